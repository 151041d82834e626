"""CPU checks of the paged KV cache: the oracle's 4-bit blocks, and what the C ABI and the Python binding
refuse before anything is launched."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

import dli_sm100 as C
from oracle import paged as R

OK, INVALID, UNSUPPORTED, WORKSPACE = 0, 1, 2, 4
F32, I64, BF16, F16, I32, FP4 = range(6)


def test_oracle_blocks_hold_their_own_values():
    """Every representable block (codes x scale with a 6 in it) comes back unchanged."""
    for s in (1, 7, 8, 55, 126):
        x = np.concatenate([R.E2M1, -R.E2M1])[None] * R.E4M3[s]
        codes, scales = R.fp4_codes(x)
        assert scales[0, 0] == s
        np.testing.assert_array_equal(R.fp4_values(codes, scales), x)


def test_oracle_ties_zeros_saturation_and_nan():
    x = np.zeros((1, 16))
    x[0, :8] = [6, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5]  # scale 1: every border, ties to the even code
    codes, scales = R.fp4_codes(x)
    assert R.E4M3[scales[0, 0]] == 1.0
    np.testing.assert_array_equal(R.E2M1[codes[0, :8]], [6, 0, 1, 1, 2, 2, 4, 4])
    np.testing.assert_array_equal(R.fp4_codes(np.zeros((2, 32)))[0], 0)
    big = np.full((1, 16), 1e9)
    np.testing.assert_array_equal(R.fp4_values(*R.fp4_codes(big)), 6 * 448.0)
    tiny = np.full((1, 16), 1e-9)
    np.testing.assert_array_equal(R.fp4_values(*R.fp4_codes(tiny)), 0.0)
    big[0, 3] = np.nan
    assert np.isnan(R.fp4_values(*R.fp4_codes(big))).all()


def test_block_bytes_round_trip():
    r = np.random.default_rng(0)
    codes, scales = r.integers(0, 16, (16, 64), np.uint8), r.integers(0, 127, (16, 4), np.uint8)
    block = R.pack_block(codes, scales)
    assert block.size == 16 * 64 * 9 // 16
    assert block[0] == codes[0, 0] | codes[0, 1] << 4 and block[16 * 32] == scales[0, 0]
    back = R.unpack_block(block, 16, 64)
    np.testing.assert_array_equal(back[0], codes)
    np.testing.assert_array_equal(back[1], scales)


def test_page_bytes():
    f = C.lib().dli_sm100_paged_kv_page_bytes
    assert f(4, 16, 128, BF16) == 4 * 16 * 128 * 2
    assert f(4, 64, 128, F32) == 4 * 64 * 128 * 4
    assert f(2, 32, 64, FP4) == 2 * 32 * 36
    for bad in ((4, 48, 128, BF16), (4, 8, 128, BF16), (4, 16, 24, FP4), (0, 16, 128, BF16), (4, 16, 128, I64)):
        assert f(*bad) == 0, bad


X = ctypes.c_void_p(4096)  # an address that no refused call follows


def append_args(**k):
    a = dict(qkv=X, cos=X, sin=X, positions=X, starts=X, table=X, q=X, kp=X, vp=X, tokens=8, batch=2, max_new=4,
             hq=4, hkv=2, d=64, pairs=32, rows=100, page=16, pages=10, most=4, ks=1.0, vs=1.0, dtype=BF16, kv=BF16,
             stream=None)
    a.update(k)
    return list(a.values())


def attend_args(**k):
    a = dict(q=X, kp=X, vp=X, positions=X, starts=X, table=X, slopes=None, out=X, tokens=8, batch=2, max_new=4, hq=4,
             hkv=2, d=64, page=16, pages=10, most=4, scale=0.0, cap=0.0, window=0, ks=1.0, vs=1.0, dtype=BF16, kv=BF16,
             ws=None, wsn=0, stream=None)
    a.update(k)
    return list(a.values())


def gather_args(**k):
    a = dict(kp=X, vp=X, table=X, first=None, lengths=None, k=X, v=X, batch=2, count=4, hkv=2, d=64, page=16, pages=10,
             most=4, ks=1.0, vs=1.0, dtype=BF16, kv=BF16, stream=None)
    a.update(k)
    return list(a.values())


COMMON = [({"page": 48}, INVALID), ({"page": 8}, INVALID), ({"hkv": 0}, INVALID), ({"d": 0}, INVALID),
          ({"batch": -1}, INVALID), ({"pages": -1}, INVALID), ({"dtype": I64, "kv": I64}, INVALID),
          ({"kv": F16}, INVALID), ({"kv": FP4, "d": 40, "pairs": 0}, INVALID), ({"kv": FP4, "ks": 0.0}, INVALID),
          ({"kv": FP4, "vs": float("nan")}, INVALID), ({"kv": FP4, "vs": float("inf")}, INVALID),
          ({"dtype": FP4, "kv": FP4}, INVALID), ({"batch": 70000, "tokens": 280000}, UNSUPPORTED),
          ({"most": 1 << 30}, UNSUPPORTED), ({"kv": FP4, "kp": ctypes.c_void_p(4104)}, INVALID),
          ({"table": None}, INVALID), ({"kp": None}, INVALID)]


@pytest.mark.parametrize("change,status", COMMON + [
    ({"tokens": -1}, INVALID), ({"positions": None}, INVALID), ({"starts": None, "tokens": 7}, INVALID),
    ({"hq": 0}, INVALID), ({"pairs": 33}, INVALID), ({"d": 63, "pairs": 1}, INVALID), ({"max_new": -1}, INVALID),
    ({"d": 1024}, UNSUPPORTED), ({"kv": FP4, "q": ctypes.c_void_p(4104)}, INVALID)])
def test_append_refusals(change, status):
    change = {k: v for k, v in change.items()}
    assert C.lib().dli_sm100_qkv_rotary_paged(*append_args(**change)) == status, C.last_error()
    assert C.last_error()


@pytest.mark.parametrize("change,status", [c for c in COMMON if "pairs" not in c[0]] + [
    ({"hq": 3}, INVALID), ({"cap": -1.0}, INVALID), ({"cap": float("nan")}, INVALID), ({"cap": float("inf")}, INVALID),
    ({"scale": float("nan")}, INVALID), ({"window": -1}, INVALID), ({"d": 320}, UNSUPPORTED),
    ({"positions": None}, INVALID), ({"starts": None, "tokens": 7}, INVALID)])
def test_attention_refusals(change, status):
    assert C.lib().dli_sm100_attention_paged(*attend_args(**change)) == status, C.last_error()
    assert C.last_error()


@pytest.mark.parametrize("change,status", [c for c in COMMON if not {"pairs", "tokens"} & set(c[0])] + [
    ({"count": -1}, INVALID), ({"batch": 60000, "hkv": 2}, UNSUPPORTED)])
def test_gather_refusals(change, status):
    assert C.lib().dli_sm100_paged_gather(*gather_args(**change)) == status, C.last_error()
    assert C.last_error()


def test_empty_calls_launch_nothing():
    L = C.lib()
    before = C.launch_count()
    assert L.dli_sm100_qkv_rotary_paged(*append_args(batch=0, tokens=0)) == OK
    assert L.dli_sm100_qkv_rotary_paged(*append_args(max_new=0, tokens=0)) == OK
    assert L.dli_sm100_attention_paged(*attend_args(tokens=0)) == OK
    assert L.dli_sm100_paged_gather(*gather_args(count=0)) == OK
    assert C.launch_count() == before


def test_binding_refuses_wrong_tensors():
    k, v = (torch.zeros(3, 2, 16, 64, dtype=torch.bfloat16) for _ in (0, 1))
    table = torch.zeros(2, 2, dtype=torch.int32)
    pos = torch.zeros(2, dtype=torch.int64)
    q = torch.zeros(2, 4, 64, dtype=torch.bfloat16)
    bad = [dict(q=q.half()), dict(q=q[0]), dict(page_table=table.long()), dict(positions=pos.int()),
           dict(positions=pos[:1]), dict(starts=pos), dict(v_pages=v[:2]), dict(k_pages=k.float()),
           dict(slopes=torch.zeros(3)), dict(out=q.float()), dict(max_new=2), dict()]  # the last: not on a GPU
    for change in bad:
        args = dict(q=q, k_pages=k, v_pages=v, positions=pos, page_table=table)
        args.update(change)
        with pytest.raises(ValueError):
            C.attention_paged(**args)
    with pytest.raises(ValueError):
        C.paged_kv_pages(4, 2, 24, 64, torch.bfloat16, device="cpu")
    with pytest.raises(ValueError):
        C.paged_kv_pages(4, 2, 16, 24, "fp4", device="cpu")
    k4, v4 = C.paged_kv_pages(4, 2, 16, 64, "fp4", device="cpu")
    assert k4.shape == (4, 2, 16 * 36) and k4.dtype == torch.uint8
    with pytest.raises(ValueError):
        C.paged_gather(k4[..., :100].contiguous(), v4[..., :100].contiguous(), table, 3, 64, torch.bfloat16)
    with pytest.raises(ValueError):
        C.qkv_rotary_paged(torch.zeros(2, 8 * 64 + 1), torch.zeros(4, 32), torch.zeros(4, 32), pos, table, k, v, 4)
