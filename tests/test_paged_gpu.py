"""GPU parity of the paged KV-cache entry points (append with rotary, gather, attention) against the 64-bit
oracle in oracle/paged.py.

Every cached row outside the sequences is NaN (4-bit: NaN scales), table entries past a sequence are -1, pages
are in random order. Bounds, u = eps/2 of the type that is rounded to:
  append   q and 16-bit k: one rounding, u |x|, plus 4 fp32 roundings of |a c| + |b s|; v and 4-bit pages: exact
  attend   with A = sum p|v| and S = the largest scale * sum |q||k| of the row:
           output rounding u |o|, P rounded to u_p gives u_p A, scores off by e = (D + 16) 2^-24 S (dot products in
           fp32, the cap and bias included) change p by at most 2 e relative (p and its sum): 2 e A; sums over keys
           in fp32, relative (keys/16 + 40) 2^-24 A (kernels add keys in chains of at most 1/16 of them, plus merges).
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

import dli_sm100 as C
from oracle import paged as R

pytestmark = pytest.mark.gpu

BF, HF, FL = torch.bfloat16, torch.float16, torch.float32
IDS = {BF: "bf16", HF: "f16", FL: "f32"}


def unit(dtype):
    return torch.finfo(dtype).eps / 2


class Pool:
    """Sequences of float64 rows (as the cache holds them) in randomly ordered GPU pages."""

    def __init__(self, seed, lengths, hkv, d, page, dtype, fp4=False, extra=3, grow=0):
        r = np.random.default_rng(seed)
        self.hkv, self.d, self.page, self.dtype, self.fp4 = hkv, d, page, dtype, fp4
        need = [-(-(n + grow) // page) for n in lengths]
        self.pages = sum(need) + extra
        order = r.permutation(self.pages)
        self.table = np.full((len(lengths), max(need + [1]) + 1), -1, np.int32)
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = order[at:at + n]
            at += n
        self.rows = [[], []]
        self.host = []
        for which in (0, 1):
            if fp4:
                host = np.full((self.pages, hkv, page * d * 9 // 16), 0xFF, np.uint8)
            else:
                host = np.full((self.pages, hkv, page, d), np.nan)
            for b, n in enumerate(lengths):
                x = r.standard_normal((hkv, n, d)) * (0.3 + r.random((hkv, 1, d)) * 1.4)
                if fp4:
                    codes, scales = R.fp4_codes(x)
                    x = R.fp4_values(codes, scales)
                    for h in range(hkv):
                        for p0 in range(0, n, page):
                            k = min(page, n - p0)
                            full = np.full((page, d), 0xF, np.uint8), np.full((page, d // 16), 0xFF, np.uint8)
                            full[0][:k], full[1][:k] = codes[h, p0:p0 + k], scales[h, p0:p0 + k]
                            host[self.table[b, p0 // page], h] = R.pack_block(*full)
                else:
                    x = torch.from_numpy(x).to(dtype).double().numpy()
                    for p0 in range(0, n, page):
                        k = min(page, n - p0)
                        host[self.table[b, p0 // page], :, :k] = x[:, p0:p0 + k]
                self.rows[which].append(x)
            self.host.append(host)
        self.k, self.v = (self.up(h) for h in self.host)
        self.gpu_table = torch.from_numpy(self.table).cuda()

    def up(self, host):
        t = torch.from_numpy(host)
        return (t if self.fp4 else t.to(self.dtype)).cuda()

    def read(self, pages, b, p):
        """(codes, scales) or float64 values [Hkv, D] of row p of sequence b."""
        block = pages[self.table[b, p // self.page]]
        if not self.fp4:
            return block[:, p % self.page]
        got = [R.unpack_block(x, self.page, self.d) for x in block]
        return np.stack([g[0][p % self.page] for g in got]), np.stack([g[1][p % self.page] for g in got])


def down(t):
    return t.cpu().numpy() if t.dtype == torch.uint8 else t.cpu().double().numpy()


def ragged(new, pad=0):
    starts = np.concatenate([[0], np.cumsum(new)]).astype(np.int64)
    return torch.from_numpy(starts).cuda(), int(starts[-1]) + pad


def dev64(x):
    return torch.tensor(x, dtype=torch.int64, device="cuda")


# ---- append ------------------------------------------------------------------------------------

APPEND = [  # dtype, fp4, hq, hkv, d, page, past, new, pairs
    (BF, False, 28, 4, 128, 16, [0, 5, 16, 31], [1, 1, 1, 1], 64),
    (HF, False, 14, 2, 64, 32, [0, 70, 3], [40, 0, 7], 32),
    (FL, False, 4, 4, 96, 64, [63, 0], [2, 130], 48),
    (BF, False, 3, 1, 80, 128, [1], [1], 24),
    (HF, False, 5, 5, 20, 16, [0, 9], [3, 8], 10),
    (FL, False, 2, 1, 6, 16, [15], [2], 2),
    (BF, False, 37, 5, 256, 16, [100], [17], 128),
    (BF, True, 28, 4, 128, 16, [0, 5, 16, 31], [1, 1, 1, 1], 64),
    (HF, True, 14, 2, 64, 32, [0, 70, 3], [40, 0, 7], 32),
    (FL, True, 4, 2, 96, 64, [63, 0], [2, 130], 40),
    (BF, True, 2, 1, 16, 128, [127], [3], 8),
]


@pytest.mark.parametrize("dtype,fp4,hq,hkv,d,page,past,new,pairs", APPEND,
                         ids=[f"{IDS[a[0]]}{'-fp4' if a[1] else ''}-h{a[2]}.{a[3]}-d{a[4]}-p{a[5]}" for a in APPEND])
def test_append(dtype, fp4, hq, hkv, d, page, past, new, pairs):
    pad = 2
    pool = Pool(1, past, hkv, d, page, dtype, fp4, grow=max(new))
    starts, tokens = ragged(new, pad)
    g = torch.Generator().manual_seed(2)
    qkv = (torch.randn(tokens, (hq + 2 * hkv) * d, generator=g) * 1.5).to(dtype)
    rows = max(p + n for p, n in zip(past, new))
    angle = np.outer(np.arange(rows), 1e4 ** (-np.arange(pairs) / pairs))
    cos, sin = np.cos(angle).astype(np.float32), np.sin(angle).astype(np.float32)
    q_out = torch.full((tokens, hq, d), 7.0, dtype=dtype, device="cuda")
    scales = dict(k_scale=0.5, v_scale=0.3) if fp4 and dtype == HF else {}
    C.qkv_rotary_paged(qkv.cuda(), torch.from_numpy(cos).cuda(), torch.from_numpy(sin).cuda(), dev64(past),
                       pool.gpu_table, pool.k, pool.v, hq, starts=starts, max_new=max(new), q_out=q_out, **scales)
    C.check_device_error()
    q, kp, vp = down(q_out), down(pool.k), down(pool.v)
    want_k, want_v = (down(pool.up(h)) for h in pool.host)
    x = qkv.double().numpy().reshape(tokens, hq + 2 * hkv, d)
    row = 0
    for b, (p0, n) in enumerate(zip(past, new)):
        for i in range(n):
            p = p0 + i
            c, s = cos[p:p + 1], sin[p:p + 1]
            r = R.rotate(x[row:row + 1, :hq + hkv], c, s)[0]
            size = R.rotate(np.abs(x[row:row + 1, :hq + hkv]), np.abs(c), -np.abs(s))[0]
            size = np.maximum(size, R.rotate(np.abs(x[row:row + 1, :hq + hkv]), np.abs(c), np.abs(s))[0])
            tol = unit(dtype) * np.abs(r) + 4 * 2.0 ** -24 * np.abs(size) + 1e-7 * (dtype == HF)
            assert (np.abs(q[row] - r[:hq]) <= tol[:hq]).all()
            vrow = x[row, hq + hkv:]
            at, pr = pool.table[b, p // page], p % page
            if fp4:
                for got, val, ks in ((kp, r[hq:], scales.get("k_scale", 1.0)), (vp, vrow, scales.get("v_scale", 1.0))):
                    codes, sc = pool.read(got, b, p)
                    wc, ws = R.fp4_codes(val, float(np.float32(ks)))
                    np.testing.assert_array_equal(sc, ws)
                    np.testing.assert_array_equal(codes, wc)
                for got, want in ((kp, want_k), (vp, want_v)):
                    for h in range(hkv):
                        cut = page * d // 2
                        want[at, h, pr * d // 2:(pr + 1) * d // 2] = got[at, h, pr * d // 2:(pr + 1) * d // 2]
                        want[at, h, cut + pr * d // 16:cut + (pr + 1) * d // 16] = \
                            got[at, h, cut + pr * d // 16:cut + (pr + 1) * d // 16]
            else:
                assert (np.abs(kp[at, :, pr] - r[hq:]) <= tol[hq:]).all()
                np.testing.assert_array_equal(vp[at, :, pr], vrow)
                want_k[at, :, pr], want_v[at, :, pr] = kp[at, :, pr], vp[at, :, pr]
            row += 1
    # every other cached row, and the rows behind the last sequence, are as they were
    np.testing.assert_array_equal(kp, want_k)
    np.testing.assert_array_equal(vp, want_v)
    assert (q[row:] == 7).all()


def test_append_fp4_borders_and_special_values():
    """v is quantised as it stands: ties at every border, zeros, saturation, infinities, a NaN block."""
    hq, hkv, d, page = 1, 1, 128, 16
    v = np.zeros(d)
    v[:8] = [6, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5]
    v[8:16] = [-6, -0.25, -0.75, -1.25, -1.75, -2.5, -3.5, -5]
    v[16:32] = 3e38
    v[32] = np.inf
    v[48], v[49] = np.nan, 1.0
    v[64:80] = 1e-30
    v[80:96] = 6 * 2.0 ** -10  # half way between the scales 0 and 2^-9: the even code 0
    v[96:112] = 6 * 1.5 * 2.0 ** -9  # half way between 1 and 2 (x 2^-9)
    v[112:128] = np.arange(16) - 8
    qkv = torch.zeros(1, 3 * d)
    qkv[0, 2 * d:] = torch.from_numpy(v).float()
    pool = Pool(3, [0], hkv, d, page, FL, True, grow=1)
    cos, sin = torch.ones(1, d // 2, device="cuda"), torch.zeros(1, d // 2, device="cuda")
    C.qkv_rotary_paged(qkv.cuda(), cos, sin, dev64([0]), pool.gpu_table, pool.k, pool.v, hq)
    codes, scales = pool.read(down(pool.v), 0, 0)
    wc, ws = R.fp4_codes(qkv[0, 2 * d:].double().numpy()[None])
    np.testing.assert_array_equal(scales, ws)
    keep = np.repeat(ws != 127, 16, -1)
    np.testing.assert_array_equal(np.where(keep, codes, 0), np.where(keep, wc, 0))
    k, got = C.paged_gather(pool.k, pool.v, pool.gpu_table, 1, d, FL)
    assert torch.isnan(got[0, 0, 0, 48:64]).all() and torch.isfinite(got[0, 0, 0, :48]).all()
    assert (k == 0).all()


def test_append_reports_positions_pages_and_rows_out_of_bounds():
    hq, hkv, d, page = 2, 1, 64, 16
    cos, sin = torch.ones(64, 32, device="cuda"), torch.zeros(64, 32, device="cuda")
    qkv = torch.ones(4, 4 * d, device="cuda", dtype=BF)

    def call(table, past, starts, cos=cos, max_new=2, match=None):
        k, v = C.paged_kv_pages(4, hkv, page, d, BF)
        q = torch.full((4, hq, d), 9.0, device="cuda", dtype=BF)
        C.qkv_rotary_paged(qkv, cos, cos * 0, dev64(past), torch.tensor(table, dtype=torch.int32, device="cuda"), k, v,
                           hq, starts=dev64(starts), max_new=max_new, q_out=q)
        if match:
            with pytest.raises(RuntimeError, match=match):
                C.check_device_error()
        C.check_device_error()
        return q, k, v

    # a page outside the pool: q is written, the page's rows are not
    q, k, v = call([[0, 1], [4, 2]], [0, 3], [0, 2, 4], match="page table entry")
    assert (q == 1).all() and k[0, 0, :2].eq(1).all() and k.sum() == 2 * d and v.sum() == 2 * d
    # past the table: the sequence is skipped
    q, k, v = call([[0, 1], [3, 2]], [0, 31], [0, 2, 4], match="capacity")
    assert (q[:2] == 1).all() and (q[2:] == 9).all() and k.sum() == 2 * d
    for starts in ([0, 3, 4], [0, 2, 5], [0, -1, 4], [2, 0, 2]):
        q, k, v = call([[0, 1], [3, 2]], [0, 0], starts, match="row starts")
    # a position past the cos/sin table: reported, not rotated
    q, k, v = call([[0, 1], [3, 2]], [0, 5], [0, 2, 4], cos=cos[:6].contiguous() * 0.5, match="cos/sin")
    assert (q[:3] == 0.5).all() and (q[3] == 1).all() and k[3, 0, 6].eq(1).all()


# ---- gather ------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype,fp4,d,page", [(BF, False, 128, 16), (HF, False, 20, 64), (FL, False, 64, 32),
                                              (BF, True, 128, 16), (HF, True, 64, 128), (FL, True, 48, 32)])
def test_gather(dtype, fp4, d, page):
    lengths = [37, 1, 130, 0]
    pool = Pool(4, lengths, 3, d, page, dtype, fp4)
    first = [0, 0, 125, 0]
    count = 40
    ks, vs = (0.25, 3.0) if fp4 else (1.0, 1.0)
    # sequence 0 ends inside the rows asked for, 2 reads its last 5 rows
    k, v = C.paged_gather(pool.k, pool.v, pool.gpu_table, count, d, dtype, first=dev64(first), lengths=dev64(lengths),
                          k_scale=ks, v_scale=vs)
    C.check_device_error()
    for got, rows, scale in ((down(k), pool.rows[0], ks), (down(v), pool.rows[1], vs)):
        for b, n in enumerate(lengths):
            want = np.zeros((3, count, d))
            part = rows[b][:, first[b]:first[b] + count] * scale
            want[:, :part.shape[1]] = part
            want = torch.from_numpy(want).float().to(dtype).double().numpy()
            np.testing.assert_array_equal(got[b], want)
    with pytest.raises(RuntimeError, match="page table"):  # no lengths: the table's -1 entries are reached
        C.paged_gather(pool.k, pool.v, pool.gpu_table, count, d, dtype)
        C.check_device_error()


# ---- attention ---------------------------------------------------------------------------------

def check_attention(got, pool, past, new, q, scale, softcap=0.0, window=0, slopes=None, p_unit=None, k_scale=1.0,
                    v_scale=1.0):
    dtype, d = q.dtype, q.shape[-1]
    x = q.double().cpu().numpy()
    p_unit = p_unit if p_unit is not None else (0.0 if dtype == FL else unit(dtype))
    row = 0
    for b, (p0, n) in enumerate(zip(past, new)):
        if n:
            o, mass, size = R.attention(x[row:row + n], pool.rows[0][b] * k_scale, pool.rows[1][b] * v_scale, p0,
                                        scale or d ** -0.5, softcap, window, slopes)
            e = (d + 16) * 2.0 ** -24 * size[..., None]
            keys = min(p0 + n, window or 1 << 60)
            tol = unit(dtype) * np.abs(o) + (p_unit + 2 * e + (keys / 16 + 40) * 2.0 ** -24) * mass * 1.01
            tol += 2.0 ** -24 * (dtype == HF)
            off = np.abs(got[row:row + n] - o)
            assert np.isfinite(got[row:row + n]).all(), f"sequence {b}: not finite"
            assert (off <= tol).all(), f"sequence {b}: off by {(off / tol).max():.2f} of the bound"
        row += n


ATTEND = [  # dtype, fp4, hq, hkv, d, page, past, new, options
    (BF, False, 28, 4, 128, 16, [0, 15, 16, 700, 64], [1, 1, 1, 1, 0], {}),
    (HF, False, 14, 2, 64, 32, [31, 333], [1, 1], {}),
    (HF, False, 8, 8, 64, 64, [63, 64, 65], [1, 1, 1], {"window": 40}),
    (BF, False, 64, 8, 128, 128, [1500, 2], [1, 1], {"softcap": 20.0}),
    (BF, False, 16, 1, 128, 64, [257, 90], [1, 1], {"slopes": True}),
    (HF, False, 40, 1, 64, 16, [129], [1], {"slopes": True, "softcap": 30.0, "window": 70}),
    (BF, False, 28, 4, 128, 16, [200, 0, 77], [2, 2, 1], {}),
    (HF, False, 8, 2, 128, 32, [100, 3], [4, 3], {"window": 3}),
    (BF, False, 4, 4, 64, 16, [500], [8], {"softcap": 5.0, "slopes": True}),
    (BF, False, 28, 4, 128, 64, [0, 0, 0], [129, 20, 65], {}),
    (HF, False, 14, 2, 64, 16, [0, 300, 5], [200, 31, 0], {}),
    (BF, False, 4, 4, 64, 32, [100, 0], [140, 300], {"window": 64}),
    (HF, False, 6, 2, 128, 128, [64, 200], [70, 33], {"softcap": 8.0}),
    (BF, False, 8, 1, 128, 16, [10, 40], [50, 20], {"slopes": True, "window": 33, "softcap": 25.0}),
    (BF, False, 130, 1, 64, 16, [40], [5], {}),
    (FL, False, 16, 4, 128, 16, [0, 90, 333], [1, 1, 1], {}),
    (FL, False, 14, 2, 64, 32, [0, 61], [33, 5], {"softcap": 10.0}),
    (FL, False, 4, 2, 96, 16, [50], [7], {"window": 20, "slopes": True}),
    (FL, False, 9, 3, 256, 64, [70], [1], {}),
    (BF, False, 6, 3, 80, 16, [20, 0], [3, 18], {}),
    (HF, False, 2, 1, 7, 16, [33], [2], {"window": 5}),
    (BF, True, 28, 4, 128, 16, [0, 15, 16, 700, 64], [1, 1, 1, 1, 0], {}),
    (HF, True, 14, 2, 64, 32, [31, 333], [1, 1], {"k_scale": 0.5, "v_scale": 3.0}),
    (BF, True, 64, 8, 128, 64, [1500, 2], [1, 1], {"softcap": 20.0}),
    (HF, True, 8, 8, 64, 128, [63, 200, 65], [1, 1, 1], {"window": 40}),
    (BF, True, 16, 1, 128, 64, [257, 90], [1, 1], {"slopes": True}),
    (BF, True, 28, 4, 128, 16, [200, 0, 77], [2, 2, 1], {}),
    (BF, True, 28, 4, 128, 32, [90, 0], [40, 129], {}),
    (HF, True, 14, 2, 64, 16, [0, 300, 5], [200, 31, 0], {"softcap": 15.0, "v_scale": 0.5}),
    (FL, True, 8, 2, 64, 16, [77, 3], [1, 20], {}),
    (BF, True, 4, 2, 96, 16, [40], [3], {}),
]


@pytest.mark.parametrize("dtype,fp4,hq,hkv,d,page,past,new,opt", ATTEND, ids=[
    f"{i}-{IDS[a[0]]}{'-fp4' if a[1] else ''}-h{a[2]}.{a[3]}-d{a[4]}-p{a[5]}-n{max(a[7])}" for i, a in enumerate(ATTEND)])
def test_attention(dtype, fp4, hq, hkv, d, page, past, new, opt):
    opt = dict(opt)
    pool = Pool(5, [p + n for p, n in zip(past, new)], hkv, d, page, dtype, fp4)
    starts, tokens = ragged(new, 3)
    q = (torch.randn(tokens, hq, d, generator=torch.Generator().manual_seed(6)) * 1.3).to(dtype)
    slopes = None
    if opt.pop("slopes", False):
        slopes = (2.0 ** (-8.0 * np.arange(1, hq + 1) / hq)).astype(np.float32)
    out = torch.full_like(q, 5.0, device="cuda")
    C.attention_paged(q.cuda(), pool.k, pool.v, dev64(past), pool.gpu_table, starts=starts, max_new=max(new),
                      slopes=None if slopes is None else torch.from_numpy(slopes).cuda(), out=out, **opt)
    C.check_device_error()
    got = down(out)
    check_attention(got, pool, past, new, q, 0.0, slopes=slopes, **opt)
    assert (got[sum(new):] == 5).all()  # rows behind the last sequence


def test_attention_equal_rows_without_starts_and_a_given_scale():
    past, new = [40, 7, 100], [2, 2, 2]
    pool = Pool(7, [p + n for p, n in zip(past, new)], 2, 128, 16, BF)
    q = torch.randn(6, 8, 128, generator=torch.Generator().manual_seed(8)).to(BF)
    out = C.attention_paged(q.cuda(), pool.k, pool.v, dev64(past), pool.gpu_table, scale=0.2)
    C.check_device_error()
    check_attention(down(out), pool, past, new, q, 0.2)


@pytest.mark.parametrize("fp4,new", [(False, 1), (False, 40), (True, 1), (True, 40)])
def test_attention_reports_bad_pages_positions_and_rows(fp4, new):
    """Sequence 1 is wrong in each case; sequence 0 keeps its result."""
    past = [50, 60]
    pool = Pool(9, [p + new for p in past], 2, 64, 16, BF, fp4)
    q = torch.randn(2 * new, 4, 64, generator=torch.Generator().manual_seed(10)).to(BF)

    def call(match, past=past, table=pool.gpu_table, starts=(0, new, 2 * new)):
        out = torch.full_like(q, 5.0, device="cuda")
        C.attention_paged(q.cuda(), pool.k, pool.v, dev64(past), table, starts=dev64(starts), max_new=new, out=out)
        with pytest.raises(RuntimeError, match=match):
            C.check_device_error()
        check_attention(down(out)[:new], pool, [50], [new], q[:new], 0.0, p_unit=unit(BF))
        return out

    bad = pool.gpu_table.clone()
    bad[1, 1] = pool.pages
    call("page table", table=bad)
    bad[1, 1] = -7
    call("page table", table=bad)
    assert (call("capacity", past=[50, 100000])[new:] == 5).all()
    assert (call("capacity", past=[50, -1])[new:] == 5).all()
    assert (call("row starts", starts=(0, new, 2 * new + 1))[new:] == 5).all()
    assert (call("row starts", starts=(0, new, new - 1))[new:] == 5).all()


def test_append_then_attend_as_one_decode_loop():
    """A prompt and four steps of three ragged sequences, one of them idle at times, both cache types, captured steps
    replayed: the cache ends with the rows of the oracle's, and every step's output is the oracle's."""
    hq, hkv, d, page = 14, 2, 64, 16
    cos, sin = (torch.from_numpy(f(np.outer(np.arange(200), 1e4 ** (-np.arange(32) / 32))).astype(np.float32))
                for f in (np.cos, np.sin))
    for fp4 in (False, True):
        pool = Pool(11, [0, 0, 0], hkv, d, page, HF, fp4, grow=150)
        pool.k.zero_(), pool.v.zero_()
        g = torch.Generator().manual_seed(12)
        past = [0, 0, 0]
        rows = [[np.zeros((hkv, 0, d))] * 3, [np.zeros((hkv, 0, d))] * 3]
        for new in ([70, 33, 1], [1, 1, 1], [1, 0, 1], [1, 1, 0], [2, 1, 3]):
            starts, tokens = ragged(new)
            qkv = (torch.randn(tokens, (hq + 2 * hkv) * d, generator=g)).to(HF)
            pos = dev64(past)

            def step(qkv=qkv.cuda(), pos=pos, starts=starts, most=max(new)):
                q = C.qkv_rotary_paged(qkv, cos.cuda(), sin.cuda(), pos, pool.gpu_table, pool.k, pool.v, hq,
                                       starts=starts, max_new=most)
                return q, C.attention_paged(q, pool.k, pool.v, pos, pool.gpu_table, starts=starts, max_new=most)

            q, out = step()
            torch.cuda.synchronize()
            C.check_device_error()
            ck, cv = C.paged_gather(pool.k, pool.v, pool.gpu_table, 150, d, HF,
                                    lengths=dev64([p + n for p, n in zip(past, new)]))
            x = qkv.double().numpy().reshape(tokens, hq + 2 * hkv, d)
            row = 0
            for b, n in enumerate(new):
                past[b] += n
                r = R.rotate(x[row:row + n, hq:hq + hkv], cos.numpy()[past[b] - n:past[b]], sin.numpy()[past[b] - n:past[b]])
                for which, (val, got) in enumerate(((r, ck), (x[row:row + n, hq + hkv:], cv))):
                    if fp4 and n:
                        val = R.fp4_values(*R.fp4_codes(val))
                    rows[which][b] = np.concatenate([rows[which][b], val.transpose(1, 0, 2)], 1)
                    have = down(got)[b][:, :past[b]]
                    assert (np.abs(have - rows[which][b]) <= 2.0 ** -11 * np.abs(rows[which][b]) + 1e-6).all()
                    rows[which][b] = have  # 16-bit k: as rounded
                row += n
            pool.rows = rows
            check_attention(down(out), pool, [p - n for p, n in zip(past, new)], new, q, 0.0)
