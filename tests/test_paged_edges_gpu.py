"""Paged KV cache on the GPU at the calls where a rule of its kernels ends: head counts that no CTA divides evenly,
NaN in every place and pattern, scales that underflow, rings that keep turning over bad or forgotten pages, tables
that change under a captured step, workspaces of calls with a window."""
from __future__ import annotations

import pytest
import torch

import dli_sm100 as C
import test_paged_gpu as plain
import test_paged_long_gpu as long

pytestmark = pytest.mark.gpu

BF, HF, FL = torch.bfloat16, torch.float16, torch.float32


@pytest.mark.parametrize("name", ["decode-fp4", "decode-fp4-many", "decode-f32-fp4"])
@pytest.mark.parametrize("window", [0, 1000])
def test_four_bit_rings_over_bad_and_forgotten_pages(name, window):
    """Pages outside the pool count as zeros, pages behind a window are not looked up, and what is read through the
    same ring entries afterwards keeps its bits, run after run."""
    c = long.case(name, window=window)
    table, page = c.table.clone(), c.k.shape[2] // (c.d * 9 // 16)
    zero = c.k.shape[0]
    c.k, c.v = (torch.cat([t, torch.zeros_like(t[:1])]) for t in (c.k, c.v))
    picked = [(b, p) for b, n in enumerate(c.past) for p in range(b % 3, n // page, 5)]
    for b, p in picked:
        c.table[b, p] = zero
    want = c.run()
    C.check_device_error()
    for b, p in picked:
        c.table[b, p] = (-5, zero + 1, 2 ** 31 - 1)[p % 3]
    for _ in range(20):
        assert torch.equal(c.run(), want)
        with pytest.raises(RuntimeError, match="page table"):
            C.check_device_error()
    if window:
        c.table = table
        want = c.run()
        for b, n in enumerate(c.past):
            c.table[b, :max(0, n - window + 1) // page] = -1
        for _ in range(20):
            assert torch.equal(c.run(), want)
        C.check_device_error()


def put_nan(c, pages, b, head, rows, dims, bits=None):
    """NaN (of the given float32 bits) in some dims of rows of sequence b; over 4-bit pages in the whole rows."""
    table = c.table[b].tolist()
    page = pages.shape[2] // (c.d * 9 // 16) if pages.dtype == torch.uint8 else pages.shape[2]
    for r in rows:
        block, r0 = pages[table[r // page], head], r % page
        if pages.dtype == torch.uint8:
            at = page * c.d // 2 + r0 * (c.d // 16)
            block[at:at + c.d // 16] = 0x7F
        elif bits is None:
            block[r0, dims] = float("nan")
        else:
            block.view(torch.int32)[r0, dims] = bits


SHORT = (FL, False, 6, 2, 64, 16, [70, 4, 333], [1, 1, 1])


@pytest.mark.parametrize("bits", [0x7FFFFFFF, 0xFFFFFFFF, 0x7F800001, 0x7FC00000], ids=hex)
@pytest.mark.parametrize("name", ["short", "decode-f32", "rows-f32"])
def test_float32_nan_of_every_pattern(name, bits):
    """A NaN in q, k or v (the GPU's own is 0x7FFFFFFF) makes NaN of what it reaches, and of nothing else."""
    c = long.Case(*SHORT) if name == "short" else long.case(name)
    want = c.run()
    group, new = c.hq // c.k.shape[1], c.new[0]
    signed = bits - (1 << 32) if bits >> 31 else bits
    q = c.q.clone()
    q.view(torch.int32)[0, 1, 5] = signed
    got = c.run(q=q)
    assert torch.isnan(got[0, 1]).all()
    got[0, 1] = want[0, 1]
    assert torch.equal(got, want)
    heads = slice(group, 2 * group)  # of KV head 1
    k = c.k.clone()
    put_nan(c, c.k, 0, 1, [3], slice(7, 8), signed)
    got = c.run()
    assert torch.isnan(got[:new, heads]).all()
    got[:new, heads] = want[:new, heads]
    assert torch.equal(got, want)
    c.k = k
    put_nan(c, c.v, 0, 1, [3], slice(7, 8), signed)
    got = c.run()
    C.check_device_error()
    assert torch.isnan(got[:new, heads, 7]).all()
    got[:new, heads, 7] = want[:new, heads, 7]
    assert torch.equal(got, want)


@pytest.mark.parametrize("name", ["short", "decode-f32", "rows-f32"])
def test_float32_infinities_in_the_cache(name):
    """A k of -infinity takes its key out of the rows with a positive q there; a v of infinity makes infinities, and
    so does a finite v next to the largest float, as it is."""
    c = long.Case(*SHORT) if name == "short" else long.case(name)
    group, n, past = c.hq // c.k.shape[1], c.new[0], c.past[0]
    heads = slice(group, 2 * group)
    c.q[:, :, 7] = c.q[:, :, 7].abs() + 0.25
    put_nan(c, c.k, 0, 1, [3, 40], slice(7, 8), 0xFF800000 - (1 << 32))
    got = c.run()[:n, heads]
    k, v = C.paged_gather(c.k, c.v, c.table, past + n, c.d, FL, lengths=c.lengths)
    s = torch.einsum("nhd,ld->nhl", c.q[:n, heads].double(), k[0, 1].double()) * c.d ** -0.5
    i = past + torch.arange(n, device="cuda")[:, None, None]
    s = s.masked_fill(torch.arange(past + n, device="cuda") > i, float("-inf"))
    want = torch.softmax(s, -1) @ v[0, 1].double()
    assert (s[..., 3] == float("-inf")).all() and torch.isfinite(want).all()
    torch.testing.assert_close(got.double(), want, rtol=0, atol=1e-5)
    before = c.run()
    put_nan(c, c.v, 0, 1, [5], slice(9, 10), 0x7F800000)
    put_nan(c, c.v, 0, 1, [5], slice(11, 12), 0x7F7FFFFF)
    out = c.run()
    p = torch.softmax(s, -1)[..., 5]
    assert (out[:n, heads, 9] == float("inf")).all()
    big = out[:n, heads, 11].double()
    torch.testing.assert_close(big, p * torch.finfo(FL).max, rtol=1e-4, atol=0)
    out[:n, heads, 9] = before[:n, heads, 9]
    out[:n, heads, 11] = before[:n, heads, 11]
    assert torch.equal(out, before)
    C.check_device_error()


def test_a_window_over_a_table_that_is_too_wide_to_share_out():
    """Units times the table's blocks pass an int, units times the window's do not: the workspace is of the size that
    was asked for, and the call is served."""
    hq, hkv, d, page, batch = 8, 8, 64, 128, 32
    rows, width = 8192, 4096
    new = [rows // batch] * batch
    g = torch.Generator("cuda").manual_seed(2)
    q = torch.randn(rows, hq, d, device="cuda", generator=g)
    k, v = C.paged_kv_pages(2 * batch, hkv, page, d, FL)
    k.normal_(generator=g), v.normal_(generator=g)
    table = torch.full((batch, width), -1, dtype=torch.int32, device="cuda")
    table[:, :2] = torch.randperm(2 * batch, device="cuda", generator=g).view(batch, 2)
    starts = torch.arange(batch + 1, device="cuda") * new[0]
    pos = torch.zeros(batch, dtype=torch.int64, device="cuda")
    out = C.attention_paged(q, k, v, pos, table, starts=starts, window=700)  # wider than any sequence
    want = C.attention_paged(q, k, v, pos, table[:, :2].contiguous(), starts=starts)
    C.check_device_error()
    assert torch.equal(out, want)
    assert torch.equal(C.attention_paged(q, k, v, pos, table, starts=starts), want)


@pytest.mark.parametrize("dtype,fp4,hq,hkv,d,past,new", [
    (BF, False, 48, 8, 96, [0, 5], [1, 1]),
    (BF, False, 16, 8, 192, [31, 3], [1, 1]),
    (FL, False, 24, 4, 96, [17], [1]),
    (FL, False, 32, 32, 96, [3, 0], [1, 2]),
    (FL, False, 32, 32, 96, [3, 0], [190, 30]),  # many tokens: several heads of a thread in flight
    (BF, True, 48, 8, 96, [0, 40], [1, 1]),
    (HF, True, 83, 1, 80, [9], [1]),
    (BF, True, 80, 21, 80, [0, 9], [150, 60]),
    (HF, False, 83, 1, 80, [0], [450]),
    (BF, False, 5, 1, 172, [2], [3]),  # 43 pairs of 4 bytes a row: not by 16-byte vectors
])
def test_append_of_heads_that_fill_no_cta_evenly(dtype, fp4, hq, hkv, d, past, new):
    plain.test_append(dtype, fp4, hq, hkv, d, 16, past, new, d // 2)


@pytest.mark.parametrize("dtype,hq,hkv,d", [(BF, 48, 8, 96), (HF, 16, 8, 80), (FL, 7, 2, 172)])
def test_append_of_views_off_their_alignment(dtype, hq, hkv, d):
    """The same bits as from 16-byte aligned tensors."""
    page, rows = 16, 7
    g = torch.Generator().manual_seed(3)
    qkv = torch.randn(rows, (hq + 2 * hkv) * d, generator=g).to(dtype).cuda()
    angle = (torch.rand(40, d // 2, generator=g) * 6).cuda()
    table = torch.tensor([[2, 0], [1, 3]], dtype=torch.int32, device="cuda")
    starts, pos = torch.tensor([0, 3, 7], device="cuda"), torch.tensor([14, 5], device="cuda")
    results = []
    for shift in (0, 1):
        flat = torch.empty(qkv.numel() + shift, dtype=dtype, device="cuda")[shift:]
        flat.copy_(qkv.view(-1))
        k, v = C.paged_kv_pages(4, hkv, page, d, dtype)
        q = C.qkv_rotary_paged(flat.view_as(qkv), angle.cos(), angle.sin(), pos, table, k, v, hq, starts=starts, max_new=4)
        results.append((q, k, v))
    C.check_device_error()
    for a, b in zip(*results):
        assert torch.equal(a, b) and a.abs().sum() > 0


@pytest.mark.parametrize("dtype,fp4,d,new", [(BF, False, 128, 1), (HF, False, 64, 2), (BF, True, 128, 1), (FL, False, 128, 1),
                                             (FL, True, 64, 1), (BF, False, 128, 60), (HF, True, 64, 60)])
def test_nan_that_fills_whole_parts_of_the_keys(dtype, fp4, d, new):
    """Keys 512 to 1535 of 2048, all of some shares and parts of them, score NaN in KV head 0: its rows are NaN, the
    other head's keep their bits."""
    c = long.Case(dtype, fp4, 16, 2, d, 64, [2048 - new], [new])
    want = c.run()
    put_nan(c, c.k, 0, 0, range(512, 1536), slice(0, d))
    got = c.run()
    C.check_device_error()
    assert torch.isnan(got[:, :8]).all()
    assert torch.equal(got[:, 8:], want[:, 8:])


@pytest.mark.parametrize("name", ["decode-fp4", "decode-f32-fp4", "parts-fp4", "tiles-fp4"])
@pytest.mark.parametrize("scales", [dict(k_scale=1e-12), dict(k_scale=1e-30, scale=1e-25), dict(scale=1e-45)], ids=str)
def test_scales_whose_product_underflows(name, scales):
    """Scores that underflow weigh all keys alike (a row of q of zeros has nothing else), whatever masks some of them."""
    c = long.case(name, amplitude=0.0, window=300, softcap=0.0)
    want = c.run()
    c.check(want)
    c.options.update(scales)
    assert torch.equal(c.run(), want)
    C.check_device_error()


@pytest.mark.parametrize("name", ["decode", "decode-f32", "parts", "tiles-bf16"])
def test_the_smallest_scale(name):
    c = long.case(name, amplitude=0.0)
    want = c.run()
    c.options.update(scale=1e-45)
    assert torch.equal(c.run(), want)
    C.check_device_error()


def test_a_warm_up_that_fails_leaves_the_open_sequences_their_pages():
    import test_paged_model_gpu as model

    shape = model._small()
    r = model._runner(shape, page_size=16, num_pages=8)
    r.open([40, 20])
    held = r.page_table(2).clone()
    step = r._step

    def fail(*a, **k):
        raise RuntimeError("out of memory")

    r._step = fail
    for call in (r.decode_graph, lambda n: r.profile_decode_step(n, None)):
        with pytest.raises(RuntimeError, match="out of memory"):
            call(2)
        assert torch.equal(r.page_table(2), held)
    r._step = step
    r.decode_graph(2)
    assert torch.equal(r.page_table(2), held)
    r.release_graphs()


@pytest.mark.parametrize("name", ["decode-many", "decode-fp4-many", "decode-f32", "parts"])
def test_a_captured_call_follows_pages_that_move(name):
    """Positions grow and pages move (their old places turn to NaN) between replays: the eager call's bits before the
    move."""
    c = long.case(name)
    positions = c.positions.clone()
    eager = []
    cuts = (200, 64, 63, 1, 0)
    for cut in cuts:
        c.positions.copy_((positions - cut).clamp_min(0))
        eager.append(c.run())
    out = torch.empty_like(c.q)
    c.run(out=out)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        c.run(out=out)
    held = set(c.table.flatten().tolist())
    spare = [p for p in range(c.k.shape[0]) if p not in held]
    for turn, cut in enumerate(cuts):
        for i in range(len(spare)):
            b, p = i % len(c.past), (turn + i) % 3 if c.past[i % len(c.past)] > 48 * 3 else 0
            old = int(c.table[b, p])
            if old < 0:
                continue
            for t in (c.k, c.v):
                t[spare[i]] = t[old]
                t[old] = 0xFF if t.dtype == torch.uint8 else float("nan")
            c.table[b, p] = spare[i]
            spare[i] = old
        c.positions.copy_((positions - cut).clamp_min(0))
        g.replay()
        assert torch.equal(out, eager[turn])
    C.check_device_error()


@pytest.mark.parametrize("fp4", [False, True], ids=["rows16", "rows4"])
def test_a_batch_of_almost_only_idle_sequences(fp4):
    """As many items as the grid may have, nearly all of them empty: none of the kernel's warps gives up waiting."""
    batch, hq, rows, d = 65535, 128, 16384, 64  # a tile is one token
    g = torch.Generator("cuda").manual_seed(3)
    k, v = C.paged_kv_pages(4, 1, 16, d, "fp4" if fp4 else BF)
    one = torch.ones(64, d // 2, device="cuda")
    table = torch.zeros(batch, 2, dtype=torch.int32, device="cuda")
    table[0], table[-1] = torch.tensor([1, 2]), torch.tensor([3, 0])
    qkv = torch.randn(40, (hq + 2) * d, device="cuda", generator=g).to(BF)
    starts = torch.full((batch + 1,), 20, dtype=torch.int64, device="cuda")
    starts[0], starts[-1] = 0, 40
    pos = torch.zeros(batch, dtype=torch.int64, device="cuda")
    q = torch.zeros(rows, hq, d, dtype=BF, device="cuda")
    q[:40] = C.qkv_rotary_paged(qkv, one, one * 0, pos, table, k, v, hq, starts=starts)
    two = torch.tensor([0, batch - 1], device="cuda")
    want = C.attention_paged(q[:40], k, v, pos[:2], table[two].contiguous(), max_new=20)
    got = C.attention_paged(q, k, v, pos, table, starts=starts)
    C.check_device_error()
    assert torch.equal(got[:40], want)
