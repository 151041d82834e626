"""Paged attention at the sizes where its kernels split, share and hand out work: long caches, many tiles, keys in
parts, rings that wrap many times; relaunches, streams, captured graphs, views; values at the ends of the types.

The reference is a plain attention in 64 bits on the device over the rows that paged_gather returns in fp32 (exact
for every page type; tested on its own against unpacked pages). Bounds, u = eps/2 of the type that is rounded to,
A = sum p|v|, S = the largest scale * sum |q||k| of a row: output u |o|; P rounded to u_p: u_p A; scores off by
e = (D + 16) 2^-24 S: 2 e A; sums over keys in fp32, chains of at most 1/16 of the keys plus merges:
(keys / 16 + 40) 2^-24 A. P in half precision (4-bit pages, and half-precision models): below 2^-14 its steps are
2^-24 wide, so a P_j = exp(x_j - m) is off by up to 2^-25 or by itself. m is at most the row's maximum, so the sum
l that it is divided by is at least 1, and key j is off by at most min(p_j, 2^-25) |v_j| in the output. That counts
where the keys that carry the row have a zero in some dim (4-bit values often do): A is then tiny there as well.
"""
from __future__ import annotations

import pytest
import torch

import dli_sm100 as C

pytestmark = pytest.mark.gpu

BF, HF, FL = torch.bfloat16, torch.float16, torch.float32
IDS = {BF: "bf16", HF: "f16", FL: "f32"}


def unit(dtype):
    return torch.finfo(dtype).eps / 2


class Case:
    """A batch with everything that a call needs: cached rows in randomly ordered pages of a pool whose other pages
    hold NaN, written by the append itself."""

    def __init__(self, dtype, fp4, hq, hkv, d, page, past, new, seed=1, slopes=False, amplitude=1.0, **options):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.dtype, self.hq, self.d, self.past, self.new, self.options = dtype, hq, d, past, new, options
        need = [-(-(p + n) // page) for p, n in zip(past, new)]
        pages = sum(need) + 2
        order = torch.randperm(pages, generator=g, device="cuda").int()
        self.table = torch.full((len(past), max(need) + 1), -1, dtype=torch.int32, device="cuda")
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = order[at:at + n]
            at += n
        self.k, self.v = C.paged_kv_pages(pages, hkv, page, d, "fp4" if fp4 else dtype)
        for t in (self.k, self.v):
            t.fill_(0xFF if fp4 else float("nan"))
        self.lengths = torch.tensor([p + n for p, n in zip(past, new)], device="cuda")
        starts = torch.cumsum(torch.tensor([0] + list(self.lengths.tolist())), 0).cuda()
        rows = int(starts[-1])
        qkv = torch.empty(rows, (hq + 2 * hkv) * d, dtype=dtype, device="cuda").normal_(generator=g)
        one = torch.ones(int(self.lengths.max()), 1, device="cuda")
        C.qkv_rotary_paged(qkv, one, one * 0, torch.zeros_like(self.lengths), self.table, self.k, self.v, hq,
                           starts=starts, max_new=int(self.lengths.max()))
        C.check_device_error()
        self.tokens = sum(new)
        self.q = (torch.randn(self.tokens, hq, d, generator=g, device="cuda") * amplitude).to(dtype)
        self.starts = torch.cumsum(torch.tensor([0] + list(new)), 0).cuda()
        self.positions = torch.tensor(past, device="cuda")
        self.slopes = (2.0 ** (-8.0 * torch.arange(1, hq + 1, device="cuda") / hq)).float() if slopes else None

    def run(self, **kw):
        kw = {"q": self.q, "table": self.table, **kw}
        return C.attention_paged(kw["q"], self.k, self.v, self.positions, kw["table"], starts=self.starts,
                                 max_new=max(self.new), slopes=self.slopes, out=kw.get("out"), **self.options)

    def check(self, got, rows=None):
        k, v = C.paged_gather(self.k, self.v, self.table, int(self.lengths.max()), self.d, FL if self.k.dtype == torch.uint8 else self.dtype,
                              lengths=self.lengths)
        group = self.hq // k.shape[1]
        u, row = unit(self.dtype), 0
        p_unit = 0.0 if self.dtype == FL else unit(HF if self.k.dtype == torch.uint8 and self.dtype == HF else self.dtype)
        for b, (past, new) in enumerate(zip(self.past, self.new)):
            for at in range(0, new, 256):
                n = min(256, new - at)
                x = self.q[row + at:row + at + n].double().transpose(0, 1).unflatten(0, (k.shape[1], group))
                kk, vv = k[b, :, :past + new].double()[:, None], v[b, :, :past + new].double()[:, None]
                s = (x @ kk.transpose(-1, -2)) * self.d ** -0.5
                size = (x.abs() @ kk.abs().transpose(-1, -2)) * self.d ** -0.5
                i = torch.arange(past + at, past + at + n, device="cuda")[:, None]
                j = torch.arange(past + new, device="cuda")[None]
                if self.options.get("softcap"):
                    s = self.options["softcap"] * torch.tanh(s / self.options["softcap"])
                seen = j <= i
                if self.options.get("window"):
                    seen &= j > i - self.options["window"]
                if self.slopes is not None:
                    bias = self.slopes.double().view(-1, group, 1, 1) * (j - i)
                    s = s + bias
                    size = size + bias.abs()
                size = size.masked_fill(~seen, 0).amax(-1, keepdim=True)
                p = torch.softmax(s.masked_fill(~seen, float("-inf")), -1)
                o, mass = p @ vv, p @ vv.abs()
                small = p.clamp(max=2.0 ** -25) @ vv.abs() * (self.dtype == HF or self.k.dtype == torch.uint8)
                e = (self.d + 16) * 2.0 ** -24 * size
                keys = min(past + new, self.options.get("window") or 1 << 60)
                tol = u * o.abs() + (p_unit + 2 * e + (keys / 16 + 40) * 2.0 ** -24) * mass * 1.01 + small + 2.0 ** -24 * (self.dtype == HF)
                have = got[row + at:row + at + n].double().transpose(0, 1).unflatten(0, (k.shape[1], group))
                assert torch.isfinite(have).all(), f"sequence {b}: not finite"
                off = (have - o).abs()
                assert (off <= tol).all(), f"sequence {b}: off by {(off / tol).max().item():.2f} of the bound"
            row += new


LONG = {
    # more tiles than the GPU holds at a time: the scheduler hands them out
    "tiles-bf16": (BF, False, 28, 4, 128, 16, [0, 1000, 300, 0, 17, 900], [700, 300, 511, 64, 640, 1]),
    "tiles-f16-window-cap": (HF, False, 16, 16, 64, 32, [0, 500, 100], [900, 333, 128], {"window": 300, "softcap": 20.0}),
    "tiles-fp4": (BF, True, 28, 4, 128, 32, [0, 1000, 300, 17], [700, 300, 511, 640]),
    "tiles-fp4-slopes": (HF, True, 14, 2, 64, 64, [0, 400, 33, 80], [1200, 800, 900, 700], {"slopes": True}),
    # few tiles: keys in many parts
    "parts": (BF, False, 28, 4, 128, 16, [5000, 30, 0], [60, 20, 33]),
    "parts-window": (HF, False, 14, 2, 64, 64, [3000, 9000], [70, 129], {"window": 2500, "slopes": True}),
    "parts-fp4": (BF, True, 28, 4, 128, 64, [4100, 333, 12], [40, 17, 0], {"softcap": 30.0}),
    # some waves of tiles over long keys: parts of long sequences, whole tiles of short ones
    "long-parts": (BF, False, 28, 4, 128, 64, [4000, 7200, 100, 0], [200, 180, 150, 66]),
    "long-parts-fp4": (HF, True, 14, 2, 64, 128, [3600, 9000, 70, 3601], [500, 512, 300, 1]),
    # decode: one share of the blocks for every CTA
    "decode": (BF, False, 28, 4, 128, 16, [30000, 511, 0, 7777], [1, 1, 1, 0]),
    "decode-many": (HF, False, 32, 8, 64, 32, [100 + 37 * i for i in range(60)], [1] * 60),
    "decode-two-tokens": (BF, False, 28, 4, 128, 128, [9000, 2500], [2, 2], {"slopes": True, "softcap": 15.0}),
    "decode-window": (HF, False, 8, 2, 128, 64, [20000, 100], [1, 1], {"window": 4097}),
    "decode-wide-group": (BF, False, 160, 1, 64, 16, [3000, 40], [1, 3]),
    "decode-fp4": (BF, True, 28, 4, 128, 16, [30000, 511, 0, 7777], [1, 1, 1, 0]),
    "decode-fp4-many": (HF, True, 32, 8, 64, 32, [100 + 37 * i for i in range(60)], [1] * 60),
    "decode-f32": (FL, False, 8, 2, 128, 64, [9000, 63, 1], [1, 1, 1]),
    "rows-f32": (FL, False, 14, 2, 64, 16, [2000, 0], [50, 90]),
    "decode-f32-fp4": (FL, True, 8, 2, 64, 32, [5000, 63], [1, 2]),
}


def case(name, **kw):
    *a, options = LONG[name] if isinstance(LONG[name][-1], dict) else (*LONG[name], {})
    return Case(*a, **{**options, **kw})


@pytest.mark.parametrize("name", LONG)
def test_against_64_bits(name):
    c = case(name)
    out = c.run()
    C.check_device_error()
    c.check(out)


@pytest.mark.parametrize("name", ["tiles-bf16", "tiles-fp4", "parts", "parts-fp4", "long-parts", "decode", "decode-fp4",
                                  "decode-f32"])
def test_relaunches_give_the_same_bits(name):
    c = case(name)
    want = c.run()
    for _ in range(25):
        assert torch.equal(c.run(), want)
    C.check_device_error()


def test_two_calls_at_once_on_two_streams():
    """Each call has its own workspace: neither disturbs the other."""
    pairs = [case("decode", seed=3), case("long-parts", seed=4)]
    want = [c.run() for c in pairs]
    streams = [torch.cuda.Stream() for _ in pairs]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, (c, s) in enumerate(zip(pairs, streams)):
            with torch.cuda.stream(s):
                got[i].append(c.run())
    torch.cuda.synchronize()
    C.check_device_error()
    for g, w in zip(got, want):
        assert all(torch.equal(x, w) for x in g)


@pytest.mark.parametrize("names", [("decode", "parts"), ("decode-fp4", "long-parts-fp4"), ("decode-f32", "tiles-bf16")])
def test_two_graphs_over_one_memory_pool(names):
    """Two captured calls that share the memory of their workspaces, replayed in turn with new inputs."""
    cases = [case(n) for n in names]
    for c in cases:
        c.run()
    torch.cuda.synchronize()
    graphs, outs, pool = [], [], None
    for c in cases:
        out = torch.empty_like(c.q)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, pool=pool):
            c.run(out=out)
        pool = pool or g.pool()
        graphs.append(g)
        outs.append(out)
    for turn in range(3):
        for c in cases:
            c.q.copy_(torch.randn(c.q.shape, generator=torch.Generator().manual_seed(turn)))
        eager = [c.run() for c in cases]
        for g in graphs + graphs[::-1]:
            g.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, eager):
            assert torch.equal(a, b)
    C.check_device_error()


def test_captured_decode_follows_positions_and_table():
    """One captured step, replayed while positions grow over pages and parts of the keys: the eager call's bits."""
    c = case("decode-many")
    table, positions = c.table.clone(), c.positions.clone()
    c.table = table
    out = torch.empty_like(c.q)
    c.run(out=out)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        c.run(out=out)
    for cut in (0, 1, 63, 64, 99):
        c.positions.copy_(positions - cut)
        g.replay()
        assert torch.equal(out, c.run())
    C.check_device_error()


@pytest.mark.parametrize("name", ["parts", "decode", "decode-fp4", "decode-f32", "tiles-fp4"])
def test_pages_behind_the_window_may_be_gone(name):
    """Pages whose rows no query of the sequence sees any more are not looked at: -1 in the table is no error there."""
    c = case(name, window=333)
    want = c.run()
    C.check_device_error()
    c.check(want)
    page = c.k.shape[2] if c.k.dim() == 4 else c.k.shape[2] // (c.d * 9 // 16)
    for b, p in enumerate(c.past):
        c.table[b, :max(0, p - 332) // page] = -1
    assert (c.table[0, :100] == -1).any()
    assert torch.equal(c.run(), want)
    C.check_device_error()


@pytest.mark.parametrize("name", ["parts", "decode", "decode-fp4", "tiles-fp4", "decode-f32"])
def test_rows_of_q_do_not_touch_each_other(name):
    """NaN and infinities in some rows of q stay there; the other rows keep their bits."""
    c = case(name)
    want = c.run()
    q = c.q.clone()
    q[0, 1, 3] = float("nan")
    q[-1, 0, 0] = float("inf")
    q[-1, -1] = float("-inf")
    got = c.run(q=q)
    touched = torch.zeros(q.shape[:2], dtype=torch.bool, device="cuda")
    touched[0, 1] = touched[-1, 0] = touched[-1, -1] = True
    assert torch.equal(got[~touched], want[~touched])
    assert torch.isnan(got[0, 1]).all()
    C.check_device_error()


@pytest.mark.parametrize("name", ["parts", "decode", "decode-fp4", "tiles-fp4", "decode-f32", "long-parts-fp4"])
@pytest.mark.parametrize("amplitude", [0.0, 2.0 ** -14, 200.0])
def test_small_and_large_scores(name, amplitude):
    """Scores of zero (equal weights), of nearly zero, and of hundreds (one key takes all)."""
    c = case(name, amplitude=amplitude)
    out = c.run()
    C.check_device_error()
    c.check(out)


@pytest.mark.parametrize("name", ["parts", "decode", "decode-fp4", "decode-f32"])
@pytest.mark.parametrize("where", ["q", "out", "k", "v"])
def test_views_off_their_alignment(name, where):
    """Contiguous views that start at an odd element (pages of bytes: an odd byte) are served, or refused where the
    kernels need whole words; nothing faults."""
    c = case(name, seed=6)
    want = c.run()

    def shifted(t):
        flat = torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")[1:]
        flat.copy_(t.reshape(-1))
        return flat.view(t.shape)

    kw = {}
    if where == "q":
        kw["q"] = shifted(c.q)
    elif where == "out":
        kw["out"] = shifted(c.q)
    else:
        setattr(c, where, shifted(getattr(c, where)))
    try:
        got = c.run(**kw)
    except ValueError as e:
        assert "align" in str(e)
        return
    C.check_device_error()
    c.k, c.v = c.k.clone(), c.v.clone()
    c.check(got)
    if c.dtype != FL:
        torch.testing.assert_close(got.float(), want.float(), rtol=2 * torch.finfo(c.dtype).eps, atol=4 * torch.finfo(c.dtype).eps)


def test_a_workspace_that_is_too_small_is_refused():
    c = case("decode")
    L = C.lib()
    hkv, page = c.k.shape[1], c.k.shape[2]
    need = L.dli_sm100_attention_paged_workspace_size(c.tokens, len(c.past), 1, c.hq, hkv, c.d, page, c.table.shape[1], C.DTYPE_CODES[BF], C.DTYPE_CODES[BF])
    assert need > 0
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    out = torch.full_like(c.q, 3.0)

    def call(workspace, nbytes):
        return L.dli_sm100_attention_paged(
            c.q.data_ptr(), c.k.data_ptr(), c.v.data_ptr(), c.positions.data_ptr(), c.starts.data_ptr(), c.table.data_ptr(),
            None, out.data_ptr(), c.tokens, len(c.past), 1, c.hq, hkv, c.d, page, c.k.shape[0], c.table.shape[1], 0.0, 0.0, 0,
            1.0, 1.0, C.DTYPE_CODES[BF], C.DTYPE_CODES[BF], workspace, nbytes, torch.cuda.current_stream().cuda_stream)

    assert call(ws.data_ptr(), need - 1) == 4 and call(None, 0) == 4
    torch.cuda.synchronize()
    assert (out == 3).all()
    assert call(ws.data_ptr(), need) == 0
    C.check_device_error()
    assert torch.equal(out, c.run())


def test_gather_and_append_on_another_stream_and_many_pages():
    """A pool above 2^31 bytes: rows of its last pages are written, read and attended to as any others."""
    hkv, d, page, hq = 8, 128, 128, 16
    pages = (2 ** 31 // (hkv * d * page * 2)) + 40
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        k, v = C.paged_kv_pages(pages, hkv, page, d, BF)
        assert k.numel() * 2 > 2 ** 31
        table = torch.tensor([[pages - 1, 3, pages - 7], [pages - 2, 0, pages - 30]], dtype=torch.int32, device="cuda")
        small = torch.tensor([[0, 1, 2], [3, 4, 5]], dtype=torch.int32, device="cuda")
        k2, v2 = C.paged_kv_pages(6, hkv, page, d, BF)
        g = torch.Generator(device="cuda").manual_seed(5)
        one = torch.ones(400, 1, device="cuda")
        results = []
        for past, new in ((0, 300), (300, 1), (301, 40)):
            qkv = torch.randn(2 * new, (hq + 2 * hkv) * d, generator=g, device="cuda").to(BF)
            pos = torch.full((2,), past, device="cuda")
            both = []
            for kk, vv, tt in ((k, v, table), (k2, v2, small)):
                q = C.qkv_rotary_paged(qkv, one, one * 0, pos, tt, kk, vv, hq)
                both.append((C.attention_paged(q, kk, vv, pos, tt), *C.paged_gather(kk, vv, tt, past + new, d, BF)))
            results.append(both)
    s.synchronize()
    C.check_device_error()
    for (a, b) in results:
        for x, y in zip(a, b):
            assert torch.equal(x, y) and torch.isfinite(x).all()


@pytest.mark.parametrize("fp4", [False, True], ids=["rows16", "rows4"])
def test_positions_and_lengths_at_the_ends_of_their_type(fp4):
    """The largest and smallest int64 as positions or lengths: reported, nothing written, the other sequences served."""
    hkv, d, page, hq = 2, 64, 16, 4
    table = torch.tensor([[0, 1], [2, 3]], dtype=torch.int32, device="cuda")
    one = torch.ones(64, 1, device="cuda")
    qkv = torch.randn(2, (hq + 2 * hkv) * d, device="cuda").to(BF)
    for far in (2 ** 63 - 1, 2 ** 63 - 2, -2 ** 63, 2 ** 32, 2 ** 31 - 1):
        k, v = C.paged_kv_pages(4, hkv, page, d, "fp4" if fp4 else BF)
        k.fill_(1), v.fill_(1)
        kept = k[2:].clone()
        pos = torch.tensor([3, far], device="cuda")
        q = torch.full((2, hq, d), 7.0, dtype=BF, device="cuda")
        C.qkv_rotary_paged(qkv, one, one * 0, pos, table, k, v, hq, q_out=q)
        with pytest.raises(RuntimeError):
            C.check_device_error()
        assert torch.equal(k[2:], kept) and (q[1] == 7).all() and torch.equal(q[0], qkv[0, :hq * d].view(hq, d))
        for rows in (1, 40):  # the decode kernel, the tcgen05 kernel
            out = torch.full((2 * rows, hq, d), 7.0, dtype=BF, device="cuda")
            big = torch.tensor([[0, 1, 0, 1], [2, 3, 2, 3]], dtype=torch.int32, device="cuda")
            C.attention_paged(torch.zeros_like(out), k, v, pos, big, out=out)
            with pytest.raises(RuntimeError):
                C.check_device_error()
            assert (out[rows:] == 7).all() and torch.isfinite(out[:rows]).all() and (out[:rows] != 7).all()
        # past every row: zeros, with an error only where a bound is outside the table's
        kk, vv = C.paged_gather(k, v, table, 5, d, BF, first=pos)
        assert (kk[1] == 0).all() and (vv[1] == 0).all() and kk[0].abs().sum() > 0
        if far < 0:
            with pytest.raises(RuntimeError):
                C.check_device_error()
        C.check_device_error()
        kk, _ = C.paged_gather(k, v, table, 32, d, BF, lengths=pos)
        assert kk[0, :, :3].abs().sum() > 0 and (kk[0, :, 3:] == 0).all()
        if far > 0:
            with pytest.raises(RuntimeError):
                C.check_device_error()
        C.check_device_error()


@pytest.mark.parametrize("name", ["tiles-bf16", "tiles-fp4", "parts", "long-parts", "decode", "decode-many", "decode-fp4",
                                  "decode-f32", "rows-f32"])
def test_the_output_may_be_q_itself(name):
    c = case(name)
    want = c.run()
    q = c.q.clone()
    assert torch.equal(c.run(q=q, out=q), want)
    C.check_device_error()


@pytest.mark.parametrize("name", ["parts", "decode", "decode-fp4", "tiles-fp4", "decode-f32", "rows-f32"])
@pytest.mark.parametrize("softcap", [2.0 ** -130, 1e-3, 0.7, 3.0, 1e4, 1e9, 1e38])
def test_caps_of_any_size(name, softcap):
    """Caps far below the scores (all keys alike), around them, and far above (no cap at all): the error is one of
    the scores' size, not of the cap's."""
    c = case(name, softcap=softcap)
    out = c.run()
    C.check_device_error()
    c.check(out)


@pytest.mark.parametrize("name", ["tiles-bf16", "parts", "decode", "decode-fp4", "parts-fp4", "decode-f32"])
def test_a_window_of_one_and_a_window_past_everything(name):
    c = case(name, window=1)
    c.check(c.run())
    c = case(name, window=2 ** 40)
    plain = case(name, window=0)
    assert torch.equal(c.run(), plain.run())
    C.check_device_error()


@pytest.mark.parametrize("name", ["decode", "decode-fp4", "parts", "long-parts", "decode-f32"])
def test_a_bound_on_new_rows_that_is_too_large(name):
    """max_new may be more than any sequence has (here: all rows of the batch); rows behind the last sequence stay."""
    c = case(name)
    q = torch.cat([c.q, c.q[:3]])
    out = torch.full_like(q, 5.0)
    C.attention_paged(q, c.k, c.v, c.positions, c.table, starts=c.starts, slopes=c.slopes, out=out, **c.options)
    C.check_device_error()
    c.check(out)
    assert (out[c.tokens:] == 5).all()
    out.fill_(5.0)  # a bound beyond any buffer costs nothing
    C.attention_paged(q, c.k, c.v, c.positions, c.table, starts=c.starts, max_new=2 ** 30, slopes=c.slopes, out=out, **c.options)
    C.check_device_error()
    c.check(out)
    hkv = c.k.shape[1]
    qkv = torch.zeros(c.tokens, (c.hq + 2 * hkv) * c.d, dtype=c.dtype, device="cuda")
    one = torch.ones(int(c.lengths.max()), 1, device="cuda")
    C.qkv_rotary_paged(qkv, one, one * 0, c.positions, c.table, c.k, c.v, c.hq, starts=c.starts, max_new=2 ** 30)
    C.check_device_error()
    # no rows at all in a batch that has some behind it
    out.fill_(5.0)
    C.attention_paged(q, c.k, c.v, c.positions, c.table, starts=torch.zeros_like(c.starts), out=out)
    C.check_device_error()
    assert (out == 5).all()


@pytest.mark.parametrize("fp4", [False, True], ids=["rows16", "rows4"])
@pytest.mark.parametrize("new", [1, 40])
def test_sequences_that_share_their_first_pages(fp4, new):
    """A common prefix cached once: the same bits as with a copy of it for every sequence."""
    c = Case(HF, fp4, 8, 2, 64, 32, [320, 320, 320], [new] * 3, seed=9)
    shared = c.table.clone()
    shared[1:, :10] = shared[0, :10]
    for t in (c.k, c.v):
        for b in (1, 2):
            t[c.table[b, :10].long()] = t[c.table[0, :10].long()]
    want = c.run()
    assert torch.equal(c.run(table=shared), want)
    C.check_device_error()
    c.check(want)
