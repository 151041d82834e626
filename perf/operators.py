"""The paged key/value cache operators, measured over their range: the append with rotary embedding
(into pages of the model's type or of 4-bit values) and the attention that reads the pages back.

Plain forms are elementary torch operations; with `own` set, run() makes the calls a program makes of
dli_sm100. A 4-bit page holds, per (page, head), page_size rows of head_dim/2 code bytes (E2M1, the even
element in the low half) followed by page_size rows of head_dim/16 scale bytes (E4M3, one for 16 elements).
"""
import math
import os
import random
import sys

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
THETA = 1e6


def _case(name, op, dtype, fp4, batch, q_heads, kv_heads, head_dim, page, new, past, ragged,
          softcap=0.0, window=0, slopes=False):
    return {"name": name, "op": op, "dtype": dtype, "fp4": fp4, "batch": batch, "q_heads": q_heads,
            "kv_heads": kv_heads, "head_dim": head_dim, "page": page, "new": new, "past": past,
            "ragged": ragged, "softcap": softcap, "window": window, "slopes": slopes}


def listed():
    return [
        # one decode step of a batch of 32: a latency-bound append
        _case("append_step_bf16", "append", "bf16", False, 32, 28, 4, 128, 16, 1, 2304, True),
        # a packed batch of prompts of a small model
        _case("append_prompts_f16", "append", "f16", False, 24, 14, 2, 64, 32, 2048, 0, True),
        # one decode step of a large model's batch into the 4-bit cache, its rows read back
        _case("append_step_fp4_bf16", "append", "bf16", True, 128, 64, 8, 128, 64, 1, 1000, True),
        # prompts into the 4-bit cache
        _case("append_prompts_fp4_bf16", "append", "bf16", True, 16, 28, 4, 128, 16, 2048, 0, True),
        # a single chat's step with a short history: the smallest call
        _case("decode_one_bf16", "attend", "bf16", False, 1, 14, 2, 64, 16, 1, 333, False),
        # the step of a full batch, every sequence of another length
        _case("decode_batch_bf16", "attend", "bf16", False, 32, 28, 4, 128, 16, 1, 2304, True),
        # few, very long sequences, capped scores
        _case("decode_long_f16_capped", "attend", "f16", False, 3, 64, 8, 128, 64, 1, 60001, True, 30.0),
        # a packed batch of whole prompts
        _case("prompts_bf16", "attend", "bf16", False, 16, 28, 4, 128, 64, 2048, 0, True),
        # a chunk of two long prompts, distance bias and a window
        _case("chunk_f16_distance", "attend", "f16", False, 2, 16, 16, 64, 32, 383, 8000, True, 0.0, 4096, True),
        # the step of a float32 model
        _case("decode_f32", "attend", "f32", False, 6, 16, 4, 128, 16, 1, 1501, True),
        # the step of a batch over the 4-bit cache
        _case("decode_batch_fp4_bf16", "attend", "bf16", True, 24, 28, 4, 128, 16, 1, 8192, True),
        # chunks of prompts over the 4-bit cache
        _case("chunk_fp4_bf16", "attend", "bf16", True, 4, 28, 4, 128, 32, 301, 3001, True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("append", "attend", "attend"))
    fp4 = rng.random() < 0.4
    dtype = rng.choice(("bf16", "bf16", "f16") if fp4 else ("bf16", "bf16", "f16", "f16", "f32"))
    q_heads, kv_heads, head_dim = rng.choice(
        ((14, 2, 64), (28, 4, 128), (64, 8, 128), (16, 16, 64), (16, 4, 128), (8, 1, 128), (24, 2, 64)))
    c = _case("", op, dtype, fp4, _log(rng, 1, 96), q_heads, kv_heads, head_dim, rng.choice((16, 32, 64, 128)),
              rng.choice((1, 1, rng.randint(2, 5), _log(rng, 6, 2048))), _log(rng, 1, 40000), rng.random() < 0.8)
    del c["name"]
    if op == "attend":
        c["softcap"] = rng.choice((0.0, 0.0, 20.0, 50.0))
        c["window"] = rng.choice((0, 0, _log(rng, 16, 4096)))
        c["slopes"] = rng.random() < 0.25
    if c["new"] > 64 and rng.random() < 0.5:
        c["past"] = 0
    most_scores, most_bytes, most_rows = 16 * 28 * 2048 * 2048, 600e6, 40000
    if dtype == "f32":  # float32 runs on the CUDA cores: smaller
        most_scores, most_bytes = 2e8, 200e6
    while True:
        length = c["past"] + c["new"]
        cache = 4 * c["batch"] * length * kv_heads * head_dim
        if op == "attend" and c["batch"] * q_heads * c["new"] * length > most_scores or cache > most_bytes or \
                c["batch"] * c["new"] * (q_heads + 2 * kv_heads) * head_dim > most_rows * 36 * 128:
            if c["batch"] > 1 and rng.random() < 0.6:
                c["batch"] = max(1, int(c["batch"] * 0.7))
            else:
                c["past"] = int(c["past"] * 0.7)
                c["new"] = max(1, int(c["new"] * 0.8))
            continue
        return c


def _lengths(case):
    """(past, new) of every sequence: by the case alone."""
    r = random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))
    past, new = [], []
    for b in range(case["batch"]):
        lo = 0.4 if case["ragged"] and b else 1.0
        past.append(int(case["past"] * r.uniform(lo, 1.0)))
        new.append(max(1, int(case["new"] * r.uniform(lo, 1.0))))
    return past, new


def _esize(case):
    return 4 if case["dtype"] == "f32" else 2


def work(case):
    past, new = _lengths(case)
    hq, hkv, d, es = case["q_heads"], case["kv_heads"], case["head_dim"], _esize(case)
    row = d * 9 / 16 if case["fp4"] else d * es
    t = sum(new)
    if case["op"] == "append":
        spots = set()
        for p, n in zip(past, new):
            spots.update(range(p, p + n))
        size = t * (hq + 2 * hkv) * d * es + t * hq * d * es + 2 * t * hkv * row + len(spots) * d * 4
        if case["fp4"]:  # the rows are read back as values
            size += 2 * t * hkv * row + 2 * case["batch"] * case["new"] * hkv * d * es
        return {"bytes": size, "flops": 3 * t * (hq + hkv) * d}
    w = case["window"] or (1 << 60)
    pairs = rows = 0
    for p, n in zip(past, new):
        full = max(0, min(p + n, w) - p)          # rows that see every key up to themselves
        pairs += full * p + full * (full + 1) // 2 + (n - full) * min(w, 1 << 40)
        rows += min(p + n, n + w - 1)
    return {"bytes": 2 * t * hq * d * es + 2 * rows * hkv * row, "flops": 4 * d * hq * pairs}


class State:
    pass


def _pack(x, page):
    """[pages, heads, page, d] values near to 4-bit pages, for prepare()."""
    n, h, p, d = x.shape
    b = x.float().unflatten(-1, (d // 16, 16))
    scale = (b.abs().amax(-1, keepdim=True) / 6).to(torch.float8_e4m3fn)
    edges = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device=x.device)
    code = torch.bucketize(b.abs() / scale.float().clamp_min(2.0 ** -9), edges).to(torch.uint8)
    code = (code | ((b < 0).to(torch.uint8) << 3)).flatten(-2)
    code = code[..., 0::2] | (code[..., 1::2] << 4)
    return torch.cat([code.flatten(-2), scale.squeeze(-1).view(torch.uint8).flatten(-2)], -1).contiguous()


def prepare(case, seed):
    past, new = _lengths(case)
    dev = "cuda"
    g = torch.Generator(device=dev).manual_seed(seed)
    dt = TYPES[case["dtype"]]
    b, hq, hkv, d, page = (case[k] for k in ("batch", "q_heads", "kv_heads", "head_dim", "page"))
    s = State()
    s.case, s.total, s.max_new = case, sum(new), max(new)
    s.max_len = max(p + n for p, n in zip(past, new))
    counts = torch.tensor(new, dtype=torch.int64)
    s.counts = counts.to(dev)
    s.starts = torch.cat([torch.zeros(1, dtype=torch.int64), counts.cumsum(0)]).to(dev)
    s.positions = torch.tensor(past, dtype=torch.int64, device=dev)
    s.lengths = s.positions + s.counts
    need = [-(-(p + n) // page) for p, n in zip(past, new)]
    width = max(need) + 1
    pool = sum(need) + max(2, sum(need) // 16)
    order = torch.randperm(pool, device=dev, generator=g).to(torch.int32)
    table = torch.zeros(b, width, dtype=torch.int32, device=dev)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    s.table = table

    def normal(*shape):
        return torch.randn(*shape, device=dev, generator=g)

    def pages():
        # channels of unlike size, as keys have them
        x = normal(pool, hkv, page, d).mul_(0.25 + 1.5 * torch.rand(hkv, 1, d, device=dev, generator=g))
        return _pack(x, page) if case["fp4"] else x.to(dt)

    s.k_pages, s.v_pages = pages(), pages()
    if case["op"] == "append":
        s.qkv = normal(s.total, (hq + 2 * hkv) * d).to(dt)
        inv = THETA ** (-torch.arange(0, d, 2, dtype=torch.float64, device=dev) / d)
        angle = torch.outer(torch.arange(s.max_len, dtype=torch.float64, device=dev), inv)
        s.cos, s.sin = angle.cos().float().contiguous(), angle.sin().float().contiguous()
    else:
        s.q = normal(s.total, hq, d).to(dt)
        s.slopes = None
        if case["slopes"]:
            s.slopes = 2.0 ** (-8.0 * torch.arange(1, hq + 1, device=dev, dtype=torch.float32) / hq)
    return s


# ---- plain forms ---------------------------------------------------------------------------------


def _tokens(s):
    """(sequence, position) of every packed row."""
    seq = torch.repeat_interleave(torch.arange(s.case["batch"], device="cuda"), s.counts, output_size=s.total)
    return seq, s.positions[seq] + torch.arange(s.total, device="cuda") - s.starts[seq]


def _planes(pages, case):
    """Code and scale views of 4-bit pages: [pages, heads, page, d/2] and [pages, heads, page, d/16]."""
    p, d = case["page"], case["head_dim"]
    cut = p * d // 2
    return pages[..., :cut].unflatten(-1, (p, d // 2)), pages[..., cut:].unflatten(-1, (p, d // 16))


def _values(code, scale):
    """float32 values of code bytes [.., d/2] and scale bytes [.., d/16]."""
    table = torch.tensor(E2M1 + tuple(-x for x in E2M1), device=code.device)
    x = table[torch.stack([code & 15, code >> 4], -1).flatten(-2).long()]
    return (x.unflatten(-1, (-1, 16)) * scale.contiguous().view(torch.float8_e4m3fn).float().unsqueeze(-1)).flatten(-2)


def _quantise(x):
    """float64 [.., d] -> (code bytes, scale bytes): nearest E4M3 to max/6, nearest E2M1 to x/scale, ties to the even code."""
    b = x.unflatten(-1, (-1, 16))
    most = b.abs().amax(-1)
    grid = torch.arange(127, dtype=torch.uint8, device=x.device).view(torch.float8_e4m3fn).double()
    edge = 6 * (grid[:-1] + grid[1:]) / 2
    edge[1::2] = torch.nextafter(edge[1::2], torch.zeros_like(edge[1::2]))  # a tie goes up to an even code
    scale = torch.bucketize(most, edge)
    unit = grid[scale].unsqueeze(-1)
    code = torch.zeros(b.shape, dtype=torch.uint8, device=x.device)
    size = b.abs()
    for cut, up in ((0.25, False), (0.75, True), (1.25, False), (1.75, True), (2.5, False), (3.5, True), (5.0, False)):
        code += (size >= cut * unit) if up else (size > cut * unit)
    code = torch.where(unit > 0, code, 0) | ((b < 0) & (unit > 0)).to(torch.uint8) << 3
    code = code.flatten(-2)
    return code[..., 0::2] | (code[..., 1::2] << 4), scale.to(torch.uint8)


def _rotate(x, cos, sin):
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)


def _plain_append(s):
    case = s.case
    hq, hkv, d, page = (case[k] for k in ("q_heads", "kv_heads", "head_dim", "page"))
    dt = s.qkv.dtype
    seq, pos = _tokens(s)
    x = s.qkv.view(s.total, hq + 2 * hkv, d)
    cos, sin = s.cos[pos].unsqueeze(1), s.sin[pos].unsqueeze(1)
    q = _rotate(x[:, :hq].float(), cos, sin).to(dt)
    spot, row = s.table[seq, pos // page].long(), pos % page
    if not case["fp4"]:
        s.k_pages[spot, :, row] = _rotate(x[:, hq:hq + hkv].float(), cos, sin).to(dt)
        s.v_pages[spot, :, row] = x[:, hq + hkv:]
        return {"q": q, "k_pages": s.k_pages, "v_pages": s.v_pages}
    out = {"q": q}
    # values next to a rounding border: 64 bits
    k = _rotate(x[:, hq:hq + hkv].double(), cos.double(), sin.double())
    rows = (torch.arange(s.total, device="cuda") - s.starts[seq])
    for name, pages, v in (("k", s.k_pages, k), ("v", s.v_pages, x[:, hq + hkv:].double())):
        codes, scales = _planes(pages, case)
        codes[spot, :, row], scales[spot, :, row] = _quantise(v)
        back = torch.zeros(case["batch"], hkv, s.max_new, d, dtype=dt, device="cuda")
        back[seq, :, rows] = _values(codes[spot, :, row], scales[spot, :, row]).to(dt)
        out[name] = back
    return out


def _plain_attend(s):
    case = s.case
    hq, hkv, d, page = (case[k] for k in ("q_heads", "kv_heads", "head_dim", "page"))
    b, n, g = case["batch"], s.max_new, hq // hkv
    j = torch.arange(s.max_len, device="cuda")
    spot, row = s.table[:, j // page].long(), (j % page).expand(b, -1)

    def dense(pages):
        if case["fp4"]:
            codes, scales = _planes(pages, case)
            return _values(codes[spot, :, row], scales[spot, :, row])
        return pages[spot, :, row].float()

    k, v = dense(s.k_pages), dense(s.v_pages)                       # [b, length, hkv, d]
    i = torch.arange(n, device="cuda")
    at = (s.starts[:-1, None] + i).clamp_max(s.total - 1)
    q = s.q[at].float().view(b, n, hkv, g, d)
    x = torch.einsum("bnhgd,blhd->bhgnl", q, k) / math.sqrt(d)
    if case["softcap"]:
        t = torch.exp(-2 / case["softcap"] * x.abs())
        x = torch.sign(x) * (case["softcap"] * (1 - t) / (1 + t))
    where = (s.positions[:, None] + i)[:, :, None]                  # [b, n, 1]
    seen = j <= where
    if case["window"]:
        seen = seen & (j > where - case["window"])
    if s.slopes is not None:
        x = x + s.slopes.view(1, hkv, g, 1, 1) * (j - where).float()[:, None, None]
    x = x.masked_fill(~seen[:, None, None], float("-inf"))
    x = torch.exp(x - x.amax(-1, keepdim=True))
    norm = x.sum(-1)                                                # [b, hkv, g, n]
    o = torch.einsum("bhgnl,blhd->bnhgd", x, v) / norm.permute(0, 3, 1, 2).unsqueeze(-1)
    seq, pos = _tokens(s)
    return o.reshape(b, n, hq, d)[seq, pos - s.positions[seq]].to(s.q.dtype)


def run(s):
    case = s.case
    if not own:
        return _plain_append(s) if case["op"] == "append" else _plain_attend(s)
    at = os.path.join(os.getcwd(), "dl-inference_b200", "python")
    if at not in sys.path:
        sys.path.insert(0, at)
    import dli_sm100 as C

    if case["op"] == "append":
        q = C.qkv_rotary_paged(s.qkv, s.cos, s.sin, s.positions, s.table, s.k_pages, s.v_pages, case["q_heads"],
                               starts=s.starts, max_new=s.max_new)
        if not case["fp4"]:
            return {"q": q, "k_pages": s.k_pages, "v_pages": s.v_pages}
        k, v = C.paged_gather(s.k_pages, s.v_pages, s.table, s.max_new, case["head_dim"], s.qkv.dtype,
                              first=s.positions, lengths=s.lengths)
        return {"q": q, "k": k, "v": v}
    return C.attention_paged(s.q, s.k_pages, s.v_pages, s.positions, s.table, starts=s.starts, max_new=s.max_new,
                             softcap=case["softcap"], window=case["window"], slopes=s.slopes)


# ---- from the definition, in 64 bits ---------------------------------------------------------------


def _near(x, grid):
    """Index of the nearest grid value (ascending, from 0), the even index on a tie, the last beyond the grid."""
    hi = torch.searchsorted(grid, x.contiguous()).clamp(1, grid.numel() - 1)
    lo = hi - 1
    up, down = grid[hi] - x, x - grid[lo]
    return torch.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)


def _through_fp4(x):
    """The values that 4-bit blocks hold for x (float64)."""
    shape = x.shape
    x = x.reshape(-1, 16)
    grid = torch.tensor([(m / 8.0) * 2.0 ** -6 if e == 0 else (1 + m / 8.0) * 2.0 ** (e - 7)
                         for e in range(16) for m in range(8)][:127], dtype=torch.float64, device=x.device)
    size = torch.tensor(E2M1, dtype=torch.float64, device=x.device)
    scale = grid[_near(x.abs().amax(1) / 6, grid)].unsqueeze(1)
    q = size[_near(torch.where(scale > 0, x.abs() / scale.clamp_min(2.0 ** -12), 0.0), size)]
    return (torch.sign(x) * q * scale).reshape(shape)


def _exact_rows(pages, table_row, length, case):
    """[hkv, length, d] float64 rows 0..length-1 of one sequence."""
    page, d = case["page"], case["head_dim"]
    x = pages[table_row[: -(-length // page)].long()]
    if case["fp4"]:
        half = x[..., : page * d // 2]
        e4 = x[..., page * d // 2:].contiguous().view(torch.float8_e4m3fn).double()
        both = torch.stack([half % 16, half // 16], -1).flatten(-2)
        mag = both % 8
        val = torch.where(mag < 2, mag.double() / 2, (1 + (mag % 2).double() / 2) * 2.0 ** ((mag // 2).double() - 1))
        x = torch.where(both >= 8, -val, val) * e4.repeat_interleave(16, -1)
        x = x.unflatten(-1, (page, d))
    return x.double().transpose(0, 1).flatten(1, 2)[:, :length]


def exact(case, seed):
    s = prepare(case, seed)
    past, new = _lengths(case)
    hq, hkv, d = case["q_heads"], case["kv_heads"], case["head_dim"]
    begin = 0
    if case["op"] == "append":
        q = torch.empty(s.total, hq, d, dtype=torch.float64, device="cuda")
        k_pages, v_pages = (None, None) if case["fp4"] else (s.k_pages.double(), s.v_pages.double())
        back = [torch.zeros(case["batch"], hkv, s.max_new, d, dtype=torch.float64, device="cuda") for _ in (0, 1)]
        for b, (p, n) in enumerate(zip(past, new)):
            x = s.qkv[begin:begin + n].double().reshape(n, hq + 2 * hkv, d // 2, 2)
            turn = torch.complex(s.cos[p:p + n].double(), s.sin[p:p + n].double()).unsqueeze(1)
            r = torch.view_as_real(torch.view_as_complex(x[:, :hq + hkv].contiguous()) * turn).flatten(-2)
            q[begin:begin + n] = r[:, :hq]
            k, v = r[:, hq:], x[:, hq + hkv:].flatten(-2)
            if case["fp4"]:
                back[0][b, :, :n], back[1][b, :, :n] = _through_fp4(k).transpose(0, 1), _through_fp4(v).transpose(0, 1)
            else:
                where = torch.arange(p, p + n, device="cuda")
                spot = s.table[b, where // case["page"]].long()
                k_pages[spot, :, where % case["page"]] = k
                v_pages[spot, :, where % case["page"]] = v
            begin += n
        return {"q": q, "k": back[0], "v": back[1]} if case["fp4"] else {"q": q, "k_pages": k_pages, "v_pages": v_pages}
    out = torch.empty(s.total, hq, d, dtype=torch.float64, device="cuda")
    for b, (p, n) in enumerate(zip(past, new)):
        first = max(0, p - case["window"] + 1) if case["window"] else 0
        k = _exact_rows(s.k_pages, s.table[b], p + n, case)[:, first:]
        v = _exact_rows(s.v_pages, s.table[b], p + n, case)[:, first:]
        gap = torch.arange(p, p + n, device="cuda")[:, None] - torch.arange(first, p + n, device="cuda")
        hidden = (gap < 0) | (gap >= case["window"]) if case["window"] else gap < 0
        for h in range(hq):
            x = s.q[begin:begin + n, h].double() @ k[h * hkv // hq].T * d ** -0.5
            if case["softcap"]:
                x = case["softcap"] * torch.tanh(x / case["softcap"])
            if s.slopes is not None:
                x = x - s.slopes[h].double() * gap
            x = torch.softmax(x.masked_fill(hidden, -math.inf), -1)
            out[begin:begin + n, h] = x @ v[h * hkv // hq]
        begin += n
    return out
