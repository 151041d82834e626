"""GPU tests of the paged KV cache in the engine and the Qwen2 runner."""
from __future__ import annotations

import json

import numpy as np
import pytest
import torch

import dli
import model_parity

pytestmark = pytest.mark.gpu


_GRAPHS = []  # an engine knows its plans by their graph's address: graphs outlive it


def _graph(nodes, inputs, outputs):
    _GRAPHS.append(dli.Graph.from_json(json.dumps({"format": "dli.graph.v1", "inputs": inputs, "outputs": outputs, "nodes": [
        {"name": f"n{i}", "op": op, "inputs": a, "outputs": b, "attrs": attrs}
        for i, (op, a, b, attrs) in enumerate(nodes)]})))
    return _GRAPHS[-1]


def _engine():
    e = dli.Engine()
    e.load_library(dli.PLUGIN_PATH)
    return e


def _pool_attrs(hq, hkv, d, page, pages, fp4):
    return {"q_heads": hq, "kv_heads": hkv, "head_dim": d, "page_size": page, "num_pages": pages, "kv_cache": "c",
            **({"kv_dtype": "fp4", "k_scale": 0.5, "v_scale": 2.0} if fp4 else {})}


@pytest.mark.parametrize("fp4", [False, True], ids=["rows16", "rows4"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=["bf16", "f16", "f32"])
def test_graph_operators_equal_the_wrappers(dtype, fp4):
    """Three runs of an engine (a prompt, a chunk, single tokens) over one pool give the bits of the wrappers."""
    import dli_sm100 as C

    hq, hkv, d, page, pages, b = 6, 2, 64, 32, 9, 2
    opts = {"softcap": 20.0, "window": 50, "scale": 0.2}
    scales = {"k_scale": 0.5, "v_scale": 2.0} if fp4 else {}
    g = _graph([("qkv_rotary_paged", ["qkv", "cos", "sin", "pos", "table"], ["q"], _pool_attrs(hq, hkv, d, page, pages, fp4)),
                ("attention_paged", ["q", "pos", "table", "slopes"], ["out"], {"kv_cache": "c", **opts, **scales})],
               ["qkv", "cos", "sin", "pos", "table", "slopes"], ["q", "out"])
    gen = torch.Generator(device="cuda").manual_seed(4)
    table = torch.tensor([[3, 8, 1, 6], [0, 5, 2, 7]], dtype=torch.int32, device="cuda")
    ang = torch.rand(128, d // 2, device="cuda", generator=gen) * 6
    cos, sin = ang.cos(), ang.sin()
    slopes = torch.rand(hq, device="cuda", generator=gen) * 0.1
    kp, vp = C.paged_kv_pages(pages, hkv, page, d, "fp4" if fp4 else dtype)
    e = _engine()
    past = torch.zeros(b, dtype=torch.int64, device="cuda")
    for s in (70, 33, 1, 1):
        qkv = torch.randn(b, s, (hq + 2 * hkv) * d, device="cuda", generator=gen).to(dtype)
        got = e.run(g, {"qkv": qkv, "cos": cos, "sin": sin, "pos": past, "table": table, "slopes": slopes})
        q = C.qkv_rotary_paged(qkv.view(b * s, -1), cos, sin, past, table, kp, vp, hq, **scales)
        out = C.attention_paged(q, kp, vp, past, table, slopes=slopes, **opts, **scales)
        assert torch.equal(got["q"].reshape(-1), q.reshape(-1))
        assert got["out"].shape == (b, s, hq * d) and torch.equal(got["out"].reshape(-1), out.reshape(-1))
        past = past + s
    k, v, _ = e.kv_cache_entry("c")
    assert torch.equal(k, kp) and torch.equal(v, vp)
    C.check_device_error()


def test_cache_entries_keep_their_form():
    e = _engine()
    d, page = 64, 16
    table = torch.zeros(1, 2, dtype=torch.int32, device="cuda")
    pos = torch.zeros(1, dtype=torch.int64, device="cuda")
    cos = torch.ones(32, d // 2, device="cuda")
    qkv = torch.zeros(1, 1, 3 * d, device="cuda", dtype=torch.bfloat16)
    feed = {"qkv": qkv, "cos": cos, "sin": cos, "pos": pos, "table": table}

    def append(**kw):
        return _graph([("qkv_rotary_paged", ["qkv", "cos", "sin", "pos", "table"], ["q"],
                        {**_pool_attrs(1, 1, d, page, 4, False), **kw})], list(feed), ["q"])

    e.run(append(), feed)
    for other in (dict(num_pages=5), dict(page_size=32), dict(kv_dtype="fp4"), dict(kv_dtype="fp8"), dict(page_size=24),
                  dict(num_pages=0), dict(head_dim=32), dict(q_heads=0), dict(kv_heads=0)):
        with pytest.raises(ValueError):
            e.run(append(**other), feed)
    q = torch.zeros(1, 1, 1, d, device="cuda", dtype=torch.bfloat16)
    flat = _graph([("qkv_rotary_cache", ["qkv", "cos", "sin", "pos"], ["q"],
                    {"q_heads": 1, "kv_heads": 1, "head_dim": d, "capacity": 32, "kv_cache": "flat"})], list(feed), ["q"])
    e.run(flat, feed)
    for op, ins, name in (("attention_kvcache", ["q", "pos"], "c"), ("attention_paged", ["q", "pos", "table"], "flat"),
                          ("attention_paged", ["q", "pos", "table"], "none"),
                          ("attention", ["q", "q", "q"], "c")):
        with pytest.raises(ValueError):
            e.run(_graph([(op, ins, ["o"], {"kv_cache": name, "causal": True})], ins, ["o"]),
                  {"q": q, "pos": pos, "table": table})
    with pytest.raises(ValueError):  # the contiguous operator under the paged entry's name
        e.run(_graph([("qkv_rotary_cache", ["qkv", "cos", "sin", "pos"], ["q"],
                       {"q_heads": 1, "kv_heads": 1, "head_dim": d, "capacity": 32, "kv_cache": "c"})], list(feed), ["q"]), feed)
    with pytest.raises(ValueError):  # a table of another batch
        e.run(append(), {**feed, "table": torch.zeros(2, 2, dtype=torch.int32, device="cuda")})
    for bad in (q[..., :32].contiguous(), q.to(torch.float16)):
        with pytest.raises(ValueError):
            e.run(_graph([("attention_paged", ["q", "pos", "table"], ["o"], {"kv_cache": "c"})], ["q", "pos", "table"], ["o"]),
                  {"q": bad, "pos": pos, "table": table})


def test_a_pool_is_not_made_under_capture():
    d = 64
    e = _engine()
    g = _graph([("qkv_rotary_paged", ["qkv", "cos", "sin", "pos", "table"], ["q"], _pool_attrs(1, 1, d, 16, 2, False))],
               ["qkv", "cos", "sin", "pos", "table"], ["q"])
    one = torch.ones(32, d // 2, device="cuda")
    feed = {"qkv": torch.zeros(1, 1, 3 * d, device="cuda", dtype=torch.bfloat16), "cos": one, "sin": one,
            "pos": torch.zeros(1, dtype=torch.int64, device="cuda"),
            "table": torch.zeros(1, 2, dtype=torch.int32, device="cuda")}
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        with pytest.raises(RuntimeError, match="before a capture"):
            e.run(g, feed)
    assert e.kv_cache_size() == 0
    e.run(g, feed)
    captured = torch.cuda.CUDAGraph()
    with torch.cuda.graph(captured):
        e.run(g, feed)
    captured.replay()
    torch.cuda.synchronize()


def _small(head_dim=64):
    from dli_export.qwen2 import Qwen2Shape

    return Qwen2Shape(hidden=6 * head_dim, layers=3, q_heads=6, kv_heads=2, head_dim=head_dim, intermediate=512, vocab=1000)


def _runner(shape, capacity=256, **kw):
    from dli.qwen2 import Qwen2Runner
    from dli_export.qwen2 import random_state, transform_weights

    st = random_state(shape, device="cuda", dtype=torch.bfloat16, seed=2, std=0.05)
    return Qwen2Runner(shape, transform_weights(st, shape, dtype=torch.bfloat16), capacity=capacity, **kw)


@pytest.mark.parametrize("kv_dtype", [None, "fp4"], ids=["rows16", "rows4"])
@pytest.mark.parametrize("head_dim", [64, 128])
def test_generate_over_pages(head_dim, kv_dtype):
    """Captured and plain decoding give the same ids, whichever pages the sequences hold, and the pages return."""
    shape = _small(head_dim)
    r = _runner(shape, page_size=32, num_pages=40, kv_dtype=kv_dtype)
    prompt = torch.randint(0, shape.vocab, (3, 45), device="cuda", generator=torch.Generator("cuda").manual_seed(8))
    a = r.generate(prompt, 60)
    r.open([1])  # the pages move
    other = [r.pool._free.pop() for _ in range(5)]
    b = r.generate(prompt, 60, use_graph=False)
    c = r.generate(prompt, 60)
    assert torch.equal(a, b) and torch.equal(a, c)
    r.pool._free.extend(other)
    r.reset()
    assert r.pool.free == 40
    r.check_device_error()
    r.release_graphs()


def test_decoding_a_sequence_that_grows():
    """Pages added between replays of one captured step: the same ids as with all of them from the start."""
    shape = _small()
    r = _runner(shape, page_size=16, num_pages=24)
    prompt = torch.randint(0, shape.vocab, (2, 30), device="cuda", generator=torch.Generator("cuda").manual_seed(9))
    want = r.generate(prompt, 40)
    r.reset()
    _, nxt = r.prefill(prompt)
    got = [nxt.clone()]
    g, ids, pos, _, next_ids = r.decode_graph(2)
    ids.copy_(nxt.view(2, 1))
    pos.fill_(30)
    for t in range(39):
        r.extend([31 + t] * 2)
        g.replay()
        got.append(next_ids.clone())
    assert torch.equal(torch.stack(got, 1), want)
    r.check_device_error()
    # one more step than there are pages for is reported, not followed
    r.open([16, 16])
    ids.zero_()
    pos.fill_(16)
    g.replay()
    with pytest.raises(RuntimeError, match="page"):
        r.check_device_error()
    r.release_graphs()


def test_cached_rows_of_the_first_layer():
    """The first layer's rows come from equal projections: equal to the contiguous cache's over 16-bit pages up to
    the rounding of the projection (two kernels, one bf16 step), within the 4-bit format's error over 4-bit pages.

    A 4-bit block's scale S is max / 6 rounded to 4 bits: off by 2^-4 of itself at most (max / 6 is above the
    smallest normal scale here, checked). Codes are at most 2 units apart, so one is S = (1 + 2^-4) max / 6 off at
    most, or at the top, where 6 S is below the block's maximum, max / 16: together below 0.18 max."""
    shape = _small()
    prompt = torch.randint(0, shape.vocab, (2, 77), device="cuda", generator=torch.Generator("cuda").manual_seed(10))
    rows = []
    for kw in ({}, dict(page_size=16, num_pages=12), dict(page_size=16, num_pages=12, kv_dtype="fp4")):
        r = _runner(shape, **kw)
        r.prefill(prompt)
        rows.append([t.double().cpu() for t in r.cached_rows(0, 77)])
        assert rows[-1][0].shape == (2, 2, 77, 64)
    for flat, paged, four in zip(*rows):
        # both round the projection and the rotation to bf16: two half steps of the pair's larger element each
        size = flat.abs().reshape(*flat.shape[:-1], 32, 2).amax(-1, keepdim=True).expand(*flat.shape[:-1], 32, 2).reshape(flat.shape)
        assert ((paged - flat).abs() <= 8 * 2.0 ** -8 * size + 1e-30).all()
        top = flat.abs().reshape(*flat.shape[:-1], 4, 16).amax(-1, keepdim=True)
        assert top.min() > 6 * 2.0 ** -6
        bound = (0.18 * 1.04 * top + 8 * 2.0 ** -8 * top).expand(*flat.shape[:-1], 4, 16).reshape(flat.shape)
        assert ((four - flat).abs() <= bound).all()


def test_paged_model_matches_the_source_model():
    """The 0.5B configuration over a paged cache, batch 4, held to the same bounds as over the contiguous cache."""
    from dli.qwen2 import Qwen2Runner
    from dli_export.qwen2 import QWEN2_0_5B, random_state, transform_weights

    shape, prompt, steps, batch = QWEN2_0_5B, 300, 48, 4
    dev = torch.device("cuda:0")
    st = random_state(shape, device=dev, dtype=torch.bfloat16, seed=11, std=0.02)
    hf = model_parity.hf_model(shape, dev, st)
    runner = Qwen2Runner(shape, transform_weights(st, shape, dtype=torch.bfloat16), capacity=512, page_size=64, num_pages=32)
    del st
    ids = torch.randint(0, shape.vocab, (batch, prompt), device=dev, generator=torch.Generator(device=dev).manual_seed(12))
    prefill = runner.prefill
    runner.prefill = lambda p: (runner.open([prompt + steps] * batch), prefill(p))[1]
    stats = model_parity.teacher_forced(runner, hf, ids, steps)
    model_parity.report("qwen2-0.5b paged", stats)
    runner.check_device_error()
    runner.release_graphs()
    model_parity.check_absolute(stats)
    assert np.isfinite(stats["max_logits_rel_err"])
