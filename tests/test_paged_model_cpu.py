"""CPU tests of the paged KV cache in the Qwen2 path: the exported graph, the graph
run by the 64-bit interpreter against the contiguous cache, the page pool, and what
the runner and the operators refuse before any GPU is touched."""
from __future__ import annotations

import json

import numpy as np
import pytest
import torch

import dli
from dli.pages import PagePool
from dli_export.qwen2 import Qwen2Shape, build_graph, export_qwen2, random_state, rotary_tables, transform_weights
from oracle.graph import GraphOracle

TINY = Qwen2Shape(hidden=64, layers=2, q_heads=4, kv_heads=2, head_dim=16, intermediate=96, vocab=50)


def test_graph_of_a_paged_cache():
    g = build_graph(TINY, 64, page_size=16, num_pages=12)
    ops = [n["op"] for n in g["nodes"]]
    assert ops.count("qkv_rotary_paged") == ops.count("attention_paged") == TINY.layers
    assert not {"qkv_rotary_cache", "linear_qkv_rotary_cache", "attention_kvcache"} & set(ops)
    assert g["inputs"] == ["input_ids", "positions", "page_table"]
    append = next(n for n in g["nodes"] if n["op"] == "qkv_rotary_paged")
    assert append["inputs"] == ["layers.0.qkv", "rotary_cos", "rotary_sin", "positions", "page_table"]
    assert append["attrs"] == {"q_heads": 4, "kv_heads": 2, "head_dim": 16, "kv_cache": "layer_0", "page_size": 16,
                               "num_pages": 12}
    four = build_graph(TINY, 64, tp_size=2, page_size=32, num_pages=3, kv_dtype="fp4")
    append = next(n for n in four["nodes"] if n["op"] == "qkv_rotary_paged")
    assert append["attrs"]["kv_dtype"] == "fp4" and append["attrs"]["kv_heads"] == 1
    assert dli.Graph.from_json(json.dumps(four)).inputs[-1] == "page_table"
    # without pages the graph is the one it was
    assert build_graph(TINY, 64) == build_graph(TINY, 64, page_size=0, num_pages=0, kv_dtype=None)


@pytest.mark.parametrize("bad", [dict(page_size=16), dict(num_pages=4), dict(page_size=-16, num_pages=4),
                                 dict(kv_dtype="fp4"), dict(page_size=16, num_pages=4, kv_dtype="fp8")])
def test_graph_refusals(bad):
    with pytest.raises(ValueError):
        build_graph(TINY, 64, **bad)


def test_export_with_a_paged_cache(tmp_path):
    st = random_state(TINY, dtype=torch.bfloat16, seed=1)
    gpath, _ = export_qwen2(st, tmp_path, "tiny", shape=TINY, capacity=64, page_size=16, num_pages=8, kv_dtype="fp4")
    assert dli.Graph.from_json_file(str(gpath)).inputs == ["input_ids", "positions", "page_table"]


def _interpreters(**paged):
    st = random_state(TINY, dtype=torch.float32, seed=5, std=0.1)
    cos, sin = rotary_tables(TINY, 64)
    consts = {k: v.double().numpy() for k, v in transform_weights(st, TINY, dtype=torch.float32).items()}
    consts.update(rotary_cos=cos.numpy(), rotary_sin=sin.numpy())
    return GraphOracle(build_graph(TINY, 64, **paged), consts)


def _prompt_and_steps(run, table):
    r = np.random.default_rng(3)
    ids = r.integers(0, TINY.vocab, (2, 21))
    feed = {} if table is None else {"page_table": table}
    outs = [run.run({"input_ids": ids, "positions": np.zeros(2, np.int64), **feed})["logits"]]
    for t in range(13):  # across a page's end
        step = r.integers(0, TINY.vocab, (2, 1))
        outs.append(run.run({"input_ids": step, "positions": np.full(2, 21 + t), **feed})["logits"])
    return np.stack(outs)


def test_interpreted_paged_graph_equals_the_contiguous_one():
    table = np.array([[7, 2, 5, -1], [0, 6, 3, -1]], np.int32)
    want = _prompt_and_steps(_interpreters(), None)
    got = _prompt_and_steps(_interpreters(page_size=16, num_pages=8), table)
    # the same sums in another order, in 64 bits: some 10^4 additions of 2^-53 each
    np.testing.assert_allclose(got, want, rtol=0, atol=1e4 * 2.0 ** -53 * np.abs(want).max())
    four = _prompt_and_steps(_interpreters(page_size=16, num_pages=8, kv_dtype="fp4"), table)
    # 4-bit rows move the logits, and by less than they are large
    rel = np.linalg.norm(four - want) / np.linalg.norm(want)
    assert 1e-6 < rel < 1.0


def test_page_pool():
    pool = PagePool(6, 16)
    a, b = [], []
    pool.grow([a, b], [33, 16])
    assert len(a) == 3 and len(b) == 1 and pool.free == 2 and not set(a) & set(b)
    first = list(a)
    pool.grow([a, b], [40, 17])  # a has room, b needs one more
    assert a == first and len(b) == 2 and pool.free == 1
    with pytest.raises(MemoryError):
        pool.grow([a, b], [49, 33])
    assert a == first and len(b) == 2 and pool.free == 1  # none given
    pool.grow([a, b], [0, 0])
    assert len(a) == 3 and len(b) == 2
    with pytest.raises(ValueError):
        pool.grow([a], [-1])
    with pytest.raises(ValueError):
        pool.grow([a], [1, 2])
    twice = list(a)
    pool.give_back(a)
    assert a == [] and pool.free == 4
    for bad in (twice, [6], [b[0], b[0]]):
        with pytest.raises(ValueError):
            pool.give_back(bad)
    pool.give_back(b)
    assert pool.free == 6
    for size in ((0, 16), (4, 0)):
        with pytest.raises(ValueError):
            PagePool(*size)


def _runner(**kw):
    from dli.qwen2 import Qwen2Runner

    st = random_state(TINY, dtype=torch.bfloat16, seed=1)
    return Qwen2Runner(TINY, transform_weights(st, TINY, dtype=torch.bfloat16), capacity=64, **kw)


def test_runner_opens_extends_and_closes_sequences():
    r = _runner(page_size=16, num_pages=7)
    r.open([17, 64])
    table = r.page_table(2)
    address = table.data_ptr()
    assert table.shape == (2, 4) and (table >= 0).sum(1).tolist() == [2, 4] and r.pool.free == 1
    assert sorted(p for s in r.sequences for p in s) == sorted(x for x in table.flatten().tolist() if x >= 0)
    before = table.clone()
    r.extend([33, 64])
    assert r.pool.free == 0 and torch.equal(table[:, :2], before[:, :2]) and int(table[0, 2]) >= 0
    with pytest.raises(MemoryError):
        r.extend([64, 64])
    assert (table[0] >= 0).sum() == 3  # left as it was
    r.open([16])
    assert r.pool.free == 6 and (table == -1).all() and int(r.page_table(1)[0, 0]) >= 0
    r.open([5, 5])
    assert r.page_table(2).data_ptr() == address
    r.reset()
    assert r.pool.free == 7 and not r.sequences and (r.page_table(2) == -1).all()


def test_runner_refusals():
    r = _runner(page_size=16, num_pages=4)
    for rows in ([], [65], [-1]):
        with pytest.raises(ValueError):
            r.open(rows)
    with pytest.raises(MemoryError):
        r.open([64, 16])
    assert r.pool.free == 4 and not r.sequences
    with pytest.raises(ValueError):
        r.extend([16])
    with pytest.raises(ValueError):
        r.forward(torch.zeros(1, 3, dtype=torch.int64), torch.zeros(1, dtype=torch.int64))
    contiguous = _runner()
    with pytest.raises(ValueError):
        contiguous.open([16])
    contiguous.reset()
    for kw in (dict(page_size=16), dict(kv_dtype="fp4")):
        with pytest.raises(ValueError):
            _runner(**kw)


def test_operators_are_registered_and_refuse_host_tensors():
    e = dli.Engine()
    e.load_library(dli.PLUGIN_PATH)
    for op, n in (("qkv_rotary_paged", 5), ("attention_paged", 3)):
        assert e.has_operator(op)
        names = [f"i{j}" for j in range(n)]
        for count in (n, n - 1):  # host tensors, then too few
            g = dli.Graph.from_json(json.dumps({"format": "dli.graph.v1", "inputs": names, "outputs": ["o"], "nodes": [
                {"name": "x", "op": op, "inputs": names[:count], "outputs": ["o"], "attrs": {"kv_cache": "c"}}]}))
            with pytest.raises(ValueError):
                e.run(g, {k: torch.zeros(2, 2) for k in names})
