"""Paged KV cache, without a GPU: calls whose refusal, size or dtype is decided on the host alone."""
from __future__ import annotations

import json

import pytest
import torch

import dli
import dli_sm100 as C
import test_paged_cpu as calls


@pytest.mark.parametrize("fp4", [False, True], ids=["rows16", "rows4"])
def test_a_table_is_needed_for_a_pool_of_no_pages_too(fp4):
    """Rows are looked up in the table before it is known that the pool has none."""
    kv = {"kv": calls.FP4} if fp4 else {}
    L = C.lib()
    for fn, args in ((L.dli_sm100_qkv_rotary_paged, calls.append_args), (L.dli_sm100_attention_paged, calls.attend_args),
                     (L.dli_sm100_paged_gather, calls.gather_args)):
        assert fn(*args(table=None, pages=0, **kv)) == calls.INVALID, C.last_error()
        assert "page_table" in C.last_error()


class _OnDevice:
    """A tensor that says it lies on a GPU."""

    def __init__(self, t, device):
        self.t, self.index = t, device

    def get_device(self):
        return self.index

    def __getattr__(self, name):
        return getattr(self.t, name)


def test_the_workspace_is_of_the_tensors_device(monkeypatch):
    """Its size goes by the device's SMs: asked for with that device current, and not kept for another one."""
    current, sms = [0], {0: 148, 1: 200}
    asked, given = [], []

    class Device:
        def __init__(self, index):
            self.index = index

        def __enter__(self):
            self.held, current[0] = current[0], self.index

        def __exit__(self, *a):
            current[0] = self.held

    class Lib:
        def dli_sm100_attention_paged_workspace_size(self, *sizes):
            asked.append(current[0])
            return sms[current[0]] * 16

        def dli_sm100_attention_paged(self, *args):
            given.append((current[0], args[-2]))
            return C.DLI_OK

    monkeypatch.setattr(C, "lib", Lib)
    monkeypatch.setattr(torch.cuda, "device", Device)
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: current[0], raising=False)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: 0, raising=False)
    C._attention_paged_workspace.cache_clear()
    k, v = (torch.zeros(3, 2, 16, 64, dtype=torch.bfloat16) for _ in (0, 1))
    q, table, pos = torch.zeros(2, 4, 64, dtype=torch.bfloat16), torch.zeros(2, 2, dtype=torch.int32), torch.zeros(2, dtype=torch.int64)
    try:
        for device in (0, 1, 1, 0):
            C.attention_paged(*(_OnDevice(t, device) for t in (q, k, v, pos, table)), out=_OnDevice(q.clone(), device))
    finally:
        C._attention_paged_workspace.cache_clear()
    assert given == [(0, 148 * 16), (1, 200 * 16), (1, 200 * 16), (0, 148 * 16)]
    assert asked == [0, 1] and current == [0]


def test_bytes_do_not_enter_the_engine(tmp_path):
    """uint8 is the type of a 4-bit pool's pages inside the engine: no input, constant, weight or operand has it."""
    e = dli.Engine()
    e.load_library(dli.PLUGIN_PATH)
    g = dli.Graph.from_json(json.dumps({"format": "dli.graph.v1", "inputs": ["x"], "outputs": ["y"], "nodes": [
        {"name": "n", "op": "reshape", "inputs": ["x"], "outputs": ["y"], "attrs": {"shape": [4]}}]}))
    for call in (lambda t: e.run(g, {"x": t}), lambda t: e.set_constants({"x": t})):
        with pytest.raises(ValueError, match="unsupported torch tensor dtype"):
            call(torch.zeros(2, 2, dtype=torch.uint8))
    (tmp_path / "w.bin").write_bytes(bytes(4))
    (tmp_path / "w.json").write_text(json.dumps({"format": "dli.weights.v1", "data": "w.bin", "tensors": {
        "a": {"dtype": "uint8", "shape": [4], "offset": 0, "nbytes": 4}}}))
    with pytest.raises(ValueError, match="unknown dtype"):
        dli.load_weights(str(tmp_path / "w.json"))
