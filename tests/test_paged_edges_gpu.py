"""Paged KV cache on the GPU at the calls where a rule of its kernels ends: head counts that no CTA divides evenly,
NaN in every place and pattern, scales that underflow, rings that keep turning over bad or forgotten pages, tables
that change under a captured step, workspaces of calls with a window."""
from __future__ import annotations

import pytest
import torch

import dli_sm100 as C
import test_paged_long_gpu as long

pytestmark = pytest.mark.gpu


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
