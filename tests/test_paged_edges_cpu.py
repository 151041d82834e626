"""Paged KV cache, without a GPU: calls whose refusal, size or dtype is decided on the host alone."""
from __future__ import annotations

import pytest

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
