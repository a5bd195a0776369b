"""Calls at the edge of what the paged entry points take, on a CPU host: argument
checks come before any device work, so the pointers are never dereferenced."""
from __future__ import annotations

import ctypes

import pytest

from test_paged import INVALID, OK, P, append, attend, desc, evict


@pytest.mark.parametrize("change", [{"table_dev": 0}, {"table_dev": 0, "k_dev": 0, "v_dev": 0, "n_pages": 0}])
def test_no_sequences_need_no_memory(qlib, change):
    """A batch that has run empty: its table has no storage, nor has a pool of no pages."""
    kv = ctypes.byref(desc(n_seqs=0, **change))
    assert attend(qlib, kv, q=None, lengths=None, out=None) == OK
    assert evict(qlib, kv, w=None, pos=None) == OK
    assert append(qlib, kv, tokens=0, qkv=None) == OK
    assert qlib.qmm_paged_attention_workspace_size(kv, 4, 1) > 0
    one = desc(n_seqs=1, **change)
    assert attend(qlib, ctypes.byref(one)) == INVALID and append(qlib, ctypes.byref(one)) == INVALID


def test_histories_whose_counts_would_not_fit(qlib):
    """A count of 2^30 would run into the flags beside it."""
    from test_paged import SHAPE, logits
    for n in (1 << 30, (1 << 31) - 1):
        assert logits(qlib, tokens=P, lens=P, ld_tokens=n, n=n) == SHAPE
        assert b"history" in qlib.qmm_last_error_message()
