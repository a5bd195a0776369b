"""Paged key/value cache and logits processing on a CPU host: what the entry
points and their Python forms refuse, and with which error. Argument checks
come before any device work, so the pointers below are never dereferenced."""
from __future__ import annotations

import ctypes

import pytest
import torch

OK, SHAPE, DTYPE, INVALID = 0, 2, 3, 8
P = 1 << 20  # a 16-byte aligned address that is never read


def desc(**changes):
    from machinelearning_b200 import _lib
    kv = dict(k_dev=P, v_dev=2 * P, dtype=_lib.KV_BF16, n_kv_heads=2, head_dim=128, page_size=16, n_pages=8,
              page_stride=2 * 16 * 128, head_stride=16 * 128, slot_stride=128, table_dev=3 * P, n_seqs=3, max_pages=4,
              table_stride=4)
    kv.update(changes)
    return _lib.PagedKv(*kv.values())


BAD_CACHES = [({"k_dev": 0}, INVALID), ({"v_dev": 0}, INVALID), ({"table_dev": 0}, INVALID), ({"dtype": 2}, DTYPE),
              ({"head_dim": 96}, SHAPE), ({"head_dim": 320}, SHAPE), ({"head_dim": 0}, SHAPE),
              ({"n_kv_heads": 0}, SHAPE), ({"n_seqs": -1}, SHAPE), ({"max_pages": 0}, SHAPE), ({"n_pages": -1}, SHAPE),
              ({"n_pages": 1 << 31}, SHAPE), ({"page_size": 8}, SHAPE), ({"page_size": 24}, SHAPE),
              ({"page_size": 2048}, SHAPE), ({"max_pages": 1 << 27}, SHAPE), ({"slot_stride": 64}, SHAPE),
              ({"page_stride": -4096}, SHAPE), ({"slot_stride": 132}, INVALID), ({"k_dev": P + 8}, INVALID)]


def append(lib, kv, qkv=P, ld=1024, tokens=1, nq=4, qn=P, kn=P, cos=P, ctx=16, pos=P, slots=P, out=P):
    return lib.qmm_paged_append_dev(kv, qkv, ld, tokens, nq, qn, kn, 0.0, 1e-6, cos, P, ctx, 0, pos, slots, None, out,
                                    None)


def attend(lib, kv, q=P, ld=512, nq=4, lengths=P, window=0, w=None, w_out=None, out=P):
    return lib.qmm_paged_attention_dev(kv, q, ld, nq, lengths, 1.0, window, w, w_out, out, None)


def evict(lib, kv, w=P, pos=P, budget=8, recent=2, lens_out=2 * P, w_out=2 * P, pos_out=2 * P):
    return lib.qmm_paged_evict_dev(kv, P, w, pos, P, budget, recent, lens_out, w_out, pos_out, None)


def logits(lib, x=P, ld=100, rows=2, vocab=100, tokens=None, ld_tokens=0, n=0, lens=None, ids=None, vals=None, nb=0,
           mask=None, n_masks=0, mask_rows=None, out=2 * P, ld_out=100):
    return lib.qmm_process_logits_dev(x, ld, rows, vocab, tokens, ld_tokens, n, lens, None, None, None, None, ids, vals,
                                      nb, mask, n_masks, mask_rows, out, ld_out, None)


@pytest.mark.parametrize("change,status", BAD_CACHES)
def test_bad_cache_is_refused_by_every_entry(qlib, change, status):
    kv = ctypes.byref(desc(**change))
    assert append(qlib, kv) == status
    assert attend(qlib, kv) == status
    assert evict(qlib, kv) == status
    assert qlib.qmm_paged_attention_workspace_size(kv, 4, 1) == 0
    assert qlib.qmm_paged_evict_workspace_size(kv, 8) == 0
    assert qlib.qmm_last_error_message()


@pytest.mark.parametrize("args,status", [
    (dict(nq=3), SHAPE), (dict(nq=0), SHAPE), (dict(qkv=None), INVALID), (dict(cos=None), INVALID),
    (dict(pos=None), INVALID), (dict(slots=None), INVALID), (dict(out=None), INVALID), (dict(qn=None), INVALID),
    (dict(kn=None), INVALID), (dict(ld=1020), SHAPE), (dict(ld=1026), INVALID), (dict(ctx=0), SHAPE),
    (dict(tokens=1 << 40), SHAPE), (dict(qkv=P + 4), INVALID), (dict(out=P + 4), INVALID), (dict(qn=P + 8), INVALID),
    (dict(tokens=0, qkv=None), OK)])
def test_append_refusals(qlib, args, status):
    assert append(qlib, ctypes.byref(desc()), **args) == status


@pytest.mark.parametrize("args,status", [
    (dict(nq=3), SHAPE), (dict(q=None), INVALID), (dict(lengths=None), INVALID), (dict(out=None), INVALID),
    (dict(w=P), INVALID), (dict(w_out=P), INVALID), (dict(ld=508), SHAPE), (dict(ld=514), INVALID),
    (dict(window=-1), SHAPE), (dict(q=P + 4), INVALID)])
def test_attention_refusals(qlib, args, status):
    assert attend(qlib, ctypes.byref(desc()), **args) == status


@pytest.mark.parametrize("args,status", [
    (dict(w=None), INVALID), (dict(pos=None), INVALID), (dict(w_out=None), INVALID), (dict(w_out=P), INVALID),
    (dict(pos_out=P), INVALID), (dict(lens_out=P), INVALID), (dict(budget=0), SHAPE), (dict(recent=-1), SHAPE),
    (dict(recent=9), SHAPE)])
def test_evict_refusals(qlib, args, status):
    assert evict(qlib, ctypes.byref(desc()), **args) == status


@pytest.mark.parametrize("args,status", [
    (dict(x=None), INVALID), (dict(out=None), INVALID), (dict(ld=99), SHAPE), (dict(ld_out=99), SHAPE),
    (dict(rows=70000), SHAPE), (dict(tokens=P, ld_tokens=4, n=4), INVALID),
    (dict(tokens=P, lens=P, ld_tokens=3, n=4), SHAPE), (dict(ids=P, nb=4), INVALID),
    (dict(ids=P, vals=P, nb=1025), SHAPE), (dict(mask=P, n_masks=1), SHAPE),
    (dict(out=P, ld=100, ld_out=104), INVALID), (dict(rows=0, x=None), OK), (dict(vocab=0), OK)])
def test_logits_refusals(qlib, args, status):
    assert logits(qlib, **args) == status


def test_empty_batches_do_nothing(qlib):
    kv = ctypes.byref(desc(n_seqs=0))
    assert attend(qlib, kv) == OK and evict(qlib, kv) == OK


def test_python_forms_refuse_host_tensors(qlib):
    from machinelearning_b200 import _lib
    from machinelearning_b200.logits import process_logits
    from machinelearning_b200.paged import PagedKVCache
    k = torch.zeros(2, 1, 16, 64)
    table = torch.zeros(1, 2, dtype=torch.int32)
    with pytest.raises(ValueError, match="GPU"):
        PagedKVCache(k, k.clone(), table)
    with pytest.raises(_lib.DTypeMismatch):
        PagedKVCache(k.double(), k.double(), table)
    with pytest.raises(_lib.ShapeMismatch):
        PagedKVCache(k, k[:1], table)
    with pytest.raises(_lib.ShapeMismatch):
        PagedKVCache(k, k.clone(), table.long())
    with pytest.raises(ValueError, match="GPU"):
        process_logits(torch.zeros(1, 4))
    with pytest.raises(_lib.DTypeMismatch):
        process_logits(torch.zeros(1, 4, dtype=torch.float16))
    with pytest.raises(_lib.ShapeMismatch):
        process_logits(torch.zeros(4))
