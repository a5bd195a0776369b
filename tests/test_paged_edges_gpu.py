"""Caches and arguments at the edge of what the Python forms take (machinelearning_b200/paged.py)."""
from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch
    assert torch.cuda.is_available()
    return torch


@pytest.mark.parametrize("pages", [0, 4])
def test_empty_batches(torch, pages):
    from machinelearning_b200.paged import PagedKVCache
    k = torch.randn(pages, 2, 16, 64, device="cuda")
    ints = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")  # noqa: E731
    cache = PagedKVCache(k, k.clone(), ints(0, 3))
    q = torch.empty(0, 4, 64, device="cuda")
    w = torch.empty(0, 2, 48, device="cuda")
    assert cache.attend(q, ints(0), 1.0).shape == (0, 4, 64)
    assert cache.attend(q, ints(0), 1.0, weights=w).shape == (0, 4, 64)
    assert [t.shape for t in cache.evict(ints(0), w, ints(0, 2, 48), ints(0), 8, 2)] == [(0,), (0, 2, 48), (0, 2, 48)]
    one = torch.ones(4, 32, device="cuda")
    assert cache.append(torch.empty(0, 8 * 64, device="cuda"), ints(0), ints(0), one, one, n_heads=4).shape == (0, 4, 64)
    # tokens of sequences that are gone: their queries, and nothing stored
    qkv = torch.randn(3, 8 * 64, device="cuda")
    before = k.clone()
    got = cache.append(qkv, ints(3), ints(3), one, torch.zeros_like(one), n_heads=4, seqs=ints(3))
    assert torch.equal(got.view(3, -1), qkv[:, :4 * 64]) and torch.equal(cache.k, before)
    assert PagedKVCache.allocate(0, 48, 2, 64).attend(q, ints(0), 1.0).shape == (0, 4, 64)


def test_strides_of_dimensions_of_size_one_do_not_matter(torch):
    """K and V from differently laid out pools that are alike but for such a stride, or
    whose stride there is no multiple of 16 bytes."""
    from machinelearning_b200.paged import PagedKVCache
    n = torch.tensor([40], dtype=torch.int32, device="cuda")
    table = torch.tensor([[2, 0, 1]], dtype=torch.int32, device="cuda")
    k = torch.randn(3, 16, 1, 64, device="cuda").transpose(1, 2)  # [slot][head] pages
    v = torch.randn(3, 1, 16, 64, device="cuda")                  # [head][slot] pages
    assert k.shape == v.shape and k.stride() != v.stride()
    q = torch.randn(1, 4, 64, device="cuda")
    want = PagedKVCache(k.contiguous(), v, table).attend(q, n, 0.1)
    assert torch.equal(PagedKVCache(k, v, table).attend(q, n, 0.1), want)
    odd = v.as_strided(v.shape, (1024, 1023, 64, 1))
    assert torch.equal(PagedKVCache(k, odd, table).attend(q, n, 0.1), want)
    assert torch.equal(PagedKVCache(odd, odd, table).attend(q, n, 0.1), PagedKVCache(v, v, table).attend(q, n, 0.1))
    one_page = v[:1].as_strided((1, 1, 16, 64), (1, 1, 64, 1))
    table0 = torch.zeros(1, 1, dtype=torch.int32, device="cuda")
    assert torch.equal(PagedKVCache(one_page, one_page, table0).attend(q, n, 0.1),
                       PagedKVCache(v[:1], v[:1], table0).attend(q, n, 0.1))


def test_reserve_refuses_what_attend_would(torch):
    from machinelearning_b200 import _lib
    from machinelearning_b200.paged import PagedKVCache
    cache = PagedKVCache.allocate(1, 64, 2, 64)
    cache.reserve(4, weights=True, budget=10)
    for heads in (3, 0, -2):
        with pytest.raises(_lib.ShapeMismatch):
            cache.reserve(heads)
    with pytest.raises(ValueError):
        cache.reserve(4, budget=-1)


@pytest.mark.parametrize("n_seqs", [1, 2, 31, 32, 33, 64, 159, 160, 161, 288, 289, 1025])
@pytest.mark.parametrize("kind", ["short", "one long", "last alone", "empty"])
def test_any_number_of_sequences(torch, n_seqs, kind):
    """The division of the work over many sequences, most of them empty or short, one or two
    divided among CTAs; with and without weights."""
    import numpy as np

    from test_paged_gpu import SPLIT, attend_ref, check, make_cache
    rng = np.random.default_rng(n_seqs)
    longest = 600 if n_seqs > 64 else 3000
    lengths = rng.integers(0, 40, n_seqs)
    if kind == "one long":
        lengths[n_seqs // 2] = longest
    if kind == "last alone":
        lengths[:] = 0
        lengths[-1] = longest
    if kind == "empty":
        lengths[:] = 0
    lengths = lengths.tolist()
    cache = make_cache(torch, n_seqs, longest, 1, 64, "f16", 16, seed=n_seqs)
    q = torch.randn(n_seqs, 3, 64, device="cuda")
    n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    w = torch.zeros(n_seqs, 1, cache.capacity, device="cuda")
    ref, tol, wr, wtol = attend_ref(cache, q, lengths, 0.125, 0, SPLIT["f16"])
    out = cache.attend(q, n, 0.125)
    check(out, ref, tol)
    assert torch.equal(cache.attend(q, n, 0.125, weights=w), out)
    check(w, wr, wtol)


@pytest.mark.parametrize("same,n", [(2, 1024), (9, 1024), (700, 1024), (1024, 1024), (3, 3), (40, 64)])
def test_logits_many_biases_of_one_token(torch, same, n):
    """A bias list padded with one id, and tokens that come up a few times: the values are added
    one after the other in the list's order, in 32 bits."""
    import numpy as np

    from machinelearning_b200.logits import process_logits
    rng = np.random.default_rng(same)
    rows, vocab = 3, 40000
    ids = rng.integers(0, vocab, (rows, n)).astype(np.int32)
    ids[:, rng.permutation(n)[:same]] = 7
    ids[1, :2] = 39999
    vals = rng.normal(0, 5, (rows, n)).astype(np.float32)
    x = rng.normal(0, 4, (rows, vocab)).astype(np.float32)
    want = x.copy()
    for r in range(rows):
        for t, v in zip(ids[r], vals[r]):
            want[r, t] = np.float32(want[r, t] + v)
    cu = lambda a: torch.from_numpy(a).cuda()  # noqa: E731
    got = process_logits(cu(x), bias_ids=cu(ids), bias_values=cu(vals))
    np.testing.assert_array_equal(got.cpu().numpy(), want)
