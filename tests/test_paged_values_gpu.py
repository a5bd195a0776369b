"""Attention over a paged cache (machinelearning_b200/paged.py) where values are
unlike each other or not finite, against the formula in 64 bits.

With scores s and weights p = e^(s - max s) / sum of the same: a score of
-infinity has weight 0 (all of them: the output is zero), one of +infinity
or NaN makes its query head's output NaN; a weight above 0 times an infinite V is
that infinity, 0 times it and the sum of both infinities are NaN. What a query
head or a column of V holds changes no other head's or column's output.

Tolerance of a finite output, u = 2^-24, stated before the first run: that of
``test_paged_gpu.py``, of the sums without the terms that are not finite.
"""
from __future__ import annotations

import numpy as np
import pytest

from test_paged_gpu import SPLIT, U, make_cache

pytestmark = pytest.mark.gpu

HEADS = [(4, 1, 256), (8, 2, 128), (24, 2, 64), (12, 1, 192)]
LENGTHS = [5, 300, 20000, 17]  # the third is divided among CTAs


@pytest.fixture(scope="module")
def torch():
    import torch
    assert torch.cuda.is_available()
    return torch


def dense(cache, pages, b, n):
    """f64 [kv heads][n][head_dim] of a sequence's first n slots."""
    slots = np.arange(n)
    table = cache.block_table[b].cpu().numpy()
    t = pages[table[slots // cache.page_size], :, slots % cache.page_size].double().cpu().numpy()
    return t.transpose(1, 0, 2)


def put(cache, pages, b, slot, head, column, value):
    pages[int(cache.block_table[b, slot // cache.page_size]), head, slot % cache.page_size, column] = value


def reference(cache, q, lengths, scale, split):
    """(out, tolerance) in 64 bits; q is finite."""
    B, nq, hd = q.shape
    g = nq // cache.n_kv_heads
    q = q.double().cpu().numpy()
    out, tol = np.zeros(q.shape), np.full(q.shape, 1e-30)
    for b, n in enumerate(lengths):
        k, v = dense(cache, cache.k, b, n), dense(cache, cache.v, b, n)
        for h in range(nq):
            kk, vv = k[h // g], v[h // g]
            with np.errstate(invalid="ignore", over="ignore"):
                s = (kk * q[b, h]).sum(-1) * scale
                finite = np.isfinite(s)
                if np.isneginf(s).all():
                    continue
                e = (np.abs(kk[finite]) @ np.abs(q[b, h])).max(initial=0.0) * scale * (split + hd * U)
                p = np.exp(s - s.max())
                p /= p.sum()
                out[b, h] = (p[:, None] * vv).sum(0)
                tol[b, h] += p @ np.where(np.isfinite(vv), np.abs(vv), 0.0) * (2 * e + split + 2.0 ** -20)
    return out, tol


def check(got, ref, tol):
    got = got.double().cpu().numpy()
    np.testing.assert_array_equal(np.isnan(got), np.isnan(ref))
    off = ~np.isfinite(ref)
    np.testing.assert_array_equal(got[off], ref[off])
    worst = np.max(np.abs(got[~off] - ref[~off]) / tol[~off])
    assert worst <= 1.0, f"off by {worst:.2f} times the tolerance"


def problem(torch, dtype, nq, nkv, hd, seed):
    cache = make_cache(torch, len(LENGTHS), max(LENGTHS), nkv, hd, dtype, 16, seed=seed)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    q = torch.randn(len(LENGTHS), nq, hd, generator=gen, device="cuda")
    return cache, q, torch.tensor(LENGTHS, dtype=torch.int32, device="cuda"), hd ** -0.5


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("nq,nkv,hd", HEADS)
@pytest.mark.parametrize("outlier", [2.0 ** 15, -3e4, 2.0 ** 7])
def test_attend_queries_with_an_outlier(torch, dtype, nq, nkv, hd, outlier):
    """One element of a query far above the others, where the keys are zero: the
    scores are those of the others, to their own accuracy."""
    cache, q, n, scale = problem(torch, dtype, nq, nkv, hd, 1)
    q[..., 7] = outlier
    cache.k[..., 7] = 0
    check(cache.attend(q, n, scale), *reference(cache, q, LENGTHS, scale, SPLIT[dtype]))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("nq,nkv,hd", HEADS)
def test_attend_infinite_keys(torch, dtype, nq, nkv, hd):
    """Keys with an infinite element: weight 0 for the query heads on its far side,
    NaN for those on its near side."""
    cache, q, n, scale = problem(torch, dtype, nq, nkv, hd, 2)
    q[..., 3] = 1.0   # exact in every type: its other parts are zero
    q[:, 1::2, 3] = 0.7
    for b, slots in enumerate(([0, 4], [16, 299], [0, 9000, 19999], [16])):
        for i, slot in enumerate(slots):
            put(cache, cache.k, b, slot, i % nkv, 3, float("-inf"))
    ref = reference(cache, q, LENGTHS, scale, SPLIT[dtype])
    assert np.isfinite(ref[0]).all()
    check(cache.attend(q, n, scale), *ref)
    q[0, 0, 3], q[2, nq - 1, 3] = -1.0, -0.3
    put(cache, cache.k, 2, 12345, nkv - 1, 3, float("-inf"))
    ref = reference(cache, q, LENGTHS, scale, SPLIT[dtype])
    assert np.isnan(ref[0]).all(-1).sum() == 2
    check(cache.attend(q, n, scale), *ref)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_attend_weights_of_infinite_keys(torch, dtype):
    """The slots' weights: 0 where the key is infinite; and all keys infinite: zeros."""
    nq, nkv, hd = 8, 2, 128
    cache, q, n, scale = problem(torch, dtype, nq, nkv, hd, 3)
    q[..., 3] = 0.9
    for slot in range(5):
        put(cache, cache.k, 0, slot, 0, 3, float("-inf"))
    put(cache, cache.k, 1, 77, 1, 3, float("-inf"))
    w = torch.zeros(len(LENGTHS), nkv, cache.capacity, device="cuda")
    out = cache.attend(q, n, scale, weights=w)
    check(out, *reference(cache, q, LENGTHS, scale, SPLIT[dtype]))
    assert not out[0, :4].any() and not w[0, 0].any() and out[0, 4:].any()
    assert float(w[1, 1, 77]) == 0.0
    np.testing.assert_allclose(w.sum(-1).cpu().numpy(), [[0, 4]] + [[4, 4]] * 3, rtol=1e-5)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_attend_queries_that_are_not_finite(torch, dtype):
    """NaN and infinite queries: NaN for their own head, and the others as without them."""
    cache, q, n, scale = problem(torch, dtype, 24, 2, 64, 5)
    ref, tol = reference(cache, q, LENGTHS, scale, SPLIT[dtype])
    bad = q.clone()
    bad[0, 1, 5], bad[1, 13, 0], bad[2, 23, 63] = float("nan"), float("inf"), float("-inf")
    for b, h in ((0, 1), (1, 13), (2, 23)):
        ref[b, h] = np.nan
    check(cache.attend(bad, n, scale), ref, tol)


def test_attend_f16_overflow_from_append(torch):
    """A key beyond f16's range is an infinity in the cache: its slot has weight 0
    for a query on its far side."""
    cache = make_cache(torch, 1, 64, 1, 64, "f16", 16, seed=6)
    qkv = torch.randn(1, 3 * 64, device="cuda")
    qkv[0, 0], qkv[0, 64], qkv[0, 128 + 5] = 1.0, -7e4, 7e4
    one = torch.ones(1, 32, device="cuda")
    n = torch.tensor([33], dtype=torch.int32, device="cuda")
    q = cache.append(qkv, torch.zeros_like(n), n - 1, one, torch.zeros_like(one), n_heads=1)
    got = cache.attend(q, n - 32, 0.125)  # one other slot alone
    assert torch.isfinite(got).all()
    with_it = cache.attend(q, n, 0.125)
    ref, tol = reference(cache, q, [33], 0.125, SPLIT["f16"])
    assert np.isnan(ref[0, 0, 5]) and np.isfinite(ref[0, 0]).sum() == 63  # weight 0 times the infinite value
    check(with_it, ref, tol)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("nq,nkv,hd", HEADS)
def test_attend_infinite_values(torch, dtype, nq, nkv, hd):
    """Values with infinities and NaN: their own columns only, of the kv head's query heads."""
    cache, q, n, scale = problem(torch, dtype, nq, nkv, hd, 4)
    inf, nan = float("inf"), float("nan")
    for b, slots in enumerate(([0, 3], [31, 150], [5, 19990], [8, 16])):
        put(cache, cache.v, b, slots[0], 0, 0, inf)
        put(cache, cache.v, b, slots[1], 0, 0, inf)
        put(cache, cache.v, b, slots[0], 0, 9, -inf)
        put(cache, cache.v, b, slots[0], nkv - 1, hd - 1, inf)
        put(cache, cache.v, b, slots[1], nkv - 1, hd - 1, -inf)  # both: NaN
        put(cache, cache.v, b, slots[1], nkv - 1, 40, nan)
    q[..., 3] = 1.0
    put(cache, cache.k, 1, 10, 0, 3, -inf)  # weight 0 of an infinity: NaN
    put(cache, cache.v, 1, 10, 0, 33, inf)
    ref = reference(cache, q, LENGTHS, scale, SPLIT[dtype])
    g = nq // nkv
    assert (ref[0][:, :g, 0] == inf).all() and (ref[0][:, :g, 9] == -inf).all()
    assert np.isnan(ref[0][:, -g:, hd - 1]).all() and np.isnan(ref[0][1, :g, 33]).all()
    check(cache.attend(q, n, scale), *ref)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("nq,nkv,hd", HEADS + [(16, 1, 128), (1, 1, 64), (9, 1, 256)])
def test_attend_is_as_exact_as_32_bit_arithmetic(torch, dtype, nq, nkv, hd):
    """Per query head, the distance from 64 bits is at most four times that of
    the formula in elementary 32-bit operations on the same inputs, or 1e-6 of
    the output's norm where that happens to be smaller."""
    lengths = [1, 40, 512, 6000]
    cache = make_cache(torch, 4, 6000, nkv, hd, dtype, 16, seed=hd)
    gen = torch.Generator(device="cuda").manual_seed(nq)
    q = torch.randn(4, nq, hd, generator=gen, device="cuda") * 2
    scale, g = hd ** -0.5, nq // nkv
    got = cache.attend(q, torch.tensor(lengths, dtype=torch.int32, device="cuda"), scale).double()
    for b, n in enumerate(lengths):
        slots = torch.arange(n, device="cuda")
        rows = cache.block_table[b].long()[slots // 16]
        k, v = (t[rows, :, slots % 16].transpose(0, 1).repeat_interleave(g, 0) for t in (cache.k, cache.v))

        def formula(kind):
            s = torch.matmul(k.to(kind), q[b].to(kind)[:, :, None])[..., 0] * scale
            e = torch.exp(s - s.amax(-1, keepdim=True))
            return torch.matmul((e / e.sum(-1, keepdim=True))[:, None, :], v.to(kind))[:, 0]
        ref = formula(torch.float64)
        size = ref.norm(dim=-1)
        plain = (formula(torch.float32).double() - ref).norm(dim=-1) / size
        mine = (got[b] - ref).norm(dim=-1) / size
        assert torch.all(mine <= torch.clamp(4 * plain, min=1e-6)), (mine.max(), plain.max())
