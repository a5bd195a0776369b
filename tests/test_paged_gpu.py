"""The paged serving operators (machinelearning_b200/paged.py, logits.py) on the
GPU against the formulas in 64 bits.

Tolerances, u = 2^-24 (f32), t = the cache type's unit roundoff (f32 0, f16
2^-11, bf16 2^-8), stated before the first run:

* append: a sum of 256 squares in tree order, a root, a reciprocal and five
  products: at most 16 u of the rotated pair's |a| + |b|, 1.5e-6 with a margin;
  cache rows add t |x| (and half of f16's smallest subnormal).
* attend: a score is off by at most e = scale * sum |q k| * (r + head_dim u) with r the
  residue of q held as values of the matrix instructions' type (two f16 or tf32
  2^-21, three bf16 less); a weight by a relative 2 e + r + 2^-20 (exponentials and the
  running sums), so an output by that times sum p |v|.
* evict: moves and choices: equal.
* logits: at most eight roundings of values no larger than |x| max(r, 1/r) + f count + p
  + sum |bias|: 8 u of that.
"""
from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
ROUNDOFF = {"f32": 0.0, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
SPLIT = {"f32": 2.0 ** -21, "f16": 2.0 ** -21, "bf16": 2.0 ** -21}
HEADS = [(4, 1, 256), (64, 8, 128), (15, 3, 64), (16, 1, 128), (12, 2, 192), (1, 1, 64), (9, 1, 256), (8, 8, 64)]


@pytest.fixture(scope="module")
def torch():
    import torch
    assert torch.cuda.is_available()
    return torch


def types(torch):
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def make_cache(torch, n_seqs, capacity, nkv, hd, dtype="bf16", page=16, layout="heads", seed=0, spare=3):
    """A cache with random contents whose pages lie in random order. layout: pages of
    [head][slot] ("heads") or [slot][head] ("slots"), or K and V interleaved in one pool ("joint")."""
    from machinelearning_b200.paged import PagedKVCache
    gen = torch.Generator(device="cuda").manual_seed(seed)
    per = -(-capacity // page)
    pages = n_seqs * per + spare
    if layout == "joint":
        pool = torch.randn(pages, 2, nkv, page, hd, generator=gen, device="cuda").to(types(torch)[dtype])
        k, v = pool[:, 0], pool[:, 1]
    elif layout == "slots":
        k, v = (torch.randn(pages, page, nkv, hd, generator=gen, device="cuda").to(types(torch)[dtype]).transpose(1, 2)
                for _ in range(2))
    else:
        k, v = (torch.randn(pages, nkv, page, hd, generator=gen, device="cuda").to(types(torch)[dtype])
                for _ in range(2))
    order = np.random.default_rng(seed).permutation(pages)[:n_seqs * per].astype(np.int32)
    return PagedKVCache(k, v, torch.from_numpy(order.reshape(n_seqs, per)).cuda())


def rows_of(cache, pages, b, slots):
    """f64 [slots][kv heads][head_dim] of a sequence's slots, and which of them have a page."""
    table = cache.block_table[b].cpu().numpy()
    page = table[slots // cache.page_size]
    ok = (page >= 0) & (page < cache.n_pages)
    t = pages[np.where(ok, page, 0), :, slots % cache.page_size].double().cpu().numpy()
    return t, ok


def attend_ref(cache, q, lengths, scale, window, split):
    """(out, out tolerance, weights, weights tolerance) in 64 bits."""
    B, nq, hd = q.shape
    nkv = cache.n_kv_heads
    g = nq // nkv
    q = q.double().cpu().numpy()
    out, tol = np.zeros(q.shape), np.full(q.shape, 1e-30)
    w, wtol = np.zeros((B, nkv, cache.capacity)), np.full((B, nkv, cache.capacity), 1e-30)
    for b in range(B):
        n = min(max(int(lengths[b]), 0), cache.capacity)
        first = max(0, n - window) if window else 0
        slots = np.arange(first, n)
        k, ok = rows_of(cache, cache.k, b, slots)
        v, _ = rows_of(cache, cache.v, b, slots)
        slots, k, v = slots[ok], k[ok], v[ok]
        if not len(slots):
            continue
        for h in range(nq):
            s = k[:, h // g] @ q[b, h] * scale
            e = (np.abs(k[:, h // g]) @ np.abs(q[b, h])).max() * scale * (split + hd * U)
            p = np.exp(s - s.max())
            p /= p.sum()
            rel = 2 * e + split + 2.0 ** -20
            out[b, h] = p @ v[:, h // g]
            tol[b, h] += p @ np.abs(v[:, h // g]) * rel
            w[b, h // g, slots] += p
            wtol[b, h // g, slots] += p * rel
    return out, tol, w, wtol


def check(got, ref, tol):
    got = got.double().cpu().numpy()
    assert np.all(np.isfinite(got)), "non-finite output"
    worst = np.max(np.abs(got - ref) / tol)
    assert worst <= 1.0, f"off by {worst:.2f} times the tolerance"


# ---- append -----------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("nq,nkv,hd", HEADS)
@pytest.mark.parametrize("interleaved,norm,layout", [(False, True, "heads"), (True, False, "slots"),
                                                     (True, True, "joint")])
def test_append(torch, dtype, nq, nkv, hd, interleaved, norm, layout):
    rng = np.random.default_rng(hd + nq)
    B, T, ctx, page = 3, 37, 70, 32
    cache = make_cache(torch, B, 64, nkv, hd, dtype, page, layout)
    pool = torch.from_numpy(rng.normal(0, 2, (T, (nq + 2 * nkv) * hd + 8)).astype(np.float32)).cuda()
    qkv = pool[:, :-8]  # rows wider than their contents
    flat = rng.permutation(B * 64)[:T]
    seqs, slots, pos = (flat // 64).astype(np.int32), (flat % 64).astype(np.int32), rng.integers(0, ctx, T, np.int32)
    slots[3], slots[4], pos[5], pos[6], seqs[7], seqs[8] = -1, 64, -1, ctx, -1, B  # rows that store nothing
    table = cache.block_table.clone()
    cache.block_table[1, 1] = -1
    cache.block_table[2, 0] = cache.n_pages
    ang = rng.uniform(0, 6, (ctx, hd // 2))
    cos, sin = np.cos(ang).astype(np.float32), np.sin(ang).astype(np.float32)
    wq, wk = (rng.normal(0, 0.3, hd).astype(np.float32) for _ in range(2))
    k0, v0 = cache.k.double().cpu().numpy(), cache.v.double().cpu().numpy()
    cu = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    q = cache.append(qkv, cu(pos), cu(slots), cu(cos), cu(sin), n_heads=nq, q_norm=cu(wq) if norm else None,
                     k_norm=cu(wk) if norm else None, offset=1.0, eps=1e-5, seqs=cu(seqs), interleaved=interleaved)
    x = qkv.double().cpu().numpy().reshape(T, nq + 2 * nkv, hd)
    qk = x[:, :nq + nkv].copy()
    if norm:
        qk /= np.sqrt((qk * qk).mean(-1, keepdims=True) + 1e-5)
        qk[:, :nq] *= wq.astype(float) + 1.0
        qk[:, nq:] *= wk.astype(float) + 1.0
    a, b = (qk[..., 0::2], qk[..., 1::2]) if interleaved else (qk[..., :hd // 2], qk[..., hd // 2:])
    placed = (pos >= 0) & (pos < ctx)
    c, s = (t.astype(float)[np.where(placed, pos, 0)][:, None] for t in (cos, sin))
    parts, size = (a * c - b * s, a * s + b * c), np.abs(a) + np.abs(b)
    join = lambda u, w: np.stack((u, w), -1).reshape(qk.shape) if interleaved else np.concatenate((u, w), -1)  # noqa: E731
    rot, tol = join(*parts), join(size, size) * 1.5e-6 + 1e-30
    check(q, np.where(placed[:, None, None], rot[:, :nq], 0.0), tol[:, :nq])
    ktol, vtol = np.full(k0.shape, 1e-30), np.full(v0.shape, 1e-30)
    floor = 2.0 ** -25 if dtype == "f16" else 0.0
    held = cache.block_table.cpu().numpy()
    for i in range(T):
        if not placed[i] or not 0 <= seqs[i] < B or not 0 <= slots[i] < 64:
            continue
        p, o = held[seqs[i], slots[i] // page], slots[i] % page
        if not 0 <= p < cache.n_pages:
            continue
        k0[p, :, o], v0[p, :, o] = rot[i, nq:], x[i, nq + nkv:]
        ktol[p, :, o] = tol[i, nq:] + np.abs(rot[i, nq:]) * (ROUNDOFF[dtype] + U) + floor
        vtol[p, :, o] = np.abs(x[i, nq + nkv:]) * ROUNDOFF[dtype] + floor + 1e-30
    check(cache.k, k0, ktol)  # the whole pool: nothing else was written
    check(cache.v, v0, vtol)
    cache.block_table.copy_(table)


def test_append_one_token_defaults_to_its_own_sequence(torch):
    cache = make_cache(torch, 2, 16, 1, 64, "f32")
    qkv = torch.randn(2, 3 * 64, device="cuda")
    one = torch.ones(4, 32, device="cuda")
    pos = torch.tensor([0, 3], dtype=torch.int32, device="cuda")
    q = cache.append(qkv, pos, pos, one, torch.zeros_like(one), n_heads=1)  # cos 1, sin 0: no rotation
    assert torch.equal(q.view(2, 64), qkv[:, :64])
    for i in range(2):
        page = cache.block_table[i, 0]
        assert torch.equal(cache.k[page, 0, pos[i]], qkv[i, 64:128])
        assert torch.equal(cache.v[page, 0, pos[i]], qkv[i, 128:])
    assert cache.append(qkv[:0], pos[:0], pos[:0], one, one, n_heads=1).shape == (0, 1, 64)


# ---- attend -----------------------------------------------------------------------------

LENGTHS = [0, 1, 2, 15, 16, 17, 31, 33, 64, 127, 129, 300, 513, 1000, -5, 4000]  # the last two are clamped


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("nq,nkv,hd", HEADS)
@pytest.mark.parametrize("page,layout,window", [(16, "heads", 0), (64, "slots", 100), (32, "joint", 1)])
def test_attend_lengths_heads_and_layouts(torch, dtype, nq, nkv, hd, page, layout, window):
    cache = make_cache(torch, len(LENGTHS), 1024, nkv, hd, dtype, page, layout, seed=hd)
    gen = torch.Generator(device="cuda").manual_seed(1)
    q = torch.randn(len(LENGTHS), nq, hd, generator=gen, device="cuda") * 2
    lengths = torch.tensor(LENGTHS, dtype=torch.int32, device="cuda")
    scale = hd ** -0.5
    before = torch.rand(len(LENGTHS), nkv, cache.capacity, generator=gen, device="cuda")
    after = torch.full_like(before, 7.0)
    ref, tol, w, wtol = attend_ref(cache, q, LENGTHS, scale, window, SPLIT[dtype])
    out = cache.attend(q, lengths, scale, window=window)
    check(out, ref, tol)
    assert not out[0].any() and not out[-2].any()  # nothing cached
    again = cache.attend(q, lengths, scale, window=window, weights=before, weights_out=after)
    assert torch.equal(again, out)  # the weights change nothing, and the sums have one order
    check(after, before.double().cpu().numpy() + w, wtol + 2 * U * (before.double().cpu().numpy() + w))
    place = before.clone()
    cache.attend(q, lengths, scale, window=window, weights=place)
    assert torch.equal(place, after)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("nq,nkv,hd", [(17, 1, 64), (24, 2, 192), (40, 1, 128), (33, 1, 256), (10, 1, 64), (16, 1, 192),
                                       (32, 2, 256)])
def test_attend_many_heads_on_one(torch, dtype, nq, nkv, hd):
    """More than eight query heads per kv head share a pass, sixteen at a time; in
    divided sequences and whole ones, with the weights of all of them."""
    lengths = [1, 700, 0, 2500]
    cache = make_cache(torch, 4, 2500, nkv, hd, dtype, 16, seed=nq)
    gen = torch.Generator(device="cuda").manual_seed(2)
    q = torch.randn(4, nq, hd, generator=gen, device="cuda")
    n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    w = torch.zeros(4, nkv, cache.capacity, device="cuda")
    ref, tol, wr, wtol = attend_ref(cache, q, lengths, hd ** -0.5, 0, SPLIT[dtype])
    check(cache.attend(q, n, hd ** -0.5, weights=w), ref, tol)
    check(w, wr, wtol)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_attend_ignores_what_unseen_slots_hold(torch, dtype):
    """NaN and infinities beyond the length, before the window, on pages of no
    sequence and behind table entries that name no page."""
    B, nq, nkv, hd = 4, 8, 2, 128
    cache = make_cache(torch, B, 512, nkv, hd, dtype, 16, seed=3)
    lengths = [37, 200, 450, 512]
    window = 190
    q = torch.randn(B, nq, hd, device="cuda")
    cache.block_table[2, 20:23] = torch.tensor([-1, cache.n_pages, 2 ** 31 - 1], dtype=torch.int32)
    cache.block_table[1, 5:] = -7  # a sequence whose pages all lie outside the pool from slot 80 on
    ref, tol, _, _ = attend_ref(cache, q, lengths, 0.1, window, SPLIT[dtype])
    seen = torch.zeros(cache.k.shape[0], 16, dtype=torch.bool)
    for b, n in enumerate(lengths):
        for t in range(max(0, n - window), n):
            p = int(cache.block_table[b, t // 16])
            if 0 <= p < cache.n_pages:
                seen[p, t % 16] = True
    bad = torch.tensor([float("nan"), float("inf"), float("-inf"), 3e4], device="cuda").to(cache.k.dtype)
    for pool, shift in ((cache.k, 0), (cache.v, 1)):
        fill = bad.roll(shift).repeat(hd // 4).expand_as(pool)
        pool.copy_(torch.where(seen.cuda()[:, None, :, None], pool, fill))
    check(cache.attend(q, torch.tensor(lengths, dtype=torch.int32, device="cuda"), 0.1, window=window), ref, tol)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("factor", [1e-6, 300.0, 1e6])
def test_attend_query_range(torch, dtype, factor):
    """Queries far outside the cache type's range: nearly equal weights, and one
    slot that takes nearly all (whose score the scale brings back in range)."""
    cache = make_cache(torch, 2, 512, 2, 128, dtype, seed=5)
    q = torch.randn(2, 8, 128, device="cuda") * factor
    lengths = torch.tensor([500, 77], dtype=torch.int32, device="cuda")
    scale = 1.0 / max(factor, 1.0)
    ref, tol, _, _ = attend_ref(cache, q, [500, 77], scale, 0, SPLIT[dtype])
    check(cache.attend(q, lengths, scale), ref, tol)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_attend_many_small_weights_beside_a_large_one(torch, dtype):
    """One slot of weight 1 and tens of thousands of 2^-26 or so each: none of
    them is lost on the way."""
    n, hd = 40000, 64
    cache = make_cache(torch, 1, n, 1, hd, dtype, seed=6)
    cache.k.zero_()
    cache.v.fill_(1.0)
    q = torch.zeros(1, 2, hd, device="cuda")
    q[:, :, 0] = 1.0
    page = cache.block_table[0, 77 // 16]
    cache.k[page, 0, 77 % 16, 0] = 18.0  # e^-18 = 2^-26 for all the others
    cache.v[page, 0, 77 % 16] = 0.0
    out = cache.attend(q, torch.tensor([n], dtype=torch.int32, device="cuda"), 1.0)
    rest = (n - 1) * np.exp(-18.0)
    np.testing.assert_allclose(out.cpu().numpy(), rest / (1 + rest), rtol=2.0 ** -14)


def test_attend_long_sequences_split_and_join(torch):
    for dtype, (nq, nkv, hd), lengths in (("bf16", (4, 1, 256), [70001]), ("f16", (64, 8, 128), [20000, 3, 0, 9000]),
                                          ("f32", (9, 1, 64), [30000, 30001])):
        cache = make_cache(torch, len(lengths), max(lengths), nkv, hd, dtype, 32, seed=8)
        q = torch.randn(len(lengths), nq, hd, device="cuda")
        n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
        w = torch.zeros(len(lengths), nkv, cache.capacity, device="cuda")
        ref, tol, wr, wtol = attend_ref(cache, q, lengths, hd ** -0.5, 0, SPLIT[dtype])
        out = cache.attend(q, n, hd ** -0.5, weights=w)
        check(out, ref, tol)
        check(w, wr, wtol)
        for _ in range(3):
            assert torch.equal(cache.attend(q, n, hd ** -0.5), out)


def test_attend_many_short_sequences(torch):
    rng = np.random.default_rng(9)
    lengths = rng.integers(0, 90, 700).tolist()
    cache = make_cache(torch, 700, 96, 2, 64, "f16", 16, seed=9)
    q = torch.randn(700, 6, 64, device="cuda")
    ref, tol, _, _ = attend_ref(cache, q, lengths, 0.125, 0, SPLIT["f16"])
    check(cache.attend(q, torch.tensor(lengths, dtype=torch.int32, device="cuda"), 0.125), ref, tol)


def test_offsets_beyond_32_bits(torch):
    """A pool of 2^31 + elements: the pages of the sequence lie at its end, and
    append, attend and evict reach them."""
    nkv, hd, page = 8, 128, 64
    from machinelearning_b200.paged import PagedKVCache
    pages = 2 ** 31 // (nkv * hd * page) + 40
    k = torch.empty(pages, nkv, page, hd, dtype=torch.bfloat16, device="cuda")
    v = torch.empty_like(k)
    table = torch.arange(pages - 4, pages, dtype=torch.int32, device="cuda").view(1, 4)
    k[-4:] = torch.randn(4, nkv, page, hd, device="cuda")
    v[-4:] = torch.randn(4, nkv, page, hd, device="cuda")
    cache = PagedKVCache(k, v, table)
    n = torch.tensor([200], dtype=torch.int32, device="cuda")
    qkv = torch.randn(1, (16 + 2 * nkv) * hd, device="cuda")
    one = torch.ones(1, hd // 2, device="cuda")
    q = cache.append(qkv, torch.zeros_like(n), n - 1, one, torch.zeros_like(one), n_heads=16)
    assert torch.equal(v[pages - 1, :, 199 - 192].float(), qkv[0, (16 + nkv) * hd:].view(nkv, hd).bfloat16().float())
    ref, tol, _, _ = attend_ref(cache, q, [200], 0.09, 0, SPLIT["bf16"])
    check(cache.attend(q, n, 0.09), ref, tol)
    w = torch.zeros(1, nkv, 256, device="cuda")
    w[:, :, 100:200] = 1.0
    pos = torch.arange(256, dtype=torch.int32, device="cuda").expand(1, nkv, 256).contiguous()
    rows = v[table[0].long()].transpose(0, 1).reshape(nkv, 256, hd)[:, 100:200].clone()
    cache.evict(n, w, pos, n, budget=100, recent=0)
    assert torch.equal(v[table[0].long()].transpose(0, 1).reshape(nkv, 256, hd)[:, :100], rows)


@pytest.mark.parametrize("n", [90, 20000])
def test_attend_back_to_back_accumulations(torch, n):
    """Calls whose launches overlap: each adds its weights to what the one before left."""
    cache = make_cache(torch, 3, n, 2, 128, "bf16", seed=n)
    q = torch.randn(3, 8, 128, device="cuda")
    lengths = torch.tensor([n, n // 2, 1], dtype=torch.int32, device="cuda")
    one = torch.zeros(3, 2, cache.capacity, device="cuda")
    cache.attend(q, lengths, 0.1, weights=one)
    torch.cuda.synchronize()
    want = torch.zeros_like(one)
    for _ in range(200):
        want += one
    for _ in range(3):
        many = torch.zeros_like(one)
        for _ in range(200):
            cache.attend(q, lengths, 0.1, weights=many)
        assert torch.equal(many, want)


def test_attend_on_another_stream_and_in_a_graph(torch):
    cache = make_cache(torch, 2, 4096, 2, 128, "bf16", seed=10)
    q = torch.randn(2, 8, 128, device="cuda")
    lengths = torch.tensor([5, 1000], dtype=torch.int32, device="cuda")
    w = torch.zeros(2, 2, cache.capacity, device="cuda")
    out = torch.empty(2, 8, 128, device="cuda")
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    cache.reserve(8, weights=True, stream=stream)
    with torch.cuda.stream(stream):
        cache.attend(q, lengths, 0.1, out=out, weights=w)
    stream.synchronize()
    assert torch.equal(out, cache.attend(q, lengths, 0.1))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        cache.attend(q, lengths, 0.1, out=out, weights=w)
    for step in (0, 1, 700):  # lengths advance in place between replays
        lengths.add_(step)
        w.zero_()
        graph.replay()
        torch.cuda.synchronize()
        ref, tol, wr, wtol = attend_ref(cache, q, lengths.tolist(), 0.1, 0, SPLIT["bf16"])
        check(out, ref, tol)
        check(w, wr, wtol)


# ---- evict ------------------------------------------------------------------------------

def evict_ref(lengths, w, pos, nxt, budget, recent):
    """(lengths, weights, positions, moves (b, h, to, of)) by sorting."""
    w, pos, moves = w.copy(), pos.copy(), []
    for b in range(w.shape[0]):
        n = min(max(int(lengths[b]), 0), w.shape[2])
        m = min(n, budget)
        for h in range(w.shape[1]):
            if n > budget:
                key = np.where(np.isnan(w[b, h, :n]), -np.inf, w[b, h, :n])
                protected = pos[b, h, :n] >= int(nxt[b]) - recent
                kept = np.zeros(n, bool)
                kept[np.lexsort((np.arange(n), np.where(protected, 0.0, -key), ~protected))[:budget]] = True
                to, of = np.flatnonzero(~kept[:budget]), budget + np.flatnonzero(kept[budget:])
                w[b, h, to], pos[b, h, to] = w[b, h, of], pos[b, h, of]
                moves += [(b, h, t, o) for t, o in zip(to, of)]
            w[b, h, m:], pos[b, h, m:] = 0.0, -1
    return np.clip(lengths, 0, np.minimum(budget, w.shape[2])), w, pos, moves


@pytest.mark.parametrize("dtype,layout", [("f32", "heads"), ("f16", "slots"), ("bf16", "joint")])
@pytest.mark.parametrize("nkv,hd", [(1, 256), (3, 64), (8, 128)])
@pytest.mark.parametrize("budget,recent,kind", [(100, 20, "random"), (1, 0, "random"), (1, 1, "ties"),
                                                (700, 700, "ties"), (1000, 3, "special"), (64, 64, "surplus"),
                                                (511, 0, "equal"), (5000, 10, "random")])
def test_evict(torch, dtype, layout, nkv, hd, budget, recent, kind):
    rng = np.random.default_rng(budget + hd)
    lengths = np.array([0, 1, 99, 100, 101, 512, 1000, 2049, 2064, -3, 3000], np.int32)
    B = len(lengths)
    cache = make_cache(torch, B, 2064, nkv, hd, dtype, 16, layout, seed=budget)
    cap = cache.capacity
    w = rng.random((B, nkv, cap)).astype(np.float32)
    if kind == "ties":
        w = np.floor(w * 4).astype(np.float32)
    if kind == "equal":
        w[:] = 0.5
    if kind == "special":
        w = rng.choice(np.array([0.0, -0.0, np.nan, np.inf, -np.inf, 1.0, -1.0, 1e-45, 3e38], np.float32), w.shape)
    pos = np.sort(rng.permuted(np.broadcast_to(np.arange(2 * cap), (B, nkv, 2 * cap)), axis=-1)[..., :cap],
                  axis=-1).astype(np.int32)
    nxt = np.array([pos[b, :, max(0, min(n, cap) - 1)].max() + 1 for b, n in enumerate(lengths)], np.int32)
    if kind == "surplus":  # every slot counts as recent
        nxt[:] = 0
    cu = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    k0, v0 = cache.k.clone(), cache.v.clone()
    wd, pd = cu(w), cu(pos)
    got = cache.evict(cu(lengths), wd, pd, cu(nxt), budget=budget, recent=recent)
    ref = evict_ref(lengths, w, pos, nxt, budget, recent)
    np.testing.assert_array_equal(got[0].cpu().numpy(), ref[0])
    np.testing.assert_array_equal(got[1].cpu().numpy(), ref[1])
    np.testing.assert_array_equal(got[2].cpu().numpy(), ref[2])
    np.testing.assert_array_equal(wd.cpu().numpy(), w)
    table = cache.block_table.cpu().numpy()
    if ref[3]:
        b, h, to, of = np.array(ref[3]).T
        tp, fp = table[b, to // 16], table[b, of // 16]
        for new, old in ((cache.k, k0), (cache.v, v0)):
            want = old.clone()
            want[tp, h, to % 16] = old[fp, h, of % 16]
            assert torch.equal(new, want)
    else:
        assert torch.equal(cache.k, k0) and torch.equal(cache.v, v0)


@pytest.mark.parametrize("n,budget", [(40001, 20000), (40001, 40000), (100000, 77), (131072, 65537)])
def test_evict_long_rows(torch, n, budget):
    rng = np.random.default_rng(n)
    cache = make_cache(torch, 2, n, 1, 64, "bf16", 64, seed=n)
    w = (rng.random((2, 1, cache.capacity)) ** 4).astype(np.float32)
    w[1] = np.floor(w[1] * 8)  # long runs of ties
    pos = np.broadcast_to(np.arange(cache.capacity, dtype=np.int32), w.shape).copy()
    lengths, nxt = np.array([n, n - 1], np.int32), np.array([n, n - 1], np.int32)
    k0 = cache.k.clone()
    cu = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    got = cache.evict(cu(lengths), cu(w), cu(pos), cu(nxt), budget=budget, recent=min(budget, 500))
    ref = evict_ref(lengths, w, pos, nxt, budget, min(budget, 500))
    for g, r in zip(got, ref):
        np.testing.assert_array_equal(g.cpu().numpy(), r)
    table = cache.block_table.cpu().numpy()
    b, h, to, of = np.array(ref[3]).T
    want = k0.clone()
    want[table[b, to // 64], h, to % 64] = k0[table[b, of // 64], h, of % 64]
    assert torch.equal(cache.k, want)


def test_evict_leaves_rows_of_missing_pages(torch):
    cache = make_cache(torch, 1, 64, 1, 64, "f32", 16, seed=11)
    cache.block_table[0, 0] = -1  # the holes' page
    k0 = cache.k.clone()
    w = torch.arange(64, dtype=torch.float32, device="cuda").view(1, 1, 64)
    pos = torch.arange(64, dtype=torch.int32, device="cuda").view(1, 1, 64)
    n = torch.tensor([64], dtype=torch.int32, device="cuda")
    _, w2, p2 = cache.evict(n, w, pos, n, budget=16, recent=0)
    assert torch.equal(cache.k, k0)
    assert p2[0, 0, :16].tolist() == list(range(48, 64)) and not w2[0, 0, 16:].any()


# ---- logits -----------------------------------------------------------------------------

def logits_ref(x, tokens, total, prompt, rep, pres, freq, ids, vals, mask, mask_rows):
    y = x.astype(np.float64)
    size = np.abs(y)
    rows, vocab = x.shape
    for r in range(rows):
        if tokens is not None:
            hist = tokens[r, :min(max(total[r], 0), tokens.shape[1])]
            out = hist[max(prompt[r], 0):]
            for t in np.unique(hist[(hist >= 0) & (hist < vocab)]):
                y[r, t] = y[r, t] / rep[r] if y[r, t] > 0 else y[r, t] * rep[r]
                n = int((out == t).sum())
                size[r, t] = abs(y[r, t]) * 2 + freq[r] * n + pres[r]
                if n:
                    y[r, t] -= float(freq[r]) * n + float(pres[r])
        if ids is not None:
            for t, b in zip(ids[r], vals[r]):
                if 0 <= t < vocab:
                    y[r, t] += float(b)
                    size[r, t] += abs(float(b))
        state = (mask_rows[r] if mask_rows is not None else r) if mask is not None else -1
        if mask is not None and 0 <= state < mask.shape[0]:
            bits = np.unpackbits(mask[state].view(np.uint8), bitorder="little")[:vocab]
            y[r, bits == 0] = -np.inf
    return y, size


def check_logits(got, ref, size):
    got = got.double().cpu().numpy()
    np.testing.assert_array_equal(np.isnan(got), np.isnan(ref))
    off = ~np.isfinite(ref)
    np.testing.assert_array_equal(got[off], ref[off])
    assert np.all(np.abs(got[~off] - ref[~off]) <= 8 * U * size[~off] + 1e-37)


@pytest.mark.parametrize("rows,vocab,hist,bias,masks", [
    (1, 262144, 300, 8, 4), (3, 32003, 2000, 300, 0), (5, 1, 4, 1, 5), (2, 31, 100, 1024, 2), (4, 8192, 0, 0, 4),
    (3, 8193, 9, 3, 2), (2, 65537, 40000, 17, 3), (6, 1001, 5000, 0, 1), (1, 50257, 1, 0, 0)])
@pytest.mark.parametrize("in_place", [False, True])
def test_logits(torch, rows, vocab, hist, bias, masks, in_place):
    from machinelearning_b200.logits import process_logits
    rng = np.random.default_rng(vocab + rows)
    pad = 5 if vocab % 2 else 0  # strided rows
    x = (rng.normal(0, 4, (rows, vocab + pad))).astype(np.float32)
    tokens = (rng.random((rows, hist)) ** 3 * vocab).astype(np.int32)
    if hist > 3:
        tokens[:, 1], tokens[:, 2] = -1, vocab  # ignored
    total = rng.integers(0, hist + 1, rows).astype(np.int32)
    total[0] = hist + 7  # clamped
    prompt = (total * rng.random(rows)).astype(np.int32)
    prompt[-1] = -2
    rep, pres, freq = (rng.uniform(*r, rows).astype(np.float32) for r in ((1.0, 1.5), (0.0, 1.0), (0.0, 0.5)))
    ids = rng.integers(-2, vocab + 2, (rows, bias)).astype(np.int32) if bias else None  # duplicates where bias > vocab
    vals = rng.normal(0, 5, (rows, bias)).astype(np.float32) if bias else None
    mask = mask_rows = None
    if masks:
        mask = rng.integers(-2 ** 31, 2 ** 31, (masks, (vocab + 31) // 32)).astype(np.int32)
        mask[-1] = 0  # nothing allowed
        mask_rows = rng.integers(-1, masks + 1, rows).astype(np.int32)
        mask_rows[0] = masks - 1 if rows > 1 else 0
    if vocab > 8:  # special values, masked or not
        x[0, :5] = [np.nan, np.inf, -np.inf, 0.0, -0.0]
    cu = lambda a: None if a is None else torch.from_numpy(a).cuda()  # noqa: E731
    xd = cu(x)[:, :vocab]
    keep = xd.clone()
    with np.errstate(invalid="ignore"):
        ref, size = logits_ref(x[:, :vocab], tokens if hist else None, total, prompt, rep, pres, freq, ids, vals, mask,
                               mask_rows)
    args = dict(bias_ids=cu(ids), bias_values=cu(vals), mask=cu(mask), mask_rows=cu(mask_rows))
    if hist:
        args.update(tokens=cu(tokens), token_lengths=cu(total), prompt_lengths=cu(prompt), repetition=cu(rep),
                    presence=cu(pres), frequency=cu(freq))
    got = process_logits(xd, out=xd if in_place else None, **args)
    check_logits(got, ref, size)
    if not in_place:
        assert torch.equal(xd.nan_to_num(), keep.nan_to_num())
        assert torch.equal(process_logits(xd, **args).nan_to_num(), got.nan_to_num())


def test_logits_without_steps_is_a_copy_and_states_default_to_rows(torch):
    from machinelearning_b200.logits import process_logits
    x = torch.randn(2, 100, device="cuda")
    assert torch.equal(process_logits(x), x)
    mask = torch.tensor([[-1, 0, 0, 0], [0, 0, 0, 1]], dtype=torch.int32, device="cuda")
    y = process_logits(x, mask=mask)
    assert torch.equal(y[0, :32], x[0, :32]) and torch.isneginf(y[0, 32:]).all()
    assert torch.equal(y[1, 96:97], x[1, 96:97]) and int(torch.isfinite(y).sum()) == 33


def test_python_refusals_on_the_gpu(torch):
    from machinelearning_b200 import _lib
    from machinelearning_b200.logits import process_logits
    cache = make_cache(torch, 2, 64, 2, 64)
    q = torch.randn(2, 4, 64, device="cuda")
    n = torch.ones(2, dtype=torch.int32, device="cuda")
    with pytest.raises(_lib.ShapeMismatch):
        cache.attend(q[:1], n, 1.0)
    with pytest.raises(_lib.ShapeMismatch):
        cache.attend(q[:, :3].contiguous(), n, 1.0)  # 3 heads on 2
    with pytest.raises(_lib.DTypeMismatch):
        cache.attend(q.half(), n, 1.0)
    with pytest.raises(_lib.DTypeMismatch):
        cache.attend(q, n.long(), 1.0)
    with pytest.raises(_lib.ShapeMismatch):
        cache.attend(q, n, 1.0, weights=torch.zeros(2, 2, 63, device="cuda"))
    with pytest.raises(ValueError):
        cache.attend(q, n, 1.0, weights_out=torch.zeros(2, 2, 64, device="cuda"))
    with pytest.raises(_lib.ShapeMismatch):
        cache.append(torch.randn(3, 8 * 64, device="cuda"), n, n, n, n, n_heads=4)
    w, pos = torch.zeros(2, 2, 64, device="cuda"), torch.zeros(2, 2, 64, dtype=torch.int32, device="cuda")
    with pytest.raises(_lib.ShapeMismatch):
        cache.evict(n, w, pos, n, budget=0, recent=0)
    x = torch.randn(2, 50, device="cuda")
    with pytest.raises(ValueError):
        process_logits(x, tokens=pos[0])
    with pytest.raises(_lib.ShapeMismatch):
        process_logits(x, mask=torch.zeros(2, 3, dtype=torch.int32, device="cuda"))
    with pytest.raises(ValueError):
        process_logits(x, presence=torch.zeros(2, device="cuda"))
