"""The library's workspaces under the paged operators, which keep live data in
them between their launches (machinelearning_b200/csrc/qmm_api.cu)."""
from __future__ import annotations

import pytest

from test_paged_gpu import make_cache

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch
    assert torch.cuda.is_available()
    return torch


@pytest.mark.parametrize("reserve", [False, True])
def test_a_new_workspace_is_cleared_before_its_first_use(torch, reserve):
    """The first calls on a side stream, behind a backlog on the default one: the
    buffer's clear comes before them, not when the backlog ends."""
    B, nq, nkv, hd = 8, 64, 8, 64
    cap = 32768 if reserve else 16384  # 67 or 34 MB of scores: more than any stream's buffer has
    cache = make_cache(torch, B, cap, nkv, hd, "bf16", 64, seed=1)
    q = torch.randn(B, nq, hd, device="cuda")
    n = torch.full((B,), cap, dtype=torch.int32, device="cuda")
    zero = torch.zeros(B, nkv, cap, device="cuda")
    pos = torch.arange(cap, dtype=torch.int32, device="cuda").expand(B, nkv, cap).contiguous()
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    torch.cuda._sleep(200_000_000)  # a tenth of a second on the default stream
    with torch.cuda.stream(stream):
        if reserve:
            cache.reserve(nq, weights=True, budget=cap // 2)
        first = zero.clone()
        out = cache.attend(q, n, 0.1, weights=first)
    stream.synchronize()
    torch.cuda.synchronize()
    again = zero.clone()
    assert torch.equal(cache.attend(q, n, 0.1, weights=again), out) and torch.equal(again, first)
    k, v = cache.k.clone(), cache.v.clone()
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    torch.cuda._sleep(200_000_000)
    with torch.cuda.stream(stream):
        got = cache.evict(n, first, pos, n, budget=cap // 2, recent=10)
    stream.synchronize()
    torch.cuda.synchronize()
    moved = cache.k.clone(), cache.v.clone()
    assert not torch.equal(moved[0], k)
    cache.k.copy_(k), cache.v.copy_(v)
    want = cache.evict(n, first, pos, n, budget=cap // 2, recent=10)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert torch.equal(cache.k, moved[0]) and torch.equal(cache.v, moved[1])


def test_a_graph_keeps_its_workspace_when_a_later_call_needs_more(torch):
    """A captured step over a small cache, then a direct call over a large one on the
    same stream: replays give the same result, and write to nobody else's memory."""
    stream = torch.cuda.Stream()
    small = make_cache(torch, 2, 4096, 2, 128, "bf16", seed=2)
    q = torch.randn(2, 8, 128, device="cuda")
    n = torch.tensor([4096, 3000], dtype=torch.int32, device="cuda")
    zero = torch.zeros(2, 2, 4096, device="cuda")
    out, w = torch.zeros_like(q), zero.clone()
    large = make_cache(torch, 8, 65536, 8, 64, "bf16", 64, seed=3)  # 268 MB of scores
    ql = torch.randn(8, 64, 64, device="cuda")
    nl = torch.full((8,), 65536, dtype=torch.int32, device="cuda")
    wl = torch.zeros(8, 8, 65536, device="cuda")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(stream):
        small.reserve(8, weights=True)
        small.attend(q, n, 0.1, out=out, weights=w, weights_out=w)
        want = out.clone(), w.clone()
        stream.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            small.attend(q, n, 0.1, out=out, weights=w, weights_out=w)
        large.attend(ql, nl, 0.1, weights=wl)
        stream.synchronize()
        # whatever was freed is handed out again, in pieces of the sizes of the buffer
        others = [torch.full((size,), 7.0, device="cuda") for size in (1 << 18, 1 << 20, 1 << 22) for _ in range(8)]
        for _ in range(3):
            out.zero_(), w.zero_()
            graph.replay()
            stream.synchronize()
            assert torch.equal(out, want[0]) and torch.equal(w, want[1])
        assert all(bool((t == 7.0).all()) for t in others)
        again = torch.zeros_like(wl)
        large.attend(ql, nl, 0.1, weights=again)  # the larger buffer serves the direct calls
        assert torch.equal(again, wl)


def test_host_threads_on_one_stream(torch, oracle):
    """Calls of several launches from three host threads on one stream: attention over
    divided sequences, evictions, and a matmul that sums its K splits in the
    same workspace. Each has the results that it has alone."""
    import threading

    import numpy as np

    from machinelearning_b200 import _lib
    from machinelearning_b200.linear import Linear, QuantWeight
    jobs = []
    for i in range(2):
        cache = make_cache(torch, 2, 8192, 2, 128, "bf16", seed=20 + i)
        q = torch.randn(2, 8, 128, device="cuda")
        n = torch.tensor([8192, 5000 - i], dtype=torch.int32, device="cuda")
        jobs.append(lambda cache=cache, q=q, n=n: cache.attend(q, n, 0.1))
    spare = make_cache(torch, 4, 2048, 2, 64, "f16", seed=22)
    w = torch.rand(4, 2, 2048, device="cuda")
    pos = torch.arange(2048, dtype=torch.int32, device="cuda").expand(4, 2, 2048).contiguous()
    full = torch.full((4,), 2048, dtype=torch.int32, device="cuda")
    jobs.append(lambda: torch.cat([t.float().flatten() for t in spare.evict(full, w, pos, full, 1000, 10)]))
    rng = np.random.default_rng(0)
    m, k, rows = 20, 1152, 256  # rows of 1224 bytes: the streaming kernel, with K split
    lin = Linear(QuantWeight.from_host(_lib.Q8_0, rows, k, oracle.quantize_q8_0(
        rng.normal(0, 0.05, rows * k).astype(np.float32)), device=0))
    x = torch.from_numpy(rng.normal(0, 1, (m, k)).astype(np.float32)).cuda()
    jobs.append(lambda: lin(x))
    want = [job().clone() for job in jobs]
    wrong = [None] * len(jobs)
    gate = threading.Barrier(len(jobs))

    def work(i):
        gate.wait()
        got = [jobs[i]() for _ in range(300)]
        wrong[i] = sum(not torch.equal(g, want[i]) for g in got)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(jobs))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert wrong == [0] * len(jobs)
    lin.weight.close()
