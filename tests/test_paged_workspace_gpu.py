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
