"""What the paged decoder (machinelearning_b200/paged_decode.py) keeps from step to
step and leaves behind."""
from __future__ import annotations

import numpy as np
import pytest

from test_decode_gpu import host_weights, small_config

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch
    assert torch.cuda.is_available()
    return torch


def bounded(model, limit):
    """Makes the model refuse more than ``limit`` steps."""
    step = model.step
    left = [limit]

    def counted(*args, **kwargs):
        left[0] -= 1
        assert left[0] >= 0, "the loop does not end"
        return step(*args, **kwargs)
    model.step = counted


def test_generate_with_a_graph_that_does_not_advance(oracle, torch):
    from machinelearning_b200.paged_decode import PagedGemma3Decoder
    cfg = small_config()
    w = host_weights(oracle, cfg, seed=71)
    prompts = [[5, 9, 14], [600]]
    model = PagedGemma3Decoder(cfg, w, batch=2)
    want = model.generate(prompts, 5)
    model.capture(advance=False)
    bounded(model, 20)
    assert model.generate(prompts, 5) == want
    model.close()


def test_generate_leaves_sequences_idle_and_refuses_first(oracle, torch):
    from machinelearning_b200.paged_decode import PagedGemma3Decoder
    cfg = small_config()
    model = PagedGemma3Decoder(cfg, host_weights(oracle, cfg, seed=72), batch=3)
    bounded(model, 30)
    idle = [-1, -1, -1]
    assert model.generate([[1, 2], [3]], 0) == [[], []] and model.host_positions == idle
    assert model.generate([], 4) == [] and model.host_positions == idle
    for prompts, n, every in (([[1] * 17], 1, 0),      # the prompt is longer than the cache
                              ([[1] * 10, [2]], 8, 0),  # the last token fed would be the 17th
                              ([[1]], -1, 0), ([[1]], 2, 3)):  # no budget to evict to
        with pytest.raises(ValueError):
            model.generate(prompts, n, evict_every=every)
        assert model.host_positions == idle and model.positions.tolist() == idle
    full = model.generate([[1] * 10], 7)  # the 16th position is fed, its token the last one out
    assert len(full[0]) == 7
    model.start(2)
    with pytest.raises(ValueError, match="started"):  # it would be fed tokens of nobody's
        model.generate([[1, 2]], 2)
    assert model.host_positions == [-1, -1, 0]
    model.close()


@pytest.mark.parametrize("use_graph", [False, True])
def test_a_repeated_step_adds_its_weights_once(oracle, torch, use_graph):
    """step(advance=False) leaves the accumulated weights as they were, like the
    position it stays at."""
    from machinelearning_b200.paged_decode import PagedGemma3Decoder
    cfg = small_config()
    w = host_weights(oracle, cfg, seed=73)
    got = []
    for repeats in (0, 3):
        model = PagedGemma3Decoder(cfg, w, batch=2, budget=4, recent=1)
        for s in range(2):
            model.start(s)
        model.step([7, 8])
        if use_graph and repeats:
            model.capture(advance=False)
        for _ in range(repeats):
            model.step([9, 10], advance=False)
        model.graph = None
        model.step([9, 10])
        got.append([model.slot_weights[li].clone() for li in model.global_layers] + [model.logits.clone()])
        model.close()
    for a, b in zip(*got):
        assert torch.equal(a, b)


def test_generate_evicts_alike_with_and_without_a_graph(oracle, torch):
    """The weights that evictions go by are those of the steps taken, however they are launched."""
    from machinelearning_b200.paged_decode import PagedGemma3Decoder
    cfg = small_config()
    w = host_weights(oracle, cfg, seed=76)
    got = []
    for graph in (None, True, False):
        model = PagedGemma3Decoder(cfg, w, batch=2, budget=3, recent=1)
        if graph is not None:
            model.capture(advance=graph)
        out = model.generate([[5, 9, 14], [600]], 8, evict_every=2)
        got.append((out, [model.slot_positions[li].tolist() for li in model.global_layers]))
        assert (model.graph is None) == (graph is None)
        model.close()
    assert got[0] == got[1] == got[2]


@pytest.mark.parametrize("use_graph", [False, True])
def test_windows_of_the_local_layers_match_the_oracle(oracle, torch, use_graph):
    """Logits at the dense decoder's 1e-3 with a window that the positions exceed."""
    from conftest import assert_close_rel
    from oracle.decode import decode_step

    from machinelearning_b200.paged_decode import PagedGemma3Decoder
    cfg = small_config()
    w = host_weights(oracle, cfg, seed=74)
    for window in (1, 3, 15):
        model = PagedGemma3Decoder(cfg, w, batch=2, cache_dtype=torch.float32, window=window)
        model.start(0)
        if use_graph:
            model.capture()
        shape = (1, cfg.n_kv_heads, cfg.ctx, cfg.head_dim)
        caches = [[[np.zeros(shape, np.float32) for _ in range(cfg.n_layers)] for _ in range(2)] for _ in range(2)]
        tokens = np.random.default_rng(window).integers(0, cfg.vocab, (2, cfg.ctx))
        for step in range(cfg.ctx):
            if step == 2:
                model.start(1)
            model.step([tokens[0, step], tokens[1, max(0, step - 2)]])
            got = model.logits.cpu().numpy()
            for s in range(2 if step >= 2 else 1):
                at = step - 2 * s
                ref = decode_step(cfg, w, tokens[s, at:at + 1], at, *caches[s], window=window)[0]
                assert_close_rel(got[s], ref, 1e-3, 1e-2)
        model.close()


def test_slots_after_every_eviction(oracle, torch):
    from machinelearning_b200.paged_decode import PagedGemma3Decoder
    cfg = small_config()
    model = PagedGemma3Decoder(cfg, host_weights(oracle, cfg, seed=75), batch=2, budget=4, recent=2)
    model.start(0)
    counts = [0, -1]
    for step in range(12):
        if step == 3:
            model.start(1)
            counts[1] = 0
        model.step([step, 20 + step])
        counts = [c + 1 if c >= 0 else c for c in counts]
        if step % 3 == 2:
            model.evict()
            counts = [min(c, 4) for c in counts]
        assert model.slots.tolist() == [max(c, 0) for c in counts]
        for li in model.global_layers:  # every held slot has a position of its own, the newest among them
            for s, c in enumerate(counts):
                held = model.slot_positions[li][s, 0, :max(c, 0)].tolist()
                assert len(set(held)) == len(held) and (c <= 0 or max(held) == model.host_positions[s] - 1)
    model.close()


def test_sequences_that_do_not_exist(oracle, torch):
    from machinelearning_b200.paged_decode import PagedGemma3Decoder
    cfg = small_config()
    model = PagedGemma3Decoder(cfg, host_weights(oracle, cfg, seed=77), batch=2)
    model.start(0), model.start(1)
    for seq in (-1, 2):
        with pytest.raises(ValueError):
            model.start(seq)
        with pytest.raises(ValueError):  # -1 named the last one
            model.stop(seq)
    assert model.host_positions == [0, 0] and model.positions.tolist() == [0, 0]
    model.stop(1)
    assert model.host_positions == [0, -1] and model.positions.tolist() == [0, -1]
    model.close()
