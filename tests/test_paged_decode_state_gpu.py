"""What the paged decoder (machinelearning_b200/paged_decode.py) keeps from step to
step and leaves behind."""
from __future__ import annotations

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
