"""The decoders (machinelearning_b200/decode.py, paged_decode.py) run on a stream of
their own: what the caller's stream does before a step is seen by it, and what it
does with the last step's logits is done before the next one."""
from __future__ import annotations

import pytest

from test_decode_gpu import host_weights, small_config

pytestmark = pytest.mark.gpu

BACKLOG = 100_000_000  # clocks: 50 ms on the caller's stream


@pytest.fixture(scope="module")
def torch():
    import torch
    assert torch.cuda.is_available()
    return torch


@pytest.mark.parametrize("use_graph", [False, True])
def test_a_grammar_state_changed_in_place_holds_for_the_next_step(oracle, torch, use_graph):
    from machinelearning_b200.paged_decode import PagedGemma3Decoder
    cfg = small_config()
    model = PagedGemma3Decoder(cfg, host_weights(oracle, cfg, seed=81), batch=2)
    mask = torch.zeros(cfg.vocab // 32, cfg.vocab // 32, dtype=torch.int32, device="cuda")
    mask.fill_diagonal_(-1)  # state i allows tokens 32 i to 32 i + 31
    state = torch.zeros(2, dtype=torch.int32, device="cuda")
    model.set_constraints(mask=mask, mask_rows=state)
    model.start(0), model.start(1)
    if use_graph:
        model.capture()
    torch.cuda.synchronize()
    for i in range(1, 8):
        torch.cuda._sleep(BACKLOG)
        state.add_(1)
        model.step([3, 4])
        assert all(32 * i <= t < 32 * (i + 1) for t in model.next_tokens.tolist())
    model.close()


@pytest.mark.parametrize("paged", [False, True])
@pytest.mark.parametrize("use_graph", [False, True])
def test_the_next_step_waits_for_readers_of_the_last_logits(oracle, torch, paged, use_graph):
    from machinelearning_b200.decode import Gemma3Decoder
    from machinelearning_b200.paged_decode import PagedGemma3Decoder
    cfg = small_config()
    model = (PagedGemma3Decoder if paged else Gemma3Decoder)(cfg, host_weights(oracle, cfg, seed=82), batch=1)
    if paged:
        model.start(0)
    if use_graph:
        model.capture()
    want, kept = [], []
    for delayed in (False, True):
        model.start(0) if paged else model.set_position(0)
        for t in range(4):
            logits = model.step([10 + t])
            if delayed:
                torch.cuda._sleep(BACKLOG)
            (kept if delayed else want).append(logits.clone())
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, kept))
    assert not torch.equal(want[0], want[1])
    model.close()


def test_a_captured_step_keeps_its_constraints_alive(oracle, torch):
    """Constraints replaced after the capture, with no other reference to the old ones:
    replays go on with those, whatever the freed memory holds."""
    import gc

    from machinelearning_b200.paged_decode import PagedGemma3Decoder
    cfg = small_config()
    model = PagedGemma3Decoder(cfg, host_weights(oracle, cfg, seed=83), batch=2)
    words = cfg.vocab // 32
    mask = torch.zeros(1, words, dtype=torch.int32, device="cuda")
    mask[0, 3] = -1
    ids = torch.tensor([[97], [110]], dtype=torch.int32, device="cuda")
    model.set_constraints(bias_ids=ids, bias_values=torch.full((2, 1), 1e4, device="cuda"), mask=mask,
                          mask_rows=torch.zeros(2, dtype=torch.int32, device="cuda"))
    model.start(0), model.start(1)
    model.capture()
    del mask, ids
    model.set_constraints()
    gc.collect()
    filled = [torch.full((n,), v, device="cuda", dtype=torch.int32) for n in (1, 2, words, 128) for v in (0, 5, -1)
              for _ in range(40)]
    for _ in range(4):
        model.step([3, 4])
        assert model.next_tokens.tolist() == [97, 110]
    assert filled
    model.capture()  # without constraints now
    model.step([3, 4])
    assert torch.equal(model.processed, model.logits)
    model.close()
