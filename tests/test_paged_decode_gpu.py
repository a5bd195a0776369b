"""The paged decoder (machinelearning_b200/paged_decode.py) against the dense one
and the oracle: sequences at positions of their own, in f32 and 16-bit caches,
directly and from a captured graph; generation with penalties and evictions."""
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


@pytest.mark.parametrize("dtype,window,use_graph", [("f32", 0, False), ("f32", 0, True), ("f16", 0, True),
                                                    ("bf16", 0, False), ("f32", 3, False)])
def test_staggered_sequences_match_the_oracle(oracle, torch, dtype, window, use_graph):
    """Three sequences started at steps 0, 2 and 5: each one's logits are those of the
    oracle's pass over it alone. f32: the 1e-3 contract of the dense decoder; 16-bit
    caches round k and v once (2^-8 in bf16), over 6 layers within 3e-2 norm-wise. A
    window that the 10 positions exceed changes the logits of the local layers."""
    from conftest import assert_close_rel
    from oracle.decode import decode_step

    from machinelearning_b200.paged_decode import PagedGemma3Decoder
    cfg = small_config()
    w = host_weights(oracle, cfg, seed=31)
    types = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
    model = PagedGemma3Decoder(cfg, w, batch=3, cache_dtype=types[dtype], window=window)
    rng = np.random.default_rng(32)
    tokens = rng.integers(0, cfg.vocab, (3, 10))
    starts = (0, 2, 5)
    dense = [([np.zeros((1, cfg.n_kv_heads, cfg.ctx, cfg.head_dim), np.float32) for _ in range(cfg.n_layers)],
              [np.zeros((1, cfg.n_kv_heads, cfg.ctx, cfg.head_dim), np.float32) for _ in range(cfg.n_layers)])
             for _ in range(3)]
    if use_graph:
        model.start(0)
        model.capture()
        model.stop(0)
    differs = False
    for step in range(10):
        for s in range(3):
            if starts[s] == step:
                model.start(s)
        feed = [tokens[s, step - starts[s]] if step >= starts[s] else 0 for s in range(3)]
        model.step(feed)
        got = model.logits.cpu().numpy()
        for s in range(3):
            at = step - starts[s]
            if at < 0:
                continue
            ref = decode_step(cfg, w, tokens[s, at:at + 1], at, *dense[s])[0]
            if window and at >= window:
                differs = differs or np.linalg.norm(got[s] - ref) > 1e-3 * np.linalg.norm(ref)
            else:
                tol = 1e-3 if dtype == "f32" else 3e-2
                assert_close_rel(got[s], ref, tol, 10 * tol)
    assert differs == bool(window)
    assert model.positions.tolist() == [10, 8, 5] and model.host_positions == [10, 8, 5]
    model.close()


def test_generate_with_penalties_and_constraints(oracle, torch):
    from machinelearning_b200.paged_decode import PagedGemma3Decoder
    cfg = small_config()
    w = host_weights(oracle, cfg, seed=41)
    model = PagedGemma3Decoder(cfg, w, batch=3)
    prompts = [[5, 9, 14], [600], [1, 2, 3, 4, 5]]
    first = model.generate(prompts, 5)
    assert [len(o) for o in first] == [5, 5, 5] and model.positions.tolist() == [-1, -1, -1]
    assert model.generate(prompts, 5) == first  # a sequence starts from nothing
    assert model.generate(prompts[:1], 5)[0] == first[0]  # beside idle ones
    # a grammar that allows 32 tokens only, for the second sequence
    mask = torch.zeros(1, cfg.vocab // 32, dtype=torch.int32, device="cuda")
    mask[0, 3] = -1
    model.set_constraints(mask=mask, mask_rows=torch.tensor([-1, 0, -1], dtype=torch.int32, device="cuda"))
    held = model.generate(prompts, 5)
    assert all(96 <= t < 128 for t in held[1]) and held[0] == first[0] and held[2] == first[2]
    model.set_constraints()
    # a presence penalty beyond every logit: no token twice
    model.set_penalties(presence=1e4)
    for o in model.generate(prompts, 8):
        assert len(set(o)) == 8
    model.close()


def test_evictions_keep_the_budget_and_the_step_going(oracle, torch):
    """With a budget that holds every slot nothing changes; with a smaller one the
    global layers hold that many slots and generation goes on."""
    from machinelearning_b200.paged_decode import PagedGemma3Decoder
    cfg = small_config()
    w = host_weights(oracle, cfg, seed=51)
    prompts = [[7, 8, 9], [100, 200]]
    plain = PagedGemma3Decoder(cfg, w, batch=2)
    want = plain.generate(prompts, 9)
    plain.close()
    roomy = PagedGemma3Decoder(cfg, w, batch=2, budget=cfg.ctx, recent=4)
    assert roomy.generate(prompts, 9, evict_every=2) == want
    roomy.close()
    tight = PagedGemma3Decoder(cfg, w, batch=2, budget=4, recent=2)
    for s in range(2):
        tight.start(s)
    tight.capture()
    for li in tight.global_layers:
        assert not tight.slot_weights[li].any()
    for step in range(10):
        tight.step([3 + step, 50 + step])
        if step % 3 == 2:
            tight.evict()
            assert tight.slots.tolist() == [min(4, step + 1)] * 2 or step < 4
    assert tight.slots.tolist() == [5, 5] and tight.positions.tolist() == [10, 10]
    held = tight.slot_positions[tight.global_layers[0]][:, :, :5]
    assert int(held.min()) >= 0 and all(9 in row.tolist() and 8 in row.tolist() for row in held[:, 0])
    # a step adds one weight per query head, and each global layer's 4 heads attend to every slot it holds
    total = tight.slot_weights[tight.global_layers[0]].sum(-1)
    assert torch.all(total > 0) and torch.all(total <= 4 * 10 + 1e-3)
    with pytest.raises(ValueError):
        plain.evict()
    for _ in range(cfg.ctx - 10):
        tight.step([1, 2])
    with pytest.raises(ValueError, match="capacity"):
        tight.step([1, 2])
    tight.close()


def test_idle_rows_and_refusals(oracle, torch):
    from machinelearning_b200.paged_decode import PagedGemma3Decoder
    cfg = small_config()
    w = host_weights(oracle, cfg, seed=61)
    with pytest.raises(ValueError):
        PagedGemma3Decoder(cfg, w, batch=1, budget=4, recent=5)
    model = PagedGemma3Decoder(cfg, w, batch=2)
    with pytest.raises(ValueError):
        model.start(2)
    with pytest.raises(ValueError):
        model.generate([[]], 1)
    with pytest.raises(NotImplementedError):
        model.set_position(3)
    model.start(1)
    model.step([9, 9])
    per = model.block_table.shape[1]
    assert not model.k_pages[:, :per].any() and model.k_pages[:, per:].any()  # sequence 0 is idle
    assert torch.isfinite(model.logits).all()
    model.close()
