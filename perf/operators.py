"""Cases and plain forms of the paged serving operators.

Four operators of a serving step over a paged key/value cache (pages of
[kv head][slot][head_dim], one block table per sequence):

* append  -- per-head RMSNorm of q and k, position rotation, k and v into the cache
* attend  -- one new token per sequence over its cached positions
             (optionally with the attention weight each slot received)
* evict   -- keep the slots with the most accumulated attention weight
* logits  -- penalties for repeated tokens, biases and a grammar mask

``own`` selects the library's kernels; otherwise ``run`` computes the same
results with elementary torch operations in 32 bits.
"""
from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZES = {"f32": 4, "f16": 2, "bf16": 2}
DEVICE = "cuda"


# ---- cases ------------------------------------------------------------------------------

# Gemma-3-1B: 4 query heads on 1 kv head of 256; Llama-70B: 64 on 8 of 128.
GEMMA = {"nq": 4, "nkv": 1, "hd": 256}
LLAMA = {"nq": 64, "nkv": 8, "hd": 128}


def listed():
    return [
        # the smallest call: one sequence, one token of a Gemma-3-1B layer
        {"name": "append_gemma_1", "op": "append", "tokens": 1, "seqs": 1, **GEMMA, "dtype": "bf16", "page": 16,
         "start": 511, "norm": True, "offset": 1.0, "interleaved": False, "ragged": 1},
        # an ordinary decode batch of a Llama-70B layer (no q/k norm, GGUF's interleaved pairs)
        {"name": "append_llama_64", "op": "append", "tokens": 64, "seqs": 64, **LLAMA, "dtype": "f16", "page": 16,
         "start": 1000, "norm": False, "offset": 0.0, "interleaved": True, "ragged": 2},
        # the largest: a prefill chunk of 8192 tokens of four sequences
        {"name": "append_prefill_8192", "op": "append", "tokens": 8192, "seqs": 4, **LLAMA, "dtype": "bf16",
         "page": 32, "start": 0, "norm": True, "offset": 0.0, "interleaved": False, "ragged": 3},
        # the smallest: one Gemma-3-1B sequence at the decoder's context of 512, cache in f32
        {"name": "attend_gemma_1x512", "op": "attend", "seqs": 1, "longest": 512, "floor": 512, **GEMMA,
         "dtype": "f32", "page": 16, "window": 0, "weights": False, "ragged": 4},
        # an ordinary serving batch: 64 ragged sequences, one of them still empty
        {"name": "attend_llama_64_ragged", "op": "attend", "seqs": 64, "longest": 8192, "floor": 0, **LLAMA,
         "dtype": "f16", "page": 16, "window": 0, "weights": False, "ragged": 5},
        # the largest: one long document
        {"name": "attend_llama_1x131071", "op": "attend", "seqs": 1, "longest": 131071, "floor": 131071, **LLAMA,
         "dtype": "bf16", "page": 64, "window": 0, "weights": False, "ragged": 6},
        # global Gemma layers under a cache budget: the weight of every slot is accumulated
        {"name": "attend_gemma_16_weights", "op": "attend", "seqs": 16, "longest": 32001, "floor": 3000, **GEMMA,
         "dtype": "bf16", "page": 32, "window": 0, "weights": True, "ragged": 7},
        # a steady state: four Gemma sequences 65 slots over their budget
        {"name": "evict_gemma_4", "op": "evict", "seqs": 4, "longest": 4161, "floor": 4161, **GEMMA, "dtype": "bf16",
         "page": 16, "budget": 4096, "recent": 256, "ragged": 8},
        # after long prompts: ragged sequences brought down to 2048 slots, some already below it
        {"name": "evict_llama_16_ragged", "op": "evict", "seqs": 16, "longest": 8192, "floor": 1500, **LLAMA,
         "dtype": "f16", "page": 32, "budget": 2048, "recent": 128, "ragged": 9},
        # one sequence over the Gemma-3 vocabulary, under a grammar
        {"name": "logits_gemma_1", "op": "logits", "rows": 1, "vocab": 262144, "history": 300, "bias": 8,
         "masks": 4, "ragged": 10},
        # a serving batch over the Gemma-3 vocabulary
        {"name": "logits_gemma_64", "op": "logits", "rows": 64, "vocab": 262144, "history": 4096, "bias": 300,
         "masks": 16, "ragged": 11},
        # an odd vocabulary with long histories, no grammar
        {"name": "logits_odd_7", "op": "logits", "rows": 7, "vocab": 32003, "history": 30000, "bias": 0,
         "masks": 0, "ragged": 12},
    ]


def _spread(rng, lo, hi):
    """A whole number spread over the logarithm of [lo, hi]."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


HEADS = [GEMMA, LLAMA, {"nq": 32, "nkv": 4, "hd": 64}, {"nq": 8, "nkv": 8, "hd": 128}, {"nq": 15, "nkv": 3, "hd": 64},
         {"nq": 12, "nkv": 2, "hd": 192}, {"nq": 16, "nkv": 1, "hd": 128}, {"nq": 7, "nkv": 1, "hd": 256}]


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "evict", "logits"])
    ragged = rng.randrange(1 << 30)
    if op == "logits":
        vocab = rng.choice([262144, 128256, 32000, 32003, 50257, _spread(rng, 1000, 262144)])
        rows = _spread(rng, 1, max(1, 64 * 262144 // vocab))
        return {"op": op, "rows": min(rows, 256), "vocab": vocab, "history": _spread(rng, 1, 30000),
                "bias": rng.choice([0, _spread(rng, 1, 512)]), "masks": rng.choice([0, _spread(rng, 1, 32)]),
                "ragged": ragged}
    heads = rng.choice(HEADS)
    base = {"op": op, **heads, "dtype": rng.choice(["f32", "f16", "bf16"]), "page": rng.choice([16, 32, 64, 128]),
            "ragged": ragged}
    if op == "append":
        cap = 8192 * 80 * 128 // ((heads["nq"] + 2 * heads["nkv"]) * heads["hd"])
        tokens = _spread(rng, 1, min(8192, cap))
        return {**base, "tokens": tokens, "seqs": _spread(rng, 1, tokens), "start": _spread(rng, 1, 4096),
                "norm": rng.random() < 0.5, "offset": rng.choice([0.0, 1.0]), "interleaved": rng.random() < 0.5}
    slot_bytes = heads["nkv"] * heads["hd"] * SIZES[base["dtype"]]
    if op == "attend":
        cap = 131072 * 1024 * 2 // slot_bytes  # slots of the largest listed case
        longest = _spread(rng, 1, min(131072, cap))
        weights = rng.random() < 0.25
        return {**base, "seqs": _spread(rng, 1, min(256, cap // longest)), "longest": longest,
                "floor": rng.choice([0, 1, longest]), "window": rng.choice([0, 0, 0, _spread(rng, 1, 4096)]),
                "weights": weights}
    longest = _spread(rng, 64, 32768)
    cap = max(1, 16 * 8192 * 2048 // (longest * slot_bytes))
    budget = max(16, int(longest * rng.uniform(0.2, 0.99)))
    return {**base, "seqs": _spread(rng, 1, min(64, cap)), "longest": longest, "floor": rng.choice([budget, longest]),
            "budget": budget, "recent": int(budget * rng.uniform(0.0, 0.5))}


def _lengths(case):
    """Cache lengths of a case: the longest first, the others spread down to the floor (0: one sequence empty)."""
    rng = random.Random(case["ragged"])
    n, longest, floor = case["seqs"], case["longest"], case["floor"]
    out = [longest] + [_spread(rng, max(1, floor), longest) for _ in range(n - 1)]
    if floor == 0 and n > 1:
        out[rng.randrange(1, n)] = 0
    return out


def _rows(case):
    """(sequence, slot) of each appended token: consecutive slots of each sequence, the sequences of uneven length."""
    rng = random.Random(case["ragged"])
    cuts = sorted(rng.sample(range(1, case["tokens"]), case["seqs"] - 1)) if case["seqs"] > 1 else []
    counts = [b - a for a, b in zip([0] + cuts, cuts + [case["tokens"]])]
    start = [rng.randint(case["start"] // 2, case["start"]) for _ in counts]
    return [(s, start[s] + i) for s, c in enumerate(counts) for i in range(c)]


def _history(case):
    """(tokens so far, tokens of them in the prompt) of each row."""
    rng = random.Random(case["ragged"])
    total = [case["history"]] + [rng.randint(0, case["history"]) for _ in range(case["rows"] - 1)]
    return [(t, rng.randint(0, t)) for t in total]


# ---- inputs -----------------------------------------------------------------------------

def _generator(seed):
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(seed)
    return gen


def _pool(case, seqs, longest, gen, seed):
    """K and V pages with random contents, and a block table whose pages lie in random order."""
    nkv, hd, page = case["nkv"], case["hd"], case["page"]
    per = max(1, -(-longest // page))
    pages = seqs * per + 3
    shape = (pages, nkv, page, hd)
    k = torch.randn(shape, generator=gen, device=DEVICE).to(DTYPES[case["dtype"]])
    v = torch.randn(shape, generator=gen, device=DEVICE).to(DTYPES[case["dtype"]])
    order = np.random.default_rng(seed).permutation(pages)[:seqs * per].astype(np.int32)
    return k, v, torch.from_numpy(order.reshape(seqs, per)).to(DEVICE)


def _inputs(case, seed):
    gen = _generator(seed)
    randn = lambda *s: torch.randn(s, generator=gen, device=DEVICE)  # noqa: E731
    rand = lambda *s: torch.rand(s, generator=gen, device=DEVICE)  # noqa: E731
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=DEVICE)  # noqa: E731
    s = {"case": case}
    if case["op"] == "logits":
        rows, vocab = case["rows"], case["vocab"]
        hist = _history(case)
        width = case["history"]
        s["logits"] = randn(rows, vocab) * 4.0
        # frequent tokens come up often, as in text
        s["tokens"] = (rand(rows, width) ** 4 * vocab).to(torch.int32).clamp_(0, vocab - 1)
        s["token_lengths"], s["prompt_lengths"] = ints([t for t, _ in hist]), ints([p for _, p in hist])
        s["repetition"] = 1.0 + 0.3 * rand(rows)
        s["presence"], s["frequency"] = 0.5 * rand(rows), 0.2 * rand(rows)
        s["bias_ids"] = s["bias_values"] = s["mask"] = s["mask_rows"] = None
        if case["bias"]:
            pick = torch.stack([torch.randperm(vocab, generator=gen, device=DEVICE)[:case["bias"]]
                                for _ in range(rows)])
            s["bias_ids"] = pick.to(torch.int32)
            s["bias_values"] = randn(rows, pick.shape[1]) * 5.0
        if case["masks"]:
            words = (vocab + 31) // 32
            # grammar states: from a few allowed tokens to nearly all
            allowed = rand(case["masks"], vocab) < torch.logspace(-3, -0.01, case["masks"], device=DEVICE)[:, None]
            bits = torch.zeros(case["masks"], words * 32, dtype=torch.int64, device=DEVICE)
            bits[:, :vocab] = allowed
            packed = (bits.view(-1, words, 32) << torch.arange(32, device=DEVICE)).sum(-1)
            s["mask"] = torch.where(packed >= 2 ** 31, packed - 2 ** 32, packed).to(torch.int32)
            rng = random.Random(seed)
            s["mask_rows"] = ints([rng.randrange(-1, case["masks"]) if r else 0 for r in range(rows)])
        return s
    nq, nkv, hd = case["nq"], case["nkv"], case["hd"]
    if case["op"] == "append":
        rows = _rows(case)
        longest = max(p for _, p in rows) + 1
        s["k"], s["v"], s["table"] = _pool(case, case["seqs"], longest, gen, seed)
        s["seqs"], s["slots"] = ints([q for q, _ in rows]), ints([p for _, p in rows])
        s["positions"] = s["slots"].clone()
        s["qkv"] = randn(case["tokens"], (nq + 2 * nkv) * hd)
        s["q_norm"] = randn(hd) * 0.1 + (1.0 - case["offset"]) if case["norm"] else None
        s["k_norm"] = randn(hd) * 0.1 + (1.0 - case["offset"]) if case["norm"] else None
        angle = torch.arange(longest, device=DEVICE, dtype=torch.float64)[:, None] * (
            10000.0 ** (-torch.arange(hd // 2, device=DEVICE, dtype=torch.float64) * 2.0 / hd))
        s["cos"], s["sin"] = angle.cos().float().contiguous(), angle.sin().float().contiguous()
        return s
    lengths = _lengths(case)
    s["k"], s["v"], s["table"] = _pool(case, case["seqs"], case["longest"], gen, seed)
    s["lengths"] = ints(lengths)
    capacity = s["table"].shape[1] * case["page"]
    live = torch.arange(capacity, device=DEVICE) < s["lengths"][:, None, None]
    s["weights"] = torch.where(live, rand(case["seqs"], nkv, capacity) ** 4 * 8.0, 0.0)
    if case["op"] == "attend":
        s["q"] = randn(case["seqs"], nq, hd) * 2.0
        s["scale"] = 1.0 / math.sqrt(hd)
        s["weights_out"] = torch.zeros_like(s["weights"]) if case["weights"] else None
        return s
    # earlier evictions left gaps in the positions: slots hold every position but some older ones
    gap = torch.randint(0, 1000, (case["seqs"],), generator=gen, device=DEVICE, dtype=torch.int32)
    slot = torch.arange(capacity, device=DEVICE, dtype=torch.int32)
    old = slot < s["lengths"][:, None, None] - case["recent"]
    positions = torch.where(old, slot, slot + gap[:, None, None])
    s["positions"] = torch.where(live, positions, -1).expand(-1, nkv, -1).to(torch.int32).contiguous()
    s["next_positions"] = s["lengths"] + gap
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if own and "k" in s:
        from machinelearning_b200.paged import PagedKVCache
        s["cache"] = PagedKVCache(s["k"], s["v"], s["table"])
    return s


# ---- one pass ---------------------------------------------------------------------------

def run(state):
    return (_own if own else _plain)[state["case"]["op"]](state)


def _own_append(s):
    c = s["case"]
    q = s["cache"].append(s["qkv"], s["positions"], s["slots"], s["cos"], s["sin"], n_heads=c["nq"],
                          q_norm=s["q_norm"], k_norm=s["k_norm"], offset=c["offset"], eps=1e-6, seqs=s["seqs"],
                          interleaved=c["interleaved"])
    return q, s["k"], s["v"]


def _own_attend(s):
    c = s["case"]
    if not c["weights"]:
        return s["cache"].attend(s["q"], s["lengths"], s["scale"], window=c["window"])
    out = s["cache"].attend(s["q"], s["lengths"], s["scale"], window=c["window"], weights=s["weights"],
                            weights_out=s["weights_out"])
    return out, s["weights_out"]


def _own_evict(s):
    c = s["case"]
    lengths, weights, positions = s["cache"].evict(s["lengths"], s["weights"], s["positions"], s["next_positions"],
                                                   budget=c["budget"], recent=c["recent"])
    return lengths, weights, positions, s["k"], s["v"]


def _own_logits(s):
    from machinelearning_b200.logits import process_logits
    return process_logits(s["logits"], tokens=s["tokens"], token_lengths=s["token_lengths"],
                          prompt_lengths=s["prompt_lengths"], repetition=s["repetition"], presence=s["presence"],
                          frequency=s["frequency"], bias_ids=s["bias_ids"], bias_values=s["bias_values"],
                          mask=s["mask"], mask_rows=s["mask_rows"])


def _plain_append(s):
    c = s["case"]
    nq, nkv, hd, half = c["nq"], c["nkv"], c["hd"], c["hd"] // 2
    x = s["qkv"].view(c["tokens"], nq + 2 * nkv, hd)
    q, k, v = x[:, :nq], x[:, nq:nq + nkv], x[:, nq + nkv:]
    if c["norm"]:
        q = q / torch.sqrt((q * q).mean(-1, keepdim=True) + 1e-6) * (s["q_norm"] + c["offset"])
        k = k / torch.sqrt((k * k).mean(-1, keepdim=True) + 1e-6) * (s["k_norm"] + c["offset"])
    pos = s["positions"].long()
    cos, sin = s["cos"][pos][:, None, :], s["sin"][pos][:, None, :]

    def rotate(t):
        if c["interleaved"]:
            a, b = t[..., 0::2], t[..., 1::2]
            return torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)
        a, b = t[..., :half], t[..., half:]
        return torch.cat((a * cos - b * sin, a * sin + b * cos), -1)

    slots = s["slots"].long()
    pages = s["table"][s["seqs"].long(), slots // c["page"]].long()
    s["k"][pages, :, slots % c["page"]] = rotate(k).to(s["k"].dtype)
    s["v"][pages, :, slots % c["page"]] = v.to(s["v"].dtype)
    return rotate(q).contiguous(), s["k"], s["v"]


def _gather(pages, table, longest):
    """[seqs][kv heads][longest][head_dim] in 32 bits from the pages."""
    seqs, per = table.shape
    t = pages[table.long()].transpose(1, 2)  # [seqs][kv heads][pages][slot][head_dim]
    return t.reshape(seqs, pages.shape[1], per * pages.shape[2], pages.shape[3])[:, :, :longest].float()


def _plain_attend(s):
    c = s["case"]
    g, longest = c["nq"] // c["nkv"], c["longest"]
    slot = torch.arange(longest, device=DEVICE)
    n = s["lengths"][:, None]
    seen = slot < n
    if c["window"]:
        seen = seen & (slot >= n - c["window"])
    seen = seen[:, None, None, :]
    k = _gather(s["k"], s["table"], longest)
    q = s["q"].view(c["seqs"], c["nkv"], g, c["hd"])
    score = torch.matmul(q, k.transpose(-1, -2)) * s["scale"]
    del k
    score = torch.where(seen, score, float("-inf"))
    top = score.amax(-1, keepdim=True)
    e = torch.exp(score - torch.where(top == float("-inf"), 0.0, top))
    total = e.sum(-1, keepdim=True)
    p = torch.where(total > 0, e / total, 0.0)
    v = torch.where(seen.transpose(-1, -2), _gather(s["v"], s["table"], longest), 0.0)
    out = torch.matmul(p, v).view(c["seqs"], c["nq"], c["hd"])
    if not c["weights"]:
        return out
    weights = s["weights"].clone()
    weights[:, :, :longest] += p.sum(2)
    return out, weights


def _plain_evict(s):
    c = s["case"]
    capacity = s["weights"].shape[-1]
    slot = torch.arange(capacity, device=DEVICE)
    n = s["lengths"].long()[:, None, None]
    valid = slot < n
    recent = s["positions"] >= (s["next_positions"] - c["recent"])[:, None, None]
    key = torch.where(valid, torch.where(recent, float("inf"), s["weights"]), float("-inf"))
    order = torch.sort(key, dim=-1, descending=True, stable=True).indices
    rank = torch.empty_like(order).scatter_(-1, order, slot.expand_as(order).contiguous())
    keep = valid & ((rank < c["budget"]) | (n <= c["budget"]))
    hole = ~keep & valid & (slot < c["budget"])
    mover = keep & (slot >= c["budget"])
    dst, src = hole.nonzero(as_tuple=True), mover.nonzero(as_tuple=True)  # both in row, slot order
    weights, positions = s["weights"].clone(), s["positions"].clone()
    weights[dst], positions[dst] = s["weights"][src], s["positions"][src]
    lengths = torch.minimum(s["lengths"], torch.full_like(s["lengths"], c["budget"]))
    gone = slot >= lengths[:, None, None]
    weights, positions = torch.where(gone, 0.0, weights), torch.where(gone, -1, positions)
    to = s["table"][dst[0], dst[2] // c["page"]].long()
    of = s["table"][src[0], src[2] // c["page"]].long()
    for t in (s["k"], s["v"]):
        t[to, dst[1], dst[2] % c["page"]] = t[of, src[1], src[2] % c["page"]]
    return lengths, weights, positions, s["k"], s["v"]


def _plain_logits(s):
    c = s["case"]
    rows, vocab = c["rows"], c["vocab"]
    at = torch.arange(c["history"], device=DEVICE)
    in_history = at < s["token_lengths"][:, None]
    in_output = in_history & (at >= s["prompt_lengths"][:, None])
    ids = s["tokens"].long()
    seen = torch.zeros(rows, vocab, dtype=torch.int32, device=DEVICE).scatter_add_(1, ids, in_history.int())
    count = torch.zeros(rows, vocab, dtype=torch.int32, device=DEVICE).scatter_add_(1, ids, in_output.int())
    x, r = s["logits"], s["repetition"][:, None]
    x = torch.where(seen > 0, torch.where(x > 0, x / r, x * r), x)
    x = x - s["frequency"][:, None] * count - s["presence"][:, None] * (count > 0)
    if s["bias_ids"] is not None:
        x = x.scatter_add(1, s["bias_ids"].long(), s["bias_values"])
    if s["mask"] is not None:
        bits = (s["mask"][s["mask_rows"].clamp(min=0).long()][:, :, None] >> torch.arange(32, device=DEVICE)) & 1
        allowed = bits.flatten(1)[:, :vocab].bool() | (s["mask_rows"] < 0)[:, None]
        x = torch.where(allowed, x, float("-inf"))
    return x


_own = {"append": _own_append, "attend": _own_attend, "evict": _own_evict, "logits": _own_logits}
_plain = {"append": _plain_append, "attend": _plain_attend, "evict": _plain_evict, "logits": _plain_logits}


# ---- what a pass cannot do without --------------------------------------------------------

def work(case):
    if case["op"] == "logits":
        rows, vocab = case["rows"], case["vocab"]
        tokens = sum(t for t, _ in _history(case))
        moved = rows * vocab * 8 + tokens * 4 + rows * case["bias"] * 8 + min(case["masks"], rows) * vocab / 8
        return {"bytes": moved, "flops": 4 * rows * vocab}
    nq, nkv, hd, size = case["nq"], case["nkv"], case["hd"], SIZES[case["dtype"]]
    if case["op"] == "append":
        t = case["tokens"]
        tables = len({p for _, p in _rows(case)}) * hd * 4
        return {"bytes": t * ((2 * nq + 2 * nkv) * hd * 4 + 2 * nkv * hd * size) + tables,
                "flops": t * (nq + nkv) * hd * 7}
    lengths = _lengths(case)
    capacity = max(1, -(-case["longest"] // case["page"])) * case["page"]
    if case["op"] == "attend":
        seen = sum(min(n, case["window"]) if case["window"] else n for n in lengths)
        moved = 2 * seen * nkv * hd * size + case["seqs"] * nq * hd * 8
        if case["weights"]:
            moved += case["seqs"] * nkv * capacity * 8
        return {"bytes": moved, "flops": 4 * seen * nq * hd}
    moved, flops = 0.0, 0.0
    budget, recent = case["budget"], case["recent"]
    for n in lengths:
        moved += nkv * (min(n, capacity) * 8 + capacity * 8)
        flops += nkv * n * 4
        if n > budget:
            # kept slots above the budget: the recent ones, and their share of the older ones
            kept = min(recent, n - budget) + max(0, n - budget - recent) * (budget - recent) / max(1, n - recent)
            moved += nkv * kept * hd * size * 4
    return {"bytes": moved, "flops": flops}


# ---- the definitions in 64 bits -----------------------------------------------------------

def exact(case, seed):
    return _exact[case["op"]](case, _inputs(case, seed))


def _exact_append(case, s):
    nq, nkv, hd = case["nq"], case["nkv"], case["hd"]
    x = s["qkv"].double().reshape(case["tokens"], -1, hd)
    if case["norm"]:
        gain = torch.cat((s["q_norm"].double().expand(nq, hd), s["k_norm"].double().expand(nkv, hd))) + case["offset"]
        r = torch.rsqrt(x[:, :nq + nkv].pow(2).sum(-1, keepdim=True) / hd + 1e-6)
        x = torch.cat((x[:, :nq + nkv] * r * gain, x[:, nq + nkv:]), 1)
    # the rotation as a product of complex numbers
    turn = torch.complex(s["cos"].double(), s["sin"].double())[s["positions"].long()][:, None]
    pairs = x[:, :nq + nkv]
    pairs = pairs.unflatten(-1, (-1, 2)) if case["interleaved"] else pairs.unflatten(-1, (2, -1)).transpose(-1, -2)
    z = torch.view_as_real(torch.complex(pairs[..., 0].contiguous(), pairs[..., 1].contiguous()) * turn)
    z = z.flatten(-2) if case["interleaved"] else z.transpose(-1, -2).flatten(-2)
    k, v = s["k"].double(), s["v"].double()
    page, off = torch.div(s["slots"], case["page"], rounding_mode="floor").long(), s["slots"].long() % case["page"]
    where = s["table"].long()[s["seqs"].long(), page]
    for h in range(nkv):
        k[where, h, off] = z[:, nq + h]
        v[where, h, off] = x[:, nq + nkv + h]
    return z[:, :nq].contiguous(), k, v


def _exact_attend(case, s):
    nq, nkv, hd, page = case["nq"], case["nkv"], case["hd"], case["page"]
    out = torch.zeros(case["seqs"], nq, hd, dtype=torch.float64, device=DEVICE)
    weights = s["weights"].double()
    for b, n in enumerate(_lengths(case)):
        first = max(0, n - case["window"]) if case["window"] else 0
        if n == first:
            continue
        slots = torch.arange(first, n, device=DEVICE)
        rows = s["table"][b].long()[slots // page]
        k = s["k"][rows, :, slots % page].double()  # [slots][kv heads][head_dim]
        v = s["v"][rows, :, slots % page].double()
        q = s["q"][b].double().view(nkv, nq // nkv, hd)
        p = torch.softmax(torch.einsum("hgd,nhd->hgn", q, k) * s["scale"], -1)
        out[b] = torch.einsum("hgn,nhd->hgd", p, v).reshape(nq, hd)
        weights[b, :, first:n] += p.sum(1)
    return (out, weights) if case["weights"] else out


def _exact_evict(case, s):
    budget, page = case["budget"], case["page"]
    table, k, v = s["table"].cpu().numpy(), s["k"], s["v"]
    weights, positions = s["weights"].double().cpu().numpy(), s["positions"].cpu().numpy().copy()
    limit = s["next_positions"].cpu().numpy().astype(np.int64) - case["recent"]
    lengths = _lengths(case)
    moves = []
    for b, n in enumerate(lengths):
        for h in range(case["nkv"]):
            m = min(n, budget)
            if n > budget:
                w = np.where(positions[b, h, :n] >= limit[b], np.inf, weights[b, h, :n])
                kept = np.zeros(n, bool)
                kept[np.lexsort((np.arange(n), -w))[:budget]] = True
                to, of = np.flatnonzero(~kept[:budget]), budget + np.flatnonzero(kept[budget:])
                weights[b, h, to], positions[b, h, to] = weights[b, h, of], positions[b, h, of]
                moves.append(np.stack([table[b, to // page], np.full_like(to, h), to % page,
                                       table[b, of // page], np.full_like(of, h), of % page]))
            weights[b, h, m:], positions[b, h, m:] = 0.0, -1
    if moves:
        tp, th, to, fp, fh, fo = torch.from_numpy(np.concatenate(moves, 1).astype(np.int64)).to(DEVICE)
        k[tp, th, to], v[tp, th, to] = k[fp, fh, fo], v[fp, fh, fo]
    short = torch.tensor([min(n, budget) for n in lengths], dtype=torch.int32, device=DEVICE)
    return short, torch.from_numpy(weights).to(DEVICE), torch.from_numpy(positions).to(DEVICE), k, v


def _exact_logits(case, s):
    x = s["logits"].double()
    for b, (total, prompt) in enumerate(_history(case)):
        text = s["tokens"][b].long()
        used = torch.unique(text[:total])
        old = x[b, used]
        rep = s["repetition"][b].double()
        x[b, used] = torch.where(old > 0, old / rep, old * rep)
        ids, count = torch.unique(text[prompt:total], return_counts=True)
        x[b, ids] -= s["frequency"][b].double() * count + s["presence"][b].double()
        if s["bias_ids"] is not None:
            x[b].index_add_(0, s["bias_ids"][b].long(), s["bias_values"][b].double())
        row = int(s["mask_rows"][b]) if s["mask"] is not None else -1
        if row >= 0:
            words = s["mask"][row].cpu().numpy()
            bits = np.unpackbits(words.view(np.uint8), bitorder="little")[:case["vocab"]]
            x[b, torch.from_numpy(bits == 0).to(DEVICE)] = float("-inf")
    return x


_exact = {"append": _exact_append, "attend": _exact_attend, "evict": _exact_evict, "logits": _exact_logits}
