"""Timed calls of the mixers that stand beside ``rosa_soft``: decayed linear attention and
attention with a sliding window and sinks, in training and in serving.

``listed()`` names the fixed cases, ``draw(rng)`` gives one more of the same ranges,
``prepare(case, seed)`` makes what a program holds before the call, ``run(state)`` is one pass,
``work(case)`` counts what a pass cannot do without and ``exact(case, seed)`` is the answer in
64 bits.  With ``own`` false a pass is the operator's formula in elementary tensor operations,
with ``own`` true the call of the framework.

The kinds of a case:

* ``decay_train`` / ``window_train``: forward and backward over a batch (``B`` x ``T``) or over
  packed sequences (``lengths``);
* ``decay_update``: ``T`` tokens for each of ``S`` slots on top of the slots' states;
* ``window_update``: the same on top of the slots' key-value caches.
"""

from __future__ import annotations

import math

import torch

own = False

DEVICE = "cuda:0"
ITEM_BYTES = {"float32": 4, "float16": 2, "bfloat16": 2}


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------

def _train(kind, name, dtype, H, Hkv, D, Dv, B=0, T=0, lengths="", window=0, sinks=0):
    case = dict(kind=kind, dtype=dtype, B=B, T=T, lengths=lengths, H=H, Hkv=Hkv, D=D, Dv=Dv)
    if kind == "window_train":
        case.update(window=window, sinks=sinks)
    if name:
        case["name"] = name
    return case


def _update(kind, name, dtype, S, T, H, Hkv, D, Dv, past, window=0, sinks=0):
    """``past``: the most tokens that a slot already holds; the slots' own numbers are drawn."""
    case = dict(kind=kind, dtype=dtype, S=S, T=T, H=H, Hkv=Hkv, D=D, Dv=Dv, past=past)
    if kind == "window_update":
        case.update(window=window, sinks=sinks)
    if name:
        case["name"] = name
    return case


def listed():
    return [
        # the smallest model that is trained in earnest: a step is a handful of launches
        _train("decay_train", "decay_train_tiny", "float32", H=4, Hkv=4, D=32, Dv=32, B=1, T=256),
        # a layer of a mid-sized model in mixed precision, a head of keys and values per query head
        _train("decay_train", "decay_train", "bfloat16", H=32, Hkv=32, D=128, Dv=128, B=2, T=4096),
        # samples as they come: odd lengths, one of a single token, shared heads, odd widths
        _train("decay_train", "decay_train_ragged", "float16", H=12, Hkv=6, D=48, Dv=80,
               lengths="1,37,129,513,1000,2047,3001"),
        # serving: four prompts of 2048 tokens, their states behind them
        _update("decay_update", "decay_prompt", "bfloat16", S=4, T=2048, H=32, Hkv=32, D=128,
                Dv=128, past=0),
        # serving: one more token for each of 64 slots
        _update("decay_update", "decay_token", "bfloat16", S=64, T=1, H=32, Hkv=32, D=128, Dv=128,
                past=4096),
        # one slot, one token, a small model: nothing but latency
        _update("decay_update", "decay_token_one", "float32", S=1, T=1, H=16, Hkv=16, D=64, Dv=64,
                past=512),
        # the smallest model again, with a window of a quarter of its context
        _train("window_train", "window_train_tiny", "float32", H=4, Hkv=2, D=32, Dv=32, B=1, T=256,
               window=64, sinks=2),
        # a layer of a mid-sized model with grouped heads; the largest step
        _train("window_train", "window_train", "bfloat16", H=32, Hkv=8, D=128, Dv=128, B=2, T=4096,
               window=1024, sinks=4),
        # samples as they come, a window that no tile divides
        _train("window_train", "window_train_ragged", "float16", H=12, Hkv=4, D=80, Dv=80,
               lengths="1,37,129,513,1000,2047,3001", window=257, sinks=3),
        # serving: the second part of long prompts, behind what the caches already hold
        _update("window_update", "window_prompt", "bfloat16", S=4, T=2048, H=32, Hkv=8, D=128,
                Dv=128, past=2500, window=1500, sinks=4),
        # serving: one more token for each of 64 slots whose caches are filled to various lengths
        _update("window_update", "window_token", "bfloat16", S=64, T=1, H=32, Hkv=8, D=128, Dv=128,
                past=9000, window=4096, sinks=4),
        # one slot with a very long window: its cache is all there is to share out
        _update("window_update", "window_token_long", "float16", S=1, T=1, H=16, Hkv=2, D=64, Dv=64,
                past=200000, window=65536, sinks=4),
    ]


def _spread(rng, low, high):
    """An integer between the bounds, even over the logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


MOST_SCORES = 5.0e8    # heads x (query, key) pairs of a drawn one, visible or not
MOST_BYTES = 2.0e8     # of a drawn single-token update


def draw(rng):
    kind = rng.choice(["decay_train", "decay_update", "window_train", "window_update"])
    dtype = rng.choice(["float32", "float16", "bfloat16"])
    kv_heads = _spread(rng, 1, 16)
    heads = kv_heads * rng.choice([1, 1, 2, 4])
    width = rng.choice([16, 32, 40, 64, 64, 72, 80, 96, 128, 128])
    value_width = width if rng.random() < 0.7 else rng.choice([24, 32, 33, 64, 100, 128])
    shape = dict(H=heads, Hkv=kv_heads, D=width, Dv=value_width)
    window, sinks = _spread(rng, 16, 4096), rng.choice([0, 1, 2, 4, 16])
    masks = dict(window=window, sinks=sinks) if kind.startswith("window") else {}
    if kind.endswith("train"):
        longest = _spread(rng, 32, 6000)
        most = max(1, min(8, int(MOST_SCORES / (heads * longest ** 2))))
        count = rng.randint(1, most)
        if rng.random() < 0.4:
            lengths = [longest if i == 0 else _spread(rng, 1, longest) for i in range(count)]
            # the plain form scores every token against every other one
            cut = int((MOST_SCORES / heads) ** 0.5)
            kept = [n for i, n in enumerate(lengths) if sum(lengths[:i + 1]) <= cut]
            case = _train(kind, "", dtype, lengths=",".join(map(str, kept or [min(longest, cut)])),
                          **shape, **masks)
        else:
            longest = min(longest, int((MOST_SCORES / heads) ** 0.5))
            case = _train(kind, "", dtype, B=count, T=longest, **shape, **masks)
        return case
    if rng.random() < 0.4:  # a prompt
        tokens = _spread(rng, 2, 4000)
        past = rng.choice([0, _spread(rng, 1, 5000)])
        if kind == "window_update":
            seen = tokens + min(window + tokens, 5000)
            tokens = max(2, min(tokens, int(MOST_SCORES / (heads * seen))))
        else:
            tokens = max(2, min(tokens, int((MOST_SCORES / heads) ** 0.5)))
        most = max(1, min(8, int(MOST_SCORES / (heads * tokens * (2 * tokens + window)))))
        return _update(kind, "", dtype, S=rng.randint(1, most), T=tokens, past=past, **shape,
                       **masks)
    past = _spread(rng, 1, 100000)
    if kind == "window_update":
        window = _spread(rng, 16, 65536)
        masks = dict(window=window, sinks=sinks)
        one = kv_heads * (window + sinks) * (width + value_width) * ITEM_BYTES[dtype]
    else:
        one = heads * width * value_width * 8
    slots = _spread(rng, 1, max(1, min(256, int(MOST_BYTES / one))))
    return _update(kind, "", dtype, S=slots, T=1, past=past, **shape, **masks)


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _lengths(case):
    if case.get("lengths"):
        return [int(item) for item in case["lengths"].split(",")]
    return [case["T"]] * case["B"]


def _log_decay(heads):
    """Heads that forget over 32 tokens up to heads that remember 4096: log(1 - 2^-5 .. 2^-12)."""
    exponents = torch.linspace(5.0, 12.0, heads, dtype=torch.float64) if heads > 1 \
        else torch.tensor([7.0], dtype=torch.float64)
    return torch.log1p(-torch.exp2(-exponents)).float().to(DEVICE)


def prepare(case, seed):
    generator = torch.Generator(device=DEVICE).manual_seed(int(seed))
    dtype = getattr(torch, case["dtype"])
    randn = lambda *dims: torch.randn(*dims, device=DEVICE, generator=generator)
    kind, H, Hkv, D, Dv = (case[name] for name in ("kind", "H", "Hkv", "D", "Dv"))
    state = dict(kind=kind, log_decay=_log_decay(H))
    if kind.startswith("window"):
        state["controls"] = dict(window=case["window"], sinks=case["sinks"])
    if kind.endswith("train"):
        lead, offsets = (case["B"], case["T"]), None
        if case["lengths"]:
            ends = torch.tensor([0, *_lengths(case)], dtype=torch.int32).cumsum(0)
            offsets = ends.to(device=DEVICE, dtype=torch.int32)
            lead = (int(ends[-1]),)
        leaves = [randn(*lead, H, D), randn(*lead, Hkv, D), randn(*lead, Hkv, Dv)]
        state.update(
            leaves=[leaf.to(dtype).requires_grad_() for leaf in leaves], offsets=offsets,
            # the gradient that the layers above hand to the operator's output
            grad_output=randn(*lead, H, Dv).to(dtype))
        return state
    S, T = case["S"], case["T"]
    state["inputs"] = [randn(S, T, H, D).to(dtype), randn(S, T, Hkv, D).to(dtype),
                       randn(S, T, Hkv, Dv).to(dtype)]
    # what the slots have seen: all of them nothing, or each a number of its own up to the most
    past = torch.rand(S, device=DEVICE, generator=generator).mul(0.75).add(0.25).mul(case["past"])
    past = past.round().to(torch.int32)
    past[-1:] = case["past"]
    state["lengths"] = past
    if kind == "decay_update":
        # sums over the tokens seen so far: as large as the number that the head remembers
        seen = torch.exp(state["log_decay"]).view(1, H, 1, 1)
        weight = (1 - seen.pow(2 * past.view(S, 1, 1, 1))) / (1 - seen.square())
        state["state"] = randn(S, H, D, Dv) * weight.sqrt()
        state["state_out"] = torch.empty_like(state["state"])
        return state
    # the ring holds the window of the first new token and all new tokens
    capacity = case["sinks"] + case["window"] + T - 1
    state["caches"] = [randn(S, Hkv, capacity, D).to(dtype), randn(S, Hkv, capacity, Dv).to(dtype)]
    return state


# ---------------------------------------------------------------------------
# the plain forms: float32, one product per contraction, no library attention
# ---------------------------------------------------------------------------

def _heads_first(tensor, heads):
    """float32 ``[..., H, T, D]`` of ``[..., T, Hkv, D]``, shared heads repeated."""
    tensor = tensor.detach().float().transpose(-2, -3)
    return tensor.repeat_interleave(heads // tensor.shape[-3], dim=-3)


def _tokens_first(tensor, shared, dtype):
    """``[..., T, Hkv, D]`` of ``[..., H, T, D]``, the gradients of a shared head summed."""
    if tensor.shape[-3] != shared:
        tensor = tensor.unflatten(-3, (shared, -1)).sum(-3)
    return tensor.transpose(-2, -3).to(dtype).contiguous()


def _distances(tokens, offsets):
    """``t - s`` of every pair of tokens, the token's own position, and whether ``s`` may be seen."""
    index = torch.arange(tokens, device=DEVICE)
    distance = index[:, None] - index[None, :]
    if offsets is None:
        return distance, index, distance >= 0
    sequence = torch.searchsorted(offsets[1:].long(), index, right=True)
    return (distance, index - offsets.long()[sequence],
            (distance >= 0) & (sequence[:, None] == sequence[None, :]))


def _plain_decay_train(state):
    query, key, value = state["leaves"]
    H, Hkv, dtype, scale = query.shape[-2], key.shape[-2], query.dtype, query.shape[-1] ** -0.5
    q, k, v = (_heads_first(leaf, H) for leaf in state["leaves"])
    grad = _heads_first(state["grad_output"], H)
    distance, _, visible = _distances(q.shape[-2], state["offsets"])
    weight = torch.exp(distance.float() * state["log_decay"].view(H, 1, 1))
    weight = torch.where(visible, weight * scale, 0.0)
    scores = torch.matmul(q, k.transpose(-1, -2)) * weight
    utility = torch.matmul(grad, v.transpose(-1, -2)) * weight
    return [_tokens_first(torch.matmul(scores, v), H, dtype),
            _tokens_first(torch.matmul(utility, k), H, dtype),
            _tokens_first(torch.matmul(utility.transpose(-1, -2), q), Hkv, dtype),
            _tokens_first(torch.matmul(scores.transpose(-1, -2), grad), Hkv, dtype)]


def _plain_decay_update(state):
    query, key, value = state["inputs"]
    H, T, dtype, scale = query.shape[-2], query.shape[1], query.dtype, query.shape[-1] ** -0.5
    q, k, v = (_heads_first(tensor, H) for tensor in state["inputs"])
    rate = state["log_decay"].view(H, 1, 1)
    distance, index, visible = _distances(T, None)
    weight = torch.where(visible, torch.exp(distance.float() * rate), 0.0)
    before = torch.exp((index + 1).float()[:, None] * rate)        # of the state, at each token
    behind = torch.exp((T - 1 - index).float()[:, None] * rate)    # of each token, in the new state
    scores = torch.matmul(q, k.transpose(-1, -2)) * weight
    output = torch.matmul(scores, v) + torch.matmul(q * before, state["state"])
    state["state_out"].copy_(
        state["state"] * torch.exp(T * rate) + torch.matmul((k * behind).transpose(-1, -2), v))
    return [_tokens_first(output * scale, H, dtype), state["state_out"]]


def _softmax(scores, visible):
    scores = torch.where(visible, scores, -torch.inf)
    weights = torch.exp(scores - scores.amax(-1, keepdim=True))
    return weights / weights.sum(-1, keepdim=True)


def _plain_window_train(state):
    query, key, value = state["leaves"]
    H, Hkv, dtype, scale = query.shape[-2], key.shape[-2], query.dtype, query.shape[-1] ** -0.5
    q, k, v = (_heads_first(leaf, H) for leaf in state["leaves"])
    grad = _heads_first(state["grad_output"], H)
    distance, position, visible = _distances(q.shape[-2], state["offsets"])
    visible = visible & ((distance < state["controls"]["window"])
                         | (position[None, :] < state["controls"]["sinks"]))
    weights = _softmax(torch.matmul(q, k.transpose(-1, -2)) * scale, visible)
    utility = torch.matmul(grad, v.transpose(-1, -2))
    slope = weights * (utility - (weights * utility).sum(-1, keepdim=True)) * scale
    return [_tokens_first(torch.matmul(weights, v), H, dtype),
            _tokens_first(torch.matmul(slope, k), H, dtype),
            _tokens_first(torch.matmul(slope.transpose(-1, -2), q), Hkv, dtype),
            _tokens_first(torch.matmul(weights.transpose(-1, -2), grad), Hkv, dtype)]


def _plain_window_update(state):
    query, key, value = state["inputs"]
    S, T, H, D = query.shape
    Hkv, scale = key.shape[-2], D ** -0.5
    window, sinks = state["controls"]["window"], state["controls"]["sinks"]
    past = state["lengths"].long()
    key_cache, value_cache = state["caches"]
    capacity = key_cache.shape[2]
    ring, row = capacity - sinks, torch.arange(capacity, device=DEVICE)
    # the position that each row of the cache holds: its own for the sinks, the newest one that
    # falls on it for the ring
    newest = past[:, None] - 1 - (past[:, None] - 1 - row) % ring
    held = torch.where(row < sinks, row, newest)
    known = (held < past[:, None]) & ((row < sinks) | (held >= sinks))
    q = _heads_first(query, H)
    keys = torch.cat([key_cache, key.transpose(1, 2)], dim=2).float()
    values = torch.cat([value_cache, value.transpose(1, 2)], dim=2).float()
    keys, values = (t.repeat_interleave(H // Hkv, dim=1) for t in (keys, values))
    fresh = past[:, None] + torch.arange(T, device=DEVICE)
    where = torch.cat([held, fresh], dim=1)[:, None, :]
    there = torch.cat([known, torch.ones_like(fresh, dtype=torch.bool)], dim=1)[:, None, :]
    distance = fresh[:, :, None] - where
    visible = there & (distance >= 0) & ((distance < window) | (where < sinks))
    weights = _softmax(torch.matmul(q, keys.transpose(-1, -2)) * scale, visible[:, None])
    output = _tokens_first(torch.matmul(weights, values), H, query.dtype)
    # the new tokens that the cache keeps: each on its row
    rows = torch.where(fresh < sinks, fresh, sinks + (fresh - sinks) % ring)
    slot, token = torch.nonzero((fresh < sinks) | (fresh >= past[:, None] + T - ring),
                                as_tuple=True)
    key_cache[slot, :, rows[slot, token]] = key[slot, token]
    value_cache[slot, :, rows[slot, token]] = value[slot, token]
    return [output, key_cache, value_cache]


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def _own_train(state):
    from rosa_soft_amd import mixers

    leaves, offsets = state["leaves"], state["offsets"]
    if state["kind"] == "decay_train":
        if offsets is None:
            output = mixers.decay_attention(*leaves, state["log_decay"])
        else:
            output = mixers.decay_attention_varlen(*leaves, offsets, state["log_decay"])
    elif offsets is None:
        output = mixers.window_attention(*leaves, **state["controls"])
    else:
        output = mixers.window_attention_varlen(*leaves, offsets, **state["controls"])
    return [output.detach(), *torch.autograd.grad(output, leaves, state["grad_output"])]


def _own_update(state):
    from rosa_soft_amd import mixers

    if state["kind"] == "decay_update":
        # the new states go to a second tensor that takes turns with the first
        output = mixers.decay_attention_update(*state["inputs"], state["log_decay"],
                                               state["state"], state_out=state["state_out"])
        return [output, state["state_out"]]
    output = mixers.window_attention_update(*state["inputs"], *state["caches"], state["lengths"],
                                            **state["controls"])
    return [output, *state["caches"]]


def run(state):
    if own:
        return _own_train(state) if "leaves" in state else _own_update(state)
    plain = {"decay_train": _plain_decay_train, "decay_update": _plain_decay_update,
             "window_train": _plain_window_train, "window_update": _plain_window_update}
    return plain[state["kind"]](state)


# ---------------------------------------------------------------------------
# what a pass needs
# ---------------------------------------------------------------------------

def _visible_pairs(tokens, past, window, sinks):
    """(query, key) pairs of ``tokens`` new tokens behind ``past`` earlier ones."""
    def upto(n):  # of the first n tokens of a sequence
        near = n * (n + 1) // 2 if n <= window else window * (window + 1) // 2 + (n - window) * window
        # token t sees, beyond its window, the sinks before position t - window + 1
        beyond = max(0, n - window)
        few = min(beyond, sinks)
        return near + few * (few + 1) // 2 + (beyond - few) * sinks
    return upto(past + tokens) - upto(past)


def work(case):
    kind, item = case["kind"], ITEM_BYTES[case["dtype"]]
    H, Hkv, D, Dv = (case[name] for name in ("H", "Hkv", "D", "Dv"))
    token = (H * (D + Dv) + Hkv * (D + Dv)) * item  # query, output, key, value
    if kind.endswith("train"):
        lengths = _lengths(case)
        size = 2 * sum(lengths) * token              # and the gradients of the four
        if kind == "decay_train":                    # output, dq, dk, dv: a state updated and read
            return {"bytes": size, "flops": 16 * sum(lengths) * H * D * Dv}
        pairs = H * sum(_visible_pairs(n, 0, case["window"], case["sinks"]) for n in lengths)
        # scores and output; scores again, go.v, dV, dK, dQ
        return {"bytes": size, "flops": 2 * pairs * (4 * D + 3 * Dv)}
    S, T = case["S"], case["T"]
    if kind == "decay_update":
        return {"bytes": S * (T * token + 2 * H * D * Dv * 4), "flops": 4 * S * T * H * D * Dv}
    past, window, sinks = case["past"], case["window"], case["sinks"]
    past = round(past * 0.625) if S > 1 else past    # on average
    rows = min(past, window - 1 + sinks)             # of the cache that the new tokens see
    pairs = _visible_pairs(T, past, window, sinks)
    return {"bytes": S * (T * token + Hkv * (rows + T) * (D + Dv) * item),
            "flops": 2 * S * H * pairs * (D + Dv)}


# ---------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------

def _group_sum(tensor, shared):
    return tensor.unflatten(-2, (shared, -1)).sum(-2)


def _exact_decay(q, k, v, rate, before):
    """The recurrence over tokens: outputs ``[B, T, H, Dv]`` and the last state."""
    state = before
    outputs = torch.empty(*q.shape[:3], v.shape[-1], dtype=q.dtype, device=DEVICE)
    for t in range(q.shape[1]):
        state = rate * state + k[:, t, :, :, None] * v[:, t, :, None, :]
        outputs[:, t] = torch.matmul(q[:, t, :, None, :], state).squeeze(-2)
    return outputs, state


def _exact_decay_train(case, state):
    H, Hkv, scale = case["H"], case["Hkv"], case["D"] ** -0.5
    leaves = [leaf.detach().double().repeat_interleave(H // leaf.shape[-2], dim=-2)
              for leaf in (*state["leaves"], state["grad_output"])]
    rate = torch.exp(state["log_decay"].double()).view(H, 1, 1)
    batches = [leaves]
    if case["lengths"]:
        ends = [0]
        for length in _lengths(case):
            ends.append(ends[-1] + length)
        batches = [[leaf[a:b].unsqueeze(0) for leaf in leaves] for a, b in zip(ends, ends[1:])]
    parts = []
    for q, k, v, go in batches:
        zero = torch.zeros(q.shape[0], H, case["D"], case["Dv"], dtype=q.dtype, device=DEVICE)
        output, _ = _exact_decay(q, k, v, rate, zero)
        # the state's row t, applied to the output's gradient, is the query's gradient
        grad_query, _ = _exact_decay(go, v, k, rate, zero.transpose(-1, -2))
        back = [tensor.flip(1) for tensor in (q, k, v, go)]
        grad_value, _ = _exact_decay(back[1], back[0], back[3], rate, zero)
        grad_key, _ = _exact_decay(back[2], back[3], back[0], rate, zero.transpose(-1, -2))
        parts.append([scale * output, scale * grad_query, scale * _group_sum(grad_key.flip(1), Hkv),
                      scale * _group_sum(grad_value.flip(1), Hkv)])
    if case["lengths"]:
        return [torch.cat([part[i][0] for part in parts]) for i in range(4)]
    return parts[0]


def _group_sum_heads(tensor, shared):
    return tensor.unflatten(0, (shared, -1)).sum(1)


def _exact_window_sequence(case, q, k, v, go):
    """One sequence: head by head over the whole square of scores."""
    H, Hkv, scale = case["H"], case["Hkv"], case["D"] ** -0.5
    t = torch.arange(q.shape[0], device=DEVICE)
    hidden = (t[None, :] > t[:, None]) | ((t[:, None] - t[None, :] >= case["window"])
                                          & (t[None, :] >= case["sinks"]))
    results = []
    for h in range(H):
        g = h // (H // Hkv)
        weights = torch.softmax((q[:, h] @ k[:, g].T * scale).masked_fill(hidden, -torch.inf), -1)
        output = weights @ v[:, g]
        slope = weights * (go[:, h] @ v[:, g].T - (go[:, h] * output).sum(-1, keepdim=True)) * scale
        results.append((output, slope @ k[:, g], slope.T @ q[:, h], weights.T @ go[:, h]))
    stacked = [torch.stack(parts) for parts in zip(*results)]
    stacked[2:] = [_group_sum_heads(part, Hkv) for part in stacked[2:]]
    return [part.transpose(0, 1) for part in stacked]


def _exact_window_update(case, state):
    H, Hkv, T, scale = case["H"], case["Hkv"], case["T"], case["D"] ** -0.5
    window, sinks = case["window"], case["sinks"]
    query, key, value = (tensor.double() for tensor in state["inputs"])
    caches = [cache.double() for cache in state["caches"]]
    ring = caches[0].shape[2] - sinks
    row = lambda p: torch.where(p < sinks, p, sinks + (p - sinks) % ring)
    outputs = torch.empty(*query.shape[:3], case["Dv"], dtype=torch.float64, device=DEVICE)
    for s, past in enumerate(state["lengths"].tolist()):
        # the history that new tokens can see: the sinks and the window of the first of them
        first = max(0, past - window + 1)
        seen = torch.cat([torch.arange(min(sinks, first)), torch.arange(first, past)]).to(DEVICE)
        fresh = torch.arange(past, past + T, device=DEVICE)
        position = torch.cat([seen, fresh])
        keys, values = (torch.cat([cache[s][:, row(seen)], new[s].transpose(0, 1)], dim=1)
                        for cache, new in zip(caches, (key, value)))
        hidden = (position > fresh[:, None]) | ((fresh[:, None] - position >= window)
                                                & (position >= sinks))
        for h in range(H):
            scores = query[s, :, h] @ keys[h // (H // Hkv)].T * scale
            outputs[s, :, h] = torch.softmax(scores.masked_fill(hidden, -torch.inf), -1) \
                @ values[h // (H // Hkv)]
        kept = fresh[(fresh < sinks) | (fresh >= past + T - ring)]
        for cache, new in zip(caches, (key, value)):
            cache[s][:, row(kept)] = new[s][kept - past].transpose(0, 1)
    return [outputs, *caches]


def exact(case, seed):
    state = prepare(case, seed)
    if case["kind"] == "decay_train":
        return _exact_decay_train(case, state)
    if case["kind"] == "decay_update":
        q, k, v = (tensor.double().repeat_interleave(case["H"] // tensor.shape[-2], dim=-2)
                   for tensor in state["inputs"])
        rate = torch.exp(state["log_decay"].double()).view(case["H"], 1, 1)
        output, last = _exact_decay(q, k, v, rate, state["state"].double())
        return [output * case["D"] ** -0.5, last]
    if case["kind"] == "window_update":
        return _exact_window_update(case, state)
    leaves = [leaf.detach().double() for leaf in (*state["leaves"], state["grad_output"])]
    if case["lengths"]:
        ends = [0]
        for length in _lengths(case):
            ends.append(ends[-1] + length)
        parts = [_exact_window_sequence(case, *(leaf[a:b] for leaf in leaves))
                 for a, b in zip(ends, ends[1:])]
        return [torch.cat([part[i] for part in parts]) for i in range(4)]
    parts = [_exact_window_sequence(case, *(leaf[b] for leaf in leaves)) for b in range(case["B"])]
    return [torch.stack([part[i] for part in parts]) for i in range(4)]
