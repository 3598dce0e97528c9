"""Timed calls of the paged cache: tables of pages built from request lengths, attention of new
tokens over the pages, and attention over the pages that a score selects for each token.

``listed()`` names the fixed cases, ``draw(rng)`` gives one more of the same ranges,
``prepare(case, seed)`` makes what a server holds before the call, ``run(state)`` is one pass,
``work(case)`` counts what a pass cannot do without and ``exact(case, seed)`` is the answer in
64 bits.  With ``own`` false a pass is the operator's formula in elementary tensor operations,
with ``own`` true the calls of the framework.

The kinds of a case:

* ``tables``: requests give pages back and take others for their new tokens;
* ``paged``: ``T`` new tokens for each of ``S`` slots, or ``lengths`` of them packed, over all that
  the slots hold;
* ``selected``: the same over the pages with the ``count`` largest scores and the token's own.
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

def _tables(name, S, page, past, T=0, lengths="", ended=0):
    """``past``: the most tokens that a slot holds; the first ``ended`` slots begin anew."""
    case = dict(kind="tables", S=S, page=page, past=past, T=T, lengths=lengths, ended=ended)
    return dict(case, name=name) if name else case


def _attention(kind, name, dtype, page, past, H, Hkv, D, Dv, S=0, T=0, lengths="", count=0):
    """``past``: the most tokens that a slot already holds; the slots' own numbers are drawn."""
    case = dict(kind=kind, dtype=dtype, S=S, T=T, lengths=lengths, page=page, past=past, H=H,
                Hkv=Hkv, D=D, Dv=Dv)
    if kind == "selected":
        case["count"] = count
    return dict(case, name=name) if name else case


def listed():
    return [
        # a step of 64 requests: eight drafted tokens were rejected, eight others take their place
        _tables("tables_draft", S=64, page=16, past=9000, T=8),
        # a busy server: a quarter of 256 requests ended, prompts of other ones take their slots
        _tables("tables_admit", S=256, page=64, past=4096, ended=64,
                lengths=",".join(["1024"] * 32 + ["37"] * 31 + ["3001"] + ["1"] * 192)),
        # one slot, one token, a small model: nothing but latency
        _attention("paged", "paged_token_one", "float32", S=1, T=1, page=16, past=512, H=16,
                   Hkv=16, D=64, Dv=64),
        # one more token for each of 64 slots of various lengths
        _attention("paged", "paged_token", "bfloat16", S=64, T=1, page=64, past=9000, H=32, Hkv=8,
                   D=128, Dv=128),
        # two slots with very long contexts: their caches are all there is to share out
        _attention("paged", "paged_token_long", "float16", S=2, T=1, page=64, past=200000, H=16,
                   Hkv=2, D=64, Dv=64),
        # drafted tokens that one pass checks
        _attention("paged", "paged_draft", "bfloat16", S=16, T=5, page=16, past=4096, H=32, Hkv=8,
                   D=128, Dv=128),
        # the second part of long prompts, behind what the caches already hold; the largest call
        _attention("paged", "paged_prompt", "bfloat16", S=4, T=2048, page=64, past=2500, H=32,
                   Hkv=8, D=128, Dv=128),
        # one step of everything at once: single tokens, drafts and prompts, odd widths
        _attention("paged", "paged_ragged", "float16", page=32, past=3001, H=12, Hkv=4, D=80,
                   Dv=80, lengths="1,37,1,513,4,1000,1,1,2047,129"),
        # one slot of a small model, a quarter of its pages selected
        _attention("selected", "selected_one", "float32", S=1, T=1, page=16, past=1000, H=8, Hkv=2,
                   D=64, Dv=64, count=16),
        # one more token for each of 32 slots with long contexts
        _attention("selected", "selected_token", "bfloat16", S=32, T=1, page=64, past=16384, H=32,
                   Hkv=8, D=128, Dv=128, count=32),
        # two slots with very long contexts
        _attention("selected", "selected_token_long", "float16", S=2, T=1, page=64, past=200000,
                   H=16, Hkv=2, D=64, Dv=64, count=64),
        # questions to long documents, packed
        _attention("selected", "selected_ragged", "bfloat16", page=32, past=6000, H=16, Hkv=4,
                   D=96, Dv=80, lengths="1,37,1,129,4,1", count=24),
    ]


def _spread(rng, low, high):
    """An integer between the bounds, even over the logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


MOST_SCORES = 5.0e8    # heads x (query, key) pairs of a drawn one, visible or not
MOST_BYTES = 6.0e8     # of a drawn cache
MOST_GATHERED = 8.0e9  # bytes of the selected pages of all new tokens, in float32


def draw(rng):
    kind = rng.choice(["tables", "paged", "paged", "selected", "selected"])
    page = rng.choice([16, 16, 32, 64, 64, 128, 256])
    past = rng.choice([0, _spread(rng, 1, 20000), _spread(rng, 1, 20000), _spread(rng, 1000, 200000)])
    if kind == "tables":
        slots = _spread(rng, 1, 512)
        past = min(past, 20000)
        ended = rng.choice([0, rng.randint(0, slots)])
        if rng.random() < 0.5:
            return _tables("", S=slots, page=page, past=past, T=_spread(rng, 1, 200), ended=ended)
        most = _spread(rng, 1, 1000)
        parts = [rng.choice([0, 1, _spread(rng, 1, most)]) for _ in range(slots - 1)] + [most]
        return _tables("", S=slots, page=page, past=past, ended=ended,
                       lengths=",".join(map(str, parts)))
    dtype = rng.choice(["float32", "float16", "bfloat16"])
    kv_heads = _spread(rng, 1, 16)
    heads = kv_heads * rng.choice([1, 2, 4, 4, 8])
    width = rng.choice([16, 32, 40, 64, 64, 72, 80, 96, 128, 128])
    value_width = width if rng.random() < 0.7 else rng.choice([24, 32, 33, 64, 100, 128])
    shape = dict(page=page, H=heads, Hkv=kv_heads, D=width, Dv=value_width)
    if kind == "selected":
        shape["count"] = _spread(rng, 1, 64)
    # how long the slots' contexts may be, and then how many of them
    one = kv_heads * (width + value_width) * ITEM_BYTES[dtype]
    past = min(past, int(MOST_BYTES / one))
    # the plain form gathers the selected pages of every new token
    gathered = (shape["count"] + 1) * page * one * 4 // ITEM_BYTES[dtype] if kind == "selected" else 1
    if rng.random() < 0.5:
        tokens = rng.choice([1, 1, 1, rng.randint(2, 8)])
        slots = _spread(rng, 1, max(1, min(128, int(MOST_BYTES / (one * (past + 1))),
                                           int(MOST_GATHERED / (gathered * tokens)))))
        return _attention(kind, "", dtype, S=slots, T=tokens, past=past, **shape)
    # and scores every new token against all that the longest slot holds
    most = 300 if kind == "selected" else 4000
    past = min(past, 20000)
    tokens = _spread(rng, 2, most)
    tokens = max(2, min(tokens, int(MOST_SCORES / (heads * (past + tokens)))))
    slots = max(1, min(8, int(MOST_SCORES / (heads * tokens * (past + tokens))),
                       int(MOST_BYTES / (one * (past + tokens)))))
    tokens = max(2, min(tokens, int(MOST_GATHERED / gathered)))
    slots = max(1, min(slots, int(MOST_GATHERED / (gathered * tokens))))
    slots = rng.randint(1, slots)
    if rng.random() < 0.5:
        return _attention(kind, "", dtype, S=slots, T=tokens, past=past, **shape)
    parts = [rng.choice([0, 1, _spread(rng, 1, tokens)]) for _ in range(slots - 1)] + [tokens]
    return _attention(kind, "", dtype, past=past, lengths=",".join(map(str, parts)), **shape)


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _chunk(case):
    """The new tokens of every slot."""
    if case["lengths"]:
        return [int(item) for item in case["lengths"].split(",")]
    return [case["T"]] * case["S"]


def _held(case, generator):
    """What the slots hold: a number of their own between a quarter of the most and the most."""
    slots = len(_chunk(case))
    past = torch.rand(slots, device=DEVICE, generator=generator).mul(0.75).add(0.25)
    past = past.mul(case["past"]).round().to(torch.int32)
    past[-1:] = case["past"]
    return past


def _ceil(a, b):
    return -(-a // b)


def prepare(case, seed):
    generator = torch.Generator(device=DEVICE).manual_seed(int(seed))
    chunk, page = _chunk(case), case["page"]
    most = case["past"] + max(chunk)
    slots, columns = len(chunk), _ceil(most, page) + 3
    past = _held(case, generator)
    if case["kind"] == "tables":
        past[:case["ended"]] = 0
    new = torch.tensor(chunk, dtype=torch.int32, device=DEVICE)
    # a pool with a tenth more pages than the requests need, handed out in any order
    pages = slots * (_ceil(case["past"], page) + 1) + sum(_ceil(n, page) + 1 for n in chunk)
    pages += pages // 10
    order = torch.randperm(pages, device=DEVICE, generator=generator)
    pool = torch.cat([torch.full_like(order[:1], pages), order]).to(torch.int32)
    tables = torch.full((slots, columns), -1, dtype=torch.int32, device=DEVICE)
    state = dict(kind=case["kind"], page=page, tables=tables, pool=pool, lengths=past,
                 tokens=sum(chunk) if case["lengths"] else case["T"], offsets=None)
    if case["lengths"]:
        state["offsets"] = torch.cat([new[:1] * 0, new.cumsum(0)]).to(torch.int32)
    # the tables as earlier steps have left them, and the pages of this one's tokens
    _plain_update(tables, past * 0, pool, past, page)
    _plain_update(tables, past, pool, new, page)
    if case["kind"] == "tables":
        # the step is done over: its pages go back and come again
        state["after"] = past + new
        return state
    state["rows"] = _plain_rows(tables, past, state["offsets"], state["tokens"], page, pages)
    state["most"], state["longest"] = most, max(chunk)
    dtype = getattr(torch, case["dtype"])
    H, Hkv, D, Dv = (case[name] for name in ("H", "Hkv", "D", "Dv"))
    randn = lambda *dims: torch.randn(*dims, device=DEVICE, generator=generator)
    lead = (sum(chunk),) if case["lengths"] else (slots, case["T"])
    state["inputs"] = [randn(*lead, H, D).to(dtype), randn(*lead, Hkv, D).to(dtype),
                       randn(*lead, Hkv, Dv).to(dtype)]
    # the keys of neighbouring tokens are alike: a page has a direction of its own
    keys = (randn(pages, Hkv, page, D) + 0.7 * randn(pages, Hkv, 1, D)).to(dtype)
    state["pages"] = [keys, randn(pages, Hkv, page, Dv).to(dtype)]
    if case["kind"] == "selected":
        state["count"] = case["count"]
        bounds = torch.full((pages, Hkv, 2, D), torch.inf, device=DEVICE, dtype=dtype)
        bounds[:, :, 1] = -torch.inf
        spans = torch.arange(columns, device=DEVICE) * page
        slot, column = torch.nonzero(spans < past[:, None], as_tuple=True)
        held = (past.long()[slot] - column * page).clamp(max=page)
        hidden = torch.arange(page, device=DEVICE) >= held[:, None]
        at = tables[slot, column].long()
        mine = keys[at].float()
        hidden = hidden[:, None, :, None]
        bounds[at, :, 0] = mine.masked_fill(hidden, torch.inf).amin(2).to(dtype)
        bounds[at, :, 1] = mine.masked_fill(hidden, -torch.inf).amax(2).to(dtype)
        state["bounds"] = bounds
    return state


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------

def _plain_update(tables, lengths, pool, new, page):
    """Pages for ``new`` more tokens of every slot, from the top of the pool's stack."""
    columns, free = tables.shape[1], pool[0].long()
    have = _ceil(lengths.long().clamp(min=0), page).clamp(max=columns)
    need = _ceil(lengths.long().clamp(min=0) + new.long(), page).clamp(max=columns)
    column = torch.arange(columns, device=DEVICE)
    fresh = (column >= have[:, None]) & (column < need[:, None])
    taken = (need - have).cumsum(0) - (need - have)
    number = taken[:, None] + column - have[:, None]
    entry = torch.where(number < free, pool[(free - number).clamp(min=0)], -1)
    tables.copy_(torch.where(fresh, entry.to(torch.int32), tables))
    pool[0] = (free - (need - have).sum()).clamp(min=0)


def _plain_release(tables, lengths, keep, pool, page):
    """The pages behind the first ``keep`` tokens go back, the first of them on top."""
    pages, columns, free = pool.shape[0] - 1, tables.shape[1], pool[0].long()
    have = _ceil(lengths.long().clamp(min=0), page).clamp(max=columns)
    kept = torch.minimum(_ceil(keep.long().clamp(min=0), page), have)
    column = torch.arange(columns, device=DEVICE)
    gone = (column >= kept[:, None]) & (column < have[:, None])
    back = (gone & (tables >= 0) & (tables < pages)).flatten()
    number = back.long().cumsum(0) - 1
    place = free + back.sum() - number
    # (an element behind the pool takes what has no place in it)
    place = torch.where(back & (place <= pages), place, pages + 1)
    wider = torch.cat([pool, pool[:1]]).index_copy_(0, place, tables.flatten())
    pool.copy_(wider[:-1])
    pool[0] = (free + back.sum()).clamp(max=pages)
    tables.masked_fill_(gone, -1)


def _positions(lengths, offsets, tokens):
    """The slot and the position of every new token, packed or ``(slots, T)``."""
    past = lengths.long().clamp(min=0)
    if offsets is None:
        index = torch.arange(tokens, device=DEVICE).expand(past.shape[0], tokens)
        return torch.arange(past.shape[0], device=DEVICE)[:, None].expand_as(index), past[:, None] + index
    index = torch.arange(tokens, device=DEVICE)
    slot = torch.searchsorted(offsets[1:].long(), index, right=True)
    return slot, past[slot] + index - offsets.long()[slot]


def _plain_rows(tables, lengths, offsets, tokens, page, pages):
    slot, position = _positions(lengths, offsets, tokens)
    column = position // page
    entry = tables[slot, column.clamp(max=tables.shape[1] - 1)].long()
    there = (column < tables.shape[1]) & (entry >= 0) & (entry < pages)
    return torch.where(there, entry * page + position % page, -1)


def _new_of(state):
    if state["offsets"] is None:
        return torch.full_like(state["lengths"], state["tokens"])
    return state["offsets"].diff()


def _plain_tables(state):
    tables, pool, lengths, page = (state[n] for n in ("tables", "pool", "lengths", "page"))
    _plain_release(tables, state["after"], lengths, pool, page)
    _plain_update(tables, lengths, pool, _new_of(state), page)
    rows = _plain_rows(tables, lengths, state["offsets"], state["tokens"], page, pool.shape[0] - 1)
    return [rows, tables, pool]


def _put(state):
    """The new tokens on their rows."""
    page, rows = state["page"], state["rows"].flatten()
    for_rows = lambda tensor: tensor.reshape(rows.shape[0], *tensor.shape[-2:])
    keys, values = state["pages"]
    keys[rows // page, :, rows % page] = for_rows(state["inputs"][1])
    values[rows // page, :, rows % page] = for_rows(state["inputs"][2])


def _padded(state, tensor):
    """``[slots, heads, tokens, width]`` in float32, and where the real tokens lie in it."""
    if state["offsets"] is None:
        return tensor.transpose(1, 2).float(), None
    slot, position = _positions(state["lengths"] * 0, state["offsets"], state["tokens"])
    out = torch.zeros(state["lengths"].shape[0], state["longest"], *tensor.shape[1:], device=DEVICE)
    out[slot, position] = tensor.float()
    return out.transpose(1, 2), (slot, position)


def _tokens_first(state, tensor, places, dtype):
    tensor = tensor.transpose(1, 2)
    return (tensor if places is None else tensor[places]).to(dtype).contiguous()


def _softmax(scores, visible):
    scores = torch.where(visible, scores, -torch.inf)
    weights = torch.exp(scores - scores.amax(-1, keepdim=True))
    return weights / weights.sum(-1, keepdim=True)


def _plain_paged(state):
    query, (keys, values) = state["inputs"][0], state["pages"]
    Hkv, page, scale = keys.shape[1], state["page"], query.shape[-1] ** -0.5
    _put(state)
    table = state["tables"][:, :_ceil(state["most"], page)].long().clamp(min=0)
    in_order = lambda pool: pool[table].float().transpose(1, 2).flatten(2, 3)
    q, places = _padded(state, query)
    S, H, T, D = q.shape
    t = state["lengths"].view(-1, 1, 1) + torch.arange(T, device=DEVICE).view(1, -1, 1)
    visible = torch.arange(table.shape[1] * page, device=DEVICE) <= t
    scores = torch.matmul(q.reshape(S, Hkv, -1, D), in_order(keys).transpose(-1, -2).contiguous())
    scores = scores.view(S, Hkv, H // Hkv, T, -1) * scale
    weights = _softmax(scores, visible[:, None, None]).view(S, Hkv, H // Hkv * T, -1)
    output = torch.matmul(weights, in_order(values)).view(S, H, T, -1)
    return [_tokens_first(state, output, places, query.dtype), keys, values]


def _plain_bounds(state):
    """The bounds of the pages that the new tokens lie on."""
    page, (keys, _), bounds = state["page"], state["pages"], state["bounds"]
    slot, position = _positions(state["lengths"], state["offsets"], state["tokens"])
    at = state["rows"].flatten() // page
    # a page holds its first tokens up to the slot's last one
    last = (state["lengths"] + _new_of(state)).long()[slot.flatten()] - 1
    held = last - position.flatten() // page * page
    hidden = (torch.arange(page, device=DEVICE) > held[:, None])[:, None, :, None]
    mine = keys[at]
    bounds[at, :, 0] = mine.masked_fill(hidden, torch.inf).amin(2)
    bounds[at, :, 1] = mine.masked_fill(hidden, -torch.inf).amax(2)


def _plain_selected(state):
    query, (keys, values), count = state["inputs"][0], state["pages"], state["count"]
    Hkv, page, scale = keys.shape[1], state["page"], query.shape[-1] ** -0.5
    _put(state)
    _plain_bounds(state)
    table = state["tables"][:, :_ceil(state["most"], page)].long().clamp(min=0)
    q, places = _padded(state, query)
    S, H, T, D = q.shape
    position = state["lengths"].view(-1, 1).long() + torch.arange(T, device=DEVICE)
    # the largest product that a key within a page's bounds can have, in 64 bits: ranks are compared
    low, high = (state["bounds"][table, :, i].permute(0, 2, 3, 1).double().contiguous() for i in (0, 1))
    wide = q.double().reshape(S, Hkv, -1, D)
    scores = torch.matmul(wide.clamp(min=0), high) + torch.matmul(wide.clamp(max=0), low)
    scores = scores.view(S, Hkv, H // Hkv, T, -1).amax(2)
    own_page = (position // page).clamp(max=table.shape[1] - 1).view(S, 1, T, 1)
    earlier = torch.arange(table.shape[1], device=DEVICE) < own_page
    scores = torch.where(earlier, scores, -torch.inf)
    best = scores.sort(dim=-1, descending=True, stable=True).indices[..., :count]
    chosen = torch.cat([best, own_page.expand(S, Hkv, T, 1)], dim=-1)
    ranked = torch.arange(chosen.shape[-1] - 1, device=DEVICE) < own_page
    there = torch.cat([ranked, torch.ones_like(ranked[..., :1])], dim=-1).expand_as(chosen)
    at = table.view(S, 1, 1, -1).expand(S, Hkv, T, -1).gather(-1, chosen)
    head = torch.arange(Hkv, device=DEVICE).view(1, -1, 1, 1)
    spans = chosen[..., None] * page + torch.arange(page, device=DEVICE)
    visible = there[..., None] & (spans <= position.view(S, 1, T, 1, 1))
    # [slots, kv heads, tokens, members of the group, keys]
    q = q.view(S, Hkv, H // Hkv, T, D).transpose(2, 3)
    weights = torch.matmul(q, keys[at, head].float().flatten(3, 4).transpose(-1, -2).contiguous()) * scale
    weights = _softmax(weights, visible.flatten(3)[..., None, :])
    output = torch.matmul(weights, values[at, head].float().flatten(3, 4))
    output = output.transpose(2, 3).reshape(S, H, T, -1)
    return [_tokens_first(state, output, places, query.dtype), keys, values, state["bounds"]]


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def _own(state):
    from rosa_soft_amd import paged

    tables, lengths, offsets = state["tables"], state["lengths"], state["offsets"]
    if state["kind"] == "tables":
        paged.page_tables_release(tables, state["after"], lengths, state["pool"], page=state["page"])
        rows = paged.page_tables_update(tables, lengths, state["pool"], offsets,
                                        tokens=state["tokens"], page=state["page"])
        return [rows, tables, state["pool"]]
    if state["kind"] == "paged":
        output = paged.paged_attention_update(*state["inputs"], *state["pages"], tables,
                                              state["rows"], lengths, offsets)
        return [output, *state["pages"]]
    output = paged.selected_attention_update(*state["inputs"], *state["pages"], state["bounds"],
                                             tables, state["rows"], lengths, offsets,
                                             count=state["count"])
    return [output, *state["pages"], state["bounds"]]


def run(state):
    if own:
        return _own(state)
    plain = {"tables": _plain_tables, "paged": _plain_paged, "selected": _plain_selected}
    return plain[state["kind"]](state)


# ---------------------------------------------------------------------------
# what a pass needs
# ---------------------------------------------------------------------------

def work(case):
    chunk, page = _chunk(case), case["page"]
    slots, tokens = len(chunk), sum(chunk)
    if case["kind"] == "tables":
        # lengths twice and chunks, the entries that come and go and their pages, the rows
        changed = sum(_ceil(n, page) for n in chunk)
        return {"bytes": 12 * slots + 16 * changed + 8 * tokens, "flops": tokens + changed}
    item, H, Hkv, D, Dv = ITEM_BYTES[case["dtype"]], *(case[n] for n in ("H", "Hkv", "D", "Dv"))
    size = tokens * ((H + Hkv) * (D + Dv) * item + 8)
    pairs = products = 0
    for i, new in enumerate(chunk):
        past = case["past"] if i == slots - 1 else round(0.625 * case["past"])  # on average
        if new == 0:
            continue
        if case["kind"] == "paged":
            size += past * Hkv * (D + Dv) * item
            pairs += new * past + new * (new + 1) // 2
            continue
        kept = min(past, (case["count"] + 0.5) * page)      # of a token
        size += min(past, kept * new) * Hkv * (D + Dv) * item + past / page * Hkv * 2 * D * item
        pairs += new * kept
        products += new * past / page
    return {"bytes": int(size), "flops": int(2 * H * (pairs * (D + Dv) + products * D))}


# ---------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------

def _seen_pages(case, q, low, high, own_page):
    """Whether each of the pages is seen by a token whose group of query rows is ``q``."""
    seen = torch.zeros(own_page + 1, dtype=torch.bool, device=DEVICE)
    seen[own_page] = True
    if own_page > 0:
        at_most = torch.maximum(q[:, None] * low[None, :own_page], q[:, None] * high[None, :own_page])
        rank = torch.argsort(at_most.sum(-1).amax(0), descending=True, stable=True)
        seen[rank[:case["count"]]] = True
    return seen


def exact(case, seed):
    if case["kind"] == "tables":
        return None  # whole numbers
    state = prepare(case, seed)
    page, chunk = case["page"], _chunk(case)
    if case["kind"] == "selected" and sum(chunk) * case["Hkv"] > 4000:
        return None
    H, Hkv, scale = case["H"], case["Hkv"], case["D"] ** -0.5
    flat = lambda tensor: tensor.reshape(-1, *tensor.shape[-2:])
    query, key, value = (flat(tensor).double() for tensor in state["inputs"])
    keys, values = (pool.clone() for pool in state["pages"])
    row = state["rows"].flatten()
    for pool, fresh in ((keys, state["inputs"][1]), (values, state["inputs"][2])):
        pool[row // page, :, row % page] = flat(fresh)
    output = torch.empty(sum(chunk), H, case["Dv"], dtype=torch.float64, device=DEVICE)
    first = 0
    for slot, (new, past) in enumerate(zip(chunk, state["lengths"].tolist())):
        table = state["tables"][slot, :_ceil(past + new, page)].long()
        for g in range(Hkv if new else 0):
            k, v = (pool[table, g].flatten(0, 1)[:past + new].double() for pool in (keys, values))
            t = torch.arange(past, past + new, device=DEVICE)
            s = torch.arange(past + new, device=DEVICE)
            members = range(g * (H // Hkv), (g + 1) * (H // Hkv))
            hidden = s > t[:, None]
            if case["kind"] == "selected":
                pieces = k.split(page)
                low = torch.stack([piece.amin(0) for piece in pieces])
                high = torch.stack([piece.amax(0) for piece in pieces])
                for i, at in enumerate(range(past, past + new)):
                    seen = _seen_pages(case, query[first + i, members.start:members.stop], low, high,
                                       at // page)
                    hidden[i, :at // page * page] |= ~seen[:-1].repeat_interleave(page)
            for h in members:
                scores = query[first:first + new, h] @ k.T * scale
                weights = torch.softmax(scores.masked_fill(hidden, -torch.inf), -1)
                output[first:first + new, h] = weights @ v
        first += new
    if not case["lengths"]:
        output = output.view(case["S"], case["T"], H, case["Dv"])
    return [output] + [None] * (3 if case["kind"] == "selected" else 2)
