"""Decayed linear attention and window attention against their definitions in 64 bits.

Tolerances: u is half a step of the type (2^-24, 2^-11, 2^-8).  What is rounded to the type on the
way is each term of a sum (the weights, the scores, the state, the weighted values), once, and the
result, once; ``bound`` is the sum of the absolute terms, so k roundings are k u bound.  What
stays in float32 adds its own sums (``float32_slack``).
"""

import itertools
import math

import pytest
import torch

import rosa_soft_amd
from rosa_soft_amd import mixers
from tests import mixer_reference as reference
from tests.mixer_reference import HALF_STEP, float32_slack

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
DEVICE = "cuda:0"


def randn(seed, *shape, dtype=torch.float32, scale=1.0):
    generator = torch.Generator(device=DEVICE).manual_seed(seed)
    return (torch.randn(*shape, device=DEVICE, generator=generator) * scale).to(dtype)


def rates(heads, low=0.003, high=0.4):
    return -torch.logspace(math.log10(low), math.log10(high), heads, device=DEVICE)


def offsets_of(lengths):
    return torch.tensor([0, *itertools.accumulate(lengths)], dtype=torch.int32, device=DEVICE)


def pieces(tensor, lengths):
    """The sequences of a dense or packed tensor."""
    return list(tensor) if lengths is None else list(tensor.split(lengths))


def whole(parts, lengths):
    return torch.stack(parts) if lengths is None else torch.cat(parts)


def close(got, want, tolerance, what=""):
    assert got.shape == want.shape, (what, got.shape, want.shape)
    off = (got.double() - want).abs()
    over = off > tolerance
    assert bool(torch.isfinite(got).all()) and not bool(over.any()), (
        what, float((off / tolerance.clamp(min=1e-300)).max()), int(over.sum()), got.numel())


SHAPES = [
    # dense (B, T) or packed lengths, H, Hkv, D, Dv
    ((1, 1), None, 1, 1, 1, 1),
    ((2, 63), None, 2, 1, 32, 32),
    ((1, 64), None, 4, 4, 64, 64),
    ((3, 65), None, 6, 2, 128, 128),
    ((2, 300), None, 2, 2, 80, 40),
    ((1, 700), None, 2, 1, 33, 100),
    ((1, 129), None, 3, 1, 7, 128),
    (None, [1, 0, 37, 129, 64, 200], 4, 2, 64, 64),
    (None, [5], 1, 1, 128, 32),
    (None, [0, 0, 300, 0], 2, 2, 48, 80),
    (None, [513, 1, 700], 4, 1, 128, 128),
]


def inputs_of(shape, dtype, seed=0):
    dense, lengths, H, Hkv, D, Dv = shape
    lead = dense if dense is not None else (sum(lengths),)
    tensors = [randn(seed, *lead, H, D, dtype=dtype), randn(seed + 1, *lead, Hkv, D, dtype=dtype),
               randn(seed + 2, *lead, Hkv, Dv, dtype=dtype)]
    return tensors, randn(seed + 3, *lead, H, Dv, dtype=dtype)


def decay_tolerance(dtype, bound, tokens, width):
    # the score or state, the weighted value, and the result
    return (4 * HALF_STEP[dtype] + float32_slack(tokens, width)) * bound + 1e-37


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_decay_attention_and_its_gradients(shape, dtype):
    dense, lengths, H, Hkv, D, Dv = shape
    tensors, grad_output = inputs_of(shape, dtype)
    log_decay = rates(H)
    leaves = [t.requires_grad_() for t in tensors]
    if lengths is None:
        output = mixers.decay_attention(*leaves, log_decay)
    else:
        output = mixers.decay_attention_varlen(*leaves, offsets_of(lengths), log_decay)
    gradients = torch.autograd.grad(output, leaves, grad_output)
    assert output.dtype == dtype and all(g.dtype == dtype for g in gradients)
    results = [[], [], [], []]
    for q, k, v, go in zip(*(pieces(t.detach(), lengths) for t in (*leaves, grad_output))):
        for absolute in (False, True):
            out = reference.decay(q, k, v, log_decay, absolute=absolute)[0]
            grads = reference.decay(q, k, v, log_decay, grad_output=go, absolute=absolute)
            for place, tensor in zip(results, (out, *grads)):
                place.append(tensor)
    tokens = dense[1] if dense else max(lengths)
    for name, got, parts in zip(("output", "dq", "dk", "dv"), (output, *gradients), results):
        want, bound = (whole(parts[i::2], lengths) for i in (0, 1))
        close(got.detach(), want, decay_tolerance(dtype, bound, tokens * H // Hkv, D + Dv), name)


WINDOWS = [(1, 0), (7, 3), (64, 0), (100, 4), (257, 64), (2**40, 2)]


def window_tolerances(dtype, bounds, most, tokens, width):
    # weights (or slopes) and the result; the slope takes the rounded output in as well
    relative = 4 * HALF_STEP[dtype] + float32_slack(tokens, width) * (1 + 2 * most)
    return [relative * bound + 1e-37 for bound in bounds]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape,masks", [
    (shape, WINDOWS[(i + shift) % len(WINDOWS)])
    for i, shape in enumerate(SHAPES) for shift in (0, 3)])
def test_window_attention_and_its_gradients(shape, masks, dtype):
    dense, lengths, H, Hkv, D, Dv = shape
    size, sinks = masks
    tensors, grad_output = inputs_of(shape, dtype, seed=10)
    leaves = [t.requires_grad_() for t in tensors]
    controls = dict(window=size, sinks=sinks)
    if lengths is None:
        output = mixers.window_attention(*leaves, **controls)
    else:
        output = mixers.window_attention_varlen(*leaves, offsets_of(lengths), **controls)
    gradients = torch.autograd.grad(output, leaves, grad_output)
    parts, most = [], 0.0
    for q, k, v, go in zip(*(pieces(t.detach(), lengths) for t in (*leaves, grad_output))):
        if len(q) == 0:
            parts.append([[x.double(), x.double()] for x in (go, q, k, v)])
            continue
        out, bound, here = reference.window(q, k, v, size, sinks)
        grads, bounds, _ = reference.window(q, k, v, size, sinks, grad_output=go)
        parts.append([[out, bound], *zip(grads, bounds)])
        most = max(most, here)
    tokens = dense[1] if dense else max(lengths)
    for i, (name, got) in enumerate(zip(("output", "dq", "dk", "dv"), (output, *gradients))):
        want, bound = (whole([part[i][j] for part in parts], lengths) for j in (0, 1))
        tolerance, = window_tolerances(dtype, [bound], most, tokens * H // Hkv, D + Dv)
        close(got.detach(), want, tolerance, name)


@pytest.mark.parametrize("dtype", DTYPES)
def test_sinks_of_long_sequences_collect_all_their_gradients(dtype):
    """The tokens beyond the sinks' window are walked in pieces of 1024: several of them, a last
    one of a few tokens, and sequences that begin inside a piece."""
    shape = (None, [900, 2501, 64], 4, 2, 32, 32)
    tensors, grad_output = inputs_of(shape, dtype, seed=20)
    leaves = [t.requires_grad_() for t in tensors]
    output = mixers.window_attention_varlen(*leaves, offsets_of(shape[1]), window=50, sinks=5)
    gradients = torch.autograd.grad(output, leaves, grad_output)
    parts = [reference.window(q, k, v, 50, 5, grad_output=go)
             for q, k, v, go in zip(*(t.detach().split(shape[1]) for t in (*leaves, grad_output)))]
    for i, got in enumerate(gradients):
        want, bound = (torch.cat([part[j][i] for part in parts]) for j in (0, 1))
        tolerance, = window_tolerances(dtype, [bound], max(p[2] for p in parts), 5002, 64)
        close(got, want, tolerance, i)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape,masks", [
    (((1, 1300), None, 8, 1, 32, 32), (2000, 0)),            # many parts, all causal
    ((None, [700, 3, 900], 6, 1, 64, 48), (300, 4)),         # and sinks, which the first part has
    (((1, 1600), None, 16, 1, 128, 128), (150, 0)),          # parts that end inside a head's walk
    ((None, [1100, 60], 9, 1, 20, 36), (1000, 2)),           # a last part without steps
])
def test_few_key_heads_share_out_their_walks(shape, masks, dtype):
    dense, lengths, H, Hkv, D, Dv = shape
    tensors, grad_output = inputs_of(shape, dtype, seed=25)
    leaves = [t.requires_grad_() for t in tensors]
    cu = offsets_of(lengths or [dense[1]])
    output = mixers.window_attention_varlen(*(t.view(-1, *t.shape[-2:]) for t in leaves), cu,
                                            window=masks[0], sinks=masks[1])
    gradients, again = (torch.autograd.grad(output, leaves, grad_output.view(output.shape),
                                            retain_graph=True) for _ in range(2))
    assert all(map(torch.equal, gradients, again))
    lengths = lengths or [dense[1]]
    parts = [reference.window(q, k, v, *masks, grad_output=go)
             for q, k, v, go in zip(*(t.detach().view(-1, *t.shape[-2:]).split(lengths)
                                      for t in (*leaves, grad_output)))]
    for i, got in enumerate(gradients):
        want, bound = (torch.cat([part[j][i] for part in parts]) for j in (0, 1))
        tolerance, = window_tolerances(dtype, [bound], max(p[2] for p in parts), max(lengths) * H, D + Dv)
        close(got.view(want.shape), want, tolerance, i)
    bad = cu.clone()
    bad[-1] += 1
    for gradient in torch.autograd.grad(
            mixers.window_attention_varlen(*(t.view(-1, *t.shape[-2:]) for t in leaves), bad,
                                           window=masks[0], sinks=masks[1]), leaves,
            grad_output.view(output.shape)):
        assert bool(torch.isnan(gradient).all())


# ---------------------------------------------------------------------------
# serving
# ---------------------------------------------------------------------------

CHUNKS = [[5, 1, 64, 1, 1, 130, 3], [1, 1, 1, 1], [300, 1, 1], [63, 65, 1]]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("chunks", CHUNKS)
@pytest.mark.parametrize("widths", [(4, 2, 64, 64), (2, 2, 128, 128), (3, 1, 24, 33), (2, 1, 40, 100)])
def test_decay_updates_continue_each_other(chunks, widths, dtype):
    H, Hkv, D, Dv = widths
    slots, total = 3, sum(chunks)
    tensors, _ = inputs_of(((slots, total), None, H, Hkv, D, Dv), dtype, seed=30)
    log_decay = rates(H)
    start = randn(35, slots, H, D, Dv, scale=4.0)
    state, outputs, at = start.clone(), [], 0
    for chunk in chunks:
        part = [t[:, at:at + chunk] for t in tensors]  # (strided)
        if at % 2:
            fresh = torch.full_like(state, math.nan)
            outputs.append(mixers.decay_attention_update(*part, log_decay, state, state_out=fresh))
            state = fresh
        else:
            outputs.append(mixers.decay_attention_update(*part, log_decay, state))
        at += chunk
    output = torch.cat(outputs, dim=1)
    for s in range(slots):
        rows = [t[s] for t in tensors]
        want, last = reference.decay(*rows, log_decay, state=start[s])
        bound, last_bound = reference.decay(*rows, log_decay, state=start[s], absolute=True)
        close(output[s], want, decay_tolerance(dtype, bound, total, D + Dv))
        # states are float32 sums of products that are split, not rounded: 2^-23 for the terms
        # that the split leaves out
        close(state[s], last, (float32_slack(total, D) + 2.0**-23) * last_bound + 1e-37)


def linear(cache, length, sinks):
    """The rows of a slot's cache by position, for the positions it still holds."""
    ring = cache.shape[1] - sinks
    position = torch.arange(length, device=cache.device)
    row = torch.where(position < sinks, position, sinks + (position - sinks) % ring)
    held = (position < sinks) | (position >= length - ring)
    return position[held], cache[:, row[held]]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("chunks", CHUNKS)
@pytest.mark.parametrize("masks", [(16, 4, 0), (70, 0, 0), (64, 3, 9), (1, 1, 0), (400, 64, 5)])
@pytest.mark.parametrize("widths", [(4, 2, 64, 64), (20, 1, 32, 100), (2, 2, 128, 128), (3, 1, 24, 33)])
def test_window_updates_continue_each_other(chunks, masks, widths, dtype):
    """Every chunk gives what one pass over the whole sequence gives, and the caches hold the newest
    tokens and the sinks.  What no token has been put on is NaN and stays unread."""
    H, Hkv, D, Dv = widths
    size, sinks, spare = masks
    slots, total = 2, sum(chunks)
    tensors, _ = inputs_of(((slots, total), None, H, Hkv, D, Dv), dtype, seed=40)
    caches = [torch.full((slots, Hkv, sinks + size + spare, width), math.nan, dtype=dtype,
                         device=DEVICE) for width in (D, Dv)]
    lengths, outputs, at = torch.zeros(slots, dtype=torch.int32, device=DEVICE), [], 0
    for chunk in chunks:
        part = [t[:, at:at + chunk] for t in tensors]
        outputs.append(mixers.window_attention_update(*part, *caches, lengths, window=size, sinks=sinks))
        lengths += chunk
        at += chunk
    output = torch.cat(outputs, dim=1)
    for s in range(slots):
        want, bound, most = reference.window(*(t[s] for t in tensors), size, sinks)
        tolerance, = window_tolerances(dtype, [bound], most, total, D + Dv)
        close(output[s], want, tolerance)
        for cache, tensor in zip(caches, tensors[1:]):
            position, rows = linear(cache[s], total, sinks)
            assert torch.equal(rows, tensor[s][position].transpose(0, 1))


@pytest.mark.parametrize("dtype", DTYPES)
def test_packed_updates_leave_slots_without_tokens_alone(dtype):
    H, Hkv, D, Dv, size, sinks = 4, 2, 64, 48, 20, 2
    chunks = [[3, 0, 100, 1], [0, 0, 1, 1], [70, 5, 0, 64], [1, 1, 1, 1]]
    log_decay = rates(H)
    slots = 4
    totals = [sum(c[s] for c in chunks) for s in range(slots)]
    streams = [inputs_of(((1, n), None, H, Hkv, D, Dv), dtype, seed=50 + s)[0]
               for s, n in enumerate(totals)]
    state = randn(60, slots, H, D, Dv)
    start = state.clone()
    caches = [torch.full((slots, Hkv, size + sinks, w), math.nan, dtype=dtype, device=DEVICE)
              for w in (D, Dv)]
    lengths = torch.zeros(slots, dtype=torch.int32, device=DEVICE)
    got = [[[], []] for _ in range(slots)]
    seen = [0] * slots
    for chunk in chunks:
        part = [torch.cat([streams[s][i][0, seen[s]:seen[s] + chunk[s]] for s in range(slots)])
                for i in range(3)]
        offsets = offsets_of(chunk)
        outs = (mixers.decay_attention_update(*part, log_decay, state, offsets),
                mixers.window_attention_update(*part, *caches, lengths, offsets, window=size,
                                               sinks=sinks))
        lengths += offsets.diff()
        for s in range(slots):
            for kind, out in enumerate(outs):
                got[s][kind].append(out.split(chunk)[s])
            seen[s] += chunk[s]
    for s in range(slots):
        rows = [t[0] for t in streams[s]]
        want, last = reference.decay(*rows, log_decay, state=start[s])
        bound, last_bound = reference.decay(*rows, log_decay, state=start[s], absolute=True)
        close(torch.cat(got[s][0]), want, decay_tolerance(dtype, bound, 200, D + Dv))
        close(state[s], last, (float32_slack(200, D) + 2.0**-23) * last_bound + 1e-37)
        if totals[s]:
            want, bound, most = reference.window(*rows, size, sinks)
            tolerance, = window_tolerances(dtype, [bound], most, 200, D + Dv)
            close(torch.cat(got[s][1]), want, tolerance)
            for cache, tensor in zip(caches, rows[1:]):
                position, held = linear(cache[s], totals[s], sinks)
                assert torch.equal(held, tensor[position].transpose(0, 1))


def test_a_token_beyond_two_billion_elements_of_cache():
    """Offsets into a cache pass 32 bits: five slots of 3.5 million rows of 128."""
    slots, capacity, D = 5, 3_500_000, 128
    caches = [torch.zeros(slots, 1, capacity, D, dtype=torch.bfloat16, device=DEVICE) for _ in range(2)]
    q, k, v = (randn(70 + i, slots, 1, 2 if i == 0 else 1, D, dtype=torch.bfloat16) for i in range(3))
    lengths = torch.tensor([0, 5, 100, capacity - 1, capacity + 77], dtype=torch.int32, device=DEVICE)
    recent = randn(75, slots, 40, D, dtype=torch.bfloat16)
    for s, n in enumerate(lengths.tolist()):
        for j in range(min(n, 40)):
            row = (n - 1 - j) % capacity
            caches[0][s, 0, row] = recent[s, j]
            caches[1][s, 0, row] = recent[s, j] * 0.5
    for tokens in (1, 2):  # the kernel of a single token, and that of chunks
        query, key, value = (t.repeat_interleave(tokens, dim=1) for t in (q, k, v))
        output = mixers.window_attention_update(query, key, value, *caches, lengths, window=30)
        for s, n in enumerate(lengths.tolist()):
            held = recent[s, :min(n, 40)].flip(0)
            keys = torch.cat([held, key[s, :, 0]]).unsqueeze(1)
            values = torch.cat([held * 0.5, value[s, :, 0]]).unsqueeze(1)
            want, bound, most = reference.window(query[s], keys, values, 30, 0, past=len(held))
            tolerance, = window_tolerances(torch.bfloat16, [bound], most, 32, 2 * D)
            close(output[s], want, tolerance)
    del caches


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("sizes", [(1, 16, 2, 64, 9000, 4), (2, 4, 4, 128, 4000, 0), (1, 40, 2, 32, 3000, 1)])
def test_a_long_cache_is_shared_out_and_joined(sizes, dtype):
    slots, H, Hkv, D, size, sinks = sizes
    q = randn(80, slots, 1, H, D, dtype=dtype)
    k, v = (randn(81 + i, slots, 1, Hkv, D, dtype=dtype) for i in range(2))
    caches = [randn(85 + i, slots, Hkv, size + sinks, D, dtype=dtype) for i in range(2)]
    for past in (0, 1, 31, 500, size - 1, size + sinks, 5 * size):
        lengths = torch.full((slots,), past, dtype=torch.int32, device=DEVICE)
        before = [c.clone() for c in caches]
        output = mixers.window_attention_update(q, k, v, *caches, lengths, window=size, sinks=sinks)
        first = max(0, past - size + 1)
        position = torch.tensor([*range(min(sinks, first)), *range(first, past)], device=DEVICE,
                                dtype=torch.long)
        row = torch.where(position < sinks, position, sinks + (position - sinks) % size)
        for s in range(slots):
            keys, values = (torch.cat([c[s][:, row].transpose(0, 1), n[s]])
                            for c, n in zip(before, (k, v)))
            want, bound, most = reference.window(q[s], keys, values, 2**31, 0, past=len(position))
            tolerance, = window_tolerances(dtype, [bound], most, size, 2 * D)
            close(output[s], want, tolerance, past)


# ---------------------------------------------------------------------------
# inputs as they come
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("width", [64, 36])
def test_strided_inputs_are_read_in_place(width, dtype):
    """Parts of a fused projection, an expanded gradient, heads first, a step between elements."""
    B, T, H = 2, 90, 3
    fused = randn(90, B, T, 3, H, width, dtype=dtype)
    heads_first = randn(91, B, H, T, width, dtype=dtype).transpose(1, 2)
    stepped = randn(92, B, T, H, 2 * width, dtype=dtype)[..., ::2]
    odd_base = randn(93, B * T * H * width + 1, dtype=dtype)[1:].view(B, T, H, width)
    log_decay = rates(H)
    for q, k, v in ([fused[:, :, i] for i in range(3)], [heads_first, stepped, fused[:, :, 1]],
                    [odd_base, heads_first, odd_base]):
        for run in (lambda *x: mixers.decay_attention(*x, log_decay),
                    lambda *x: mixers.window_attention(*x, window=33, sinks=2)):
            results = []
            for copy in (False, True):
                leaves = [(x.contiguous() if copy else x).detach().requires_grad_() for x in (q, k, v)]
                if copy:
                    leaves = [x.detach().clone().requires_grad_() for x in leaves]
                output = run(*leaves)
                grad = torch.ones((), dtype=dtype, device=DEVICE).expand_as(output)
                results.append([output.detach(), *torch.autograd.grad(output, leaves, grad)])
            assert all(torch.equal(a, b) for a, b in zip(*results))


@pytest.mark.parametrize("dtype", DTYPES)
def test_more_sequences_than_threads(dtype):
    """1100 sequences of 0 to 6 tokens: the search for a block's sequence takes several rounds."""
    lengths = [(7 * i + i // 5) % 7 for i in range(1100)]
    H, Hkv, D, Dv = 2, 1, 24, 40
    tensors, grad_output = inputs_of((None, lengths, H, Hkv, D, Dv), dtype, seed=99)
    log_decay, cu = rates(H), offsets_of(lengths)
    parts = [[t.detach()[begin:end] for t in (*tensors, grad_output)]
             for begin, end in zip(cu.tolist(), cu.tolist()[1:]) if end > begin]
    leaves = [t.requires_grad_() for t in tensors]
    output = mixers.decay_attention_varlen(*leaves, cu, log_decay)
    got = [output.detach(), *torch.autograd.grad(output, leaves, grad_output)]
    for i in range(4):
        want, bound = (torch.cat([
            reference.decay(*p[:3], log_decay, absolute=absolute)[0] if i == 0 else
            reference.decay(*p[:3], log_decay, grad_output=p[3], absolute=absolute)[i - 1]
            for p in parts]) for absolute in (False, True))
        close(got[i], want, decay_tolerance(dtype, bound, 12, D + Dv), i)
    output = mixers.window_attention_varlen(*leaves, cu, window=3, sinks=1)
    got = [output.detach(), *torch.autograd.grad(output, leaves, grad_output)]
    results = [(reference.window(*p[:3], 3, 1), reference.window(*p[:3], 3, 1, grad_output=p[3])) for p in parts]
    most = max(forward[2] for forward, _ in results)
    for i in range(4):
        want, bound = (torch.cat([forward[j] if i == 0 else backward[j][i - 1]
                                  for forward, backward in results]) for j in (0, 1))
        tolerance, = window_tolerances(dtype, [bound], most, 12, D + Dv)
        close(got[i], want, tolerance, i)
    q, k, v = (t.detach() for t in leaves)
    state, lengths_of = torch.zeros(len(lengths), H, D, Dv, device=DEVICE), torch.zeros(
        len(lengths), dtype=torch.int32, device=DEVICE)
    caches = [torch.zeros(len(lengths), Hkv, 4, w, dtype=dtype, device=DEVICE) for w in (D, Dv)]
    assert torch.equal(mixers.window_attention_update(q, k, v, *caches, lengths_of, cu, window=3, sinks=1), got[0])
    close(mixers.decay_attention_update(q, k, v, log_decay, state, cu),
          *(torch.cat([f(reference.decay(*p[:3], log_decay, absolute=absolute)[0]) for p in parts])
            for absolute, f in ((False, lambda x: x),
                                (True, lambda x: decay_tolerance(dtype, x, 12, D + Dv)))))


@pytest.mark.parametrize("which", ["decay", "window"])
def test_a_sequence_of_more_than_two_billion_elements(which):
    """The last tokens of 140000 with 128 heads of 128 lie beyond 32 bits in every tensor; they
    depend on the tokens just before them alone."""
    T, H, D, tail, before = 140000, 128, 128, 64, 400
    generator = torch.Generator(device=DEVICE).manual_seed(98)
    draw = lambda heads: torch.randn(1, T, heads, D, device=DEVICE, dtype=torch.bfloat16, generator=generator)
    leaves = [draw(H).requires_grad_(), draw(1).requires_grad_(), draw(1).requires_grad_()]
    log_decay = torch.full((H,), -0.3, device=DEVICE)
    output = mixers.decay_attention(*leaves, log_decay) if which == "decay" else \
        mixers.window_attention(*leaves, window=100)
    grad = draw(H)
    gradients = torch.autograd.grad(output, leaves, grad)
    rows = [t.detach()[0, -before:] for t in leaves]
    if which == "decay":
        want = [reference.decay(*rows, log_decay)[0],
                *reference.decay(*rows, log_decay, grad_output=grad[0, -before:])]
        bound = [reference.decay(*rows, log_decay, absolute=True)[0],
                 *reference.decay(*rows, log_decay, grad_output=grad[0, -before:], absolute=True)]
        # (what the tokens before count for: e^(-0.3 * 336), 1e-44)
        tolerances = [decay_tolerance(torch.bfloat16, b, before * H, 2 * D) for b in bound]
    else:
        out, b, most = reference.window(*rows, 100, 0)
        grads, bounds, _ = reference.window(*rows, 100, 0, grad_output=grad[0, -before:])
        want = [out, *grads]
        tolerances = window_tolerances(torch.bfloat16, [b, *bounds], most, before * H, 2 * D)
    for name, got, w, tolerance in zip(("output", "dq", "dk", "dv"), (output, *gradients), want, tolerances):
        close(got.detach()[0, -tail:], w[-tail:], tolerance[-tail:], name)


def test_outputs_farther_apart_than_an_offset_of_24_bits():
    """Tokens of 70000 heads are 17.9 MB of outputs apart; a gradient of the outputs that is
    expanded has no such strides itself."""
    heads, tokens = 70000, 20
    q = randn(94, 1, tokens, heads, 8, dtype=torch.bfloat16)
    k, v = randn(95, 1, tokens, 1, 8, dtype=torch.bfloat16), randn(96, 1, tokens, 1, 128, dtype=torch.bfloat16)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    output = mixers.window_attention(*leaves, window=7)
    grad = randn(97, 1, 1, 1, 128, dtype=torch.bfloat16).expand_as(output)
    got, = torch.autograd.grad(output, (q,), grad)
    few = [0, 1, 34999, heads - 1]
    rows = [q.detach()[0, :, few], k.detach()[0], v.detach()[0]]
    want, bounds, most = reference.window(*rows, 7, 0, grad_output=grad[0, :, few])
    tolerances = window_tolerances(torch.bfloat16, bounds, most, 7, 128)
    close(got[0, :, few], want[0], tolerances[0])


def test_results_do_not_change_from_run_to_run():
    shape = (None, [700, 1, 900, 64], 8, 2, 64, 64)
    tensors, grad_output = inputs_of(shape, torch.bfloat16, seed=100)
    offsets, log_decay = offsets_of(shape[1]), rates(8)
    leaves = [t.requires_grad_() for t in tensors]
    runs = []
    for _ in range(3):
        run = []
        for output in (mixers.decay_attention_varlen(*leaves, offsets, log_decay),
                       mixers.window_attention_varlen(*leaves, offsets, window=100, sinks=4)):
            run += [output.detach(), *torch.autograd.grad(output, leaves, grad_output)]
        runs.append(run)
    assert all(torch.equal(a, b) for run in runs[1:] for a, b in zip(runs[0], run))


@pytest.mark.parametrize("dtype", DTYPES)
def test_only_the_requested_gradients_are_computed_and_are_the_same(dtype):
    shape = (None, [300, 41], 4, 2, 32, 48)
    tensors, grad_output = inputs_of(shape, dtype, seed=110)
    offsets, log_decay = offsets_of(shape[1]), rates(4)
    for run in (lambda *x: mixers.decay_attention_varlen(*x, offsets, log_decay),
                lambda *x: mixers.window_attention_varlen(*x, offsets, window=30, sinks=3)):
        leaves = [t.detach().requires_grad_() for t in tensors]
        every = torch.autograd.grad(run(*leaves), leaves, grad_output)
        for needs in itertools.product((False, True), repeat=3):
            if not any(needs):
                continue
            some = [t.detach().requires_grad_(need) for t, need in zip(tensors, needs)]
            wanted = [t for t in some if t.requires_grad]
            got = iter(torch.autograd.grad(run(*some), wanted, grad_output))
            assert all(torch.equal(next(got), g) for g, need in zip(every, needs) if need)


def test_rates_of_zero_and_of_minus_infinity():
    """No decay is a plain running sum; minus infinity leaves a token nothing but itself."""
    (q, k, v), _ = inputs_of(((1, 150), None, 2, 2, 32, 32), torch.float32, seed=120)
    log_decay = torch.tensor([0.0, -math.inf], device=DEVICE)
    output = mixers.decay_attention(q, k, v, log_decay)
    want, _ = reference.decay(q[0], k[0], v[0], log_decay)
    bound, _ = reference.decay(q[0], k[0], v[0], log_decay, absolute=True)
    close(output[0], want, decay_tolerance(torch.float32, bound, 150, 64))
    state = randn(121, 1, 2, 32, 32)
    last = state.clone()
    one = mixers.decay_attention_update(q[:, :1], k[:, :1], v[:, :1], log_decay, last)
    want, after = reference.decay(q[0, :1], k[0, :1], v[0, :1], log_decay, state=state[0])
    close(one[0], want, 1e-5 * (1 + want.abs()))
    close(last[0], after, 1e-6 * (1 + after.abs()))


def test_float16_scores_and_states_beyond_its_range():
    """Scores, states and slopes that float16 cannot hold, and results that it can."""
    (q, k, v), grad = inputs_of(((1, 200), None, 2, 2, 64, 64), torch.float16, seed=130)
    q, k = q * 60, k * 60                       # scores of 10^5 and more
    v, grad = v * 2.0**-8, grad * 2.0**-12
    log_decay = rates(2, low=0.01)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    output = mixers.decay_attention(*leaves, log_decay)
    gradients = torch.autograd.grad(output, leaves, grad)
    rows = [t.detach()[0] for t in leaves]
    want = [reference.decay(*rows, log_decay)[0], *reference.decay(*rows, log_decay, grad_output=grad[0])]
    bound = [reference.decay(*rows, log_decay, absolute=True)[0],
             *reference.decay(*rows, log_decay, grad_output=grad[0], absolute=True)]
    for got, w, b in zip((output.detach(), *gradients), want, bound):
        assert float(w.abs().max()) < 65504
        # (subnormal steps of 2^-24 on the way out)
        close(got[0], w, decay_tolerance(torch.float16, b, 200, 128) + 2.0**-24)
    big = randn(131, 1, 200, 2, 64, dtype=torch.float16, scale=200.0)
    q, k = (t.detach() / 60 for t in (q, k))
    leaves = [t.requires_grad_() for t in (q, k * 2.0**-6, big)]
    output = mixers.window_attention(*leaves, window=50)
    grad = randn(132, *output.shape, dtype=torch.float16, scale=100.0)  # slopes of 10^5
    gradients = torch.autograd.grad(output, leaves, grad)
    want, bounds, most = reference.window(*(t.detach()[0] for t in leaves), 50, 0, grad_output=grad[0])
    tolerances = window_tolerances(torch.float16, bounds, most, 50, 128)
    for got, w, tolerance in zip(gradients, want, tolerances):
        if float(w.abs().max()) < 65000:
            close(got[0], w, tolerance + 2.0**-24)


@pytest.mark.parametrize("offsets", [[1, 100, 200], [0, 150, 100, 200], [0, 100, 199], [0, 300, 200]])
def test_invalid_offsets_give_nan_and_change_nothing(offsets):
    cu = torch.tensor(offsets, dtype=torch.int32, device=DEVICE)
    slots = len(offsets) - 1
    (q, k, v), grad = inputs_of((None, [200], 2, 1, 32, 48), torch.bfloat16, seed=140)
    log_decay = rates(2)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    for output in (mixers.decay_attention_varlen(*leaves, cu, log_decay),
                   mixers.window_attention_varlen(*leaves, cu, window=20, sinks=2)):
        for tensor in (output, *torch.autograd.grad(output, leaves, grad)):
            assert bool(torch.isnan(tensor).all())
    q, k, v = (t.detach() for t in (q, k, v))
    state = randn(141, slots, 2, 32, 48)
    before, other = state.clone(), torch.zeros_like(state)
    assert bool(torch.isnan(mixers.decay_attention_update(q, k, v, log_decay, state, cu)).all())
    assert bool(torch.isnan(mixers.decay_attention_update(q, k, v, log_decay, state, cu,
                                                          state_out=other)).all())
    assert torch.equal(state, before) and torch.equal(other, before)
    caches = [randn(142, slots, 1, 30, w, dtype=torch.bfloat16) for w in (32, 48)]
    kept = [c.clone() for c in caches]
    lengths = torch.full((slots,), 7, dtype=torch.int32, device=DEVICE)
    output = mixers.window_attention_update(q, k, v, *caches, lengths, cu, window=20, sinks=2)
    assert bool(torch.isnan(output).all()) and all(map(torch.equal, caches, kept))


def test_tensors_of_two_devices_are_refused():
    (q, k, v), _ = inputs_of(((2, 5), None, 2, 1, 8, 8), torch.float32, seed=145)
    log_decay, state = rates(2), torch.zeros(2, 2, 8, 8, device=DEVICE)
    caches = [torch.zeros(2, 1, 9, 8, device=DEVICE) for _ in range(2)]
    lengths = torch.zeros(2, dtype=torch.int32, device=DEVICE)
    packed, offsets = [t.flatten(0, 1) for t in (q, k, v)], offsets_of([4, 6])
    for call in (lambda: mixers.decay_attention(q, k.cpu(), v, log_decay),
                 lambda: mixers.decay_attention(q, k, v, log_decay.cpu()),
                 lambda: mixers.decay_attention_varlen(*packed, offsets.cpu(), log_decay),
                 lambda: mixers.decay_attention_update(q, k, v, log_decay, state.cpu()),
                 lambda: mixers.window_attention(q, k, v.cpu(), window=3),
                 lambda: mixers.window_attention_varlen(*packed, offsets.cpu(), window=3),
                 lambda: mixers.window_attention_update(q, k, v, caches[0].cpu(), caches[1], lengths,
                                                        window=9),
                 lambda: mixers.window_attention_update(q, k, v, *caches, lengths.cpu(), window=9)):
        with pytest.raises(ValueError, match="same device"):
            call()


def test_overlapping_states_and_caches_are_refused():
    (q, k, v), _ = inputs_of(((1, 1), None, 2, 2, 8, 8), torch.float32, seed=146)
    log_decay = rates(2)
    both = torch.zeros(2 * 128 + 4, device=DEVICE)
    with pytest.raises(ValueError, match="share no memory"):
        mixers.decay_attention_update(q, k, v, log_decay, both[:128].view(1, 2, 8, 8),
                                      state_out=both[4:132].view(1, 2, 8, 8))
    cache = torch.zeros(1, 2, 9, 8, device=DEVICE)
    lengths = torch.zeros(1, dtype=torch.int32, device=DEVICE)
    with pytest.raises(ValueError, match="share no memory"):
        mixers.window_attention_update(q, k, v, cache, cache, lengths, window=9)
    with pytest.raises(ValueError, match="share no memory"):
        mixers.window_attention_update(q, cache[:, :, :1].transpose(1, 2), v, cache,
                                       torch.zeros_like(cache), lengths, window=9)


@pytest.mark.parametrize("which", ["decay", "window"])
def test_gradients_are_differentiable_once(which):
    (q, k, v), _ = inputs_of(((1, 20), None, 2, 2, 8, 8), torch.float32, seed=147)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    output = mixers.decay_attention(*leaves, rates(2)) if which == "decay" else \
        mixers.window_attention(*leaves, window=5)
    gradients = torch.autograd.grad(output.square().sum(), leaves, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiate twice"):
        gradients[0].sum().backward()


def test_updates_are_seen_by_a_graph_that_keeps_what_they_change():
    """A state, a cache that a graph has saved: its backward refuses to use what is there now."""
    (q, k, v), _ = inputs_of(((2, 3), None, 2, 2, 8, 8), torch.float32, seed=148)
    weight = torch.ones((), device=DEVICE, requires_grad=True)
    state = torch.zeros(2, 2, 8, 8, device=DEVICE)
    state_out = torch.zeros_like(state)
    caches = [torch.zeros(2, 2, 9, 8, device=DEVICE) for _ in range(2)]
    lengths = torch.zeros(2, dtype=torch.int32, device=DEVICE)
    for changed, update in (
        ([state], lambda: mixers.decay_attention_update(q, k, v, rates(2), state)),
        ([state_out], lambda: mixers.decay_attention_update(q, k, v, rates(2), state,
                                                            state_out=state_out)),
        (caches, lambda: mixers.window_attention_update(q, k, v, *caches, lengths, window=9)),
    ):
        kept = [(weight * tensor).sum() for tensor in changed]
        with torch.no_grad():
            update()
        for total in kept:
            with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                total.backward()
    with torch.inference_mode():
        state = torch.zeros(2, 2, 8, 8, device=DEVICE)
        mixers.decay_attention_update(q, k, v, rates(2), state)
    with torch.no_grad():  # and a state made in inference mode serves outside it
        assert mixers.decay_attention_update(q, k, v, rates(2), state).shape == (2, 3, 2, 8)


def test_updates_without_tokens():
    log_decay, state = rates(2), randn(150, 3, 2, 8, 8)
    other = torch.zeros_like(state)
    empty = torch.empty(3, 0, 2, 8, device=DEVICE)
    assert mixers.decay_attention_update(empty, empty, empty, log_decay, state,
                                         state_out=other).shape == (3, 0, 2, 8)
    assert torch.equal(other, state)
    caches = [randn(151, 3, 2, 9, 8) for _ in range(2)]
    lengths = torch.zeros(3, dtype=torch.int32, device=DEVICE)
    assert mixers.window_attention_update(empty, empty, empty, *caches, lengths, window=9).numel() == 0


# ---------------------------------------------------------------------------
# streams, graphs, tracing
# ---------------------------------------------------------------------------

def test_another_stream_than_the_current_one():
    (q, k, v), grad = inputs_of(((2, 400), None, 4, 2, 64, 64), torch.bfloat16, seed=160)
    log_decay = rates(4)
    leaves = [t.requires_grad_() for t in (q, k, v)]

    def both():
        run = []
        for output in (mixers.decay_attention(*leaves, log_decay),
                       mixers.window_attention(*leaves, window=90, sinks=1)):
            run += [output.detach(), *torch.autograd.grad(output, leaves, grad)]
        return run

    want = both()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for stream in streams:  # two calls at once
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            got.append(both())
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for run in got for a, b in zip(want, run))


def test_decoding_steps_replay_from_a_graph():
    """Twelve tokens of a layer with both mixers, one captured step replayed; every replay is
    compared with the eager step, with eager work in between."""
    slots, H, Hkv, D, size, sinks, dtype = 3, 8, 2, 64, 600, 2, torch.bfloat16
    log_decay = rates(H)
    tokens = [randn(170 + i, slots, 12, H if i == 0 else Hkv, D, dtype=dtype) for i in range(3)]
    history = [randn(175 + i, slots, Hkv, size + sinks, D, dtype=dtype) for i in range(2)]

    def fresh():
        return dict(state=randn(177, slots, H, D, D), caches=[h.clone() for h in history],
                    lengths=torch.tensor([0, 599, 1000], dtype=torch.int32, device=DEVICE))

    def step(s, q, k, v):
        first = mixers.decay_attention_update(q, k, v, log_decay, s["state"])
        second = mixers.window_attention_update(q, k, v, *s["caches"], s["lengths"], window=size,
                                                sinks=sinks)
        s["lengths"] += 1
        return first, second

    eager, captured = fresh(), fresh()
    static = [t[:, :1].clone() for t in tokens]
    warm = fresh()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(warm, *static)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outputs = step(captured, *static)
    for i in range(12):
        part = [t[:, i:i + 1] for t in tokens]
        for s, p in zip(static, part):
            s.copy_(p)
        graph.replay()
        want = step(eager, *part)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outputs, want)), i
        assert torch.equal(captured["state"], eager["state"])
        assert all(torch.equal(a, b) for a, b in zip(captured["caches"], eager["caches"]))


def test_forwards_replay_from_a_graph_and_backwards_are_refused():
    shape = (None, [300, 0, 411], 4, 2, 64, 64)
    (q, k, v), grad = inputs_of(shape, torch.bfloat16, seed=180)
    offsets, log_decay = offsets_of(shape[1]), rates(4)
    run = lambda: (mixers.decay_attention_varlen(q, k, v, offsets, log_decay),
                   mixers.window_attention_varlen(q, k, v, offsets, window=90, sinks=3))
    run()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outputs = run()
    for i in range(4):
        q.copy_(randn(181 + i, *q.shape, dtype=q.dtype))
        graph.replay()
        want = run()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outputs, want))
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for call in (lambda: mixers.decay_attention_varlen(*leaves, offsets, log_decay),
                     lambda: mixers.window_attention_varlen(*leaves, offsets, window=9)):
            with pytest.raises(RuntimeError, match="cannot be recorded"):
                call()
        with pytest.raises(RuntimeError, match="cannot be recorded"):
            torch.ops.rosa_soft.decay_attention_vjp(q, k, v, offsets, log_decay, grad, 1.0, 7)


def test_tracing_keeps_the_operators():
    (q, k, v), _ = inputs_of(((1, 70), None, 2, 1, 16, 16), torch.float32, seed=190)
    log_decay = rates(2)

    def block(q, k, v):
        return mixers.decay_attention(q, k, v, log_decay) + mixers.window_attention(q, k, v, window=9)

    compiled = torch.compile(block, backend="aot_eager", fullgraph=True)
    results = []
    for call in (block, compiled):
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        output = call(*leaves)
        results.append([output.detach(), *torch.autograd.grad(output.square().sum(), leaves)])
    assert all(torch.equal(a, b) for a, b in zip(*results))


# ---------------------------------------------------------------------------
# gradients by differences, and the mixers together
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("which", ["decay", "window"])
def test_gradients_against_differences(which):
    """Central differences of a scalar along a random direction.  Truncation is the third
    derivative, at most of the order of the value times step^2 = 2^-12; rounding is 2^-24 times the
    sum of the terms over the step."""
    (q, k, v), grad = inputs_of(((1, 100), None, 2, 1, 16, 16), torch.float32, seed=200)
    log_decay = rates(2)
    run = (lambda *x: mixers.decay_attention(*x, log_decay)) if which == "decay" else \
        (lambda *x: mixers.window_attention(*x, window=20, sinks=2))
    leaves = [t.requires_grad_() for t in (q, k, v)]
    gradients = torch.autograd.grad(run(*leaves), leaves, grad)
    step = 2.0**-6
    for i, (leaf, gradient) in enumerate(zip(leaves, gradients)):
        direction = randn(205 + i, *leaf.shape)
        direction /= direction.norm()
        values = []
        for sign in (1, -1):
            moved = [t.detach() for t in leaves]
            moved[i] = moved[i] + sign * step * direction
            terms = run(*moved).double() * grad.double()
            values.append(terms.sum())
            rounding = float32_slack(100, 32) * float(terms.abs().sum())
        slope = float((values[0] - values[1]) / (2 * step))
        want = float((gradient.double() * direction.double()).sum())
        assert abs(slope - want) <= 2.0**-12 * float(gradient.double().norm()) + rounding / step


def hybrid(parameters, symbols, log_decay, offsets):
    """The framework's mixer and the two beside it, on the same packed tokens, added up."""
    q, k, v = parameters
    exact = rosa_soft_amd.rosa_soft_varlen(*symbols, offsets, max_suffix_length=16)
    return exact + mixers.decay_attention_varlen(q, k, v, offsets, log_decay) \
        + mixers.window_attention_varlen(q, k, v, offsets, window=24, sinks=2)


def test_a_hybrid_block_trains_and_serves_the_same_tokens():
    """One block of three mixers: its gradients are the sums of theirs, and serving the tokens of
    each sequence chunk by chunk gives the block's outputs."""
    H, D, dtype, lengths = 4, 8, torch.float32, [61, 90]
    offsets, log_decay = offsets_of(lengths), rates(H)
    symbols = [randn(210 + i, sum(lengths), H, D).sign().mul(0.5).requires_grad_() for i in range(3)]
    parameters = [randn(215 + i, sum(lengths), H, D).requires_grad_() for i in range(3)]
    output = hybrid(parameters, symbols, log_decay, offsets)
    grad = randn(218, *output.shape)
    together = torch.autograd.grad(output, [*symbols, *parameters], grad)
    parts = [rosa_soft_amd.rosa_soft_varlen(*symbols, offsets, max_suffix_length=16),
             mixers.decay_attention_varlen(*parameters, offsets, log_decay),
             mixers.window_attention_varlen(*parameters, offsets, window=24, sinks=2)]
    alone = [torch.autograd.grad(part, leaves, grad)
             for part, leaves in zip(parts, (symbols, parameters, parameters))]
    for i in range(3):  # (the operator's own backward adds with atomics)
        assert torch.allclose(together[i], alone[0][i], rtol=1e-4, atol=1e-6)
        assert torch.equal(together[3 + i], alone[1][i] + alone[2][i]) or torch.equal(
            together[3 + i], alone[2][i] + alone[1][i])

    runtime = rosa_soft_amd.RosaRuntime(H, H, D, D, 16)
    state = torch.zeros(2, H, D, D, device=DEVICE)
    caches = [torch.zeros(2, H, 26, D, device=DEVICE) for _ in range(2)]
    seen = torch.zeros(2, dtype=torch.int32, device=DEVICE)
    served, at = [[], []], [0, 0]
    for chunk in ([40, 1], [1, 0], [0, 60], [20, 29]):
        pick = lambda t: torch.cat([t.detach().split(lengths)[s][at[s]:at[s] + chunk[s]] for s in (0, 1)])
        cu = offsets_of(chunk)
        exact, _ = runtime.update(*(pick(t) for t in symbols), cu_seqlens=cu)
        q, k, v = (pick(t) for t in parameters)
        out = exact + mixers.decay_attention_update(q, k, v, log_decay, state, cu) \
            + mixers.window_attention_update(q, k, v, *caches, seen, cu, window=24, sinks=2)
        seen += cu.diff()
        for s, part in enumerate(out.split(chunk)):
            served[s].append(part)
            at[s] += chunk[s]
    want = output.detach()
    got = torch.cat([torch.cat(parts) for parts in served])
    # both are float32 sums of the same terms in another order: 2^-24 each, of sums below 100
    assert float((got - want).abs().max()) <= 200 * float32_slack(100, 16)
