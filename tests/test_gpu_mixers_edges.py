"""The mixers where their arithmetic or their launches reach an end: factors that follow the data's
range, rows that are not finite, outputs and scratch off 16 bytes, more blocks than one launch
dimension holds.  Tolerances as in ``test_gpu_mixers``."""

import ctypes

import pytest
import torch

from rosa_soft_amd import cabi, mixers
from tests import mixer_reference as reference
from tests.test_gpu_mixers import (DEVICE, close, decay_tolerance, offsets_of, randn, rates,
                                   window_tolerances)
from tests.mixer_reference import HALF_STEP, float32_slack

pytestmark = pytest.mark.gpu

# half a step of float16's smallest numbers, on the way to a product and on the way out
SMALLEST = 2.0**-24


# ---------------------------------------------------------------------------
# float16: what is rounded is scaled by a power of two that follows the data
# ---------------------------------------------------------------------------

def decay_results(leaves, log_decay, grad):
    output = mixers.decay_attention(*leaves, log_decay)
    return [output.detach(), *torch.autograd.grad(output, leaves, grad)]


def check_decay(tensors, log_decay, grad, what=""):
    """One sequence, forward and backward, every element against the definition."""
    leaves = [t.requires_grad_() for t in tensors]
    got = decay_results(leaves, log_decay, grad)
    rows, go = [t.detach()[0] for t in leaves], grad[0]
    want, bound = ([reference.decay(*rows, log_decay, absolute=absolute)[0],
                    *reference.decay(*rows, log_decay, grad_output=go, absolute=absolute)]
                   for absolute in (False, True))
    tokens, width = rows[0].shape[0], rows[0].shape[-1] + rows[2].shape[-1]
    share = rows[0].shape[1] // rows[1].shape[1]
    for name, g, w, b in zip(("output", "dq", "dk", "dv"), got, want, bound):
        close(g[0], w, decay_tolerance(g.dtype, b, tokens * share, width) + SMALLEST, (what, name))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("zeros", ["keys", "values", "gradients", "queries"])
@pytest.mark.parametrize("spans", [((0, 1900),), ((90, 1800),), ((10, 70), (130, 700), (710, 1999))])
def test_decayed_states_pass_through_every_exponent(zeros, spans, dtype):
    """Over tokens that are exactly zero (padding, a loss that masks a prompt) states, and the
    gradients' states, only decay, through every exponent down to zero."""
    heads = 6
    q, k, v = (randn(300 + i, 1, 2000, heads if i == 0 else 3, 32, dtype=dtype) for i in range(3))
    grad = randn(303, 1, 2000, heads, 32, dtype=dtype)
    for begin, end in spans:
        dict(keys=k, values=v, gradients=grad, queries=q)[zeros][:, begin:end] = 0
    # e^-0.02 passes 2^-128 after 4400 tokens, e^-5 after 18
    check_decay([q, k, v], rates(heads, low=0.02, high=5.0), grad)


@pytest.mark.parametrize("rate", [0.9, 1.1, 1.3, 1.35, 1.4, 1.45, 1.6, 3.0])
def test_scores_that_are_nothing_but_a_far_key(rate):
    """One key in 60 tokens: the scores behind it are powers of the rate alone, 2^-90 and less."""
    q, k, v = (randn(310 + i, 1, 256, 2, 32, dtype=torch.float16) for i in range(3))
    keep = torch.zeros(256, dtype=torch.bool, device=DEVICE)
    keep[::60] = True
    k[:, ~keep] = 0
    check_decay([q, k, v], torch.full((2,), -rate, device=DEVICE),
                randn(313, 1, 256, 2, 32, dtype=torch.float16), rate)


@pytest.mark.parametrize("exponent", [-149, -140, -127, -120, -114, -100, -60, -20, 0])
@pytest.mark.parametrize("zeros", [False, True])
def test_updates_on_top_of_states_of_every_size(exponent, zeros):
    log_decay = rates(2)
    q, k, v = (randn(320 + i, 1, 70, 2, 32, dtype=torch.float16) for i in range(3))
    if zeros:
        k[:, :66] = 0
    start = (randn(323, 1, 2, 32, 32).double() * 2.0**exponent).float()
    state = start.clone()
    output = mixers.decay_attention_update(q, k, v, log_decay, state)
    rows = [t[0] for t in (q, k, v)]
    want, last = reference.decay(*rows, log_decay, state=start[0])
    bound, last_bound = reference.decay(*rows, log_decay, state=start[0], absolute=True)
    close(output[0], want, decay_tolerance(torch.float16, bound, 70, 64) + SMALLEST)
    # (2^-126: what float32 products may flush)
    close(state[0], last, (float32_slack(70, 32) + 2.0**-23) * last_bound + 70 * 2.0**-126)


def peaked(tokens, heads, low_keys, seed):
    """Queries and keys along one direction: keys in ``low_keys`` score 56 to 100 nats, head by
    head, below the others; values and output gradients as usual."""
    scale = 32**-0.5
    gap = torch.linspace(56.0, 100.0, heads, device=DEVICE)
    q, k, v = (randn(seed + i, 1, tokens, heads, 32, scale=0.25) for i in range(3))
    q[..., 0] = 16.0
    k[..., 0] = (gap / (2 * scale * 16.0)) * torch.where(low_keys, -1.0, 1.0).view(1, -1, 1)
    return [t.half() for t in (q, k, v)], randn(seed + 3, 1, tokens, heads, 32, dtype=torch.float16)


@pytest.mark.parametrize("tokens,window,sinks", [
    (100, 30, 1),      # the sink's own block walks the tokens beyond its window
    (2000, 50, 1),     # kernels of their own
    (1500, 300, 20),   # sums of dO . o from the output
])
@pytest.mark.parametrize("low", ["sinks", "blocks"])
@pytest.mark.parametrize("small", [1.0, 2.0**-12])
def test_slopes_of_keys_far_below_the_maximum(low, small, tokens, window, sinks):
    position = torch.arange(tokens, device=DEVICE)
    low_keys = position < sinks if low == "sinks" else position // 16 % 3 != 1
    tensors, grad = peaked(tokens, 12, low_keys, seed=330)
    grad = grad * small
    leaves = [t.requires_grad_() for t in tensors]
    output = mixers.window_attention(*leaves, window=window, sinks=sinks)
    got = [output.detach(), *torch.autograd.grad(output, leaves, grad)]
    rows = [t.detach()[0] for t in leaves]
    out, bound, most = reference.window(*rows, window, sinks)
    grads, bounds, _ = reference.window(*rows, window, sinks, grad_output=grad[0])
    tolerances = window_tolerances(torch.float16, [bound, *bounds], most, tokens, 64)
    for name, g, w, tolerance in zip(("output", "dq", "dk", "dv"), got, (out, *grads), tolerances):
        close(g[0], w, tolerance + SMALLEST, name)


# ---------------------------------------------------------------------------
# the sinks' gradients by pieces of tokens
# ---------------------------------------------------------------------------

def check_window_sequences(tensors, grad, lengths, window, sinks, checked=None):
    """A packed batch, forward and backward; sequences ``checked`` against the definition."""
    leaves = [t.requires_grad_() for t in tensors]
    output = mixers.window_attention_varlen(*leaves, offsets_of(lengths), window=window, sinks=sinks)
    got = [output.detach(), *torch.autograd.grad(output, leaves, grad)]
    parts = [[t.detach().split(lengths)[s] for t in (*leaves, grad)]
             for s in (range(len(lengths)) if checked is None else checked)]
    results = [t.split(lengths) for t in got]
    share = leaves[0].shape[1] // leaves[1].shape[1]
    width = leaves[0].shape[2] + leaves[2].shape[2]
    # results below 2^-14 have steps of 2^-24 in float16, whatever their terms: rounding is off by
    # 2^-25 where the tolerance, relative to the terms, may be less (the last key of a sequence has
    # the one term p dO)
    step = SMALLEST if leaves[0].dtype == torch.float16 else 0.0
    for place, (q, k, v, go) in zip(range(len(lengths)) if checked is None else checked, parts):
        if len(q) == 0:
            continue
        out, bound, most = reference.window(q, k, v, window, sinks)
        grads, bounds, _ = reference.window(q, k, v, window, sinks, grad_output=go)
        tolerances = window_tolerances(q.dtype, [bound, *bounds], most, len(q) * share, width)
        for name, g, w, tolerance in zip(("output", "dq", "dk", "dv"), results, (out, *grads), tolerances):
            close(g[place], w, tolerance + step, (place, len(q), name))


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("heads", [(8, 8), (8, 2), (9, 1)])
def test_pieces_of_packed_sequences_keep_apart(heads, dtype):
    """Sequences of one token more and less than the shortest with pieces (64 or 128 keys, a window
    of 20, up to eight more steps of 64 tokens) beside long, short and empty ones; pieces of 256
    tokens that begin and end everywhere."""
    lengths = [84, 83, 1, 596, 595, 0, 660, 659, 84, 257, 1300, 511, 148, 147, 3, 276, 275, 700, 85]
    tensors = [randn(340 + i, sum(lengths), heads[i > 0], 24, dtype=dtype) for i in range(3)]
    grad = randn(343, sum(lengths), heads[0], 24, dtype=dtype)
    check_window_sequences(tensors, grad, lengths, 20, 5)


def test_pieces_get_longer_where_their_sums_would_take_too_much():
    """16 heads on one, 64 sinks, a window of 8: sums of pieces of 256 tokens would take 4.8 GB,
    those of 512 take half, and sequences of up to 512 tokens have none."""
    lengths = [700, 90, 200, 1500, 513, 512, 64, 1, 1024, 400] * 43
    tensors = [randn(350 + i, sum(lengths), 16 if i == 0 else 1, 128, dtype=torch.bfloat16) for i in range(3)]
    grad = randn(353, sum(lengths), 16, 128, dtype=torch.bfloat16)
    checked = [*range(10), 213, 218, *range(len(lengths) - 10, len(lengths))]
    check_window_sequences(tensors, grad, lengths, 8, 64, checked)


# ---------------------------------------------------------------------------
# arrays off 16 bytes
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("widths", [(7, 12), (5, 64), (33, 100), (1, 4)])
def test_scratch_of_odd_widths(widths, dtype):
    """Gradients of shared heads go through two float32 arrays, the second behind odd rows."""
    D, Dv = widths
    tensors = [randn(360, 1, 1301, 4, D, dtype=dtype), randn(361, 1, 1301, 1, D, dtype=dtype),
               randn(362, 1, 1301, 1, Dv, dtype=dtype)]
    grad = randn(363, 1, 1301, 4, Dv, dtype=dtype)
    check_decay(tensors, rates(4), grad)
    check_window_sequences([t.detach()[0] for t in tensors], grad[0], [1301], 1301, 0)


class Shifted:
    """Memory for an output ``shift`` elements behind a 16-byte address, NaN around it."""

    def __init__(self, like, shift):
        self.shift, self.like = shift, like
        self.memory = torch.full((like.numel() + 16,), float("nan"), dtype=like.dtype, device=DEVICE)

    @property
    def pointer(self):
        return self.memory.data_ptr() + self.shift * self.memory.element_size()

    def check(self, want):
        inside = self.memory[self.shift:self.shift + want.numel()]
        assert torch.equal(inside.view(want.shape), want)
        outside = torch.cat([self.memory[:self.shift], self.memory[self.shift + want.numel():]])
        assert bool(torch.isnan(outside).all())


def described(tensor):
    return ctypes.byref(cabi.RosaMixerTensor(tensor.data_ptr(), tensor.stride(0), *tensor.stride()[1:3]))


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("shift", [0, 1, 2, 3, 4, 6])
@pytest.mark.parametrize("width", [64, 36])
def test_c_entries_write_outputs_at_any_element(width, shift, dtype):
    """Callers of the C interface choose where outputs and gradients lie."""
    library = cabi.load()
    q, k, v = (randn(370 + i, 2, 150, 4 if i == 0 else 2, width, dtype=dtype) for i in range(3))
    grad = randn(373, 2, 150, 4, width, dtype=dtype)
    log_decay, scale = rates(4), width**-0.5
    code = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}[dtype]
    problem = ctypes.byref(cabi.RosaMixerProblem(code, 2, 150, 300, 0, 4, 2, width, width, scale, None))
    rows, go = [described(t) for t in (q, k, v)], described(grad)
    stream = torch.cuda.current_stream().cuda_stream
    workspace = torch.empty(1 << 24, dtype=torch.uint8, device=DEVICE)
    space = (workspace.data_ptr(), workspace.numel(), stream)

    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    want = decay_results(leaves, log_decay, grad)
    outs = [Shifted(t, shift) for t in want]
    assert library.rosa_hip_decay_forward(problem, *rows, log_decay.data_ptr(), outs[0].pointer, *space) == 0
    assert library.rosa_hip_decay_backward(problem, *rows, go, log_decay.data_ptr(),
                                           *(o.pointer for o in outs[1:]), *space) == 0
    for out, tensor in zip(outs, want):
        out.check(tensor)

    output, log_sum = torch.ops.rosa_soft.window_attention(*leaves, None, 40, 2, None, True)
    want = [output.detach(), *torch.autograd.grad(output, leaves, grad)]
    outs = [Shifted(t, shift) for t in want]
    sums = torch.empty_like(log_sum)
    assert library.rosa_hip_window_forward(problem, 40, 2, *rows, outs[0].pointer, sums.data_ptr(), stream) == 0
    # (the forward's output is read where it was written)
    assert library.rosa_hip_window_backward(problem, 40, 2, *rows, outs[0].pointer, sums.data_ptr(), go,
                                            *(o.pointer for o in outs[1:]), *space) == 0
    for out, tensor in zip(outs, want):
        out.check(tensor)
    assert torch.equal(sums, log_sum)


# ---------------------------------------------------------------------------
# packed as dense
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("lengths", [[32] * 64, [32] * 20 + [600] + [1, 400, 7, 513, 512] * 2])
def test_packed_sequences_have_the_gradients_that_they_have_alone(lengths, dtype):
    """Under a window that none of them fills: the sums dO . o are exact where a sequence is short,
    whatever it is packed with, and come from the output where it is long."""
    heads, masks = 2, dict(window=1024, sinks=0)
    tensors = [randn(380 + i, sum(lengths), heads, 40, dtype=dtype) for i in range(3)]
    grad = randn(383, sum(lengths), heads, 40, dtype=dtype)
    leaves = [t.requires_grad_() for t in tensors]
    output = mixers.window_attention_varlen(*leaves, offsets_of(lengths), **masks)
    got = [t.split(lengths) for t in (output.detach(), *torch.autograd.grad(output, leaves, grad))]
    for s in range(len(lengths)):
        alone = [t.detach().split(lengths)[s].unsqueeze(0).clone().requires_grad_() for t in leaves]
        output = mixers.window_attention(*alone, **masks)
        want = [output.detach(), *torch.autograd.grad(output, alone, grad.split(lengths)[s].unsqueeze(0))]
        for name, g, w in zip(("output", "dq"), got, want):
            assert torch.equal(g[s], w[0]), (s, lengths[s], name)
        # dk and dv are float32 sums over the tokens, in parts whose number goes by all tokens of a
        # call: the order of a sum may differ, float32_slack of its terms, and with it the rounding
        # of the result, half a step on either side
        rows = [t.detach()[0] for t in alone]
        _, bounds, _ = reference.window(*rows, *masks.values(), grad_output=grad.split(lengths)[s])
        for g, w, bound in zip(got[2:], want[2:], bounds[1:]):
            step = 2 * HALF_STEP[dtype] * w[0].double().abs() + (SMALLEST if dtype == torch.float16 else 0.0)
            close(g[s], w[0].double(), step + float32_slack(lengths[s], 80) * bound, (s, lengths[s]))


# ---------------------------------------------------------------------------
# more threads than one dimension of a launch has
# ---------------------------------------------------------------------------

def test_more_blocks_than_a_launch_dimension_holds():
    """Sequences of one token, whose answers are one line each: o = scale (q . k) v for the decay,
    o = v for the window, and dv = scale (q . k) dO, or dO.  2^32 threads are 4.2 million heads of
    128 columns in the decay's forward, 1.4 million in its backward, 16.8 million in the window's."""
    count, H, D = 66000, 64, 128
    ones = dict(dtype=torch.bfloat16, device=DEVICE)
    mark = (torch.arange(count, device=DEVICE) % 5 - 2).to(torch.bfloat16).view(count, 1, 1, 1)
    q = mark.expand(count, 1, H, D).contiguous()
    k, v = torch.ones(count, 1, 1, D, **ones), torch.full((count, 1, 1, D), 0.5, **ones)
    log_decay = rates(H)
    output = mixers.decay_attention(q, k, v, log_decay, scale=2.0**-7)
    assert torch.equal(output, (mark * 0.5).expand_as(output))
    del output
    few = q[:24000].detach().requires_grad_(), k[:24000].clone().requires_grad_(), v[:24000].clone().requires_grad_()
    output = mixers.decay_attention(*few, log_decay, scale=2.0**-7)
    dq, dk, dv = torch.autograd.grad(output, few, torch.ones((), **ones).expand_as(output))
    # sums of 64 heads and, in the products, of 128 columns: exact in float32 and in bfloat16
    assert torch.equal(dq, torch.full_like(dq, 0.5))
    assert torch.equal(dk, (32 * mark[:24000]).expand_as(dk))
    assert torch.equal(dv, (64 * mark[:24000]).expand_as(dv))
    del q, k, v, few, output, dq, dk, dv

    count, H, D = 270000, 64, 4
    mark = (torch.arange(count * H, device=DEVICE) % 251).to(torch.bfloat16).view(count, 1, H, 1)
    v = mark.expand(count, 1, H, D).contiguous().requires_grad_()
    q = torch.ones(count, 1, H, D, **ones)
    for output in (mixers.window_attention(q, q, v, window=3, sinks=1),
                   mixers.window_attention_varlen(q[:, 0], q[:, 0], v[:, 0], torch.arange(
                       count + 1, dtype=torch.int32, device=DEVICE), window=3)):
        assert torch.equal(output.view_as(v), v)
        dv, = torch.autograd.grad(output, (v,), output.detach())
        assert torch.equal(dv, v)
    v = v.detach()
    caches = [torch.zeros(count, H, 3, D, **ones) for _ in range(2)]
    lengths = torch.zeros(count, dtype=torch.int32, device=DEVICE)
    assert torch.equal(mixers.window_attention_update(q, q, v, *caches, lengths, window=3), v)
    assert torch.equal(caches[1][:, :, 0], v[:, 0])
    log_decay, state = rates(H), torch.zeros(count, H, D, D, device=DEVICE)
    output = mixers.decay_attention_update(q, q, v, log_decay, state, scale=0.25)
    assert torch.equal(output, v) and torch.equal(state[:, :, 1], v[:, 0].float())


# ---------------------------------------------------------------------------
# rows that are not finite
# ---------------------------------------------------------------------------

def results_with(run, tensors, grad, spoiled=None, row=0, value=float("nan")):
    """Output, dq, dk, dv with one row of one input replaced."""
    tensors = [t.detach().clone() for t in (*tensors, grad)]
    if spoiled is not None:
        tensors["q k v go".split().index(spoiled)][row] = value
    leaves = [t.requires_grad_() for t in tensors[:3]]
    output = run(*leaves)
    gradients = torch.autograd.grad(output, leaves, tensors[3])
    return dict(zip(("output", "dq", "dk", "dv"), (output.detach(), *gradients)))


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_rows_that_are_not_finite_in_the_decay(value, dtype):
    lengths, row = [300, 900, 200], 300 + 421
    tensors = [randn(390 + i, sum(lengths), 4 if i == 0 else 2, 40, dtype=dtype) for i in range(3)]
    grad, log_decay, cu = randn(393, sum(lengths), 4, 40, dtype=dtype), rates(4), offsets_of(lengths)
    run = lambda *x: mixers.decay_attention_varlen(*x, cu, log_decay)
    clean = results_with(run, tensors, grad)
    own = (row, row + 1)
    later, around_later = (row, 1200), (row - 63, 1200)
    earlier, around_earlier = (300, row + 1), (300, row + 64)
    reach = {"q": dict(output=own, dk=around_earlier, dv=earlier),
             "k": dict(output=later, dq=around_later, dv=own),
             "v": dict(output=around_later, dq=later, dk=own),
             "go": dict(dq=own, dk=earlier, dv=around_earlier)}
    for spoiled, reached in reach.items():
        got = results_with(run, tensors, grad, spoiled, row, value)
        for name, tensor in got.items():
            begin, end = reached.get(name, (row, row))
            for part in (slice(0, begin), slice(end, None)):
                assert torch.equal(tensor[part], clean[name][part]), (spoiled, name)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("window,sinks,Hkv", [(40, 0, 4), (40, 5, 2), (300, 33, 1)])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_rows_that_are_not_finite_in_the_window(value, window, sinks, Hkv, dtype):
    lengths, row = [300, 2500, 200], 300 + 1203
    tensors = [randn(395 + i, sum(lengths), 4 if i == 0 else Hkv, 40, dtype=dtype) for i in range(3)]
    grad, cu = randn(398, sum(lengths), 4, 40, dtype=dtype), offsets_of(lengths)
    run = lambda *x: mixers.window_attention_varlen(*x, cu, window=window, sinks=sinks)
    clean = results_with(run, tensors, grad)
    seen_by = (row, row + window)                        # the tokens that see the row
    sees = (row - window + 1, row + 1)                   # what its token sees, but for the sinks
    wide = lambda span: (span[0] - 127, span[1] + 127)
    # whoever has a NaN output has NaN slopes, and hands them to what it sees
    back = lambda span: (span[0] - window + 1 - 127, span[1] + 127)
    own = (row, row + 1)
    reach = {"q": dict(output=own, dq=own, dk=wide(sees), dv=wide(sees)),
             "k": dict(output=seen_by, dq=wide(seen_by), dk=back(seen_by), dv=back(seen_by)),
             "v": dict(output=wide(seen_by), dq=wide(seen_by), dk=back(wide(seen_by))),
             "go": dict(dq=own, dk=wide(sees), dv=wide(sees))}
    for spoiled, reached in reach.items():
        got = results_with(run, tensors, grad, spoiled, row, value)
        for name, tensor in got.items():
            begin, end = reached.get(name, (row, row))
            same = torch.equal(tensor[end:], clean[name][end:]) and torch.equal(tensor[:300], clean[name][:300])
            first = 364 if sinks and name in ("dk", "dv") else 300
            assert same and torch.equal(tensor[first:begin], clean[name][first:begin]), (spoiled, name)
