"""Mixers without a GPU: argument checks, schemas, fake tensors, C entry points, the definitions."""

import ctypes
import inspect
import math

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from rosa_soft_amd import cabi, mixers
from tests import mixer_reference as reference


def fake(*shape, dtype=torch.bfloat16, device="cuda"):
    return torch.empty(*shape, dtype=dtype, device=device)


def host(*shape, dtype=torch.bfloat16):
    return torch.zeros(*shape, dtype=dtype)


def arguments(make=host, **changes):
    """A dense call that passes every check but that of the device; ``changes`` replace parts."""
    parts = dict(q=make(2, 5, 4, 16), k=make(2, 5, 2, 16), v=make(2, 5, 2, 8),
                 log_decay=make(4, dtype=torch.float32), state=make(2, 4, 16, 8, dtype=torch.float32),
                 keys=make(2, 2, 12, 16), values=make(2, 2, 12, 8),
                 lengths=make(2, dtype=torch.int32), window=9, sinks=3)
    parts.update(changes)
    return parts


def calls(p):
    masks = dict(window=p["window"], sinks=p["sinks"])
    qkv = p["q"], p["k"], p["v"]
    extra = {"scale": p["scale"]} if "scale" in p else {}
    return {
        "decay": lambda: mixers.decay_attention(*qkv, p["log_decay"], **extra),
        "decay_update": lambda: mixers.decay_attention_update(
            *qkv, p["log_decay"], p["state"], state_out=p.get("state_out"), **extra),
        "window": lambda: mixers.window_attention(*qkv, **masks, **extra),
        "window_update": lambda: mixers.window_attention_update(
            *qkv, p["keys"], p["values"], p["lengths"], **masks, **extra),
    }


def test_calls_that_pass_give_outputs_of_the_right_shape():
    with FakeTensorMode():
        for name, call in calls(arguments(fake)).items():
            output = call()
            assert output.shape == (2, 5, 4, 8) and output.dtype == torch.bfloat16, name
        packed = [fake(7, 4, 16), fake(7, 2, 16), fake(7, 2, 8)]
        offsets = fake(3, dtype=torch.int32)
        log_decay = fake(4, dtype=torch.float32)
        assert mixers.decay_attention_varlen(*packed, offsets, log_decay).shape == (7, 4, 8)
        assert mixers.window_attention_varlen(*packed, offsets, window=3).shape == (7, 4, 8)
        gradients = torch.ops.rosa_soft.window_attention_vjp(
            *packed, offsets, fake(7, 4, 8), fake(4, 7, dtype=torch.float32), fake(7, 4, 8), 3, 0,
            0.25, 5)
        assert [g.shape for g in gradients] == [(7, 4, 16), (0,), (7, 2, 8)]
        assert all(g.dtype == torch.bfloat16 for g in gradients)


EVERY = ("decay", "decay_update", "window", "window_update")


@pytest.mark.parametrize("names,changes,error,message", [
    (EVERY, lambda: dict(q=host(5, 4, 16)), ValueError, "must have shape"),
    (EVERY, lambda: dict(k=host(2, 6, 2, 16)), ValueError, "share their token dimensions"),
    (EVERY, lambda: dict(v=host(2, 5, 1, 8)), ValueError, "key and value head counts"),
    (EVERY, lambda: dict(q=host(2, 5, 3, 16)), ValueError, "divisible by key heads"),
    (EVERY, lambda: dict(q=host(2, 5, 4, 17)), ValueError, "query and key widths"),
    (EVERY, lambda: dict(q=host(2, 5, 4, 129), k=host(2, 5, 2, 129)), ValueError, r"\[1, 128\]"),
    (EVERY, lambda: dict(v=host(2, 5, 2, 0)), ValueError, r"\[1, 128\]"),
    (EVERY, lambda: dict(k=host(2, 5, 2, 16, dtype=torch.float16)), ValueError, "same dtype"),
    (EVERY, lambda: {n: host(2, 5, 2, 8, dtype=torch.float64) for n in "qkv"}, ValueError,
     "float32, float16, and bfloat16"),
    (EVERY, lambda: {}, ValueError, "require CUDA tensors"),
    (EVERY, lambda: dict(scale=0.0), ValueError, "positive normal"),
    (EVERY, lambda: dict(scale=math.inf), ValueError, "positive normal"),
    (EVERY, lambda: dict(scale=1e-40), ValueError, "positive normal"),
    (("decay", "window"), lambda: dict(q=host(2, 0, 4, 16), k=host(2, 0, 2, 16), v=host(2, 0, 2, 8)),
     ValueError, "must be >= 1"),
    (("decay_update", "window_update"),
     lambda: dict(q=host(0, 5, 4, 16), k=host(0, 5, 2, 16), v=host(0, 5, 2, 8)), ValueError,
     "at least one slot"),
    (EVERY[:2], lambda: dict(log_decay=host(2, dtype=torch.float32)), ValueError,
     "one entry per query head"),
    (EVERY[:2], lambda: dict(log_decay=host(4)), ValueError, "dtype float32"),
    (EVERY[:1], lambda: dict(log_decay=host(4, dtype=torch.float32).requires_grad_()), ValueError,
     "takes no gradient"),
    (EVERY[1:2], lambda: dict(log_decay=host(4, dtype=torch.float32).requires_grad_()), RuntimeError,
     "have no backward"),
    (EVERY[1:2], lambda: dict(state=host(2, 2, 16, 8, dtype=torch.float32)), ValueError, "shape"),
    (EVERY[1:2], lambda: dict(state=host(2, 4, 16, 8)), ValueError, "float32"),
    (EVERY[1:2], lambda: dict(state=host(2, 4, 8, 16, dtype=torch.float32).transpose(2, 3)),
     ValueError, "contiguous"),
    (EVERY[1:2], lambda: dict(state_out=host(2, 4, 16, 9, dtype=torch.float32)), ValueError, "shape"),
    (EVERY[2:], lambda: dict(window=0), ValueError, "window must be >= 1"),
    (EVERY[2:], lambda: dict(window=True), TypeError, "window must be an integer"),
    (EVERY[2:], lambda: dict(window=2.5), TypeError, "window must be an integer"),
    (EVERY[2:], lambda: dict(sinks=-1), ValueError, "sinks"),
    (EVERY[2:], lambda: dict(sinks=65), ValueError, "sinks"),
    (EVERY[3:], lambda: dict(keys=host(2, 2, 11, 16), values=host(2, 2, 11, 8)), ValueError,
     "hold the sinks and the window"),
    (EVERY[3:], lambda: dict(values=host(2, 2, 13, 8)), ValueError, "shape"),
    (EVERY[3:], lambda: dict(keys=host(2, 2, 12, 16, dtype=torch.float16)), ValueError, "dtype"),
    (EVERY[3:], lambda: dict(keys=host(2, 12, 2, 16).transpose(1, 2)), ValueError, "contiguous"),
    (EVERY[3:], lambda: dict(lengths=host(2, dtype=torch.int64)), ValueError, "lengths"),
    (EVERY[3:], lambda: dict(lengths=host(3, dtype=torch.int32)), ValueError, "lengths"),
    (("decay_update", "window_update"), lambda: dict(q=host(2, 5, 4, 16).requires_grad_()),
     RuntimeError, "have no backward"),
])
def test_refusals(names, changes, error, message):
    """Every check is made before the device is looked at: host tensors meet all of them."""

    for name in names:
        with pytest.raises(error, match=message):
            calls(arguments(**changes()))[name]()


@pytest.mark.parametrize("masks,message", [
    (dict(window=-2**70), "window must be >= 1"), (dict(sinks=2**70), "sinks must be in"),
    (dict(sinks=-2**70), "sinks must be in"), (dict(window=2**63, sinks=2**63), "sinks must be in"),
])
def test_masks_of_more_than_64_bits(masks, message):
    for name in EVERY[2:]:
        with pytest.raises(ValueError, match=message):
            calls(arguments(**masks))[name]()
    with pytest.raises(ValueError, match="require CUDA tensors"):  # an endless window
        calls(arguments(window=2**70))["window"]()


@pytest.mark.parametrize("tokens,refused", [(2**31 - 1025, False), (2**31 - 1024, True), (2**31 - 1, True)])
def test_sequences_end_where_counts_past_their_last_tile_still_fit(tokens, refused):
    """Kernels count up to a tile of tokens past the last one, in 32 bits."""
    long = torch.zeros(1, 1, 1, 1).expand(1, tokens, 1, 1)
    message = "at most 2\\^31 - 1025" if refused else "require CUDA tensors"
    offsets = torch.tensor([0, 5], dtype=torch.int32)
    for call in (lambda: mixers.decay_attention(long, long, long, torch.zeros(1)),
                 lambda: mixers.window_attention(long, long, long, window=3),
                 lambda: mixers.window_attention_varlen(long[0], long[0], long[0], offsets, window=3),
                 lambda: mixers.decay_attention_update(long, long, long, torch.zeros(1), torch.zeros(1, 1, 1, 1))):
        with pytest.raises(ValueError, match=message):
            call()
    library = cabi.load()
    for fields in (dict(B=1, T=tokens), dict(B=0, T=0, S=3, cu_seqlens=1)):
        p = ctypes.byref(problem(N=tokens, H=1, Hkv=1, D=1, Dv=1, **fields))
        assert (library.rosa_hip_decay_workspace_bytes(p, 0) == 0) == refused
        assert (library.rosa_hip_window_workspace_bytes(p, 10, 2, 0) == 0) == refused


@pytest.mark.parametrize("names,which", [
    (EVERY, "q"), (EVERY, "k"), (EVERY, "v"), (EVERY[:2], "log_decay"), (EVERY[1:2], "state"),
    (EVERY[3:], "keys"), (EVERY[3:], "values"),
])
def test_tangents_are_refused(names, which):
    """Forward-mode derivatives do not exist: a dual input is an error, not an output without one."""
    from torch.autograd import forward_ad

    with FakeTensorMode():
        for name in names:
            with forward_ad.dual_level():
                parts = arguments(fake)
                parts[which] = forward_ad.make_dual(parts[which], torch.ones_like(parts[which]))
                with pytest.raises(NotImplementedError, match="forward-mode"):
                    calls(parts)[name]()
            calls(arguments(fake))[name]()
        with forward_ad.dual_level():
            q, k, v = (fake(2, 5, 2, 8) for _ in range(3))
            dual = forward_ad.make_dual(q, q)
            for call in (
                    lambda: torch.ops.rosa_soft.window_attention(dual, k, v, None, 3, 0),
                    lambda: torch.ops.rosa_soft.decay_attention_vjp(
                        q, k, v, None, fake(2, dtype=torch.float32), dual, None, 7)):
                with pytest.raises(NotImplementedError, match="forward-mode"):
                    call()


def test_states_share_no_memory_with_what_is_read():
    """A block may store a state while another still reads its keys or rates."""
    memory = torch.zeros(2 * 4 * 16 * 8 + 64)
    state = memory[:1024].view(2, 4, 16, 8)
    q, k, v = (torch.zeros(2, 1, 4, 16), torch.zeros(2, 1, 4, 16), torch.zeros(2, 1, 4, 8))
    rates = torch.zeros(4)
    inside = memory[512:640].view(2, 1, 4, 16)
    for arguments in ((inside, k, v, rates), (q, inside, v, rates), (q, k, memory[960:1024].view(2, 1, 4, 8), rates),
                      (q, k, v, memory[1020:1024])):
        with pytest.raises(ValueError, match="share no memory"):
            mixers.decay_attention_update(*arguments, state)
        with pytest.raises(ValueError, match="share no memory"):
            mixers.decay_attention_update(*arguments, torch.zeros_like(state), state_out=state)
    with pytest.raises(ValueError, match="require CUDA tensors"):  # behind the state is none of it
        mixers.decay_attention_update(q, k, v, memory[1024:1028], state)


def test_packed_refusals():
    packed = [host(7, 4, 16), host(7, 2, 16), host(7, 2, 8)]
    log_decay = host(4, dtype=torch.float32)
    for offsets, message in ((host(3, dtype=torch.int64), "int32"),
                             (host(1, dtype=torch.int32), "one-dimensional")):
        for call in (lambda: mixers.decay_attention_varlen(*packed, offsets, log_decay),
                     lambda: mixers.window_attention_varlen(*packed, offsets, window=2)):
            with pytest.raises(ValueError, match=message):
                call()


def test_signatures_and_schemas():
    assert mixers.__all__ == [
        "decay_attention", "decay_attention_update", "decay_attention_varlen",
        "window_attention", "window_attention_update", "window_attention_varlen",
    ]
    keyword = inspect.Parameter.KEYWORD_ONLY
    for name in mixers.__all__:
        parameters = inspect.signature(getattr(mixers, name)).parameters
        assert parameters["scale"].kind is keyword and parameters["scale"].default is None
        if name.startswith("window"):
            assert parameters["window"].kind is keyword and parameters["sinks"].default == 0
    for name in ("decay_attention", "decay_attention_vjp", "decay_attention_update",
                 "decay_attention_update_out", "window_attention", "window_attention_vjp",
                 "window_attention_update"):
        assert torch._C._dispatch_has_kernel_for_dispatch_key(f"rosa_soft::{name}", "CUDA")
    written = lambda op: {a.name for a in getattr(torch.ops.rosa_soft, op).default._schema.arguments
                          if a.alias_info is not None and a.alias_info.is_write}
    assert written("decay_attention_update") == {"state"}
    assert written("decay_attention_update_out") == {"state_out"}
    assert written("window_attention_update") == {"key_cache", "value_cache"}
    assert not written("decay_attention") and not written("window_attention")


def problem(**changes):
    fields = dict(dtype=2, B=2, T=100, N=200, S=0, H=4, Hkv=2, D=64, Dv=64, scale=0.125)
    fields.update(changes)
    return cabi.RosaMixerProblem(**fields)


@pytest.mark.parametrize("changes,message", [
    (dict(dtype=3), b"dtype"), (dict(B=0), b"dense layout"), (dict(N=199), b"N = B \\* T"),
    (dict(B=0, T=0, S=0, cu_seqlens=1), b"packed layout"), (dict(H=3), b"multiple"),
    (dict(Hkv=0), b"multiple"), (dict(D=129), b"128"), (dict(Dv=0), b"128"),
    (dict(scale=0.0), b"scale"), (dict(scale=math.nan), b"scale"),
    (dict(B=1, T=2**30, N=2**30, H=2**10), b"too many blocks"),
])
def test_c_entries_refuse_bad_problems_before_any_launch(changes, message):
    """Host arithmetic only; each entry reports the problem instead of dividing by it."""
    library, bad = cabi.load(), problem(**changes)
    tensor = cabi.RosaMixerTensor(1, 0, 64, 64)
    p, t = ctypes.byref(bad), ctypes.byref(tensor)
    assert library.rosa_hip_decay_workspace_bytes(p, 1) == 0
    assert library.rosa_hip_window_workspace_bytes(p, 10, 2, 0) == 0
    assert library.rosa_hip_window_workspace_bytes(p, 10, 2, 12) == 0
    assert library.rosa_hip_decay_forward(p, t, t, t, 1, 1, 1, 1 << 40, None) == 1
    assert library.rosa_hip_decay_backward(p, t, t, t, t, 1, 1, 1, 1, 1, 1 << 40, None) == 1
    assert library.rosa_hip_decay_update(p, t, t, t, 1, 1, 1, 1, 1, 1 << 40, None) == 1
    assert library.rosa_hip_window_forward(p, 10, 2, t, t, t, 1, None, None) == 1
    assert library.rosa_hip_window_backward(p, 10, 2, t, t, t, 1, 1, t, 1, 1, 1, 1, 1 << 40, None) == 1
    assert library.rosa_hip_window_update(p, 10, 2, t, t, t, 1, 1, 12, 1, 1, 1, 1 << 40, None) == 1
    import re
    assert re.search(message, library.rosa_hip_last_error())


def test_c_entries_refuse_null_pointers_masks_and_small_workspaces():
    library, good = cabi.load(), problem()
    packed = problem(B=0, T=0, S=3, cu_seqlens=1)  # (never dereferenced on the host)
    tensor, null = cabi.RosaMixerTensor(1, 0, 64, 64), cabi.RosaMixerTensor(None, 0, 64, 64)
    t, n = ctypes.byref(tensor), ctypes.byref(null)
    for p in (ctypes.byref(good), ctypes.byref(packed)):
        assert library.rosa_hip_decay_forward(p, n, t, t, 1, 1, 1, 1 << 40, None) == 2
        assert library.rosa_hip_decay_forward(p, t, t, t, None, 1, 1, 1 << 40, None) == 2
        assert library.rosa_hip_decay_backward(p, t, t, t, None, 1, 1, 1, 1, 1, 1 << 40, None) == 2
        assert library.rosa_hip_decay_update(p, t, t, t, 1, None, 1, 1, 1, 1 << 40, None) == 2
        assert library.rosa_hip_window_forward(p, 10, 2, t, t, t, None, None, None) == 2
        assert library.rosa_hip_window_forward(p, 0, 2, t, t, t, 1, None, None) == 1
        assert library.rosa_hip_window_forward(p, 10, 65, t, t, t, 1, None, None) == 1
        assert library.rosa_hip_window_update(p, 10, 2, t, t, t, 1, 1, 11, 1, 1, 1, 1 << 40, None) == 1
        assert library.rosa_hip_window_update(p, 10, 2, t, t, t, 1, 1, 12, None, 1, 1, 1 << 40, None) == 2
        size = library.rosa_hip_window_workspace_bytes(p, 10, 2, 0)
        assert size >= 4 * 200 * 4  # a float per token and head, and the sums of the sinks
        assert library.rosa_hip_window_backward(p, 10, 2, t, t, t, 1, 1, t, 1, 1, 1, 1, size - 1, None) == 3
        assert library.rosa_hip_decay_backward(p, t, t, t, t, 1, 1, 1, 1, 1, 255, None) == 3
        # no gradient is wanted: nothing is launched
        assert library.rosa_hip_decay_backward(p, t, t, t, t, 1, None, None, None, 1, 1 << 40, None) == 0
    assert library.rosa_hip_decay_workspace_bytes(ctypes.byref(good), 3) == 0


def test_c_entries_refuse_misaligned_workspaces():
    library, good = cabi.load(), problem()
    p, t = ctypes.byref(good), ctypes.byref(cabi.RosaMixerTensor(1, 0, 64, 64))
    assert library.rosa_hip_decay_forward(p, t, t, t, 1, 1, 8, 1 << 40, None) == 1
    assert library.rosa_hip_decay_backward(p, t, t, t, t, 1, 1, 1, 1, 8, 1 << 40, None) == 1
    assert library.rosa_hip_decay_update(p, t, t, t, 1, 1, 1, 1, 8, 1 << 40, None) == 1
    assert library.rosa_hip_window_backward(p, 10, 2, t, t, t, 1, 1, t, 1, 1, 1, 8, 1 << 40, None) == 1
    assert library.rosa_hip_window_update(p, 10, 2, t, t, t, 1, 1, 12, 1, 1, 8, 1 << 40, None) == 1
    assert b"16-byte aligned" in library.rosa_hip_last_error()


def test_workspaces_of_extreme_shapes_stay_bounded():
    """States between segments take at most 2 GiB, however many short sequences a call has."""
    library = cabi.load()
    for fields in (dict(B=0, T=0, S=100_000, N=200_000, H=64, Hkv=64, D=128, Dv=128, cu_seqlens=1),
                   dict(B=1, T=2**21, N=2**21, H=16, Hkv=16, D=128, Dv=128),
                   dict(B=0, T=0, S=1, N=2**20, H=128, Hkv=128, D=128, Dv=128, cu_seqlens=1)):
        for call in (0, 1, 2):
            size = library.rosa_hip_decay_workspace_bytes(ctypes.byref(problem(**fields)), call)
            assert 0 < size <= (2 << 30) + 256
    token = problem(B=64, T=1, N=64, H=32, Hkv=8, D=128, Dv=128)
    assert library.rosa_hip_decay_workspace_bytes(ctypes.byref(token), 2) == 256  # unused


def test_every_array_of_a_workspace_begins_on_its_own_256_bytes():
    """Of odd widths too: kernels store four float32 at once, whose address has to be whole."""
    library = cabi.load()
    up = lambda size: (size + 255) // 256 * 256
    p = problem(B=1, T=129, N=129, H=3, Hkv=1, D=7, Dv=12)
    parts = up(129 * 3 * 7 * 4) + up(129 * 3 * 12 * 4)  # (one segment: no states)
    assert library.rosa_hip_decay_workspace_bytes(ctypes.byref(p), 1) == parts
    # 8192 tokens, 4 heads on 1: 128 blocks of 64 keys, whose walk of 8128 tokens is shared by four
    p = problem(B=1, T=8191, N=8191, H=4, Hkv=1, D=7, Dv=11)
    sums = up(4 * 8191 * 7 * 4) + up(4 * 8191 * 11 * 4)
    assert library.rosa_hip_window_workspace_bytes(ctypes.byref(p), 8191, 0, 0) == up(4 * 8191 * 4) + sums


@pytest.mark.parametrize("fields", [
    dict(S=8192, N=65536, H=32, Hkv=32),                       # many short sequences
    dict(S=100_000, N=200_000, H=64, Hkv=64),
    dict(S=100_000, N=200_000, H=64, Hkv=4),
    dict(S=1, N=2**20, H=64, Hkv=8),                           # one that may be long
    dict(B=512, T=2048, N=2**20, H=64, Hkv=8),
    dict(B=2**15, T=40, N=40 * 2**15, H=16, Hkv=1),
])
@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("window,sinks", [(1, 64), (128, 16), (100, 64), (1024, 4)])
def test_workspaces_of_sinks_stay_bounded(fields, dtype, window, sinks):
    """The backward's sums of sinks go by tokens, not by sequences: 2 GiB, or the bytes of queries
    and output gradients in 16 bits; the parts of shared walks take up to 512 blocks of keys."""
    library = cabi.load()
    packed = dict(B=0, T=0, cu_seqlens=1) if "S" in fields else {}
    p = problem(**{**dict(D=128, Dv=128, dtype=dtype), **packed, **fields})
    size = library.rosa_hip_window_workspace_bytes(ctypes.byref(p), window, sinks, 0)
    delta = p.N * p.H * 4
    sums = max(2 << 30, 2 * p.N * p.H * (p.D + p.Dv))
    parts = 512 * 128 * (p.D + p.Dv) * 4
    assert delta <= size <= delta + sums + parts + 4 * 256


def test_the_definitions_agree_with_step_by_step_evaluation():
    """The 64-bit definitions the GPU tests use, against one token at a time."""
    generator = torch.Generator().manual_seed(0)
    randn = lambda *shape: torch.randn(*shape, generator=generator, dtype=torch.float64)
    q, k, v, start = randn(9, 4, 3), randn(9, 2, 3), randn(9, 2, 5), randn(4, 3, 5)
    log_decay = torch.tensor([-0.1, -0.5, 0.0, -2.0])
    output, last = reference.decay(q, k, v, log_decay, state=start)
    state = start.clone()
    for t in range(9):
        for h in range(4):
            state[h] = log_decay[h].double().exp() * state[h] + k[t, h // 2, :, None] * v[t, h // 2]
            assert torch.allclose(output[t, h], 3 ** -0.5 * q[t, h] @ state[h])
    assert torch.allclose(last, state)
    leaves = [x.clone().requires_grad_() for x in (q, k, v)]
    grad = randn(9, 4, 5)
    want = torch.autograd.grad(reference.decay(*leaves, log_decay)[0], leaves, grad)
    got = reference.decay(q, k, v, log_decay, grad_output=grad)
    assert all(torch.allclose(a, b) for a, b in zip(got, want))
    for size, sinks in ((1, 0), (3, 2), (20, 1)):
        output, _, _ = reference.window(q, k, v, size, sinks)
        for t in range(9):
            rows = [s for s in range(t + 1) if t - s < size or s < sinks]
            for h in range(4):
                p = torch.softmax(3 ** -0.5 * k[rows, h // 2] @ q[t, h], 0)
                assert torch.allclose(output[t, h], p @ v[rows, h // 2])
        want = torch.autograd.grad(reference.window(*leaves, size, sinks)[0], leaves, grad)
        got, bounds, _ = reference.window(q, k, v, size, sinks, grad_output=grad)
        assert all(torch.allclose(a, b) for a, b in zip(got, want))
        assert all(bool((a.abs() <= b + 1e-12).all()) for a, b in zip(got, bounds))
