"""Mixers that stand beside ``rosa_soft`` in a model's blocks, in training and in serving.

``rosa_soft`` answers with one exact, far match.  A block that uses it carries what a suffix
match cannot in other mixers over the same tokens and slots:

* ``decay_attention``: linear attention with a decay for each head, a running summary of all
  tokens so far in a state of fixed size;
* ``window_attention``: softmax attention over the last ``window`` tokens and a few first tokens
  (sinks) that stay visible.

Both take the layouts of ``rosa_soft``: dense ``(B, T, heads, width)`` or, in the ``_varlen``
forms, ``(N, heads, width)`` with device ``cu_seqlens``; heads of keys and values may be shared by
groups of query heads; dtypes float32, float16 and bfloat16, head widths 1 to 128.  Inputs may be
strided (the parts of a fused projection) as long as the elements of a head are neighbours;
others are copied.  Gradients come in the dtype of their input, the same on every run, once
differentiable, and like that of ``rosa_soft`` the backward cannot be recorded into a HIP graph;
everything else can.

The ``_update`` forms serve slots, like ``RosaRuntime.update``: a chunk of one or more tokens per
slot (or a packed chunk with ``cu_seqlens``, in which slots may bring none) on top of the slots'
states or caches, which are advanced in place.  They have no backward.

Invalid device ``cu_seqlens`` cannot be seen without a synchronisation: they make every output and
gradient NaN and leave states and caches as they were.  A row of values that is not finite makes
the outputs NaN of every token that sees it, and may do so for up to 63 tokens before it.
"""

from __future__ import annotations

import math
import operator
from typing import Optional

import torch
from torch import Tensor
from torch.autograd.function import once_differentiable

__all__ = [
    "decay_attention",
    "decay_attention_update",
    "decay_attention_varlen",
    "window_attention",
    "window_attention_update",
    "window_attention_varlen",
]

MAX_HEAD_WIDTH = 128
MAX_SINKS = 64

_DEVICE_DTYPES = (torch.float32, torch.float16, torch.bfloat16)
_GRADIENT_BITS = (1, 2, 4)  # query, key, value
_INT32_MAX = 2**31 - 1


# ---------------------------------------------------------------------------
# argument checks
# ---------------------------------------------------------------------------

def _require(condition: bool, message: str) -> None:
    if not condition:
        raise ValueError(message)


def _integer(name: str, value) -> int:
    if isinstance(value, bool):
        raise TypeError(f"{name} must be an integer")
    try:
        return operator.index(value)
    except TypeError as error:
        raise TypeError(f"{name} must be an integer") from error


def _check_inputs(name: str, query: Tensor, key: Tensor, value: Tensor,
                  cu_seqlens: Optional[Tensor], empty: bool = False) -> None:
    rank = 4 if cu_seqlens is None else 3
    layout = "(B, T, heads, width)" if cu_seqlens is None else "(N, heads, width)"
    tensors = (query, key, value)
    _require(all(t.ndim == rank for t in tensors), f"query, key, and value must have shape {layout}")
    lead = [tuple(t.shape[:-2]) for t in tensors]
    _require(lead[0] == lead[1] == lead[2], "all inputs must share their token dimensions")
    _require(key.size(-2) == value.size(-2), "key and value head counts must match")
    _require(query.size(-2) >= 1 and key.size(-2) >= 1, "query and key must have at least one head")
    _require(query.size(-2) % key.size(-2) == 0, "query heads must be divisible by key heads")
    _require(query.size(-1) == key.size(-1), "query and key widths must match")
    _require(1 <= query.size(-1) <= MAX_HEAD_WIDTH and 1 <= value.size(-1) <= MAX_HEAD_WIDTH,
             f"head widths must be in [1, {MAX_HEAD_WIDTH}]")
    if empty:
        _require(cu_seqlens is not None or query.size(0) >= 1, "an update needs at least one slot")
    else:
        _require(all(size >= 1 for size in lead[0]), "batch and sequence dimensions must be >= 1")
    _require(query.device == key.device == value.device, "all inputs must be on the same device")
    _require(query.dtype == key.dtype == value.dtype, "all inputs must have the same dtype")
    if cu_seqlens is not None:
        _require(cu_seqlens.device == query.device,
                 "all inputs and cu_seqlens must be on the same device")
        _require(cu_seqlens.dtype == torch.int32, "cu_seqlens must have dtype int32")
        _require(cu_seqlens.ndim == 1 and cu_seqlens.numel() >= 2,
                 "cu_seqlens must be a one-dimensional int32 tensor")
    _require(query.is_cuda, f"{name} requires CUDA tensors")
    _require(query.dtype in _DEVICE_DTYPES, f"{name} supports float32, float16, and bfloat16")


def _check_scale(scale: Optional[float], width: int) -> float:
    if scale is None:
        return width ** -0.5
    limits = torch.finfo(torch.float32)
    _require(not isinstance(scale, bool) and math.isfinite(float(scale))
             and limits.tiny <= float(scale) <= limits.max,
             "scale must be representable as a positive normal float32 value")
    return float(scale)


def _check_log_decay(log_decay: Tensor, query: Tensor) -> None:
    _require(log_decay.ndim == 1 and log_decay.size(0) == query.size(-2),
             "log_decay must have one entry per query head")
    _require(log_decay.dtype == torch.float32, "log_decay must have dtype float32")
    _require(log_decay.device == query.device,
             "all inputs and log_decay must be on the same device")
    if log_decay.requires_grad and torch.is_grad_enabled():
        raise ValueError("log_decay is a constant of each head and takes no gradient: detach it")


def _check_window(window: int, sinks: int):
    window, sinks = _integer("window", window), _integer("sinks", sinks)
    _require(window >= 1, "window must be >= 1")
    _require(0 <= sinks <= MAX_SINKS, f"sinks must be in [0, {MAX_SINKS}]")
    return min(window, _INT32_MAX), sinks


def _needs_backward(*tensors: Tensor) -> bool:
    return torch.is_grad_enabled() and any(tensor.requires_grad for tensor in tensors)


def _refuse_training_capture(name: str) -> None:
    if torch.compiler.is_compiling():  # tracing: nothing is being launched
        return
    if torch.cuda.is_current_stream_capturing():
        raise RuntimeError(
            f"{name}: the backward cannot be recorded into a HIP graph in this build; capture "
            "the forward under torch.no_grad() or run the training step eagerly"
        )


def _refuse_gradients(name: str, *tensors: Tensor) -> None:
    if _needs_backward(*tensors):
        raise RuntimeError(f"{name} has no backward: call it under torch.no_grad()")


# ---------------------------------------------------------------------------
# shape functions for FakeTensor / torch.compile tracing
# ---------------------------------------------------------------------------

def _fake_output(query: Tensor, value: Tensor) -> Tensor:
    return query.new_empty((*query.shape[:-1], value.shape[-1]))


def _fake_gradients(query: Tensor, key: Tensor, value: Tensor, gradient_mask: int):
    return tuple(
        tensor.new_empty(tensor.shape if gradient_mask & bit else (0,))
        for bit, tensor in zip(_GRADIENT_BITS, (query, key, value))
    )


def _register_fakes() -> None:
    register = torch.library.register_fake

    @register("rosa_soft::decay_attention")
    def _(query, key, value, cu_seqlens, log_decay, scale):
        return _fake_output(query, value)

    @register("rosa_soft::decay_attention_vjp")
    def _(query, key, value, cu_seqlens, log_decay, grad_output, scale, gradient_mask):
        return _fake_gradients(query, key, value, gradient_mask)

    @register("rosa_soft::decay_attention_update")
    def _(query, key, value, cu_seqlens, log_decay, state, scale):
        return _fake_output(query, value)

    @register("rosa_soft::decay_attention_update_out")
    def _(query, key, value, cu_seqlens, log_decay, state, state_out, scale):
        return _fake_output(query, value)

    @register("rosa_soft::window_attention")
    def _(query, key, value, cu_seqlens, window, sinks, scale, want_log_sum):
        tokens = math.prod(query.shape[:-2])
        shape = (query.shape[-2], tokens) if want_log_sum else (0,)
        return _fake_output(query, value), query.new_empty(shape, dtype=torch.float32)

    @register("rosa_soft::window_attention_vjp")
    def _(query, key, value, cu_seqlens, output, log_sum, grad_output, window, sinks, scale,
          gradient_mask):
        return _fake_gradients(query, key, value, gradient_mask)

    @register("rosa_soft::window_attention_update")
    def _(query, key, value, key_cache, value_cache, lengths, cu_seqlens, window, sinks, scale):
        return _fake_output(query, value)


def _device_operators() -> bool:
    from . import BUILD_CAPABILITIES

    return BUILD_CAPABILITIES.rosa_soft_cuda


def _require_device_operators(name: str) -> None:
    if not _device_operators():
        from . import _BUILD_HINT, _raise_unavailable

        _raise_unavailable(name, _BUILD_HINT)


if _device_operators():
    _register_fakes()


# ---------------------------------------------------------------------------
# autograd nodes
# ---------------------------------------------------------------------------

def _gradient_mask(needs) -> int:
    return sum(bit for bit, need in zip(_GRADIENT_BITS, needs[:3]) if need)


def _requested(gradients, needs):
    return tuple(gradient if need else None for gradient, need in zip(gradients, needs[:3]))


class _DecayAttention(torch.autograd.Function):

    @staticmethod
    def forward(ctx, query, key, value, cu_seqlens, log_decay, scale):
        ctx.scale = scale
        ctx.save_for_backward(query, key, value, cu_seqlens, log_decay)
        return torch.ops.rosa_soft.decay_attention(query, key, value, cu_seqlens, log_decay, scale)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_output):
        query, key, value, cu_seqlens, log_decay = ctx.saved_tensors
        gradients = torch.ops.rosa_soft.decay_attention_vjp(
            query, key, value, cu_seqlens, log_decay, grad_output, ctx.scale,
            _gradient_mask(ctx.needs_input_grad),
        )
        return (*_requested(gradients, ctx.needs_input_grad), None, None, None)


class _WindowAttention(torch.autograd.Function):

    @staticmethod
    def forward(ctx, query, key, value, cu_seqlens, window, sinks, scale):
        output, log_sum = torch.ops.rosa_soft.window_attention(
            query, key, value, cu_seqlens, window, sinks, scale, True
        )
        ctx.controls = (window, sinks, scale)
        ctx.save_for_backward(query, key, value, cu_seqlens, output, log_sum)
        return output

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_output):
        query, key, value, cu_seqlens, output, log_sum = ctx.saved_tensors
        gradients = torch.ops.rosa_soft.window_attention_vjp(
            query, key, value, cu_seqlens, output, log_sum, grad_output, *ctx.controls,
            _gradient_mask(ctx.needs_input_grad),
        )
        return (*_requested(gradients, ctx.needs_input_grad), None, None, None, None)


# ---------------------------------------------------------------------------
# linear attention with a decay for each head
# ---------------------------------------------------------------------------

def _decay_attention(name, query, key, value, cu_seqlens, log_decay, scale) -> Tensor:
    _require_device_operators(name)
    _check_inputs(name, query, key, value, cu_seqlens)
    _check_log_decay(log_decay, query)
    scale = _check_scale(scale, query.size(-1))
    if not _needs_backward(query, key, value):
        return torch.ops.rosa_soft.decay_attention(query, key, value, cu_seqlens, log_decay, scale)
    _refuse_training_capture(name)
    return _DecayAttention.apply(query, key, value, cu_seqlens, log_decay.detach(), scale)


def decay_attention(query: Tensor, key: Tensor, value: Tensor, log_decay: Tensor, *,
                    scale: Optional[float] = None) -> Tensor:
    """Causal linear attention whose memory decays at a rate of each head.

    ``S_t = exp(log_decay) S_{t-1} + k_t v_t^T`` and ``o_t = scale q_t^T S_t``, from ``S = 0``.
    ``query`` is ``(B, T, H, D)``, ``key`` ``(B, T, Hkv, D)`` and ``value`` ``(B, T, Hkv, Dv)`` with
    ``H % Hkv == 0``; ``log_decay`` is float32 ``(H,)``, zero or negative (``-inf`` forgets
    everything but the token itself), and takes no gradient.  ``scale`` defaults to ``D ** -0.5``.
    Returns ``(B, T, H, Dv)``.
    """

    return _decay_attention("decay_attention", query, key, value, None, log_decay, scale)


def decay_attention_varlen(query: Tensor, key: Tensor, value: Tensor, cu_seqlens: Tensor,
                           log_decay: Tensor, *, scale: Optional[float] = None) -> Tensor:
    """``decay_attention`` applied independently to sequences packed along dim 0.

    ``cu_seqlens`` is a device int32 tensor of ``S + 1`` cumulative offsets.
    """

    return _decay_attention("decay_attention_varlen", query, key, value, cu_seqlens, log_decay, scale)


def decay_attention_update(query: Tensor, key: Tensor, value: Tensor, log_decay: Tensor,
                           state: Tensor, cu_seqlens: Optional[Tensor] = None, *,
                           scale: Optional[float] = None,
                           state_out: Optional[Tensor] = None) -> Tensor:
    """New tokens of every slot on top of the slots' states; no backward.

    ``query`` is ``(slots, T, H, D)``, or ``(N, H, D)`` with ``cu_seqlens`` of ``slots + 1`` offsets.
    ``state`` is float32 ``(slots, H, D, Dv)``, zeros for a fresh slot, and is advanced in place;
    with ``state_out`` (of the same shape) the new states go there and ``state`` is left as it is.
    Returns the outputs of the new tokens.
    """

    name = "decay_attention_update"
    _require_device_operators(name)
    _check_inputs(name, query, key, value, cu_seqlens, empty=True)
    _check_log_decay(log_decay, query)
    scale = _check_scale(scale, query.size(-1))
    _refuse_gradients(name, query, key, value, state)
    slots = query.size(0) if cu_seqlens is None else cu_seqlens.numel() - 1
    shape = (slots, query.size(-2), query.size(-1), value.size(-1))
    for tensor in (state,) if state_out is None else (state, state_out):
        _require(tuple(tensor.shape) == shape,
                 "state must have shape (slots, heads, key width, value width)")
        _require(tensor.dtype == torch.float32, "state must have dtype float32")
        _require(tensor.device == query.device, "all inputs and state must be on the same device")
        _require(tensor.is_contiguous(), "state must be contiguous")
    operators = torch.ops.rosa_soft
    if state_out is None or state_out is state:
        return operators.decay_attention_update(query, key, value, cu_seqlens, log_decay, state,
                                                scale)
    return operators.decay_attention_update_out(query, key, value, cu_seqlens, log_decay, state,
                                                state_out, scale)


# ---------------------------------------------------------------------------
# attention with a sliding window and sinks
# ---------------------------------------------------------------------------

def _window_attention(name, query, key, value, cu_seqlens, window, sinks, scale) -> Tensor:
    _require_device_operators(name)
    _check_inputs(name, query, key, value, cu_seqlens)
    window, sinks = _check_window(window, sinks)
    scale = _check_scale(scale, query.size(-1))
    if not _needs_backward(query, key, value):
        return torch.ops.rosa_soft.window_attention(
            query, key, value, cu_seqlens, window, sinks, scale, False)[0]
    _refuse_training_capture(name)
    return _WindowAttention.apply(query, key, value, cu_seqlens, window, sinks, scale)


def window_attention(query: Tensor, key: Tensor, value: Tensor, *, window: int, sinks: int = 0,
                     scale: Optional[float] = None) -> Tensor:
    """Causal softmax attention over the last ``window`` tokens and the first ``sinks`` ones.

    Token ``t`` sees token ``s <= t`` when ``t - s < window`` or ``s < sinks``; a window as long
    as the sequence is full causal attention.  ``query`` is ``(B, T, H, D)``, ``key``
    ``(B, T, Hkv, D)`` and ``value`` ``(B, T, Hkv, Dv)`` with ``H % Hkv == 0``; ``sinks`` is at most
    64 and ``scale`` defaults to ``D ** -0.5``.  Returns ``(B, T, H, Dv)``.
    """

    return _window_attention("window_attention", query, key, value, None, window, sinks, scale)


def window_attention_varlen(query: Tensor, key: Tensor, value: Tensor, cu_seqlens: Tensor, *,
                            window: int, sinks: int = 0, scale: Optional[float] = None) -> Tensor:
    """``window_attention`` applied independently to sequences packed along dim 0.

    ``cu_seqlens`` is a device int32 tensor of ``S + 1`` cumulative offsets.
    """

    return _window_attention("window_attention_varlen", query, key, value, cu_seqlens, window, sinks,
                             scale)


def window_attention_update(query: Tensor, key: Tensor, value: Tensor, key_cache: Tensor,
                            value_cache: Tensor, lengths: Tensor,
                            cu_seqlens: Optional[Tensor] = None, *, window: int, sinks: int = 0,
                            scale: Optional[float] = None) -> Tensor:
    """New tokens of every slot on top of the slots' caches; no backward.

    ``query`` is ``(slots, T, H, D)``, or ``(N, H, D)`` with ``cu_seqlens`` of ``slots + 1`` offsets.
    The caches are contiguous ``(slots, Hkv, capacity, width)`` of the inputs' dtype with
    ``capacity >= sinks + window``: position ``p`` lies on row ``p`` for ``p < sinks`` and on row
    ``sinks + (p - sinks) % (capacity - sinks)`` otherwise, so that a slot of any length fits.
    ``lengths`` is a device int32 tensor of the tokens that each slot has seen.  The new tokens
    attend to what their slot holds and to each other, and are then put on their rows;
    ``lengths`` is left to the caller, who advances it once for all layers of a model:
    ``lengths += T``.  Returns the outputs of the new tokens.
    """

    name = "window_attention_update"
    _require_device_operators(name)
    _check_inputs(name, query, key, value, cu_seqlens, empty=True)
    window, sinks = _check_window(window, sinks)
    scale = _check_scale(scale, query.size(-1))
    _refuse_gradients(name, query, key, value, key_cache, value_cache)
    slots = query.size(0) if cu_seqlens is None else cu_seqlens.numel() - 1
    for cache, tensor in ((key_cache, key), (value_cache, value)):
        _require(cache.ndim == 4 and cache.size(0) == slots and cache.size(1) == tensor.size(-2)
                 and cache.size(2) == key_cache.size(2) and cache.size(3) == tensor.size(-1),
                 "caches must have shape (slots, key heads, capacity, width)")
        _require(cache.dtype == query.dtype, "caches must have the dtype of the inputs")
        _require(cache.device == query.device, "all inputs and caches must be on the same device")
        _require(cache.is_contiguous(), "caches must be contiguous")
    _require(window + sinks <= key_cache.size(2) <= _INT32_MAX,
             "caches must hold the sinks and the window, and fewer than 2^31 tokens")
    _require(lengths.ndim == 1 and lengths.size(0) == slots and lengths.dtype == torch.int32,
             "lengths must be an int32 tensor with one entry per slot")
    _require(lengths.device == query.device, "all inputs and lengths must be on the same device")
    return torch.ops.rosa_soft.window_attention_update(
        query, key, value, key_cache, value_cache, lengths, cu_seqlens, window, sinks, scale)
