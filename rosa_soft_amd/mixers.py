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
differentiable and in reverse mode alone (dual tensors are refused), and like that of
``rosa_soft`` the backward cannot be recorded into a HIP graph; everything else can.

The ``_update`` forms serve slots, like ``RosaRuntime.update``: a chunk of one or more tokens per
slot (or a packed chunk with ``cu_seqlens``, in which slots may bring none) on top of the slots'
states or caches, which are advanced in place.  They have no backward.  One token for every slot is
fastest dense: packed it runs as a chunk, whose blocks walk a slot's window alone.

Invalid device ``cu_seqlens`` cannot be seen without a synchronisation: they make every output and
gradient NaN and leave states and caches as they were.  States and caches share no memory with the
inputs, and the updates count a version of them.

A row that is not finite makes NaN of every result that depends on it, and may do so to others near
those, because masked weights of a tile are zeros that multiply its rows.  With ``decay_attention``
these are results of up to 63 tokens before the row (values in outputs, keys in the gradients of
queries) or behind it (queries and output gradients in those of keys and values).  With
``window_attention`` they are up to 127 tokens away on either side, among outputs for values, among
gradients for all inputs, and the gradients of a sequence's first 64 keys and values where there are
sinks.  What is farther away, and other sequences, keep their results.
"""

from __future__ import annotations

import math
import operator
from typing import Optional

import torch
from torch import Tensor

from . import _BUILD_HINT, _raise_unavailable, BUILD_CAPABILITIES

__all__ = [
    "decay_attention",
    "decay_attention_update",
    "decay_attention_varlen",
    "window_attention",
    "window_attention_update",
    "window_attention_varlen",
]

_GRADIENT_BITS = (1, 2, 4)  # query, key, value
_INT64_MAX = 2**63 - 1


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
    def _(query, key, value, cu_seqlens, log_decay, scale=None):
        return _fake_output(query, value)

    @register("rosa_soft::decay_attention_vjp")
    def _(query, key, value, cu_seqlens, log_decay, grad_output, scale, gradient_mask):
        return _fake_gradients(query, key, value, gradient_mask)

    @register("rosa_soft::decay_attention_update")
    def _(query, key, value, cu_seqlens, log_decay, state, scale=None):
        return _fake_output(query, value)

    @register("rosa_soft::decay_attention_update_out")
    def _(query, key, value, cu_seqlens, log_decay, state, state_out, scale=None):
        return _fake_output(query, value)

    @register("rosa_soft::window_attention")
    def _(query, key, value, cu_seqlens, window, sinks, scale=None, want_log_sum=False):
        tokens = math.prod(query.shape[:-2])
        shape = (query.shape[-2], tokens) if want_log_sum else (0,)
        return _fake_output(query, value), query.new_empty(shape, dtype=torch.float32)

    @register("rosa_soft::window_attention_vjp")
    def _(query, key, value, cu_seqlens, output, log_sum, grad_output, window, sinks, scale,
          gradient_mask):
        return _fake_gradients(query, key, value, gradient_mask)

    @register("rosa_soft::window_attention_update")
    def _(query, key, value, key_cache, value_cache, lengths, cu_seqlens, window, sinks,
          scale=None):
        return _fake_output(query, value)


def _unavailable(*args, **kwargs):
    _raise_unavailable("rosa_soft mixer", _BUILD_HINT)


# The operators check their arguments themselves (ValueError and TypeError as everywhere in this
# package) and carry their autograd, so that a call costs little more than its launches.
if BUILD_CAPABILITIES.rosa_soft_cuda:
    _register_fakes()
    _decay = torch.ops.rosa_soft.decay_attention.default
    _decay_update = torch.ops.rosa_soft.decay_attention_update.default
    _decay_update_out = torch.ops.rosa_soft.decay_attention_update_out.default
    _window = torch.ops.rosa_soft.window_attention.default
    _window_update = torch.ops.rosa_soft.window_attention_update.default
else:
    _decay = _decay_update = _decay_update_out = _window = _window_update = _unavailable


def _integer(name: str, value) -> int:
    if isinstance(value, bool):
        raise TypeError(f"{name} must be an integer")
    try:
        return max(-1, min(operator.index(value), _INT64_MAX))
    except TypeError as error:
        raise TypeError(f"{name} must be an integer") from error


def _number(name: str, value) -> Optional[float]:
    if value is None or type(value) is float:
        return value
    if isinstance(value, bool):
        raise TypeError(f"{name} must be a number")
    return float(value)


# ---------------------------------------------------------------------------
# linear attention with a decay for each head
# ---------------------------------------------------------------------------

def decay_attention(query: Tensor, key: Tensor, value: Tensor, log_decay: Tensor, *,
                    scale: Optional[float] = None) -> Tensor:
    """Causal linear attention whose memory decays at a rate of each head.

    ``S_t = exp(log_decay) S_{t-1} + k_t v_t^T`` and ``o_t = scale q_t^T S_t``, from ``S = 0``.
    ``query`` is ``(B, T, H, D)``, ``key`` ``(B, T, Hkv, D)`` and ``value`` ``(B, T, Hkv, Dv)`` with
    ``H % Hkv == 0``; ``log_decay`` is float32 ``(H,)``, zero or negative (``-inf`` forgets
    everything but the token itself), and takes no gradient.  ``scale`` defaults to ``D ** -0.5``.
    Returns ``(B, T, H, Dv)``.
    """

    return _decay(query, key, value, None, log_decay, _number("scale", scale))


def decay_attention_varlen(query: Tensor, key: Tensor, value: Tensor, cu_seqlens: Tensor,
                           log_decay: Tensor, *, scale: Optional[float] = None) -> Tensor:
    """``decay_attention`` applied independently to sequences packed along dim 0.

    ``cu_seqlens`` is a device int32 tensor of ``S + 1`` cumulative offsets.
    """

    return _decay(query, key, value, cu_seqlens, log_decay, _number("scale", scale))


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

    scale = _number("scale", scale)
    if state_out is None or state_out is state:
        return _decay_update(query, key, value, cu_seqlens, log_decay, state, scale)
    return _decay_update_out(query, key, value, cu_seqlens, log_decay, state, state_out, scale)


# ---------------------------------------------------------------------------
# attention with a sliding window and sinks
# ---------------------------------------------------------------------------

def _masks(window, sinks):
    # (integers that the operators do not take at all are cut to ones that they refuse, or to an
    # endless window)
    if type(window) is int and type(sinks) is int and 0 <= window <= _INT64_MAX >= sinks >= 0:
        return window, sinks
    return _integer("window", window), _integer("sinks", sinks)


def _window_attention(query, key, value, cu_seqlens, window, sinks, scale) -> Tensor:
    window, sinks = _masks(window, sinks)
    return _window(query, key, value, cu_seqlens, window, sinks, _number("scale", scale))[0]


def window_attention(query: Tensor, key: Tensor, value: Tensor, *, window: int, sinks: int = 0,
                     scale: Optional[float] = None) -> Tensor:
    """Causal softmax attention over the last ``window`` tokens and the first ``sinks`` ones.

    Token ``t`` sees token ``s <= t`` when ``t - s < window`` or ``s < sinks``; a window as long
    as the sequence is full causal attention.  ``query`` is ``(B, T, H, D)``, ``key``
    ``(B, T, Hkv, D)`` and ``value`` ``(B, T, Hkv, Dv)`` with ``H % Hkv == 0``; ``sinks`` is at most
    64 and ``scale`` defaults to ``D ** -0.5``.  Returns ``(B, T, H, Dv)``.
    """

    return _window_attention(query, key, value, None, window, sinks, scale)


def window_attention_varlen(query: Tensor, key: Tensor, value: Tensor, cu_seqlens: Tensor, *,
                            window: int, sinks: int = 0, scale: Optional[float] = None) -> Tensor:
    """``window_attention`` applied independently to sequences packed along dim 0.

    ``cu_seqlens`` is a device int32 tensor of ``S + 1`` cumulative offsets.
    """

    return _window_attention(query, key, value, cu_seqlens, window, sinks, scale)


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

    window, sinks = _masks(window, sinks)
    return _window_update(query, key, value, key_cache, value_cache, lengths, cu_seqlens, window,
                          sinks, _number("scale", scale))
