"""The mixers in 64 bits, from their definitions, and how far 32-bit and 16-bit arithmetic may be off.

A bound is the answer with every term replaced by its absolute value: a relative error of each
term, and of each rounded intermediate, is at most that error times the bound.
"""

import math

import torch

HALF_STEP = {torch.float32: 2.0**-24, torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}


def float32_slack(*sums):
    """Relative error of float32 sums of that many terms: six standard deviations of a random walk
    of half steps."""
    return 6 * math.sqrt(sum(sums) + 16) * 2.0**-24


def repeated(tensor, heads):
    return tensor.double().repeat_interleave(heads // tensor.shape[-2], dim=-2)


def group_sum(tensor, shared):
    return tensor.unflatten(-2, (shared, -1)).sum(-2)


def decay(query, key, value, log_decay, state=None, grad_output=None, absolute=False):
    """One sequence: ``[T, heads, width]``.  The output and the state behind it, or the gradients."""
    heads, scale = query.shape[-2], query.shape[-1] ** -0.5
    q, k, v = (repeated(t, heads).transpose(0, 1) for t in (query, key, value))
    go = None if grad_output is None else grad_output.double().transpose(0, 1)
    if absolute:
        q, k, v = q.abs(), k.abs(), v.abs()
        go = None if go is None else go.abs()
        state = None if state is None else state.abs()
    tokens = q.shape[1]
    rate = torch.exp(log_decay.double()).view(-1, 1, 1)
    t = torch.arange(tokens, device=query.device)
    apart = (t[:, None] - t[None, :])
    weight = torch.where(apart >= 0, rate ** apart.clamp(min=0).double(), 0.0)
    scores = torch.matmul(q, k.transpose(1, 2)) * weight * scale
    if go is not None:
        utility = torch.matmul(go, v.transpose(1, 2)) * weight * scale
        shared = key.shape[-2]
        back = lambda x: x.transpose(0, 1)
        return (back(utility @ k), group_sum(back(utility.transpose(1, 2) @ q), shared),
                group_sum(back(scores.transpose(1, 2) @ go), shared))
    output = scores @ v
    last = (k * rate ** (tokens - 1 - t).double().view(1, -1, 1)).transpose(1, 2) @ v
    if state is not None:
        output = output + scale * (rate ** (t + 1).double().view(1, -1, 1)) * (q @ state.double())
        last = last + rate ** float(tokens) * state.double()
    return output.transpose(0, 1), last


def visible(t, s, window, sinks):
    return (s <= t) & ((t - s < window) | (s < sinks))


def window(query, key, value, window, sinks, grad_output=None, past=0):
    """One sequence: keys and values of all ``past + T`` tokens, queries of the last ``T``.

    ``(output, bound)`` or ``(gradients, bounds)``, and the most of ``scale sum |q||k|``.
    """
    heads, scale = query.shape[-2], query.shape[-1] ** -0.5
    q, k, v = (repeated(x, heads).transpose(0, 1) for x in (query, key, value))
    t = torch.arange(past, past + q.shape[1], device=query.device)[:, None]
    s = torch.arange(k.shape[1], device=query.device)[None, :]
    seen = visible(t, s, window, sinks)
    # (a token that nobody sees stays out of every sum, whatever it holds)
    hidden = ~seen.any(0)
    k, v = (torch.where(hidden.view(1, -1, 1), 0.0, x) for x in (k, v))
    scores = (q @ k.transpose(1, 2) * scale).masked_fill(~seen, -math.inf)
    p = torch.softmax(scores, -1)
    most = float((q.detach().abs() @ k.detach().abs().transpose(1, 2) * scale).max())
    output, bound = p @ v, p @ v.abs()
    back = lambda x: x.transpose(0, 1)
    if grad_output is None:
        return back(output), back(bound), most
    go, shared = grad_output.double().transpose(0, 1), key.shape[-2]
    slope = p * (go @ v.transpose(1, 2) - (go * output).sum(-1, keepdim=True)) * scale
    steep = p * (go.abs() @ v.abs().transpose(1, 2) + (go.abs() * bound).sum(-1, keepdim=True)) * scale
    sums = lambda x: group_sum(back(x), shared)
    gradients = (back(slope @ k), sums(slope.transpose(1, 2) @ q), sums(p.transpose(1, 2) @ go))
    bounds = (back(steep @ k.abs()), sums(steep.transpose(1, 2) @ q.abs()),
              sums(p.transpose(1, 2) @ go.abs()))
    return gradients, bounds, most
