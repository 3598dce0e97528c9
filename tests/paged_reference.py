"""The paged cache from its definitions: the pool as a Python list, attention in 64 bits."""

import math

import torch

from tests.mixer_reference import repeated


def ceil(a, b):
    return -(-a // b)


class Tables:
    """Page tables of lists, as a server without a GPU would keep them."""

    def __init__(self, slots, columns, pages, page, order=None, free=None):
        self.columns, self.pages, self.page = columns, pages, page
        self.stack = list(range(pages) if order is None else order)   # the top is the last one
        self.free = len(self.stack) if free is None else free
        self.table = [[-1] * columns for _ in range(slots)]

    def columns_of(self, tokens):
        return min(ceil(max(tokens, 0), self.page), self.columns)

    def row(self, slot, position):
        column = position // self.page
        entry = self.table[slot][column] if column < self.columns else -1
        return entry * self.page + position % self.page if 0 <= entry < self.pages else -1

    def update(self, lengths, fresh):
        """Rows of the new tokens, slot by slot."""
        for slot, (n, new) in enumerate(zip(lengths, fresh)):
            n = max(n, 0)
            for column in range(self.columns_of(n), self.columns_of(n + new)):
                if self.free > 0:
                    self.free -= 1
                    self.table[slot][column] = self.stack[self.free]
                else:
                    self.table[slot][column] = -1
        return [[self.row(slot, max(n, 0) + i) for i in range(new)]
                for slot, (n, new) in enumerate(zip(lengths, fresh))]

    def release(self, lengths, keep):
        for slot in reversed(range(len(self.table))):
            n = max(lengths[slot], 0)
            kept = self.columns_of(min(max(keep[slot], 0), n))
            for column in reversed(range(kept, self.columns_of(n))):
                entry, self.table[slot][column] = self.table[slot][column], -1
                if 0 <= entry < self.pages:
                    if self.free < self.pages:
                        self.stack[self.free:self.free + 1] = [entry]
                    self.free = min(self.free + 1, self.pages)

    def tensors(self, device):
        pool = torch.full((self.pages + 1,), -7, dtype=torch.int32)
        pool[0] = self.free
        pool[1:1 + len(self.stack)] = torch.tensor(self.stack, dtype=torch.int32)
        return (torch.tensor(self.table, dtype=torch.int32, device=device), pool.to(device))


def bounds_of(keys, page):
    """Least and largest elements of the pages of one head, ``[pages, 2, D]``."""
    return torch.stack([torch.stack([part.amin(0), part.amax(0)]) for part in keys.split(page)])


def selected(query, keys, page, count, position):
    """Pages that a token of a group of query rows sees: its own and the best of those before."""
    own = position // page
    bounds = bounds_of(keys[:position + 1], page).double()[:own]
    q = query.double()[:, None]
    score = torch.maximum(q * bounds[None, :, 0], q * bounds[None, :, 1]).sum(-1)
    score = torch.nan_to_num(score.amax(0), nan=math.inf)
    return sorted(sorted(range(own), key=lambda j: (-float(score[j]), j))[:count]) + [own]


def attention(query, key, value, past, page=None, count=None):
    """One slot: keys and values of all ``past + T`` tokens, queries of the last ``T``; the output, the
    sum of the absolute terms, and the most of ``scale sum |q||k|``."""
    heads, scale = query.shape[-2], query.shape[-1] ** -0.5
    shared = key.shape[-2]
    q, k, v = (repeated(x, heads).transpose(0, 1) for x in (query, key, value))
    t = torch.arange(past, past + q.shape[1], device=query.device)[:, None]
    seen = torch.arange(k.shape[1], device=query.device)[None, :] <= t
    seen = seen.expand(heads, *seen.shape).clone()
    if count is not None:
        for i in range(q.shape[1]):
            for g in range(shared):
                members = slice(g * (heads // shared), (g + 1) * (heads // shared))
                pages = selected(query[i, members], key[:, g], page, count, past + i)
                kept = torch.zeros(k.shape[1], dtype=torch.bool, device=query.device)
                for j in pages:
                    kept[j * page:(j + 1) * page] = True
                seen[members, i] &= kept
    scores = (q @ k.transpose(1, 2) * scale).masked_fill(~seen, -math.inf)
    p = torch.softmax(scores, -1)
    most = float((q.abs() @ k.abs().transpose(1, 2) * scale).max())
    back = lambda x: x.transpose(0, 1)
    return back(p @ v), back(p @ v.abs()), most
