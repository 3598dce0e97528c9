"""The paged cache where its uses meet.  Tolerances as in ``test_gpu_paged``."""

import math

import pytest
import torch

from rosa_soft_amd import paged
from tests.test_gpu_paged import DEVICE, DTYPES, Server, i32, offsets_of

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------------------
# what a token does not see
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("widths", [(4, 2, 64, 64), (3, 1, 24, 33), (8, 1, 128, 128)])
@pytest.mark.parametrize("chunk", [2, 6, 30, 200])
@pytest.mark.parametrize("past", [0, 500])
def test_later_tokens_leave_every_bit_of_earlier_ones(past, chunk, widths, dtype):
    """Keys and values of later tokens, ordinary, large or infinite: rows that do not see them share
    tiles and waves with rows that do, and no rounding."""
    server = Server(1900, [past + chunk, past // 2 + chunk], *widths, 16, dtype, bounds=False)
    if past:
        server.step([past, past // 2], packed=True)
    rows = paged.page_tables_update(server.tables, server.lengths, server.pool, tokens=chunk, page=16)
    inputs = [torch.stack([stream[i][at:at + chunk] for stream, at in zip(server.streams, server.seen)])
              for i in range(3)]
    where = server.tables, rows, server.lengths
    first = paged.paged_attention_update(*inputs, *[c.clone() for c in server.caches], *where)
    for factor in (-1.0, 30.0, math.inf):
        for token in {1, chunk // 2, chunk - 1}:
            later = [t.clone() for t in inputs]
            for tensor in later:
                tensor[0, token:] *= factor
            output = paged.paged_attention_update(*later, *[c.clone() for c in server.caches], *where)
            assert torch.equal(output[0, :token], first[0, :token])
            assert torch.equal(output[1], first[1])


# ---------------------------------------------------------------------------
# the largest finite numbers
# ---------------------------------------------------------------------------

# in float32 the first of a number's three bfloat16 parts is infinite from 2^128 - 2^119 on
EXTREMES = {torch.float32: [2.0**128 - 2.0**104, 2.0**128 - 2.0**119, 2.0**128 - 2.0**119 - 2.0**104],
            torch.float16: [65504.0], torch.bfloat16: [2.0**128 - 2.0**120]}
CASES = [(dtype, sign * value) for dtype, values in EXTREMES.items() for value in values for sign in (-1.0, 1.0)]


@pytest.mark.parametrize("dtype,value", CASES)
@pytest.mark.parametrize("count", [None, 2])
def test_padding_of_the_largest_numbers(count, dtype, value):
    """A dense batch of prompts padded with the lowest or the largest finite value."""
    lengths, most = [70, 33, 1, 48], 70
    server = Server(2000, [n + 1 for n in lengths], 4, 2, 64, 64, 16, dtype)
    padded = []
    for i in range(3):
        batch = torch.full((4, most, *server.streams[0][i].shape[1:]), value, dtype=dtype, device=DEVICE)
        assert bool(torch.isfinite(batch).all())
        for s, n in enumerate(lengths):
            batch[s, :n] = server.streams[s][i][:n]
        padded.append(batch)
    packed_rows = paged.page_tables_update(server.tables, server.lengths, server.pool, offsets_of(lengths),
                                           tokens=sum(lengths), page=16)
    rows = torch.full((4, most), -1, dtype=torch.int64, device=DEVICE)
    for s, part in enumerate(packed_rows.split(lengths)):
        rows[s, :lengths[s]] = part
    where = server.tables, rows, server.lengths
    if count is None:
        output = paged.paged_attention_update(*padded, *server.caches, *where, key_bounds=server.bounds)
    else:
        output = paged.selected_attention_update(*padded, *server.caches, server.bounds, *where, count=count)
    server.lengths += i32(lengths)
    server.seen = list(lengths)
    server.check([output[s, :n] for s, n in enumerate(lengths)], [0] * 4, count)
    server.check(server.step([1] * 4, False, count), lengths, count)


@pytest.mark.parametrize("dtype,value", CASES)
@pytest.mark.parametrize("widths", [(4, 2, 64, 64), (3, 1, 24, 33), (8, 1, 128, 128)])
@pytest.mark.parametrize("chunk", [2, 6, 30, 200])
@pytest.mark.parametrize("past", [0, 500])
def test_the_largest_numbers_stay_with_those_that_see_them(past, chunk, widths, dtype, value):
    server = Server(2050, [past + chunk, past // 2 + chunk], *widths, 16, dtype, bounds=False)
    if past:
        server.step([past, past // 2], packed=True)
    rows = paged.page_tables_update(server.tables, server.lengths, server.pool, tokens=chunk, page=16)
    inputs = [torch.stack([stream[i][at:at + chunk] for stream, at in zip(server.streams, server.seen)])
              for i in range(3)]
    where = server.tables, rows, server.lengths
    clean = paged.paged_attention_update(*inputs, *[c.clone() for c in server.caches], *where)
    group = widths[0] // widths[1]
    for what in (1, 2):
        for token in {chunk // 2, chunk - 1}:
            hurt = [t.clone() for t in inputs]
            hurt[what][0, token, 0, -1] = value
            output = paged.paged_attention_update(*hurt, *[c.clone() for c in server.caches], *where)
            assert torch.equal(output[0, :token], clean[0, :token])
            assert torch.equal(output[0, :, group:], clean[0, :, group:])
            assert torch.equal(output[1], clean[1])
