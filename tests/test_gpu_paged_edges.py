"""The paged cache where its uses meet.  Tolerances as in ``test_gpu_paged``."""

import math

import pytest
import torch

from rosa_soft_amd import paged
from tests.test_gpu_paged import DTYPES, Server

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
