"""The paged cache against its definitions: page tables as lists, attention in 64 bits.

Tolerances: u is half a step of the type (2^-24, 2^-11, 2^-8).  Rounded to the type on the way are each
weight (once, or as the operand that is summed as well) and the result; ``bound`` is the sum of the
absolute terms, so k roundings are k u bound.  What stays in float32 adds its own sums, and a score is
off by as much relative to ``most`` (``float32_slack``).
"""

import itertools
import math

import pytest
import torch

from rosa_soft_amd import paged
from tests import paged_reference as reference
from tests.mixer_reference import HALF_STEP, float32_slack

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
DEVICE = "cuda:0"


def randn(seed, *shape, dtype=torch.float32, scale=1.0):
    generator = torch.Generator(device=DEVICE).manual_seed(seed)
    return (torch.randn(*shape, device=DEVICE, generator=generator) * scale).to(dtype)


def i32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


def offsets_of(lengths):
    return i32([0, *itertools.accumulate(lengths)])


def close(got, want, tolerance, what=""):
    assert got.shape == want.shape, (what, got.shape, want.shape)
    off = (got.double() - want).abs()
    over = off > tolerance
    assert bool(torch.isfinite(got).all()) and not bool(over.any()), (
        what, float((off / tolerance.clamp(min=1e-300)).max()), int(over.sum()), got.numel())


def tolerance_of(dtype, bound, most, tokens, width):
    return (4 * HALF_STEP[dtype] + float32_slack(tokens, width) * (1 + 2 * most)) * bound + 1e-37


# ---------------------------------------------------------------------------
# tables
# ---------------------------------------------------------------------------

def shuffled(seed, count):
    return torch.randperm(count, generator=torch.Generator().manual_seed(seed)).tolist()


def check_tables(want, tables, pool):
    assert tables.tolist() == want.table
    pool = pool.tolist()
    assert pool[0] == want.free
    assert pool[1:1 + want.free] == want.stack[:want.free]


@pytest.mark.parametrize("slots,columns,pages,page,packed", [
    (1, 1, 1, 16, False), (1, 9, 40, 16, True), (3, 4, 20, 64, False), (5, 7, 12, 32, True),
    (70, 11, 300, 16, True), (70, 11, 900, 256, False), (1030, 5, 3000, 16, True), (8192, 3, 9000, 32, False),
    (8192, 2, 20000, 16, True),
])
def test_pages_come_and_go(slots, columns, pages, page, packed):
    """Steps of growth, rejected tokens and ended requests, with pools and tables that run out."""
    generator = torch.Generator().manual_seed(slots)
    random = lambda high: torch.randint(0, high + 1, (slots,), generator=generator).tolist()
    want = reference.Tables(slots, columns, pages, page, order=shuffled(slots, pages))
    tables, pool = want.tensors(DEVICE)
    lengths = [0] * slots
    for step in range(6):
        most = (3, page, 2 * page + 1, 1, 0, 3 * page)[step]
        fresh = random(most) if packed else [most] * slots
        offsets = offsets_of(fresh) if packed else None
        tokens = sum(fresh) if packed else most
        rows = paged.page_tables_update(tables, i32(lengths), pool, offsets, tokens=tokens, page=page)
        assert rows.dtype == torch.int64 and rows.shape == ((tokens,) if packed else (slots, tokens))
        assert rows.flatten().tolist() == [r for part in want.update(lengths, fresh) for r in part]
        check_tables(want, tables, pool)
        after = [n + new for n, new in zip(lengths, fresh)]
        # some requests end, some take back a part of what is new, the others keep all (or more)
        choice = random(3)
        keep = [(0, n + new // 2, n + new, n + new + 5)[c] for c, n, new in zip(choice, lengths, fresh)]
        paged.page_tables_release(tables, i32(after), i32(keep), pool, page=page)
        want.release(after, keep)
        check_tables(want, tables, pool)
        lengths = [min(k, n) for k, n in zip(keep, after)]


def test_rows_of_many_tokens():
    """More than one block writes: the tables are made first."""
    for packed in (False, True):
        fresh = [9000, 1, 0, 20000, 7] if packed else [6001] * 5
        want = reference.Tables(5, 700, 2000, 64, order=shuffled(1, 2000))
        tables, pool = want.tensors(DEVICE)
        lengths = [5, 63, 64, 0, 1000]
        want.update([0] * 5, lengths)
        paged.page_tables_update(tables, i32([0] * 5), pool, offsets_of(lengths), tokens=sum(lengths), page=64)
        rows = paged.page_tables_update(tables, i32(lengths), pool, offsets_of(fresh) if packed else None,
                                         tokens=sum(fresh) if packed else 6001, page=64)
        assert rows.flatten().tolist() == [r for part in want.update(lengths, fresh) for r in part]
        check_tables(want, tables, pool)


def test_a_release_takes_back_an_update():
    want = reference.Tables(4, 30, 100, 16, order=shuffled(2, 100))
    tables, pool = want.tensors(DEVICE)
    paged.page_tables_update(tables, i32([0] * 4), pool, offsets_of([40, 0, 16, 1]), tokens=57, page=16)
    before = tables.clone(), pool.clone()
    lengths = i32([40, 0, 16, 1])
    paged.page_tables_update(tables, lengths, pool, tokens=200, page=16)
    assert not torch.equal(tables, before[0])
    paged.page_tables_release(tables, lengths + 200, lengths, pool, page=16)
    assert torch.equal(tables, before[0]) and torch.equal(pool, before[1])


def test_pools_and_tables_that_hold_nonsense():
    """Numbers that are no page are passed over, none leaves the pool or the tables."""
    pages, page, guard = 6, 16, 64
    whole = torch.full((guard + pages + 1 + guard,), 12345, dtype=torch.int32, device=DEVICE)
    pool = whole[guard:guard + pages + 1]
    pool.copy_(i32([2**31 - 1, 3, -5, 2, 99, 1, 0]))   # more free pages than there are
    tables = torch.full((2, 3), -1, dtype=torch.int32, device=DEVICE)
    rows = paged.page_tables_update(tables, i32([-7, 0]), pool, tokens=40, page=page)
    assert tables.tolist() == [[0, 1, 99], [2, -5, 3]] and pool[0].item() == 0
    assert rows[0].tolist() == [*range(32), *[-1] * 8]
    assert rows[1].tolist() == [*range(32, 48), *[-1] * 16, *range(48, 56)]
    paged.page_tables_release(tables, i32([40, 2**31 - 1]), i32([-3, 0]), pool, page=page)
    assert pool.tolist()[:5] == [4, 3, 2, 1, 0] and tables.tolist() == [[-1] * 3] * 2
    # pages that come back twice have no place
    tables.copy_(i32([[0, 1, 2], [3, 4, 5]]))
    paged.page_tables_release(tables, i32([48, 48]), i32([0, 0]), pool, page=page)
    assert pool.tolist() == [6, 3, 2, 1, 0, 5, 4]
    pool[0] = -9
    paged.page_tables_update(tables, i32([0, 0]), pool, tokens=1, page=page)
    assert tables[:, 0].tolist() == [-1, -1] and pool[0].item() == 0
    assert bool((whole[:guard] == 12345).all()) and bool((whole[-guard:] == 12345).all())


@pytest.mark.parametrize("offsets", [[1, 3, 5], [0, 4, 3], [0, 3, 4], [0, -1, 5], [0, 6, 5]])
def test_invalid_offsets_change_no_table(offsets):
    tables, pool = reference.Tables(2, 4, 9, 16).tensors(DEVICE)
    before = tables.clone(), pool.clone()
    rows = paged.page_tables_update(tables, i32([0, 0]), pool, i32(offsets), tokens=5, page=16)
    assert rows.tolist() == [-1] * 5
    assert torch.equal(tables, before[0]) and torch.equal(pool, before[1])
    many = i32([0, 20000, 17000])
    rows = paged.page_tables_update(tables, i32([0, 0]), pool, many, tokens=20000, page=16)
    assert bool((rows == -1).all()) and torch.equal(tables, before[0])


# ---------------------------------------------------------------------------
# a server of one layer
# ---------------------------------------------------------------------------

class Server:
    """Tables, pages and bounds of some slots, whose streams of tokens are known from the start."""

    def __init__(self, seed, totals, H, Hkv, D, Dv, page, dtype, columns=None, spare=3, bounds=True):
        self.page, self.dtype, self.slots = page, dtype, len(totals)
        most = max(totals)
        columns = -(-most // page) + 1 if columns is None else columns
        pages = sum(-(-n // page) for n in totals) + spare
        self.pages = pages
        order = [0] + [n + 1 for n in shuffled(seed, pages - 1)]   # page 0 is among the spare ones
        self.tables, self.pool = reference.Tables(self.slots, columns, pages, page, order=order).tensors(DEVICE)
        self.lengths = torch.zeros(self.slots, dtype=torch.int32, device=DEVICE)
        self.seen = [0] * self.slots
        # what no token has been put on is NaN and stays unread
        self.caches = [torch.full((pages, Hkv, page, width), math.nan, dtype=dtype, device=DEVICE)
                       for width in (D, Dv)]
        self.bounds = torch.full((pages, Hkv, 2, D), math.nan, dtype=dtype, device=DEVICE) if bounds else None
        self.streams = [[randn(seed + 10 * s, n, H, D, dtype=dtype), randn(seed + 10 * s + 1, n, Hkv, D, dtype=dtype),
                         randn(seed + 10 * s + 2, n, Hkv, Dv, dtype=dtype)] for s, n in enumerate(totals)]

    def step(self, fresh, packed, count=None):
        """Outputs of every slot's new tokens."""
        parts = [[stream[i][at:at + n] for stream, at, n in zip(self.streams, self.seen, fresh)] for i in range(3)]
        if packed:
            offsets, tokens = offsets_of(fresh), sum(fresh)
            inputs = [torch.cat(part) for part in parts]
        else:
            offsets, tokens = None, fresh[0]
            inputs = [torch.stack(part) for part in parts]
        rows = paged.page_tables_update(self.tables, self.lengths, self.pool, offsets, tokens=tokens, page=self.page)
        where = self.tables, rows, self.lengths, offsets
        if count is None:
            output = paged.paged_attention_update(*inputs, *self.caches, *where, key_bounds=self.bounds)
        else:
            output = paged.selected_attention_update(*inputs, *self.caches, self.bounds, *where, count=count)
        self.lengths += i32(fresh)
        self.seen = [at + n for at, n in zip(self.seen, fresh)]
        return list(output.split(fresh) if packed else output)

    def held(self, cache, slot):
        """A slot's rows of a cache, ``[tokens, heads, width]``."""
        table = self.tables[slot, :-(-self.seen[slot] // self.page)].long()
        return cache[table].transpose(1, 2).flatten(0, 1)[:self.seen[slot]]

    def check(self, outputs, before, count=None, slots=None):
        for s in range(self.slots) if slots is None else slots:
            q, k, v = self.streams[s]
            past, end = before[s], self.seen[s]
            for cache, stream in zip(self.caches, (k, v)):
                assert torch.equal(self.held(cache, s), stream[:end])
            if self.bounds is not None:
                table = self.tables[s, :-(-end // self.page)].long()
                for g in range(k.shape[1]):
                    assert torch.equal(self.bounds[table, g], reference.bounds_of(k[:end, g], self.page)
                                       if end else self.bounds[table, g])
            if end > past:
                want, bound, most = reference.attention(q[past:end], k[:end], v[:end], past, self.page, count)
                close(outputs[s], want, tolerance_of(self.dtype, bound, most, end, q.shape[-1] + v.shape[-1]), s)


WIDTHS = [(4, 2, 64, 64), (2, 2, 128, 128), (20, 1, 32, 100), (3, 1, 24, 33), (40, 1, 40, 16), (1, 1, 1, 1)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("chunks", [[5, 1, 64, 1, 1, 130, 3], [1, 1, 1, 1], [300, 1, 1, 15, 2], [8, 9, 40]])
@pytest.mark.parametrize("page", [16, 64, 256])
@pytest.mark.parametrize("widths", WIDTHS)
def test_updates_continue_each_other(chunks, page, widths, dtype):
    """Every chunk gives what one pass over the whole sequence gives, the pages hold the tokens, and
    the bounds are those of their keys."""
    server = Server(100, [sum(chunks)] * 2, *widths, page, dtype)
    for chunk in chunks:
        before = list(server.seen)
        server.check(server.step([chunk] * 2, packed=False), before)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("widths", WIDTHS)
@pytest.mark.parametrize("page", [32, 128])
def test_packed_updates_of_everything_at_once(page, widths, dtype):
    chunks = [[3, 0, 100, 1, 200], [0, 0, 1, 1, 1], [70, 5, 0, 64, 16], [1, 1, 1, 1, 1], [2, 260, 33, 0, 5]]
    server = Server(200, [sum(c[s] for c in chunks) for s in range(5)], *widths, page, dtype)
    for fresh in chunks:
        before = list(server.seen)
        server.check(server.step(fresh, packed=True), before)


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("slots", [64, 65, 150, 300])
def test_many_slots(slots, packed):
    """Up to 64 slots a wave looks at all of them, beyond a block does."""
    lengths = [(s * 37) % 90 + 1 for s in range(slots)]
    server = Server(300, [n + 22 for n in lengths], 4, 2, 32, 32, 16, torch.bfloat16)
    for fresh, as_packed in ((lengths, True), ([1] * slots, packed), ([1 + s % 20 for s in range(slots)], True),
                             ([1] * slots, packed)):
        before = list(server.seen)
        server.check(server.step(fresh, as_packed), before, slots=range(0, slots, 7))


@pytest.mark.parametrize("slots", [63, 130, 700])
def test_selected_pages_of_many_packed_slots(slots):
    lengths = [(s * 37) % 150 + 1 for s in range(slots)]
    server = Server(350, [n + 5 for n in lengths], 4, 2, 32, 32, 16, torch.bfloat16)
    for fresh, count in ((lengths, None), ([s % 3 for s in range(slots)], 2), ([1] * slots, 3)):
        before = list(server.seen)
        server.check(server.step(fresh, True, count), before, count, slots=range(0, slots, 13))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("widths,chunk", [((8, 1, 64, 64), 1), ((8, 2, 128, 128), 1), ((8, 2, 128, 128), 6),
                                          ((8, 2, 64, 64), 90), ((6, 2, 48, 80), 20)])
def test_long_caches_are_shared_out(widths, chunk, dtype):
    """Few rows over many keys: portions of all sizes, joined."""
    totals = [20000, 700, 63, 1, 5000]
    server = Server(400, [n + 3 * chunk for n in totals], *widths, 64, dtype, columns=700, bounds=False)
    server.step(totals, packed=True)
    for packed in (False, True, False):
        before = list(server.seen)
        server.check(server.step([chunk] * 5, packed), before)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("page,count", [(16, 1), (16, 7), (32, 3), (64, 2), (16, 1000), (256, 1)])
@pytest.mark.parametrize("widths", [(4, 2, 64, 64), (2, 2, 128, 128), (20, 1, 32, 100), (3, 1, 24, 33), (40, 1, 40, 16)])
def test_selected_pages(page, count, widths, dtype):
    """Prompts in full, then tokens, drafts and packed mixes over the pages that matter most."""
    server = Server(500, [900, 330, 70], *widths, page, dtype)
    server.step([700, 257, 0], packed=True)
    for fresh, packed in (([1] * 3, False), ([5] * 3, False), ([1] * 3, True), ([40, 0, 18], True), ([17] * 3, False)):
        before = list(server.seen)
        server.check(server.step(fresh, packed, count), before, count)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("widths", [(4, 2, 96, 96), (4, 1, 80, 96), (2, 2, 96, 64), (8, 2, 72, 100)])
def test_widths_between_two_tiles(widths, dtype):
    """Columns that no head has are left out of the products of many rows."""
    server = Server(450, [2400, 300], *widths, 32, dtype)
    server.step([2000, 100], packed=True)
    for fresh, packed in (([150, 150], False), ([70, 0], True), ([1, 1], False), ([20, 20], False)):
        before = list(server.seen)
        server.check(server.step(fresh, packed), before)


@pytest.mark.parametrize("fresh", [[1] * 15 + [6], [1] * 15 + [700], [0] * 15 + [1], [130] * 15 + [1]])
def test_packed_single_tokens_beside_a_prompt(fresh):
    """Slots of few rows have their own kernel, or the one of the prompts."""
    totals = [(s * 331) % 3000 + 5 for s in range(16)]
    server = Server(470, [a + b for a, b in zip(totals, fresh)], 8, 1, 64, 64, 16, torch.bfloat16)
    server.step(totals, packed=True)
    before = list(server.seen)
    server.check(server.step(fresh, packed=True), before)


def test_more_scores_than_are_kept_at_once():
    """Tables so wide that the scores of a prompt are made in parts."""
    server = Server(650, [800], 4, 2, 32, 32, 16, torch.float16, columns=70000)
    server.step([500], packed=False)
    before = list(server.seen)
    server.check(server.step([300], packed=False, count=5), before, count=5)


def test_selection_among_many_pages():
    """Thousands of scores, with a count from one to nearly all of them."""
    server = Server(600, [40000], 4, 1, 16, 16, 16, torch.bfloat16, columns=2600)
    server.step([39900], packed=False)
    for count in (1, 63, 255, 1024):
        before = list(server.seen)
        server.check(server.step([2], packed=False, count=count), before, count)


def test_equal_scores_go_to_the_first_pages():
    """Pages with the same keys rank alike; the values tell which were taken."""
    page, pages, count = 16, 12, 4
    keys = randn(1, 1, 2, page, 32, dtype=torch.float16).expand(pages, 2, page, 32).contiguous()
    keys[7] = keys[7] * 40  # larger bounds for any query
    values = torch.zeros(pages, 2, page, 32, dtype=torch.float16, device=DEVICE)
    values += (2.0 ** -torch.arange(pages, device=DEVICE)).view(-1, 1, 1, 1).half()
    bounds = torch.stack([keys.amin(2), keys.amax(2)], dim=2)
    tables = torch.arange(pages, dtype=torch.int32, device=DEVICE).view(1, -1)
    lengths = i32([(pages - 1) * page])
    q = torch.zeros(1, 1, 4, 32, dtype=torch.float16, device=DEVICE)
    q[..., :1] = 2.0 ** -14   # weights of the same size everywhere
    rows = lengths.long().view(1, 1)
    zeros = torch.zeros(1, 1, 2, 32, dtype=torch.float16, device=DEVICE)
    output = paged.selected_attention_update(q, zeros, zeros, keys, values, bounds, tables, rows, lengths, count=count)
    want = sum(2.0 ** -j for j in (0, 1, 2, 7)) * page / (4 * page + 1)
    assert torch.allclose(output.float(), torch.full_like(output.float(), want), rtol=2e-3)


def test_scores_that_are_no_number_rank_first():
    page, pages = 16, 6
    server = Server(700, [pages * page], 2, 1, 32, 32, page, torch.float32)
    server.step([pages * page - 1], packed=False)
    hurt = int(server.tables[0, 2])
    server.caches[0][hurt, 0, 3, 5] = math.nan
    server.bounds[hurt, 0, :, 5] = math.nan
    output, = server.step([1], packed=False, count=1)
    assert bool(torch.isnan(output).all())
    server.caches[0][hurt] = 0.0
    server.seen, server.lengths = [n - 1 for n in server.seen], server.lengths - 1
    output, = server.step([1], packed=False, count=1)
    assert bool(torch.isfinite(output).all())  # it was this page that was taken, and no other


# ---------------------------------------------------------------------------
# what is missing, and what is left alone
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("chunk", [1, 4, 30, 100])
def test_missing_pages_make_nan_of_the_tokens_that_see_them(chunk, dtype):
    """A page number that is none: tokens before it keep their results, whatever lies on page 0."""
    page, totals = 16, [400, 100]
    server = Server(800, [n + chunk for n in totals], 8, 2, 64, 64, page, dtype)
    server.step(totals, packed=True)
    before = list(server.seen)
    pages = server.pages
    rows = paged.page_tables_update(server.tables, server.lengths, server.pool, tokens=chunk, page=page)
    last = (400 + chunk - 1) // page
    server.caches[0][0], server.caches[1][0] = math.nan, math.nan
    inputs = [torch.stack([stream[i][at:at + chunk] for stream, at in zip(server.streams, before)]) for i in range(3)]
    for column, number in ((3, -1), (3, pages), (3, 2**31 - 1), (last, -2**31)):
        tables, caches = server.tables.clone(), [c.clone() for c in server.caches]
        tables[0, column] = number
        output = paged.paged_attention_update(*inputs, *caches, tables, rows, server.lengths)
        visible = [400 + i >= column * page for i in range(chunk)]
        assert [bool(torch.isnan(output[0, i]).all()) for i in range(chunk)] == visible
        assert bool(torch.isfinite(output[1]).all())
        if not all(visible):
            k, v = server.streams[0][1:]
            upto = visible.index(True)
            want, bound, most = reference.attention(inputs[0][0, :upto], k[:400 + upto], v[:400 + upto], 400)
            close(output[0, :upto], want, tolerance_of(dtype, bound, most, 500, 128))


@pytest.mark.parametrize("chunk", [1, 4])
def test_a_missing_page_among_those_to_select_from(chunk):
    """It ranks first: its slot's tokens are NaN, and no others."""
    server = Server(980, [400 + chunk] * 2, 4, 2, 64, 64, 16, torch.bfloat16)
    server.step([400] * 2, packed=True)
    for entry in (-1, server.pages, 2**31 - 1, -2**31):
        tables = server.tables.clone()
        rows = paged.page_tables_update(tables, server.lengths, server.pool.clone(), tokens=chunk, page=16)
        inputs = [torch.stack([stream[i][400:] for stream in server.streams]) for i in range(3)]
        results = []
        for hurt in (False, True):
            if hurt:
                tables[0, 3] = entry
            results.append(paged.selected_attention_update(
                *inputs, *[c.clone() for c in server.caches], server.bounds.clone(), tables, rows,
                server.lengths, count=2))
        assert bool(torch.isnan(results[1][0]).all()) and torch.equal(results[0][1], results[1][1])
        assert bool(torch.isfinite(results[0]).all())


def test_tokens_behind_their_table_are_nan_and_lengths_without_sense_end():
    """A slot that claims two billion tokens walks its table, not them."""
    page, columns = 16, 4
    server = Server(900, [60, 60], 4, 2, 32, 32, page, torch.bfloat16, columns=columns)
    server.step([50, 50], packed=False)
    for chunk in (1, 3, 40):
        inputs = [randn(5 + i, 2, chunk, 4 if i == 0 else 2, 32, dtype=torch.bfloat16) for i in range(3)]
        rows = torch.full((2, chunk), -1, dtype=torch.int64, device=DEVICE)
        for first in (64, 2**31 - 1):
            lengths = i32([first, 50])
            caches = [c.clone() for c in server.caches]
            output = paged.paged_attention_update(*inputs, *caches, server.tables, rows, lengths)
            assert bool(torch.isnan(output[0]).all())
            assert all(torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0)) for a, b in zip(caches, server.caches))
            output = paged.selected_attention_update(*inputs, *caches, server.bounds.clone(), server.tables, rows,
                                                      lengths, count=2)
            assert bool(torch.isnan(output[0]).all())
        negative = paged.paged_attention_update(*inputs, *[c.clone() for c in server.caches], server.tables,
                                                 torch.where(rows < 0, -2**40, rows), i32([-3, -2**31]))
        assert negative.shape == (2, chunk, 4, 32)


@pytest.mark.parametrize("count", [None, 2])
@pytest.mark.parametrize("offsets", [[1, 30, 40], [0, 35, 30], [0, 30, 39], [0, -1, 40], [0, 41, 40], [0, 2**31 - 1, 40]])
def test_invalid_offsets_are_nan_and_leave_the_cache(offsets, count):
    server = Server(1000, [200, 200], 4, 2, 64, 32, 16, torch.float16)
    server.step([100, 90], packed=True)
    inputs = [randn(5 + i, 40, 4 if i == 0 else 2, 64 if i < 2 else 32, dtype=torch.float16) for i in range(3)]
    rows = torch.arange(40, device=DEVICE)
    caches, bounds = [c.clone() for c in server.caches], server.bounds.clone()
    where = server.tables, rows, server.lengths, i32(offsets)
    if count is None:
        output = paged.paged_attention_update(*inputs, *caches, *where, key_bounds=bounds)
    else:
        output = paged.selected_attention_update(*inputs, *caches, bounds, *where, count=count)
    assert bool(torch.isnan(output).all())
    for got, want in zip((*caches, bounds), (*server.caches, server.bounds)):
        assert torch.equal(got.nan_to_num(7.0), want.nan_to_num(7.0))
    # more slots than a wave has lanes
    slots = 70
    tables = server.tables[:1].expand(slots, -1).contiguous()
    bad = torch.arange(slots + 1, dtype=torch.int32, device=DEVICE).clamp(max=40)
    bad[20] = 3
    output = paged.paged_attention_update(*inputs, *caches, tables, rows, server.lengths[:1].expand(slots), bad)
    assert bool(torch.isnan(output).all())
    assert all(torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0)) for a, b in zip(caches, server.caches))


@pytest.mark.parametrize("chunk", [1, 3, 50])
def test_tokens_without_a_row_are_not_stored(chunk):
    """Padding behind a slot's real tokens, rows outside the pool, and rows of pages that nobody has."""
    server = Server(1100, [200, 200], 4, 2, 64, 64, 16, torch.bfloat16)
    server.step([100, 90], packed=True)
    inputs = [randn(5 + i, 2, chunk, 4 if i == 0 else 2, 64, dtype=torch.bfloat16) for i in range(3)]
    for bad in (-1, server.pages * 16, 2**62, -2**62):
        rows = torch.full((2, chunk), bad, dtype=torch.int64, device=DEVICE)
        caches, bounds = [c.clone() for c in server.caches], server.bounds.clone()
        paged.paged_attention_update(*inputs, *caches, server.tables, rows, server.lengths, key_bounds=bounds)
        for got, want in zip((*caches, bounds), (*server.caches, server.bounds)):
            assert torch.equal(got.nan_to_num(7.0), want.nan_to_num(7.0))
    # real tokens in front of padding are as they would be alone
    if chunk > 1:
        rows = paged.page_tables_update(server.tables, server.lengths, server.pool, tokens=chunk, page=16)
        caches = [c.clone() for c in server.caches]
        full = paged.paged_attention_update(*inputs, *[c.clone() for c in caches], server.tables, rows, server.lengths)
        cut = rows.clone()
        cut[:, chunk // 2:] = -1
        part = paged.paged_attention_update(*inputs, *caches, server.tables, cut, server.lengths)
        assert torch.equal(part[:, :chunk // 2], full[:, :chunk // 2])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("widths", [(4, 2, 64, 64), (3, 1, 24, 33), (8, 1, 128, 128), (2, 1, 80, 96)])
@pytest.mark.parametrize("chunk", [1, 2, 6, 30, 200])
@pytest.mark.parametrize("past", [0, 500])
def test_what_is_not_finite_stays_with_those_that_see_it(past, chunk, widths, dtype):
    server = Server(1150, [past + chunk, past // 2 + chunk], *widths, 16, dtype, bounds=False)
    if past:
        server.step([past, past // 2], packed=True)
    rows = paged.page_tables_update(server.tables, server.lengths, server.pool, tokens=chunk, page=16)
    inputs = [torch.stack([stream[i][at:at + chunk] for stream, at in zip(server.streams, server.seen)])
              for i in range(3)]
    where = server.tables, rows, server.lengths
    clean = paged.paged_attention_update(*inputs, *[c.clone() for c in server.caches], *where)
    for what, value in ((1, math.nan), (2, math.inf), (2, math.nan)):
        for token in {0, chunk // 2, chunk - 1}:
            hurt = [t.clone() for t in inputs]
            hurt[what][0, token, 0, -1] = value
            output = paged.paged_attention_update(*hurt, *[c.clone() for c in server.caches], *where)
            group = widths[0] // widths[1]
            assert not bool(torch.isfinite(output[0, token:, :group, -1]).any())
            assert torch.equal(output[0, :token], clean[0, :token])
            assert torch.equal(output[0, :, group:], clean[0, :, group:])
            assert torch.equal(output[1], clean[1])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("count", [None, 2])
def test_padding_that_is_not_finite(count, dtype):
    """A dense batch of prompts of several lengths, padded with what is no number: outputs, pages and
    bounds are those of the real tokens, and so are those of the next step."""
    lengths, most = [70, 33, 1, 48], 70
    server = Server(1160, [n + 1 for n in lengths], 4, 2, 64, 64, 16, dtype)
    padded = []
    for i in range(3):
        batch = torch.full((4, most, *server.streams[0][i].shape[1:]), math.nan, dtype=dtype, device=DEVICE)
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


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("width", [24, 33, 40, 128])
@pytest.mark.parametrize("both", [False, True])
def test_pages_with_a_key_that_is_not_finite(both, width, dtype):
    """Minus infinity in a bound against queries above zero ranks last; who sees no such key is as ever."""
    server = Server(1170, [101], 1, 1, width, width, 16, dtype)
    for stream in (server.streams[0][0], server.streams[0][1]):
        stream.abs_().add_(0.125)
    if both:
        server.streams[0][1][20, 0, -1] = -math.inf    # page 1, whose bounds from above stay finite
    server.streams[0][1][32:48, 0, -1] = -math.inf  # page 2
    server.step([100], True)
    for count in (1, 4):
        rows = paged.page_tables_update(server.tables, server.lengths, server.pool, tokens=1, page=16)
        output = paged.selected_attention_update(
            *(t[100:].unsqueeze(0) for t in server.streams[0]), *[c.clone() for c in server.caches],
            server.bounds.clone(), server.tables, rows, server.lengths, count=count)
        q, k, v = server.streams[0]
        pages = reference.selected(q[100], k[:, 0], 16, count, 100)
        kept = torch.cat([torch.arange(j * 16, min(101, j * 16 + 16), device=DEVICE) for j in pages])
        assert 2 not in pages
        if not bool(torch.isfinite(k[kept]).all()) and not bool(torch.isfinite(output).all()):
            continue    # (a key that is seen may make the output what it is)
        weights = torch.softmax(k[kept, 0].double() @ q[100, 0].double() * width ** -0.5, 0)
        bound = (weights[:, None] * v[kept, 0].double().abs()).sum(0)
        finite = torch.where(torch.isfinite(k[kept, 0]), k[kept, 0], 0).double()
        most = float((finite.abs() @ q[100, 0].double().abs()).max()) * width ** -0.5
        close(output[0, 0, 0], (weights[:, None] * v[kept, 0].double()).sum(0),
              tolerance_of(dtype, bound, most, len(kept), 2 * width))


def test_slots_share_pages_that_nobody_writes():
    """A prompt in common: two tables begin with the same pages."""
    page = 32
    server = Server(1200, [96 + 20, 96 + 20], 4, 2, 64, 64, page, torch.float16)
    server.streams[1] = [torch.cat([a[:96], b[96:]]) for a, b in zip(*server.streams)]
    server.step([96, 0], packed=True)
    server.tables[1, :3] = server.tables[0, :3]
    server.lengths[1], server.seen[1] = 96, 96
    for fresh in ([1, 1], [7, 7], [12, 12]):
        before = list(server.seen)
        server.check(server.step(fresh, packed=False), before)


def test_nobody_brings_a_token():
    server = Server(1300, [40], 4, 2, 32, 32, 16, torch.bfloat16)
    server.step([30], packed=False)
    caches = [c.clone() for c in server.caches]
    empty = [torch.empty(1, 0, h, 32, dtype=torch.bfloat16, device=DEVICE) for h in (4, 2, 2)]
    rows = paged.page_tables_update(server.tables, server.lengths, server.pool, tokens=0, page=16)
    assert rows.shape == (1, 0)
    assert paged.paged_attention_update(*empty, *server.caches, server.tables, rows, server.lengths).shape == (1, 0, 4, 32)
    packed = [t[0] for t in empty]
    assert paged.selected_attention_update(*packed, *server.caches, server.bounds, server.tables, rows[0],
                                            server.lengths, i32([0, 0]), count=1).shape == (0, 4, 32)
    assert all(torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0)) for a, b in zip(caches, server.caches))


# ---------------------------------------------------------------------------
# layouts, streams, graphs
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("chunk", [1, 5, 70])
def test_strides_and_addresses(chunk, dtype):
    """Parts of a fused projection, transposed layouts, odd addresses: the same results."""
    H, Hkv, D, page = 4, 2, 64, 16
    server = Server(1400, [300, 300], H, Hkv, D, D, page, dtype)
    server.step([200, 120], packed=True)
    rows = paged.page_tables_update(server.tables, server.lengths, server.pool, tokens=chunk, page=page)
    fused = randn(3, 2, chunk, H + 2 * Hkv, D, dtype=dtype)
    plain = [t.contiguous() for t in fused.split([H, Hkv, Hkv], dim=2)]
    odd = torch.empty(2 * chunk * 8 * D + 1, dtype=dtype, device=DEVICE)[1:].view(2, chunk, 8, D)
    odd.copy_(fused)
    spread = torch.empty(2, chunk, 8, 2 * D, dtype=dtype, device=DEVICE)[..., ::2].copy_(fused)
    heads_first = fused.transpose(1, 2).contiguous().transpose(1, 2)
    results = []
    for variant in (plain, *(t.split([H, Hkv, Hkv], dim=2) for t in (fused, odd, spread, heads_first))):
        caches = [c.clone() for c in server.caches]
        table = torch.cat([server.tables.flatten(), server.tables.flatten()])[server.tables.numel():].view_as(server.tables)
        output = paged.paged_attention_update(*variant, *caches, table, rows, server.lengths)
        results.append([output, *caches])
    for other in results[1:]:
        assert all(torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0)) for a, b in zip(results[0], other))
    # pages at odd addresses
    moved = [torch.empty(c.numel() + 1, dtype=dtype, device=DEVICE)[1:].view_as(c).copy_(c) for c in server.caches]
    strided = torch.stack([server.lengths, server.lengths], dim=1)[:, 0]
    output = paged.paged_attention_update(*plain, *moved, server.tables, rows, strided)
    assert torch.equal(output, results[0][0])
    assert torch.equal(moved[0].nan_to_num(7.0), results[0][1].nan_to_num(7.0))


def test_results_are_the_same_on_every_run():
    server = Server(1500, [6000, 900, 40], 8, 2, 128, 128, 64, torch.bfloat16)
    server.step([5900, 800, 0], packed=True)
    for chunk in (1, 3, 30):
        rows = paged.page_tables_update(server.tables, server.lengths, server.pool, tokens=chunk, page=64)
        inputs = [randn(5 + i, 3, chunk, 8 if i == 0 else 2, 128, dtype=torch.bfloat16) for i in range(3)]
        where = server.tables, rows, server.lengths
        first = [paged.paged_attention_update(*inputs, *server.caches, *where),
                 paged.selected_attention_update(*inputs, *server.caches, server.bounds, *where, count=5)]
        for _ in range(3):
            again = [paged.paged_attention_update(*inputs, *server.caches, *where),
                     paged.selected_attention_update(*inputs, *server.caches, server.bounds, *where, count=5)]
            assert all(torch.equal(a, b) for a, b in zip(first, again))


def test_rows_beyond_two_billion_elements():
    """Offsets into the pool pass 32 bits."""
    page, D = 128, 128
    pages = 2**31 // (page * D) + 40
    caches = [torch.zeros(pages, 1, page, D, dtype=torch.bfloat16, device=DEVICE) for _ in range(2)]
    bounds = torch.zeros(pages, 1, 2, D, dtype=torch.bfloat16, device=DEVICE)
    tables = i32([[pages - 1, 3, pages - 2], [0, pages - 30, 5]])
    stream = [randn(1 + i, 2, 300, 2 if i == 0 else 1, D, dtype=torch.bfloat16) for i in range(3)]
    position = torch.arange(300, device=DEVICE)
    rows = tables.long()[:, position // page] * page + position % page
    lengths, outputs, at = i32([0, 0]), [], 0
    for chunk, count in ((257, None), (1, None), (40, None), (2, 2)):
        part = [t[:, at:at + chunk] for t in stream]
        where = tables, rows[:, at:at + chunk], lengths
        outputs.append(paged.paged_attention_update(*part, *caches, *where, key_bounds=bounds) if count is None else
                       paged.selected_attention_update(*part, *caches, bounds, *where, count=count))
        lengths += chunk
        at += chunk
    output = torch.cat(outputs, dim=1)
    for s in range(2):
        want, bound, most = reference.attention(*(t[s] for t in stream), 0)
        close(output[s], want, tolerance_of(torch.bfloat16, bound, most, 300, 2 * D))
        assert torch.equal(caches[0].view(-1, D)[rows[s]], stream[1][s, :, 0])


def test_streams_and_graphs():
    """A step of tables and attention on another stream, recorded and replayed; two graphs at once."""
    def build(seed):
        server = Server(seed, [400, 250], 8, 2, 64, 64, 16, torch.bfloat16, spare=80, columns=60)
        server.step([300, 200], packed=True)
        return server

    def step(server, inputs, state):
        tables, pool, lengths = state
        rows = paged.page_tables_update(tables, lengths, pool, tokens=inputs[0].shape[1], page=16)
        full = paged.paged_attention_update(*inputs, *server.caches, tables, rows, lengths, key_bounds=server.bounds)
        few = paged.selected_attention_update(*inputs, *server.caches, server.bounds, tables, rows, lengths, count=4)
        lengths += inputs[0].shape[1]
        return full, few

    for chunk in (1, 2, 24):
        graphs = []
        for seed in (1600, 1700):
            eager, recorded = build(seed), build(seed)
            inputs = [torch.zeros(2, chunk, h, 64, dtype=torch.bfloat16, device=DEVICE) for h in (8, 2, 2)]
            state = recorded.tables, recorded.pool, recorded.lengths
            saved = [t.clone() for t in (*state, *recorded.caches, recorded.bounds)]
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                step(recorded, inputs, state)
            torch.cuda.current_stream().wait_stream(side)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                outputs = step(recorded, inputs, state)
            for tensor, value in zip((*state, *recorded.caches, recorded.bounds), saved):
                tensor.copy_(value)
            graphs.append((graph, inputs, outputs, eager, recorded))
        for replay in range(5):
            wanted = []
            for i, (graph, inputs, outputs, eager, recorded) in enumerate(graphs):
                fresh = [randn(50 + 10 * replay + i + j, *t.shape, dtype=t.dtype) for j, t in enumerate(inputs)]
                for tensor, value in zip(inputs, fresh):
                    tensor.copy_(value)
                wanted.append(step(eager, fresh, (eager.tables, eager.pool, eager.lengths)))
            for graph, *_ in graphs:
                graph.replay()
            torch.cuda.synchronize()
            for (_, _, outputs, eager, recorded), want in zip(graphs, wanted):
                assert all(torch.equal(a, b) for a, b in zip(outputs, want))
                assert torch.equal(recorded.tables, eager.tables) and torch.equal(recorded.pool, eager.pool)
                assert torch.equal(recorded.bounds.nan_to_num(7.0), eager.bounds.nan_to_num(7.0))


def test_two_servers_on_two_streams():
    """Steps of two servers that run at once."""
    totals, plans = [1500, 900, 40], [[700, 1, 30], [2, 5, 1], [1] * 3, [3] * 3, [1] * 3]
    servers = [Server(seed, totals, 8, 2, 64, 64, 16, torch.bfloat16) for seed in (1710, 1750)]
    streams = [torch.cuda.Stream() for _ in servers]
    torch.cuda.synchronize()
    outputs = [[], []]
    for i, fresh in enumerate(plans):
        for server, stream, kept in zip(servers, streams, outputs):
            with torch.cuda.stream(stream):
                kept.append((list(server.seen), fresh, server.step(fresh, len(set(fresh)) > 1, 4 if i > 2 else None)))
    torch.cuda.synchronize()
    for server, kept in zip(servers, outputs):
        for i, (before, fresh, output) in enumerate(kept):
            for s in range(3):
                q, k, v = server.streams[s]
                end = before[s] + fresh[s]
                want, bound, most = reference.attention(q[before[s]:end], k[:end], v[:end], before[s], 16,
                                                        4 if i > 2 else None)
                close(output[s], want, tolerance_of(torch.bfloat16, bound, most, end, 128))


def test_changed_tensors_get_new_versions():
    server = Server(1800, [40], 4, 2, 32, 32, 16, torch.bfloat16)
    watched = server.tables, server.pool, *server.caches, server.bounds
    before = [t._version for t in watched]
    server.step([30], packed=False)
    assert all(t._version > v for t, v in zip(watched, before))
    before = [t._version for t in watched]
    server.step([1], packed=False, count=1)
    assert all(t._version > v for t, v in zip(watched, before))
    before = [t._version for t in watched[:2]]
    paged.page_tables_release(server.tables, server.lengths, server.lengths, server.pool, page=16)
    assert all(t._version > v for t, v in zip(watched, before))
