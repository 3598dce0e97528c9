"""The paged cache where its uses meet.  Tolerances as in ``test_gpu_paged``."""

import math

import pytest
import torch

from rosa_soft_amd import paged
from tests import paged_reference as reference
from tests.test_gpu_paged import (DEVICE, DTYPES, Server, check_tables, close, i32, offsets_of, randn,
                                  shuffled, tolerance_of)

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


# ---------------------------------------------------------------------------
# pages that several slots hold
# ---------------------------------------------------------------------------

def release(want, lengths, keep):
    """A release of ``want``'s tables in which a page that a slot keeps stays with it, and a page that
    several slots give back goes back once."""
    columns = [(want.columns_of(min(max(k, 0), max(n, 0))), want.columns_of(n)) for n, k in zip(lengths, keep)]
    kept = {entry for row, (begin, _) in zip(want.table, columns) for entry in row[:begin]}
    for slot in reversed(range(len(want.table))):
        begin, end = columns[slot]
        for column in reversed(range(begin, end)):
            entry, want.table[slot][column] = want.table[slot][column], -1
            if 0 <= entry < want.pages and entry not in kept:
                kept.add(entry)
                if want.free < want.pages:
                    want.stack[want.free:want.free + 1] = [entry]
                want.free = min(want.free + 1, want.pages)


def share(server, giver, taker, tokens):
    """A prompt in common: the taker's table begins with the giver's pages."""
    columns = tokens // server.page
    assert tokens % server.page == 0 and server.seen[taker] == 0
    server.tables[taker, :columns] = server.tables[giver, :columns]
    server.lengths[taker], server.seen[taker] = tokens, tokens


def free_pages(pool):
    pool = pool.tolist()
    return pool[1:1 + pool[0]]


@pytest.mark.parametrize("ends", [0, 1])
@pytest.mark.parametrize("keep", [0, 40])
def test_a_page_that_another_slot_keeps_stays_with_it(ends, keep):
    """One of two slots with a prompt in common ends, or goes back into it; a third takes the pages
    on top of the stack; the other one's pages and outputs are as they were."""
    page, prompt = 16, 96
    stays = 1 - ends
    server = Server(2100, [prompt + 30, prompt + 30, 400], 4, 2, 64, 64, page, torch.bfloat16,
                    bounds=False)
    server.streams[1] = [torch.cat([a[:prompt], b[prompt:]]) for a, b in zip(*server.streams[:2])]
    server.step([prompt, 0, 0], packed=True)
    share(server, 0, 1, prompt)
    server.step([10, 20, 0], packed=True)
    kept = [keep if s == ends else n for s, n in enumerate(server.seen)]
    paged.page_tables_release(server.tables, server.lengths, i32(kept), server.pool, page=page)
    server.seen[ends] = keep
    server.lengths[ends] = keep
    free = free_pages(server.pool)
    held = server.tables[stays, :-(-server.seen[stays] // page)].tolist()
    assert len(free) == len(set(free)) and not set(free) & set(held)
    server.step([0, 0, min(400, len(free) * page)], packed=True)
    before = list(server.seen)
    fresh = [0, 0, 0]
    fresh[stays] = min(10, page - before[stays] % page)
    server.check(server.step(fresh, packed=True), before)
    # and when all of them have ended every page is free, once
    paged.page_tables_release(server.tables, server.lengths, i32([0] * 3), server.pool, page=page)
    assert sorted(free_pages(server.pool)) == list(range(server.pages))
    assert bool((server.tables == -1).all())


def test_slots_with_a_prompt_in_common_end_at_once():
    """Their pages go back once, in an order that does not depend on the run."""
    page, slots = 16, 300
    pools = []
    for _ in range(3):
        want = reference.Tables(slots, 20, 4000, page, order=shuffled(7, 4000))
        tables, pool = want.tensors(DEVICE)
        paged.page_tables_update(tables, i32([0] * slots), pool, offsets_of([160] + [0] * (slots - 1)),
                                 tokens=160, page=page)
        tables[1:, :10] = tables[:1, :10]
        lengths = i32([160] * slots)
        paged.page_tables_update(tables, lengths, pool, tokens=40, page=page)
        paged.page_tables_release(tables, lengths + 40, lengths * 0, pool, page=page)
        assert bool((tables == -1).all())
        free = free_pages(pool)
        assert sorted(free) == list(range(4000))
        pools.append(free)
    assert pools[0] == pools[1] == pools[2]


@pytest.mark.parametrize("slots,columns,pages,page", [
    (2, 3, 9, 16), (5, 40, 90, 32), (64, 70, 3000, 16), (300, 30, 5000, 16), (1500, 9, 4000, 64), (7, 3000, 9000, 16),
    (40, 50, 300000, 16), (8192, 4, 140000, 16), (3, 2, 131073, 16),
    (40, 50, 1200000, 16), (3, 2, 2**19 + 1, 16),
])
def test_releases_of_shared_pages_are_those_of_lists(slots, columns, pages, page):
    """Any page in any number of tables, what is kept and what goes at random."""
    generator = torch.Generator().manual_seed(slots)
    random = lambda high, count=slots: torch.randint(0, high + 1, (count,), generator=generator).tolist()
    for step in range(4):
        want = reference.Tables(slots, columns, pages, page, order=[], free=0)
        few = (3, columns, pages - 1, pages - 1)[step]   # of which most slots have the same, or hardly any
        spread = random(min(few, pages - 1), slots * columns)
        if step == 3:   # and numbers that are no page
            spread = [(n, -1, pages, -2**31, 2**31 - 1)[c] for n, c in zip(spread, random(4, slots * columns))]
        want.table = [spread[s * columns:(s + 1) * columns] for s in range(slots)]
        tables, pool = want.tensors(DEVICE)
        lengths = random(columns * page + 40)
        keep = [(0, n // 3, n, n + 9)[c] for n, c in zip(lengths, random(3))]
        paged.page_tables_release(tables, i32(lengths), i32(keep), pool, page=page)
        release(want, lengths, keep)
        check_tables(want, tables, pool)


def test_a_release_of_shared_pages_in_a_graph():
    page, slots = 16, 5
    build = lambda: reference.Tables(slots, 8, 60, page, order=shuffled(8, 60))
    lengths = i32([100, 100, 50, 100, 0])
    keep = i32([0, 100, 0, 32, 0])
    want = build()
    tables, pool = want.tensors(DEVICE)
    saved = tables.clone(), pool.clone()

    def step():
        paged.page_tables_update(tables, lengths * 0, pool, offsets_of([100, 0, 0, 0, 0]), tokens=100, page=page)
        tables[1:4] = tables[:1]
        paged.page_tables_release(tables, lengths, keep, pool, page=page)

    step()
    result = tables.clone(), pool.clone()
    graph = torch.cuda.CUDAGraph()
    recorded = i32([0, 100, 100, 100, 100, 100])
    tables.copy_(saved[0]), pool.copy_(saved[1])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=side):
        paged.page_tables_update(tables, lengths * 0, pool, recorded, tokens=100, page=page)
        tables[1:4] = tables[:1]
        paged.page_tables_release(tables, lengths, keep, pool, page=page)
    for _ in range(4):
        tables.copy_(saved[0]), pool.copy_(saved[1])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(tables, result[0]) and torch.equal(pool, result[1])
    assert sorted(free_pages(pool) + tables[1, :7].tolist()) == list(range(60))


# ---------------------------------------------------------------------------
# bounds that are infinite
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("width", [24, 33, 40, 128])
@pytest.mark.parametrize("share", [1, 4, 6])
@pytest.mark.parametrize("bound", [math.inf, -math.inf])
def test_a_query_of_zero_and_an_infinite_bound_are_no_number(bound, share, width, dtype):
    """Their product, whichever of the two bounds it is: the page ranks first, and makes NaN of the
    token that sees it; the other heads' tokens have their own pages."""
    server = Server(2200, [101], 2 * share, 2, width, width, 16, dtype)
    for column in {0, width // 2, width - 1}:
        server.caches = [torch.full_like(c, math.nan) for c in server.caches]
        server.bounds = torch.full_like(server.bounds, math.nan)
        server.tables, server.pool = reference.Tables(1, 8, server.pages, 16).tensors(DEVICE)
        server.lengths, server.seen = i32([0]), [0]
        q, k, v = server.streams[0] = [randn(2201 + i, 101, 2 * share if i == 0 else 2, width, dtype=dtype)
                                       for i in range(3)]
        k[35, 0, column] = bound             # on page 2
        q[100, share - 1, column] = 0.0      # one member of the group
        server.step([100], True)
        output, = server.step([1], False, count=1)
        pages = reference.selected(q[100, :share], k[:, 0], 16, 1, 100)
        assert pages[0] == 2
        assert bool(torch.isnan(output[0, share - 1]).all())
        want, terms, most = reference.attention(q[100:, share:], k[:, 1:], v[:, 1:], 100, 16, 1)
        close(output[:, share:], want, tolerance_of(dtype, terms, most, 101, 2 * width))


# ---------------------------------------------------------------------------
# steps that are undone
# ---------------------------------------------------------------------------

def test_a_step_that_ran_out_of_pages_is_undone_and_done_again():
    page = 16
    want = reference.Tables(3, 10, 12, page, order=shuffled(3, 12))
    tables, pool = want.tensors(DEVICE)
    lengths = [40, 70, 30]
    paged.page_tables_update(tables, i32([0] * 3), pool, offsets_of(lengths), tokens=sum(lengths), page=page)
    want.update([0] * 3, lengths)
    rows = paged.page_tables_update(tables, i32(lengths), pool, tokens=30, page=page)
    assert bool((rows == -1).any()) and pool[0].item() == 0
    paged.page_tables_release(tables, i32(lengths) + 30, i32(lengths), pool, page=page)
    check_tables(want, tables, pool)
    # a request ends, and the step has room
    paged.page_tables_release(tables, i32(lengths), i32([40, 0, 30]), pool, page=page)
    want.release(lengths, [40, 0, 30])
    rows = paged.page_tables_update(tables, i32([40, 0, 30]), pool, tokens=30, page=page)
    assert rows.tolist() == want.update([40, 0, 30], [30] * 3)
    assert bool((rows >= 0).all())
    check_tables(want, tables, pool)


def test_a_step_of_which_a_part_is_kept_loses_no_page():
    """A dense step whose tokens are not all real: the rest's pages are given back before the next."""
    page, slots, step = 16, 4, 40
    want = reference.Tables(slots, 30, 60, page, order=shuffled(4, 60))
    tables, pool = want.tensors(DEVICE)
    lengths = [0] * slots
    for real in ([40, 1, 0, 17], [3, 40, 16, 15], [0, 0, 40, 1]):
        rows = paged.page_tables_update(tables, i32(lengths), pool, tokens=step, page=page)
        assert rows.tolist() == want.update(lengths, [step] * slots)
        upto, lengths = [n + step for n in lengths], [n + r for n, r in zip(lengths, real)]
        paged.page_tables_release(tables, i32(upto), i32(lengths), pool, page=page)
        want.release(upto, lengths)
        check_tables(want, tables, pool)
        held = [entry for row in tables.tolist() for entry in row if entry >= 0]
        assert len(held) == sum(-(-n // page) for n in lengths)
        assert sorted(held + free_pages(pool)) == list(range(60))


# ---------------------------------------------------------------------------
# many slots whose tiles are cut
# ---------------------------------------------------------------------------

MIXED = [(lambda s: 1, False), (lambda s: 3, False), (lambda s: 6, False), (lambda s: s % 2, True),
         (lambda s: (0, 1, 5, 90)[s % 4], True), (lambda s: 0 if s % 10 else 70, True)]


@pytest.mark.parametrize("widths", [(8, 2, 64, 64), (6, 2, 40, 33)])
@pytest.mark.parametrize("slots", [64, 65, 130, 300])
def test_long_and_short_caches_of_many_slots(slots, widths):
    """Single tokens, drafts and packed mixes for slots of a few or thousands of tokens, among them
    slots without new ones: every slot against the definition."""
    lengths = [3000 + 7 * s if s % 10 == 0 else 0 if s % 10 == 3 else (s * 37) % 90 + 1 for s in range(slots)]
    totals = [n + sum(fresh(s) for fresh, _ in MIXED) for s, n in enumerate(lengths)]
    server = Server(2300, totals, *widths, 16, torch.bfloat16, columns=400, bounds=False)
    server.step(lengths, packed=True)
    for fresh, packed in MIXED:
        before = list(server.seen)
        server.check(server.step([fresh(s) for s in range(slots)], packed), before)


@pytest.mark.parametrize("totals,steps", [
    ([(s * 37) % 60 + 25 for s in range(2500)], [lambda s: s % 25, lambda s: 1, lambda s: 0 if s % 50 else 20]),
    ([30000, 3, 20000], [lambda s: (29000, 0, 17)[s], lambda s: (5, 1, 19000)[s]]),
])
def test_bounds_of_many_pages_in_packed_calls(totals, steps):
    """More pages that new tokens touch than blocks run at once."""
    slots = len(totals)
    server = Server(2400, totals, 4, 4, 32, 32, 16, torch.bfloat16)
    for fresh in steps:
        before = list(server.seen)
        output = server.step([fresh(s) for s in range(slots)], packed=True)
        if slots > 3:
            server.check(output, before, slots=range(0, slots, 41))
    for s in range(0, slots, 41 if slots > 3 else 1):
        end, table = server.seen[s], server.tables[s, :-(-server.seen[s] // 16)].long()
        for cache, stream in zip(server.caches, server.streams[s][1:]):
            assert torch.equal(server.held(cache, s), stream[:end])
        for g in range(4):
            assert torch.equal(server.bounds[table, g], reference.bounds_of(server.streams[s][1][:end, g], 16))


def test_batches_of_calls_are_refused():
    """``torch.vmap`` has no rule for operators that change their arguments."""
    server = Server(2500, [40], 4, 2, 32, 32, 16, torch.bfloat16)
    server.step([30], packed=False)
    inputs = [randn(5 + i, 3, 1, 1, 4 if i == 0 else 2, 32, dtype=torch.bfloat16) for i in range(3)]
    rows = torch.full((1, 1), -1, dtype=torch.int64, device=DEVICE)
    before = [c.clone() for c in (*server.caches, server.bounds)]
    where = server.tables, rows, server.lengths
    for call in (lambda *x: paged.paged_attention_update(*x, *server.caches, *where),
                 lambda *x: paged.paged_attention_update(*x, *server.caches, *where, key_bounds=server.bounds),
                 lambda *x: paged.selected_attention_update(*x, *server.caches, server.bounds, *where, count=1)):
        with pytest.raises(RuntimeError, match="[Bb]atching rule"):
            torch.vmap(call)(*inputs)
    for got, want in zip((*server.caches, server.bounds), before):
        assert torch.equal(got.nan_to_num(7.0), want.nan_to_num(7.0))
