"""The paged cache without a GPU: argument checks, schemas, fake tensors, C entry points, the definitions."""

import ctypes
import inspect
import re

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from rosa_soft_amd import cabi, paged
from tests import paged_reference as reference


def fake(*shape, dtype=torch.bfloat16, device="cuda"):
    return torch.empty(*shape, dtype=dtype, device=device)


def host(*shape, dtype=torch.bfloat16):
    return torch.zeros(*shape, dtype=dtype)


I32, I64 = dict(dtype=torch.int32), dict(dtype=torch.int64)


def arguments(make=host, **changes):
    """Dense calls that pass every check but that of the device; ``changes`` replace parts."""
    parts = dict(q=make(2, 5, 4, 16), k=make(2, 5, 2, 16), v=make(2, 5, 2, 8),
                 keys=make(9, 2, 32, 16), values=make(9, 2, 32, 8), bounds=make(9, 2, 2, 16),
                 tables=make(2, 4, **I32), rows=make(2, 5, **I64), lengths=make(2, **I32),
                 pool=make(10, **I32), keep=make(2, **I32), tokens=5, page=32, count=2, offsets=None)
    parts.update(changes)
    return parts


def calls(p):
    cache = p["q"], p["k"], p["v"], p["keys"], p["values"]
    where = p["tables"], p["rows"], p["lengths"], p["offsets"]
    extra = {"scale": p["scale"]} if "scale" in p else {}
    return {
        "paged": lambda: paged.paged_attention_update(*cache, *where, **extra),
        "bounds": lambda: paged.paged_attention_update(*cache, *where, key_bounds=p["bounds"], **extra),
        "selected": lambda: paged.selected_attention_update(*cache, p["bounds"], *where,
                                                             count=p["count"], **extra),
        "update": lambda: paged.page_tables_update(p["tables"], p["lengths"], p["pool"], p["offsets"],
                                                    tokens=p["tokens"], page=p["page"]),
        "release": lambda: paged.page_tables_release(p["tables"], p["lengths"], p["keep"], p["pool"],
                                                      page=p["page"]),
    }


ATTENTION, TABLES = ("paged", "bounds", "selected"), ("update", "release")


def test_calls_that_pass_give_outputs_of_the_right_shape():
    with FakeTensorMode():
        made = {name: call() for name, call in calls(arguments(fake)).items()}
        for name in ATTENTION:
            assert made[name].shape == (2, 5, 4, 8) and made[name].dtype == torch.bfloat16, name
        assert made["update"].shape == (2, 5) and made["update"].dtype == torch.int64
        assert made["release"] is None
        packed = arguments(fake, q=fake(7, 4, 16), k=fake(7, 2, 16), v=fake(7, 2, 8),
                           rows=fake(7, **I64), offsets=fake(3, **I32), tokens=7)
        made = {name: call() for name, call in calls(packed).items()}
        assert all(made[name].shape == (7, 4, 8) for name in ATTENTION)
        assert made["update"].shape == (7,)


@pytest.mark.parametrize("names,changes,error,message", [
    (ATTENTION, lambda: dict(q=host(5, 4, 16)), ValueError, "must have shape"),
    (ATTENTION, lambda: dict(k=host(2, 6, 2, 16)), ValueError, "share their token dimensions"),
    (ATTENTION, lambda: dict(v=host(2, 5, 1, 8)), ValueError, "key and value head counts"),
    (ATTENTION, lambda: dict(q=host(2, 5, 3, 16)), ValueError, "divisible by key heads"),
    (ATTENTION, lambda: dict(q=host(2, 5, 4, 129), k=host(2, 5, 2, 129)), ValueError, r"\[1, 128\]"),
    (ATTENTION, lambda: dict(k=host(2, 5, 2, 16, dtype=torch.float16)), ValueError, "same dtype"),
    (ATTENTION, lambda: {n: host(2, 5, 2, 16, dtype=torch.float64) for n in "qkv"}, ValueError,
     "float32, float16, and bfloat16"),
    (ATTENTION, lambda: dict(scale=0.0), ValueError, "positive normal"),
    (ATTENTION, lambda: dict(q=host(0, 5, 4, 16), k=host(0, 5, 2, 16), v=host(0, 5, 2, 8)), ValueError,
     "at least one slot"),
    (ATTENTION, lambda: dict(keys=host(9, 32, 2, 16).transpose(1, 2)), ValueError, "contiguous"),
    (ATTENTION, lambda: dict(keys=host(9, 2, 32, 17)), ValueError, "pages must have shape"),
    (ATTENTION, lambda: dict(values=host(8, 2, 32, 8)), ValueError, "pages must have shape"),
    (ATTENTION, lambda: dict(values=host(9, 2, 16, 8)), ValueError, "pages must have shape"),
    (ATTENTION, lambda: dict(keys=host(9, 2, 24, 16), values=host(9, 2, 24, 8)), ValueError, "power of two"),
    (ATTENTION, lambda: dict(keys=host(9, 2, 8, 16), values=host(9, 2, 8, 8)), ValueError, "power of two"),
    (ATTENTION, lambda: dict(keys=host(9, 2, 512, 16), values=host(9, 2, 512, 8)), ValueError, "power of two"),
    (ATTENTION, lambda: dict(keys=host(0, 2, 32, 16), values=host(0, 2, 32, 8), bounds=host(0, 2, 2, 16)),
     ValueError, "1 to 2"),
    (ATTENTION, lambda: dict(keys=host(9, 2, 32, 16, dtype=torch.float16)), ValueError, "dtype of the inputs"),
    (ATTENTION[1:], lambda: dict(bounds=host(9, 2, 16)), ValueError, "key_bounds must have shape"),
    (ATTENTION[1:], lambda: dict(bounds=host(9, 2, 2, 16, dtype=torch.float32)), ValueError, "dtype of the inputs"),
    (ATTENTION, lambda: dict(tables=host(3, 4, **I32)), ValueError, "tables must be"),
    (ATTENTION, lambda: dict(tables=host(2, 0, **I32)), ValueError, "tables must be"),
    (ATTENTION, lambda: dict(tables=host(2, 4, **I64)), ValueError, "tables must be"),
    (ATTENTION, lambda: dict(tables=host(4, 2, **I32).t()), ValueError, "tables must be contiguous"),
    (ATTENTION, lambda: dict(rows=host(2, 5, **I32)), ValueError, "rows must be"),
    (ATTENTION, lambda: dict(rows=host(10, **I64)), ValueError, "rows must be"),
    (ATTENTION, lambda: dict(lengths=host(3, **I32)), ValueError, "lengths must be"),
    (ATTENTION, lambda: dict(lengths=host(2, **I64)), ValueError, "lengths must be"),
    (ATTENTION, lambda: dict(q=host(2, 5, 4, 16).requires_grad_()), RuntimeError, "have no backward"),
    (ATTENTION, lambda: dict(keys=host(9, 2, 32, 16).requires_grad_()), RuntimeError, "have no backward"),
    (ATTENTION[2:], lambda: dict(count=0), ValueError, "count must be"),
    (ATTENTION[2:], lambda: dict(count=1025), ValueError, "count must be"),
    (ATTENTION[2:], lambda: dict(count=2**70), ValueError, "count must be"),
    (ATTENTION[2:], lambda: dict(count=2.0), TypeError, "count must be an integer"),
    (ATTENTION[2:], lambda: dict(count=True), TypeError, "count must be an integer"),
    (TABLES, lambda: dict(tables=host(8, **I32)), ValueError, "tables must have shape"),
    (TABLES, lambda: dict(tables=host(0, 4, **I32)), ValueError, "tables must have shape"),
    (TABLES, lambda: dict(tables=host(2, 4, **I64)), ValueError, "tables must have dtype int32"),
    (TABLES, lambda: dict(tables=host(4, 2, **I32).t()), ValueError, "contiguous"),
    (TABLES, lambda: dict(tables=host(8193, 1, **I32), lengths=host(8193, **I32), keep=host(8193, **I32)),
     ValueError, "at most 8192"),
    (TABLES, lambda: dict(lengths=host(3, **I32)), ValueError, "one entry per slot"),
    (TABLES, lambda: dict(lengths=host(2, **I64)), ValueError, "lengths must have dtype int32"),
    (TABLES, lambda: dict(pool=host(10, **I64)), ValueError, "pool must have dtype int32"),
    (TABLES, lambda: dict(pool=host(1, **I32)), ValueError, "pool must have shape"),
    (TABLES, lambda: dict(pool=host(20, **I32)[::2]), ValueError, "contiguous"),
    (TABLES, lambda: dict(page=0), ValueError, "power of two"),
    (TABLES, lambda: dict(page=48), ValueError, "power of two"),
    (TABLES, lambda: dict(page=2**70), ValueError, "power of two"),
    (TABLES, lambda: dict(page=16.0), TypeError, "page must be an integer"),
    (TABLES[:1], lambda: dict(tokens=-1), ValueError, "tokens must be >= 0"),
    (TABLES[:1], lambda: dict(tokens=2**30), ValueError, "fit in int32"),
    (TABLES[:1], lambda: dict(tokens=2**70), ValueError, "fit in int32"),
    (TABLES[:1], lambda: dict(offsets=host(4, **I32)), ValueError, "slots \\+ 1 entries"),
    (TABLES[:1], lambda: dict(offsets=host(3, **I64)), ValueError, "cu_seqlens must have dtype"),
    (TABLES[1:], lambda: dict(keep=host(3, **I32)), ValueError, "one entry per slot"),
    (TABLES[1:], lambda: dict(keep=host(2, **I64)), ValueError, "keep must have dtype"),
    (ATTENTION + TABLES, lambda: {}, ValueError, "require CUDA tensors"),
])
def test_refusals(names, changes, error, message):
    """Every check is made before the device is looked at: host tensors meet all of them."""
    for name in names:
        with pytest.raises(error, match=message):
            calls(arguments(**changes()))[name]()


def test_what_a_call_changes_shares_no_memory_with_what_it_reads():
    memory = torch.zeros(4096, **I32)
    tables, rest = memory[:8].view(2, 4), memory[4:]
    for changes in (dict(tables=tables, pool=rest[:10]), dict(tables=tables, lengths=rest[:2]),
                    dict(pool=memory[:10], lengths=rest[:2])):
        for name in TABLES:
            with pytest.raises(ValueError, match="share no memory"):
                calls(arguments(**changes))[name]()
    with pytest.raises(ValueError, match="share no memory"):
        calls(arguments(tables=tables, keep=rest[:2]))["release"]()
    with pytest.raises(ValueError, match="share no memory"):
        calls(arguments(tables=tables, offsets=rest[:3]))["update"]()
    pages = torch.zeros(9 * 2 * 32 * 16 + 4096, dtype=torch.bfloat16)
    keys, tail = pages[:9216].view(9, 2, 32, 16), pages[9000:]
    for names, changes in (
            (ATTENTION, dict(q=tail[:640].view(2, 5, 4, 16))), (ATTENTION, dict(k=tail[:320].view(2, 5, 2, 16))),
            (ATTENTION, dict(v=tail[:160].view(2, 5, 2, 8))),
            (ATTENTION, dict(values=pages[:4608].view(9, 2, 32, 8))),
            (ATTENTION, dict(lengths=pages.view(torch.int32)[100:102])),
            (ATTENTION, dict(tables=pages.view(torch.int32)[100:108].view(2, 4))),
            (ATTENTION[1:], dict(bounds=tail[:576].view(9, 2, 2, 16)))):
        for name in names:
            with pytest.raises(ValueError, match="share no memory"):
                calls(arguments(keys=keys, **changes))[name]()


@pytest.mark.parametrize("which", ["q", "k", "v", "keys", "values", "bounds"])
def test_tangents_are_refused(which):
    from torch.autograd import forward_ad

    with FakeTensorMode():
        for name in ATTENTION:
            if which == "bounds" and name == "paged":
                continue
            with forward_ad.dual_level():
                parts = arguments(fake)
                parts[which] = forward_ad.make_dual(parts[which], torch.ones_like(parts[which]))
                with pytest.raises(NotImplementedError, match="forward-mode"):
                    calls(parts)[name]()


def test_changed_tensors_are_declared_and_get_new_versions():
    def written(name):
        schema = getattr(torch.ops.rosa_soft, name).default._schema
        return {a.name for a in schema.arguments if a.alias_info is not None and a.alias_info.is_write}

    assert written("page_tables_update") == written("page_tables_release") == {"tables", "pool"}
    assert written("paged_attention_update") == {"key_pages", "value_pages"}
    bounded = {"key_pages", "value_pages", "key_bounds"}
    assert written("paged_attention_update_bounds") == written("selected_attention_update") == bounded


def test_every_function_is_documented():
    for name in paged.__all__:
        assert len(inspect.getdoc(getattr(paged, name))) > 80


# ---------------------------------------------------------------------------
# C entry points
# ---------------------------------------------------------------------------

def problem(**changes):
    fields = dict(dtype=2, B=2, T=100, N=200, S=0, H=4, Hkv=2, D=64, Dv=64, scale=0.125)
    fields.update(changes)
    return cabi.RosaMixerProblem(**fields)


def cache(**changes):
    fields = dict(key_pages=1, value_pages=1, key_bounds=1, tables=1, lengths=1, rows=1, columns=8,
                  pages=9, page=64)
    fields.update(changes)
    return cabi.RosaPagedCache(**fields)


def tables(**changes):
    fields = dict(tables=1, lengths=1, pool=1, slots=2, columns=8, pages=9, page=64)
    fields.update(changes)
    return cabi.RosaPageTables(**fields)


TENSOR = cabi.RosaMixerTensor(1, 0, 64, 64)


def update(p, c, count=0, workspace=16, size=1 << 40, output=1, query=TENSOR):
    t = ctypes.byref(TENSOR)
    return cabi.load().rosa_hip_paged_update(ctypes.byref(p), ctypes.byref(c), count, ctypes.byref(query),
                                             t, t, output, workspace, size, None)


@pytest.mark.parametrize("problems,caches,count,message", [
    (dict(dtype=3), {}, 0, b"dtype"), (dict(B=0), {}, 0, b"dense layout"), (dict(N=199), {}, 0, b"N = B"),
    (dict(B=0, T=0, S=0, cu_seqlens=1), {}, 0, b"packed layout"), (dict(H=3), {}, 0, b"multiple"),
    (dict(Hkv=0), {}, 0, b"multiple"), (dict(D=129), {}, 0, b"128"), (dict(Dv=0), {}, 0, b"128"),
    (dict(scale=0.0), {}, 0, b"scale"), (dict(B=1, T=2**30, N=2**30, H=2**10), {}, 0, b"too many blocks"),
    (dict(B=0, T=0, S=2**26, N=1, H=2**6, Hkv=2**6, cu_seqlens=1), {}, 0, b"too many blocks"),
    ({}, dict(page=0), 0, b"power of two"), ({}, dict(page=8), 0, b"power of two"),
    ({}, dict(page=65), 0, b"power of two"), ({}, dict(page=512), 0, b"power of two"),
    ({}, dict(columns=0), 0, b"columns"), ({}, dict(pages=0), 0, b"pages"),
    ({}, {}, -1, b"count"), ({}, {}, 1025, b"count"),
])
def test_c_entries_refuse_bad_problems_before_any_launch(problems, caches, count, message):
    p, c = problem(**problems), cache(**caches)
    assert cabi.load().rosa_hip_paged_workspace_bytes(ctypes.byref(p), ctypes.byref(c), count) == 0
    assert update(p, c, count) == 1
    assert re.search(message, cabi.load().rosa_hip_last_error())


def test_c_entries_refuse_null_pointers_and_small_or_misaligned_workspaces():
    library, packed = cabi.load(), problem(B=0, T=0, S=3, cu_seqlens=1)
    for p in (problem(), problem(T=1, N=2), packed):
        for name in ("key_pages", "value_pages", "tables", "lengths", "rows"):
            assert update(p, cache(**{name: None})) == 2
        assert update(p, cache(key_bounds=None), count=3) == 2
        assert update(p, cache(), output=None) == 2
        assert update(p, cache(), query=cabi.RosaMixerTensor(None, 0, 64, 64)) == 2
        for count in (0, 3):
            size = library.rosa_hip_paged_workspace_bytes(ctypes.byref(p), ctypes.byref(cache()), count)
            assert size > 256
            assert update(p, cache(), count, size=size - 1) == 3
            assert update(p, cache(), count, workspace=None) == 2
            assert update(p, cache(), count, workspace=8) == 1
    t = ctypes.byref(tables())
    for bad, message in ((dict(slots=0), b"slots"), (dict(slots=8193), b"slots"), (dict(columns=0), b"columns"),
                         (dict(pages=0), b"pages"), (dict(page=20), b"power of two"),
                         (dict(slots=4096, columns=2**20), b"2\\^31 entries")):
        for code in (library.rosa_hip_page_tables_update(ctypes.byref(tables(**bad)), None, 1, 2, 1, None),
                     library.rosa_hip_page_tables_release(ctypes.byref(tables(**bad)), 1, None)):
            assert code == 1
            assert re.search(message, library.rosa_hip_last_error())
    for name in ("tables", "lengths", "pool"):
        null = ctypes.byref(tables(**{name: None}))
        assert library.rosa_hip_page_tables_update(null, None, 1, 2, 1, None) == 2
        assert library.rosa_hip_page_tables_release(null, 1, None) == 2
    assert library.rosa_hip_page_tables_update(t, None, 1, 3, 1, None) == 1   # not slots * T
    assert library.rosa_hip_page_tables_update(t, 1, 0, -1, 1, None) == 1
    assert library.rosa_hip_page_tables_update(t, None, 1, 2, None, None) == 2
    assert library.rosa_hip_page_tables_release(t, None, None) == 2
    assert library.rosa_hip_page_tables_update(t, None, 0, 0, None, None) == 0  # nobody brings a token
    assert library.rosa_hip_paged_workspace_bytes(None, ctypes.byref(cache()), 0) == 0
    assert library.rosa_hip_paged_workspace_bytes(ctypes.byref(problem()), None, 0) == 0


@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("fields", [
    dict(B=1, T=1, N=1, H=1, Hkv=1), dict(B=256, T=1, N=256, H=64, Hkv=8), dict(B=1, T=2**20, N=2**20, H=64, Hkv=8),
    dict(S=8192, N=2**20, H=32, Hkv=4), dict(S=3, N=5, H=128, Hkv=1), dict(B=4096, T=8, N=2**15, H=32, Hkv=32),
])
def test_workspaces_stay_bounded(fields, dtype):
    """Partial sums go by portions, of which there are a fixed number, not by tokens or slots; scores
    of selected pages take 256 MiB, or one token's."""
    packed = dict(B=0, T=0, cu_seqlens=1) if "S" in fields else {}
    p = problem(**{**dict(D=128, Dv=128, dtype=dtype), **packed, **fields})
    c = cache(columns=1 << 14)
    size = cabi.load().rosa_hip_paged_workspace_bytes(ctypes.byref(p), ctypes.byref(c), 0)
    assert 0 < size <= 2 * (1024 + p.Hkv) * (128 + 32) * 132 * 4 + (1 << 20)
    size = cabi.load().rosa_hip_paged_workspace_bytes(ctypes.byref(p), ctypes.byref(c), 7)
    assert 0 < size <= (1 << 28) + p.N * p.Hkv * 8 * 8 + 4 * (1024 + p.N) * 32 * 132 * 4 + (1 << 20)


# ---------------------------------------------------------------------------
# the definitions
# ---------------------------------------------------------------------------

def test_a_release_takes_back_an_update():
    tables = reference.Tables(3, 6, 12, 16, order=[5, 3, 8, 1, 0, 2, 4, 6, 7, 9, 10, 11])
    rows = tables.update([0, 0, 0], [17, 0, 40])
    assert rows[0] == [11 * 16 + i for i in range(16)] + [10 * 16] and tables.free == 7
    assert rows[2][:2] == [9 * 16, 9 * 16 + 1]
    before = ([list(row) for row in tables.table], list(tables.stack), tables.free)
    assert tables.update([17, 0, 40], [100, 40, 9])[0][0] == 10 * 16 + 1
    assert tables.free == 0 and tables.table[2][3] == -1  # the pool ran out
    tables.release([117, 40, 49], [17, 0, 40])
    assert (tables.table, tables.free) == (before[0], before[2])
    assert tables.stack[:tables.free] == before[1][:tables.free]


def test_the_definition_of_attention_agrees_with_step_by_step_evaluation():
    generator = torch.Generator().manual_seed(0)
    randn = lambda *shape: torch.randn(*shape, generator=generator, dtype=torch.float64)
    past, q, k, v = 43, randn(9, 4, 3), randn(52, 2, 3), randn(52, 2, 5)
    for count in (None, 1, 2, 50):
        output, bound, _ = reference.attention(q, k, v, past, 16, count)
        for i in range(9):
            t = past + i
            for h in range(4):
                rows = range(t + 1)
                if count is not None:
                    best = []
                    for j in range(t // 16):
                        page = k[j * 16:(j + 1) * 16, h // 2]
                        most = [sum(max(q[i, m, d] * page[:, d].min(), q[i, m, d] * page[:, d].max())
                                    for d in range(3)) for m in (h // 2 * 2, h // 2 * 2 + 1)]
                        best.append((-float(max(most)), j))
                    pages = {j for _, j in sorted(best)[:count]} | {t // 16}
                    rows = [s for s in rows if s // 16 in pages]
                rows = list(rows)
                p = torch.softmax(3 ** -0.5 * k[rows, h // 2] @ q[i, h], 0)
                assert torch.allclose(output[i, h], p @ v[rows, h // 2])
                assert torch.allclose(bound[i, h], p @ v[rows, h // 2].abs())
