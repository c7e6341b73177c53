"""The paged cache's entry points refuse what they cannot do, before any
device work (no GPU here), and their struct has its declared layout."""
import ctypes as C
import random

import pytest

import needle_cs_amd as N
from needle_cs_amd.paged import PagedCache, PagedCacheView

A = 0x10000  # a 16-byte aligned address; every call here is refused before it could be used
BIG = 1 << 40


def cache(**other):
    dims = dict(layers=2, pages=8, page_size=16, kv_heads=2, qk_dim=48, v_dim=64, sequences=4, width=6)
    names = ("keys", "key_scales", "values", "value_scales", "tables", "lengths", "refs")
    buffers = {n: other.pop(n, A) for n in names}
    return PagedCache(**{**dims, **other}, buffers=buffers)


def refused(match):
    return pytest.raises(N.NeedleHipError, match=match)


def test_struct_layout():
    assert C.sizeof(PagedCacheView) == 88
    assert PagedCacheView.tables.offset == 32 and PagedCacheView.layers.offset == 56
    assert PagedCacheView.width.offset == 84


@pytest.mark.parametrize("other,match", [
    ({"page_size": 24}, "page size"), ({"page_size": 8}, "page size"), ({"page_size": 512}, "page size"),
    ({"page_size": 0}, "page size"), ({"page_size": -16}, "page size"),
    ({"qk_dim": 64, "v_dim": 48}, "head dims"), ({"qk_dim": 128, "v_dim": 64}, "head dims"),
    ({"qk_dim": 32, "v_dim": 32}, "head dims"),
    ({"layers": 0}, "layers"), ({"pages": 0}, "pages"), ({"pages": (1 << 20) + 1}, "pages"),
    ({"kv_heads": 0}, "kv heads"), ({"kv_heads": 257}, "kv heads"), ({"sequences": 0}, "sequences"),
    ({"sequences": 65537}, "sequences"), ({"width": 0}, "pages a sequence"),
    ({"width": (1 << 26) + 1}, "pages a sequence"), ({"keys": None}, "null"), ({"refs": None}, "null"),
    ({"values": A + 8}, "aligned"), ({"key_scales": A + 4}, "aligned"), ({"tables": A + 2}, "aligned"),
])
def test_a_malformed_cache_is_refused_by_every_call(other, match):
    c = cache(**other)
    for call in (lambda: c.reset(), lambda: c.append(0, A, 4096, A, 4096, A, A, 1),
                 lambda: c.decode(0, A, A, 1, 2, A, A, A, 16, A, BIG, A),
                 lambda: c.prompt(0, A, A, 1, 2, 1, A, A, A, 0, 16, A, BIG, A),
                 lambda: c.copy(1, A, A), lambda: c.fork(1, A, A, None, A, BIG),
                 lambda: c.resize(1, A, A, None, A, BIG), lambda: c.free(1, A, A, BIG),
                 lambda: c.compact(None, A, BIG)):
        with refused(match):
            call()
    assert c.pages_workspace(1) == 0 and c.decode_workspace(1, 2, 16) == 0 and c.prompt_workspace(1, 2, 1, 16) == 0


def test_no_cache_is_refused():
    lib = N.lib()
    assert lib.nhip_paged_reset_dev(None, None) == -1
    assert lib.nhip_paged_compact_dev(None, None, A, BIG, None) == -1
    assert lib.nhip_paged_pages_workspace(None, 4) == 0


def test_a_closed_cache_refuses_its_calls():
    c = cache()
    c.close()
    with refused("null"):
        c.reset()


@pytest.mark.parametrize("args,match", [
    ((2, A, 96, A, 128, A, A, 1), "layer"), ((-1, A, 96, A, 128, A, A, 1), "layer"),
    ((0, A, 95, A, 128, A, A, 1), "strides"), ((0, A, 96, A, 127, A, A, 1), "strides"),
    ((0, None, 96, A, 128, A, A, 1), "null"), ((0, A, 96, None, 128, A, A, 1), "null"),
    ((0, A, 96, A, 128, None, A, 1), "null"), ((0, A, 96, A, 128, A, None, 1), "null"),
    ((0, A, 96, A, 128, A, A, -1), "rows"), ((0, A, 96, A, 128, A, A, (1 << 20) + 1), "rows"),
])
def test_append_refuses(args, match):
    with refused(match):
        cache().append(*args)


@pytest.mark.parametrize("change,match", [
    ({"layer": 2}, "layer"), ({"q": None}, "null"), ({"q_scales": None}, "null"), ({"out": None}, "null"),
    ({"q": A + 8}, "aligned"), ({"out": A + 8}, "aligned"), ({"rows": -1}, "rows"), ({"rows": (1 << 20) + 1}, "rows"),
    ({"heads": 3}, "heads"), ({"heads": 0}, "heads"), ({"heads": 34}, "heads"), ({"heads": -2}, "heads"),
    ({"max_count": -1}, "max_count"), ({"max_count": 97}, "max_count"), ({"a": None}, "null"),
    ({"b": None}, "null"), ({"c": None}, "null"),
])
def test_attention_refuses(change, match):
    d = dict(layer=0, q=A, q_scales=A, rows=3, heads=12, a=A, b=A, c=A, max_count=96, out=A)
    d.update(change)
    with refused(match):
        cache().decode(d["layer"], d["q"], d["q_scales"], d["rows"], d["heads"], d["a"], d["b"], d["c"],
                       d["max_count"], A, BIG, d["out"])
    with refused(match):
        cache().prompt(d["layer"], d["q"], d["q_scales"], d["rows"], d["heads"], 1, d["a"], d["b"], d["c"], 0,
                       d["max_count"], A, BIG, d["out"])


def test_prompt_refuses_its_own():
    for runs, window in ((-1, 0), ((1 << 20) + 1, 0), (1, -1)):
        with refused("runs"):
            cache().prompt(0, A, A, 3, 12, runs, A, A, A, window, 96, A, BIG, A)


def test_prompt_refuses_more_tiles_than_a_grid_holds():
    with refused("too many"):
        cache(kv_heads=16).prompt(0, A, A, 3, 16, 1 << 20, A, A, A, 0, 96, A, BIG, A)
    with refused("too many"):
        cache(kv_heads=256).prompt(0, A, A, 1 << 20, 4096, 1, A, A, A, 0, 96, A, BIG, A)


def test_workspace_sizes_need_no_device():
    """They are the same before and after a device is chosen, and a window never needs more."""
    c = cache(pages=4096, width=4096)
    assert c.decode_workspace(4, 12, 300) == 0
    assert c.decode_workspace(1, 12, 60000) >= 4 * 12 * 2 * 66
    assert c.prompt_workspace(4000, 12, 3, 60000) == 0
    assert c.prompt_workspace(20, 12, 1, 60000) >= 4 * 20 * 12 * 2 * 66


#: (pages of 16, kv heads, query heads, rows, runs, max_count) -> decode's and a prompt's workspace for dims of 48 / 64:
#: rows * heads * parts * (64 + 2) * 4 bytes, with the parts that the rules make of max_count // 64 + 2 blocks
WORKSPACES = [
    ((4096, 2, 12, 4, 1, 300), (0, 4 * 12 * 3 * 264)),
    ((4096, 2, 12, 1, 1, 60000), (1 * 12 * 63 * 264, 1 * 12 * 63 * 264)),
    ((4096, 2, 12, 20, 1, 60000), (20 * 12 * 50 * 264, 20 * 12 * 63 * 264)),
    ((4096, 16, 16, 300, 3, 8000), (0, 300 * 16 * 10 * 264)),  # 80 workgroups of 127 blocks: 14 a part
    ((4096, 16, 16, 300, 3, 1500), (0, 300 * 16 * 9 * 264)),  # of 25: 3 a part
    ((4096, 16, 16, 4000, 3, 60000), (0, 0)),
]


@pytest.mark.parametrize("call,want", WORKSPACES)
def test_workspace_sizes(call, want):
    """Here without a device; tests/test_paged_gpu.py asks for the same with one."""
    width, kv, heads, rows, runs, max_count = call
    c = cache(pages=width, width=width, kv_heads=kv)
    assert (c.decode_workspace(rows, heads, max_count), c.prompt_workspace(rows, heads, runs, max_count)) == want


def test_a_window_never_needs_more_workspace():
    """A prompt call whose workspace is as large as the query says is refused for
    its missing arrays, never for the workspace, whatever its window."""
    rng = random.Random(5)
    split = 0
    for _ in range(400):
        kv, group = rng.choice([1, 2, 3, 8, 16, 48]), rng.choice([1, 2, 3, 5, 6, 16])
        width = int(2 ** rng.uniform(0, 13))
        max_count = rng.randint(0, 16 * width)
        rows, runs = int(2 ** rng.uniform(0, 12)), int(2 ** rng.uniform(0, 8))
        c = cache(pages=width, width=width, kv_heads=kv)
        need = c.prompt_workspace(rows, kv * group, runs, max_count)
        split += need > 0
        for window in [0, 1, max_count, max_count + 1, 2 ** 31 - 1] + [int(2 ** rng.uniform(0, 17)) for _ in range(6)]:
            with refused("prompt: null pointer"):
                c.prompt(0, A, A, rows, kv * group, runs, None, None, None, window, max_count, A, need, A)
    assert split > 100


def test_attention_workspaces_are_checked():
    c = cache(pages=4096, width=4096)
    need = c.decode_workspace(1, 12, 60000)
    for ws, size in ((None, need), (A, need - 1), (A + 8, need)):
        with refused("workspace"):
            c.decode(0, A, A, 1, 12, A, A, A, 60000, ws, size, A)
    need = c.prompt_workspace(20, 12, 1, 60000)
    for ws, size in ((None, need), (A, need - 1), (A + 8, need)):
        with refused("workspace"):
            c.prompt(0, A, A, 20, 12, 1, A, A, A, 0, 60000, ws, size, A)


def test_workspaces_are_checked():
    c = cache()
    need = c.pages_workspace(4)
    assert need > 0
    for ws, size in ((None, need), (A, need - 1), (A + 2, need)):
        with refused("workspace"):
            c.fork(4, A, A, None, ws, size)
        with refused("workspace"):
            c.resize(4, A, A, None, ws, size)
        with refused("workspace"):
            c.free(4, A, ws, size)
    for ws, size in ((None, BIG), (A, c.pages_workspace(0) - 1)):
        with refused("workspace"):
            c.compact(None, ws, size)


@pytest.mark.parametrize("count", [-1, 1025])
def test_entry_counts_are_checked(count):
    c = cache()
    for call in (lambda: c.copy(count, A, A), lambda: c.fork(count, A, A, None, A, BIG),
                 lambda: c.resize(count, A, A, None, A, BIG), lambda: c.free(count, A, A, BIG)):
        with refused("entries"):
            call()
    assert c.pages_workspace(count) == 0


def test_null_entries_are_refused():
    c = cache()
    for call in (lambda: c.copy(1, None, A), lambda: c.copy(1, A, None), lambda: c.fork(1, None, A, None, A, BIG),
                 lambda: c.fork(1, A, None, None, A, BIG), lambda: c.resize(1, None, A, None, A, BIG),
                 lambda: c.resize(1, A, None, None, A, BIG), lambda: c.free(1, None, A, BIG)):
        with refused("null"):
            call()


def test_nothing_to_do_is_no_error():
    c = cache()
    c.append(0, None, 96, None, 128, None, None, 0)
    c.decode(0, None, None, 0, 12, None, None, None, 16, None, 0, None)
    c.prompt(0, None, None, 0, 12, 0, None, None, None, 0, 16, None, 0, None)
    c.prompt(0, A, A, 5, 12, 0, None, None, None, 0, 16, None, 0, A)
    c.copy(0, None, None)
    c.fork(0, None, None, None, None, 0)
    c.resize(0, None, None, None, None, 0)
    c.free(0, None, None, 0)


def test_a_cache_of_its_own_needs_sizes():
    with pytest.raises(ValueError):
        PagedCache(1, 0, 16, 1, 64, 64, 1, 1)
