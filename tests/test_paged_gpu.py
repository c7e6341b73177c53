"""The paged cache on the GPU against plain numpy (paged_f64.py): append bit
for bit with the oracle's QuantizeInt8, attention within the bound of its
arithmetic, bookkeeping and moved pages exactly, and all of it together as a
server runs it.  Positions that no sequence holds have NaN scales."""
import ctypes as C

import numpy as np
import pytest

from paged_f64 import Books, Pool
from test_paged import WORKSPACES

pytestmark = pytest.mark.gpu

DIMS = [(48, 64), (64, 64), (128, 128)]


class Gpu:
    """A Pool on the device, and the calls on it."""

    def __init__(self, hip, pool):
        from needle_cs_amd.paged import PagedCache
        self.hip, self.pool = hip, pool
        self.bufs = {n: hip.DeviceBuffer.from_array(getattr(pool, n)) for n in Pool.NAMES}
        self.cache = PagedCache(pool.layers, pool.pages, pool.page, pool.kv, pool.qk, pool.v, pool.sequences,
                                pool.width, buffers={n: b.ptr for n, b in self.bufs.items()})
        self.keep = []

    def dev(self, a, dtype=np.int32):
        b = self.hip.DeviceBuffer.from_array(np.ascontiguousarray(a, dtype=dtype))
        self.keep.append(b)
        return b

    def get(self, name):
        a = getattr(self.pool, name)
        return self.bufs[name].download(a.dtype).reshape(a.shape)

    def workspace(self, size):
        b = self.hip.DeviceBuffer.from_array(np.full(max(size, 16), 0xA5, dtype=np.uint8))
        self.keep.append(b)
        return b.ptr, size

    def decode(self, layer, q, qs, seq, first, count, max_count, stream=None):
        rows, heads = q.shape[:2]
        out = self.dev(np.full((rows, heads, self.pool.v), np.nan), np.float32)
        ws = self.workspace(self.cache.decode_workspace(rows, heads, max_count))
        self.cache.decode(layer, self.dev(q, np.int8).ptr, self.dev(qs, np.float32).ptr, rows, heads,
                          self.dev(seq).ptr, self.dev(first).ptr, self.dev(count).ptr, max_count, *ws, out.ptr, stream)
        return out.download(np.float32).reshape(rows, heads, self.pool.v)

    def prompt(self, layer, q, qs, run_rows, run_seq, run_pos, window, max_count):
        rows, heads = q.shape[:2]
        out = self.dev(np.full((rows, heads, self.pool.v), -77.0), np.float32)
        ws = self.workspace(self.cache.prompt_workspace(rows, heads, len(run_seq), max_count))
        self.cache.prompt(layer, self.dev(q, np.int8).ptr, self.dev(qs, np.float32).ptr, rows, heads, len(run_seq),
                          self.dev(run_rows).ptr, self.dev(run_seq).ptr, self.dev(run_pos).ptr, window, max_count,
                          *ws, out.ptr)
        return out.download(np.float32).reshape(rows, heads, self.pool.v)

    def books(self):
        return self.get("tables"), self.get("lengths"), self.get("refs")


def queries(rng, rows, heads, qk, sharp=0.03):
    return (rng.integers(-128, 128, (rows, heads, qk), dtype=np.int8),
            rng.uniform(0.2 * sharp, sharp, (rows, heads)).astype(np.float32))


def close(got, want, far):
    off = np.abs(got - want)
    assert np.all(off <= far), (float(off.max()), np.argwhere(off > far)[:4].tolist(), float(far.max()))
    rms = np.sqrt(np.mean(want ** 2))
    if rms:
        assert np.sqrt(np.mean(off ** 2)) <= 1e-5 * rms


def check_decode(gpu, layer, q, qs, spec, max_count):
    pool = gpu.pool
    seq, first, count = (np.array(x) for x in zip(*spec))
    got = gpu.decode(layer, q, qs, seq, first, count, max_count)
    want, far = np.zeros(got.shape), np.zeros(got.shape)
    span = pool.width * pool.page
    for r, (s, f, n) in enumerate(spec):
        if 0 <= s < pool.sequences and f >= 0 and 0 <= n <= max_count and f + n <= span:
            want[r], far[r] = pool.attend(layer, s, q[r], qs[r], f, n)
    close(got, want, far)
    return got


# ---------------------------------------------------------------- decode --

@pytest.mark.parametrize("qk,v", DIMS)
@pytest.mark.parametrize("kv,group", [(1, 1), (2, 6), (3, 16), (16, 1), (2, 5)])
def test_decode_lengths_and_spans(hip, qk, v, kv, group):
    rng = np.random.default_rng(100 * qk + 10 * kv + group)
    lengths = [0, 1, 2, 15, 16, 17, 63, 64, 65, 130, 300]
    pool = Pool(rng, 2, 60, 16, kv, qk, v, len(lengths), 20)
    pool.give(rng, lengths)
    spec = [(s, 0, n) for s, n in enumerate(lengths)] + [(10, 7, 200), (10, 64, 1), (10, 299, 1), (9, 33, 64),
                                                          (10, 0, 257), (8, 64, 1)]
    q, qs = queries(rng, len(spec), kv * group, qk)
    check_decode(Gpu(hip, pool), 1, q, qs, spec, 300)


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("qk,v", DIMS)
def test_decode_pages(hip, page, qk, v):
    rng = np.random.default_rng(page + qk)
    lengths = [1, page - 1, page, page + 1, 3 * page + 5, 1100]
    width = -(-1100 // page) + 1
    pool = Pool(rng, 1, sum(-(-n // page) for n in lengths) + 2, page, 2, qk, v, len(lengths), width)
    pool.give(rng, lengths)
    spec = [(s, 0, n) for s, n in enumerate(lengths)] + [(5, 1000, 100), (4, 2 * page - 3, page + 6)]
    q, qs = queries(rng, len(spec), 8, qk)
    check_decode(Gpu(hip, pool), 0, q, qs, spec, width * page)


def test_decode_long_and_split(hip):
    """Few rows of a long context: the length is split; the bound of the rows
    (max_count) may be far above them."""
    rng = np.random.default_rng(5)
    lengths = [9001, 5, 4096]
    pool = Pool(rng, 1, 260, 64, 1, 64, 64, 3, 300)
    pool.give(rng, lengths)
    gpu = Gpu(hip, pool)
    q, qs = queries(rng, 4, 4, 64)
    spec = [(0, 0, 9001), (1, 0, 5), (2, 0, 4096), (0, 8000, 1001)]
    a = check_decode(gpu, 0, q, qs, spec, 9001)
    b = check_decode(gpu, 0, q, qs, spec, 300 * 64)
    assert np.allclose(a, b, rtol=1e-4, atol=1e-4)


@pytest.mark.parametrize("rows,kv,lo,hi", [(2, 1, 1000, 1300), (1, 2, 700, 900), (9, 64, 700, 730)])
def test_decode_sixteen_heads_of_128(hip, rows, kv, lo, hi):
    """The largest joins: eight waves and four, of 16 heads of 128."""
    rng = np.random.default_rng(8)
    pool = Pool(rng, 1, 50, 64, kv, 128, 128, 2, 21)
    pool.give(rng, [hi, lo])
    q, qs = queries(rng, rows, 16 * kv, 128)
    check_decode(Gpu(hip, pool), 0, q, qs, [(i % 2, 3 * i, lo - 3 * i) for i in range(rows)], hi)


def test_decode_many_rows(hip):
    rng = np.random.default_rng(6)
    lengths = rng.integers(1, 90, 300)
    pool = Pool(rng, 1, 1900, 16, 2, 64, 64, 300, 6)
    pool.give(rng, lengths)
    spec = [(s, 0, int(n)) for s, n in enumerate(lengths)]
    q, qs = queries(rng, 300, 4, 64)
    check_decode(Gpu(hip, pool), 0, q, qs, spec, 90)


@pytest.mark.parametrize("kv,group,rows", [(48, 1, 11), (100, 1, 64), (8, 2, 64), (8, 1, 63), (256, 1, 2)])
def test_decode_rows_in_order_of_their_length(hip, kv, group, rows):
    """More workgroups than CUs, rows of many lengths, equal ones and none."""
    rng = np.random.default_rng(39)
    pool = Pool(rng, 1, 80, 16, kv, 48, 64, 4, 20)
    pool.give(rng, [300, 150, 64, 10])
    q, qs = queries(rng, rows, kv * group, 48)
    spec = []
    for _ in range(rows):
        s = int(rng.integers(0, 4))
        n = int(rng.integers(0, pool.lengths[s] + 1) // (1 + 3 * rng.integers(0, 2)))
        spec.append((s, int(rng.integers(0, pool.lengths[s] - n + 1)), n))
    spec[rows // 2], spec[rows // 3] = (0, 0, 0), (5, 0, 9)
    spec[-1] = (0, 0, 300)
    check_decode(Gpu(hip, pool), 0, q, qs, spec, 300)


@pytest.mark.parametrize("kv,group,rows,qk,v", [(5, 1, 60, 48, 64), (5, 3, 60, 48, 64), (8, 1, 40, 64, 64),
                                                (8, 2, 63, 64, 64), (8, 1, 48, 128, 128), (16, 2, 17, 128, 128)])
def test_decode_rows_in_order_of_their_length_by_eight_waves(hip, kv, group, rows, qk, v):
    """257 to 511 workgroups of rows of 11 to 40 blocks: whole rows, sorted, eight waves each."""
    rng = np.random.default_rng(47)
    assert 256 < kv * rows < 512
    pool = Pool(rng, 1, 60, 64, kv, qk, v, 5, 30)
    pool.give(rng, [1900, 1100, 300, 64, 5])
    q, qs = queries(rng, rows, kv * group, qk)
    spec = []
    for _ in range(rows):
        s = int(rng.integers(0, 5))
        n = int(rng.integers(0, pool.lengths[s] + 1) // (1 + 5 * rng.integers(0, 2)))
        spec.append((s, int(rng.integers(0, pool.lengths[s] - n + 1)), n))
    spec[rows // 2], spec[rows // 3] = (0, 0, 0), (9, 0, 9)
    spec[-1] = (0, 0, 1900)
    gpu = Gpu(hip, pool)
    assert gpu.cache.decode_workspace(rows, kv * group, 1900) == 0
    seq, first, count = (np.array(x) for x in zip(*spec))
    got = gpu.decode(0, q, qs, seq, first, count, 1900)
    want, far = np.zeros(got.shape), np.zeros(got.shape)
    for r, (s, f, n) in enumerate(spec):
        if s < 5 and n:
            want[r], far[r] = pool.attend_products(0, s, q[r], qs[r], f, n)
    close(got, want, far)


def test_decode_rows_out_of_range_give_zeros(hip):
    rng = np.random.default_rng(7)
    pool = Pool(rng, 1, 40, 16, 2, 64, 64, 3, 8)
    pool.give(rng, [100, 20, 60])
    gpu = Gpu(hip, pool)
    q, qs = queries(rng, 9, 4, 64)
    big = 2 ** 31 - 1
    bad = [(-1, 0, 10), (3, 0, 10), (0, -1, 10), (0, 0, -5), (0, 0, 101), (0, 120, 10), (0, big, big), (0, big, 5),
           (big, 0, 10)]
    got = check_decode(gpu, 0, q, qs, bad, 100)
    assert not got.any()
    assert not gpu.decode(0, q, qs, *zip(*[(0, 0, 0)] * 9), 0).any()


def test_decode_leaves_out_pages_outside_the_pool(hip):
    rng = np.random.default_rng(8)
    pool = Pool(rng, 1, 40, 16, 2, 64, 64, 3, 8)
    pool.give(rng, [100, 20, 60])
    pool.tables[0, 2], pool.tables[0, 5], pool.tables[1, :2], pool.tables[2, 0] = -7, 40, 2 ** 31 - 1, -2 ** 31
    q, qs = queries(rng, 4, 8, 64)
    got = check_decode(Gpu(hip, pool), 0, q, qs, [(0, 0, 100), (1, 0, 20), (2, 0, 60), (0, 32, 16)], 128)
    assert not got[1].any() and not got[3].any()


@pytest.mark.parametrize("sharp", [0.0005, 0.3])
@pytest.mark.parametrize("spread", [0.0, 3.0])
def test_decode_flat_and_peaked_scores_and_uneven_scales(hip, sharp, spread):
    """Scores from nearly equal to one position taking all; value scales that
    differ by e^10 within a sequence."""
    rng = np.random.default_rng(9)
    pool = Pool(rng, 1, 80, 16, 2, 64, 64, 2, 40)
    pool.give(rng, [600, 333], spread)
    pool.key_scales[:] = np.where(np.isnan(pool.key_scales), np.nan, 0.02)
    pool.value_scales[0, pool.tables[1, 3], :, 2] = 0.0
    q, qs = queries(rng, 2, 12, 64, sharp)
    check_decode(Gpu(hip, pool), 0, q, qs, [(0, 0, 600), (1, 0, 333)], 640)


def test_decode_offsets_past_32_bits(hip):
    """A pool of over 4 GB a kind: the pages used are its first and its last."""
    from needle_cs_amd.paged import PagedCache
    layers, pages, page, kv, d = 2, 2300, 256, 32, 128
    rng = np.random.default_rng(11)
    cells = layers * pages * kv * page
    assert cells * d > 2 ** 32 and cells > 2 ** 25
    bufs = {"keys": hip.DeviceBuffer(cells * d), "values": hip.DeviceBuffer(cells * d),
            "key_scales": hip.DeviceBuffer(4 * cells), "value_scales": hip.DeviceBuffer(4 * cells)}
    small = Pool(rng, 1, 3, page, kv, d, d, 1, 3)
    small.give(rng, [600])
    at = [pages - 1, 0, pages - 2]  # where the small pool's pages lie in layer 1
    for name in ("keys", "key_scales", "values", "value_scales"):
        a = getattr(small, name)
        for p in range(3):
            bufs[name].upload(a[0, p], offset=(pages + at[p]) * a[0, p].nbytes)
    tables = np.array([[at[p] for p in small.tables[0]]], dtype=np.int32)
    more = {"tables": hip.DeviceBuffer.from_array(tables), "lengths": hip.DeviceBuffer.from_array(small.lengths),
            "refs": hip.DeviceBuffer(4 * pages)}
    more["refs"].zero()
    cache = PagedCache(layers, pages, page, kv, d, d, 1, 3, buffers={n: b.ptr for n, b in {**bufs, **more}.items()})
    q, qs = queries(rng, 1, kv, d)
    dq, ds = hip.DeviceBuffer.from_array(q), hip.DeviceBuffer.from_array(qs)
    spans = hip.DeviceBuffer.from_array(np.array([0, 0, 600, 0, 1, 599], dtype=np.int32))
    out = hip.DeviceBuffer(4 * kv * d)
    want, far = small.attend(0, 0, q[0], qs[0], 0, 600)
    need = cache.decode_workspace(1, kv, 768)
    ws = hip.DeviceBuffer(max(need, 16))
    cache.decode(1, dq.ptr, ds.ptr, 1, kv, spans.ptr, spans.ptr + 4, spans.ptr + 8, 768, ws.ptr, need, out.ptr)
    close(out.download(np.float32).reshape(kv, d), want, far)
    need = cache.prompt_workspace(1, kv, 1, 768)
    ws2 = hip.DeviceBuffer(max(need, 16))
    cache.prompt(1, dq.ptr, ds.ptr, 1, kv, 1, spans.ptr + 12, spans.ptr, spans.ptr + 20, 0, 768, ws2.ptr, need,
                 out.ptr)
    close(out.download(np.float32).reshape(kv, d), want, far)
    # an append and a page copy there
    x = rng.standard_normal((1, 2 * kv * d)).astype(np.float32)
    dx, row = hip.DeviceBuffer.from_array(x), hip.DeviceBuffer.from_array(np.array([0, 600], dtype=np.int32))
    cache.append(1, dx.ptr, 2 * kv * d, dx.ptr + 4 * kv * d, 2 * kv * d, row.ptr, row.ptr + 4, 1)
    pair = hip.DeviceBuffer.from_array(np.array([pages - 1, 7], dtype=np.int32))
    cache.copy(1, pair.ptr, pair.ptr + 4)
    hip.check(hip.lib().nhip_device_sync())
    page_bytes = kv * page * d
    for name in ("keys", "values"):
        a = bufs[name].download(np.int8, page_bytes, offset=(2 * pages - 1) * page_bytes)
        b = bufs[name].download(np.int8, page_bytes, offset=(pages + 7) * page_bytes)
        assert np.array_equal(a, b)
    p = int(tables[0, 600 // page])
    scales = bufs["key_scales"].download(np.float32, kv * page, offset=4 * (pages + p) * kv * page).reshape(kv, page)
    assert np.array_equal(scales[:, 600 % page], np.abs(x[0, :kv * d].reshape(kv, d)).max(1) / np.float32(127))


def test_workspace_sizes_with_a_device(hip):
    """The same as without one (tests/test_paged.py)."""
    from needle_cs_amd.paged import PagedCache
    names = ("keys", "key_scales", "values", "value_scales", "tables", "lengths", "refs")
    for (width, kv, heads, rows, runs, max_count), want in WORKSPACES:
        c = PagedCache(2, width, 16, kv, 48, 64, 4, width, buffers={n: 0x10000 for n in names})
        assert (c.decode_workspace(rows, heads, max_count), c.prompt_workspace(rows, heads, runs, max_count)) == want


# ---------------------------------------------------------------- prompt --

def check_prompt(gpu, layer, q, qs, runs, window, max_count, rows_behind=0):
    pool = gpu.pool
    run_rows = np.cumsum([0] + [n for n, _, _ in runs])
    assert run_rows[-1] + rows_behind == q.shape[0]
    got = gpu.prompt(layer, q, qs, run_rows, [s for _, s, _ in runs], [p for _, _, p in runs], window, max_count)
    want, far = np.zeros(got.shape), np.zeros(got.shape)
    want[run_rows[-1]:] = -77.0
    for i, (n, s, pos) in enumerate(runs):
        for j in range(n):
            p, r = pos + j, run_rows[i] + j
            if 0 <= s < pool.sequences and pos >= 0 and p < min(max_count, pool.width * pool.page):
                first = max(0, p - window + 1) if window else 0
                want[r], far[r] = pool.attend(layer, s, q[r], qs[r], first, p + 1 - first, True)
    assert np.array_equal(got[run_rows[-1]:], want[run_rows[-1]:].astype(np.float32))
    close(got[:run_rows[-1]], want[:run_rows[-1]], far[:run_rows[-1]])
    return got


@pytest.mark.parametrize("qk,v", DIMS)
@pytest.mark.parametrize("kv,group", [(1, 1), (2, 6), (1, 16), (4, 1), (2, 5)])
def test_prompt_runs_of_different_lengths(hip, qk, v, kv, group):
    rng = np.random.default_rng(qk + 7 * kv + group)
    runs = [(1, 0, 0), (70, 1, 0), (0, 2, 5), (17, 3, 30), (1, 4, 129), (33, 5, 31), (64, 6, 0)]
    pool = Pool(rng, 2, 40, 16, kv, qk, v, 7, 9)
    pool.give(rng, [n + p for n, _, p in runs])
    q, qs = queries(rng, sum(n for n, _, _ in runs), kv * group, qk)
    check_prompt(Gpu(hip, pool), 1, q, qs, runs, 0, 144)


@pytest.mark.parametrize("window", [1, 2, 63, 64, 65, 100])
def test_prompt_windows(hip, window):
    rng = np.random.default_rng(window)
    runs = [(150, 0, 0), (40, 1, 170), (1, 2, 0)]
    pool = Pool(rng, 1, 40, 16, 2, 64, 64, 3, 14)
    pool.give(rng, [n + p for n, _, p in runs])
    q, qs = queries(rng, 191, 4, 64)
    check_prompt(Gpu(hip, pool), 0, q, qs, runs, window, 224)


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("qk,v", DIMS)
def test_prompt_pages(hip, page, qk, v):
    rng = np.random.default_rng(page + qk)
    runs = [(2 * page // 3 + 5, 0, page - 3), (page + 1, 1, 0), (9, 2, 2 * page)]
    pool = Pool(rng, 1, 12, page, 2, qk, v, 3, 4)
    pool.give(rng, [n + p for n, _, p in runs])
    q, qs = queries(rng, sum(n for n, _, _ in runs), 2, qk)
    check_prompt(Gpu(hip, pool), 0, q, qs, runs, 0, 4 * page)


def test_prompt_few_rows_of_a_long_context(hip):
    rng = np.random.default_rng(15)
    runs = [(5, 0, 6000), (1, 1, 0), (3, 2, 2047)]
    pool = Pool(rng, 1, 140, 64, 1, 64, 64, 3, 100)
    pool.give(rng, [n + p for n, _, p in runs])
    gpu = Gpu(hip, pool)
    q, qs = queries(rng, 9, 4, 64)
    check_prompt(gpu, 0, q, qs, runs, 0, 6400)
    check_prompt(gpu, 0, q, qs, runs, 1500, 6005)


@pytest.mark.parametrize("window", [0, 1, 700, 3000])
def test_prompt_split_over_the_length(hip, window):
    """Few tiles of a long context, in parts that are joined: runs shorter and
    longer than a part, pages outside the pool, rows behind the last run."""
    rng = np.random.default_rng(20 + window)
    runs = [(3, 0, 3000), (2, 1, 20), (0, 2, 0), (1, 3, 1500)]
    pool = Pool(rng, 1, 330, 16, 2, 48, 64, 4, 200)
    pool.give(rng, [n + p for n, _, p in runs])
    pool.tables[0, 7:40] = -1
    gpu = Gpu(hip, pool)
    assert gpu.cache.prompt_workspace(8, 12, 4, 3200) > 0
    q, qs = queries(rng, 8, 12, 48)
    check_prompt(gpu, 0, q, qs, runs, window, 3200, rows_behind=2)


def test_prompt_spoilt_positions(hip):
    """NaN and infinite scales in a row's future do not reach it; they spoil
    the rows that attend them."""
    rng = np.random.default_rng(23)
    pool = Pool(rng, 1, 40, 16, 2, 64, 64, 1, 8)
    pool.give(rng, [120])
    keys, values = pool.key_scales.copy(), pool.value_scales.copy()
    for scales, pos, bad in ((pool.value_scales, 50, np.nan), (pool.value_scales, 90, np.inf),
                             (pool.key_scales, 70, np.nan)):
        scales[0, pool.tables[0, pos // 16], :, pos % 16] = bad
    gpu = Gpu(hip, pool)
    q, qs = queries(rng, 120, 4, 64)
    got = gpu.prompt(0, q, qs, [0, 120], [0], [0], 0, 128)
    assert np.isnan(got[50:]).all() and np.isfinite(got[:50]).all()
    count = gpu.decode(0, q, qs, [0] * 120, [0] * 120, list(range(1, 121)), 120)
    assert np.isnan(count[50:]).all() and np.isfinite(count[:50]).all()
    pool.key_scales, pool.value_scales = keys, values
    for r in range(50):
        want, far = pool.attend(0, 0, q[r], qs[r], 0, r + 1, True)
        assert np.all(np.abs(got[r] - want) <= far) and np.all(np.abs(count[r] - want) <= far)


@pytest.mark.parametrize("kv,group", [(2, 1), (1, 6)])
@pytest.mark.parametrize("window", [0, 1, 40, 130])
def test_large_scales_reach_only_the_rows_that_attend_them(hip, window, kv, group):
    """Value scales 2^40 to 2^58 times the others: a row before such a position,
    or whose window has left it, is as exact as without it."""
    rng = np.random.default_rng(29)
    pool = Pool(rng, 1, 40, 16, kv, 64, 64, 1, 20)
    pool.give(rng, [310])
    for pos, e in ((40, 46), (63, 40), (64, 50), (170, 58), (309, 58)):
        pool.value_scales[0, pool.tables[0, pos // 16], :, pos % 16] = 2.0 ** e
    gpu = Gpu(hip, pool)
    q, qs = queries(rng, 310, kv * group, 64)
    got = gpu.prompt(0, q, qs, [0, 310], [0], [0], window, 310)
    first = [max(0, p - window + 1) if window else 0 for p in range(310)]
    count = [p + 1 - f for p, f in enumerate(first)]
    single = gpu.decode(0, q, qs, [0] * 310, first, count, 310)
    for p in range(310):
        want, far = pool.attend(0, 0, q[p], qs[p], first[p], count[p], True)
        assert np.all(np.abs(got[p] - want) <= far), p
        want, far = pool.attend(0, 0, q[p], qs[p], first[p], count[p])
        assert np.all(np.abs(single[p] - want) <= far), p


def zero_values_among_small_ones(rng, peak, qk, v, kv, lengths):
    """A cache whose values have peaks up to `peak`, every seventh of them all 0
    with the scale 1 that QuantizeInt8 gives it."""
    pool = Pool(rng, 1, sum(-(-n // 16) for n in lengths) + 1, 16, kv, qk, v, len(lengths), 40)
    pool.give(rng, lengths)
    pool.value_scales *= np.float32(peak / 127 / 0.03)
    for s, n in enumerate(lengths):
        for pos in range(s % 3, n, 7):
            p, at = pool.tables[s, pos // 16], pos % 16
            pool.values[0, p, :, at // 16, :, at % 16] = 0
            pool.value_scales[0, p, :, at] = 1.0
    return pool


@pytest.mark.parametrize("qk,v", DIMS)
@pytest.mark.parametrize("peak", [100.0, 1e-2, 1e-4, 1e-9])
def test_prompt_zero_values_among_small_ones(hip, qk, v, peak):
    """Values that are all 0 cost the others no digits (the first tile has some,
    with an attended whole tile after it; a run of zeros alone gives zeros)."""
    rng = np.random.default_rng(61)
    pool = zero_values_among_small_ones(rng, peak, qk, v, 2, [200, 90, 20])
    for p in pool.tables[2, :2]:
        pool.values[0, p], pool.value_scales[0, p] = 0, 1.0
    runs = [(60, 0, 140), (90, 1, 0), (20, 2, 0)]
    q, qs = queries(rng, 170, 4, qk)
    got = Gpu(hip, pool).prompt(0, q, qs, [0, 60, 150, 170], [0, 1, 2], [140, 0, 0], 0, 200)
    assert not got[150:].any()
    off = rms = 0.0
    for r, (s, p) in enumerate([(s, pos + j) for n, s, pos in runs[:2] for j in range(n)]):
        want, far = pool.attend_products(0, s, q[r], qs[r], 0, p + 1, True)
        assert np.all(np.abs(got[r] - want) <= far), r
        off, rms = off + np.sum((got[r] - want) ** 2), rms + np.sum(want ** 2)
    assert np.sqrt(off) <= 1e-5 * np.sqrt(rms)


@pytest.mark.parametrize("qk,v", DIMS)
@pytest.mark.parametrize("kv,group", [(2, 2), (2, 1)])
@pytest.mark.parametrize("peak", [100.0, 1e-4, 1e-9])
def test_decode_zero_values_among_small_ones(hip, peak, qk, v, kv, group):
    """As above, whole and in parts; a row of zeros alone gives zeros."""
    rng = np.random.default_rng(63)
    pool = zero_values_among_small_ones(rng, peak, qk, v, kv, [600, 90, 20])
    for p in pool.tables[2, :2]:
        pool.values[0, p], pool.value_scales[0, p] = 0, 1.0
    spec = [(0, 0, 600), (1, 0, 90), (0, 130, 77), (0, 599, 1), (1, 1, 1), (2, 0, 20)]
    q, qs = queries(rng, 6, kv * group, qk)
    gpu = Gpu(hip, pool)
    for max_count in (600, 640):
        got = gpu.decode(0, q, qs, *zip(*spec), max_count)
        assert not got[5].any()
        want, far = (np.stack(x) for x in zip(*[pool.attend_products(0, s, q[r], qs[r], f, n)
                                                for r, (s, f, n) in enumerate(spec)]))
        close(got, want, far)


@pytest.mark.parametrize("far_apart", [13, 40])
@pytest.mark.parametrize("window", [0, 300])
def test_prompt_large_scales_of_small_weight(hip, far_apart, window):
    """Value scales 2^13 and 2^40 times the others where the weight is about
    e^-30: the row is exact to its largest product of the two."""
    rng = np.random.default_rng(67)
    pool = Pool(rng, 1, 45, 16, 2, 64, 64, 1, 45)
    pool.give(rng, [700])
    pool.keys = rng.integers(-20, 21, pool.keys.shape, dtype=np.int8)
    for pos in (5, 64, 200, 207, 480):
        p, at = pool.tables[0, pos // 16], pos % 16
        pool.keys[0, p, :, at] = -120
        pool.key_scales[0, p, :, at] = 0.02
        pool.value_scales[0, p, :, at] *= np.float32(2.0 ** far_apart)
    gpu = Gpu(hip, pool)
    rows = 690
    q = rng.integers(60, 128, (rows, 4, 64), dtype=np.int8)
    qs = rng.uniform(0.015, 0.02, (rows, 4)).astype(np.float32)
    got = gpu.prompt(0, q, qs, [0, rows], [0], [10], window, 700)
    off, rms = 0.0, 0.0
    for r in range(0, rows, 3):
        first = max(0, 10 + r - window + 1) if window else 0
        want, far = pool.attend_products(0, 0, q[r], qs[r], first, 10 + r + 1 - first, True)
        assert np.all(np.abs(got[r] - want) <= far), r
        off, rms = off + np.sum((got[r] - want) ** 2), rms + np.sum(want ** 2)
    assert np.sqrt(off) <= 1e-5 * np.sqrt(rms)


@pytest.mark.parametrize("codes,scale", [(0, 1.0), (0, 0.0), (100, 0.0), (100, 1e-44)])
@pytest.mark.parametrize("kv,group", [(2, 2), (4, 1)])
def test_values_of_nothing_that_take_the_weight(hip, codes, scale, kv, group):
    """Every twentieth position has about e^14 times the others' weight and a
    value of 0, by its codes or by its scale: the others' digits stay."""
    rng = np.random.default_rng(73)
    pool = Pool(rng, 1, 45, 16, kv, 128, 128, 1, 45)
    pool.give(rng, [700])
    pool.keys = rng.integers(-20, 21, pool.keys.shape, dtype=np.int8)
    for pos in range(7, 700, 20):
        p, at = pool.tables[0, pos // 16], pos % 16
        pool.keys[0, p, :, at] = 100
        pool.key_scales[0, p, :, at] = 0.008
        pool.values[0, p, :, at // 16, :, at % 16] = codes
        pool.value_scales[0, p, :, at] = scale
    gpu = Gpu(hip, pool)
    q = rng.integers(90, 128, (700, kv * group, 128), dtype=np.int8)
    qs = rng.uniform(0.015, 0.016, (700, kv * group)).astype(np.float32)
    both = {True: gpu.prompt(0, q, qs, [0, 700], [0], [0], 0, 700),
            False: gpu.decode(0, q, qs, [0] * 700, [0] * 700, np.arange(1, 701), 700)}
    for prompt, got in both.items():
        for r in range(0, 700, 9):
            want, far = pool.attend_products(0, 0, q[r], qs[r], 0, r + 1, prompt)
            assert np.all(np.abs(got[r] - want) <= far), (prompt, r)


@pytest.mark.parametrize("score", [30.0, 100.0, 1000.0, -1000.0, 1e5])
@pytest.mark.parametrize("qk,v", DIMS)
@pytest.mark.parametrize("group", [1, 4])
def test_large_scores_that_nearly_tie(hip, score, qk, v, group):
    """Every position has the score up to its key scale's rounding.  In fp32 a
    score is off by three roundings of its own (those that a row's scores share
    move all its weights alike), each at most 2^-24 of it: 2^-24 |score| in the
    mean square, under 1e-7 |score|; 1e-5 where that is less."""
    rng = np.random.default_rng(83)
    pool = Pool(rng, 1, 20, 16, 2, qk, v, 1, 20)
    pool.give(rng, [300])
    base = rng.integers(60, 120, qk)
    pool.keys = (base + rng.integers(-7, 8, pool.keys.shape)).astype(np.int8)
    q = np.broadcast_to(rng.integers(60, 128, qk), (300, 2 * group, qk)).astype(np.int8)
    qs = rng.uniform(0.7, 1.0, (300, 2 * group)).astype(np.float32)
    dots = pool.keys.astype(np.float64) @ q[0, 0].astype(np.float64)
    live = ~np.isnan(pool.key_scales)
    pool.key_scales[live] = (score * np.sqrt(qk) / dots)[live]
    gpu, rows = Gpu(hip, pool), np.arange(0, 300, 5)
    both = {True: gpu.prompt(0, q, qs, [0, 300], [0], [0], 0, 300),
            False: gpu.decode(0, q, qs, [0] * 300, [0] * 300, np.arange(1, 301), 300)}
    for prompt, got in both.items():
        off = rms = 0.0
        for r in rows:
            want, far = pool.attend_products(0, 0, q[r], qs[r], 0, r + 1, prompt)
            assert np.all(np.abs(got[r] - want) <= far), (prompt, r)
            off, rms = off + np.sum((got[r] - want) ** 2), rms + np.sum(want ** 2)
        assert np.sqrt(off / rms) <= max(1e-5, 1e-7 * abs(score)), prompt


@pytest.mark.parametrize("scale", [0.0, 1e-44, 1e-30])
def test_prompt_scales_of_nothing(hip, scale):
    """Value scales of 0 or next to it, some of a sequence's and all of one's:
    what they hide is 0, the rest as exact as without it."""
    rng = np.random.default_rng(71)
    pool = Pool(rng, 1, 30, 16, 2, 64, 64, 2, 12)
    pool.give(rng, [170, 75])
    for pos in list(range(30, 90)) + [3, 100, 131]:
        pool.value_scales[0, pool.tables[0, pos // 16], :, pos % 16] = scale
    pool.value_scales[0, pool.tables[1, :5]] = scale
    q, qs = queries(rng, 245, 4, 64, 0.1)
    got = Gpu(hip, pool).prompt(0, q, qs, [0, 170, 245], [0, 1], [0, 0], 0, 170)
    assert np.abs(got[170:]).max() <= 128 * scale
    for r in range(0, 170, 3):
        want, far = pool.attend_products(0, 0, q[r], qs[r], 0, r + 1, True)
        assert np.all(np.abs(got[r] - want) <= far), r


@pytest.mark.parametrize("e", [-58, 58])
def test_scales_far_from_one(hip, e):
    """All value scales times 2^e, rows whole and in parts."""
    rng = np.random.default_rng(31)
    pool = Pool(rng, 1, 80, 16, 2, 64, 64, 1, 80)
    pool.give(rng, [1250])
    pool.value_scales *= np.float32(2.0 ** e)
    gpu = Gpu(hip, pool)
    q, qs = queries(rng, 30, 4, 64)
    check_prompt(gpu, 0, q, qs, [(30, 0, 1220)], 0, 1250)
    check_prompt(gpu, 0, q, qs, [(30, 0, 100)], 0, 130)
    check_decode(gpu, 0, q, qs, [(0, 0, 1250 - r) for r in range(30)], 1250)
    check_decode(gpu, 0, q, qs, [(0, r, 300) for r in range(30)], 300)


@pytest.mark.parametrize("runs,rows,kv", [(63, 40, 1), (65, 9, 1), (700, 3, 1), (4200, 2, 1), (255, 6, 3), (100, 4, 64),
                                          (256, 2, 1), (257, 2, 1)])
def test_prompt_many_runs(hip, runs, rows, kv):
    """Runs of 0 to `rows` rows, many of them empty, some longer than a tile."""
    rng = np.random.default_rng(33)
    pool = Pool(rng, 1, 60, 16, kv, 64, 64, 3, 20)
    pool.give(rng, [300, 150, 64])  # (every run lies in its sequence)
    spec = [(int(n), int(s), int(rng.integers(0, 8))) for n, s in zip(rng.integers(0, rows + 1, runs),
                                                                     rng.integers(0, 3, runs))]
    spec[runs // 3] = (131, 0, 100)
    spec[-1] = (70, 1, 3)
    spec[-2] = spec[0] = (0, 0, 0)
    q, qs = queries(rng, sum(n for n, _, _ in spec) + 5, 2 * kv if kv < 9 else kv, 64)
    check_prompt(Gpu(hip, pool), 0, q, qs, spec, 0, 300, rows_behind=5)


@pytest.mark.parametrize("kv,window", [(48, 0), (100, 0), (48, 20)])
def test_prompt_tiles_in_order_of_their_length(hip, kv, window):
    """More workgroups than CUs, of runs of different ends: each tile is taken once."""
    rng = np.random.default_rng(37)
    pool = Pool(rng, 1, 60, 16, kv, 48, 64, 4, 16)
    pool.give(rng, [200, 150, 40, 10])
    runs = [(3, 2, 37), (0, 1, 0), (133, 0, 40), (9, 1, 120), (1, 3, 9), (4, 9, 0), (20, 1, 0), (2, 0, 198)]
    q, qs = queries(rng, sum(n for n, _, _ in runs) + 2, kv, 48)
    check_prompt(Gpu(hip, pool), 0, q, qs, runs, window, 200, rows_behind=2)


def test_prompt_rows_out_of_range_and_behind(hip):
    """Runs of unknown sequences, before position 0 or past the table give
    zeros where a row is out of range; rows behind the last run stay."""
    rng = np.random.default_rng(16)
    big = 2 ** 31 - 1
    runs = [(3, -1, 0), (4, 9, 0), (5, 0, -2), (6, 0, 125), (2, 1, big), (3, 1, 0), (2, 0, 98)]
    pool = Pool(rng, 1, 40, 16, 2, 64, 64, 2, 8)
    pool.give(rng, [128, 30])
    gpu = Gpu(hip, pool)
    q, qs = queries(rng, 25 + 7, 4, 64)
    check_prompt(gpu, 0, q, qs, runs, 0, 128, rows_behind=7)
    got = check_prompt(gpu, 0, q, qs, runs, 0, 99, rows_behind=7)
    assert got[23].any() and not got[24].any()


def test_prompt_ignores_what_run_rows_may_not_say(hip):
    """Rows of a run outside [0, rows) are not touched, descending ends hold no rows."""
    rng = np.random.default_rng(17)
    pool = Pool(rng, 1, 40, 16, 1, 64, 64, 3, 8)
    pool.give(rng, [60, 60, 60])
    gpu = Gpu(hip, pool)
    q, qs = queries(rng, 10, 2, 64)
    got = gpu.prompt(0, q, qs, [-5, 4, 2, 2 ** 31 - 1], [0, 1, 2], [8, 0, 3], 0, 128)
    for r in range(10):  # run 0 has rows -5..3 (row r at position 8 + 5 + r), run 1 none, run 2 rows from 2 on
        want, far = pool.attend(0, 0, q[r], qs[r], 0, 14 + r, True)
        alt, alt_far = pool.attend(0, 2, q[r], qs[r], 0, 3 + r - 2 + 1, True) if r >= 2 else (want, far)
        ok = [np.abs(got[r] - w) <= f for w, f in ((want, far), (alt, alt_far))]
        assert np.all(ok[1] if r >= 4 else ok[0] | ok[1])


@pytest.mark.parametrize("left", [0xA5, 0x3F])
@pytest.mark.parametrize("group,window", [(1, 0), (1, 900), (3, 0)])
def test_prompt_split_of_runs_that_overlap(hip, left, group, window):
    """Ends that do not ascend, in a call that is split: the tiles of the last
    run find no place, so its own rows stay as they were whatever the workspace
    held; the other runs say the same of their rows, which are right."""
    rng = np.random.default_rng(17)
    heads, rows, ends = group, 300, [0, 260, 0, 260, 0, 260, 0, 260, 0, 260, 0, 260, 0, 300]
    pool = Pool(rng, 1, 45, 32, 1, 64, 64, 1, 48)
    pool.give(rng, [1400])
    gpu = Gpu(hip, pool)
    need = gpu.cache.prompt_workspace(rows, heads, 13, 1500)
    assert need > 0
    q, qs = queries(rng, rows, heads, 64)
    out = gpu.dev(np.full((rows, heads, 64), -77.0), np.float32)
    ws = gpu.dev(np.full(need, left), np.uint8)
    ends, zeros, pos = gpu.dev(ends), gpu.dev([0] * 13), gpu.dev([1100] * 13)
    gpu.cache.prompt(0, gpu.dev(q, np.int8).ptr, gpu.dev(qs, np.float32).ptr, rows, heads, 13, ends.ptr, zeros.ptr,
                     pos.ptr, window, 1500, ws.ptr, need, out.ptr)
    got = out.download(np.float32).reshape(rows, heads, 64)
    assert (got[260:] == -77.0).all()
    for r in range(0, 260, 7):
        first = max(0, 1100 + r - window + 1) if window else 0
        want, far = pool.attend(0, 0, q[r], qs[r], first, 1100 + r + 1 - first, True)
        assert np.all(np.abs(got[r] - want) <= far), r


def test_prompt_leaves_out_pages_outside_the_pool(hip):
    rng = np.random.default_rng(18)
    pool = Pool(rng, 1, 40, 16, 2, 64, 64, 2, 8)
    pool.give(rng, [100, 40])
    pool.tables[0, 0], pool.tables[0, 3], pool.tables[1, :] = -1, 40, 99999
    q, qs = queries(rng, 140, 4, 64)
    got = check_prompt(Gpu(hip, pool), 0, q, qs, [(100, 0, 0), (40, 1, 0)], 0, 128)
    assert not got[:16].any() and not got[100:].any()


def test_prompt_of_one_row_is_decode(hip):
    rng = np.random.default_rng(19)
    pool = Pool(rng, 1, 90, 16, 2, 48, 64, 4, 40)
    pool.give(rng, [600, 1, 77, 500])
    gpu = Gpu(hip, pool)
    q, qs = queries(rng, 4, 12, 48)
    a = check_prompt(gpu, 0, q, qs, [(1, 0, 599), (1, 1, 0), (1, 2, 76), (1, 3, 499)], 0, 640)
    b = check_decode(gpu, 0, q, qs, [(0, 0, 600), (1, 0, 1), (2, 0, 77), (3, 0, 500)], 640)
    assert np.sqrt(np.mean((a - b) ** 2)) <= 2e-5 * np.sqrt(np.mean(a ** 2))


# ---------------------------------------------------------------- append --

def expected_append(orc, pool, layer, k, v, seq, pos):
    for r in range(len(seq)):
        if not (0 <= seq[r] < pool.sequences and 0 <= pos[r] < pool.width * pool.page):
            continue
        p, at = pool.tables[seq[r], pos[r] // pool.page], pos[r] % pool.page
        if not 0 <= p < pool.pages:
            continue
        (qk, ks), (qv, vs) = orc.quantize_rows(k[r]), orc.quantize_rows(v[r])
        pool.keys[layer, p, :, at], pool.key_scales[layer, p, :, at] = qk, ks
        pool.values[layer, p, :, at // 16, :, at % 16], pool.value_scales[layer, p, :, at] = qv, vs


@pytest.mark.parametrize("qk,v", DIMS)
@pytest.mark.parametrize("page,kv", [(16, 2), (64, 3), (256, 1)])
def test_append(hip, orc, qk, v, page, kv):
    """Rows of any order and offset in strided columns; a long run, single
    tokens, rows that go nowhere."""
    rng = np.random.default_rng(qk + page + kv)
    pool = Pool(rng, 2, 40, page, kv, qk, v, 4, 8)
    pool.give(rng, [8 * page, 5 * page + 3, 2, 7 * page])
    pool.tables[2, 0] = -3
    spec = [(0, p) for p in range(3, 3 + 4 * page // 3)] + [(1, 5 * page + 2), (2, 1), (3, page), (-1, 0), (4, 0),
                                                             (1, -1), (3, 8 * page), (3, 7 * page - 1), (1, 0)]
    seq, pos = (np.array(x, dtype=np.int32) for x in zip(*spec))
    rows, ld = len(spec), 11 + kv * (qk + v) + 5
    x = (rng.standard_normal((rows, ld)) * np.exp(rng.standard_normal((rows, 1)) * 3)).astype(np.float32)
    x[3], x[5, 11:20] = 0.0, -0.0
    x[7] = np.round(x[7])
    gpu = Gpu(hip, pool)
    dx = gpu.dev(x, np.float32)
    gpu.cache.append(1, dx.ptr + 4 * 11, ld, dx.ptr + 4 * (11 + kv * qk), ld, gpu.dev(seq).ptr, gpu.dev(pos).ptr, rows)
    expected_append(orc, pool, 1, x[:, 11:11 + kv * qk].reshape(rows, kv, qk),
                    x[:, 11 + kv * qk:11 + kv * (qk + v)].reshape(rows, kv, v), seq, pos)
    for name in Pool.NAMES:
        assert np.array_equal(gpu.get(name), getattr(pool, name), equal_nan=name.endswith("scales")), name


@pytest.mark.parametrize("qk,v", DIMS)
def test_append_writes_no_page_that_others_hold(hip, orc, qk, v):
    """A step whose resize finds too few pages appends all the same (a graph
    does): no byte of a shared page changes, rows on pages of their own are
    written, and the step goes through once pages are free."""
    rng = np.random.default_rng(qk)
    pool = Pool(rng, 2, 5, 16, 2, qk, v, 4, 6)
    pool.give(rng, [40, 0, 0, 5])
    gpu, books = Gpu(hip, pool), Books(pool)
    ws = gpu.workspace(gpu.cache.pages_workspace(4))
    gpu.cache.fork(2, gpu.dev([1, 2]).ptr, gpu.dev([0, 0]).ptr, gpu.dev([20, 40]).ptr, *ws)
    books.fork([1, 2], [0, 0], [20, 40])
    before = pools(gpu)
    status = gpu.dev([9, 9])
    seq, length = [0, 1, 2, 3], [41, 21, 41, 6]
    gpu.cache.resize(4, gpu.dev(seq).ptr, gpu.dev(length).ptr, status.ptr, *ws)
    assert tuple(status.download(np.int32)) == books.resize(seq, length) == (1, 0)
    pos = [40, 20, 40, 5]
    x = rng.standard_normal((4, 2 * (qk + v))).astype(np.float32)
    dx, dseq, dpos = gpu.dev(x, np.float32), gpu.dev(seq), gpu.dev(pos)

    def append():
        gpu.cache.append(1, dx.ptr, x.shape[1], dx.ptr + 8 * qk, x.shape[1], dseq.ptr, dpos.ptr, 4)

    def expect(rows):
        for name in ("keys", "key_scales", "values", "value_scales"):
            setattr(pool, name, before[name].copy())
        pool.tables = books.tables
        for a, b in books.moved:
            for name in ("keys", "key_scales", "values", "value_scales"):
                getattr(pool, name)[:, b] = before[name][:, a]
        expected_append(orc, pool, 1, x[rows, :2 * qk].reshape(-1, 2, qk), x[rows, 2 * qk:].reshape(-1, 2, v),
                        [seq[r] for r in rows], [pos[r] for r in rows])
        for name in ("keys", "key_scales", "values", "value_scales"):
            assert np.array_equal(gpu.get(name), getattr(pool, name), equal_nan=True), name
        check_books(gpu, books)

    append()
    expect([3])
    gpu.cache.free(1, dseq.ptr + 8, *ws)  # sequence 2 ends: the last page of sequence 0 is its own
    books.resize([2], [0])
    append()
    expect([0, 3])
    before = pools(gpu)
    gpu.cache.resize(2, dseq.ptr, gpu.dev(length).ptr, status.ptr, *ws)
    assert tuple(status.download(np.int32)) == books.resize(seq[:2], length[:2]) == (0, 0)
    assert len(books.moved) == 1
    append()
    expect([0, 1, 3])


def test_append_of_over_a_million_workgroups(hip, orc):
    """70,000 rows of 256 kv heads, four of which go somewhere."""
    rng = np.random.default_rng(43)
    rows, kv, at = 70000, 256, [0, 17, 40000, 69999]
    pool = Pool(rng, 1, 6, 16, kv, 48, 64, 1, 6)
    pool.give(rng, [90])
    k = rng.standard_normal((4, kv, 48)).astype(np.float32)
    v = rng.standard_normal((4, kv, 64)).astype(np.float32)
    bufs = [hip.DeviceBuffer(4 * rows * kv * d) for d in (48, 64)]
    for b, x in zip(bufs, (k, v)):
        b.zero()
        for i, r in enumerate(at):
            b.upload(x[i], offset=r * x[i].nbytes)
    seq, pos = np.full(rows, -1, dtype=np.int32), np.arange(rows, dtype=np.int32)
    seq[at], pos[at] = 0, [3, 88, 50, 51]
    gpu = Gpu(hip, pool)
    gpu.cache.append(0, bufs[0].ptr, kv * 48, bufs[1].ptr, kv * 64, gpu.dev(seq).ptr, gpu.dev(pos).ptr, rows)
    expected_append(orc, pool, 0, k, v, seq[at], pos[at])
    for name in Pool.NAMES:
        assert np.array_equal(gpu.get(name), getattr(pool, name), equal_nan=name.endswith("scales")), name


# ----------------------------------------------------------------- pages --

def check_books(gpu, books, pool_before=None):
    tables, lengths, refs = gpu.books()
    assert np.array_equal(lengths, books.lengths)
    assert np.array_equal(tables, books.tables)
    assert np.array_equal(refs, books.refs)
    if pool_before is not None:
        for name in ("keys", "key_scales", "values", "value_scales"):
            want = pool_before[name].copy()
            for a, b in books.moved:
                want[:, b] = pool_before[name][:, a]
            assert np.array_equal(gpu.get(name), want, equal_nan=True), name


def pools(gpu):
    return {n: gpu.get(n) for n in ("keys", "key_scales", "values", "value_scales")}


def make(hip, seed, lengths, page=16, pages=40, width=8, layers=3, kv=2, qk=48, v=64):
    rng = np.random.default_rng(seed)
    pool = Pool(rng, layers, pages, page, kv, qk, v, len(lengths), width)
    pool.give(rng, lengths)
    return Gpu(hip, pool), Books(pool)


def test_reset(hip):
    gpu, books = make(hip, 1, [30, 0, 100])
    gpu.cache.reset()
    books.tables[:], books.lengths[:], books.refs[:] = -1, 0, 0
    check_books(gpu, books)


def test_copy(hip):
    gpu, books = make(hip, 2, [30, 17, 100])
    before = pools(gpu)
    src, dst = [3, 5, 3, -1, 40, 6, 7], [30, 31, 32, 33, 34, 40, 7]
    gpu.cache.copy(7, gpu.dev(src).ptr, gpu.dev(dst).ptr)
    books.moved = [(3, 30), (5, 31), (3, 32)]
    check_books(gpu, books, before)


@pytest.mark.parametrize("lengths", [None, [5, 200, 33, -4, 48, 7, 16, 9, 1]])
def test_fork(hip, lengths):
    """A permutation with repeats, a sequence onto itself, a name given twice,
    entries out of range."""
    gpu, books = make(hip, 3, [30, 17, 100, 0, 64, 1])
    before = pools(gpu)
    dst, src = [0, 1, 2, 3, 4, 0, 6, -1, 5], [2, 0, 2, 2, 1, 4, 1, 1, 99]
    ws = gpu.workspace(gpu.cache.pages_workspace(9))
    gpu.cache.fork(9, gpu.dev(dst).ptr, gpu.dev(src).ptr, gpu.dev(lengths).ptr if lengths else None, *ws)
    books.fork(dst, src, lengths)
    check_books(gpu, books, before)


def test_resize(hip):
    gpu, books = make(hip, 4, [30, 17, 100, 0, 64, 1], pages=40)
    before = pools(gpu)
    status = gpu.dev([9, 9])
    seq, length = [5, 3, 0, 2, 1, 4, 5, 7, 2], [1, 33, 31, 40, 128, 0, 100, 3, 129]
    ws = gpu.workspace(gpu.cache.pages_workspace(9))
    gpu.cache.resize(9, gpu.dev(seq).ptr, gpu.dev(length).ptr, status.ptr, *ws)
    want = books.resize(seq, length)
    assert tuple(status.download(np.int32)) == want == (0, 2)
    check_books(gpu, books, before)


def test_resize_changes_nothing_when_pages_are_missing(hip):
    gpu, books = make(hip, 5, [30, 17, 100, 0], pages=13)
    before = pools(gpu)
    status = gpu.dev([9, 9])
    seq, length = [3, 0, 2, -1], [50, 0, 110, 4]
    ws = gpu.workspace(gpu.cache.pages_workspace(4))
    for _ in range(2):
        gpu.cache.resize(4, gpu.dev(seq).ptr, gpu.dev(length).ptr, status.ptr, *ws)
        assert books.resize(seq, length) == (2, 1)
        assert tuple(status.download(np.int32)) == (2, 1)
        check_books(gpu, books, before)
    # once the pages given up are free the same growth succeeds
    gpu.cache.free(1, gpu.dev([0]).ptr, *ws)
    books.resize([0], [0])
    gpu.cache.resize(4, gpu.dev(seq).ptr, gpu.dev(length).ptr, None, *ws)
    assert books.resize(seq, length) == (0, 1)
    check_books(gpu, books, before)


def test_resize_of_more_than_the_pool(hip):
    gpu, books = make(hip, 6, [1] * 3, page=256, pages=20, width=1 << 22, layers=1)
    status = gpu.dev([9, 9])
    ws = gpu.workspace(gpu.cache.pages_workspace(3))
    gpu.cache.resize(3, gpu.dev([0, 1, 2]).ptr, gpu.dev([1 << 30] * 3).ptr, status.ptr, *ws)
    missing, refused = status.download(np.int32)
    assert refused == 0 and missing == 3 * 21 - 17
    assert np.array_equal(gpu.get("lengths"), books.lengths) and np.array_equal(gpu.get("refs"), books.refs)


@pytest.mark.parametrize("growers", [[0, 1, 2, 3], [2, 0], [3, 1, 2]])
def test_shared_pages_are_copied_before_they_grow(hip, growers):
    """Four holders of a partly filled page: all that grow copy it, except
    the last of them when nobody else holds it."""
    gpu, books = make(hip, 7, [40, 20, 0, 5], pages=40)
    dst, src = [1, 2, 3], [0, 0, 0]
    ws = gpu.workspace(gpu.cache.pages_workspace(4))
    gpu.cache.fork(3, gpu.dev(dst).ptr, gpu.dev(src).ptr, None, *ws)
    books.fork(dst, src)
    check_books(gpu, books)
    before = pools(gpu)
    length = [41 + 9 * g for g in growers]
    gpu.cache.resize(len(growers), gpu.dev(growers).ptr, gpu.dev(length).ptr, None, *ws)
    assert books.resize(growers, length) == (0, 0)
    assert len(books.moved) == min(len(growers), 3)
    check_books(gpu, books, before)


@pytest.mark.parametrize("pages", [1, 37, 5000, 20000])
def test_compact(hip, pages):
    rng = np.random.default_rng(pages)
    lengths = [int(n) for n in rng.integers(0, 16 * 30, 40)]
    while sum(-(-n // 16) for n in lengths) > pages:
        lengths.pop()
    lengths = lengths or [0]
    gpu, books = make(hip, pages, lengths, pages=pages, width=32, layers=2, kv=1)
    ws = gpu.workspace(gpu.cache.pages_workspace(len(lengths)))
    gone = list(range(0, len(lengths), 3))
    gpu.cache.free(len(gone), gpu.dev(gone).ptr, *ws)
    books.resize(gone, [0] * len(gone))
    if len(lengths) > 5:
        gpu.cache.fork(1, gpu.dev([0]).ptr, gpu.dev([4]).ptr, None, *ws)
        books.fork([0], [4])
    before = pools(gpu)
    status = gpu.dev([-1])
    gpu.cache.compact(status.ptr, *ws)
    n = books.compact()
    assert status.download(np.int32)[0] == n
    check_books(gpu, books, before)
    assert not gpu.get("refs")[n:].any()
    before = pools(gpu)  # a second time nothing moves
    gpu.cache.compact(None, *ws)
    books.compact()
    check_books(gpu, books, before)


def test_bookkeeping_against_the_model_at_random(hip):
    rng = np.random.default_rng(123)
    n, width = 60, 12
    gpu, books = make(hip, 8, [int(x) for x in rng.integers(0, 100, n)], pages=420, width=width, layers=1, kv=1)
    ws = gpu.workspace(gpu.cache.pages_workspace(n))
    for step in range(12):
        dst, src = rng.permutation(n)[:30], rng.integers(0, n, 30)
        length = rng.integers(0, 16 * width, 30)
        gpu.cache.fork(30, gpu.dev(dst).ptr, gpu.dev(src).ptr, gpu.dev(length).ptr if step % 2 else None, *ws)
        books.fork(dst, src, length if step % 2 else None)
        check_books(gpu, books)
        before = pools(gpu)
        seq = rng.permutation(n)
        length = np.clip(books.lengths[seq] + rng.integers(-20, 21, n), 0, 16 * width)
        status = gpu.dev([7, 7])
        gpu.cache.resize(n, gpu.dev(seq).ptr, gpu.dev(length).ptr, status.ptr, *ws)
        books.moved = []
        assert tuple(status.download(np.int32)) == books.resize(seq, length)
        check_books(gpu, books, before)
        if step % 4 == 3:
            before = pools(gpu)
            gpu.cache.compact(None, *ws)
            books.compact()
            check_books(gpu, books, before)


def test_1024_entries(hip):
    rng = np.random.default_rng(9)
    n = 1024
    gpu, books = make(hip, 9, [int(x) for x in rng.integers(1, 33, n)], pages=4000, width=4, layers=1, kv=1)
    ws = gpu.workspace(gpu.cache.pages_workspace(n))
    dst, src = rng.permutation(n), rng.integers(0, n, n)
    gpu.cache.fork(n, gpu.dev(dst).ptr, gpu.dev(src).ptr, None, *ws)
    books.fork(dst, src)
    check_books(gpu, books)
    before = pools(gpu)
    seq = rng.permutation(n)
    length = books.lengths[seq] + rng.integers(0, 20, n)
    gpu.cache.resize(n, gpu.dev(seq).ptr, gpu.dev(length).ptr, None, *ws)
    assert books.resize(seq, length) == (0, 0)
    check_books(gpu, books, before)


# ------------------------------------------------------------- together --

def test_a_server_s_steps(hip, orc):
    """Prompts enter, are attended, branch into beams, grow token by token
    (pages copied on write), one request ends, the pool is compacted and
    decoding goes on: after every step the attention of every live beam
    equals plain attention over the quantized keys and values of its own
    history, kept on the host."""
    from needle_cs_amd.paged import PagedCache
    rng = np.random.default_rng(77)
    layers, pages, page, kv, qk, v, heads, seqs, width = 2, 30, 16, 2, 48, 64, 12, 6, 6
    cache = PagedCache(layers, pages, page, kv, qk, v, seqs, width)
    keep = []

    def dev(a, dtype=np.int32):
        keep.append(hip.DeviceBuffer.from_array(np.ascontiguousarray(a, dtype=dtype)))
        return keep[-1].ptr

    wsn = cache.pages_workspace(seqs)
    ws = (hip.DeviceBuffer(wsn), wsn)
    history = {s: [] for s in range(seqs)}  # per position: (k, v) fp32 per layer

    def oracle(s, layer, q, qs, count):
        """Plain attention over the first `count` positions of s's history."""
        pool = Pool(rng, 1, -(-count // 16), 16, kv, qk, v, 1, -(-count // 16))
        pool.give(rng, [count])
        k = np.array([history[s][p][layer][0] for p in range(count)], dtype=np.float32).reshape(count, kv, qk)
        x = np.array([history[s][p][layer][1] for p in range(count)], dtype=np.float32).reshape(count, kv, v)
        expected_append(orc, pool, 0, k, x, [0] * count, list(range(count)))
        return pool.attend(0, 0, q, qs, 0, count, True)

    def feed(spec):
        """spec: (sequence, positions); appends random rows and checks their attention in every layer."""
        lens = {s: len(history[s]) for s, _ in spec}
        status = hip.DeviceBuffer.from_array(np.array([5, 5], dtype=np.int32))
        cache.resize(len(spec), dev([s for s, _ in spec]), dev([lens[s] + n for s, n in spec]), status.ptr, ws[0].ptr,
                     ws[1])
        assert not status.download(np.int32).any()
        rows = sum(n for _, n in spec)
        seq = [s for s, n in spec for _ in range(n)]
        pos = [lens[s] + j for s, n in spec for j in range(n)]
        raw = rng.standard_normal((layers, rows, kv * (qk + v))).astype(np.float32)
        r = 0
        for s, n in spec:
            for _ in range(n):
                history[s] = history[s] + [[(raw[l, r, :kv * qk], raw[l, r, kv * qk:]) for l in range(layers)]]
                r += 1
        for layer in range(layers):
            q, qs = queries(rng, rows, heads, qk)
            x = dev(raw[layer], np.float32)
            cache.append(layer, x, kv * (qk + v), x + 4 * kv * qk, kv * (qk + v), dev(seq), dev(pos), rows)
            out = hip.DeviceBuffer(4 * rows * heads * v)
            if all(n == 1 for _, n in spec):
                need = cache.decode_workspace(rows, heads, width * page)
                cache.decode(layer, dev(q, np.int8), dev(qs, np.float32), rows, heads, dev(seq), dev([0] * rows),
                             dev([p + 1 for p in pos]), width * page, dev(np.zeros(need + 16), np.uint8), need,
                             out.ptr)
            else:
                need = cache.prompt_workspace(rows, heads, len(spec), width * page)
                cache.prompt(layer, dev(q, np.int8), dev(qs, np.float32), rows, heads, len(spec),
                             dev(np.cumsum([0] + [n for _, n in spec])), dev([s for s, _ in spec]),
                             dev([lens[s] for s, _ in spec]), 0, width * page, dev(np.zeros(need + 16), np.uint8),
                             need, out.ptr)
            got = out.download(np.float32).reshape(rows, heads, v)
            for r in range(rows):
                want, far = oracle(seq[r], layer, q[r], qs[r], pos[r] + 1)
                assert np.all(np.abs(got[r] - want) <= far)

    feed([(0, 37), (3, 21)])
    for parents in ([0, 0, 0, 3, 3, 3], [1, 0, 1, 5, 4, 3], [2, 2, 0, 4, 4, 4]):
        cache.fork(6, dev(range(6)), dev(parents), None, ws[0].ptr, ws[1])
        history = dict(enumerate([list(history[p]) for p in parents]))
        feed([(s, 1) for s in range(6)])
    cache.free(2, dev([0, 4]), ws[0].ptr, ws[1])
    history[0], history[4] = [], []
    live = hip.DeviceBuffer.from_array(np.array([-1], dtype=np.int32))
    cache.compact(live.ptr, ws[0].ptr, ws[1])
    refs = cache.buffers["refs"].download(np.int32)
    n = int(live.download(np.int32)[0])
    assert (refs[:n] > 0).all() and not refs[n:].any()
    feed([(s, 1) for s in (1, 2, 3, 5)])
    feed([(0, 30), (1, 2), (4, 3)])
    cache.close()


def test_in_a_graph(hip, orc):
    """A decode step (branch, grow, append, attend both ways, one of them split
    over the length, compact) captured once and replayed: every replay equals
    the same calls made eagerly on a twin."""
    rng = np.random.default_rng(31)
    lengths = [40, 23, 16, 70]
    pool = Pool(rng, 1, 40, 16, 2, 64, 64, 4, 64)
    pool.give(rng, lengths)
    twins = [Gpu(hip, pool), Gpu(hip, pool)]
    q, qs = queries(rng, 4, 8, 64)
    x = rng.standard_normal((4, 256)).astype(np.float32)
    stream = hip.Stream()
    sets = []
    for gpu in twins:
        out = gpu.dev(np.zeros((4, 8, 64)), np.float32)
        seq, parents, grown, last, first, count = (gpu.dev(a) for a in ([0, 1, 2, 3], [1, 1, 3, 3], [24, 24, 71, 71],
                                                                        [23, 23, 70, 70], [0] * 4, [24, 24, 71, 71]))
        out2 = gpu.dev(np.zeros((4, 8, 64)), np.float32)
        runs = gpu.dev([0, 1, 2, 3, 4])
        parts = gpu.workspace(gpu.cache.prompt_workspace(4, 8, 4, 1024))
        dx, dq, ds = gpu.dev(x, np.float32), gpu.dev(q, np.int8), gpu.dev(qs, np.float32)
        pages, att = (gpu.workspace(n) for n in (gpu.cache.pages_workspace(4),
                                                 gpu.cache.decode_workspace(4, 8, 128)))
        status = gpu.dev([9, 9])

        def step(st, gpu=gpu, out=out, seq=seq, parents=parents, grown=grown, last=last, first=first, count=count,
                 dx=dx, dq=dq, ds=ds, pages=pages, att=att, status=status, out2=out2, runs=runs, parts=parts):
            c = gpu.cache
            c.fork(4, seq.ptr, parents.ptr, last.ptr, *pages, stream=st)
            c.resize(4, seq.ptr, grown.ptr, status.ptr, *pages, stream=st)
            c.append(0, dx.ptr, 256, dx.ptr + 512, 256, seq.ptr, last.ptr, 4, stream=st)
            c.decode(0, dq.ptr, ds.ptr, 4, 8, seq.ptr, first.ptr, count.ptr, 128, *att, out.ptr, stream=st)
            c.prompt(0, dq.ptr, ds.ptr, 4, 8, 4, runs.ptr, seq.ptr, last.ptr, 0, 1024, *parts, out2.ptr, stream=st)
            c.compact(None, *pages, stream=st)
        assert parts[1] > 0
        sets.append((gpu, out, step, out2))
    with hip.Graph.capture(stream) as graph:
        sets[0][2](stream.ptr)
    check_books(twins[0], Books(pool))  # capturing ran nothing
    other = hip.Stream()
    for _ in range(4):
        graph.launch()
        stream.sync()
        sets[1][2](other.ptr)
        other.sync()
        a, b = (s[1].download(np.float32) for s in sets)
        assert np.array_equal(a, b) and np.abs(a).max() > 0
        a2, b2 = (s[3].download(np.float32) for s in sets)
        assert np.array_equal(a2, b2) and np.abs(a2 - a).max() <= 1e-4 * np.abs(a).max()
        for name in Pool.NAMES:
            assert np.array_equal(twins[0].get(name), twins[1].get(name), equal_nan=True), name
    graph.close()


def test_two_streams_with_a_workspace_each(hip):
    rng = np.random.default_rng(41)
    pool = Pool(rng, 1, 200, 16, 2, 64, 64, 8, 60)
    pool.give(rng, [int(n) for n in rng.integers(100, 300, 8)])
    gpu = Gpu(hip, pool)
    q, qs = queries(rng, 8, 8, 64)
    streams = [hip.Stream(), hip.Stream()]
    calls = []
    for k in range(2):
        seq = [(s + k) % 8 for s in range(8)]
        count = [int(pool.lengths[s]) for s in seq]
        out = gpu.dev(np.zeros((8, 8, 64)), np.float32)
        ws = gpu.workspace(gpu.cache.decode_workspace(8, 8, 960))
        calls.append((gpu.dev(q, np.int8).ptr, gpu.dev(qs, np.float32).ptr, 8, 8, gpu.dev(seq).ptr,
                      gpu.dev([0] * 8).ptr, gpu.dev(count).ptr, 960, *ws, out.ptr, out, seq, count))
    for _ in range(20):
        for st, c in zip(streams, calls):
            gpu.cache.decode(0, *c[:11], stream=st.ptr)
    for st in streams:
        st.sync()
    for c in calls:
        got = c[11].download(np.float32).reshape(8, 8, 64)
        for r in range(8):
            want, far = pool.attend(0, c[12][r], q[r], qs[r], 0, c[13][r])
            assert np.all(np.abs(got[r] - want) <= far)
