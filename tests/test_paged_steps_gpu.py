"""The paged cache's rotated append, its read back and attention with sinks on
the GPU: bit for bit with the calls that they join, and against 64 bits within
the bound of paged_f64."""
import numpy as np
import pytest

from paged_f64 import FLOOR, PROMPT_LAG, Pool, bound
from test_layer_rows_gpu import dev, quantize, rotated, table
from test_paged_gpu import DIMS, Gpu, close, queries

pytestmark = pytest.mark.gpu


class Rows:
    """Rows of a fused projection, and where they go."""

    def __init__(self, hip, rng, pool, heads, spec, dim, positions, interleaved, pad=0):
        from needle_cs_amd.rotary import Rotary
        self.hip, self.pool, self.heads, self.dim, self.interleaved, self.positions = hip, pool, heads, dim, interleaved, positions
        self.rows, kv = len(spec), pool.kv
        self.width = heads * pool.qk + kv * (pool.qk + pool.v) + pad
        self.x = rng.standard_normal((self.rows, self.width)).astype(np.float32) * 3
        self.seq, self.pos = (np.array(a, dtype=np.int32) for a in zip(*spec))
        self.cos, self.sin = table(rng, positions, dim)
        self.dx, self.dseq, self.dpos = dev(hip, self.x), dev(hip, self.seq), dev(hip, self.pos)
        self.dc, self.ds = dev(hip, self.cos), dev(hip, self.sin)
        self.table = Rotary(self.dc.ptr, self.ds.ptr, positions, dim, interleaved)
        self.codes = dev(hip, np.full(self.rows * heads * pool.qk, 77, np.int8))
        self.scales = dev(hip, np.full(self.rows * heads, -7, np.float32))

    def append(self, cache, layer, stream=None):
        a, b = self.heads * self.pool.qk, (self.heads + self.pool.kv) * self.pool.qk
        cache.rotary_append(layer, self.table, self.dx.ptr, self.width, self.heads, self.dx.ptr + 4 * a, self.width,
                            self.dx.ptr + 4 * b, self.width, self.dseq.ptr, self.dpos.ptr, self.rows, self.codes.ptr,
                            self.scales.ptr, stream)

    def parts(self):
        """The rows' query heads rotated, keys rotated and values; rows out of the table have zeros."""
        qk, kv, n = self.pool.qk, self.pool.kv, self.rows
        known = (self.pos >= 0) & (self.pos < self.positions)
        at = np.where(known, self.pos, 0)
        x = self.x[:, :(self.heads + kv) * qk].reshape(n, -1, qk)
        y = rotated(x, self.cos[at], self.sin[at], self.dim, self.interleaved) * known[:, None, None].astype(np.float32)
        return y[:, :self.heads], y[:, self.heads:], self.x[:, (self.heads + kv) * qk:][:, :kv * self.pool.v].reshape(n, kv, -1)

    def check_queries(self):
        codes, scales = quantize(self.parts()[0])
        assert np.array_equal(self.codes.download(np.int8).reshape(codes.shape), codes)
        assert np.array_equal(self.scales.download(np.float32).reshape(scales.shape), scales)


def appended(pool, layer, rows):
    """The pool with the rows' keys and values in it, by position."""
    _, k, v = rows.parts()
    (kc, ks), (vc, vs) = quantize(k), quantize(v)
    for r in range(rows.rows):
        s, p = int(rows.seq[r]), int(rows.pos[r])
        if not (0 <= s < pool.sequences and 0 <= p < rows.positions and p // pool.page < pool.width):
            continue
        page, at = int(pool.tables[s, p // pool.page]), p % pool.page
        if not 0 <= page < pool.pages or pool.refs[page] > 1:
            continue
        pool.keys[layer, page, :, at], pool.key_scales[layer, page, :, at] = kc[r], ks[r]
        pool.values[layer, page, :, at // 16, :, at % 16], pool.value_scales[layer, page, :, at] = vc[r], vs[r]


def same_pools(gpu, pool):
    for name in ("keys", "key_scales", "values", "value_scales"):
        assert np.array_equal(gpu.get(name), getattr(pool, name), equal_nan=name.endswith("scales")), name


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("qk,v", DIMS)
@pytest.mark.parametrize("kv,group,dim,page,pad", [(1, 1, 0, 16, 0), (2, 6, 0, 16, 5), (3, 2, 20, 64, 1), (8, 4, 32, 32, 0),
                                                   (2, 1, 2, 256, 0), (1, 16, 46, 128, 3)])
def test_rotary_append(hip, qk, v, kv, group, dim, page, pad, interleaved):
    rng = np.random.default_rng(qk + 10 * kv + dim)
    pool = Pool(rng, 2, 60, page, kv, qk, v, 5, max(2, -(-330 // page) + 1))
    lengths = [1, 17, 330 if page < 256 else 200, 40, 0]
    pool.give(rng, lengths)
    gpu = Gpu(hip, pool)
    spec = [(0, 0), (1, 16), (3, 39)] + [(2, p) for p in range(3, min(lengths[2], 103))] + [(1, 3), (1, 2), (4, 0)]
    rows = Rows(hip, rng, pool, kv * group, spec, dim or qk, 330, interleaved, pad)
    rows.append(gpu.cache, 1)
    appended(pool, 1, rows)
    rows.check_queries()
    same_pools(gpu, pool)


@pytest.mark.parametrize("qk,v", DIMS)
def test_rotary_append_is_the_calls_one_after_the_other(hip, qk, v):
    rng = np.random.default_rng(qk)
    pool = Pool(rng, 1, 40, 16, 2, qk, v, 3, 12)
    pool.give(rng, [150, 33, 90])
    one, two = Gpu(hip, pool), Gpu(hip, pool)
    spec = [(0, p) for p in range(29, 150)] + [(2, p) for p in range(90)] + [(1, 32)]
    rows = Rows(hip, rng, pool, 12, spec, qk, 150, False)
    rows.append(one.cache, 0)
    n, y = rows.rows, hip.DeviceBuffer(4 * rows.rows * 14 * qk)
    rows.table.rotate(rows.dx.ptr, rows.width, 14, qk, rows.dpos.ptr, n, y.ptr, 14 * qk)
    two.cache.append(0, y.ptr + 4 * 12 * qk, 14 * qk, rows.dx.ptr + 4 * 14 * qk, rows.width, rows.dseq.ptr, rows.dpos.ptr, n)
    heads = np.ascontiguousarray(y.download(np.float32).reshape(n, 14, qk)[:, :12])
    q, scales = hip.DeviceBuffer(n * 12 * qk), hip.DeviceBuffer(4 * n * 12)
    dh = dev(hip, heads)
    hip.check(hip.lib().nhip_quantize_rows_dev(dh.ptr, n * 12, qk, q.ptr, scales.ptr, None))
    assert np.array_equal(q.download(np.int8), rows.codes.download(np.int8))
    assert np.array_equal(scales.download(np.float32), rows.scales.download(np.float32))
    for name in ("keys", "key_scales", "values", "value_scales"):
        assert np.array_equal(one.get(name), two.get(name), equal_nan=name.endswith("scales"))


def test_rotary_append_rows_out_of_range(hip):
    """They write nothing to the cache; outside the table their queries are 0 of scale 1, else rotated and quantized."""
    rng = np.random.default_rng(6)
    pool = Pool(rng, 1, 20, 16, 2, 64, 64, 4, 8)
    pool.give(rng, [64, 40, 128, 5])
    pool.refs[pool.tables[1, 1]] = 2  # shared
    pool.tables[2, 3], pool.tables[2, 4] = 20, -5
    gpu = Gpu(hip, pool)
    spec = [(0, 3), (-1, 4), (4, 4), (0, -1), (0, 100), (0, 63), (1, 17), (1, 15), (2, 50), (2, 70), (2, 90), (2, 2 ** 31 - 1),
            (0, -2 ** 31), (3, 20)]
    rows = Rows(hip, rng, pool, 4, spec, 64, 90, False)
    rows.append(gpu.cache, 0)
    appended(pool, 0, rows)
    rows.check_queries()
    same_pools(gpu, pool)
    assert (rows.scales.download(np.float32).reshape(-1, 4)[[3, 4, 10, 11, 12]] == 1).all()


def read(hip, gpu, layer, seq, pos, pads=(0, 0), keys=True, values=True):
    pool, n = gpu.pool, len(seq)
    ldk, ldv = pool.kv * pool.qk + pads[0], pool.kv * pool.v + pads[1]
    k, v = dev(hip, np.full((n, ldk), -7, np.float32)), dev(hip, np.full((n, ldv), -7, np.float32))
    ds, dp = dev(hip, seq, np.int32), dev(hip, pos, np.int32)
    gpu.cache.read(layer, ds.ptr, dp.ptr, n, k.ptr if keys else None, ldk, v.ptr if values else None, ldv)
    return k.download(np.float32).reshape(n, ldk), v.download(np.float32).reshape(n, ldv)


def check_read(hip, gpu, layer, spec, pads=(0, 0)):
    pool = gpu.pool
    seq, pos = zip(*spec)
    k, v = read(hip, gpu, layer, seq, pos, pads)
    a, b = pool.kv * pool.qk, pool.kv * pool.v
    assert (k[:, a:] == -7).all() and (v[:, b:] == -7).all()
    for r, (s, p) in enumerate(spec):
        for h in range(pool.kv):
            found = pool.position(layer, s, h, p) if 0 <= s < pool.sequences and 0 <= p < pool.width * pool.page else None
            want = (np.zeros(pool.qk), np.zeros(pool.v)) if found is None else (
                found[0].astype(np.float32) * found[1], found[2].astype(np.float32) * found[3])
            assert np.array_equal(k[r, h * pool.qk:(h + 1) * pool.qk], want[0])
            assert np.array_equal(v[r, h * pool.v:(h + 1) * pool.v], want[1])


@pytest.mark.parametrize("qk,v", DIMS)
@pytest.mark.parametrize("kv,page", [(1, 16), (2, 32), (3, 256), (16, 64)])
def test_read(hip, qk, v, kv, page):
    rng = np.random.default_rng(qk + kv + page)
    pool = Pool(rng, 2, 30, page, kv, qk, v, 4, -(-150 // page) + 1)
    pool.give(rng, [1, 150, 17, 0])
    gpu = Gpu(hip, pool)
    check_read(hip, gpu, 1, [(0, 0)])
    check_read(hip, gpu, 1, [(1, p) for p in range(150)], pads=(1, 2))
    check_read(hip, gpu, 1, [(1, p) for p in range(13, 130)] + [(2, p) for p in range(17)] + [(0, 0)])
    check_read(hip, gpu, 1, [(1, int(p)) for p in rng.permutation(150)[:60]] + [(2, 3)] * 5)


@pytest.mark.parametrize("consecutive", [False, True])
def test_read_many_rows(hip, consecutive):
    """More than 32 MB, stored past the caches."""
    rng = np.random.default_rng(7)
    pool = Pool(rng, 1, 40, 64, 4, 128, 128, 2, 8)
    pool.give(rng, [500, 300])
    at = np.tile(np.arange(499), 17) if consecutive else rng.integers(0, 500, 8400)
    check_read(hip, Gpu(hip, pool), 0, [(0, int(p)) for p in at], pads=(1, 2))


@pytest.mark.parametrize("qk,v", DIMS)
@pytest.mark.parametrize("consecutive", [False, True])
def test_read_more_than_the_last_cache_keeps(hip, qk, v, consecutive):
    """160 MB and more: the rows of a few positions over and over, as small calls give them."""
    rng = np.random.default_rng(8)
    pool = Pool(rng, 1, 40, 64, 4, qk, v, 2, 8)
    pool.give(rng, [500, 300])
    gpu = Gpu(hip, pool)
    few = np.arange(497) if consecutive else rng.integers(0, 500, 497)
    check_read(hip, gpu, 0, [(0, int(p)) for p in few], pads=(1, 2))
    want = read(hip, gpu, 0, [0] * 497, few, (1, 2))
    times = 40_000_000 // (497 * 4 * (qk + v)) + 1
    got = read(hip, gpu, 0, np.zeros(497 * times), np.tile(few, times), (1, 2))
    for a, b in zip(got, want):
        assert (a.reshape(times, *b.shape) == b).all()


def test_read_out_of_range(hip):
    rng = np.random.default_rng(2)
    pool = Pool(rng, 1, 12, 16, 2, 48, 64, 3, 6)
    pool.give(rng, [60, 30, 16])
    pool.tables[0, 1], pool.tables[0, 2] = 12, -7
    gpu = Gpu(hip, pool)
    check_read(hip, gpu, 0, [(0, p) for p in range(60)] + [(-1, 0), (3, 0), (0, -1), (0, 96), (0, 2 ** 31 - 1), (1, 40), (1, -2 ** 31)])
    k, v = read(hip, gpu, 0, [1], [5], keys=False)
    assert (k == -7).all() and (v != -7).all()
    k, v = read(hip, gpu, 0, [1], [5], values=False)
    assert (k != -7).all() and (v == -7).all()


def test_read_gives_what_append_wrote(hip):
    """Within half a step of QuantizeInt8's scale, the largest exactly (127 steps)."""
    rng = np.random.default_rng(3)
    pool = Pool(rng, 1, 40, 64, 4, 128, 128, 2, 8)
    pool.give(rng, [500, 300])
    gpu = Gpu(hip, pool)
    rows = Rows(hip, rng, pool, 8, [(0, p) for p in range(500)] + [(1, p) for p in range(300)], 64, 500, True)
    rows.append(gpu.cache, 0)
    k, v = read(hip, gpu, 0, rows.seq, rows.pos)
    _, wk, wv = rows.parts()
    for got, want in ((k.reshape(wk.shape), wk), (v.reshape(wv.shape), wv)):
        step = np.abs(want).max(-1, keepdims=True) / 127
        # half a step; the scale, its inverse, the product and the code's product each round (4 * 2^-24 of 127 steps)
        assert (np.abs(got - want) <= step * (0.5 + 127 * 4 * 2.0 ** -24)).all()


# ----------------------------------------------------------------- sinks --

def attend(pool, layer, seq, q, qs, at, prompt=False):
    """As Pool.attend, over the positions `at`."""
    heads = q.shape[0]
    out, far = np.zeros((heads, pool.v)), np.zeros((heads, pool.v))
    at = np.array(sorted(set(at)), dtype=np.int64)
    page = pool.tables[seq, at // pool.page]
    at, page = at[(page >= 0) & (page < pool.pages)], page[(page >= 0) & (page < pool.pages)]
    if not len(at):
        return out, far
    for h in range(heads):
        j = h // (heads // pool.kv)
        k = pool.keys[layer, page, j, at % pool.page].astype(np.float64)
        ks = pool.key_scales[layer, page, j, at % pool.page].astype(np.float64)
        v = pool.values[layer, page, j, at % pool.page // 16, :, at % 16].astype(np.float64)
        vs = pool.value_scales[layer, page, j, at % pool.page].astype(np.float64)
        z = (k @ q[h].astype(np.float64)) * ks * float(qs[h]) / np.sqrt(pool.qk)
        w = np.exp(z - z.max())
        w /= w.sum()
        out[h] = (w * vs) @ v
        far[h] = bound(len(at), np.abs(z).max(), vs) * ((w * np.abs(vs)) @ np.abs(v))
        far[h] += FLOOR * 2 * (vs.max() * PROMPT_LAG if prompt else (w * np.abs(vs)).max()) * np.abs(v).sum(0)
    return out, far


def run_decode(gpu, layer, q, qs, spec, sinks, max_count, stream=None):
    rows, heads = q.shape[:2]
    seq, first, count = (np.array(x) for x in zip(*spec))
    out = gpu.dev(np.full((rows, heads, gpu.pool.v), np.nan), np.float32)
    ws = gpu.workspace(gpu.cache.decode_sinks_workspace(rows, heads, sinks, max_count))
    gpu.cache.decode_sinks(layer, gpu.dev(q, np.int8).ptr, gpu.dev(qs, np.float32).ptr, rows, heads, gpu.dev(seq).ptr,
                           gpu.dev(first).ptr, gpu.dev(count).ptr, sinks, max_count, *ws, out.ptr, stream)
    return out.download(np.float32).reshape(rows, heads, gpu.pool.v)


def check_decode(gpu, layer, q, qs, spec, sinks, max_count):
    pool = gpu.pool
    got = run_decode(gpu, layer, q, qs, spec, sinks, max_count)
    want, far = np.zeros(got.shape), np.zeros(got.shape)
    for r, (s, f, n) in enumerate(spec):
        if 0 <= s < pool.sequences and f >= 0 and 0 < n <= max_count and f + n <= pool.width * pool.page:
            want[r], far[r] = attend(pool, layer, s, q[r], qs[r], [*range(min(sinks, f)), *range(f, f + n)])
    close(got, want, far)
    return got


def run_prompt(gpu, layer, q, qs, runs, window, sinks, max_count):
    rows, heads = q.shape[:2]
    starts = np.cumsum([0] + [n for _, _, n in runs])
    out = gpu.dev(np.full((rows, heads, gpu.pool.v), -77.0), np.float32)
    ws = gpu.workspace(gpu.cache.prompt_sinks_workspace(rows, heads, len(runs), sinks, max_count))
    gpu.cache.prompt_sinks(layer, gpu.dev(q, np.int8).ptr, gpu.dev(qs, np.float32).ptr, rows, heads, len(runs),
                           gpu.dev(starts).ptr, gpu.dev([s for s, _, _ in runs]).ptr, gpu.dev([p for _, p, _ in runs]).ptr,
                           window, sinks, max_count, *ws, out.ptr)
    return out.download(np.float32).reshape(rows, heads, gpu.pool.v)


def check_prompt(gpu, layer, q, qs, runs, window, sinks, max_count, every=1):
    """runs: (sequence, first position, rows); rows behind the last run stay as they are."""
    pool = gpu.pool
    got = run_prompt(gpu, layer, q, qs, runs, window, sinks, max_count)
    at, rows, want, far = 0, [], [], []
    for s, pos, n in runs:
        for i in range(0, n, every):
            p = pos + i
            rows.append(at + i)
            seen = [x for x in range(p + 1) if x > p - window or x < sinks] if window else range(p + 1)
            ok = 0 <= s < pool.sequences and pos >= 0 and p < max_count
            a = attend(pool, layer, s, q[at + i], qs[at + i], seen, prompt=True) if ok else (np.zeros(got.shape[1:]),) * 2
            want.append(a[0]), far.append(a[1])
        at += n
    close(got[rows], np.array(want), np.array(far))
    assert (got[at:] == -77).all()
    return got


@pytest.mark.parametrize("qk,v", DIMS)
@pytest.mark.parametrize("kv,group", [(1, 1), (2, 6), (3, 16), (16, 1), (2, 5)])
@pytest.mark.parametrize("sinks", [1, 4, 70])
def test_decode_sinks(hip, qk, v, kv, group, sinks):
    rng = np.random.default_rng(100 * qk + 10 * kv + group)
    lengths = [0, 1, 2, 64, 65, 130, 300, 500]
    pool = Pool(rng, 2, 90, 16, kv, qk, v, len(lengths), 33)
    pool.give(rng, lengths)
    spec = [(s, max(0, n - 64), min(n, 64)) for s, n in enumerate(lengths)]
    spec += [(7, 0, 300), (7, 1, 100), (7, 3, 1), (7, 63, 2), (7, 64, 64), (7, 65, 100), (7, 71, 3), (7, 130, 129), (7, 499, 1),
             (7, 200, 0), (6, 128, 172)]
    q, qs = queries(rng, len(spec), kv * group, qk)
    check_decode(Gpu(hip, pool), 1, q, qs, spec, sinks, 300)


@pytest.mark.parametrize("page", [16, 64, 256])
@pytest.mark.parametrize("sinks", [5, 64, 200])
def test_decode_sinks_pages(hip, page, sinks):
    rng = np.random.default_rng(page + sinks)
    pool = Pool(rng, 1, 3 * (1100 // page + 1), page, 2, 64, 64, 3, 1100 // page + 2)
    pool.give(rng, [1100, 700, 260])
    spec = [(0, 1000, 100), (0, 600, 500), (1, 193, 507), (2, 259, 1), (1, sinks, 65), (1, sinks - 1, 65), (0, sinks + 1, 63)]
    q, qs = queries(rng, len(spec), 8, 64)
    check_decode(Gpu(hip, pool), 0, q, qs, spec, sinks, 600)


@pytest.mark.parametrize("qk,v", DIMS)
@pytest.mark.parametrize("rows,kv,group", [(3, 1, 4), (2, 2, 1), (1, 4, 16)])
def test_decode_sinks_split(hip, qk, v, rows, kv, group):
    """Long windows of few rows: the length is split, the sinks in its first part (or parts)."""
    rng = np.random.default_rng(rows + kv)
    pool = Pool(rng, 1, 260, 64, kv, qk, v, 2, 200)
    pool.give(rng, [9001, 5000])
    gpu = Gpu(hip, pool)
    spec = [(0, 4000, 5001), (1, 900, 4100), (0, 70, 3000)][:rows]
    q, qs = queries(rng, rows, kv * group, qk)
    for sinks in (4, 700):
        check_decode(gpu, 0, q, qs, spec, sinks, 5001)


@pytest.mark.parametrize("qk,v", DIMS)
@pytest.mark.parametrize("sinks", [0, 4, 65])
def test_decode_sinks_at_the_longest_whole_rows(hip, qk, v, sinks):
    """Rows of 17 to 21 blocks, with and without sinks: whole, and in parts."""
    rng = np.random.default_rng(qk + sinks)
    pool = Pool(rng, 1, 200, 16, 2, qk, v, 2, 110)
    pool.give(rng, [1700, 1450])
    gpu = Gpu(hip, pool)
    q, qs = queries(rng, 4, 12, qk)
    for blocks in range(17, 22):
        n = 64 * (blocks - 2 - -(-sinks // 64)) + 20
        # (63 positions into a block: as many blocks as a row of n can have)
        check_decode(gpu, 0, q, qs, [(0, 127, n), (1, 191, n - 200), (1, 1450 - n, n), (0, 66, 5)], sinks, n)


@pytest.mark.parametrize("kv", [16, 48])
def test_decode_sinks_sorted(hip, kv):
    """Many whole rows, dealt out by their length."""
    rng = np.random.default_rng(kv)
    pool = Pool(rng, 1, 700, 16, kv, 64, 64, 40, 40)
    lengths = [int(n) for n in rng.integers(1, 260, 40)]
    pool.give(rng, lengths)
    spec = [(s, max(0, n - 100), min(n, 100)) for s, n in enumerate(lengths)]
    q, qs = queries(rng, 40, kv, 64)
    check_decode(Gpu(hip, pool), 0, q, qs, spec, 7, 100)


def test_decode_sinks_out_of_range_and_given_up_pages(hip):
    rng = np.random.default_rng(77)
    pool = Pool(rng, 1, 80, 16, 2, 64, 64, 3, 30)
    pool.give(rng, [400, 400, 100])
    pool.tables[0, 1:18] = [-1, 80, 2 ** 31 - 1, -2 ** 31] * 4 + [-1]  # between sinks and window
    pool.tables[1, 0] = -1  # the sinks' own page
    pool.key_scales[0, pool.tables[1, 3]] = np.nan  # positions that no row attends
    spec = [(0, 288, 112), (1, 100, 300), (1, 16, 20), (-1, 10, 5), (3, 10, 5), (2, 90, 391), (2, -1, 4), (2, 10, -1), (0, 380, 101),
            (2, 50, 50)]
    q, qs = queries(rng, len(spec), 4, 64)
    check_decode(Gpu(hip, pool), 0, q, qs, spec, 16, 390)


def test_no_sinks_is_the_call_without(hip):
    rng = np.random.default_rng(7)
    pool = Pool(rng, 1, 60, 16, 2, 128, 128, 2, 20)
    pool.give(rng, [300, 200])
    gpu = Gpu(hip, pool)
    spec = [(0, 100, 200), (1, 0, 200)]
    q, qs = queries(rng, 2, 8, 128)
    assert np.array_equal(run_decode(gpu, 0, q, qs, spec, 0, 300), gpu.decode(0, q, qs, *zip(*spec), 300))
    # sinks that the window holds already
    assert np.allclose(run_decode(gpu, 0, q, qs, [(0, 0, 300), (1, 0, 200)], 50, 300),
                       gpu.decode(0, q, qs, *zip(*[(0, 0, 300), (1, 0, 200)]), 300), rtol=1e-5, atol=1e-5)
    q, qs = queries(rng, 250, 8, 128)
    runs = [(0, 150, 150), (1, 100, 100)]
    a = gpu.prompt(0, q, qs, [0, 150, 250], [0, 1], [150, 100], 64, 300)
    assert np.array_equal(run_prompt(gpu, 0, q, qs, runs, 64, 0, 300), a)
    a = gpu.prompt(0, q, qs, [0, 150, 250], [0, 1], [150, 100], 0, 300)
    assert np.array_equal(run_prompt(gpu, 0, q, qs, runs, 0, 9, 300), a)


@pytest.mark.parametrize("qk,v", DIMS)
@pytest.mark.parametrize("kv,group", [(1, 1), (2, 6), (1, 16), (4, 3)])
@pytest.mark.parametrize("window,sinks", [(1, 1), (16, 4), (100, 70), (64, 64), (7, 130)])
def test_prompt_sinks(hip, qk, v, kv, group, window, sinks):
    rng = np.random.default_rng(qk + 10 * kv + window)
    pool = Pool(rng, 1, 90, 16, kv, qk, v, 4, 32)
    pool.give(rng, [330, 70, 1, 500])
    runs = [(0, 0, 330), (1, 3, 67), (2, 0, 1), (3, 450, 50), (1, 0, 0)]
    q, qs = queries(rng, sum(r[2] for r in runs) + 3, kv * group, qk)
    check_prompt(Gpu(hip, pool), 0, q, qs, runs, window, sinks, 500, every=3)


@pytest.mark.parametrize("qk,v", DIMS)
def test_prompt_sinks_split(hip, qk, v):
    """Few rows far into a stream with a wide window: the length is split."""
    rng = np.random.default_rng(qk)
    pool = Pool(rng, 1, 260, 64, 2, qk, v, 2, 200)
    pool.give(rng, [9001, 5000])
    gpu = Gpu(hip, pool)
    runs = [(0, 8981, 20), (1, 4995, 5)]
    q, qs = queries(rng, 25, 8, qk)
    for window, sinks in ((4000, 4), (3000, 900), (100, 300), (20000, 8)):
        check_prompt(gpu, 0, q, qs, runs, window, sinks, 9001, every=4)


def test_prompt_sinks_many_runs_and_pages_given_up(hip):
    rng = np.random.default_rng(5)
    pool = Pool(rng, 1, 900, 16, 8, 64, 64, 60, 16)
    pool.give(rng, [int(n) for n in rng.integers(150, 240, 60)])
    for s in range(0, 60, 2):
        pool.tables[s, 1:3] = -1
    for s in (1, 7):
        pool.tables[s, 0] = -1
    runs = [(s, int(pool.lengths[s]) - 60, 60) for s in range(60)] + [(-1, 0, 3), (60, 0, 2), (3, -5, 4)]
    q, qs = queries(rng, sum(r[2] for r in runs), 16, 64)
    check_prompt(Gpu(hip, pool), 0, q, qs, runs, 40, 6, 240, every=7)
