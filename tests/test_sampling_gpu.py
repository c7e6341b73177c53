"""Token ids drawn on the GPU against the definition in plain numpy: weights of
64 bits as whole multiples of 2^-42, sums of Python's or int64's whole numbers."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

INF = np.float32(np.inf)


def reference(x, mask, u, t, k, p, m):
    """(id, log-probability, margin) of one row; mask: booleans.  margin: how
    far (in weights' units) the draw is from another id, and the sums from a rule's border."""
    x = x.astype(np.float32)
    live = mask & (x > -INF)  # (NaN is not)
    ids = np.nonzero(live)[0]
    if not len(ids):
        return -1, -np.inf
    v = x[ids].astype(np.float64)
    order = np.lexsort((ids, -v))
    ids, v = ids[order], v[order]
    if not t > 0:
        return int(ids[0]), 0.0
    with np.errstate(invalid="ignore", over="ignore"):
        z = np.where(v == v[0], 0.0, (v - v[0]) / np.float64(t))
    z = np.where(np.isnan(z), -np.inf, z)
    w = np.rint(np.exp(z) * 2.0 ** 42).astype(np.int64)
    if k > 0:
        w[k:] = 0
    before = np.cumsum(w) - w
    keep = np.ones(len(w), dtype=bool)
    if p < 1:
        keep = before.astype(np.float64) < np.float64(p) * np.float64(w.sum())
        keep[0] = True
    if m > 0:
        keep &= w.astype(np.float64) >= min(np.float64(m), 1.0) * 2.0 ** 42
    w[~keep] = 0
    by_id = np.argsort(ids, kind="stable")
    upto = np.cumsum(w[by_id])
    total = int(upto[-1])
    r = min(max(np.float64(u), 0.0), 1.0) if u == u else 0.0
    at = min(int(np.floor(r * np.float64(total))), total - 1)
    j = by_id[int(np.searchsorted(upto, at, side="right"))]
    return int(ids[j]), z[j] - np.log(total / 2.0 ** 42)


class Call:
    def __init__(self, hip, x, random, temperature=None, top_k=None, top_p=None, min_p=None, mask=None, pad=0, offset=0, words=None):
        from needle_cs_amd.sampling import Sampling, sample_workspace
        self.hip, (self.rows, self.n) = hip, x.shape
        self.x, self.pad, self.offset, self.mask = x, pad, offset, mask
        self.settings = [None if a is None else np.broadcast_to(np.asarray(a, dtype=d), self.rows) for a, d in (
            (random, np.float32), (temperature, np.float32), (top_k, np.int32), (top_p, np.float32), (min_p, np.float32))]
        wide = np.full((self.rows, self.n + pad), np.float32(1e30))  # (what is not a logit is never taken)
        wide[:, :self.n] = x
        self.dx = hip.DeviceBuffer.from_array(np.concatenate([np.full(offset, 1e30, np.float32), wide.ravel()]))
        self.ds = [None if a is None else hip.DeviceBuffer.from_array(np.ascontiguousarray(a)) for a in self.settings]
        self.sampling = Sampling(*[None if d is None else d.ptr for d in self.ds])
        self.words = self.mask_ld = 0
        self.dm = None
        if mask is not None:
            self.words = -(-self.n // 32) if words is None else words
            self.mask_ld = self.words + 1
            bits = np.zeros((self.rows, self.mask_ld * 32), dtype=bool)
            full = mask[:, :min(self.n, 32 * self.words)]
            bits[:, :full.shape[1]] = full
            bits[:, min(32 * self.words, self.n):] = True  # (bits past the ids say nothing)
            self.mask = mask.copy()
            self.mask[:, 32 * self.words:] = False
            packed = np.packbits(bits, axis=1, bitorder="little").view(np.uint32)
            self.dm = hip.DeviceBuffer.from_array(packed)
        size = sample_workspace(self.rows, self.n)
        self.ws, self.size = hip.DeviceBuffer.from_array(np.full(max(size, 16), 0xA5, np.uint8)), size
        self.ids, self.logprobs = hip.DeviceBuffer(4 * self.rows), hip.DeviceBuffer(4 * self.rows)

    def run(self, stream=None, logprobs=True):
        from needle_cs_amd.sampling import sample
        sample(self.dx.ptr + 4 * self.offset, self.n + self.pad, self.n, self.rows, self.sampling, self.dm and self.dm.ptr,
               self.mask_ld, self.words, self.ws.ptr, self.size, self.ids.ptr, self.logprobs.ptr if logprobs else None, stream)

    def get(self):
        return self.ids.download(np.int32), self.logprobs.download(np.float32)

    def want(self):
        u, t, k, p, m = ([d] * self.rows if a is None else a for a, d in zip(self.settings, (0, 1.0, 0, 1.0, 0.0)))
        mask = np.ones(self.x.shape, dtype=bool) if self.mask is None else self.mask
        found = [reference(self.x[r], mask[r], u[r], t[r], int(k[r]), p[r], m[r]) for r in range(self.rows)]
        return np.array([f[0] for f in found]), np.array([f[1] for f in found])

    def check(self):
        self.run()
        ids, logprobs = self.get()
        want, exact = self.want()
        assert np.array_equal(ids, want), (np.nonzero(ids != want)[0][:5], ids[ids != want][:5], want[ids != want][:5])
        # rounded to fp32 once; 64 bits before
        none = want < 0
        assert (logprobs[none] == -np.inf).all()
        assert (np.abs(logprobs[~none] - exact[~none]) <= 2.0 ** -24 * np.abs(exact[~none]) + 1e-12).all()
        return ids


def logits(rng, rows, n, grid=0.0, size=2.5):
    x = rng.standard_normal((rows, n)) * size + np.minimum(np.exp(1.5 * rng.standard_normal((rows, n))), 12)
    return (np.round(x / grid) * grid if grid else x).astype(np.float32)


@pytest.mark.parametrize("n", [1, 2, 3, 4, 5, 63, 255, 256, 257, 1000, 4095, 4096, 4097, 32000, 40001, 131072, 1 << 19])
def test_widths(hip, n):
    rng = np.random.default_rng(n)
    rows = 6 if n < 100000 else 3
    x, u = logits(rng, rows, n), rng.random(rows)
    Call(hip, x, u).check()
    Call(hip, x, u, temperature=0.7, top_k=40, top_p=0.9, min_p=0.02, pad=3, offset=1).check()
    Call(hip, x, u, temperature=1.3, top_p=0.97).check()
    Call(hip, x, u, top_k=max(1, n // 2)).check()


@pytest.mark.parametrize("temperature", [0.0, 0.05, 0.7, 1.0, 3.0, 100.0])
@pytest.mark.parametrize("top_k", [0, 1, 2, 50, 1000, 3000])
@pytest.mark.parametrize("top_p", [0.1, 0.9, 0.999, 1.0])
def test_rules(hip, temperature, top_k, top_p):
    rng = np.random.default_rng(int(temperature * 10) + top_k)
    for grid in (0.0, 0.25):
        x = logits(rng, 8, 5003, grid)
        for min_p in (0.0, 0.05):
            Call(hip, x, rng.random(8), temperature, top_k, top_p, min_p).check()


def test_every_row_has_its_own_settings(hip):
    rng = np.random.default_rng(1)
    rows = 300
    x = logits(rng, rows, 3001, 0.125)
    Call(hip, x, rng.random(rows), rng.choice([0, 0.5, 1, 2], rows), rng.choice([0, 1, 7, 300, 5000], rows),
         rng.choice([0.3, 0.95, 1.0], rows), rng.choice([0.0, 0.01, 0.3], rows), rng.random((rows, 3001)) < 0.7).check()


def test_odd_settings(hip):
    """What counts as 'all ids', as 'the first', and what a number outside [0, 1) means."""
    rng = np.random.default_rng(2)
    x = logits(rng, 1, 700)
    nan, tiny = np.nan, 1e-30
    for t, k, p, m in ((nan, 0, 1.0, 0.0), (-1.0, 0, 1.0, 0.0), (1.0, -5, 2.0, -1.0), (1.0, 10 ** 9, nan, nan), (tiny, 0, 0.9, 0.0),
                       (1e-44, 5, 0.9, 0.1), (INF, 0, 1.0, 0.0), (INF, 9, 0.5, 0.5), (1e30, 20, 0.25, 0.0), (1.0, 0, 0.0, 0.0),
                       (1.0, 5, -1.0, 0.0), (1.0, 0, 1e-30, 0.0), (1.0, 0, 1.0, 7.0), (1.0, 0, 0.99999994, 1e-30)):
        for u in (0.0, 0.5, 0.99999994, 1.0, 5.0, -2.0, nan):
            Call(hip, x, u, t, k, p, m).check()


@pytest.mark.parametrize("n", [10, 5000, 70000])
def test_ties(hip, n):
    """Equal logits, more of them than are ranked one by one, cut inside by either rule: lower ids first."""
    rng = np.random.default_rng(n)
    flat = np.full((4, n), 1.5, dtype=np.float32)
    two = np.where(rng.random((4, n)) < 0.5, np.float32(2.0), np.float32(1.0))
    zero = np.where(rng.random((4, n)) < 0.5, np.float32(0.0), np.float32(-0.0))  # one value
    for x in (flat, two, zero):
        for k in (0, 1, n // 3, n - 1, n, n + 1):
            for p in (1.0, 0.5, 0.01):
                Call(hip, x, [0.0, 0.3, 0.8, 0.99999], 0.9, k, p, 0.0, rng.random((4, n)) < 0.8).check()


@pytest.mark.parametrize("n", [300, 4096, 4097, 5119, 40001, 262147])
@pytest.mark.parametrize("temperature", [0.3, 1.0, 2.0, 10.0, 1e6, 1e30, np.inf])
def test_a_share_of_the_mass(hip, n, temperature):
    """top_p alone, from bins of one id to bins of the whole row; draws in every part of a row and at its ends."""
    rng = np.random.default_rng(n)
    rows = 8 if n < 100000 else 4
    u = np.concatenate([[0.0, 1.0 - 2.0 ** -24], rng.random(rows - 2)])
    for grid in (0.0, 0.5):
        x = logits(rng, rows, n, grid)
        for p in (0.02, 0.5, 0.9, 0.999, 1.0 - 2.0 ** -24):
            Call(hip, x, u, temperature, None, p).check()
    Call(hip, x, u, temperature, None, 0.9, None, rng.random((rows, n)) < 0.3).check()
    wide = x.clip(-11.3, 11.3) * np.float32(3e37)
    Call(hip, wide, u, temperature, None, 0.7).check()


@pytest.mark.parametrize("n", [700, 4096, 16384, 1 << 17, (1 << 19) - 1, 1 << 19])
def test_neighbours(hip, n):
    """What is kept side by side in the row, at its start, its end and across powers of two."""
    rng = np.random.default_rng(n)
    kept = min(n // 2, 2000)
    for first in (0, n // 2 - kept // 2, n - kept, n // 4):
        x = rng.standard_normal((3, n)).astype(np.float32) - 12
        x[:, first:first + kept] += 11
        for k, p in ((kept - 100, 1.0), (kept, 0.9), (0, 0.8)):
            Call(hip, x, rng.random(3), 1.5, k, p).check()


@pytest.mark.parametrize("min_p", [1e-13, 1.5e-13, 2.0 ** -42, 4e-13, 7e-12])
def test_the_least_weights(hip, min_p):
    """Weights around min_p's, a few units of 2^-42 each, which round to it from below, in sum as much as the draw has left."""
    n, units = 1 << 19, min_p * 2.0 ** 42
    for first in (0.51, 0.9, 1.0, 1.1):
        x = np.full((2, n), np.float32(np.log((np.ceil(units) - 1 + first) / 2.0 ** 42)), dtype=np.float32)
        x[:, 0] = 0.0
        Call(hip, x, [1.0 - 2.0 ** -24, 0.5], 1.0, 0, 1.0, min_p).check()
        Call(hip, x, [1.0 - 2.0 ** -24, 0.5], 1.0, 0, 1.0 - 2.0 ** -24, min_p).check()


@pytest.mark.parametrize("rows,n", [(2, 2049), (2, 8192), (2, 8193), (2, 32767), (2, 32768), (2, 32769), (2, 100003), (258, 2048),
                                    (258, 2049), (258, 8192), (258, 8193)])
@pytest.mark.parametrize("top_k", [64, 65, 256, 257, 1800, 2300, 5000, 7900, 8300])
def test_many_kept(hip, rows, n, top_k):
    """Up to what a list holds and above, from rows that threads hold and from those that they read again."""
    rng = np.random.default_rng(n + top_k)
    for grid in (0.0, 0.125):
        Call(hip, logits(rng, rows, n, grid), rng.random(rows), 1.3, top_k, rng.choice([0.97, 1.0], rows)).check()
    x = np.sort(logits(rng, rows, n), axis=1)[:, ::-1]  # (all of them in a few threads' shares)
    x[0, 5] = np.inf
    Call(hip, np.ascontiguousarray(x), rng.random(rows), 1.3, top_k, None, None, rng.random((rows, n)) < 0.9).check()


def test_the_largest_weights(hip):
    """min_p = 1 keeps what rounds to the largest weight, also beside a largest logit of 0."""
    x = np.full((4, 5000), -30, dtype=np.float32)
    x[:, 40:60] = -np.float32(10.0) ** -np.arange(20)
    x[:, 60] = 0.0
    for t in (1e-5, 0.5, 1.0, 1e4):
        call = Call(hip, x, [0.0, 0.3, 0.7, 0.99], t, 0, 1.0, 1.0)
        call.check()
        call = Call(hip, x, [0.0, 0.3, 0.7, 0.99], t, 0, 0.8, 1.0)
        call.check()


@pytest.mark.parametrize("rows,n", [(257, 16384), (257, 16385), (256, 16384), (300, 5000)])
def test_many_rows(hip, rows, n):
    rng = np.random.default_rng(rows + n)
    Call(hip, logits(rng, rows, n, 0.125), rng.random(rows), rng.choice([0.0, 0.7, 1.0, 1.5], rows),
         rng.choice([0, 1, 40, 700, 3000, n - 1], rows), rng.choice([0.2, 0.9, 0.99, 1.0], rows),
         rng.choice([0.0, 0.0, 0.02], rows), rng.random((rows, n)) < 0.9).check()


def test_near_ties(hip):
    """Logits one step of fp32 apart, in one bin of the first histogram."""
    rng = np.random.default_rng(4)
    steps = rng.integers(0, 6000, (6, 20000))
    x = (np.float32(20).view(np.int32) + steps).astype(np.int32).view(np.float32)
    for k in (0, 17, 9000):
        for p in (1.0, 0.4):
            Call(hip, x, rng.random(6), 1.0, k, p).check()
    Call(hip, np.concatenate([x, np.full((6, 1), 20.5, np.float32)], 1), rng.random(6), 0.5, 7000, 0.8).check()


def test_values_that_are_no_numbers(hip):
    rng = np.random.default_rng(5)
    x = logits(rng, 12, 3000)
    x[0, ::3] = np.nan
    x[1, 5:] = -INF
    x[2] = -INF
    x[3] = np.nan
    x[4, [7, 9, 2999]] = INF
    x[5] = INF
    x[6, 0] = np.nan
    x[7] = np.finfo(np.float32).min  # the type's lowest, every one
    x[8, :1500] = np.finfo(np.float32).min
    x[9, 3], x[9, 4] = np.finfo(np.float32).max, np.finfo(np.float32).min
    x[10, :2000] = -INF
    x[11] = 1e-45
    for k, p, m in ((0, 1.0, 0.0), (2, 1.0, 0.0), (0, 0.5, 0.0), (40, 0.9, 0.1)):
        for t in (0.0, 1.0, 1e38, INF):
            Call(hip, x, rng.random(12), t, k, p, m).check()


@pytest.mark.parametrize("rows,n", [(64, 5000), (300, 9000), (64, 20000)])
@pytest.mark.parametrize("top_k", [3, 16, 17, 64, 65, 128, 200, 512])
def test_few_kept_of_those_listed(hip, rows, n, top_k):
    """min_p behind top_k alone: of the ids that are ranked against one another, by 16, 4 and 2 threads each, any
    number is dropped before the draw, none among them."""
    rng = np.random.default_rng(n + top_k)
    for grid in (0.0, 0.5):
        x = logits(rng, rows, n, grid)
        for min_p in (0.9, 0.3, 0.05, 1e-4):
            Call(hip, x, rng.random(rows), 1.0, top_k, None, min_p).check()


@pytest.mark.parametrize("n", [3, 900, 3001, 40003])
def test_signalling_nans(hip, n):
    """A NaN of any pattern is no id: quiet and signalling ones of both signs, in every row but the last alone
    among numbers, beside an infinity, and everywhere."""
    rng = np.random.default_rng(n)
    patterns = np.array([0x7F800001, 0xFF800001, 0x7FBFFFFF, 0xFFBFFFFF, 0x7FC00000, 0xFFFFFFFF], dtype=np.uint32)
    for k, p, m in ((0, 1.0, 0.0), (1, 1.0, 0.0), (40, 0.9, 0.0), (0, 0.5, 0.0), (700, 0.9, 0.01)):
        x = logits(rng, 16, n)
        bits = x.view(np.uint32)
        for r in range(6):
            bits[r, ::2] = patterns[r]
            bits[r + 6, 0] = patterns[r]
        bits[12, 1:] = rng.choice(patterns, n - 1)
        bits[13] = rng.choice(patterns, n)
        bits[14, 2:] = rng.choice(patterns, n - 2)
        x[14, 1] = INF
        mask = rng.random((16, n)) < 0.9
        for t in (0.0, 1.0):
            Call(hip, x, rng.random(16), t, k, p, m).check()
            Call(hip, x, rng.random(16), t, k, p, m, mask, pad=1, offset=1).check()


def test_masks(hip):
    rng = np.random.default_rng(6)
    x = logits(rng, 9, 10000)
    x[:, 9999] = 50  # the largest
    mask = rng.random((9, 10000)) < 0.5
    mask[0] = False
    mask[1] = True
    mask[2] = False
    mask[2, 9999] = True
    mask[3] = False
    mask[3, [0, 31, 32, 63]] = True
    for words in (313, 312, 5, 1, 0, 400):
        ids = Call(hip, x, rng.random(9), 1.0, 30, 0.95, 0.0, mask, words=words).check()
        assert ids[0] == -1


def test_whole_range_of_the_draw(hip):
    """Every id is drawn as often as it weighs: one row's distribution by 4096 numbers in [0, 1)."""
    rng = np.random.default_rng(7)
    x = logits(rng, 1, 300, size=1.0)
    u = (np.arange(4096) + 0.5) / 4096
    ids = Call(hip, np.repeat(x, 4096, 0), u, 1.0, 100).check()
    order = np.argsort(-x[0].astype(np.float64), kind="stable")[:100]
    e = np.exp(x[0, order].astype(np.float64) - x[0].max())
    share = np.zeros(300)
    share[order] = e / e.sum()
    # evenly spaced numbers meet an interval of length s within one of 4096 s times
    assert (np.abs(np.bincount(ids, minlength=300) - 4096 * share) <= 1).all()
    assert (np.diff(ids) >= 0).all()


def test_unaligned_rows(hip):
    rng = np.random.default_rng(8)
    for offset in (1, 2, 3):
        Call(hip, logits(rng, 5, 2049), rng.random(5), 0.8, 50, 0.9, 0.01, pad=offset, offset=offset).check()


def test_without_logprobs_and_settings(hip):
    rng = np.random.default_rng(9)
    call = Call(hip, logits(rng, 4, 900), rng.random(4))
    call.logprobs.upload(np.full(4, 3.0, np.float32))
    call.run(logprobs=False)
    ids, logprobs = call.get()
    assert np.array_equal(ids, call.want()[0]) and (logprobs == 3).all()


@pytest.mark.parametrize("n", [700, 32000, 131071])
def test_without_a_workspace(hip, n):
    """None of 0 bytes serves every way to a draw."""
    from needle_cs_amd.sampling import sample, sample_workspace
    rng = np.random.default_rng(n)
    for t, k, p, m in ((0.0, 0, 1.0, 0.0), (1.0, 0, 1.0, 0.0), (1.0, 50, 0.9, 0.0), (1.0, 0, 0.9, 0.0), (1.0, 600, 1.0, 0.01)):
        call = Call(hip, logits(rng, 3, n), rng.random(3), t, k, p, m)
        assert sample_workspace(3, n) == 0
        sample(call.dx.ptr, n, n, 3, call.sampling, None, 0, 0, None, 0, call.ids.ptr, call.logprobs.ptr)
        assert np.array_equal(call.get()[0], call.want()[0])


@pytest.mark.parametrize("rows,n", [(1, 32000), (3, 200000), (40, 32000)])
def test_captured_and_replayed(hip, rows, n):
    """A graph on a stream of its own with new logits and numbers for every replay, eager calls on the same
    buffers between, and another call with a workspace of its own at the same time."""
    rng = np.random.default_rng(rows)
    stream = hip.Stream()
    a = Call(hip, logits(rng, rows, n), rng.random(rows), 0.9, 60, 0.9, 0.01)
    b = Call(hip, logits(rng, rows, n, 0.25), rng.random(rows), 1.2, 0, 0.8)
    b.run()
    with hip.Graph.capture(stream) as graph:
        a.run(stream.ptr)
    want_b = b.want()[0]
    for k in range(4):
        x, u = logits(rng, rows, n, 0.0625 * (k % 2)), rng.random(rows).astype(np.float32)
        a.x, a.settings[0] = x, u
        a.dx.upload(x), a.ds[0].upload(u)
        hip.check(hip.lib().nhip_device_sync())
        graph.launch()
        b.run()
        stream.sync()
        want = a.want()[0]
        assert np.array_equal(a.get()[0], want) and np.array_equal(b.get()[0], want_b)
        a.run()
        assert np.array_equal(a.get()[0], want)


def test_fuzz(hip):
    rng = np.random.default_rng(10)
    for _ in range(60):
        n = int(np.exp(rng.uniform(0, np.log(30000))))
        rows = int(rng.integers(1, 12))
        x = logits(rng, rows, n, float(rng.choice([0, 0, 0.03125, 0.5])), float(rng.choice([0.01, 1, 5, 40])))
        Call(hip, x, rng.random(rows), rng.choice([0.0, 0.2, 0.8, 1.0, 5.0], rows), rng.choice([0, 1, 3, 50, 700, 20000], rows),
             rng.choice([0.05, 0.5, 0.9, 0.99, 1.0], rows), rng.choice([0.0, 0.001, 0.1], rows),
             rng.random((rows, n)) < 0.6 if rng.random() < 0.5 else None, int(rng.integers(0, 4)), int(rng.integers(0, 4))).check()
