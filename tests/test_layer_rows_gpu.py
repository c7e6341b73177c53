"""The residual's norm with QuantizeInt8, rows of codes read back, and rotary
positions on the GPU against plain numpy, bit for bit where every operation is
one rounding, and against 64 bits."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def dev(hip, a, dtype=None):
    return hip.DeviceBuffer.from_array(np.ascontiguousarray(a, dtype=dtype))


def quantize(h):
    """QuantizeInt8 of every row (src/Needle/Scalar.cs:67-74)."""
    peak = np.abs(h).max(-1, keepdims=True)
    scale = np.where(peak > 0, peak / np.float32(127), np.float32(1)).astype(np.float32)
    codes = np.clip(np.rint(h * (np.float32(1) / scale)), -128, 127).astype(np.int8)
    return codes, scale[..., 0]


def norm(x, delta, gain, centered, eps):
    s = x if delta is None else x + delta
    mean = (s.astype(np.float64) ** 2).sum(-1, keepdims=True) / s.shape[-1]
    r = (1.0 / np.sqrt(mean + np.float64(np.float32(eps)))).astype(np.float32)
    g = np.ones(s.shape[-1], np.float32) if gain is None else gain + np.float32(1) if centered else gain
    return s, *quantize((s * r) * g)


class NormCall:
    def __init__(self, hip, rng, rows, cols, pads=(0, 0, 0), delta=True, gain=True, centered=False, eps=1e-5, size=1.0):
        self.hip, self.rows, self.cols, self.centered, self.eps = hip, rows, cols, centered, eps
        self.ld = [cols + p for p in pads]
        self.x, self.delta = (rng.standard_normal((rows, ld)).astype(np.float32) * np.float32(size) for ld in self.ld[:2])
        self.gain = rng.standard_normal(cols).astype(np.float32) if gain else None
        self.dx, self.dd = dev(hip, self.x), dev(hip, self.delta) if delta else None
        self.dg = dev(hip, self.gain) if gain else None
        self.sum = dev(hip, np.full((rows, self.ld[2]), -7, np.float32))
        self.q, self.scales = dev(hip, np.full(rows * cols + 8, 77, np.int8)), dev(hip, np.full(rows, -7, np.float32))

    def run(self, total="sum", stream=None):
        from needle_cs_amd.rows import add_rms_quantize
        to, ld = {"sum": (self.sum, self.ld[2]), "x": (self.dx, self.ld[0]), "delta": (self.dd, self.ld[1]),
                  None: (None, 0)}[total]
        add_rms_quantize(self.dx.ptr, self.ld[0], self.dd.ptr if self.dd else None, self.ld[1],
                         self.dg.ptr if self.dg else None, self.centered, self.eps, self.rows, self.cols,
                         to.ptr if to else None, ld, self.q.ptr, self.scales.ptr, stream)
        return to, ld

    def check(self, total="sum"):
        c = self.cols
        want = norm(self.x[:, :c], self.delta[:, :c] if self.dd else None, self.gain, self.centered, self.eps)
        before = {"sum": np.full((self.rows, self.ld[2]), -7, np.float32), "x": self.x, "delta": self.delta}.get(total)
        to, ld = self.run(total)
        if to:
            got = to.download(np.float32).reshape(self.rows, ld)
            assert np.array_equal(got[:, :c], want[0]) and np.array_equal(got[:, c:], before[:, c:])
        q = self.q.download(np.int8)
        assert np.array_equal(q[:self.rows * c].reshape(self.rows, c), want[1]) and (q[self.rows * c:] == 77).all()
        assert np.array_equal(self.scales.download(np.float32), want[2])


@pytest.mark.parametrize("cols", [1, 2, 3, 4, 5, 63, 64, 255, 256, 257, 768, 1023, 1024, 1025, 2048, 4095, 4096, 4099, 8192,
                                  16384, 16385, 33000])
def test_norm_widths(hip, cols):
    rng = np.random.default_rng(cols)
    NormCall(hip, rng, 5, cols).check()
    NormCall(hip, rng, 3, cols, pads=(1, 2, 5), centered=True).check()


@pytest.mark.parametrize("cols", [100, 4000, 9001, 20001])
@pytest.mark.parametrize("total", [None, "x", "delta"])
def test_norm_in_place_and_without_sums(hip, cols, total):
    NormCall(hip, np.random.default_rng(cols), 7, cols, pads=(3, 3, 3)).check(total)


@pytest.mark.parametrize("cols", [96, 5000])
def test_norm_options(hip, cols):
    rng = np.random.default_rng(cols)
    NormCall(hip, rng, 4, cols, delta=False).check()
    NormCall(hip, rng, 4, cols, gain=False).check()
    NormCall(hip, rng, 4, cols, gain=False, centered=True).check()
    NormCall(hip, rng, 4, cols, eps=1.0).check()


@pytest.mark.parametrize("size", [1e-30, 1e-20, 1e15, 3e37])
def test_norm_of_extreme_rows(hip, size):
    """Squares that fp32 does not hold; 64 bits do."""
    NormCall(hip, np.random.default_rng(3), 6, 1500, size=size, eps=1e-38).check()


@pytest.mark.parametrize("rows,cols", [(1, 64), (4, 64), (5, 64), (70000, 16), (3001, 1000), (1000, 4096), (300, 10000)])
def test_norm_row_counts(hip, rows, cols):
    NormCall(hip, np.random.default_rng(rows), rows, cols).check()


@pytest.mark.parametrize("rows", [256, 257, 512, 513])
@pytest.mark.parametrize("cols", [33, 65, 128, 129, 300, 512, 513, 1000, 1024, 1030, 4093, 4100, 8192, 8193])
def test_norm_rows_by_columns(hip, rows, cols):
    """Every number of threads a row and of elements a thread, full and with ends inside a thread's four."""
    NormCall(hip, np.random.default_rng(rows + cols), rows, cols, pads=(0, 3, 1)).check()


@pytest.mark.parametrize("rows,cols", [(2101, 4003), (1030, 8192), (420, 20001), (140001, 60)])
@pytest.mark.parametrize("total", ["sum", "x"])
def test_norm_of_many_rows(hip, rows, cols, total):
    """More than 32 MB, whose sums are stored past the caches."""
    NormCall(hip, np.random.default_rng(cols), rows, cols, pads=(1, 2, 1)).check(total)


def test_norm_rows_of_zeros_and_of_nothing(hip):
    call = NormCall(hip, np.random.default_rng(1), 6, 520)
    call.x[1] = call.delta[1] = 0
    call.x[2, 7], call.x[3, 9], call.x[4, 11] = np.nan, np.inf, -np.inf
    call.dx.upload(call.x), call.dd.upload(call.delta)
    with np.errstate(invalid="ignore"):
        want = norm(call.x, call.delta, call.gain, False, call.eps)
    call.run()
    q, scales = call.q.download(np.int8, 6 * 520).reshape(6, 520), call.scales.download(np.float32)
    for r in (0, 1, 5):
        assert np.array_equal(q[r], want[1][r]) and scales[r] == want[2][r]
    assert (q[1] == 0).all() and scales[1] == 1


def test_norm_is_the_rows_calls_one_after_the_other(hip):
    """Its codes are nhip_quantize_rows_dev's of the normed rows."""
    call = NormCall(hip, np.random.default_rng(9), 33, 2048)
    call.run()
    s = call.x + call.delta
    r = (1.0 / np.sqrt((s.astype(np.float64) ** 2).sum(1, keepdims=True) / 2048 + float(np.float32(1e-5)))).astype(np.float32)
    h, q, scales = dev(hip, (s * r) * call.gain), hip.DeviceBuffer(33 * 2048), hip.DeviceBuffer(4 * 33)
    hip.check(hip.lib().nhip_quantize_rows_dev(h.ptr, 33, 2048, q.ptr, scales.ptr, None))
    assert np.array_equal(q.download(np.int8), call.q.download(np.int8, 33 * 2048))
    assert np.array_equal(scales.download(np.float32), call.scales.download(np.float32))


@pytest.mark.parametrize("rows,cols,pad", [(1, 1, 0), (7, 3, 2), (1000, 48, 0), (333, 50, 1), (99, 64, 0), (65, 65, 3), (64, 128, 0),
                                           (300000, 5, 0), (20, 4096, 8), (3, 70001, 0),
                                           (40, 129, 1), (9, 511, 0), (33, 512, 4), (31, 513, 0),
                                           (70001, 121, 2), (8200, 1024, 0)])
def test_dequantize(hip, rows, cols, pad):
    from needle_cs_amd.rows import dequantize_rows
    rng = np.random.default_rng(rows + cols)
    q = rng.integers(-128, 128, (rows, cols), dtype=np.int8)
    scales = rng.uniform(0.001, 3, rows).astype(np.float32)
    x = dev(hip, np.full((rows, cols + pad), -7, np.float32))
    dq, ds = dev(hip, q), dev(hip, scales)
    dequantize_rows(dq.ptr, ds.ptr, rows, cols, x.ptr, cols + pad)
    got = x.download(np.float32).reshape(rows, cols + pad)
    assert np.array_equal(got[:, :cols], q.astype(np.float32) * scales[:, None]) and (got[:, cols:] == -7).all()


# ---------------------------------------------------------------- rotary --

def frequencies(dim, theta=10000.0, kind=0, factor=1.0, low=1.0, high=32.0, original=0.0, magnitude=1.0):
    """In 64 bits, from the header's formulas."""
    out = []
    for i in range(dim // 2):
        f = math.exp(-2 * i / dim * math.log(theta))
        if kind == 1:
            f /= factor
        if kind == 2:
            f = math.exp(-2 * i / dim * (math.log(theta) + dim / (dim - 2) * math.log(factor)))
        if kind == 3:
            b = [dim * math.log(original / (2 * math.pi * t)) / (2 * math.log(theta)) for t in (high, low)]
            lo, hi = max(math.floor(b[0]), 0), min(math.ceil(b[1]), dim - 1)
            r = min(max((i - lo) / (hi - lo if hi != lo else 0.001), 0), 1)
            f = f / factor * r + f * (1 - r)
        if kind == 4:
            r = min(max((original * f / (2 * math.pi) - low) / (high - low), 0), 1)
            f = f / factor * (1 - r) + f * r
        out.append(f)
    return np.array(out)


SCALINGS = [{}, {"theta": 500000.0}, {"kind": 1, "factor": 4.0}, {"kind": 2, "factor": 8.0},
            {"kind": 3, "factor": 16.0, "original": 4096.0, "magnitude": 1.277}, {"kind": 3, "factor": 2.0, "original": 1.0},
            {"kind": 4, "factor": 8.0, "low": 1.0, "high": 4.0, "original": 8192.0}]


@pytest.mark.parametrize("scaling", SCALINGS)
@pytest.mark.parametrize("first,count,dim", [(0, 1, 4), (0, 300, 64), (5, 129, 48), (1000000, 77, 128), (2 ** 30 - 50, 50, 6),
                                             (131, 33, 512), (64, 64, 50)])
def test_table(hip, scaling, first, count, dim):
    """Values are rounded to fp32 once (2^-24 of themselves); an angle p f is
    off by up to 4 roundings of 64 bits (two of f on either side)."""
    from needle_cs_amd.rotary import rotary_table
    half = dim // 2
    c, s = (dev(hip, np.full(count * half + 3, -7, np.float32)) for _ in range(2))
    rotary_table(c.ptr, s.ptr, first, count, dim, **scaling)
    f = frequencies(dim, **scaling)
    angles = np.outer(np.arange(first, first + count, dtype=np.float64), f)
    for got, exact in ((c, np.cos(angles)), (s, np.sin(angles))):
        got = got.download(np.float32)
        exact = exact * scaling.get("magnitude", 1.0)
        far = 2.0 ** -24 * np.abs(exact) + (8 * np.abs(angles) + 8) * 2.0 ** -53 * 2
        assert (np.abs(got[:count * half].reshape(count, half) - exact) <= far).all()
        assert (got[count * half:] == -7).all()


def test_a_table_that_grows_is_the_same(hip):
    from needle_cs_amd.rotary import Rotary, rotary_table
    whole = Rotary.make(1000, 64, kind=3, factor=4.0, original=512.0)
    c, s = hip.DeviceBuffer(4 * 1000 * 32), hip.DeviceBuffer(4 * 1000 * 32)
    for first, count in ((0, 100), (100, 1), (101, 630), (731, 269)):
        rotary_table(c.ptr + 128 * first, s.ptr + 128 * first, first, count, 64, kind=3, factor=4.0, original=512.0)
    for a, b in zip(whole.buffers, (c, s)):
        assert np.array_equal(a.download(np.float32), b.download(np.float32))


def rotated(x, cos, sin, dim, interleaved):
    """x [rows][heads][head_dim] by the rows' cos and sin [rows][dim/2], every operation rounded to fp32."""
    y, half = x.copy(), dim // 2
    a, b = (slice(0, dim, 2), slice(1, dim, 2)) if interleaved else (slice(0, half), slice(half, dim))
    c, s = cos[:, None], sin[:, None]
    y[..., a] = x[..., a] * c - x[..., b] * s
    y[..., b] = x[..., b] * c + x[..., a] * s
    return y


def table(rng, positions, dim):
    """Cos and sin of angles of its own (rotation does not ask for a table made here)."""
    angles = rng.uniform(-3, 3, (positions, dim // 2))
    return np.cos(angles).astype(np.float32), np.sin(angles).astype(np.float32)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("rows,heads,head_dim,dim,pad,offset", [
    (1, 1, 2, 2, 0, 0), (3, 12, 48, 48, 0, 0), (5, 2, 64, 64, 4, 0), (70, 3, 128, 64, 1, 1), (33, 40, 128, 128, 0, 0),
    (9, 5, 50, 50, 3, 1), (9, 5, 50, 26, 2, 3), (17, 7, 80, 20, 0, 0), (4, 1, 512, 512, 0, 0), (2, 3, 600, 10, 0, 0),
    (11, 4, 6, 4, 1, 1), (2000, 2, 32, 24, 0, 0), (300, 9, 96, 40, 8, 0), (3, 2, 4096, 512, 0, 0), (5, 300, 64, 2, 0, 0),
])
def test_rotate(hip, rows, heads, head_dim, dim, pad, offset, interleaved):
    from needle_cs_amd.rotary import Rotary
    rng = np.random.default_rng(rows * 7 + head_dim + dim)
    cos, sin = table(rng, 90, dim)
    width = heads * head_dim
    x = rng.standard_normal((rows, width + pad)).astype(np.float32)
    pos = rng.integers(0, 90, rows).astype(np.int32)
    pos[rows // 2:rows // 2 + 1] = 89
    dc, ds, dp = dev(hip, cos), dev(hip, sin), dev(hip, pos)
    dx = dev(hip, np.concatenate([np.zeros(offset, np.float32), x.ravel()]))
    dy = dev(hip, np.full(offset + rows * (width + pad), -7, np.float32))
    r = Rotary(dc.ptr, ds.ptr, 90, dim, interleaved)
    want = rotated(x[:, :width].reshape(rows, heads, head_dim), cos[pos], sin[pos], dim, interleaved).reshape(rows, width)
    r.rotate(dx.ptr + 4 * offset, width + pad, heads, head_dim, dp.ptr, rows, dy.ptr + 4 * offset, width + pad)
    got = dy.download(np.float32)[offset:].reshape(rows, -1)
    assert np.array_equal(got[:, :width], want) and (got[:, width:] == -7).all()
    r.rotate(dx.ptr + 4 * offset, width + pad, heads, head_dim, dp.ptr, rows, dx.ptr + 4 * offset, width + pad)  # in place
    got = dx.download(np.float32)[offset:].reshape(rows, -1)
    assert np.array_equal(got[:, :width], want) and np.array_equal(got[:, width:], x[:, width:])


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("heads,head_dim,dim", [(32, 128, 128), (32, 128, 72), (40, 104, 8), (33, 64, 56)])
def test_rotate_many_rows(hip, heads, head_dim, dim, interleaved):
    """More than 32 MB, stored past the caches."""
    test_rotate(hip, 8500000 // (heads * head_dim) + 1, heads, head_dim, dim, 3, 1, interleaved)


@pytest.mark.parametrize("heads,head_dim,dim,interleaved", [(32, 128, 128, False), (33, 64, 56, True)])
def test_rotate_more_than_the_last_cache_keeps(hip, heads, head_dim, dim, interleaved):
    """160 MB and more, apart and in place."""
    test_rotate(hip, 40_000_000 // (heads * head_dim) + 1, heads, head_dim, dim, 3, 1, interleaved)


@pytest.mark.parametrize("dim,head_dim", [(64, 64), (12, 20)])
def test_rotate_leaves_rows_out_of_range(hip, dim, head_dim):
    from needle_cs_amd.rotary import Rotary
    rng = np.random.default_rng(4)
    cos, sin = table(rng, 30, dim)
    pos = np.array([0, -1, 29, 30, 2 ** 31 - 1, -2 ** 31, 7], dtype=np.int32)
    x = rng.standard_normal((7, 2 * head_dim)).astype(np.float32)
    dc, ds, dp, dx, dy = dev(hip, cos), dev(hip, sin), dev(hip, pos), dev(hip, x), dev(hip, np.full(x.shape, -7, np.float32))
    Rotary(dc.ptr, ds.ptr, 30, dim).rotate(dx.ptr, 2 * head_dim, 2, head_dim, dp.ptr, 7, dy.ptr, 2 * head_dim)
    got = dy.download(np.float32).reshape(x.shape)
    known = [0, 2, 6]
    want = rotated(x[known].reshape(3, 2, head_dim), cos[pos[known]], sin[pos[known]], dim, False).reshape(3, -1)
    assert np.array_equal(got[known], want) and (got[[1, 3, 4, 5]] == -7).all()


def test_rotate_past_32_bits(hip):
    """Rows and a table whose offsets pass 2^32 bytes (and 2^31 elements), sparse in what is looked at."""
    from needle_cs_amd.rotary import Rotary
    rng = np.random.default_rng(8)
    ld, rows, dim, positions = 1 << 21, 1100, 64, (1 << 25) + 9
    x, t = hip.DeviceBuffer(4 * ld * rows), hip.DeviceBuffer(4 * positions * (dim // 2))
    cos, sin = table(rng, 1, dim)
    head = rng.standard_normal((2, 64)).astype(np.float32)
    for at, h in zip((0, rows - 1), head):
        x.upload(h, 4 * ld * at)
    # (one array for cos and sin, at its two ends)
    t.upload(cos, 4 * (positions - 1) * (dim // 2))
    t.upload(cos, 0)
    pos = np.full(rows, -1, np.int32)
    pos[[0, -1]] = 0, positions - 1
    dp = dev(hip, pos)
    Rotary(t.ptr, t.ptr, positions, dim).rotate(x.ptr, ld, 1, 64, dp.ptr, rows, x.ptr, ld)
    for at, h in zip((0, rows - 1), head):
        want = rotated(h.reshape(1, 1, 64), cos, cos, dim, False).ravel()
        assert np.array_equal(x.download(np.float32, 64, 4 * ld * at), want)


def test_rows_on_a_stream_captured_and_replayed(hip):
    """Norm, read back and rotation recorded in a graph and replayed with new inputs, eager work on the same buffers between."""
    from needle_cs_amd.rotary import Rotary
    from needle_cs_amd.rows import dequantize_rows
    rng = np.random.default_rng(12)
    stream = hip.Stream()
    call = NormCall(hip, rng, 17, 768)
    cos, sin = table(rng, 64, 48)
    dc, ds, dp = dev(hip, cos), dev(hip, sin), dev(hip, np.zeros(17, np.int32))
    back, turned = hip.DeviceBuffer(4 * 17 * 768), hip.DeviceBuffer(4 * 17 * 768)
    r = Rotary(dc.ptr, ds.ptr, 64, 48)

    def steps(s):
        call.run("sum", s)
        dequantize_rows(call.q.ptr, call.scales.ptr, 17, 768, back.ptr, 768, s)
        r.rotate(back.ptr, 768, 16, 48, dp.ptr, 17, turned.ptr, 768, s)

    with hip.Graph.capture(stream) as graph:
        steps(stream.ptr)
    for k in range(4):
        call.x = rng.standard_normal((17, 768)).astype(np.float32)
        pos = rng.integers(0, 64, 17).astype(np.int32)
        call.dx.upload(call.x), dp.upload(pos)
        graph.launch()
        stream.sync()
        _, q, scales = norm(call.x, call.delta, call.gain, False, call.eps)
        values = q.astype(np.float32) * scales[:, None]
        want = rotated(values.reshape(17, 16, 48), cos[pos], sin[pos], 48, False).reshape(17, 768)
        assert np.array_equal(turned.download(np.float32).reshape(17, 768), want)
        turned.zero()
        steps(None)
        assert np.array_equal(turned.download(np.float32).reshape(17, 768), want)


def test_a_table_made_on_a_stream_is_read_by_another(hip):
    """Behind work of that stream; the other reads at once."""
    from needle_cs_amd.rotary import Rotary, rotary_table
    stream, other = hip.Stream(), hip.Stream()
    want = [b.download(np.float32) for b in Rotary.make(3000, 64, theta=500.0).buffers]
    room = hip.DeviceBuffer(4 << 20), hip.DeviceBuffer(4 << 20)
    for _ in range(20):
        rotary_table(room[0].ptr, room[1].ptr, 0, 1 << 15, 64, stream=stream.ptr)
    r = Rotary.make(3000, 64, theta=500.0, stream=stream.ptr)
    x, pos = np.ones((3000, 64), dtype=np.float32), np.arange(3000, dtype=np.int32)
    dx, dp, dy = hip.DeviceBuffer.from_array(x), hip.DeviceBuffer.from_array(pos), hip.DeviceBuffer(x.nbytes)
    r.rotate(dx.ptr, 64, 1, 64, dp.ptr, 3000, dy.ptr, 64, other.ptr)
    other.sync()
    cos, sin = (w.reshape(3000, 32) for w in want)
    assert np.array_equal(dy.download(np.float32).reshape(3000, 64), np.concatenate([cos - sin, cos + sin], axis=1))
