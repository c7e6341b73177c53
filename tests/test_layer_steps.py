"""The entry points between a layer's int8 products (norm, rotary positions,
append and read, attention with sinks, sampling) refuse what they cannot do,
before any device work (no GPU here), and their structs have their declared
layouts."""
import ctypes as C

import pytest

import needle_cs_amd as N
from needle_cs_amd.rotary import BANDS, BASE, LINEAR, PARTS, Rotary, RotaryScaling, RotaryView, rotary_table
from needle_cs_amd.rows import add_rms_quantize, dequantize_rows
from needle_cs_amd.sampling import Sampling, sample, sample_workspace
from test_paged import A, BIG, cache, refused


def test_struct_layouts():
    assert C.sizeof(RotaryView) == 32 and RotaryView.positions.offset == 16 and RotaryView.interleaved.offset == 24
    assert C.sizeof(RotaryScaling) == 56 and RotaryScaling.kind.offset == 48
    assert C.sizeof(Sampling) == 40 and Sampling.min_p.offset == 32


@pytest.mark.parametrize("change,match", [
    ({"rows": -1}, "rows"), ({"rows": (1 << 26) + 1}, "rows"), ({"cols": 0}, "rows"), ({"cols": (1 << 20) + 1}, "rows"),
    ({"ldx": 63}, "strides"), ({"ldd": 63}, "strides"), ({"lds": 63}, "strides"), ({"x": None}, "null"),
    ({"q": None}, "null"), ({"scales": None}, "null"), ({"eps": 0.0}, "eps"), ({"eps": -1e-6}, "eps"),
    ({"eps": float("nan")}, "eps"), ({"eps": 2.0}, "eps"), ({"centered": 2}, "zero_centered"),
    ({"total": 0x10000, "x": 0x10000, "lds": 65}, "in place"), ({"total": 0x20000, "delta": 0x20000, "lds": 65}, "in place"),
])
def test_norm_refuses(change, match):
    d = dict(x=A, ldx=64, delta=A + 64, ldd=64, gain=A, centered=0, eps=1e-5, rows=2, cols=64, total=A + 128, lds=64, q=A,
             scales=A)
    d.update(change)
    with refused(match):
        add_rms_quantize(*d.values())


@pytest.mark.parametrize("args,match", [
    ((A, A, -1, 64, A, 64), "rows"), ((A, A, (1 << 26) + 1, 64, A, 64), "rows"), ((A, A, 1, 0, A, 64), "rows"),
    ((A, A, 1, 64, A, 63), "stride"), ((None, A, 1, 64, A, 64), "null"), ((A, None, 1, 64, A, 64), "null"),
    ((A, A, 1, 64, None, 64), "null"),
])
def test_dequantize_refuses(args, match):
    with refused(match):
        dequantize_rows(*args)


@pytest.mark.parametrize("change,match", [
    ({"dim": 0}, "even"), ({"dim": 7}, "even"), ({"dim": 514}, "even"), ({"first": -1}, "positions"),
    ({"count": -1}, "positions"), ({"first": 1 << 30, "count": 1}, "positions"), ({"cos": None}, "null"),
    ({"sin": None}, "null"), ({"theta": 1.0}, "theta"), ({"theta": float("nan")}, "theta"), ({"kind": 5}, "kind"),
    ({"kind": -1}, "kind"), ({"magnitude": 0.0}, "magnitude"), ({"magnitude": float("inf")}, "magnitude"),
    ({"kind": LINEAR, "factor": 0.5}, "factor"), ({"kind": BASE, "factor": float("nan")}, "factor"),
    ({"kind": BASE, "factor": 2.0, "dim": 2}, "2 dimensions"), ({"kind": PARTS, "original": 0.0}, "original"),
    ({"kind": PARTS, "original": 4096.0, "low": 0.0}, "low"), ({"kind": BANDS, "original": 4096.0, "low": 4.0, "high": 4.0}, "low"),
    ({"kind": BANDS, "original": 4096.0, "high": float("nan")}, "low"),
])
def test_rotary_table_refuses(change, match):
    d = dict(cos=A, sin=A, first=0, count=4, dim=64)
    d.update(change)
    with refused(match):
        rotary_table(**d)


def test_a_table_needs_a_scaling():
    assert N.lib().nhip_rotary_table_dev(A, A, 0, 4, 64, None, None) == -1
    with pytest.raises(ValueError):
        Rotary.make(0, 64)


@pytest.mark.parametrize("table,change,match", [
    ({"dim": 0}, {}, "even"), ({"dim": 63}, {}, "even"), ({"dim": 514}, {}, "even"), ({"positions": 0}, {}, "positions"),
    ({"cos": None}, {}, "table"), ({"sin": None}, {}, "table"), ({"interleaved": 2}, {}, "interleaved"),
    ({}, {"rows": -1}, "rows"), ({}, {"rows": (1 << 20) + 1}, "rows"), ({}, {"head_dim": 48}, "rotated"),
    ({}, {"head_dim": 4097, "ldx": 1 << 20, "ldy": 1 << 20}, "dimensions"), ({}, {"heads": 0}, "heads"),
    ({}, {"heads": 1 << 20, "ldx": 1 << 30, "ldy": 1 << 30}, "heads"), ({}, {"ldx": 255}, "strides"), ({}, {"ldy": 255}, "strides"),
    ({}, {"x": None}, "null"), ({}, {"pos": None}, "null"), ({}, {"y": None}, "null"), ({}, {"y": A, "ldy": 257}, "in place"),
])
def test_rotate_refuses(table, change, match):
    t = dict(cos=A, sin=A, positions=100, dim=64, interleaved=0)
    t.update(table)
    d = dict(x=A, ldx=256, heads=4, head_dim=64, pos=A, rows=3, y=A + 4096, ldy=256)
    d.update(change)
    with refused(match):
        Rotary(**t).rotate(*d.values())
    if table:  # the same table in the append
        with refused(match):
            cache(qk_dim=64).rotary_append(0, Rotary(**t), A, 256, 4, A, 128, A, 128, A, A, 3, A, A)


def test_no_table_is_refused():
    lib = N.lib()
    assert lib.nhip_rotary_dev(None, A, 64, 1, 64, A, 1, A, 64, None) == -1
    assert lib.nhip_paged_rotary_append_dev(cache().ptr, 0, None, A, 576, 12, A, 96, A, 128, A, A, 1, A, A, None) == -1
    with refused("rotary: null"):
        table = Rotary(A, A, 4, 4)
        table.close()
        table.rotate(A, 64, 1, 64, A, 1, A, 64)


@pytest.mark.parametrize("change,match", [
    ({"layer": 2}, "layer"), ({"layer": -1}, "layer"), ({"rows": -1}, "rows"), ({"rows": (1 << 20) + 1}, "rows"),
    ({"ldq": 575}, "strides"), ({"ldk": 95}, "strides"), ({"ldv": 127}, "strides"), ({"heads": 3}, "heads"),
    ({"heads": 0}, "heads"), ({"heads": 4098}, "heads"), ({"q": None}, "null"), ({"k": None}, "null"), ({"v": None}, "null"),
    ({"seq": None}, "null"), ({"pos": None}, "null"), ({"codes": None}, "null"), ({"scales": None}, "null"),
    ({"codes": A + 2}, "aligned"),
])
def test_rotary_append_refuses(change, match):
    d = dict(layer=0, rotary=Rotary(A, A, 100, 48), q=A, ldq=576, heads=12, k=A, ldk=96, v=A, ldv=128, seq=A, pos=A,
             rows=3, codes=A, scales=A)
    d.update(change)
    with refused(match):
        cache().rotary_append(*d.values())


def test_rotary_append_refuses_more_dimensions_than_a_head_has():
    with refused("rotated"):
        cache().rotary_append(0, Rotary(A, A, 100, 50), A, 576, 12, A, 96, A, 128, A, A, 3, A, A)


@pytest.mark.parametrize("args,match", [
    ((2, A, A, 1, A, 96, A, 128), "layer"), ((0, A, A, -1, A, 96, A, 128), "rows"), ((0, None, A, 1, A, 96, A, 128), "null"),
    ((0, A, None, 1, A, 96, A, 128), "null"), ((0, A, A, 1, None, 96, None, 128), "null"), ((0, A, A, 1, A, 95, A, 128), "strides"),
    ((0, A, A, 1, A, 96, A, 127), "strides"), ((0, A, A, 1, None, 0, A, 127), "strides"),
])
def test_read_refuses(args, match):
    with refused(match):
        cache().read(*args)


@pytest.mark.parametrize("other,match", [({"page_size": 24}, "page size"), ({"keys": None}, "null"), ({"width": 0}, "pages")])
def test_a_malformed_cache_is_refused_by_the_new_calls(other, match):
    c = cache(**other)
    for call in (lambda: c.rotary_append(0, Rotary(A, A, 9, 48), A, 576, 12, A, 96, A, 128, A, A, 1, A, A),
                 lambda: c.read(0, A, A, 1, A, 96, A, 128),
                 lambda: c.decode_sinks(0, A, A, 1, 2, A, A, A, 4, 16, A, BIG, A),
                 lambda: c.prompt_sinks(0, A, A, 1, 2, 1, A, A, A, 8, 4, 16, A, BIG, A)):
        with refused(match):
            call()
    assert c.decode_sinks_workspace(1, 2, 4, 16) == 0 and c.prompt_sinks_workspace(1, 2, 1, 4, 16) == 0


@pytest.mark.parametrize("change,match", [
    ({"layer": 2}, "layer"), ({"q": None}, "null"), ({"out": A + 8}, "aligned"), ({"rows": -1}, "rows"), ({"heads": 3}, "heads"),
    ({"max_count": 97}, "max_count"), ({"a": None}, "null"), ({"sinks": -1}, "sinks"),
])
def test_attention_with_sinks_refuses(change, match):
    d = dict(layer=0, q=A, q_scales=A, rows=3, heads=12, a=A, b=A, c=A, sinks=4, max_count=96, out=A)
    d.update(change)
    with refused(match):
        cache().decode_sinks(d["layer"], d["q"], d["q_scales"], d["rows"], d["heads"], d["a"], d["b"], d["c"], d["sinks"],
                             d["max_count"], A, BIG, d["out"])
    with refused(match):
        cache().prompt_sinks(d["layer"], d["q"], d["q_scales"], d["rows"], d["heads"], 1, d["a"], d["b"], d["c"], 8,
                             d["sinks"], d["max_count"], A, BIG, d["out"])


def test_sinks_workspaces():
    """Decode: rows * heads * parts * (64 + 2) * 4 bytes, with the sinks' blocks
    of 64 among a row's; no sinks: the other call's.  A prompt's covers its sinks,
    whatever they and its window are."""
    c = cache(pages=4096, width=4096)
    assert c.decode_sinks_workspace(4, 12, 4, 300) == 0
    assert c.decode_sinks_workspace(4, 12, 0, 60000) == c.decode_workspace(4, 12, 60000)
    # 1 row of 2 kv heads, 1024 / 64 + 2 + 1 = 19 blocks: 8 a part, 3 parts
    assert c.decode_sinks_workspace(1, 12, 4, 1088) == 12 * 3 * 264
    # sinks past what a sequence holds count as all of it
    assert c.decode_sinks_workspace(1, 12, 2 ** 31 - 1, 1024) == c.decode_sinks_workspace(1, 12, 4096 * 16, 1024)
    need = c.prompt_workspace(20, 12, 1, 60000)
    assert need > 0 and c.prompt_sinks_workspace(20, 12, 1, 99, 60000) == need
    for window in (1, 64, 4096, 60000, 2 ** 31 - 1):
        for sinks in (0, 1, 64, 50000, 2 ** 31 - 1):
            with refused("prompt: null"):
                c.prompt_sinks(0, A, A, 20, 12, 1, None, None, None, window, sinks, 60000, A, need, A)
    for ws, size in ((None, need), (A, need - 1), (A + 8, need)):
        with refused("workspace"):
            c.prompt_sinks(0, A, A, 20, 12, 1, A, A, A, 0, 4, 60000, ws, size, A)
    need = c.decode_sinks_workspace(1, 12, 4, 60000)
    for ws, size in ((None, need), (A, need - 1), (A + 8, need)):
        with refused("workspace"):
            c.decode_sinks(0, A, A, 1, 12, A, A, A, 4, 60000, ws, size, A)


@pytest.mark.parametrize("change,match", [
    ({"n": 0}, "ids"), ({"n": (1 << 19) + 1, "ldx": 1 << 20}, "ids"), ({"rows": -1}, "rows"), ({"rows": 65537}, "rows"),
    ({"ldx": 99}, "stride"), ({"x": None}, "null"), ({"ids": None}, "null"), ({"s": Sampling(None, A, A, A, A)}, "null"),
    ({"words": -1}, "mask"), ({"mask_ld": 3}, "mask"),
])
def test_sample_refuses(change, match):
    d = dict(x=A, ldx=100, n=100, rows=2, s=Sampling(A, None, None, None, None), mask=A, mask_ld=4, words=4, ws=A, size=BIG,
             ids=A, logprobs=A)
    d.update(change)
    with refused(match):
        sample(*d.values())


def test_sample_needs_its_settings_and_workspace():
    assert N.lib().nhip_sample_dev(A, 100, 100, 2, None, None, 0, 0, A, BIG, A, A, None) == -1
    assert sample_workspace(-1, 100) == 0 and sample_workspace(1, 0) == 0
    need = sample_workspace(1, 1 << 19)
    if need:
        for ws, size in ((None, need), (A, need - 1), (A + 8, need)):
            with refused("workspace"):
                sample(A, 1 << 19, 1 << 19, 1, Sampling(A), None, 0, 0, ws, size, A, A)


@pytest.mark.parametrize("rows,n", [(1, 1), (1, 1 << 19), (65536, 100), (300, 131071), (0, 5)])
def test_sampling_needs_no_workspace(rows, n):
    """Of whatever size; that it is not asked for says tests/test_sampling_gpu.py."""
    assert sample_workspace(rows, n) == 0


@pytest.mark.parametrize("rows,n", [(65537, 100), (-1, 100), (1, 0), (1, (1 << 19) + 1)])
def test_a_workspace_of_no_call_is_an_error(rows, n):
    """0 like those that need none, so the reason is left for last_error."""
    N.lib().nhip_rotary_table_dev(A, A, 0, 1, 3, None, None)
    assert sample_workspace(rows, n) == 0 and "sample" in N.last_error()


def test_nothing_to_do_is_no_error():
    c = cache()
    add_rms_quantize(None, 64, None, 0, None, 0, 1e-5, 0, 64, None, 0, None, None)
    dequantize_rows(None, None, 0, 64, None, 64)
    rotary_table(None, None, 5, 0, 64)
    Rotary(A, A, 100, 64).rotate(None, 64, 1, 64, None, 0, None, 64)
    c.rotary_append(0, Rotary(A, A, 100, 48), None, 576, 12, None, 96, None, 128, None, None, 0, None, None)
    c.read(0, None, None, 0, None, 96, None, 128)
    c.decode_sinks(0, None, None, 0, 12, None, None, None, 4, 16, None, 0, None)
    c.prompt_sinks(0, None, None, 0, 12, 0, None, None, None, 8, 4, 16, None, 0, None)
    sample(None, 100, 100, 0, Sampling(), None, 0, 0, None, 0, None, None)


@pytest.mark.parametrize("dims,whole", [((48, 64), 19), ((64, 64), 19), ((128, 128), 18)])
@pytest.mark.parametrize("sinks", [0, 1, 64, 65, 300])
def test_rows_are_cut_by_their_blocks_alone(dims, whole, sinks):
    """Where a decode call of few workgroups keeps a row in one part (and needs no workspace) is a number of blocks
    of 64 positions, whichever of them hold sinks."""
    c = cache(pages=4096, width=4096, qk_dim=dims[0], v_dim=dims[1])
    for blocks in range(10, 24):
        for extra in (0, 63):
            max_count = 64 * (blocks - 2 - -(-sinks // 64)) + extra
            need = c.decode_sinks_workspace(3, 12, sinks, max_count)
            parts = -(-blocks // 8)
            assert need == (0 if blocks <= whole else 3 * 12 * parts * (dims[1] + 2) * 4)
            if sinks == 0:
                assert need == c.decode_workspace(3, 12, max_count)


class Recorded:
    """A library that does nothing and says what was called, in order, and on which stream."""

    def __init__(self):
        self.calls, self.at = [], 0x100000

    def nhip_malloc(self, p, size):
        p._obj.value = self.at
        self.at += size
        return 0

    def nhip_free(self, p):
        return 0

    def nhip_rotary_table_dev(self, *args):
        self.calls.append(("table", args[-1]))
        return 0

    def nhip_stream_sync(self, stream):
        self.calls.append(("sync", stream))
        return 0


@pytest.mark.parametrize("stream", [None, 0x7000])
def test_a_table_is_whole_when_it_is_given_out(monkeypatch, stream):
    """Rotary.make waits for the stream that fills its table, whichever that is."""
    import needle_cs_amd.rotary
    fake = Recorded()
    for module in (N, needle_cs_amd.rotary):
        monkeypatch.setattr(module, "lib", lambda: fake)
    made = Rotary.make(10, 8, True, theta=500.0, stream=stream)
    assert fake.calls == [("table", stream), ("sync", stream)]
    made.close()
