"""The steps of a server's own layers around the paged int8 cache, as a program
of its users calls them, for timing and comparing.

kind "norm"     residual + delta, its root-mean-square norm with gains, and
                QuantizeInt8 per row (the rows of the next int8 product); the
                codes are read back as the values they stand for
kind "table"    cos and sin of positions times a head's frequencies, scaled
                for long contexts
kind "rotate"   query and key heads of a fused projection rotated by position,
                the first `dim` dimensions of each head
kind "append"   queries rotated and quantized per head, keys rotated, and keys
                and values quantized into their sequences' pages; the codes
                and the cached rows are read back as the values they stand for
kind "decode"   attention of one new token of each of `rows` sequences over the
                last `window` positions and the first `sinks`
kind "prompt"   causal attention of packed prompts over the same positions
kind "sample"   one token id per row of logits: temperature, the first top_k by
                value, the smallest set of mass top_p, weights of min_p of the
                largest; drawn with a given number in [0, 1)

The cache's arrays:

    keys    int8 [layers][pages][kv_heads][page][qk]        key_scales   fp32 [layers][pages][kv_heads][page]
    values  int8 [layers][pages][kv_heads][page/16][v][16]  value_scales fp32 [layers][pages][kv_heads][page]
    tables  int32 [sequences][width] (-1 past a sequence's pages), lengths int32 [sequences],
    refs    int32 [pages], the number of sequences that hold a page (0: free)

`own` False computes them in elementary torch operations, True through
needle_cs_amd.
"""
from __future__ import annotations

import math
import random

import torch

own = False

#: Weights of a row's ids are whole multiples of this part of the largest one's.
UNIT = 2.0 ** -42


def listed() -> list[dict]:
    return [
        # a beam-3 step's rows of Needle 3's width: launch latency
        {"name": "norm_beam3", "kind": "norm", "rows": 3, "cols": 768, "pad": 0, "centered": True},
        # a batch of prompts through a wide layer, the rows in a wider matrix: the bytes bound it
        {"name": "norm_prompts", "kind": "norm", "rows": 4099, "cols": 4096, "pad": 64, "centered": False},
        # a server starts with room for long contexts
        {"name": "table_long", "kind": "table", "positions": 131072, "dim": 128, "scaling": "parts"},
        # one step of 16 sequences, the benchmark decoder's heads
        {"name": "rotate_step", "kind": "rotate", "rows": 16, "heads": 32, "head_dim": 64, "dim": 64, "pad": 1024,
         "interleaved": False, "positions": 2048},
        # packed prompts of 40 query and key heads of 128, half of each head rotated, pairs side by side
        {"name": "rotate_prompts", "kind": "rotate", "rows": 8185, "heads": 40, "head_dim": 128, "dim": 64,
         "pad": 1024, "interleaved": True, "positions": 40000},
        # one decode step's rows of 16 sequences, Needle 3's heads: launch latency
        {"name": "append_step", "kind": "append", "sequences": 16, "run": 1, "heads": 12, "kv_heads": 2, "qk": 48,
         "v": 64, "page": 16, "context": 1000, "dim": 48, "interleaved": False},
        # a batch of prompts entering the cache, wide grouped heads, ends inside pages
        {"name": "append_prompts", "kind": "append", "sequences": 5, "run": 1637, "heads": 32, "kv_heads": 8,
         "qk": 128, "v": 128, "page": 64, "context": 2048, "dim": 128, "interleaved": False},
        # a beam-3 step far into a stream, Needle 3's heads and window
        {"name": "decode_beam3", "kind": "decode", "rows": 3, "heads": 12, "kv_heads": 2, "qk": 48, "v": 64,
         "page": 16, "window": 1024, "sinks": 4, "lo": 900, "hi": 5000},
        # many long streams, grouped heads: the attended positions' bytes bound it
        {"name": "decode_streams", "kind": "decode", "rows": 48, "heads": 32, "kv_heads": 8, "qk": 128, "v": 128,
         "page": 64, "window": 8192, "sinks": 16, "lo": 4097, "hi": 32768},
        # prompts longer than the window, one behind a prefix
        {"name": "prompt_streams", "kind": "prompt", "runs": 3, "lo": 417, "hi": 6000, "prefix": 2500, "heads": 12,
         "kv_heads": 2, "qk": 48, "v": 64, "page": 16, "window": 1024, "sinks": 4},
        # one answer's next token with the usual settings, the benchmark decoder's vocabulary
        {"name": "sample_one", "kind": "sample", "rows": 1, "n": 32000, "pad": 0, "temperature": 0.8, "top_k": 50,
         "top_p": 0.95, "min_p": 0.0, "masked": False, "grid": 0.0},
        # a server's batch, every request with settings of its own, some under a grammar's mask; logits on a
        # coarse grid, as 16-bit heads leave them, so that many tie
        {"name": "sample_batch", "kind": "sample", "rows": 250, "n": 131071, "pad": 1, "temperature": -1.0,
         "top_k": -1, "top_p": -1.0, "min_p": -1.0, "masked": True, "grid": 0.0625},
    ]


def _log(rng, lo: int, hi: int) -> int:
    """An integer in [lo, hi], even over its logarithm."""
    return min(max(int(round(math.exp(rng.uniform(math.log(lo), math.log(hi))))), lo), hi)


def draw(rng) -> dict:
    kind = rng.choice(["norm", "norm", "table", "rotate", "append", "append", "decode", "decode", "prompt", "prompt",
                       "sample", "sample", "sample"])
    if kind == "norm":
        cols = _log(rng, 1, 16384)
        return {"kind": kind, "rows": _log(rng, 1, min(100000, 16_000_000 // cols)), "cols": cols,
                "pad": rng.choice([0, 0, 1, 64]), "centered": rng.random() < 0.5}
    if kind == "table":
        dim = 2 * rng.randint(2, 64)
        return {"kind": kind, "positions": _log(rng, 1, 131072), "dim": dim, "scaling": rng.choice(sorted(SCALINGS))}
    if kind == "rotate":
        head_dim = rng.choice([32, 48, 50, 64, 80, 128, 256])
        heads = rng.randint(1, 40)
        return {"kind": kind, "rows": _log(rng, 1, 8000 * 40 * 128 // (heads * head_dim)), "heads": heads,
                "head_dim": head_dim, "dim": 2 * rng.randint(1, head_dim // 2) if rng.random() < 0.5 else head_dim,
                "pad": rng.choice([0, 3, 512]), "interleaved": rng.random() < 0.5,
                "positions": _log(rng, 16, 100000)}
    if kind == "sample":
        n = _log(rng, 2, 150000)
        mixed = rng.random() < 0.3
        return {"kind": kind, "rows": _log(rng, 1, max(1, min(512, 30_000_000 // n))), "n": n,
                "pad": rng.choice([0, 0, 5]), "temperature": -1.0 if mixed else rng.choice([0.0, 0.3, 0.7, 1.0, 2.0]),
                "top_k": -1 if mixed else rng.choice([0, 0, 1, 20, 200, 5000]),
                "top_p": -1.0 if mixed else rng.choice([1.0, 1.0, 0.5, 0.9, 0.99]),
                "min_p": -1.0 if mixed else rng.choice([0.0, 0.0, 0.02, 0.1]), "masked": rng.random() < 0.3,
                "grid": rng.choice([0.0, 0.0, 0.03125, 0.25])}
    qk, v = rng.choice([(48, 64), (64, 64), (128, 128)])
    kv = rng.choice([1, 2, 3, 4, 8, 16])
    heads = kv * rng.choice([g for g in (1, 2, 3, 4, 6, 8, 16) if kv * g <= 64])
    dims = {"heads": heads, "kv_heads": kv, "qk": qk, "v": v, "page": rng.choice([16, 32, 64, 128, 256])}
    if kind == "append":
        sequences = _log(rng, 1, 64)
        run = _log(rng, 1, max(1, min(4000, 8000 * 48 * 128 // (sequences * (heads + 2 * kv) * v))))
        dim = qk if rng.random() < 0.5 else 2 * rng.randint(1, qk // 2)
        return {"kind": kind, "sequences": sequences, "run": run, "context": _log(rng, run + 1, run + 4000),
                "dim": dim, "interleaved": rng.random() < 0.5, **dims}
    sinks = rng.choice([0, 1, 4, 16, 100])
    if kind == "decode":
        rows = _log(rng, 1, 64)
        window = _log(rng, 1, max(2, min(16384, 48 * 8000 * 8 * 128 // (rows * kv * v))))
        hi = _log(rng, 2, max(3, min(32768, 48 * 16000 * 8 * 128 // (rows * kv * v))))
        return {"kind": kind, "rows": rows, "window": window, "sinks": sinks, "lo": rng.randint(1, hi), "hi": hi,
                **dims}
    runs = _log(rng, 1, 12)
    hi = _log(rng, 2, min(6000, int(math.sqrt(12 * 6000 * 8500 * 4 / (runs * heads)))))
    return {"kind": kind, "runs": runs, "lo": rng.randint(1, hi), "hi": hi,
            "prefix": rng.choice([0, rng.randint(1, 2500)]), "window": _log(rng, 16, 2048), "sinks": sinks, **dims}


# ---------------------------------------------------------------- inputs --

#: Ways to stretch a head's frequencies, (kind of the framework's table, factor, low, high, original positions, magnitude).
SCALINGS = {
    "plain": (0, 1.0, 0.0, 0.0, 0.0, 1.0),
    "linear": (1, 4.0, 0.0, 0.0, 0.0, 1.0),
    "base": (2, 8.0, 0.0, 0.0, 0.0, 1.0),
    "parts": (3, 16.0, 1.0, 32.0, 4096.0, 0.1 * math.log(16.0) + 1.0),
    "bands": (4, 8.0, 1.0, 4.0, 8192.0, 1.0),
}
THETA = 10000.0
EPS = 1e-5


def _spread(count: int, lo: int, hi: int) -> list[int]:
    """`count` lengths in [lo, hi], the same for every seed (work() counts
    them); both ends are among them where there is room."""
    rng = random.Random(1009 * count + 31 * lo + hi)
    got = [rng.randint(lo, hi) for _ in range(count)]
    got[0] = hi
    if count > 1:
        got[-1] = lo
    return got


def _runs(case) -> tuple[list[int], list[int]]:
    """The prompts' lengths, and the positions before each (every other one
    follows a prefix)."""
    lengths = _spread(case["runs"], case["lo"], case["hi"])
    return lengths, [case["prefix"] if i % 2 == 0 else 0 for i in range(case["runs"])]


def _generator(seed: int) -> torch.Generator:
    return torch.Generator(device="cuda").manual_seed(seed * 1000003 + 31)


def _ints(lst) -> torch.Tensor:
    return torch.tensor(lst, dtype=torch.int32, device="cuda")


def _randn(g, *shape) -> torch.Tensor:
    return torch.randn(*shape, generator=g, device="cuda")


def _codes(g, *shape) -> torch.Tensor:
    """int8 codes of normal values, most of them under half the range, as QuantizeInt8 leaves them."""
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float16).mul_(42).clamp_(-127, 127).to(torch.int8)


def _cache(case, g, lengths: list[int], filled: bool) -> dict:
    """A cache of one layer whose sequence i holds pages for lengths[i] positions, scattered over the pool."""
    kv, page, qk, v = case["kv_heads"], case["page"], case["qk"], case["v"]
    need = [-(-n // page) for n in lengths]
    pages, width = sum(need) + 3, max(need) + 2
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    tables = torch.full((len(need), width), -1, dtype=torch.int32, device="cuda")
    at = 0
    for i, n in enumerate(need):
        tables[i, :n] = order[at:at + n]
        at += n
    refs = torch.zeros(pages, dtype=torch.int32, device="cuda")
    refs[tables[tables >= 0].long()] = 1
    make = _codes if filled else lambda g, *shape: torch.zeros(shape, dtype=torch.int8, device="cuda")
    return {"pages": pages, "width": width, "tables": tables, "lengths": _ints(lengths), "refs": refs,
            "keys": make(g, 1, pages, kv, page, qk), "values": make(g, 1, pages, kv, page // 16, v, 16),
            "key_scales": torch.rand(1, pages, kv, page, generator=g, device="cuda") * 0.03 + 0.015,
            "value_scales": torch.rand(1, pages, kv, page, generator=g, device="cuda") * 0.02 + 0.01}


def _prepare_norm(case, seed) -> dict:
    g = _generator(seed)
    rows, cols, wide = case["rows"], case["cols"], case["cols"] + case["pad"]
    gain = _randn(g, cols) * 0.1
    # a residual stream: rows of different size, a few large columns
    x = _randn(g, rows, wide) * torch.exp(_randn(g, rows, 1)) * torch.exp(0.5 * _randn(g, 1, wide))
    return {"x": x, "delta": _randn(g, rows, wide) * 0.3, "gain": gain if case["centered"] else gain + 1,
            "sum": torch.empty(rows, wide, device="cuda"),
            "codes": torch.empty(rows, cols, dtype=torch.int8, device="cuda"),
            "scales": torch.empty(rows, device="cuda"), "values": torch.empty(rows, cols, device="cuda")}


def _frequencies(dim: int, scaling: str) -> torch.Tensor:
    kind, factor, low, high, original, _ = SCALINGS[scaling]
    i = torch.arange(dim // 2, dtype=torch.float64, device="cuda")
    theta = THETA * factor ** (dim / (dim - 2)) if kind == 2 else THETA
    f = theta ** (-2 * i / dim)
    if kind == 1:
        return f / factor
    if kind == 3:
        first, last = (dim * math.log(original / (2 * math.pi * turns)) / (2 * math.log(THETA)) for turns in (high, low))
        first, last = max(math.floor(first), 0), min(math.ceil(last), dim - 1)
        ramp = torch.clamp((i - first) / (last - first if last != first else 0.001), 0, 1)
        return f / factor * ramp + f * (1 - ramp)
    if kind == 4:
        part = torch.clamp((original * f / (2 * math.pi) - low) / (high - low), 0, 1)
        return f / factor * (1 - part) + f * part
    return f


def _table(positions: int, dim: int, scaling: str) -> dict:
    angles = torch.arange(positions, dtype=torch.float64, device="cuda")[:, None] * _frequencies(dim, scaling)
    magnitude = SCALINGS[scaling][5]
    return {"cos": (torch.cos(angles) * magnitude).float(), "sin": (torch.sin(angles) * magnitude).float()}


def _prepare_table(case, seed) -> dict:
    # (what a seed changes: where the table starts, as one that grows with its contexts)
    n, half = case["positions"], case["dim"] // 2
    return {"first": seed % 50021, "cos": torch.empty(n, half, device="cuda"), "sin": torch.empty(n, half, device="cuda")}


def _prepare_rotate(case, seed) -> dict:
    g = _generator(seed)
    rows, width = case["rows"], case["heads"] * case["head_dim"]
    return {"x": _randn(g, rows, width + case["pad"]), "y": torch.empty(rows, width, device="cuda"),
            "row_pos": torch.randint(0, case["positions"], (rows,), generator=g, device="cuda", dtype=torch.int32),
            **_table(case["positions"], case["dim"], "plain")}


def _prepare_append(case, seed) -> dict:
    g = _generator(seed)
    n, run, heads, kv, qk, v = (case[x] for x in ("sequences", "run", "heads", "kv_heads", "qk", "v"))
    ends = [run + (case["context"] - run) * (i + 1) // n for i in range(n)]  # the run's last position, different offsets
    s = _cache(case, g, ends, False)
    rows = n * run
    s["rows"] = rows
    s["projected"] = _randn(g, rows, heads * qk + kv * (qk + v)) * 3
    s["row_seq"] = torch.arange(n, device="cuda", dtype=torch.int32).repeat_interleave(run)
    s["row_pos"] = (_ints(ends)[:, None] - run + torch.arange(run, device="cuda", dtype=torch.int32)).reshape(-1).contiguous()
    s |= _table(max(ends), case["dim"], "plain")
    s["codes"] = torch.empty(rows, heads, qk, dtype=torch.int8, device="cuda")
    s["scales"] = torch.empty(rows, heads, device="cuda")
    s["q"] = torch.empty(rows, heads, qk, device="cuda")
    s["k"], s["vs"] = torch.empty(rows, kv, qk, device="cuda"), torch.empty(rows, kv, v, device="cuda")
    return s


def _queries(g, rows: int, heads: int, qk: int):
    return _codes(g, rows, heads, qk), torch.rand(rows, heads, generator=g, device="cuda") * 0.04 + 0.02


def _prepare_decode(case, seed) -> dict:
    g = _generator(seed)
    rows = case["rows"]
    s = _cache(case, g, _spread(rows, case["lo"], case["hi"]), True)
    s["q"], s["q_scales"] = _queries(g, rows, case["heads"], case["qk"])
    s["row_seq"] = torch.randperm(rows, generator=g, device="cuda").to(torch.int32)
    length = s["lengths"][s["row_seq"].long()]
    s["row_first"] = torch.clamp(length - case["window"], min=0)
    s["row_count"] = length - s["row_first"]
    s["rows"], s["max_count"] = rows, min(case["window"], case["hi"])
    s["out"] = torch.empty(rows, case["heads"], case["v"], device="cuda")
    return s


def _prepare_prompt(case, seed) -> dict:
    g = _generator(seed)
    lengths, before = _runs(case)
    s = _cache(case, g, [a + b for a, b in zip(lengths, before)], True)
    s["rows"] = sum(lengths)
    s["q"], s["q_scales"] = _queries(g, s["rows"], case["heads"], case["qk"])
    s["run_rows"] = _ints([sum(lengths[:i]) for i in range(len(lengths) + 1)])
    s["run_seq"], s["run_pos"] = _ints(list(range(len(lengths)))), _ints(before)
    s["max_run"], s["max_count"] = max(lengths), max(a + b for a, b in zip(lengths, before))
    s["out"] = torch.empty(s["rows"], case["heads"], case["v"], device="cuda")
    return s


def _choose(g, rows: int, given, choices, dtype) -> torch.Tensor:
    """The case's setting for every row, or (where it is -1) one of the choices for each."""
    if given >= 0:
        return torch.full((rows,), given, dtype=dtype, device="cuda")
    at = torch.randint(0, len(choices), (rows,), generator=g, device="cuda")
    return torch.tensor(choices, dtype=dtype, device="cuda")[at]


def _prepare_sample(case, seed) -> dict:
    g = _generator(seed)
    rows, n = case["rows"], case["n"]
    x = _randn(g, rows, n + case["pad"]) * 2.5
    # some ids stand out, as they do where a model is sure
    x += torch.exp(1.5 * _randn(g, rows, n + case["pad"])).clamp_(max=12) * 0.8
    if case["grid"]:
        x = torch.round(x / case["grid"]) * case["grid"]
    s = {"x": x.contiguous(), "temperature": _choose(g, rows, case["temperature"], [0.0, 0.6, 0.8, 1.0, 1.3], torch.float32),
         "top_k": _choose(g, rows, case["top_k"], [0, 0, 1, 40, 1000], torch.int32),
         "top_p": _choose(g, rows, case["top_p"], [1.0, 0.9, 0.95, 0.999], torch.float32),
         "min_p": _choose(g, rows, case["min_p"], [0.0, 0.0, 0.01, 0.1], torch.float32),
         "random": torch.rand(rows, generator=g, device="cuda"), "words": (n + 31) // 32,
         "ids": torch.empty(rows, dtype=torch.int32, device="cuda"), "logprobs": torch.empty(rows, device="cuda")}
    if case["masked"]:
        # half of the rows take any id, the others every second one at random, the last none
        mask = torch.randint(-2 ** 31, 2 ** 31, (rows, s["words"]), generator=g, device="cuda", dtype=torch.int64)
        mask[::2] = -1
        if rows > 1:
            mask[-1] = 0
        s["mask"] = mask.to(torch.int32)
    return s


def prepare(case: dict, seed: int) -> dict:
    s = {"norm": _prepare_norm, "table": _prepare_table, "rotate": _prepare_rotate, "append": _prepare_append,
         "decode": _prepare_decode, "prompt": _prepare_prompt, "sample": _prepare_sample}[case["kind"]](case, seed)
    s["case"] = case
    return s


# ----------------------------------------------------------- plain forms --

def _quantize(x: torch.Tensor):
    """QuantizeInt8 over the last axis (absmax / 127, half to even): codes and scales."""
    peak = x.abs().amax(-1, keepdim=True)
    # (a division by a tensor: by a number, torch multiplies with its reciprocal)
    scale = torch.where(peak > 0, peak / torch.full_like(peak, 127.0), torch.ones_like(peak))
    return torch.clamp(torch.round(x * (1.0 / scale)), -128, 127), scale


def _norm_plain(s) -> dict:
    c = s["case"]
    total = s["x"][:, :c["cols"]] + s["delta"][:, :c["cols"]]
    r = (1.0 / torch.sqrt(total.double().square().mean(-1, keepdim=True) + EPS)).float()
    codes, scale = _quantize(total * r * (s["gain"] + 1.0 if c["centered"] else s["gain"]))
    return {"sum": total, "scales": scale.squeeze(-1), "values": codes * scale}


def _table_plain(s) -> dict:
    c = s["case"]
    angles = torch.arange(s["first"], s["first"] + c["positions"], dtype=torch.float64, device="cuda")[:, None]
    angles = angles * _frequencies(c["dim"], c["scaling"])
    magnitude = SCALINGS[c["scaling"]][5]
    return {"cos": (torch.cos(angles) * magnitude).float(), "sin": (torch.sin(angles) * magnitude).float()}


def _rotated(x, cos, sin, dim: int, interleaved: bool):
    """x [rows][heads][head_dim], its first `dim` dimensions rotated by the rows' cos and sin [rows][dim/2]."""
    c, s, half = cos[:, None], sin[:, None], dim // 2
    a, b = (x[..., 0:dim:2], x[..., 1:dim:2]) if interleaved else (x[..., :half], x[..., half:dim])
    y, z = a * c - b * s, b * c + a * s
    turned = torch.stack((y, z), -1).flatten(-2) if interleaved else torch.cat((y, z), -1)
    return torch.cat((turned, x[..., dim:]), -1)


def _rotate_plain(s) -> torch.Tensor:
    c, at = s["case"], s["row_pos"].long()
    x = s["x"][:, :c["heads"] * c["head_dim"]].reshape(c["rows"], c["heads"], c["head_dim"])
    return _rotated(x, s["cos"][at], s["sin"][at], c["dim"], c["interleaved"]).reshape(c["rows"], -1)


def _append_plain(s) -> dict:
    c = s["case"]
    page, heads, kv, qk, v, rows = c["page"], c["heads"], c["kv_heads"], c["qk"], c["v"], s["rows"]
    pos, at = s["row_pos"].long(), s["row_pos"].long() % page
    x = s["projected"][:, :(heads + kv) * qk].reshape(rows, heads + kv, qk)
    x = _rotated(x, s["cos"][pos], s["sin"][pos], c["dim"], c["interleaved"])
    codes, scales = _quantize(x)
    value_codes, value_scales = _quantize(s["projected"][:, (heads + kv) * qk:].reshape(rows, kv, v))
    p = s["tables"][s["row_seq"].long(), pos // page].long()
    s["keys"][0][p, :, at] = codes[:, heads:].to(torch.int8)
    s["key_scales"][0][p, :, at] = scales[:, heads:, 0]
    s["values"][0][p, :, at // 16, :, at % 16] = value_codes.to(torch.int8)
    s["value_scales"][0][p, :, at] = value_scales.squeeze(-1)
    return {"q": (codes * scales)[:, :heads],
            "k": s["keys"][0][p, :, at].float() * s["key_scales"][0][p, :, at][..., None],
            "v": s["values"][0][p, :, at // 16, :, at % 16].float() * s["value_scales"][0][p, :, at][..., None]}


def _softmax_values(z, live, v, vs):
    """Weights of the scores z over the live positions, and the values' weighted mean (0 where nothing is live)."""
    z = torch.where(live, z, torch.full_like(z, -math.inf))
    peak = z.amax(-1, keepdim=True)
    e = torch.exp(z - torch.where(torch.isfinite(peak), peak, torch.zeros_like(peak)))
    total = e.sum(-1, keepdim=True)
    out = torch.matmul(e * vs, v)
    return torch.where(total > 0, out / total, torch.zeros_like(out))


def _cached(s, seq, pos):
    """Keys [n][kv][positions][qk], values [n][kv][positions][v] and their scales at pos [n][positions], fp32."""
    page = s["case"]["page"]
    p, at = s["tables"][seq[:, None], pos // page].clamp(min=0).long(), pos % page
    k, v = s["keys"][0][p, :, at].transpose(1, 2).float(), s["values"][0][p, :, at // 16, :, at % 16].transpose(1, 2).float()
    return k, s["key_scales"][0][p, :, at].transpose(1, 2), v, s["value_scales"][0][p, :, at].transpose(1, 2)


def _decode_plain(s) -> torch.Tensor:
    c = s["case"]
    kv, group, rows, sinks = c["kv_heads"], c["heads"] // c["kv_heads"], s["rows"], c["sinks"]
    step = torch.arange(sinks + s["max_count"], device="cuda")[None, :]
    first, count = s["row_first"].long()[:, None], s["row_count"].long()[:, None]
    # the sinks' places, then the window's
    live = torch.where(step < sinks, step < first, step - sinks < count)
    pos = torch.where(live, torch.where(step < sinks, step, first + step - sinks), torch.zeros_like(step))
    k, ks, v, vs = _cached(s, s["row_seq"].long(), pos)
    q = s["q"].float().view(rows, kv, group, c["qk"])
    z = torch.matmul(q, k.transpose(-1, -2)) * ks[:, :, None] * (s["q_scales"] / math.sqrt(c["qk"])).view(
        rows, kv, group, 1)
    return _softmax_values(z, live[:, None, None, :], v, vs[:, :, None]).reshape(rows, c["heads"], c["v"])


def _prompt_plain(s) -> torch.Tensor:
    """The packed runs laid out as [runs][longest run], and their rows picked out again."""
    c = s["case"]
    kv, group, runs, longest = c["kv_heads"], c["heads"] // c["kv_heads"], c["runs"], s["max_run"]
    pos = torch.arange(s["max_count"], device="cuda")[None, :]
    k, ks, v, vs = _cached(s, s["run_seq"].long(), pos.expand(runs, -1))
    step = torch.arange(longest, device="cuda")
    starts = s["run_rows"][:-1].long()
    at = torch.clamp(starts[:, None] + step, max=s["rows"] - 1)
    q = s["q"][at].float().view(runs, longest, kv, group, c["qk"]).permute(0, 2, 3, 1, 4)
    qs = (s["q_scales"][at] / math.sqrt(c["qk"])).view(runs, longest, kv, group).permute(0, 2, 3, 1)
    z = torch.matmul(q, k[:, :, None].transpose(-1, -2)) * ks[:, :, None, None] * qs[..., None]
    here = (s["run_pos"][:, None] + step)[:, :, None]  # the rows' positions
    live = (pos[:, None] <= here) & ((pos[:, None] > here - c["window"]) | (pos[:, None] < c["sinks"]))
    o = _softmax_values(z, live[:, None, None], v[:, :, None], vs[:, :, None, None])
    lengths = (s["run_rows"][1:] - s["run_rows"][:-1]).long()
    run = torch.repeat_interleave(torch.arange(runs, device="cuda"), lengths, output_size=s["rows"])
    row = torch.arange(s["rows"], device="cuda") - starts[run]
    return o[run, :, :, row].reshape(s["rows"], c["heads"], c["v"])


def _allowed(s) -> torch.Tensor:
    """The rows' logits, -inf at the ids that the mask leaves out."""
    n = s["case"]["n"]
    x = s["x"][:, :n]
    if "mask" not in s:
        return x
    ids = torch.arange(n, device="cuda")
    return torch.where((s["mask"][:, ids // 32] >> (ids % 32)) & 1 != 0, x, torch.full_like(x, -math.inf))


def _sample_plain(s) -> dict:
    x = _allowed(s)
    v, order = torch.sort(x, dim=-1, descending=True, stable=True)  # ties to the lower id
    greedy = ~(s["temperature"] > 0)[:, None]
    t = torch.where(greedy, torch.ones_like(s["temperature"][:, None]), s["temperature"][:, None]).double()
    some = v[:, :1] > -math.inf
    peak = torch.where(some, v[:, :1], torch.zeros_like(v[:, :1])).double()
    w = torch.round(torch.exp((v.double() - peak) / t) / UNIT).to(torch.int64)
    rank = torch.arange(v.shape[1], device="cuda")[None, :]
    k = torch.where(greedy, torch.ones_like(s["top_k"][:, None]), s["top_k"][:, None])
    w = torch.where((k <= 0) | (rank < k), w, torch.zeros_like(w))
    p = s["top_p"][:, None].double()
    before = torch.cumsum(w, -1) - w
    keep = (rank == 0) | ~(p < 1) | (before.double() < p * w.sum(-1, keepdim=True).double())
    keep = keep & (w.double() >= s["min_p"][:, None].double() / UNIT)
    w = torch.where(keep, w, torch.zeros_like(w))
    upto = torch.cumsum(torch.zeros_like(w).scatter_(1, order, w), -1)
    total = upto[:, -1:]
    at = torch.minimum(torch.floor(s["random"][:, None].double() * total.double()).to(torch.int64), total - 1)
    ids = (upto <= at).sum(-1, keepdim=True)
    ids = torch.where(some, ids, torch.zeros_like(ids))
    logprobs = (x.gather(1, ids).double() - peak) / t - torch.log(total.double() * UNIT)
    return {"ids": torch.where(some, ids, torch.full_like(ids, -1)).squeeze(-1).to(torch.int32),
            "logprobs": torch.where(some, logprobs, torch.full_like(logprobs, -math.inf)).squeeze(-1).float()}


# --------------------------------------------------- the framework's calls --

def _handle(s):
    """The program's handles, workspace and addresses, made once."""
    if "at" not in s:
        from needle_cs_amd.paged import PagedCache
        from needle_cs_amd.rotary import Rotary
        from needle_cs_amd.sampling import Sampling, sample_workspace
        c, kind = s["case"], s["case"]["kind"]
        at = {n: t.data_ptr() for n, t in s.items() if isinstance(t, torch.Tensor)}
        size = 0
        if kind in ("append", "decode", "prompt"):
            names = ("keys", "key_scales", "values", "value_scales", "tables", "lengths", "refs")
            s["cache"] = h = PagedCache(1, s["pages"], c["page"], c["kv_heads"], c["qk"], c["v"], s["tables"].shape[0],
                                        s["width"], buffers={n: at[n] for n in names})
            if kind == "decode":
                size = h.decode_sinks_workspace(s["rows"], c["heads"], c["sinks"], s["max_count"])
            elif kind == "prompt":
                size = h.prompt_sinks_workspace(s["rows"], c["heads"], c["runs"], c["sinks"], s["max_count"])
        if kind in ("rotate", "append"):
            s["rotary"] = Rotary(at["cos"], at["sin"], s["cos"].shape[0], c["dim"], c["interleaved"])
        if kind == "table":
            way, factor, low, high, original, magnitude = SCALINGS[c["scaling"]]
            s["scaling"] = dict(theta=THETA, kind=way, factor=factor, low=low, high=high, original=original,
                                magnitude=magnitude)
        if kind == "sample":
            s["sampling"] = Sampling(at["random"], at["temperature"], at["top_k"], at["top_p"], at["min_p"])
            size = sample_workspace(c["rows"], c["n"])
        s["size"], s["workspace"] = size, torch.empty(max(size, 16), dtype=torch.uint8, device="cuda")
        s["ws"] = s["workspace"].data_ptr()
        s["at"] = at
    return s["at"]


def _own(s):
    import needle_cs_amd as N
    at, c, kind = _handle(s), s["case"], s["case"]["kind"]
    if kind == "norm":
        from needle_cs_amd.rows import add_rms_quantize, dequantize_rows
        wide = c["cols"] + c["pad"]
        add_rms_quantize(at["x"], wide, at["delta"], wide, at["gain"], c["centered"], EPS, c["rows"], c["cols"],
                         at["sum"], wide, at["codes"], at["scales"])
        dequantize_rows(at["codes"], at["scales"], c["rows"], c["cols"], at["values"], c["cols"])
        return {"sum": s["sum"][:, :c["cols"]], "scales": s["scales"], "values": s["values"]}
    if kind == "table":
        from needle_cs_amd.rotary import rotary_table
        rotary_table(at["cos"], at["sin"], s["first"], c["positions"], c["dim"], **s["scaling"])
        return {"cos": s["cos"], "sin": s["sin"]}
    if kind == "rotate":
        width = c["heads"] * c["head_dim"]
        s["rotary"].rotate(at["x"], width + c["pad"], c["heads"], c["head_dim"], at["row_pos"], c["rows"], at["y"], width)
        return s["y"]
    if kind == "append":
        heads, kv, qk, v = c["heads"], c["kv_heads"], c["qk"], c["v"]
        ld, x = s["projected"].shape[1], at["projected"]
        s["cache"].rotary_append(0, s["rotary"], x, ld, heads, x + 4 * heads * qk, ld, x + 4 * (heads + kv) * qk, ld,
                                 at["row_seq"], at["row_pos"], s["rows"], at["codes"], at["scales"])
        from needle_cs_amd.rows import dequantize_rows
        dequantize_rows(at["codes"], at["scales"], s["rows"] * heads, qk, at["q"], qk)
        s["cache"].read(0, at["row_seq"], at["row_pos"], s["rows"], at["k"], kv * qk, at["vs"], kv * v)
        return {"q": s["q"], "k": s["k"], "v": s["vs"]}
    if kind == "decode":
        s["cache"].decode_sinks(0, at["q"], at["q_scales"], s["rows"], c["heads"], at["row_seq"], at["row_first"],
                                at["row_count"], c["sinks"], s["max_count"], s["ws"], s["size"], at["out"])
        return s["out"]
    if kind == "prompt":
        s["cache"].prompt_sinks(0, at["q"], at["q_scales"], s["rows"], c["heads"], c["runs"], at["run_rows"],
                                at["run_seq"], at["run_pos"], c["window"], c["sinks"], s["max_count"], s["ws"],
                                s["size"], at["out"])
        return s["out"]
    from needle_cs_amd.sampling import sample
    sample(at["x"], c["n"] + c["pad"], c["n"], c["rows"], s["sampling"], at.get("mask"), s["words"], s["words"],
           s["ws"], s["size"], at["ids"], at["logprobs"])
    return {"ids": s["ids"], "logprobs": s["logprobs"]}


def run(state: dict):
    if own:
        return _own(state)
    return {"norm": _norm_plain, "table": _table_plain, "rotate": _rotate_plain, "append": _append_plain,
            "decode": _decode_plain, "prompt": _prompt_plain, "sample": _sample_plain}[state["case"]["kind"]](state)


# ------------------------------------------------------------------ work --

def work(case: dict) -> dict:
    kind = case["kind"]
    if kind == "norm":
        n = case["rows"] * case["cols"]
        return {"bytes": n * (4 + 4 + 4 + 1 + 4) + 4 * case["rows"] + 4 * case["cols"], "flops": 9 * n}
    if kind == "table":
        n = case["positions"] * case["dim"] // 2
        return {"bytes": 8 * n, "flops": 10 * n}
    if kind == "rotate":
        n = case["rows"] * case["heads"] * case["head_dim"]
        table = 4 * min(case["rows"], case["positions"]) * case["dim"]
        return {"bytes": 8 * n + table + 4 * case["rows"], "flops": 3 * case["rows"] * case["heads"] * case["dim"]}
    if kind == "sample":
        return {"bytes": case["rows"] * (4 * case["n"] + (case["n"] // 8 if case["masked"] else 0) + 28),
                "flops": 4 * case["rows"] * case["n"]}
    heads, kv, qk, v = case["heads"], case["kv_heads"], case["qk"], case["v"]
    cell = kv * (qk + v + 8)  # one position of one layer
    if kind == "append":
        rows, width = case["sequences"] * case["run"], heads * qk + kv * (qk + v)
        return {"bytes": rows * (4 * width + cell + heads * (qk + 4) + 4 * width + 4 * case["dim"] + 8),
                "flops": 8 * rows * width}
    if kind == "decode":
        attended = [min(n, case["window"] + case["sinks"]) for n in _spread(case["rows"], case["lo"], case["hi"])]
        return {"bytes": sum(attended) * cell + case["rows"] * (heads * (qk + 4 + 4 * v) + 12),
                "flops": 2 * (qk + v) * heads * sum(attended)}
    attended, held, rows, reach = 0, 0, 0, case["window"] + case["sinks"]
    for n, b in zip(*_runs(case)):
        attended += sum(min(b + i + 1, reach) for i in range(n))
        held += min(n + b, n + reach - 1)
        rows += n
    return {"bytes": held * cell + rows * heads * (qk + 4 + 4 * v), "flops": 2 * (qk + v) * heads * attended}


# ----------------------------------------------------------------- exact --

def _exact_norm(case, s) -> dict:
    cols = case["cols"]
    total = s["x"][:, :cols].double() + s["delta"][:, :cols].double()
    gain = s["gain"].double() + (1.0 if case["centered"] else 0.0)
    y = total * torch.rsqrt((total * total).sum(1, keepdim=True) / cols + EPS) * gain
    peak = torch.maximum(y.max(1).values, -y.min(1).values)
    # (a code has no other value than the one that its roundings give)
    return {"sum": total, "scales": torch.where(peak == 0, 1.0, peak / 127), "values": None}


def _exact_table(case, s) -> dict:
    import numpy as np
    way, factor, low, high, original, magnitude = SCALINGS[case["scaling"]]
    dim, tau = case["dim"], 2 * math.pi
    found = []
    for i in range(dim // 2):
        f = math.exp(-math.log(THETA) * 2 * i / dim)
        turns = original * f / tau  # over the original positions
        if way == 1:
            f /= factor
        elif way == 2:
            f = math.exp(-(math.log(THETA) + math.log(factor) * dim / (dim - 2)) * 2 * i / dim)
        elif way == 3:
            place = lambda t: dim * math.log(original / (t * tau)) / math.log(THETA) / 2  # noqa: E731
            a, b = max(math.floor(place(high)), 0), min(math.ceil(place(low)), dim - 1)
            part = min(max((i - a) / ((b - a) or 0.001), 0.0), 1.0)
            f = part * f / factor + (1 - part) * f
        elif way == 4:
            part = min(max((turns - low) / (high - low), 0.0), 1.0)
            f = part * f + (1 - part) * f / factor
        found.append(f)
    angles = np.outer(np.arange(s["first"], s["first"] + case["positions"], dtype=np.float64), np.array(found))
    return {"cos": torch.from_numpy(np.cos(angles) * magnitude), "sin": torch.from_numpy(np.sin(angles) * magnitude)}


def _exact_rotate(case, s) -> torch.Tensor:
    rows, head_dim, dim = case["rows"], case["head_dim"], case["dim"]
    y = s["x"][:, :case["heads"] * head_dim].double().clone().view(rows, case["heads"], head_dim)
    c, sn = s["cos"].double()[s["row_pos"].long()], s["sin"].double()[s["row_pos"].long()]
    turn = torch.complex(c, sn)[:, None]
    i = torch.arange(dim // 2, device="cuda")
    a, b = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + dim // 2)
    z = torch.complex(y[:, :, a], y[:, :, b]) * turn
    y[:, :, a], y[:, :, b] = z.real, z.imag
    return y.view(rows, -1)


def _exact_rows(case, s, seq: int, q, qs, first, last):
    """Attention in 64 bits of the rows q [n][heads][qk] over positions first[i]..last[i] of a sequence, and the sinks before."""
    kv, group = case["kv_heads"], case["heads"] // case["kv_heads"]
    pages = s["tables"][seq]
    pages = pages[pages >= 0].long()
    pos = torch.arange(pages.numel() * case["page"], device="cuda")
    out = torch.empty(q.shape[0], case["heads"], case["v"], dtype=torch.float64, device="cuda")
    dead = ((pos[None, :] < first[:, None]) & (pos[None, :] >= case["sinks"])) | (pos[None, :] > last[:, None])
    for h in range(case["heads"]):
        j = h // group
        k = s["keys"][0, pages, j].reshape(-1, case["qk"]).double() * s["key_scales"][0, pages, j].reshape(-1, 1).double()
        v = s["values"][0, pages, j].transpose(-1, -2).reshape(-1, case["v"]).double()
        v = v * s["value_scales"][0, pages, j].reshape(-1, 1).double()
        z = (q[:, h].double() * qs[:, h, None].double()) @ k.t() / math.sqrt(case["qk"])
        out[:, h] = torch.softmax(z.masked_fill_(dead, -math.inf), dim=-1) @ v
    return out


def _exact_sample(case, s) -> dict:
    x = _allowed(s).double()
    found = []
    for r in range(case["rows"]):
        v, order = torch.sort(x[r], descending=True, stable=True)
        n = int((v > -math.inf).sum())
        if n == 0:
            found.append(-math.inf)
            continue
        t, k, p, least = (float(s[name][r]) for name in ("temperature", "top_k", "top_p", "min_p"))
        if t <= 0:
            found.append(0.0)
            continue
        n = min(n, int(k)) if k > 0 else n
        e = torch.exp((v[:n] - v[0]) / t)
        mass = torch.cumsum(e, 0) / e.sum()
        kept = torch.ones_like(e, dtype=torch.bool)
        if p < 1:
            kept[1:] = mass[:-1] < p
        kept &= e >= least
        by_id = torch.zeros_like(x[r])
        by_id[order[:n][kept]] = e[kept]
        upto = torch.cumsum(by_id, 0)
        total = upto[-1]
        at = min(int(torch.searchsorted(upto, float(s["random"][r]) * total, right=True)), case["n"] - 1)
        found.append(float((x[r, at] - v[0]) / t - torch.log(total)))
    return {"ids": None, "logprobs": torch.tensor(found, dtype=torch.float64)}


def exact(case: dict, seed: int):
    """Every number in 64 bits; codes and ids have no other value than the plain form's."""
    s, kind = prepare(case, seed), case["kind"]
    if kind in ("norm", "table", "rotate", "sample"):
        return {"norm": _exact_norm, "table": _exact_table, "rotate": _exact_rotate, "sample": _exact_sample}[kind](case, s)
    if kind == "append":
        return None
    if kind == "decode":
        parts = [_exact_rows(case, s, int(s["row_seq"][r]), s["q"][r:r + 1], s["q_scales"][r:r + 1],
                             s["row_first"][r:r + 1], s["row_first"][r:r + 1] + s["row_count"][r:r + 1] - 1)
                 for r in range(s["rows"])]
        return torch.cat(parts)
    parts, at = [], 0
    for i, (n, before) in enumerate(zip(*_runs(case))):
        for b in range(0, n, 4096):
            m = min(4096, n - b)
            last = torch.arange(before + b, before + b + m, device="cuda")
            first = torch.clamp(last - case["window"] + 1, min=0)
            parts.append(_exact_rows(case, s, i, s["q"][at + b:at + b + m], s["q_scales"][at + b:at + b + m], first,
                                     last))
        at += n
    return torch.cat(parts)
