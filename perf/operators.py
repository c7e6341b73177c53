"""The paged int8 cache's operators as a program of its users calls them, for timing and comparing.

A paged cache keeps every sequence's keys and values in pages of `page`
positions that a table names, for all layers:

    keys    int8 [layers][pages][kv_heads][page][qk]        key_scales   fp32 [layers][pages][kv_heads][page]
    values  int8 [layers][pages][kv_heads][page/16][v][16]  value_scales fp32 [layers][pages][kv_heads][page]
    tables  int32 [sequences][width] (-1 past a sequence's pages), lengths int32 [sequences],
    refs    int32 [pages], the number of sequences that hold a page (0: free)

kind "append"   rows of fp32 keys and values, columns of a wider matrix (a
                fused Q/K/V projection's output), QuantizeInt8 per head into
                their sequences' pages; `run` rows of each sequence
kind "decode"   attention of one new token of each of `rows` sequences
kind "prompt"   causal attention of packed prompts of different lengths, with
                positions already in the cache before some of them
kind "branch"   a beam step: every beam becomes a copy of its parent (shared
                pages) and grows by one position (a page that others hold is
                copied before it is written, new pages are taken)
kind "compact"  sequences leave, and the pages that remain move to the front
                of the pool

`own` False computes them in elementary torch operations, True through
needle_cs_amd.paged.
"""
from __future__ import annotations

import math
import random

import torch

own = False


def listed() -> list[dict]:
    return [
        # one decode step's new keys and values of 16 sequences, Needle 3's heads: launch latency
        {"name": "append_step", "kind": "append", "sequences": 16, "run": 1, "heads": 12, "kv_heads": 2, "qk": 48,
         "v": 64, "page": 16, "context": 1000, "layers": 2},
        # a batch of prompts entering the cache, wide grouped heads, ends inside pages
        {"name": "append_prompt", "kind": "append", "sequences": 5, "run": 1637, "heads": 32, "kv_heads": 8,
         "qk": 128, "v": 128, "page": 64, "context": 2048, "layers": 1},
        # a beam-3 step of a short context, Needle 3's heads: the smallest attention a server issues
        {"name": "decode_beam3", "kind": "decode", "rows": 3, "heads": 12, "kv_heads": 2, "qk": 48, "v": 64,
         "page": 16, "lo": 128, "hi": 192},
        # 16 independent sequences of 32 to 2048 positions, one kv head per query head
        {"name": "decode_ragged16", "kind": "decode", "rows": 16, "heads": 16, "kv_heads": 16, "qk": 64, "v": 64,
         "page": 64, "lo": 32, "hi": 2048},
        # long contexts, grouped heads: the cache's bytes bound it
        {"name": "decode_long", "kind": "decode", "rows": 32, "heads": 32, "kv_heads": 8, "qk": 128, "v": 128,
         "page": 64, "lo": 4097, "hi": 32768},
        # one request's prompt in a window of 1024, Needle 3's heads
        {"name": "prompt_short", "kind": "prompt", "runs": 1, "lo": 61, "hi": 61, "prefix": 0, "heads": 12,
         "kv_heads": 2, "qk": 48, "v": 64, "page": 16, "window": 1024},
        # a server's packed prompts of 1 to 700 tokens, some after a shared prefix
        {"name": "prompt_packed", "kind": "prompt", "runs": 16, "lo": 1, "hi": 700, "prefix": 333, "heads": 16,
         "kv_heads": 16, "qk": 64, "v": 64, "page": 32, "window": 0},
        # one long prompt, wide grouped heads: the products bound it
        {"name": "prompt_long", "kind": "prompt", "runs": 1, "lo": 8192, "hi": 8192, "prefix": 0, "heads": 32,
         "kv_heads": 8, "qk": 128, "v": 128, "page": 64, "window": 0},
        # a beam-3 step of one request over Needle 3's 20 layers
        {"name": "branch_beam3", "kind": "branch", "requests": 1, "beams": 3, "lo": 187, "hi": 187, "layers": 20,
         "kv_heads": 2, "qk": 48, "v": 64, "page": 16},
        # beam-4 steps of 32 requests over the 12-layer decoder's cache
        {"name": "branch_many", "kind": "branch", "requests": 32, "beams": 4, "lo": 65, "hi": 1500, "layers": 12,
         "kv_heads": 16, "qk": 64, "v": 64, "page": 64},
        # two of eight short sequences leave a Needle 3 cache
        {"name": "compact_few", "kind": "compact", "sequences": 8, "lo": 20, "hi": 300, "every": 4, "layers": 20,
         "kv_heads": 2, "qk": 48, "v": 64, "page": 16},
        # a third of 96 sequences leaves the 12-layer decoder's cache: a copy bounds it
        {"name": "compact_many", "kind": "compact", "sequences": 96, "lo": 100, "hi": 2000, "every": 3, "layers": 12,
         "kv_heads": 8, "qk": 64, "v": 64, "page": 64},
    ]


def _log(rng, lo: int, hi: int) -> int:
    """An integer in [lo, hi], even over its logarithm."""
    return min(max(int(round(math.exp(rng.uniform(math.log(lo), math.log(hi))))), lo), hi)


def draw(rng) -> dict:
    kind = rng.choice(["append", "append", "decode", "decode", "decode", "prompt", "prompt", "prompt", "branch",
                       "compact"])
    qk, v = rng.choice([(48, 64), (64, 64), (128, 128)])
    kv = rng.choice([1, 2, 3, 4, 8, 16])
    heads = kv * rng.choice([g for g in (1, 2, 3, 4, 6, 8, 16) if kv * g <= 64])
    page = rng.choice([16, 32, 64, 128, 256])
    dims = {"heads": heads, "kv_heads": kv, "qk": qk, "v": v, "page": page}
    if kind == "append":
        sequences = _log(rng, 1, 64)
        run = _log(rng, 1, max(1, min(4000, 8000 * 8 * 128 // (sequences * kv * v))))
        return {"kind": kind, "sequences": sequences, "run": run, "context": _log(rng, run + 1, run + 4000),
                "layers": rng.randint(1, 2), **dims}
    if kind == "decode":
        rows = _log(rng, 1, 64)
        hi = _log(rng, 2, min(32768, 32 * 20000 * 8 * 128 // (rows * kv * v)))
        return {"kind": kind, "rows": rows, "lo": rng.randint(1, hi), "hi": hi, **dims}
    if kind == "prompt":
        runs = _log(rng, 1, 24)
        hi = _log(rng, 2, min(6000, int(math.sqrt(32 * 8192 * 8192 * 128 / 4 / (runs * heads * v)))))
        return {"kind": kind, "runs": runs, "lo": rng.randint(1, hi), "hi": hi,
                "prefix": rng.choice([0, 0, rng.randint(1, 900)]), "window": rng.choice([0, 0, 0, 100, 1024]), **dims}
    dims.pop("heads")
    layers = rng.randint(1, 20)
    page_bytes = page * kv * (qk + v + 8) * layers
    if kind == "branch":
        beams = rng.randint(2, 6)
        requests = _log(rng, 1, 32)
        most = 1_500_000_000 // (page_bytes * requests * (beams + 1))
        hi = _log(rng, 2, max(3, min(2000, most * page)))
        return {"kind": kind, "requests": requests, "beams": beams, "lo": rng.randint(1, hi), "hi": hi,
                "layers": layers, **dims}
    sequences = _log(rng, 4, 128)
    hi = _log(rng, 2, max(3, min(4000, 1_500_000_000 // (page_bytes * sequences) * page)))
    return {"kind": kind, "sequences": sequences, "lo": rng.randint(1, hi), "hi": hi, "every": rng.randint(2, 5),
            "layers": layers, **dims}


# ---------------------------------------------------------------- inputs --

def _spread(case, count: int, lo: int, hi: int, salt: int = 0) -> list[int]:
    """`count` lengths in [lo, hi], the same for every seed (work() counts
    them); both ends are among them where there is room."""
    rng = random.Random(1009 * count + 31 * lo + hi + 7919 * salt)
    got = [rng.randint(lo, hi) for _ in range(count)]
    got[0] = hi
    if count > 1:
        got[-1] = lo
    return got


def _runs(case) -> tuple[list[int], list[int]]:
    """The prompts' lengths, and the positions before each (every other one
    follows a prefix)."""
    lengths = _spread(case, case["runs"], case["lo"], case["hi"])
    return lengths, [case["prefix"] if i % 2 == 0 else 0 for i in range(case["runs"])]


def _generator(seed: int) -> torch.Generator:
    return torch.Generator(device="cuda").manual_seed(seed * 1000003 + 29)


def _ints(lst) -> torch.Tensor:
    return torch.tensor(lst, dtype=torch.int32, device="cuda")


def _codes(g, *shape) -> torch.Tensor:
    """int8 codes of normal values, most of them under half the range, as QuantizeInt8 leaves them."""
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float16).mul_(42).clamp_(-127, 127).to(torch.int8)


def _pool(case, g, pages: int, layers: int) -> dict:
    kv, page, qk, v = case["kv_heads"], case["page"], case["qk"], case["v"]
    keys = torch.empty(layers, pages, kv, page, qk, dtype=torch.int8, device="cuda")
    values = torch.empty(layers, pages, kv, page // 16, v, 16, dtype=torch.int8, device="cuda")
    for layer in range(layers):
        keys[layer] = _codes(g, pages, kv, page, qk)
        values[layer] = _codes(g, pages, kv, page // 16, v, 16)
    key_scales = torch.rand(layers, pages, kv, page, generator=g, device="cuda") * 0.03 + 0.015
    value_scales = torch.rand(layers, pages, kv, page, generator=g, device="cuda") * 0.02 + 0.01
    return {"keys": keys, "values": values, "key_scales": key_scales, "value_scales": value_scales}


def _tables(g, need: list[int], pages: int, width: int) -> torch.Tensor:
    """Each sequence's pages, scattered over the pool."""
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    tables = torch.full((len(need), width), -1, dtype=torch.int32, device="cuda")
    at = 0
    for i, n in enumerate(need):
        tables[i, :n] = order[at:at + n]
        at += n
    return tables


def _cache(case, g, lengths: list[int], spare: int, layers: int) -> dict:
    """A cache whose sequence i holds pages for lengths[i] positions."""
    page = case["page"]
    need = [-(-n // page) for n in lengths]
    pages, width = sum(need) + spare, max(need) + 2
    tables = _tables(g, need, pages, width)
    refs = torch.zeros(pages, dtype=torch.int32, device="cuda")
    refs[tables[tables >= 0].long()] = 1
    return {"pages": pages, "width": width, "layers": layers, "tables": tables, "lengths": _ints(lengths),
            "refs": refs, **_pool(case, g, pages, layers)}


def _queries(g, rows: int, heads: int, qk: int):
    return _codes(g, rows, heads, qk), torch.rand(rows, heads, generator=g, device="cuda") * 0.04 + 0.02


def _prepare_append(case, seed) -> dict:
    g = _generator(seed)
    n, run, kv, qk, v = case["sequences"], case["run"], case["kv_heads"], case["qk"], case["v"]
    ends = [run + (case["context"] - run) * (i + 1) // n for i in range(n)]  # the run's last position, different offsets
    s = _cache(case, g, ends, 3, case["layers"])
    columns = case["heads"] * qk
    s["projected"] = torch.randn(n * run, columns + kv * (qk + v), generator=g, device="cuda") * 3
    s["k_column"], s["v_column"] = columns, columns + kv * qk
    s["row_seq"] = _ints([i for i in range(n) for _ in range(run)])
    s["row_pos"] = _ints([ends[i] - run + j for i in range(n) for j in range(run)])
    s["rows"], s["layer"] = n * run, case["layers"] - 1
    return s


def _prepare_decode(case, seed) -> dict:
    g = _generator(seed)
    counts = _spread(case, case["rows"], case["lo"], case["hi"])
    s = _cache(case, g, counts, 3, 1)
    s["q"], s["q_scales"] = _queries(g, case["rows"], case["heads"], case["qk"])
    s["row_seq"] = torch.randperm(case["rows"], generator=g, device="cuda").to(torch.int32)
    s["row_first"] = torch.zeros(case["rows"], dtype=torch.int32, device="cuda")
    s["row_count"] = s["lengths"][s["row_seq"].long()].contiguous()
    s["rows"], s["max_count"] = case["rows"], max(counts)
    s["out"] = torch.empty(case["rows"], case["heads"], case["v"], device="cuda")
    return s


def _prepare_prompt(case, seed) -> dict:
    g = _generator(seed)
    lengths, before = _runs(case)
    s = _cache(case, g, [a + b for a, b in zip(lengths, before)], 3, 1)
    s["rows"] = sum(lengths)
    s["q"], s["q_scales"] = _queries(g, s["rows"], case["heads"], case["qk"])
    s["run_rows"] = _ints([sum(lengths[:i]) for i in range(len(lengths) + 1)])
    s["run_seq"], s["run_pos"] = _ints(list(range(len(lengths)))), _ints(before)
    s["max_run"], s["max_count"] = max(lengths), max(a + b for a, b in zip(lengths, before))
    s["out"] = torch.empty(s["rows"], case["heads"], case["v"], device="cuda")
    return s


def _beam_pages(case) -> tuple[list[int], list[int]]:
    """Per request: the beams' length, and the full pages they share."""
    lengths = _spread(case, case["requests"], case["lo"], case["hi"])
    return lengths, [(n // case["page"]) * 3 // 4 for n in lengths]


def _parents(case) -> list[int]:
    """Every beam's parent: beams of its request, the better ones more than once."""
    rng = random.Random(case["requests"] * 100 + case["beams"])
    return [r * case["beams"] + rng.randint(0, b) for r in range(case["requests"]) for b in range(case["beams"])]


def _prepare_branch(case, seed) -> dict:
    g = _generator(seed)
    page, beams, n = case["page"], case["beams"], case["requests"] * case["beams"]
    lengths, shared = _beam_pages(case)
    need = [-(-a // page) for a in lengths]
    width = max(need) + 2
    pages = sum(c + beams * (a - c + 2) for a, c in zip(need, shared))
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    tables = torch.full((n, width), -1, dtype=torch.int32, device="cuda")
    refs = torch.zeros(pages, dtype=torch.int32, device="cuda")
    at = 0
    for r, (a, c) in enumerate(zip(need, shared)):
        tables[r * beams:(r + 1) * beams, :c] = order[at:at + c]
        refs[order[at:at + c].long()] = beams
        at += c
        for b in range(r * beams, (r + 1) * beams):
            tables[b, c:a] = order[at:at + a - c]
            refs[order[at:at + a - c].long()] = 1
            at += a - c
    every = [a for a in lengths for _ in range(beams)]
    return {"pages": pages, "width": width, "layers": case["layers"], "tables": tables, "lengths": _ints(every),
            "refs": refs, **_pool(case, g, pages, case["layers"]), "beams": _ints(list(range(n))),
            "parents": _ints(_parents(case)), "held": _ints(every), "grown": _ints([a + 1 for a in every]),
            "count": n, "status": torch.zeros(2, dtype=torch.int32, device="cuda")}


def _prepare_compact(case, seed) -> dict:
    g = _generator(seed)
    n = case["sequences"]
    s = _cache(case, g, _spread(case, n, case["lo"], case["hi"]), 0, case["layers"])
    # the bookkeeping in one buffer, and a copy to start every pass from (the pages keep what they hold:
    # a pass moves pages into freed ones and leaves the moved ones' old bytes alone)
    book = torch.cat([s["tables"].reshape(-1), s["lengths"], s["refs"]])
    s["book"], s["kept"] = book, book.clone()
    a, b = n * s["width"], n * s["width"] + n
    s["tables"], s["lengths"], s["refs"] = book[:a].view(n, s["width"]), book[a:b], book[b:]
    leave = list(range(0, n, case["every"]))
    s["leave"], s["count"] = _ints(leave), len(leave)
    s["status"] = torch.zeros(2, dtype=torch.int32, device="cuda")
    return s


def prepare(case: dict, seed: int) -> dict:
    s = {"append": _prepare_append, "decode": _prepare_decode, "prompt": _prepare_prompt, "branch": _prepare_branch,
         "compact": _prepare_compact}[case["kind"]](case, seed)
    s["case"] = case
    return s


# ----------------------------------------------------------- plain forms --

def _quantize(x: torch.Tensor):
    """QuantizeInt8 over the last axis: absmax / 127, half to even."""
    peak = x.abs().amax(-1, keepdim=True)
    # (a division by a tensor: by a number, torch multiplies with its reciprocal)
    scale = torch.where(peak > 0, peak / torch.full_like(peak, 127.0), torch.ones_like(peak))
    return torch.clamp(torch.round(x * (1.0 / scale)), -128, 127).to(torch.int8), scale.squeeze(-1)


def _append_plain(s) -> dict:
    c = s["case"]
    page, kv, rows = c["page"], c["kv_heads"], s["rows"]
    k = s["projected"][:, s["k_column"]:s["k_column"] + kv * c["qk"]].reshape(rows, kv, c["qk"])
    v = s["projected"][:, s["v_column"]:s["v_column"] + kv * c["v"]].reshape(rows, kv, c["v"])
    (qk, ks), (qv, vs) = _quantize(k), _quantize(v)
    pos, at = s["row_pos"].long(), s["row_pos"].long() % page
    p = s["tables"][s["row_seq"].long(), pos // page].long()
    layer = s["layer"]
    s["keys"][layer][p, :, at] = qk
    s["key_scales"][layer][p, :, at] = ks
    s["values"][layer][p, :, at // 16, :, at % 16] = qv
    s["value_scales"][layer][p, :, at] = vs
    return _contents(s)


def _contents(s) -> dict:
    return {n: s[n] for n in ("keys", "key_scales", "values", "value_scales")}


def _gather(c, pool, tables):
    """[n][pages of a sequence] -> keys [n][kv][T][qk], values [n][kv][T][v] and their scales [n][kv][T], fp32."""
    t = tables.clamp(min=0).long()
    n, kv, span = t.shape[0], c["kv_heads"], t.shape[1] * c["page"]
    k = pool["keys"][0][t].permute(0, 2, 1, 3, 4).reshape(n, kv, span, c["qk"]).float()
    v = pool["values"][0][t].permute(0, 2, 1, 3, 5, 4).reshape(n, kv, span, c["v"]).float()
    ks, vs = (pool[x][0][t].permute(0, 2, 1, 3).reshape(n, kv, span) for x in ("key_scales", "value_scales"))
    return k, ks, v, vs


def _softmax_values(z, live, v, vs):
    """Weights of the scores z over the live positions, and the values' weighted mean (0 where nothing is live)."""
    z = torch.where(live, z, torch.full_like(z, -math.inf))
    peak = z.amax(-1, keepdim=True)
    e = torch.exp(z - torch.where(torch.isfinite(peak), peak, torch.zeros_like(peak)))
    total = e.sum(-1, keepdim=True)
    out = torch.matmul(e * vs, v)
    return torch.where(total > 0, out / total, torch.zeros_like(out))


def _decode_plain(s) -> torch.Tensor:
    c = s["case"]
    kv, group, rows = c["kv_heads"], c["heads"] // c["kv_heads"], s["rows"]
    k, ks, v, vs = _gather(c, s, s["tables"][s["row_seq"].long(), :-(-s["max_count"] // c["page"])])
    q = s["q"].float().view(rows, kv, group, c["qk"])
    z = torch.matmul(q, k.transpose(-1, -2)) * ks[:, :, None] * (s["q_scales"] / math.sqrt(c["qk"])).view(
        rows, kv, group, 1)
    pos = torch.arange(k.shape[2], device="cuda")[None, :]
    live = (pos >= s["row_first"][:, None]) & (pos < (s["row_first"] + s["row_count"])[:, None])
    return _softmax_values(z, live[:, None, None, :], v, vs[:, :, None]).reshape(rows, c["heads"], c["v"])


def _prompt_plain(s) -> torch.Tensor:
    """The packed runs laid out as [runs][longest run], and their rows picked out again."""
    c = s["case"]
    kv, group, runs, longest = c["kv_heads"], c["heads"] // c["kv_heads"], c["runs"], s["max_run"]
    k, ks, v, vs = _gather(c, s, s["tables"][s["run_seq"].long(), :-(-s["max_count"] // c["page"])])
    step = torch.arange(longest, device="cuda")
    starts = s["run_rows"][:-1].long()
    at = torch.clamp(starts[:, None] + step, max=s["rows"] - 1)
    q = s["q"][at].float().view(runs, longest, kv, group, c["qk"]).permute(0, 2, 3, 1, 4)
    qs = (s["q_scales"][at] / math.sqrt(c["qk"])).view(runs, longest, kv, group).permute(0, 2, 3, 1)
    z = torch.matmul(q, k[:, :, None].transpose(-1, -2)) * ks[:, :, None, None] * qs[..., None]
    here = (s["run_pos"][:, None] + step)[:, :, None]  # the rows' positions
    pos = torch.arange(k.shape[2], device="cuda")[None, None, :]
    live = pos <= here
    if c["window"]:
        live = live & (pos > here - c["window"])
    o = _softmax_values(z, live[:, None, None], v[:, :, None], vs[:, :, None, None])
    lengths = (s["run_rows"][1:] - s["run_rows"][:-1]).long()
    run = torch.repeat_interleave(torch.arange(runs, device="cuda"), lengths, output_size=s["rows"])
    row = torch.arange(s["rows"], device="cuda") - starts[run]
    return o[run, :, :, row].reshape(s["rows"], c["heads"], c["v"])


def _add_refs(s, pages, live, by):
    """refs[page] += by for the live entries of `pages`."""
    s["refs"].index_add_(0, torch.where(live, pages, torch.zeros_like(pages)).reshape(-1).long(),
                         (live.to(torch.int32) * by).reshape(-1))


def _fork_plain(s, dst, src, held):
    c, steps = s["case"], torch.arange(s["width"], device="cuda")[None, :]
    old = s["tables"][dst]
    kept = steps < ((held + c["page"] - 1) // c["page"])[:, None]
    new = torch.where(kept, s["tables"][src], torch.full_like(old, -1))
    _add_refs(s, new, kept, 1)
    _add_refs(s, old, steps < ((s["lengths"][dst] + c["page"] - 1) // c["page"])[:, None], -1)
    s["tables"][dst] = new
    s["lengths"][dst] = held


def _resize_plain(s, seq, length):
    c, page = s["case"], s["case"]["page"]
    steps = torch.arange(s["width"], device="cuda")[None, :]
    old, rows = s["lengths"][seq], s["tables"][seq]
    has, want = (old + page - 1) // page, (length + page - 1) // page
    grows = (length > old) & (old % page != 0)  # into a page that it holds already
    tail = rows.gather(1, torch.clamp(has - 1, min=0)[:, None].long()).squeeze(1)
    earlier = (tail[:, None] == tail[None, :]) & grows[None, :] & torch.ones_like(
        tail[:, None] * tail[None, :], dtype=torch.bool).tril(-1)
    copies = grows & (earlier.sum(1) < s["refs"][tail.clamp(min=0).long()] - 1)
    takes = copies.to(torch.int32) + torch.clamp(want - has, min=0)
    start = torch.cumsum(takes, 0) - takes
    free = torch.argsort((s["refs"] != 0).to(torch.int8), stable=True).to(torch.int32)  # the free pages first
    s["status"][0] = torch.clamp(takes.sum() - (s["refs"] == 0).sum(), min=0)
    copy = torch.where(copies, free[start.long()], tail)  # (a tail that stays is copied onto itself)
    for name in ("keys", "key_scales", "values", "value_scales"):
        s[name][:, copy.long()] = s[name][:, tail.long()]
    fresh = (steps >= has[:, None]) & (steps < want[:, None])
    at = torch.clamp(start[:, None] + copies[:, None] + steps - has[:, None], min=0, max=free.numel() - 1)
    new = torch.where(fresh, free[at.long()], torch.where(steps < want[:, None], rows, torch.full_like(rows, -1)))
    new = torch.where(copies[:, None] & (steps == has[:, None] - 1), copy[:, None], new)
    _add_refs(s, rows, (steps >= want[:, None]) & (steps < has[:, None]), -1)
    _add_refs(s, tail, copies, -1)
    _add_refs(s, copy, copies, 1)
    _add_refs(s, new, fresh, 1)
    s["tables"][seq] = new
    s["lengths"][seq] = length.to(torch.int32)


def _branch_plain(s) -> dict:
    seq = s["beams"].long()
    _fork_plain(s, seq, s["parents"].long(), s["held"])
    _resize_plain(s, seq, s["grown"])
    return _books(s)


def _books(s) -> dict:
    return {**{n: s[n] for n in ("tables", "lengths", "refs", "status")}, **_contents(s)}


def _compact_plain(s) -> dict:
    s["book"].copy_(s["kept"])
    leave, steps = s["leave"].long(), torch.arange(s["width"], device="cuda")[None, :]
    rows = s["tables"][leave]
    _add_refs(s, rows, rows >= 0, -1)
    s["tables"][leave] = -1
    s["lengths"][leave] = 0
    live, index = s["refs"] > 0, torch.arange(s["pages"], device="cuda")
    total = live.sum()
    src, dst = torch.nonzero(live & (index >= total)).squeeze(1), torch.nonzero(~live & (index < total)).squeeze(1)
    for name in ("keys", "key_scales", "values", "value_scales"):
        s[name][:, dst] = s[name][:, src]
    remap = index.to(torch.int32)
    remap[src] = dst.to(torch.int32)
    s["tables"].copy_(torch.where(s["tables"] >= 0, remap[s["tables"].clamp(min=0).long()], s["tables"]))
    s["refs"][dst] = s["refs"][src]
    s["refs"][src] = 0
    s["status"][0] = total
    return _books(s)


# --------------------------------------------------- the framework's calls --

def _handle(s):
    """The program's handle on its cache, its workspace and addresses, made once."""
    if "handle" not in s:
        from needle_cs_amd.paged import PagedCache
        c = s["case"]
        s["handle"] = PagedCache(s["layers"], s["pages"], c["page"], c["kv_heads"], c["qk"], c["v"],
                                 s["tables"].shape[0], s["width"],
                                 buffers={n: s[n].data_ptr() for n in ("keys", "key_scales", "values", "value_scales",
                                                                       "tables", "lengths", "refs")})
        s["at"] = {n: t.data_ptr() for n, t in s.items() if isinstance(t, torch.Tensor)}
        h, kind = s["handle"], c["kind"]
        s["size"] = (h.decode_workspace(s["rows"], c["heads"], s["max_count"]) if kind == "decode" else
                     h.prompt_workspace(s["rows"], c["heads"], c["runs"], s["max_count"]) if kind == "prompt" else
                     0 if kind == "append" else h.pages_workspace(s["count"]))
        s["workspace"] = torch.empty(max(s["size"], 16), dtype=torch.uint8, device="cuda")
        s["ws"] = s["workspace"].data_ptr()
    return s["handle"], s["at"]


def _own(s):
    h, at = _handle(s)
    c, kind = s["case"], s["case"]["kind"]
    if kind == "append":
        ld = s["projected"].shape[1]
        h.append(s["layer"], at["projected"] + 4 * s["k_column"], ld, at["projected"] + 4 * s["v_column"], ld,
                 at["row_seq"], at["row_pos"], s["rows"])
        return _contents(s)
    if kind == "decode":
        h.decode(0, at["q"], at["q_scales"], s["rows"], c["heads"], at["row_seq"], at["row_first"], at["row_count"],
                 s["max_count"], s["ws"], s["size"], at["out"])
        return s["out"]
    if kind == "prompt":
        h.prompt(0, at["q"], at["q_scales"], s["rows"], c["heads"], c["runs"], at["run_rows"], at["run_seq"],
                 at["run_pos"], c["window"], s["max_count"], s["ws"], s["size"], at["out"])
        return s["out"]
    if kind == "branch":
        h.fork(s["count"], at["beams"], at["parents"], at["held"], s["ws"], s["size"])
        h.resize(s["count"], at["beams"], at["grown"], at["status"], s["ws"], s["size"])
        return _books(s)
    import needle_cs_amd as N
    N.check(N.lib().nhip_copy_dev(at["book"], at["kept"], 4 * s["book"].numel(), None))
    h.free(s["count"], at["leave"], s["ws"], s["size"])
    h.compact(at["status"], s["ws"], s["size"])
    return _books(s)


def run(state: dict):
    if own:
        return _own(state)
    return {"append": _append_plain, "decode": _decode_plain, "prompt": _prompt_plain, "branch": _branch_plain,
            "compact": _compact_plain}[state["case"]["kind"]](state)


# ------------------------------------------------------------------ work --

def work(case: dict) -> dict:
    kv, qk, v, page = case["kv_heads"], case["qk"], case["v"], case["page"]
    cell = kv * (qk + v + 8)  # one position of one layer
    if case["kind"] == "append":
        rows = case["sequences"] * case["run"]
        return {"bytes": rows * (4 * kv * (qk + v) + cell + 8), "flops": 3 * rows * kv * (qk + v)}
    if case["kind"] == "decode":
        counts = _spread(case, case["rows"], case["lo"], case["hi"])
        per_row = case["heads"] * (qk + 4 + 4 * v) + 12
        return {"bytes": sum(counts) * cell + len(counts) * per_row,
                "flops": 2 * (qk + v) * case["heads"] * sum(counts)}
    if case["kind"] == "prompt":
        attended, held, rows = 0, 0, 0
        for n, b in zip(*_runs(case)):
            w = case["window"] or n + b
            attended += sum(min(b + i + 1, w) for i in range(n))
            held += min(n + b, n + w - 1)
            rows += n
        return {"bytes": held * cell + rows * case["heads"] * (qk + 4 + 4 * v),
                "flops": 2 * (qk + v) * case["heads"] * attended}
    if case["kind"] == "branch":
        lengths, _ = _beam_pages(case)
        parents, beams = _parents(case), case["beams"]
        copied = sum(beams - len(set(parents[r * beams:(r + 1) * beams])) for r in range(case["requests"])
                     if lengths[r] % page)
        entries = sum(-(-n // page) + 1 for n in lengths) * beams
        return {"bytes": 2 * copied * page * cell * case["layers"] + 4 * entries * 4, "flops": 0}
    need = [-(-n // page) for n in _spread(case, case["sequences"], case["lo"], case["hi"])]
    gone = sum(need[::case["every"]])
    # the pages left sit evenly over the pool: that share of the part behind them moves
    moved = gone * (sum(need) - gone) / sum(need)
    return {"bytes": 2 * moved * page * cell * case["layers"] + 8 * sum(need), "flops": 0}


# ----------------------------------------------------------------- exact --

def _exact_rows(c, s, seq: int, q, qs, first, last):
    """Attention in 64 bits of the rows q [n][heads][qk] over positions first[i]..last[i] of a sequence."""
    kv, group, page = c["kv_heads"], c["heads"] // c["kv_heads"], c["page"]
    pages = s["tables"][seq]
    pages = pages[pages >= 0].long()
    pos = torch.arange(pages.numel() * page, device="cuda")
    out = torch.empty(q.shape[0], c["heads"], c["v"], dtype=torch.float64, device="cuda")
    dead = (pos[None, :] < first[:, None]) | (pos[None, :] > last[:, None])
    for h in range(c["heads"]):
        j = h // group
        k = s["keys"][0, pages, j].reshape(-1, c["qk"]).double() * s["key_scales"][0, pages, j].reshape(-1, 1).double()
        v = s["values"][0, pages, j].transpose(-1, -2).reshape(-1, c["v"]).double()
        v = v * s["value_scales"][0, pages, j].reshape(-1, 1).double()
        z = (q[:, h].double() * qs[:, h, None].double()) @ k.t() / math.sqrt(c["qk"])
        out[:, h] = torch.softmax(z.masked_fill_(dead, -math.inf), dim=-1) @ v
    return out


def exact(case: dict, seed: int):
    """Attention, and an append's scales, in 64 bits; codes, tables and moved pages have no other value than the plain form's."""
    kind = case["kind"]
    if kind in ("branch", "compact"):
        return None
    s = prepare(case, seed)
    if kind == "append":
        ks, vs = s["key_scales"].double(), s["value_scales"].double()
        pos = s["row_pos"].long()
        p = s["tables"][s["row_seq"].long(), pos // case["page"]].long()
        for scales, column, n in ((ks, s["k_column"], case["qk"]), (vs, s["v_column"], case["v"])):
            for j in range(case["kv_heads"]):
                x = s["projected"][:, column + j * n:column + (j + 1) * n].double()
                peak = torch.maximum(x.max(1).values, -x.min(1).values)
                scales[s["layer"], p, j, pos % case["page"]] = torch.where(peak == 0, 1.0, peak / 127)
        return {"keys": None, "key_scales": ks, "values": None, "value_scales": vs}
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
            first = torch.clamp(last - case["window"] + 1, min=0) if case["window"] else torch.zeros_like(last)
            parts.append(_exact_rows(case, s, i, s["q"][at + b:at + b + m], s["q_scales"][at + b:at + b + m], first,
                                     last))
        at += n
    return torch.cat(parts)
