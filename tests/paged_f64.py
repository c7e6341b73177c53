"""The paged cache in plain numpy: attention in 64 bits from the formula, and
the pages' bookkeeping one entry at a time."""
import numpy as np


class Pool:
    """A paged cache's arrays on the host, filled with random codes and with
    NaN scales where no sequence holds a position."""

    def __init__(self, rng, layers, pages, page, kv, qk, v, sequences, width):
        self.dims = (layers, pages, page, kv, qk, v, sequences, width)
        self.layers, self.pages, self.page, self.kv, self.qk, self.v, self.sequences, self.width = self.dims
        self.keys = rng.integers(-128, 128, (layers, pages, kv, page, qk), dtype=np.int8)
        self.values = rng.integers(-128, 128, (layers, pages, kv, page // 16, v, 16), dtype=np.int8)
        self.key_scales = np.full((layers, pages, kv, page), np.nan, dtype=np.float32)
        self.value_scales = np.full((layers, pages, kv, page), np.nan, dtype=np.float32)
        self.tables = np.full((sequences, width), -1, dtype=np.int32)
        self.lengths = np.zeros(sequences, dtype=np.int32)
        self.refs = np.zeros(pages, dtype=np.int32)

    NAMES = ("keys", "key_scales", "values", "value_scales", "tables", "lengths", "refs")

    def give(self, rng, lengths, spread=0.0):
        """Sequence i holds lengths[i] positions on scattered pages.  Scales
        are uniform in [0.01, 0.03], times e^(spread * normal)."""
        order = iter(rng.permutation(self.pages))
        for i, n in enumerate(lengths):
            self.lengths[i] = n
            for t in range(-(-n // self.page)):
                p = next(order)
                self.tables[i, t] = p
                self.refs[p] = 1
                live = min(n - t * self.page, self.page)
                for s in (self.key_scales, self.value_scales):
                    x = rng.uniform(0.01, 0.03, (self.layers, self.kv, live))
                    s[:, p, :, :live] = x * np.exp(spread * rng.standard_normal(x.shape))

    def position(self, layer, seq, kvh, pos):
        """(k, ks, v, vs) of one position, None on a page outside the pool."""
        p = self.tables[seq, pos // self.page]
        if not 0 <= p < self.pages:
            return None
        at = pos % self.page
        return (self.keys[layer, p, kvh, at], self.key_scales[layer, p, kvh, at],
                self.values[layer, p, kvh, at // 16, :, at % 16], self.value_scales[layer, p, kvh, at])

    def attend(self, layer, seq, q, q_scales, first, count, prompt=False):
        """One row's [heads][v] in 64 bits, and per output the bound of the
        kernel's error (see `bound` and FLOOR)."""
        heads = q.shape[0]
        out, far = np.zeros((heads, self.v)), np.zeros((heads, self.v))
        for h in range(heads):
            cells = [self.position(layer, seq, h // (heads // self.kv), p) for p in range(first, first + count)]
            cells = [c for c in cells if c is not None]
            if not cells:
                continue
            k = np.array([c[0] for c in cells], dtype=np.float64)
            ks = np.array([c[1] for c in cells], dtype=np.float64)
            v = np.array([c[2] for c in cells], dtype=np.float64)
            vs = np.array([c[3] for c in cells], dtype=np.float64)
            z = (k @ q[h].astype(np.float64)) * ks * float(q_scales[h]) / np.sqrt(self.qk)
            w = np.exp(z - z.max())
            w /= w.sum()
            out[h] = (w * vs) @ v
            far[h] = bound(len(cells), np.abs(z).max(), vs) * ((w * np.abs(vs)) @ np.abs(v))
            largest = vs.max() * PROMPT_LAG if prompt else (w * np.abs(vs)).max()
            far[h] += FLOOR * 2 * largest * np.abs(v).sum(0)
        return out, far

    def attend_products(self, layer, seq, q, q_scales, first, count, prompt=False):
        """As attend, with the bound that holds whatever the scales are: the
        floor is that of the largest weight times scale (PROMPT_LAG behind it in
        a prompt), and values whose codes are all 0 have no part in it."""
        heads = q.shape[0]
        out, far = np.zeros((heads, self.v)), np.zeros((heads, self.v))
        at = np.arange(first, first + count)
        t, at = self.tables[seq, at // self.page], at % self.page
        for h in range(heads):
            j = h // (heads // self.kv)
            k, ks = self.keys[layer, t, j, at].astype(np.float64), self.key_scales[layer, t, j, at].astype(np.float64)
            v = self.values[layer, t, j, at // 16, :, at % 16].astype(np.float64)
            vs = np.where(v.any(1), self.value_scales[layer, t, j, at].astype(np.float64), 0.0)
            z = (k @ q[h].astype(np.float64)) * ks * float(q_scales[h]) / np.sqrt(self.qk)
            w = np.exp(z - z.max())
            w /= w.sum()
            out[h] = (w * vs) @ v
            far[h] = bound(count, np.abs(z).max(), vs[vs > 0] if vs.any() else np.ones(1)) * ((w * vs) @ np.abs(v))
            far[h] += FLOOR * 2 * (w * vs).max() * (PROMPT_LAG if prompt else 1.0) * np.abs(v).sum(0)
        return out, far


#: The weights w vs enter the value product as two fp16 numbers.  Below 2^-14
#: fp16 has a step of 2^-24, so a weight is off by up to 2^-25 besides its
#: relative error, where the largest is scaled to [2^14, 2^15): 2^-39 of it (an
#: output whose large weights all meet code 0 shows this floor alone).
FLOOR = 2.0 ** -39

#: A prompt's weights are scaled by the running maximum that is up to 2^8 behind
#: and by the largest value scale that the row attends, not by the product.
PROMPT_LAG = 2.0 ** 8


def bound(count, z, vs):
    """The relative error that fp32 allows a weighted mean of `count` terms
    with scores up to z, in units of half a step (2^-24).  A score is a
    product of four factors, two of them rounded constants (6 roundings of
    |z|), taken to base 2 with the scale's exponent added (2 of |z| + |log2
    vs|), less the maximum (the same again); e^x is within 4 steps and a
    weight's rounding, scale and split within 8; weights enter both sums, so
    all of it twice.  A sum of n terms by chains and trees rounds at most n
    times, 4 + n / 4 allowed for the matrix units' inner sums and 64 for
    joining parts."""
    exponent = np.abs(np.log2(np.maximum(np.abs(vs), 2.0 ** -60))).max()
    score = 1.4427 * z
    return 2.0 ** -24 * (2 * (6 * score + 4 * (score + exponent) + 12) + 68 + count / 4)


class Books:
    """tables, lengths and refs, changed one entry at a time."""

    def __init__(self, pool):
        self.page, self.width, self.pages = pool.page, pool.width, pool.pages
        self.tables, self.lengths, self.refs = pool.tables.copy(), pool.lengths.copy(), pool.refs.copy()
        self.moved = []  # (from, to) pages whose contents were copied, in one call

    def count(self, n):
        return -(-int(n) // self.page)

    def fork(self, dst, src, length=None):
        before, lengths = self.tables.copy(), self.lengths.copy()
        seen = set()
        for i, (d, s) in enumerate(zip(dst, src)):
            if d in seen:
                continue
            seen.add(d)
            if not (0 <= d < len(lengths) and 0 <= s < len(lengths)):
                continue
            n = int(lengths[s]) if length is None else min(max(int(length[i]), 0), int(lengths[s]))
            for t in range(self.count(lengths[d])):
                self.refs[before[d, t]] -= 1
            self.tables[d] = -1
            for t in range(self.count(n)):
                self.tables[d, t] = before[s, t]
                self.refs[before[s, t]] += 1
            self.lengths[d] = n

    def resize(self, seq, length):
        """Returns (missing, refused)."""
        free = [p for p in range(self.pages) if self.refs[p] == 0]
        plan, refused, seen, growers = [], 0, set(), {}
        for s, n in zip(seq, length):
            if not (0 <= s < len(self.lengths) and 0 <= n <= self.width * self.page):
                refused += 1
                seen.add(s)
                continue
            if s in seen:
                continue
            seen.add(s)
            old = int(self.lengths[s])
            copy = False
            if n > old and old % self.page:
                tail = self.tables[s, self.count(old) - 1]
                copy = growers.get(tail, 0) < self.refs[tail] - 1
                growers[tail] = growers.get(tail, 0) + 1
            plan.append((s, int(n), old, copy))
        need = sum(c + max(self.count(n) - self.count(o), 0) for _, n, o, c in plan)
        if need > len(free):
            return need - len(free), refused
        self.moved = []
        at = iter(free)
        for s, n, old, copy in plan:
            a, b = self.count(old), self.count(n)
            if copy:
                p = next(at)
                self.moved.append((int(self.tables[s, a - 1]), p))
                self.refs[self.tables[s, a - 1]] -= 1
                self.refs[p] += 1
                self.tables[s, a - 1] = p
            for t in range(a, b):
                self.tables[s, t] = next(at)
                self.refs[self.tables[s, t]] += 1
            for t in range(b, a):
                self.refs[self.tables[s, t]] -= 1
                self.tables[s, t] = -1
            self.lengths[s] = n
        return 0, refused

    def compact(self):
        n = int((self.refs > 0).sum())
        holes = [p for p in range(n) if self.refs[p] == 0]
        movers = [p for p in range(n, self.pages) if self.refs[p] > 0]
        self.moved = list(zip(movers, holes))
        to = dict(self.moved)
        for s in range(len(self.lengths)):
            for t in range(self.width):
                self.tables[s, t] = to.get(int(self.tables[s, t]), self.tables[s, t])
        for a, b in self.moved:
            self.refs[b], self.refs[a] = self.refs[a], 0
        return n
