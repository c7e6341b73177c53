"""A server's program over the paged cache, all of its layer steps together:
prompts packed, then one token a sequence and step, window and sinks, ids drawn
from the logits.  Every step against the oracle's and numpy's, then the same
tokens by a captured graph."""
import numpy as np
import pytest

from paged_f64 import Pool
from test_layer_rows_gpu import norm, quantize, rotated
from test_paged_steps_gpu import attend
from test_sampling_gpu import reference

pytestmark = pytest.mark.gpu

LAYERS, D, HEADS, KV, HD, FFN, VOCAB = 2, 256, 8, 2, 64, 512, 600
WINDOW, SINKS, PAGE, WIDTH, SEQUENCES, POSITIONS = 24, 4, 16, 12, 4, 192
SETTINGS = (0.9, 40, 0.95, 0.001)


class Program:
    def __init__(self, hip, orc, seed):
        from needle_cs_amd.paged import PagedCache
        from needle_cs_amd.rotary import Rotary
        self.hip, self.orc = hip, orc
        self.rng = rng = np.random.default_rng(seed)
        st = orc.state(seed)

        def linear(rows, cols):
            w = orc.synth_int8(st, rows * cols).reshape(rows, cols)
            s = orc.synth_half_uniform(st, rows * cols // 32, 0.0002, 0.001).reshape(rows, cols // 32)
            return w, s, hip.Weights.int8(w, s)

        shapes = {"qkv": ((HEADS + 2 * KV) * HD, D), "o": (D, HEADS * HD), "up": (FFN, D), "down": (D, FFN)}
        self.w = [{n: linear(*s) for n, s in shapes.items()} for _ in range(LAYERS)]
        self.head = linear(VOCAB, D)
        self.gains = rng.standard_normal((2 * LAYERS + 1, D)).astype(np.float32) * 0.2
        self.emb = rng.standard_normal((VOCAB, D)).astype(np.float32)
        self.cache = PagedCache(LAYERS, 40, PAGE, KV, HD, HD, SEQUENCES, WIDTH)
        self.table = Rotary.make(POSITIONS, 32, True, kind=3, factor=4.0, original=64.0)
        self.cos, self.sin = (b.download(np.float32).reshape(POSITIONS, 16) for b in self.table.buffers)
        self.bufs = {}
        self.dev("gains", self.gains)

    def dev(self, name, a):
        """A device buffer of the name, made once and filled."""
        a = np.ascontiguousarray(a)
        if name not in self.bufs or self.bufs[name].nbytes < a.nbytes:
            self.bufs[name] = self.hip.DeviceBuffer(max(a.nbytes, 1 << 16))
        self.bufs[name].upload(a)
        return self.bufs[name]

    def room(self, name, nbytes):
        if name not in self.bufs or self.bufs[name].nbytes < nbytes:
            self.bufs[name] = self.hip.DeviceBuffer(max(nbytes, 16))
        return self.bufs[name].ptr

    def grow(self, lengths):
        seq, length = self.dev("seq", np.arange(SEQUENCES, dtype=np.int32)), self.dev("length", np.array(lengths, np.int32))
        status, size = self.dev("status", np.zeros(2, np.int32)), self.cache.pages_workspace(SEQUENCES)
        self.cache.resize(SEQUENCES, seq.ptr, length.ptr, status.ptr, self.room("pages", size), size)
        assert status.download(np.int32, 2).tolist() == [0, 0]

    def upload(self, tokens, seq, pos):
        self.rows = len(tokens)
        self.tokens, self.seq, self.pos = np.array(tokens), np.array(seq, np.int32), np.array(pos, np.int32)
        self.dev("x", self.emb[self.tokens]), self.dev("row_seq", self.seq), self.dev("row_pos", self.pos)
        first = np.maximum(self.pos - WINDOW + 1, 0)
        self.dev("first", first.astype(np.int32)), self.dev("count", (self.pos + 1 - first).astype(np.int32))
        self.heads = np.array([r for r in range(self.rows) if r + 1 == self.rows or seq[r + 1] != seq[r]], np.int32)
        self.random = self.rng.random(len(self.heads)).astype(np.float32)
        self.dev("random", self.random)
        for n, v, t in zip(("temperature", "top_k", "top_p", "min_p"), SETTINGS, (np.float32, np.int32, np.float32, np.float32)):
            self.dev(n, np.full(len(self.heads), v, t))
        starts = np.concatenate([[0], self.heads + 1]).astype(np.int32)
        self.dev("run_rows", starts), self.dev("run_seq", self.seq[self.heads]), self.dev("run_pos", self.pos[starts[:-1]])
        self.reserve()

    def reserve(self):
        """Everything that a step uses, so that a captured one allocates nothing."""
        n = self.rows
        for name, size in (("q", n * FFN), ("qs", 4 * n), ("qkv", 4 * n * (HEADS + 2 * KV) * HD), ("qc", n * HEADS * HD),
                           ("qcs", 4 * n * HEADS), ("att", 4 * n * HEADS * HD), ("delta", 4 * n * D), ("up", 4 * n * FFN),
                           ("logits", 4 * n * VOCAB), ("ids", 4 * n), ("logprobs", 4 * n)):
            self.room(name, size)

    def step(self, stream=None, see=lambda name: None):
        """One forward of the uploaded rows: ids of every run's last row."""
        from needle_cs_amd.rows import add_rms_quantize
        from needle_cs_amd.sampling import Sampling, sample, sample_workspace
        N, n, at = self.hip, self.rows, {k: b.ptr for k, b in self.bufs.items()}
        lib, width = N.lib(), (HEADS + 2 * KV) * HD
        prompt = len(self.heads) < n

        def normed(k, delta):
            add_rms_quantize(at["x"], D, at["delta"] if delta else None, D, at["gains"] + 4 * D * k, True, 1e-6, n, D, at["x"], D,
                             at["q"], at["qs"], stream)

        def product(w, y):
            N.check(lib.nhip_matmul_i8_dev(w[2].handle, at["q"], at["qs"], n, at[y], w[0].shape[0], 0, w[0].shape[0], stream))

        def quantized(x, cols):
            N.check(lib.nhip_quantize_rows_dev(at[x], n, cols, at["q"], at["qs"], stream))

        for layer, w in enumerate(self.w):
            normed(2 * layer, layer > 0), see("norm")
            product(w["qkv"], "qkv"), see("qkv")
            q, k = at["qkv"], at["qkv"] + 4 * HEADS * HD
            self.cache.rotary_append(layer, self.table, q, width, HEADS, k, width, k + 4 * KV * HD, width, at["row_seq"],
                                     at["row_pos"], n, at["qc"], at["qcs"], stream)
            if prompt:
                size = self.cache.prompt_sinks_workspace(n, HEADS, len(self.heads), SINKS, POSITIONS)
                self.cache.prompt_sinks(layer, at["qc"], at["qcs"], n, HEADS, len(self.heads), at["run_rows"], at["run_seq"],
                                        at["run_pos"], WINDOW, SINKS, POSITIONS, self.room("ws", size), size, at["att"], stream)
            else:
                size = self.cache.decode_sinks_workspace(n, HEADS, SINKS, WINDOW)
                self.cache.decode_sinks(layer, at["qc"], at["qcs"], n, HEADS, at["row_seq"], at["first"], at["count"], SINKS,
                                        WINDOW, self.room("ws", size), size, at["att"], stream)
            see("attention")
            quantized("att", HEADS * HD), product(w["o"], "delta")
            normed(2 * layer + 1, True), see("norm")
            product(w["up"], "up"), quantized("up", FFN), product(w["down"], "delta")
        normed(2 * LAYERS, True), see("norm")
        product(self.head, "logits")
        if prompt:  # the runs' last rows
            for i, r in enumerate(self.heads):
                N.check(lib.nhip_copy_dev(at["logits"] + 4 * VOCAB * i, at["logits"] + 4 * VOCAB * int(r), 4 * VOCAB, stream))
        size = sample_workspace(len(self.heads), VOCAB)
        sample(at["logits"], VOCAB, VOCAB, len(self.heads),
               Sampling(at["random"], at["temperature"], at["top_k"], at["top_p"], at["min_p"]), None, 0, 0,
               self.room("sample", size), size, at["ids"], at["logprobs"], stream)

    def get(self, name, dtype, *shape):
        return self.bufs[name].download(dtype, int(np.prod(shape))).reshape(shape)

    def ids(self):
        return self.get("ids", np.int32, len(self.heads))


class Mirror:
    """The same steps on the host, each from what the device had before it."""

    def __init__(self, program):
        self.p = program
        self.x, self.delta, self.k = program.emb[program.tokens], None, 0
        self.order = iter([(layer, s) for layer in range(LAYERS) for s in ("norm", "qkv", "attention", "norm")] + [(LAYERS, "norm")])

    def product(self, w, q, qs):
        y = np.zeros((len(q), w[0].shape[0]), dtype=np.float32)
        self.p.orc.matmul_rows_i8(w[0], w[1], q, qs, len(q), y, w[0].shape[0], 0, w[0].shape[0])
        return y

    def see(self, name):
        p, n = self.p, self.p.rows
        p.hip.check(p.hip.lib().nhip_stream_sync(None))
        layer, want = next(self.order)
        assert name == want
        if name == "norm":
            if self.delta is not None and self.delta.shape[1] == FFN:
                q, qs = quantize(self.delta)
                self.delta = self.product(p.w[layer - 1]["down"], q, qs)
            s, q, qs = norm(self.x, self.delta, p.gains[self.k], True, 1e-6)
            assert np.array_equal(p.get("x", np.float32, n, D), s)
            assert np.array_equal(p.get("q", np.int8, n, D), q) and np.array_equal(p.get("qs", np.float32, n), qs)
            self.x, self.k = s, self.k + 1
            self.q, self.qs = q, qs
            if self.k > 1 and self.k % 2 == 0 and layer < LAYERS:  # behind the attention
                self.delta = self.product(p.w[layer]["up"], q, qs)
            elif layer == LAYERS:
                self.logits = self.product(p.head, q, qs)
        elif name == "qkv":
            self.qkv = self.product(p.w[layer]["qkv"], self.q, self.qs)
            assert np.array_equal(p.get("qkv", np.float32, n, (HEADS + 2 * KV) * HD), self.qkv)
        else:
            heads = self.qkv.reshape(n, -1, HD)
            turned = rotated(heads[:, :HEADS + KV], p.cos[p.pos], p.sin[p.pos], 32, True)
            codes, scales = quantize(turned[:, :HEADS])
            assert np.array_equal(p.get("qc", np.int8, n, HEADS, HD), codes)
            assert np.array_equal(p.get("qcs", np.float32, n, HEADS), scales)
            pool = self.pool()
            (kc, ks), (vc, vs) = quantize(turned[:, HEADS:]), quantize(heads[:, HEADS + KV:])
            out = p.get("att", np.float32, n, HEADS, HD)
            for r in range(n):
                s, pos = int(p.seq[r]), int(p.pos[r])
                for h in range(KV):
                    got = pool.position(layer, s, h, pos)
                    assert np.array_equal(got[0], kc[r, h]) and got[1] == ks[r, h]
                    assert np.array_equal(got[2], vc[r, h]) and got[3] == vs[r, h]
                seen = [x for x in range(pos + 1) if x > pos - WINDOW or x < SINKS]
                exact, far = attend(pool, layer, s, codes[r], scales[r], seen, prompt=True)
                assert (np.abs(out[r] - exact) <= far).all()
            q, qs = quantize(out.reshape(n, -1))
            self.delta = self.product(p.w[layer]["o"], q, qs)

    def pool(self):
        """The cache's arrays as they are."""
        pool = Pool(np.random.default_rng(0), LAYERS, 40, PAGE, KV, HD, HD, SEQUENCES, WIDTH)
        for name in Pool.NAMES:
            a = getattr(pool, name)
            a[:] = self.p.cache.buffers[name].download(a.dtype).reshape(a.shape)
        return pool

    def ids(self):
        p = self.p
        return [reference(self.logits[r], np.ones(VOCAB, bool), u, *SETTINGS)[0] for r, u in zip(p.heads, p.random)]


PROMPTS = [37, 1, 60, 12]


def prompts(rng):
    return [rng.integers(0, VOCAB, n).tolist() for n in PROMPTS]


def test_prompts_and_steps_against_the_host(hip, orc):
    p = Program(hip, orc, 11)
    lengths = [0] * SEQUENCES
    new = prompts(p.rng)
    for step in range(4):
        rows = [(t, s, lengths[s] + i) for s in range(SEQUENCES) for i, t in enumerate(new[s])]
        lengths = [a + len(b) for a, b in zip(lengths, new)]
        p.grow(lengths)
        p.upload(*zip(*rows))
        mirror = Mirror(p)
        p.step(see=mirror.see)
        ids = p.ids()
        assert ids.tolist() == mirror.ids()
        new = [[int(t)] for t in ids]


def test_steps_by_a_graph_are_the_steps(hip, orc):
    """One program eager, one whose decode step is a graph on a stream of its own: the same tokens and logits."""
    a, b = Program(hip, orc, 12), Program(hip, orc, 12)
    stream, graph, lengths = hip.Stream(), None, [0] * SEQUENCES
    new = prompts(np.random.default_rng(5))
    for step in range(12):
        rows = [(t, s, lengths[s] + i) for s in range(SEQUENCES) for i, t in enumerate(new[s])]
        lengths = [x + len(y) for x, y in zip(lengths, new)]
        for p in (a, b):
            p.grow(lengths)
            p.upload(*zip(*rows))
        a.step()
        ids = a.ids()
        if step == 0:
            b.step()
        else:
            hip.check(hip.lib().nhip_device_sync())
            if graph is None:
                b.room("ws", 16)
                with hip.Graph.capture(stream) as graph:
                    b.step(stream.ptr)
            graph.launch()
            stream.sync()
        assert np.array_equal(b.ids(), ids)
        assert np.array_equal(a.get("logits", np.float32, SEQUENCES, VOCAB), b.get("logits", np.float32, SEQUENCES, VOCAB))
        assert np.array_equal(a.get("logprobs", np.float32, SEQUENCES), b.get("logprobs", np.float32, SEQUENCES))
        new = [[int(t)] for t in ids]
    graph.close()
