"""The paged cache as a server uses it: tables with room for far more than they hold, calls captured and replayed while
sequences grow, calls on several streams and threads at once, and a layer of a model from its input to its output."""
import ctypes
import threading

import numpy as np
import pytest

import serving
import test_gpu_kv_cache as kv_cache
from layers import Matrix, block64, linear64, quantize, rounded
from serving import Ints, Pool, Serving, attend64, close, held64, turned64
from simdonnx_amd import native as N
from simdonnx_amd import synth
from simdonnx_amd.backend import HipBlockNorm, HipKvBatch, HipKvCache, HipQuantLinear, HipRotary
from test_gpu_block_norm import inside, params
from test_gpu_kv_cache import normal

pytestmark = pytest.mark.gpu
FORMATS = [("f16", "f16"), ("bf16", "bf16"), ("f32", "f32"), ("f16", "i8"), ("bf16", "i8"), ("f32", "i8")]


class Stream:
    def __enter__(self):
        self.h = N.c_void_p()
        N.check(N.thin().sox_stream_create(ctypes.byref(self.h)), "stream")
        return self.h

    def __exit__(self, *_):
        N.thin().sox_stream_destroy(self.h)


def captured(stream, call):
    T = N.thin()
    N.check(T.sox_graph_begin(stream), "capture")
    call()
    graph = N.c_void_p()
    N.check(T.sox_graph_end(stream, ctypes.byref(graph)), "capture end")
    return graph


# ---- tables with room to grow: the kernel over tiles of 128 pairs, and splits that find no token ----
@pytest.mark.parametrize("storage,fmt", FORMATS)
@pytest.mark.parametrize("case", range(len(kv_cache.ATTENDS)))
def test_attend_with_room(hip, monkeypatch, case, storage, fmt):
    monkeypatch.setattr(serving, "TABLE_TOKENS", 1 << 19)
    kv_cache.test_attend(hip, case, storage, fmt)


@pytest.mark.parametrize("storage", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("case", [([(90, 40)], 1, 2, 72, 16, 0), ([(150, 150)], 1, 1, 128, 8, 20), ([(300, 130), (33, 2)], 2, 2, 64, 16, 0)])
def test_values_that_are_not_finite_with_room(hip, monkeypatch, case, storage):
    monkeypatch.setattr(serving, "TABLE_TOKENS", 1 << 19)
    kv_cache.test_values_that_are_not_finite(hip, case, storage)


def test_other_contents_with_room(hip, monkeypatch):
    """Infinite values in 8 bits, scales far apart, pages that are not there, tables of none."""
    monkeypatch.setattr(serving, "TABLE_TOKENS", 1 << 19)
    kv_cache.test_infinite_v_in_8_bits(hip)
    for fmt in ("bf16", "i8"):
        kv_cache.test_scales_far_apart(hip, fmt)
    kv_cache.test_no_page_at_all(hip)


# ---- 8 bits of values next to the middle between two integers ----
@pytest.mark.parametrize("storage", ["f16", "bf16", "f32"])
def test_halves_of_turned_keys(hip, storage):
    """Keys at position 0, which turn by nothing: n + 1/2 of 127 steps rounds to even, whatever the row's scale, and so do its
    neighbours in fp32 to either side."""
    rows, kv, dim = 60, 3, 64
    rng = np.random.default_rng(1)
    k = rng.integers(-63, 63, (rows, kv, dim)).astype(np.float32) + 0.5
    k[..., rng.integers(dim)] = 127
    if storage == "f32":
        k[1::3], k[2::3] = np.nextafter(k[1::3], np.float32(1e9)), np.nextafter(k[2::3], np.float32(-1e9))
    by = np.exp2(rng.integers(-4, 4, (rows, kv, 1))) if storage == "f16" else np.exp2(rng.integers(-100, 100, (rows, kv, 1)))
    k = (k * by).astype(np.float32)
    assert np.array_equal(rounded(k, storage), k)
    s = Serving(hip, [(1, 1)] * rows, kv, dim, 4, "i8")
    r = HipRotary(hip, dim)
    K, V = Matrix(k.reshape(rows, -1), storage), Matrix(normal(2, storage, rows, kv * dim), storage)
    K2, V2 = Matrix(None, "f32", rows, kv * dim), Matrix(None, "f32", rows, kv * dim)
    s.cache.write(s.batch, K.ptr, V.ptr, storage, rotary=r)
    s.cache.read(s.batch, K2.ptr, V2.ptr, "f32")
    q, scale = quantize(k.reshape(-1, dim))
    want = (q.astype(np.float32) * scale.astype(np.float32)[:, None]).reshape(rows, -1)
    assert np.array_equal(K2.read(), want)
    for m in (K, V, K2, V2):
        m.free()
    r.close()
    s.free()


# ---- the ends of what is allowed ----
@pytest.mark.parametrize("room", [0, 1 << 19])
@pytest.mark.parametrize("fmt", ["f16", "i8"])
def test_widest_window(hip, monkeypatch, fmt, room):
    """A window of 2^31 - 1 tokens is none, also where a sequence has more rows than tokens."""
    monkeypatch.setattr(serving, "TABLE_TOKENS", room)
    case = ([(300, 150), (40, 40), (70, 1)], 2, 2, 64, 16, 0)
    s, k, v, q, K, V, Q, Y, W = kv_cache.attend_case(hip, case, "f16", fmt)
    s.d_lengths.write([300, 25, 70])
    for window in (0, 2 ** 31 - 1, 2 ** 30):
        Y.refill()
        s.cache.attend(s.batch, Q.ptr, 4, Y.ptr, "f16", window=window, workspace=W.ptr, workspace_bytes=W.cols)
        y = Y.read()
        if window == 0:
            first = y
            hk, hv = held64(k, "f16", fmt), held64(v, "f16", fmt)
            rows = slice(s.starts[1] + 15, s.starts[2])  # (25 tokens: rows 15 .. 39 hold them)
            want, tol = attend64(q[rows].astype(np.float64), hk[300:325], hv[300:325], 0, 0.125, 0, "f16")
            close(y[rows].reshape(want.shape), want, tol, "y")
        own = s.positions() >= 0
        own[s.starts[1]:s.starts[1] + 15] = False
        assert np.array_equal(y[own], first[own]) and kv_cache.untouched(Y, ~own)
    for m in (K, V, Q, Y, W):
        m.free()
    s.free()


def test_page_past_2_gib(hip):
    """A page whose scales stand behind 2^31 bytes."""
    kv, dim, n = 1024, 256, 9
    cache = HipKvCache(hip, kv, dim, page=4096, format="i8")
    assert 2 ** 31 < cache.page_bytes < 2 ** 32
    p = ctypes.c_void_p()
    N.check(N.thin().sox_malloc(ctypes.byref(p), cache.page_bytes), "page")
    T, S, L, S1 = Ints([0]), Ints([0, n]), Ints([n]), Ints([0, 1])
    k, v, q = normal(1, "f16", n, kv, dim), normal(2, "f16", n, kv, dim), normal(3, "f16", n, kv, dim)
    K, V, Q = (Matrix(x.reshape(n, -1), "f16") for x in (k, v, q))
    Y, K2, V2 = (Matrix(None, "f16", n, kv * dim) for _ in range(3))
    W = Matrix(None, "i8", 1, cache.workspace(n, 1, kv))
    whole = HipKvBatch(p.value, 1, T.ptr, 1, S.ptr, L.ptr, 1, n)
    print("[gpu] page past 2 GiB", flush=True)
    cache.write(whole, K.ptr, V.ptr, "f16")
    cache.read(whole, K2.ptr, V2.ptr, "f16")
    hk, hv = held64(k, "f16", "i8"), held64(v, "f16", "i8")
    for m, want in ((K2, hk), (V2, hv)):
        close(m.read().reshape(want.shape), want, (2.0 ** -11 + 2.0 ** -24) * np.abs(want) + 2.0 ** -25, "read")
    want, tol = attend64(q.astype(np.float64), hk, hv, 0, 1 / 16, 0, "f16")
    cache.attend(whole, Q.ptr, kv, Y.ptr, "f16", workspace=W.ptr, workspace_bytes=W.cols)
    close(Y.read().reshape(want.shape), want, tol, "rows")
    one = HipKvBatch(p.value, 1, T.ptr, 1, S1.ptr, L.ptr, 1, 1)  # (row 0 as the last token)
    want, tol = attend64(q[:1].astype(np.float64), hk, hv, n - 1, 1 / 16, 0, "f16")
    cache.attend(one, Q.ptr, kv, Y.ptr, "f16", workspace=W.ptr, workspace_bytes=W.cols)
    close(Y.read().reshape(q.shape)[:1], want, tol, "one row")
    for m in (T, S, L, S1, K, V, Q, Y, K2, V2, W):
        m.free()
    N.thin().sox_free(p)
    cache.close()


# ---- weights that are small each and count together ----
@pytest.mark.parametrize("room", [0, 1 << 19])
@pytest.mark.parametrize("storage,fmt", FORMATS)
@pytest.mark.parametrize("new", [1, 64])
def test_many_small_weights(hip, monkeypatch, storage, fmt, room, new):
    """One token of weight 1 and 4095 of 2^-16, below fp16's normal numbers, with the opposite value."""
    monkeypatch.setattr(serving, "TABLE_TOKENS", room)
    n, dim = 4096, 64
    s = Serving(hip, [(n, new)], 1, dim, 16, fmt)
    k, v, q = np.zeros((n, 1, dim), np.float32), -np.ones((n, 1, dim), np.float32), np.zeros((new, 2, dim), np.float32)
    k[100, 0, 0], v[100] = rounded(np.array([[16 * np.log(2.0)]], np.float32), storage)[0, 0], 1
    q[..., 0] = 8  # (scale 1 / 8: the score is k's first value)
    K, V, Q, Y = Matrix(k.reshape(n, -1), storage), Matrix(v.reshape(n, -1), storage), Matrix(q.reshape(new, -1), storage), Matrix(None, storage, new, 2 * dim)
    W = Matrix(None, "i8", 1, s.cache.workspace(new, 1, 2))
    s.cache.write(s.every, K.ptr, V.ptr, storage)
    s.cache.attend(s.batch, Q.ptr, 2, Y.ptr, storage, workspace=W.ptr, workspace_bytes=W.cols)
    want, tol = attend64(q.astype(np.float64), held64(k, storage, fmt), held64(v, storage, fmt), n - new, dim ** -0.5, 0, storage)
    assert 0.87 < want.min() and want.max() < 0.9  # (without the small weights it would be 1)
    close(Y.read().reshape(want.shape), want, tol, "y")
    for m in (K, V, Q, Y, W):
        m.free()
    s.free()


# ---- captured ----
class Side:
    """A batch, its workspace and its stream, with room for its sequences to grow."""

    def __init__(self, hip, cache, rotary, heads, lengths, seed, storage, stream, room=512):
        self.cache, self.rotary, self.heads, self.storage, self.stream = cache, rotary, heads, storage, stream
        n, kv, dim = len(lengths), cache.kv_heads, cache.head_dim
        per = room // cache.page
        self.pages = n * per + 3
        self.rng = np.random.default_rng(seed)
        self.pool = Pool(cache, self.pages)
        self.tables = self.rng.permutation(self.pages)[:n * per].reshape(n, per)
        self.lengths = np.array(lengths)
        self.d = [Ints(self.tables), Ints(np.arange(n + 1)), Ints(self.lengths)]
        self.batch = HipKvBatch(self.pool.ptr, self.pages, self.d[0].ptr, per, self.d[1].ptr, self.d[2].ptr, n, n)
        self.width = (heads + 2 * kv) * dim
        self.F, self.Q, self.Y = (Matrix(None, storage, n, w) for w in (self.width, heads * dim, heads * dim))
        self.W = Matrix(None, "i8", 1, cache.workspace(n, n, heads))
        # what the cache holds so far
        self.k, self.v = [], []
        for i, length in enumerate(self.lengths):
            past = [normal(seed + 2 + i, storage, length - 1, kv, dim), normal(seed + 40 + i, storage, length - 1, kv, dim)]
            if length > 1:
                T, S, L = Ints(self.tables[i]), Ints([0, length - 1]), Ints([length - 1])
                b = HipKvBatch(self.pool.ptr, self.pages, T.ptr, per, S.ptr, L.ptr, 1, length - 1)
                K, V = (Matrix(x.reshape(length - 1, -1), storage) for x in past)
                cache.write(b, K.ptr, V.ptr, storage, rotary=rotary)
                for m in (T, S, L, K, V):
                    m.free()
            self.k.append(held64(turned64(past[0], np.arange(length - 1), rotary.frequencies, False)[0], storage, cache.format))
            self.v.append(held64(past[1], storage, cache.format))

    def call(self):
        e, dim, kv = self.F.elem * self.cache.head_dim, self.cache.head_dim, self.cache.kv_heads
        self.cache.write(self.batch, self.F.ptr + self.heads * e, self.F.ptr + (self.heads + kv) * e, self.storage, self.F.ld, self.F.ld,
                         rotary=self.rotary, q=self.F.ptr, ldq=self.F.ld, q_heads=self.heads, y=self.Q.ptr, stream=self.stream)
        self.cache.attend(self.batch, self.Q.ptr, self.heads, self.Y.ptr, self.storage, workspace=self.W.ptr, workspace_bytes=self.W.cols,
                          stream=self.stream)

    def feed(self, seed, grow, move=False):
        """The next token of each sequence, `grow` further on than the last; the pages that hold nothing yet in another order."""
        n, dim, kv = len(self.lengths), self.cache.head_dim, self.cache.kv_heads
        x = normal(seed, self.storage, n, self.heads + 2 * kv, dim)
        X = Matrix(x.reshape(n, -1), self.storage)
        N.check(N.thin().sox_memcpy_d2d(self.F.ptr, X.ptr, x.size * X.elem, self.stream), "next tokens")
        N.check(N.thin().sox_stream_sync(self.stream), "sync")
        X.free()
        self.lengths = self.lengths + grow
        if move:
            for i, length in enumerate(self.lengths):
                first = -(-(length - 1) // self.cache.page)
                self.tables[i, first:] = self.rng.permutation(self.tables[i, first:])
            self.d[0].write(self.tables)
        self.d[2].write(self.lengths)
        pos = self.lengths - 1
        k = turned64(x[:, self.heads:self.heads + kv], pos, self.rotary.frequencies, False)[0]
        for i in range(n):
            for held, new in ((self.k, k[i:i + 1]), (self.v, x[i:i + 1, self.heads + kv:])):
                held[i] = np.concatenate([held[i][:pos[i]], held64(new, self.storage, self.cache.format)])

    def check(self, what):
        q, y = (m.read().reshape(len(self.lengths), self.heads, -1) for m in (self.Q, self.Y))
        for i in range(len(self.lengths)):
            want, tol = attend64(q[i:i + 1].astype(np.float64), self.k[i], self.v[i], self.lengths[i] - 1, self.cache.head_dim ** -0.5, 0, self.storage)
            close(y[i:i + 1], want, tol, f"{what}, sequence {i}")

    def free(self):
        for m in (self.pool, self.F, self.Q, self.Y, self.W, *self.d):
            m.free()


def test_captured_steps_while_sequences_grow(hip):
    """Two sides with a cache object in common, each captured once: every replay reads lengths, tables and tokens as they are,
    gives the eager call's bits, and both sides replay on their streams at once."""
    cache, rotary, T = HipKvCache(hip, 2, 64, page=16, format="i8"), HipRotary(hip, 64), N.thin()
    with Stream() as s0, Stream() as s1:
        sides = [Side(hip, cache, rotary, 8, lengths, seed, "f16", st) for lengths, seed, st in (([1, 40, 300], 100, s0), ([17, 16, 129, 64], 200, s1))]
        graphs = []
        for i, side in enumerate(sides):
            print(f"[gpu] serving capture {i}", flush=True)
            side.feed(300 + i, 0)
            graphs.append(captured(side.stream, side.call))
        for step in range(4):
            eager = []
            for i, side in enumerate(sides):
                side.feed(400 + 10 * step + i, int(step > 0), move=step == 2)
                side.call()
                N.check(T.sox_stream_sync(side.stream), "sync")
                side.check(f"step {step} side {i}")
                eager.append(side.Y.read())
                side.Y.refill()
                side.Q.refill()
            for rep in range(2):
                for side, g in zip(sides, graphs):
                    N.check(T.sox_graph_launch(g, side.stream), "replay")
            for side, want in zip(sides, eager):
                N.check(T.sox_stream_sync(side.stream), "sync")
                assert np.array_equal(side.Y.read(), want), step
        for g in graphs:
            T.sox_graph_destroy(g)
        for side in sides:
            side.free()
    cache.close()
    rotary.close()


def test_calls_from_threads(hip):
    """Threads with streams, batches and workspaces of their own share a cache object and a rotary."""
    cache, rotary, T = HipKvCache(hip, 1, 128, page=8, format="bf16"), HipRotary(hip, 128, rotary_dim=64), N.thin()
    with Stream() as s0, Stream() as s1, Stream() as s2:
        sides = [Side(hip, cache, rotary, 4, [30 + 50 * i, 200], 500 + 100 * i, "bf16", st) for i, st in enumerate((s0, s1, s2))]
        want = []
        for i, side in enumerate(sides):
            side.feed(600 + i, 0)
            side.call()
            N.check(T.sox_stream_sync(side.stream), "sync")
            want.append(side.Y.read())
        errors = []

        def work(side):
            try:
                for _ in range(20):
                    side.call()
                N.check(T.sox_stream_sync(side.stream), "sync")
            except Exception as e:  # noqa: BLE001
                errors.append(e)

        print("[gpu] serving threads", flush=True)
        threads = [threading.Thread(target=work, args=(side,)) for side in sides]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        assert not errors
        for side, w in zip(sides, want):
            assert np.array_equal(side.Y.read(), w)
            side.free()
    cache.close()
    rotary.close()


# ---- a layer ----
def test_layer_as_served(hip):
    """A decoder layer's first half over three prompts and then their next tokens: an 8-bit projection to queries, keys and
    values, positions and cache, attention, the 8-bit projection back, residual and norm. Each step against the 64-bit
    step of what the device had before it; the single tokens' run is captured once and replayed as the sequences grow."""
    storage, c, kv, heads, dim, page = "f16", 128, 2, 4, 32, 8
    T = N.thin()
    prompts, room = [37, 5, 20], 64
    w1, w2 = synth.normal(900, 1, (c, (heads + 2 * kv) * dim), 0.1), synth.normal(900, 2, (heads * dim, c), 0.1)
    b1 = synth.uniform(900, 3, ((heads + 2 * kv) * dim,), -0.2, 0.2)
    p = params(901, c, "none", "rms")
    qkv, back, norm = HipQuantLinear(hip, w1, b1, c, w1.shape[1]), HipQuantLinear(hip, w2, None, heads * dim, c), HipBlockNorm(hip, c, **p)
    cache, rotary = HipKvCache(hip, kv, dim, page=page, format="i8"), HipRotary(hip, dim, base=5e5, factor=8.0, original=4096)
    pages = 3 * room // page + 1
    pool, tables = Pool(cache, pages), np.random.default_rng(3).permutation(pages)[:3 * room // page].reshape(3, -1)
    d_tables = Ints(tables)
    held = [[np.zeros((0, kv, dim))] * 2 for _ in prompts]

    class Run:
        def __init__(self, counts, lengths, stream):
            self.counts, self.stream, self.rows = counts, stream, sum(counts)
            self.starts, self.lengths = Ints(np.cumsum([0] + counts)), Ints(lengths)
            self.batch = HipKvBatch(pool.ptr, pages, d_tables.ptr, tables.shape[1], self.starts.ptr, self.lengths.ptr, 3, self.rows)
            mk = lambda cols: Matrix(None, storage, self.rows, cols)  # noqa: E731
            self.X, self.F, self.Q, self.A, self.O, self.H, self.Z = (mk(n) for n in (c, w1.shape[1], heads * dim, heads * dim, c, c, c))
            need = max(qkv.workspace(self.rows), back.workspace(self.rows), cache.workspace(self.rows, 3, heads), 1)
            self.W = Matrix(None, "i8", 1, need)
            self.every = (self.F, self.Q, self.A, self.O, self.H, self.Z)

        def feed(self, seed, lengths):
            x = normal(seed, storage, self.rows, c)
            X = Matrix(x, storage)
            N.check(T.sox_memcpy_d2d(self.X.ptr, X.ptr, x.size * 2, self.stream), "input")
            N.check(T.sox_stream_sync(self.stream), "sync")
            X.free()
            self.lengths.write(lengths)

        def layer(self):
            F, W, st, e = self.F, self.W, self.stream, 2 * dim
            qkv.run(self.X.ptr, self.rows, F.ptr, storage, workspace=W.ptr, workspace_bytes=W.cols, stream=st)
            cache.write(self.batch, F.ptr + heads * e, F.ptr + (heads + kv) * e, storage, F.ld, F.ld, rotary=rotary, q=F.ptr, ldq=F.ld,
                        q_heads=heads, y=self.Q.ptr, stream=st)
            cache.attend(self.batch, self.Q.ptr, heads, self.A.ptr, storage, workspace=W.ptr, workspace_bytes=W.cols, stream=st)
            back.run(self.A.ptr, self.rows, self.O.ptr, storage, workspace=W.ptr, workspace_bytes=W.cols, stream=st)
            norm.run(self.X.ptr, self.rows, storage, x=self.O.ptr, h=self.H.ptr, y=self.Z.ptr, stream=st)

        def check(self, lengths):
            N.check(T.sox_stream_sync(self.stream), "sync")
            x = self.X.read().astype(np.float64)
            f, q, a, o, h, z = (m.read().astype(np.float64) for m in self.every)

            def linear(x, w, b, y):
                xq, xs = quantize(x)
                wq, ws = quantize(w.T)
                want, tol = linear64(xq, xs, wq.T, ws.astype(np.float32), b, None, "none", storage)
                assert (np.abs(y - want) <= tol).all()

            linear(x, w1, b1, f)
            parts = f.reshape(self.rows, -1, dim)
            at = 0
            for i, n in enumerate(self.counts):
                r = slice(at, at + n)
                at += n
                pos = np.arange(lengths[i] - n, lengths[i])
                wq, err = turned64(parts[r, :heads], pos, rotary.frequencies, False)
                close(q[r].reshape(wq.shape), wq, 2.0 ** -11 * np.abs(wq) + 2.0 ** -25 + err * 1.001, "turned")
                k = held64(turned64(parts[r, heads:heads + kv], pos, rotary.frequencies, False)[0], storage, "i8")
                held[i] = [np.concatenate([past[:pos[0]], new]) for past, new in zip(held[i], (k, held64(parts[r, heads + kv:], storage, "i8")))]
                want, tol = attend64(q[r].reshape(n, heads, dim), *held[i], pos[0], dim ** -0.5, 0, storage)
                close(a[r].reshape(want.shape), want, tol, "attended")
            linear(a, w2, None, o)
            wh, wy, eh, ey = block64(x, o, None, p, storage)
            inside(h, wh, eh, storage)
            inside(z, wy, ey, storage)

        def free(self):
            for m in self.every + (self.X, self.W, self.starts, self.lengths):
                m.free()

    with Stream() as st:
        lengths = np.array(prompts)
        first = Run(prompts, prompts, st)
        print("[gpu] layer: prompts", flush=True)
        first.feed(910, lengths)
        first.layer()
        first.check(lengths)
        step = Run([1, 1, 1], lengths + 1, st)
        graph = None
        for t in range(5):
            lengths = lengths + 1
            step.feed(920 + t, lengths)
            print(f"[gpu] layer: token {t}", flush=True)
            if graph is None:
                step.layer()
                graph = captured(st, step.layer)
            else:
                N.check(T.sox_graph_launch(graph, st), "replay")
            step.check(lengths)
            got = [m.read() for m in step.every]
            step.layer()  # eager, over the same token again
            N.check(T.sox_stream_sync(st), "sync")
            for m, g in zip(step.every, got):
                assert np.array_equal(m.read(), g), t
        T.sox_graph_destroy(graph)
        first.free()
        step.free()
    for m in (pool, d_tables):
        m.free()
    for o in (qkv, back, norm, cache, rotary):
        o.close()
