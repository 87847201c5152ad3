"""Rotary positions, the paged cache and the attention over it on the GPU, against the operators in 64 bits."""
import ctypes
import math

import numpy as np
import pytest

from layers import SMALL, UNIT, Matrix, rounded
from serving import U32, Ints, Serving, attend64, close, held64, turned64
from simdonnx_amd import native as N
from simdonnx_amd.backend import HipRotary

pytestmark = pytest.mark.gpu


def normal(seed, storage, *shape, by=1.0):
    return rounded(by * np.random.default_rng(seed).standard_normal(shape).astype(np.float32), storage)


def untouched(m, rows):
    """The matrix's rows as they were filled."""
    return np.array_equal(m._view(m.fill.copy())[rows].tobytes(), raw(m)[rows].tobytes())


def raw(m):
    host = np.empty_like(m.fill)
    m._copy(host, up=False)
    return m._view(host).copy()


# ---- rotary positions ----
@pytest.mark.parametrize("storage", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("rows,heads,dim,rotary,interleaved,pad,skip", [
    (1, 1, 8, 2, False, 0, 0), (1, 12, 64, 64, False, 0, 0), (5, 3, 40, 20, False, 3, 1), (5, 3, 40, 20, True, 3, 1),
    (9, 7, 128, 128, False, 0, 0), (9, 7, 128, 64, True, 8, 0), (3, 2, 256, 256, False, 0, 0), (3, 2, 256, 254, True, 0, 3),
    (2100, 2, 72, 36, False, 8, 0), (70, 5, 96, 96, True, 0, 0)])
def test_rotary(hip, storage, rows, heads, dim, rotary, interleaved, pad, skip):
    x = normal(1, storage, rows, heads, dim)
    pos = np.random.default_rng(2).integers(-5, 200000, rows)
    pos[0] = 0
    pos[-1] = 2 ** 31 - 1
    if rows > 2:
        pos[1] = -2 ** 31
    r = HipRotary(hip, dim, rotary_dim=rotary, interleaved=interleaved, base=5e5, factor=8.0, original=4096, amplitude=1.25)
    X, Y = Matrix(x.reshape(rows, -1), storage, ld=heads * dim + pad, skip=skip), Matrix(None, storage, rows, heads * dim, ld=heads * dim + 2 * pad, skip=skip)
    P = Ints(pos)
    print(f"[gpu] rotary {storage} {rows} x {heads} x {dim}, {rotary} {'interleaved' if interleaved else 'halves'}", flush=True)
    r.run(X.ptr, P.ptr, rows, heads, Y.ptr, storage, X.ld, Y.ld)
    # far positions: the 64-bit angle is off by position * frequency * 2^-53 itself, and the device's by position * 2^-65 of a turn
    want, err = turned64(x, pos, r.frequencies, interleaved, 1.25)
    far = np.abs(pos).astype(np.float64)[:, None, None] * 2.0 ** -50 * 1.25 * 2 * np.abs(x).max()
    tol = UNIT[storage] * np.abs(want) + SMALL[storage] + (err if storage != "f32" else 2.0 ** -40 * np.abs(x).max()) * (1 + UNIT[storage]) + far
    close(Y.read().reshape(x.shape), want, tol, "turned")
    r.run(X.ptr, P.ptr, rows, heads, X.ptr, storage, X.ld, X.ld)  # in place
    assert np.array_equal(X.read(), Y.read())
    for m in (X, Y, P):
        m.free()
    r.close()


def test_rotary_given_frequencies(hip):
    """Frequencies one by one: over one turn a position, none, backwards."""
    f = np.array([7.0, 0.0, -0.3, 2 * math.pi])
    r = HipRotary(hip, 16, rotary_dim=8, frequencies=f)
    assert np.array_equal(r.frequencies, f)
    x, pos = normal(3, "f32", 50, 2, 16), np.arange(50) * 41
    X, P = Matrix(x.reshape(50, -1), "f32"), Ints(pos)
    r.run(X.ptr, P.ptr, 50, 2, X.ptr, "f32")
    want, _ = turned64(x, pos, f, False)
    close(X.read().reshape(x.shape), want, U32 * np.abs(want) + 2.0 ** -33 * np.abs(x).max(), "turned")
    for m in (X, P):
        m.free()
    r.close()


# ---- the cache ----
CACHES = [  # sequences (tokens, new), kv heads, head_dim, page
    ([(1, 1)], 1, 8, 1),
    ([(77, 77)], 2, 64, 16),
    ([(5, 5), (0, 0), (130, 3), (64, 1)], 3, 40, 8),
    ([(300, 200), (17, 0), (33, 33)], 2, 128, 64),
    ([(20, 7), (9, 9)], 2, 72, 4),
    ([(40, 40), (41, 1)], 1, 256, 32),
    ([(i % 7 + 1, 1) for i in range(150)], 2, 96, 2),
]


@pytest.mark.parametrize("storage,fmt", [("f16", "f16"), ("bf16", "bf16"), ("f32", "f32"), ("f16", "i8"), ("bf16", "i8"), ("f32", "i8")])
@pytest.mark.parametrize("case", range(len(CACHES)))
@pytest.mark.parametrize("interleaved", [False, True])
def test_write_and_read(hip, case, storage, fmt, interleaved):
    sequences, kv, dim, page = CACHES[case]
    s = Serving(hip, sequences, kv, dim, page, fmt, seed=case, before=2, behind=3)
    rows, heads = s.rows, 2 * kv
    fused = normal(case, storage, rows, (heads + 2 * kv) * dim, by=2.0)
    fused[rows // 2, heads * dim:] = 0  # a row of zeros
    r = HipRotary(hip, dim, rotary_dim=dim // 2, interleaved=interleaved)
    F = Matrix(fused, storage, ld=fused.shape[1] + 5)
    Y, K, V = (Matrix(None, storage, rows, n * dim, ld=n * dim + 8) for n in (heads, kv, kv))
    e = F.elem * dim
    print(f"[gpu] cache {storage} {fmt} {case} {interleaved}", flush=True)
    s.cache.write(s.batch, F.ptr + heads * e, F.ptr + (heads + kv) * e, storage, F.ld, F.ld, rotary=r, q=F.ptr, ldq=F.ld, q_heads=heads, y=Y.ptr, ldy=Y.ld)
    s.cache.read(s.batch, K.ptr, V.ptr, storage, K.ld, V.ld)
    pos = s.positions()
    own = pos >= 0
    parts = fused.reshape(rows, -1, dim)
    q, k, v = parts[:, :heads], parts[:, heads:heads + kv], parts[:, heads + kv:]
    half = UNIT[storage]
    wq, eq = turned64(q, pos, r.frequencies, interleaved)
    tq = half * np.abs(wq) + SMALL[storage] + eq * (1 + half)
    close(Y.read().reshape(q.shape)[own], wq[own], tq[own], "q")
    wk, ek = turned64(k, pos, r.frequencies, interleaved)
    if fmt == "i8":
        # k is turned in 64 bits and rounded once to fp32: the whole numbers are the definition's
        wk, wv = held64(wk, storage, fmt), held64(v, storage, fmt)
        tk, tv = ((half + U32) * np.abs(w) + SMALL[storage] for w in (wk, wv))
    else:
        wv, tk, tv = v, half * np.abs(wk) + SMALL[storage] + ek * (1 + half), 0.0
    close(K.read().reshape(k.shape)[own], wk[own], np.broadcast_to(tk, wk.shape)[own], "k")
    close(V.read().reshape(v.shape)[own], wv[own], np.broadcast_to(tv, wv.shape)[own], "v")
    for m in (Y, K, V):
        assert untouched(m, ~own)
    s.pool.read()
    for m in (F, Y, K, V):
        m.free()
    r.close()
    s.free()


@pytest.mark.parametrize("fmt", ["f16", "i8"])
def test_pages_that_are_not_there(hip, fmt):
    """Table entries outside of the pool, a table that ends early, and more rows than tokens: nothing is written, the
    tokens read as zeros and are not attended to, rows before the first token stay as they are."""
    kv, dim, page, storage = 2, 64, 16, "f16"
    s = Serving(hip, [(60, 60), (40, 40), (10, 10)], kv, dim, page, fmt)
    tables = s.tables.copy()
    tables[0, 1], tables[1, 0] = -7, s.pages
    s.d_tables.write(tables)
    s.d_lengths.write([60, 100, 4])  # (sequence 1's tokens 60 .. 99: table_pages * page = 80 of them are held at most)
    k, v, q = (normal(i, storage, s.rows, n, dim) for i, n in ((1, kv), (2, kv), (3, 2 * kv)))
    K, V, Q = (Matrix(x.reshape(s.rows, -1), storage) for x in (k, v, q))
    K2, V2, Y = (Matrix(None, storage, s.rows, n * dim) for n in (kv, kv, 2 * kv))
    W = Matrix(None, "i8", 1, s.cache.workspace(s.rows, 3, 2 * kv))
    print(f"[gpu] pages that are not there {fmt}", flush=True)
    s.cache.write(s.batch, K.ptr, V.ptr, storage)
    s.cache.read(s.batch, K2.ptr, V2.ptr, storage)
    s.cache.attend(s.batch, Q.ptr, 2 * kv, Y.ptr, storage, workspace=W.ptr, workspace_bytes=W.cols)
    gk, gv, gy = (m.read().reshape(x.shape) for m, x in ((K2, k), (V2, v), (Y, q)))
    hk, hv = held64(k, storage, fmt), held64(v, storage, fmt)
    where = np.concatenate([np.arange(60), np.arange(60, 100), np.arange(-6, 4)])
    held = np.ones(s.rows, bool)
    held[16:32] = False                              # page 1 of sequence 0
    held[60:100] = (where[60:100] >= 64) & (where[60:100] < 64)  # sequence 1: its table ends at 5 pages, -1 behind its own 3
    held[100:] = True
    left = where < 0
    for got, want in ((gk, hk), (gv, hv)):
        close(got[held & ~left], want[held & ~left], (UNIT[storage] + U32) * np.abs(want[held & ~left]) + SMALL[storage], "held")
        assert (got[~held & ~left] == 0).all()
    for m in (K2, V2, Y):
        assert untouched(m, left)
    # sequence 0 without tokens 16 .. 31
    absent = np.zeros(60, bool)
    absent[16:32] = True
    want, tol = attend64(q[:60].astype(np.float64), hk[:60], hv[:60], 0, dim ** -0.5, 0, storage, absent)
    close(gy[:60], want, tol, "y")
    assert np.isnan(gy[60:100]).all()                # sequence 1 sees its pages 1 and 2, which nothing has written since the fill
    want, tol = attend64(q[106:].astype(np.float64), hk[106:], hv[106:], 0, dim ** -0.5, 0, storage)
    close(gy[106:], want, tol, "y")
    s.pool.read()
    for m in (K, V, Q, K2, V2, Y, W):
        m.free()
    s.free()


def test_no_page_at_all(hip):
    """A table of none: zeros, in the single-token kernel and over pieces."""
    for new in (1, 50):
        s = Serving(hip, [(60, new)], 2, 64, 16, "bf16")
        s.d_tables.write(np.full_like(s.tables, -1))
        Q, Y = Matrix(normal(1, "bf16", new, 256), "bf16"), Matrix(None, "bf16", new, 256)
        W = Matrix(None, "i8", 1, s.cache.workspace(new, 1, 4))
        s.cache.attend(s.batch, Q.ptr, 4, Y.ptr, "bf16", workspace=W.ptr, workspace_bytes=W.cols)
        assert (Y.read() == 0).all()
        for m in (Q, Y, W):
            m.free()
        s.free()


# ---- attention ----
ATTENDS = [  # sequences (tokens, new), kv heads, query heads of each, head_dim, page, window
    ([(1, 1)], 1, 1, 8, 1, 0),
    ([(77, 1)], 3, 1, 64, 16, 0),
    ([(2000, 1)], 2, 4, 128, 16, 0),
    ([(1500, 1)], 1, 5, 80, 4, 0),
    ([(700, 1)], 1, 16, 256, 64, 0),
    ([(300, 1), (1, 1), (0, 0), (64, 1), (65, 1), (513, 1)], 2, 3, 72, 8, 0),
    ([(40, 40)], 2, 1, 64, 16, 0),
    ([(129, 129)], 1, 2, 128, 32, 0),
    ([(200, 70)], 2, 3, 40, 8, 0),
    ([(100, 100)], 1, 1, 256, 16, 0),
    ([(70, 5)], 1, 20, 128, 16, 0),
    ([(600, 3), (300, 90), (17, 17), (5, 0), (33, 1)], 2, 2, 96, 16, 0),
    ([(400, 1), (90, 90)], 1, 4, 128, 16, 33),
    ([(500, 150)], 2, 1, 64, 16, 64),
    ([(300, 40)], 1, 7, 128, 2, 1),
    ([(3000, 20)], 1, 1, 64, 128, 0),
    ([(900, 2), (901, 2), (1024, 2)], 1, 8, 128, 16, 100),
]


def attend_case(hip, case, storage, fmt, pad=0, by=1.5):
    sequences, kv, group, dim, page, window = case
    heads = kv * group
    s = Serving(hip, sequences, kv, dim, page, fmt, seed=7, before=1, behind=2)
    total = int(s.whole[-1])
    k, v = normal(11, storage, total, kv, dim), normal(12, storage, total, kv, dim)
    q = normal(13, storage, s.rows, heads, dim, by=by)
    K, V = Matrix(k.reshape(total, -1), storage), Matrix(v.reshape(total, -1), storage)
    Q, Y = Matrix(q.reshape(s.rows, -1), storage, ld=heads * dim + pad), Matrix(None, storage, s.rows, heads * dim, ld=heads * dim + pad)
    W = Matrix(None, "i8", 1, s.cache.workspace(s.rows, len(sequences), heads))
    s.cache.write(s.every, K.ptr, V.ptr, storage)
    return s, k, v, q, K, V, Q, Y, W


def expect(s, q, hk, hv, case, storage, scale=None):
    sequences, kv, group, dim, page, window = case
    want, tol = np.zeros(q.shape), np.zeros(q.shape)
    for i, (length, new) in enumerate(sequences):
        a, b = s.whole[i], s.whole[i + 1]
        r = slice(s.starts[i], s.starts[i + 1])
        want[r], tol[r] = attend64(q[r].astype(np.float64), hk[a:b], hv[a:b], length - new, scale or dim ** -0.5, window, storage)
    return want, tol


@pytest.mark.parametrize("storage,fmt", [("f16", "f16"), ("bf16", "bf16"), ("f32", "f32"), ("f16", "i8"), ("bf16", "i8"), ("f32", "i8")])
@pytest.mark.parametrize("case", range(len(ATTENDS)))
def test_attend(hip, case, storage, fmt):
    c = ATTENDS[case]
    s, k, v, q, K, V, Q, Y, W = attend_case(hip, c, storage, fmt, pad=5 if case % 2 else 0)
    print(f"[gpu] attend {storage} {fmt} {case}", flush=True)
    s.cache.attend(s.batch, Q.ptr, c[1] * c[2], Y.ptr, storage, Q.ld, Y.ld, window=c[5], workspace=W.ptr, workspace_bytes=W.cols)
    want, tol = expect(s, q, held64(k, storage, fmt), held64(v, storage, fmt), c, storage)
    got = Y.read().reshape(q.shape)
    own = s.positions() >= 0
    close(got[own], want[own], tol[own], "y")
    assert untouched(Y, ~own)
    W.read()  # (nothing behind the workspace)
    for m in (K, V, Q, Y, W):
        m.free()
    s.free()


@pytest.mark.parametrize("storage", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("case", [([(90, 40)], 1, 2, 72, 16, 0), ([(150, 150)], 1, 1, 128, 8, 20), ([(70, 3), (33, 2)], 2, 4, 64, 16, 9)])
def test_values_that_are_not_finite(hip, case, storage):
    """NaN and infinities in K and V reach the rows that see their token and no other, in tiles seen in part too."""
    sequences, kv, group, dim, page, window = case
    heads = kv * group
    s, k, v, q, K, V, Q, Y, W = attend_case(hip, case, storage, storage)
    length, new = sequences[0]
    last = length - 1
    spots = [(last, np.nan, 3), (last, np.inf, 5), (last - new // 2, -np.inf, 5), (last - new // 2, np.inf, dim - 1), (last - 1, np.nan, dim - 1)]
    for t, x, c in spots:
        v[t, 0, c] = x
    k[last - new // 3, 0, 1] = np.nan  # (a row that sees it is NaN throughout)
    if len(sequences) > 1:
        k[-1, 1, 0], v[-1, 0, 2] = np.inf, np.inf
    for m, x in ((K, k), (V, v)):
        m.free()
    K, V = Matrix(k.reshape(k.shape[0], -1), storage), Matrix(v.reshape(v.shape[0], -1), storage)
    s.cache.write(s.every, K.ptr, V.ptr, storage)
    print(f"[gpu] not finite {storage} {case}", flush=True)
    s.cache.attend(s.batch, Q.ptr, heads, Y.ptr, storage, window=window, workspace=W.ptr, workspace_bytes=W.cols)
    got = Y.read().reshape(q.shape)
    # a row that sees such a token: NaN where K is NaN or its score infinite, else as its V's channels say; others as ever
    clean_k, clean_v = np.where(np.isfinite(k), k, 0), np.where(np.isfinite(v), v, 0)
    for i, (length, new) in enumerate(sequences):
        a, r0 = int(s.whole[i]), int(s.starts[i])
        for j in range(new):
            pos = length - new + j
            lo = max(0, pos - window + 1) if window else 0
            for g in range(kv):
                kk, vv = k[a + lo:a + pos + 1, g], v[a + lo:a + pos + 1, g]
                row = slice(g * group, (g + 1) * group)
                mine = got[r0 + j, row]
                if np.isnan(kk).any():
                    assert np.isnan(mine).all()
                    continue
                with np.errstate(invalid="ignore"):
                    scores = q[r0 + j, row].astype(np.float64) @ kk.T.astype(np.float64)
                up = (scores == np.inf).any(axis=1)
                assert np.isnan(mine[up]).all()
                down = np.where(np.isinf(kk).any(axis=1))[0]
                want, tol = attend64(q[r0 + j:r0 + j + 1].astype(np.float64), clean_k[a:a + length], clean_v[a:a + length], pos, dim ** -0.5, window, storage,
                                     np.isin(np.arange(length), lo + down))
                special = np.where(np.isfinite(vv), 0, vv)
                special[down] = 0  # (their weight is exp(-inf) = 0: left to the formula's 0 * v, finite here)
                with np.errstate(invalid="ignore"):
                    add = special.sum(axis=0)
                w, t = want[0, row] + add, tol[0, row]
                close(mine[~up], w[~up], t[~up], "y")
    for m in (K, V, Q, Y, W):
        m.free()
    s.free()


def test_infinite_v_in_8_bits(hip):
    """A head of v that is not finite is held as NaN, for the rows that see its token alone."""
    case = ([(90, 40)], 1, 2, 72, 16, 0)
    s, k, v, q, K, V, Q, Y, W = attend_case(hip, case, "f16", "i8")
    v[75, 0, 3] = np.inf
    V.free()
    V = Matrix(v.reshape(90, -1), "f16")
    s.cache.write(s.every, K.ptr, V.ptr, "f16")
    s.cache.attend(s.batch, Q.ptr, 2, Y.ptr, "f16", workspace=W.ptr, workspace_bytes=W.cols)
    got = Y.read().reshape(q.shape)[1:41]
    assert np.isnan(got[25:]).all()
    want, tol = attend64(q[1:41].astype(np.float64), held64(k, "f16", "i8"), held64(np.where(np.isfinite(v), v, 0), "f16", "i8"), 50, 72 ** -0.5, 0, "f16")
    close(got[:25], want[:25], tol[:25], "y")
    for m in (K, V, Q, Y, W):
        m.free()
    s.free()


@pytest.mark.parametrize("fmt", ["bf16", "i8"])
def test_scales_far_apart(hip, fmt):
    """Values of v from 2^-80 to 2^100 and rows of zeros, scores of some hundred: no overflow, and the small ones exact where
    they are all that counts."""
    storage, n, dim = "bf16", 200, 64
    case = ([(n, n)], 1, 1, dim, 16, 0)
    s, k, v, q, K, V, Q, Y, W = attend_case(hip, case, storage, fmt, by=40.0)
    v *= np.exp2(np.random.default_rng(5).integers(-80, 100, (n, 1, 1))).astype(np.float32)
    v[0], v[7], v[50:60] = v[0] * 2.0 ** -40, 0, 0
    k[8] = 0
    for m in (K, V):
        m.free()
    K, V = Matrix(k.reshape(n, -1), storage), Matrix(v.reshape(n, -1), storage)
    s.cache.write(s.every, K.ptr, V.ptr, storage)
    s.cache.attend(s.batch, Q.ptr, 1, Y.ptr, storage, workspace=W.ptr, workspace_bytes=W.cols)
    own = s.positions() >= 0
    want, tol = expect(s, q, held64(k, storage, fmt), held64(v, storage, fmt), case, storage)
    close(Y.read().reshape(q.shape)[own], want[own], tol[own], "y")
    for m in (K, V, Q, Y, W):
        m.free()
    s.free()


@pytest.mark.parametrize("fmt", ["f16", "i8"])
def test_pool_past_4_gib(hip, fmt):
    """Pages on both sides of 2^32 bytes."""
    storage, kv, dim, page = "f16", 8, 128, 16
    s = Serving(hip, [(40, 40), (300, 1)], kv, dim, page, fmt)
    pages = (5 << 30) // s.cache.page_bytes
    p = ctypes.c_void_p()
    N.check(N.thin().sox_malloc(ctypes.byref(p), pages * s.cache.page_bytes), "pool")
    tables = np.where(s.tables >= 0, pages - 1 - s.tables * (pages // s.pages // 2), -1)
    first, last = int(tables[tables >= 0].min()), int(tables.max())
    assert last * s.cache.page_bytes > 2 ** 32 > first * s.cache.page_bytes
    s.d_tables.write(tables)
    for b in (s.batch, s.every):
        b.p.pool, b.p.pages = p.value, pages
    k, v, q = normal(1, storage, 340, kv, dim), normal(2, storage, 340, kv, dim), normal(3, storage, s.rows, 2 * kv, dim)
    K, V, Q = (Matrix(x.reshape(x.shape[0], -1), storage) for x in (k, v, q))
    K2, V2, Y = Matrix(None, storage, 340, kv * dim), Matrix(None, storage, 340, kv * dim), Matrix(None, storage, s.rows, 2 * kv * dim)
    W = Matrix(None, "i8", 1, s.cache.workspace(s.rows, 2, 2 * kv))
    print(f"[gpu] 5 GiB pool {fmt}", flush=True)
    s.cache.write(s.every, K.ptr, V.ptr, storage)
    s.cache.read(s.every, K2.ptr, V2.ptr, storage)
    s.cache.attend(s.batch, Q.ptr, 2 * kv, Y.ptr, storage, workspace=W.ptr, workspace_bytes=W.cols)
    hk, hv = held64(k, storage, fmt), held64(v, storage, fmt)
    for m, want in ((K2, hk), (V2, hv)):
        close(m.read().reshape(want.shape), want, (UNIT[storage] + U32) * np.abs(want) + SMALL[storage], "read")
    want, tol = expect(s, q, hk, hv, ([(40, 40), (300, 1)], kv, 2, dim, page, 0), storage)
    close(Y.read().reshape(q.shape), want, tol, "y")
    for m in (K, V, Q, K2, V2, Y, W):
        m.free()
    N.thin().sox_free(p)
    s.free()


def test_scale_given(hip):
    case = ([(50, 20)], 1, 2, 64, 16, 0)
    s, k, v, q, K, V, Q, Y, W = attend_case(hip, case, "f32", "f32")
    s.cache.attend(s.batch, Q.ptr, 2, Y.ptr, "f32", scale=0.7, workspace=W.ptr, workspace_bytes=W.cols)
    own = s.positions() >= 0
    want, tol = expect(s, q, k.astype(np.float64), v.astype(np.float64), case, "f32", scale=float(np.float32(0.7)))
    close(Y.read().reshape(q.shape)[own], want[own], tol[own], "y")
    for m in (K, V, Q, Y, W):
        m.free()
    s.free()
