"""The paged cache and its attention at the ends of what a call may hold: positions next to 2^31, scores of 2^30, weights and scales far
apart, rows by the thousand, on the GPU against the operators in 64 bits."""
import numpy as np
import pytest

import serving
import test_gpu_kv_cache as kv_cache
from layers import SMALL, UNIT, Matrix, rounded
from serving import U32, Ints, Serving, attend64, close, held64, turned64
from simdonnx_amd.backend import HipRotary
from test_gpu_kv_cache import normal, untouched

pytestmark = pytest.mark.gpu
FORMATS = [("f16", "f16"), ("bf16", "bf16"), ("f32", "f32"), ("f16", "i8"), ("bf16", "i8"), ("f32", "i8")]
ROOM = 1 << 19  # tokens that tables have room for where every piece is to go to the kernel over 128 pairs


def attended(s, k, v, q, storage, scale=0.0, window=0, written=None):
    """The attention of q [rows, heads, dim] over k and v [tokens, kv, dim], written from another storage type where one is named."""
    written = written or storage
    K, V = Matrix(k.reshape(k.shape[0], -1), written), Matrix(v.reshape(v.shape[0], -1), written)
    Q, Y = Matrix(q.reshape(q.shape[0], -1), storage), Matrix(None, storage, q.shape[0], q.shape[1] * q.shape[2])
    W = Matrix(None, "i8", 1, s.cache.workspace(s.rows, len(s.sequences), q.shape[1]))
    s.cache.write(s.every, K.ptr, V.ptr, written)
    s.cache.attend(s.batch, Q.ptr, q.shape[1], Y.ptr, storage, scale=scale, window=window, workspace=W.ptr, workspace_bytes=W.cols)
    y = Y.read().reshape(q.shape)
    for m in (K, V, Q, Y, W):
        m.free()
    return y


# ---- the longest sequences ----
@pytest.mark.parametrize("storage,fmt", FORMATS)
def test_window_behind_the_table(hip, monkeypatch, storage, fmt):
    """Sequences of 2^31 - 1 tokens whose window lies behind what their tables hold, split nine ways (the last split's first
    token would be 2^31): zeros, whatever the workspace held; the other sequences as ever. Then a piece of 50 rows likewise."""
    monkeypatch.setattr(serving, "TABLE_TOKENS", 4096)
    dim, window = 64, 1023
    lengths = [(10, 1)] + [(20, 4)] * 39
    s = Serving(hip, lengths, 1, dim, 16, fmt)
    s.d_lengths.write([2 ** 31 - 1] + [20] * 39)
    total = int(s.whole[-1])
    k, v, q = normal(1, storage, total, 1, dim), normal(2, storage, total, 1, dim), normal(3, storage, s.rows, 1, dim)
    K, V, Q = (Matrix(x.reshape(x.shape[0], -1), storage) for x in (k, v, q))
    size = s.cache.workspace(s.rows, len(lengths), 1)
    Y, W = Matrix(None, storage, s.rows, dim), Matrix(np.full((1, size // 4), 7.0, np.float32), "f32")
    s.d_lengths.write([10] + [20] * 39)
    s.cache.write(s.every, K.ptr, V.ptr, storage)
    s.d_lengths.write([2 ** 31 - 1] + [20] * 39)
    print(f"[gpu] window behind the table {storage} {fmt}", flush=True)
    s.cache.attend(s.batch, Q.ptr, 1, Y.ptr, storage, window=window, workspace=W.ptr, workspace_bytes=size)
    y = Y.read().reshape(q.shape)
    assert (y[0] == 0).all()
    hk, hv = held64(k, storage, fmt), held64(v, storage, fmt)
    for i in range(1, 40):
        a, r = s.whole[i], slice(s.starts[i], s.starts[i + 1])
        want, tol = attend64(q[r].astype(np.float64), hk[a:a + 20], hv[a:a + 20], 16, dim ** -0.5, window, storage)
        close(y[r], want, tol, f"sequence {i}")
    W.read()
    for m in (K, V, Q, Y, W):
        m.free()
    s.free()
    for window in (255, 1023, 4095, 2 ** 31 - 1):  # (the last: all that the table holds, and nothing is in a page there)
        s = Serving(hip, [(60, 50)], 1, dim, 16, fmt)
        s.d_lengths.write([2 ** 31 - 1])
        s.d_tables.write(np.full_like(s.tables, -1))
        Q, Y = Matrix(normal(4, storage, 50, 4 * dim), storage), Matrix(None, storage, 50, 4 * dim)
        size = s.cache.workspace(50, 1, 4)
        W = Matrix(np.full((1, size // 4), 7.0, np.float32), "f32")
        s.cache.attend(s.batch, Q.ptr, 4, Y.ptr, storage, window=window, workspace=W.ptr, workspace_bytes=size)
        assert (Y.read() == 0).all()
        W.read()
        for m in (Q, Y, W):
            m.free()
        s.free()


# ---- scores ----
@pytest.mark.parametrize("storage,fmt", FORMATS)
@pytest.mark.parametrize("new,room", [(1, 0), (40, 0), (40, ROOM)])
@pytest.mark.parametrize("power", [10, 16, 24])
def test_large_scores(hip, monkeypatch, storage, fmt, new, room, power):
    """Scores so large that a step of fp32 is more than the softmax's range (2^30 with power 16): each row is the value of the token
    with the largest. Half a step of the storage type for its weight's product with v, half for the output, and a unit of fp32
    each for the product, the sum, the quotient and the last product."""
    power = min(power, 17) if storage == "f16" else power
    monkeypatch.setattr(serving, "TABLE_TOKENS", room)
    n, dim, heads = 300, 64, 6
    rng = np.random.default_rng(power)
    s = Serving(hip, [(n, new)], 2, dim, 16, fmt)
    k, q, by = np.zeros((n, 2, dim), np.float32), np.zeros((new, heads, dim), np.float32), 2.0 ** (power - 8)
    # (whole numbers of 7 bits, so that every form of the cache holds them as they are; token 0's leads by a sixth)
    k[:, :, 5] = np.stack([rng.permutation(n) % 100 for _ in range(2)], 1) * by
    k[0, :, 5] = rng.integers(120, 127, 2) * by
    k[:, :, 9] = 127 * by  # every head's amax in 8 bits, where q holds zeros
    q[..., 5] = rng.integers(100, 127, (new, heads)) * by
    assert np.array_equal(rounded(k, storage), k) and np.array_equal(rounded(q, storage), q)
    v = normal(3, storage, n, 2, dim)
    print(f"[gpu] large scores {storage} {fmt} {new} {room} {power}", flush=True)
    y = attended(s, k, v, q, storage, scale=0.7)
    want = np.repeat(held64(v, storage, fmt)[0], heads // 2, axis=0)
    close(y, np.broadcast_to(want, y.shape), (2 * UNIT[storage] + 4 * U32) * np.abs(want) + SMALL[storage], "y")
    s.free()


# ---- weights and scales far apart in fp16 ----
@pytest.mark.parametrize("fmt", ["f16", "i8"])
@pytest.mark.parametrize("new,room", [(1, 0), (40, 0), (40, ROOM)])
@pytest.mark.parametrize("power", [20.7, 26.3])
def test_small_weights_in_fp16(hip, monkeypatch, fmt, new, room, power):
    """One token in 32 of weight 1, the others' 2^-20.7 or 2^-26.3, which fp16 alone would hold in 3 bits or not at all: their
    values stand in the channels where the first ones hold zeros. The tolerance is attend64's, but for the part of weights below
    fp16's normal numbers: the largest weights stand at 2^7 there (half of it at least where v's scale takes its part), so
    a token is off by half of 2^-24 of 2^-6 of its value at most, and the sum is their number at least."""
    monkeypatch.setattr(serving, "TABLE_TOKENS", room)
    n, dim = 4096, 64
    s = Serving(hip, [(n, new)], 1, dim, 16, fmt)
    k, v, q = np.zeros((n, 1, dim), np.float32), np.zeros((n, 1, dim), np.float32), np.zeros((new, 2, dim), np.float32)
    v[..., 1:] = np.random.default_rng(5).uniform(30000, 60000, (n, 1, dim - 1))
    k[::32, 0, 0], v[::32] = power * np.log(2.0), 0
    v[::32, 0, 0] = 1
    q[..., 0] = 8  # (scale 1 / 8: the score is k's first value)
    k, v = rounded(k, "f16"), rounded(v, "f16")
    print(f"[gpu] small weights {fmt} {new} {room} {power}", flush=True)
    y = attended(s, k, v, q, "f16")
    hk, hv = held64(k, "f16", fmt), held64(v, "f16", fmt)
    want, tol = attend64(q.astype(np.float64), hk, hv, n - new, dim ** -0.5, 0, "f16")
    seen = np.arange(n - new + 1, n + 1)[:, None, None]
    tol -= seen * 2.0 ** -25 * np.abs(hv).max(axis=0) * (1 - 2.0 ** -6 / (seen // 32))
    assert (tol[..., 1:] < 0.07 * want[..., 1:]).all()  # (2^-31 / 2^-26.3 / 0.75, and the rest)
    close(y, want, tol, "y")
    s.free()


@pytest.mark.parametrize("written,large,small", [("f16", 1000, 1e-3), ("f16", 60000, 1e-2), ("f16", 60000, 1e-3), ("f16", 1, 3e-5), ("f16", 2e-6, 6e-8),
                                                 ("f32", 1.5e5, 0.1), ("f32", 1.0, 1e-12), ("bf16", 1e-20, 1e-30)])
@pytest.mark.parametrize("new,room", [(1, 0), (40, 0), (40, ROOM)])
@pytest.mark.parametrize("by", [0.0, 1.5])
def test_scales_far_apart_in_fp16(hip, monkeypatch, written, large, small, new, room, by):
    """fp16 rows over 8 bits, where some tokens' values of v are far larger than the others' in one channel and zero in the rest:
    there the others count, to their last bits."""
    monkeypatch.setattr(serving, "TABLE_TOKENS", room)
    n, kv, dim, heads = 200, 2, 72, 4
    s = Serving(hip, [(n, new)], kv, dim, 8, "i8")
    k, v, q = normal(1, written, n, kv, dim), normal(2, written, n, kv, dim, by=small), normal(3, "f16", new, heads, dim, by=by)
    for token in (0, 90, 159):
        v[token], v[token, :, 3] = 0, large
    v = rounded(v, written)
    print(f"[gpu] scales far apart {written} {large} {small} {new} {room} {by}", flush=True)
    y = attended(s, k, v, q, "f16", written=written)
    want, tol = attend64(q.astype(np.float64), held64(k, written, "i8"), held64(v, written, "i8"), n - new, dim ** -0.5, 0, "f16")
    close(y, want, tol, "y")
    s.free()


@pytest.mark.parametrize("new,room", [(1, 0), (40, 0), (40, ROOM)])
def test_rows_of_zeros_in_fp16(hip, monkeypatch, new, room):
    """One token of large values and 4095 of zeros, in 8 bits: their weights of 2^-18 take the sum up by 2^-6."""
    monkeypatch.setattr(serving, "TABLE_TOKENS", room)
    n, dim = 4096, 64
    s = Serving(hip, [(n, new)], 1, dim, 16, "i8")
    k, v, q = np.zeros((n, 1, dim), np.float32), np.zeros((n, 1, dim), np.float32), np.zeros((new, 2, dim), np.float32)
    k[0, 0, 0], v[0] = 18 * np.log(2.0), 30000 * (1 + np.arange(dim) / dim)
    q[..., 0] = 8
    k, v = rounded(k, "f16"), rounded(v, "f16")
    print(f"[gpu] rows of zeros {new} {room}", flush=True)
    y = attended(s, k, v, q, "f16")
    hk, hv = held64(k, "f16", "i8"), held64(v, "f16", "i8")
    want, tol = attend64(q.astype(np.float64), hk, hv, n - new, dim ** -0.5, 0, "f16")
    tol -= np.arange(n - new + 1, n + 1)[:, None, None] * 2.0 ** -25 * np.abs(hv).max(axis=0) * (1 - 2.0 ** -6)  # (as above)
    assert (want < 0.99 * hv[0]).all() and (tol < 0.004 * want).all()
    close(y, want, tol, "y")
    s.free()


# ---- far positions ----
def turns_of(positions, frequencies):
    """[positions, frequencies]: position * frequency as a fraction of a turn, from whole numbers: pi to 1400 bits by Machin's
    formula, 16 arctan(1 / 5) - 4 arctan(1 / 239)."""
    bits = 1400

    def arctan_inverse(n):
        total, term, i = 0, (1 << bits) // n, 0
        while term:
            total += (-term if i & 1 else term) // (2 * i + 1)
            term //= n * n
            i += 1
        return total

    turn = 2 * (16 * arctan_inverse(5) - 4 * arctan_inverse(239))
    out = np.empty((len(positions), len(frequencies)))
    for i, p in enumerate(positions):
        for j, f in enumerate(frequencies):
            a, b = float(f).as_integer_ratio()
            out[i, j] = ((int(p) * a << bits) // b) % turn / turn
    return out


@pytest.mark.parametrize("scale", [1e-6, 1.0, 3e3, 1e6, 1e9, 1e12])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_far_and_fast(hip, scale, interleaved):
    """Positions up to both ends of 32 bits with frequencies of many turns a position: angles are off by 2^-33 of a turn at most."""
    rows, heads, dim = 64, 3, 32
    rng = np.random.default_rng(int(np.log10(scale)) + 50)
    f = scale * rng.uniform(0.5, 2.0, dim // 2) * rng.choice([-1, 1], dim // 2)
    pos = np.concatenate([[0, 1, -1, 2 ** 31 - 1, -2 ** 31, 2 ** 30], rng.integers(-2 ** 31, 2 ** 31, rows - 6)])
    x = normal(8, "f32", rows, heads, dim)
    r = HipRotary(hip, dim, interleaved=interleaved, frequencies=f)
    X, P = Matrix(x.reshape(rows, -1), "f32"), Ints(pos)
    print(f"[gpu] rotary far {scale} {interleaved}", flush=True)
    r.run(X.ptr, P.ptr, rows, heads, X.ptr, "f32")
    angle = 2 * np.pi * turns_of(pos, f)[:, None]
    i, j = (slice(0, dim, 2), slice(1, dim, 2)) if interleaved else (slice(0, dim // 2), slice(dim // 2, dim))
    a, b, want = x[..., i].astype(np.float64), x[..., j].astype(np.float64), np.empty(x.shape)
    want[..., i], want[..., j] = a * np.cos(angle) - b * np.sin(angle), b * np.cos(angle) + a * np.sin(angle)
    # (cos, sin, products and sums in 64 bits here and there: a hundred units are plenty)
    tol = U32 * np.abs(want) + (2 * np.pi * 2.0 ** -33 + 100 * 2.0 ** -53) * 2 * np.abs(x).max()
    close(X.read().reshape(x.shape), want, tol, "turned")
    for m in (X, P):
        m.free()
    r.close()


# ---- rows by the thousand: four to a workgroup ----
@pytest.mark.parametrize("storage,fmt", FORMATS)
@pytest.mark.parametrize("kv,dim,page", [(3, 40, 8), (2, 128, 64), (1, 8, 1)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_write_and_read_many(hip, monkeypatch, kv, dim, page, storage, fmt, interleaved):
    """2062 rows with two ahead of the sequences and three behind, borders between sequences within a workgroup's rows."""
    monkeypatch.setattr(kv_cache, "CACHES", [([(1500, 1301), (5, 5), (0, 0), (900, 751)], kv, dim, page)])
    kv_cache.test_write_and_read(hip, 0, storage, fmt, interleaved)


@pytest.mark.parametrize("room", [0, ROOM])
@pytest.mark.parametrize("storage", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("case", [([(90, 40)], 1, 2, 256, 16, 0), ([(170, 150)], 1, 1, 200, 8, 20)])
def test_wide_heads_that_are_not_finite(hip, monkeypatch, case, storage, room):
    monkeypatch.setattr(serving, "TABLE_TOKENS", room)
    kv_cache.test_values_that_are_not_finite(hip, case, storage)


@pytest.mark.parametrize("room", [0, ROOM])
@pytest.mark.parametrize("storage", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("dim", [72, 128, 256])
def test_heads_that_are_not_finite_in_8_bits(hip, monkeypatch, dim, storage, room):
    """Heads of k and v with an infinity or a NaN, in tiles that some rows see in part: NaN for the rows that see their token."""
    monkeypatch.setattr(serving, "TABLE_TOKENS", room)
    n, new = 140, 90
    s = Serving(hip, [(n, new)], 1, dim, 16, "i8")
    k, v, q = normal(1, storage, n, 1, dim), normal(2, storage, n, 1, dim), normal(3, storage, new, 2, dim)
    clean = held64(k, storage, "i8"), held64(v, storage, "i8")
    k[131, 0, 5], v[118, 0, 7], v[130, 0, 0] = np.nan, np.inf, -np.inf
    print(f"[gpu] not finite in 8 bits {storage} {dim} {room}", flush=True)
    y = attended(s, k, v, q, storage)
    first = 118 - (n - new)
    assert np.isnan(y[first:]).all()
    want, tol = attend64(q[:first].astype(np.float64), *clean, n - new, dim ** -0.5, 0, storage)
    close(y[:first], want, tol, "y")
    s.free()


# ---- weights of few rows over 8 bits ----
@pytest.mark.parametrize("storage", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("sequences,kv,group,dim", [([(5, 1)], 2, 4, 128), ([(300, 1), (40, 2)], 1, 5, 72), ([(3000, 1)], 2, 2, 64), ([(77, 3)], 1, 4, 256)])
def test_weights_of_few_rows(hip, sequences, kv, group, dim, storage):
    """Up to 16 pairs a sequence: weights with their scales meet v in two parts, so what 16 bits leave of them is the square of their
    half step, and an output is off by little more than its own rounding. (The rest of the tolerance is attend64's; fp16's as in
    test_small_weights_in_fp16.)"""
    s = Serving(hip, sequences, kv, dim, 16, "i8")
    total, heads = int(s.whole[-1]), kv * group
    k, v, q = normal(1, storage, total, kv, dim), normal(2, storage, total, kv, dim), normal(3, storage, s.rows, heads, dim, by=1.5)
    print(f"[gpu] weights of few rows {sequences} {dim} {storage}", flush=True)
    y = attended(s, k, v, q, storage)
    hk, hv, half = held64(k, storage, "i8"), held64(v, storage, "i8"), UNIT[storage]
    for i, (length, new) in enumerate(sequences):
        a, r = s.whole[i], slice(s.starts[i], s.starts[i + 1])
        kk, vv, qq = hk[a:a + length], hv[a:a + length], q[r].astype(np.float64)
        want, _ = attend64(qq, kk, vv, length - new, dim ** -0.5, 0, storage)
        tol = np.empty(want.shape)
        for j in range(new):
            for h in range(heads):
                g, n = h // group, length - new + j + 1
                p = np.exp(dim ** -0.5 * (kk[:n, g] @ qq[j, h]))
                size = p @ np.abs(vv[:n, g]) / p.sum()
                e = (dim + 6) * U32 * dim ** -0.5 * (np.abs(kk[:n, g]) @ np.abs(qq[j, h])).max()
                tiny = n * (2.0 ** -31 if storage == "f16" else 2.0 ** -126) * np.abs(vv[:n, g]).max(axis=0)
                left = 0.0 if storage == "f32" else half * half
                tol[j, h] = (left + 4 * e + (2 * n + 16) * U32) * size + tiny + half * np.abs(want[j, h]) * 1.001 + SMALL[storage]
        close(y[r], want, tol, f"sequence {i}")
    s.free()


@pytest.mark.parametrize("storage,fmt", FORMATS)
@pytest.mark.parametrize("new,room", [(1, 0), (3, 0), (40, ROOM)])
def test_infinite_values_seen_whole(hip, monkeypatch, storage, fmt, new, room):
    """Infinities and NaN of v in tiles that every row sees whole: they reach their channels and no other (in 8 bits, which hold
    such a head as NaN, all of its head's)."""
    monkeypatch.setattr(serving, "TABLE_TOKENS", room)
    n, kv, dim = 600, 2, 72
    s = Serving(hip, [(n, new)], kv, dim, 16, fmt)
    k, v, q = normal(1, storage, n, kv, dim), normal(2, storage, n, kv, dim), normal(3, storage, new, 2 * kv, dim)
    want, tol = attend64(q.astype(np.float64), held64(k, storage, fmt), held64(v, storage, fmt), n - new, dim ** -0.5, 0, storage)
    v[5, 0, 3], v[37, 0, 4], v[38, 0, 5], v[70, 0, 5], v[200, 0, 71] = np.inf, -np.inf, np.inf, -np.inf, np.nan
    want[:, :2, 3], want[:, :2, 4], want[:, :2, 5], want[:, :2, 71] = np.inf, -np.inf, np.nan, np.nan
    if fmt == "i8":
        want[:, :2] = np.nan
    print(f"[gpu] infinite values seen whole {storage} {fmt} {new} {room}", flush=True)
    y = attended(s, k, v, q, storage)
    close(y, want, tol, "y")
    s.free()
