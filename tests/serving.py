"""What the tests of the paged cache and its attention share: batches on the device, and the operators in 64 bits."""
import numpy as np

from layers import SMALL, UNIT, Matrix, quantize, to_bits
from simdonnx_amd.backend import HipKvBatch, HipKvCache

U32 = 2.0 ** -24
TABLE_TOKENS = 0  # tokens that a Serving's tables have room for at least, beyond what its sequences hold


class Ints(Matrix):
    """int32 values [rows, cols] on the device."""

    def __init__(self, data, stream=None):
        data = np.ascontiguousarray(np.atleast_2d(data), np.int32)
        super().__init__(data.view(np.float32), "f32", stream=stream)  # (their bits)

    def read(self):
        return super().read().view(np.int32)

    def write(self, data):
        host = self.fill.copy()
        self._view(host)[:] = np.atleast_2d(np.asarray(data, np.int32)).view(np.float32)
        self._copy(host, up=True)


class Pool(Matrix):
    """A cache's pages; every byte 0xff first: NaN as a float, -1 as 8 bits with NaN scales."""

    def __init__(self, cache, pages, stream=None):
        super().__init__(None, "i8", 1, cache.page_bytes * pages, stream=stream)
        host = self.fill.copy()
        self._view(host)[:] = -1
        self._copy(host, up=True)


class Serving:
    """Sequences of (tokens, new tokens) over a cache, their pages in a shuffled order. `before` rows stand ahead of the first
    sequence's, `behind` after the last's."""

    def __init__(self, hip, sequences, kv, dim, page, fmt, seed=0, before=0, behind=0, spare=2, stream=None):
        rng = np.random.default_rng(seed)
        self.sequences, self.kv, self.dim, self.page, self.fmt, self.stream = sequences, kv, dim, page, fmt, stream
        self.cache = HipKvCache(hip, kv, dim, page=page, format=fmt)
        counts = [-(-length // page) for length, _ in sequences]
        self.pages = sum(counts) + spare
        order = rng.permutation(self.pages)
        self.tables = np.full((len(sequences), max(max(counts + [1]) + 1, TABLE_TOKENS // page)), -1, np.int32)
        at = 0
        for s, n in enumerate(counts):
            self.tables[s, :n] = order[at:at + n]
            at += n
        self.pool = Pool(self.cache, self.pages, stream)
        self.starts = before + np.cumsum([0] + [n for _, n in sequences])
        self.rows = int(self.starts[-1]) + behind
        self.lengths = np.array([n for n, _ in sequences])
        self.whole = np.cumsum([0] + [n for n, _ in sequences])
        self.d_tables, self.d_starts, self.d_lengths, self.d_whole = (Ints(v, stream) for v in (self.tables, self.starts, self.lengths, self.whole))
        self.batch, self.every = self.of(self.d_starts, self.rows), self.of(self.d_whole, int(self.whole[-1]))

    def of(self, starts, rows):
        return HipKvBatch(self.pool.ptr, self.pages, self.d_tables.ptr, self.tables.shape[1], starts.ptr, self.d_lengths.ptr, len(self.sequences), rows)

    def positions(self):
        """[rows]: each row's token, -1 where it is no sequence's."""
        p = np.full(self.rows, -1)
        for s, (length, new) in enumerate(self.sequences):
            p[self.starts[s]:self.starts[s + 1]] = np.arange(length - new, length)
        return p

    def free(self):
        for m in (self.pool, self.d_tables, self.d_starts, self.d_lengths, self.d_whole):
            m.free()
        self.cache.close()


def turned64(x, positions, frequencies, interleaved, amplitude=1.0):
    """x [rows, heads, dim] turned, and what one product and sum of fp32 with rounded cosines may be off by (each of cos, sin,
    the product and the fma half a step of the term it joins: two for each term, and one for the sum)."""
    x = np.asarray(x, np.float64)
    n = 2 * len(frequencies)
    angle = np.asarray(positions, np.float64)[:, None] * frequencies
    c, s = amplitude * np.cos(angle)[:, None], amplitude * np.sin(angle)[:, None]
    i, j = (slice(0, n, 2), slice(1, n, 2)) if interleaved else (slice(0, n // 2), slice(n // 2, n))
    y, err = x.copy(), np.zeros_like(x)
    a, b = x[..., i], x[..., j]
    y[..., i], y[..., j] = a * c - b * s, b * c + a * s
    err[..., i], err[..., j] = (3 * U32 * (abs(a * c) + abs(b * s)), 3 * U32 * (abs(b * c) + abs(a * s)))
    return y, err


def held64(x, storage, fmt):
    """What the cache holds of values x [tokens, heads, dim] (fp32 or 64 bits, the turned ones rounded here)."""
    if fmt != "i8":
        from layers import from_bits
        return from_bits(to_bits(x, storage), storage).astype(np.float64)
    x = np.asarray(x, np.float32).astype(np.float64)
    q, scale = quantize(x.reshape(-1, x.shape[-1]))
    with np.errstate(invalid="ignore"):
        return (q * scale[:, None]).reshape(x.shape)


def attend64(q, k, v, first, scale, window, storage, absent=None):
    """(y, tolerance) [new, heads, dim] of one sequence: q [new, heads, dim] at positions first .., over k, v [tokens, kv, dim].

    A score: dim products summed in fp32, each partial sum off by a unit of the sum of magnitudes, and four more for the scales
    and the exponential's argument; e is the largest of a row. p is off by that twice over (its own and the reference's,
    which the sum divides out) and by half a step of the storage type where 16 bits hold it for its product; the sum may take p as
    it is or as rounded, and then is off by at most that half step of itself, y by that half step of |y|; p too
    small for fp16's normal numbers by half of 2^-24 of the largest value for each token, and p below fp32's normal numbers by
    itself, 2^-126 at most (the reference is no larger than the largest score, so the sum that divides is 1 or more). The
    sums of n terms: n units, twice."""
    new, heads, dim = q.shape
    tokens, kv, _ = k.shape
    y, tol = np.zeros((new, heads, dim)), np.zeros((new, heads, dim))
    t = np.arange(tokens)
    for i in range(new):
        pos = first + i
        sees = (t <= pos) & ((t > pos - window) if window else True)
        if absent is not None:
            sees &= ~absent
        if not sees.any():
            continue
        for g in range(kv):
            mine = slice(g * (heads // kv), (g + 1) * (heads // kv))
            kk, vv = k[sees, g], v[sees, g]
            s = scale * (q[i, mine] @ kk.T)
            e = (dim + 6) * U32 * scale * (np.abs(q[i, mine]) @ np.abs(kk).T).max(axis=1, keepdims=True)
            with np.errstate(invalid="ignore"):
                p = np.exp(s - np.fmax.reduce(s, axis=1, keepdims=True))
                total = p.sum(axis=1, keepdims=True)
                y[i, mine] = p @ vv / total
                size = p @ np.abs(vv) / total
            n = int(sees.sum())
            half = 0.0 if storage == "f32" else UNIT[storage]
            tiny = n * (2.0 ** -25 if storage == "f16" else 2.0 ** -126) * np.abs(vv).max(axis=0)
            tol[i, mine] = (half + 4 * e + (2 * n + 16) * U32) * size + tiny + (half + UNIT[storage]) * np.abs(y[i, mine]) + SMALL[storage]
    return y, tol


def close(got, want, tol, what):
    """Within the tolerance; NaN and infinities where they are wanted."""
    fin = np.isfinite(want)
    with np.errstate(invalid="ignore"):
        bad = np.where(fin, ~(np.abs(got - want) <= tol), ~((got == want) | (np.isnan(got) & np.isnan(want))))
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.size}, first at {np.argwhere(bad)[0]}: {got[bad][0]} for {want[bad][0]}, tolerance {np.broadcast_to(tol, bad.shape)[bad][0]}"
