"""What the tests of the 8-bit layers share: device matrices in the three storage types, and the layers in 64 bits."""
import ctypes
import math

import numpy as np

from simdonnx_amd import native as N

UNIT = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}  # half a step, relative to the value
SMALL = {"f32": 2.0 ** -149, "f16": 2.0 ** -25, "bf16": 2.0 ** -133}  # and near zero


def to_bits(x, storage):
    """fp32 values as the storage type's bits, rounded to nearest even."""
    x = np.ascontiguousarray(x, np.float32)
    if storage == "f32":
        return x
    if storage == "f16":
        with np.errstate(over="ignore"):
            return x.astype(np.float16)
    b = x.view(np.uint32)
    r = ((b + 0x7fff + ((b >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7fc0), r)


def from_bits(b, storage):
    if storage == "bf16":
        return (b.astype(np.uint32) << 16).view(np.float32)
    return b.astype(np.float32)


def rounded(x, storage):
    return from_bits(to_bits(x, storage), storage)


# (rows, inner, columns) of floating products that one launch of 32 x 128 outputs rounds and multiplies, at both ends of the
# range of K of each of its instances
PANELS = [(90, 2, 40), (21, 256, 72), (90, 257, 72), (64, 512, 100), (70, 513, 33), (100, 768, 129), (100, 769, 136),
          (65, 1000, 40), (257, 1023, 301), (786, 1024, 760), (66, 1024, 1)]


class Matrix:
    """rows x cols of a storage type (or "i8") on the device, `ld` elements from row to row, `skip` elements behind an
    aligned base; every byte around the elements holds a pattern that `untouched` looks for."""

    def __init__(self, data=None, storage="f16", rows=0, cols=0, ld=None, skip=0, stream=None):
        if data is not None:
            rows, cols = data.shape
        self.rows, self.cols, self.storage, self.ld, self.skip, self.stream = rows, cols, storage, ld or cols, skip, stream
        self.dtype = {"f32": np.float32, "f16": np.float16, "bf16": np.uint16, "i8": np.int8}[storage]
        self.elem = np.dtype(self.dtype).itemsize
        count = skip + max(rows, 1) * self.ld + 64
        self.fill = np.frombuffer((b"\xa5\x5b\x3c\xd2" * (count * self.elem // 4 + 1))[:count * self.elem], np.uint8)
        host = self.fill.copy()
        if data is not None:
            self._view(host)[:] = data if storage == "i8" else to_bits(data, storage)
        p = N.c_void_p()
        N.check(N.thin().sox_malloc(ctypes.byref(p), host.size), "sox_malloc")
        self.base = p
        self._copy(host, up=True)

    def _view(self, host):
        flat = host.view(self.dtype)
        return np.lib.stride_tricks.as_strided(flat[self.skip:], (self.rows, self.cols), (self.ld * self.elem, self.elem))

    def _copy(self, host, up):
        T = N.thin()
        if up:
            N.check(T.sox_memcpy_h2d(self.base, host.ctypes.data, host.size, self.stream), "h2d")
        else:
            N.check(T.sox_memcpy_d2h(host.ctypes.data, self.base, host.size, self.stream), "d2h")
        N.check(T.sox_stream_sync(self.stream), "sync")

    @property
    def ptr(self):
        return self.base.value + self.skip * self.elem

    def refill(self):
        """Every byte back to the pattern."""
        self._copy(self.fill.copy(), up=True)

    def read(self):
        """The elements as fp32 (int8 as they are), after a check that nothing around them was written."""
        host = np.empty_like(self.fill)
        self._copy(host, up=False)
        got = self._view(host).copy()
        self._view(host)[:] = self._view(self.fill.copy())
        assert np.array_equal(host, self.fill), "bytes outside of the matrix were written"
        return got if self.storage == "i8" else from_bits(got, self.storage)

    def free(self):
        N.thin().sox_free(self.base)


def quantize(x):
    """(q, scale) of rows, exactly: 127 x is exact in 64 bits, so its quotient falls on the right side of every half."""
    x = np.asarray(x, np.float64)
    ok = np.isfinite(x).all(axis=1)
    amax = np.where(ok, np.abs(np.where(ok[:, None], x, 0)).max(axis=1), 0.0)
    q = np.where(ok[:, None] & (amax > 0)[:, None], np.rint(127 * np.where(ok[:, None], x, 0) / np.where(amax > 0, amax, 1)[:, None]), 0)
    scale = np.where(ok, (amax.astype(np.float32) / np.float32(127)).astype(np.float64), np.nan)
    return q.astype(np.int64), scale


_erf = np.vectorize(math.erf, otypes=[np.float64])


def act64(v, act):
    if act == "relu":
        return np.where(v < 0, 0.0, v)
    if act == "gelu":
        return 0.5 * v * (1 + _erf(v * math.sqrt(0.5)))
    if act in ("sigmoid", "swish"):
        s = 1 / (1 + np.exp(-np.clip(v, -700, 700)))
        return s if act == "sigmoid" else v * s
    if act == "hardswish":
        return v * np.clip(v / 6 + 0.5, 0, 1)
    return v


def act_error(ref, act, storage):
    """What the activation's own formula may be off by: gelu_fast 3.9e-6 absolute and 2.7e-5 relative where 16 bits
    follow, the erf of Abramowitz and Stegun 7.1.26 1.5e-7 times |v| / 2 in fp32 (on top of its exponential's 2e-7); the
    polynomial exponential of the sigmoids 2e-7 relative, taken as ten times that for the quotient around it."""
    if act == "gelu":
        return 4e-6 + 2.8e-5 * np.abs(ref) if storage != "f32" else 4e-7 * (1 + np.abs(ref))
    return 2e-6 * np.abs(ref) if act in ("sigmoid", "swish") else 0.0


def linear64(q, scale, w, ws, bias, res, act, storage):
    """(y, tolerance): the product over whole numbers, and what fp32 and the output's rounding may be off by. The sum is
    exact; its conversion, two scale products, the fma, the residual's addition and the row scale's own rounding
    are at most one unit of fp32 each of the terms they join; every activation's slope is below 1.13."""
    s = q.astype(np.float64) @ np.asarray(w, np.float64)  # (whole numbers below 2^53: exact)
    prod = s * scale[:, None] * np.asarray(ws, np.float64)
    v, size = prod, np.abs(prod)
    for t in (bias, res):
        if t is not None:
            v, size = v + t, size + np.abs(t)
    y = act64(v, act)
    return y, UNIT[storage] * np.abs(y) + SMALL[storage] + 1.13 * 6 * 2.0 ** -24 * size + act_error(y, act, storage) * (1 + UNIT[storage])


def norm64(v, kind, gamma, beta, eps):
    """(result, deviation before the gamma, 1 / root)."""
    if kind == "none":
        return v, v, np.ones((v.shape[0], 1))
    d = v - v.mean(axis=1, keepdims=True) if kind == "layer" else v
    r = 1 / np.sqrt((d * d).mean(axis=1, keepdims=True) + eps)
    out = d * r * (1.0 if gamma is None else gamma)
    return (out + beta if kind == "layer" and beta is not None else out), d, r


def block64(res, x, gate, p, storage):
    """(h, y, tolerance of h before its rounding, of y before its rounding). p: the HipBlockNorm keywords.

    A row's sums have at most 32 additions in a lane, 6 in a wave and 16 across waves: 56 units of fp32 of the sum of
    magnitudes. A mean square of that error moves the root by half of it, a mean of it the deviations by that times the
    mean magnitude; the other steps (square, division, root, gamma, beta, scale, gate, residual) are one unit each, ten
    in all. So a norm's result is off by at most (28 + 10) units of itself and 57 units of mean |v| * gamma / root, and
    by the deviations' own error over the root, which an input error reaches at most three times (itself, through
    the mean and through the root)."""
    u = 2.0 ** -24
    f = lambda k: None if p.get(k) is None else np.asarray(p[k], np.float64)  # noqa: E731
    eps = lambda k: float(np.float32(p.get(k, 1e-5)))  # noqa: E731

    def step(v, err, kind, gamma, beta, e):
        y, d, r = norm64(v, kind, gamma, beta, e)
        if kind == "none":
            return y, err
        g = 1.0 if gamma is None else np.abs(gamma)
        top = np.maximum(np.abs(v), err).max(axis=1, keepdims=True) * r  # |normed| at most, in units of gamma
        rel = err.max(axis=1, keepdims=True) * r * (1 + 2 * np.minimum(top, 1e9))
        return y, 38 * u * (np.abs(d) * r * g + (0 if beta is None else np.abs(beta))) + 57 * u * np.abs(v).mean(axis=1, keepdims=True) * r * g + rel * g

    rs = float(np.float32(p.get("res_scale", 1.0)))
    h = np.zeros_like(res if res is not None else x)
    eh = np.zeros_like(h)
    if x is not None:
        a, ea = step(x, np.zeros_like(x), p.get("post", "none"), f("post_gamma"), f("post_beta"), eps("post_eps"))
        if f("scale") is not None:
            a, ea = a * f("scale"), ea * np.abs(f("scale"))
        if gate is not None:
            g = act64(gate, p.get("gate_act", "none"))
            g = np.repeat(g, x.shape[0] // g.shape[0], axis=0)
            ea = ea * np.abs(g) + np.abs(a) * (4e-7 * (1 + np.abs(g)) if p.get("gate_act", "none") == "gelu" else 3e-6 * np.abs(g))
            a = a * g
        h, eh = h + a, eh + ea + 4 * u * np.abs(a)
    if res is not None:
        h, eh = h + rs * res, eh + 2 * u * np.abs(rs * res)
    eh = eh + 2 * u * np.abs(h)
    y, ey = step(h, eh, p.get("pre", "layer"), f("pre_gamma"), f("pre_beta"), eps("pre_eps"))
    return h, y, eh, ey
