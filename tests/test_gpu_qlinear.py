"""The product in 8-bit integers with row and channel scales (sox_qlinear_*, HipQuantLinear) against the same product in
whole numbers and 64 bits. Tolerances are the steps' roundings (tests/layers.py); what the 8-bit rounding itself does
is exact on both sides."""
import ctypes
import os
import subprocess
import sys
import threading

import numpy as np
import pytest

from simdonnx_amd import native as N
from simdonnx_amd import synth
from simdonnx_amd.backend import HipQuantLinear
from simdonnx_amd.native import SoxError
from tests.layers import PANELS, Matrix, from_bits, linear64, quantize, rounded, to_bits

pytestmark = pytest.mark.gpu

TILES = ["256x256_w8k128s2", "256x192_w8k128s2", "256x128_w8k128s2", "128x128_w4k128s2", "64x64_w4k128s4"]


def weights8(seed, k, n):
    w = np.rint(synth.uniform(seed, 1, (k, n), -127.4, 127.4)).astype(np.int8)
    return w, synth.uniform(seed, 2, (n,), 0.5, 1.5) / (70 * np.sqrt(k))


def rows_of(seed, rows, k, storage):
    """Normal rows of different sizes, a few large channels, one row of zeros where there are several."""
    x = synth.normal(seed, 3, (rows, k), 1.0) * np.exp2(np.arange(rows) % 7 - 3)[:, None].astype(np.float32)
    x[:, ::61] *= 12
    if rows > 3:
        x[2] = 0
    return rounded(x, storage)


def check(got, want, tol):
    assert np.array_equal(np.isnan(got), np.isnan(want))
    ok = ~np.isnan(want)
    over = np.abs(got[ok].astype(np.float64) - want[ok]) - tol[ok]
    assert (over <= 0).all(), f"{(over > 0).sum()} of {over.size} values, worst {over.max():.3g} over its tolerance"


def both_ways(hip, seed, rows, k, n, storage, act="none", bias=True, res=False, pad=0, skip=0, inplace=False):
    """The layer over floating rows and over the 8-bit rows they become, with outputs at odd strides and places."""
    w, ws = weights8(seed, k, n)
    b = synth.uniform(seed, 4, (n,), -1, 1) if bias else None
    x = rows_of(seed, rows, k, storage)
    r = rounded(synth.normal(seed, 5, (rows, n), 1.0), storage) if res else None
    q, scale = quantize(x)
    want, tol = linear64(q, scale, w, ws, b, r, act, storage)
    lin = HipQuantLinear(hip, w, b, k, n, scales=ws)
    X = Matrix(x, storage, ld=k + pad, skip=skip)
    Y = Matrix(r if inplace else None, storage, rows, n, ld=n + pad, skip=skip)
    R = Y if inplace else (Matrix(r, storage, ld=n + pad, skip=skip) if res else None)
    k16 = -(-k // 16) * 16
    q8 = np.full((rows, k16), 77, np.int8)  # what lies past inner is not used
    q8[:, :k] = q
    Q = Matrix(q8, "i8", ld=k16 + 16 * (pad % 5))
    S = Matrix(scale.astype(np.float32)[None], "f32")
    W = Matrix(None, "i8", 1, max(1, lin.workspace(rows)))
    given = dict(ldy=Y.ld, act=act, residual=R.ptr if R else None, ldr=R.ld if R else None)
    lin.run(X.ptr, rows, Y.ptr, storage, ldx=X.ld, workspace=W.ptr, workspace_bytes=lin.workspace(rows), **given)
    got = Y.read()
    check(got, want, tol)
    if not inplace:
        Y.refill()
        lin.run_quantized(Q.ptr, S.ptr, rows, Y.ptr, storage, ldq=Q.ld, **given)
        assert np.array_equal(Y.read(), got, equal_nan=True)  # whole numbers: the same bits either way
    W.read()
    for m in {X, Y, Q, S, W} | ({R} if R else set()):
        m.free()
    lin.close()


@pytest.mark.parametrize("storage", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("rows,k,n", [(1, 1, 1), (1, 768, 768), (2, 16, 15), (3, 65, 33), (7, 4096, 80), (16, 1000, 17), (16, 4097, 40), (16, 4096, 24),
                                      (17, 577, 301), (33, 129, 64), (64, 320, 100), (1, 9000, 31)])
def test_few_rows(hip, storage, rows, k, n):
    print(f"[gpu] qlinear {storage} {rows} x {k} -> {n}", flush=True)
    both_ways(hip, 1000 + rows + k, rows, k, n, storage)


@pytest.mark.parametrize("storage", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("rows,k,n", [(1, 1025, 40), (2, 1100, 33), (16, 1536, 72), (5, 2047, 17), (16, 2048, 48)])
def test_few_rows_of_two_steps_a_wave(hip, storage, rows, k, n):
    print(f"[gpu] qlinear {storage} {rows} x {k} -> {n}", flush=True)
    both_ways(hip, 1500 + rows + k, rows, k, n, storage)
    both_ways(hip, 1600 + rows + k, rows, k, n, storage, act="gelu", bias=False, res=True, pad=5, skip=1)


@pytest.mark.parametrize("tile", TILES)
@pytest.mark.parametrize("storage,rows,k,n,pad,skip", [
    ("f16", 300, 768, 520, 0, 0), ("bf16", 65, 1, 1, 0, 0), ("bf16", 257, 64, 300, 8, 0), ("f16", 130, 200, 257, 3, 1),
    ("f32", 513, 65, 259, 0, 0), ("f32", 128, 129, 256, 4, 1), ("bf16", 1000, 16, 96, 0, 0)])
def test_tiles(hip, monkeypatch, tile, storage, rows, k, n, pad, skip):
    """Every tiling, also where the choice would not take it: one slice of K and many, partial tiles on both sides."""
    if tile[:7] == "256x256" and (storage == "f32" or n % 8):
        pytest.skip("the largest tiling takes 16-bit outputs of whole 16-byte chunks")
    monkeypatch.setenv("SIMDONNX_HIP_QGEMM", tile)
    print(f"[gpu] qlinear {tile} {storage} {rows} x {k} -> {n}", flush=True)
    both_ways(hip, 2000 + k, rows, k, n, storage, act="none", res=pad > 0, pad=pad, skip=skip)


@pytest.mark.parametrize("tile", TILES)
@pytest.mark.parametrize("storage", ["f16", "bf16", "f32"])
def test_outputs_on_lines_and_off(hip, monkeypatch, tile, storage):
    """Output rows on 128-byte lines (a kernel of their own), on 16-byte boundaries only, and on neither, a residual on less
    than they are: the same bits each time."""
    if storage == "f32" and tile.startswith("256x256"):
        pytest.skip("16-bit outputs only")
    monkeypatch.setenv("SIMDONNX_HIP_QGEMM", tile)
    rows, k, n, line = 300, 200, 328, 384
    w, ws = weights8(3, k, n)
    x = rows_of(4, rows, k, storage)
    r = rounded(synth.normal(5, 5, (rows, n), 1.0), storage)
    q, scale = quantize(x)
    want, tol = linear64(q, scale, w, ws, None, r, "swish", storage)
    lin = HipQuantLinear(hip, w, None, k, n, scales=ws)
    q8 = np.zeros((rows, lin.pitch), np.int8)
    q8[:, :k] = q
    Q, S = Matrix(q8, "i8"), Matrix(scale.astype(np.float32)[None], "f32")
    chunk = 16 // (4 if storage == "f32" else 2)
    outs = []
    for (ld, skip), (ldr, skipr) in (((line, 0), (line, 0)), ((line, 0), (n, chunk)), ((line, 0), (n + 1, 0)),
                                     ((n, 0), (line, 0)), ((line, chunk), (line, 0)), ((line, 1), (line, 0)), ((n + 3, 0), (n, 1))):
        print(f"[gpu] {tile} {storage} y {ld} {skip} residual {ldr} {skipr}", flush=True)
        Y, R = Matrix(None, storage, rows, n, ld=ld, skip=skip), Matrix(r, storage, ld=ldr, skip=skipr)
        lin.run_quantized(Q.ptr, S.ptr, rows, Y.ptr, storage, ldq=Q.ld, ldy=ld, act="swish", residual=R.ptr, ldr=ldr)
        outs.append(Y.read())
        Y.free()
        R.free()
    check(outs[0], want, tol)
    for o in outs[1:]:
        assert np.array_equal(o, outs[0], equal_nan=True)
    Q.free()
    S.free()
    lin.close()


@pytest.mark.parametrize("tile", TILES)
def test_many_tiles_per_workgroup(hip, monkeypatch, tile):
    """More tiles than workgroups, with one slice of K each: a workgroup's slices run several tiles ahead."""
    monkeypatch.setenv("SIMDONNX_HIP_QGEMM", tile)
    rows, n = {"256": (12000, 3304), "128": (9000, 2500), "64x": (4200, 2200)}[tile[:3].rstrip("x") if tile[0] != "6" else "64x"]
    print(f"[gpu] qlinear {tile} {rows} x 40 -> {n}", flush=True)
    both_ways(hip, 2100, rows, 40, n, "bf16")


@pytest.mark.parametrize("storage", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("rows,k,n", PANELS)
def test_panels(hip, storage, rows, k, n):
    """Rows rounded and multiplied by one launch, at the ends of each instance's range of K: the bits of the same rows given
    in 8 bits, with whole rows and with a residual and rows off every boundary."""
    print(f"[gpu] qlinear panel {storage} {rows} x {k} -> {n}", flush=True)
    both_ways(hip, 2200 + k, rows, k, n, storage)
    both_ways(hip, 2300 + k, rows, k, n, storage, act="swish", bias=False, res=True, pad=3, skip=1)


@pytest.mark.parametrize("act", ["none", "relu", "sigmoid", "gelu", "hardswish", "swish"])
@pytest.mark.parametrize("storage,rows", [("f16", 5), ("bf16", 100), ("f32", 70)])
def test_activations(hip, act, storage, rows):
    print(f"[gpu] qlinear {act} {storage} {rows}", flush=True)
    both_ways(hip, 3000, rows, 96, 72, storage, act=act, res=True)


@pytest.mark.parametrize("rows", [9, 40, 200])
def test_residual_in_place(hip, rows):
    print(f"[gpu] qlinear in place {rows}", flush=True)
    both_ways(hip, 3100, rows, 192, 104, "f16", res=True, inplace=True)
    both_ways(hip, 3101, rows, 192, 99, "bf16", res=True, inplace=True, bias=False, pad=2, skip=3)


@pytest.mark.parametrize("storage", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("rows", [4, 48, 150])
def test_rows_that_are_not_finite(hip, storage, rows):
    """A NaN or an infinity makes its own row NaN and leaves the others alone, at the ends of the range too."""
    k, n = 100, 40
    w, ws = weights8(5, k, n)
    x = rows_of(5, rows, k, storage)
    big = {"f16": 65504.0, "bf16": 3.3e38, "f32": 3.4e38}[storage]
    tiny = {"f16": 2.0 ** -24, "bf16": 2.0 ** -133, "f32": 2.0 ** -140}[storage]
    x[0] = np.sign(x[0]) * big
    x[1] = rounded(tiny * np.rint(3 * np.abs(x[1])), storage)
    x[3, 50] = np.inf
    if rows > 20:
        x[17, 99] = np.nan
        x[20] = -np.inf
    x = rounded(x, storage)
    q, scale = quantize(x)
    want, tol = linear64(q, scale, w, ws, None, None, "relu", storage)
    # outputs past the type's largest value are infinite, and fp32's scale of the smallest rows is a subnormal with its
    # own half step, times at most the row's sum of products
    tol += 2.0 ** -150 * np.abs(q @ w.astype(np.int64)) * ws
    lin = HipQuantLinear(hip, w, None, k, n, scales=ws)
    X, Y, W = Matrix(x, storage), Matrix(None, storage, rows, n), Matrix(None, "i8", 1, max(1, lin.workspace(rows)))
    print(f"[gpu] qlinear not finite {storage} {rows}", flush=True)
    lin.run(X.ptr, rows, Y.ptr, storage, act="relu", workspace=W.ptr, workspace_bytes=lin.workspace(rows))
    got = Y.read()
    assert np.isnan(got[3]).all() and (rows <= 20 or np.isnan(got[17]).all() and np.isnan(got[20]).all())
    top = np.float64({"f16": 65504.0, "bf16": 3.3895e38, "f32": 3.4028e38}[storage])
    fits = np.abs(want) + tol < top
    keep = fits | np.isnan(want)
    check(np.where(keep, got, 0), np.where(keep, want, 0), np.where(keep, tol, 0))
    for m in (X, Y, W):
        m.free()
    lin.close()


def test_halves_round_to_even(hip):
    """Rows whose values lie on halves of their step (x = amax / 2 is 63.5 steps) and one place beside: an identity of
    weights and a channel scale of 1 give q times the row's scale back."""
    k = 64
    w = (np.eye(k) * 1).astype(np.int8)
    lin = HipQuantLinear(hip, w, None, k, k, scales=np.ones(k, np.float32))
    for storage, step in (("f16", 2.0 ** -10), ("bf16", 2.0 ** -7), ("f32", 2.0 ** -23)):
        x = np.zeros((200, k), np.float32)
        amax = (1 + np.arange(200) * (1 / 256 if storage != "bf16" else 1 / 128) % 1).astype(np.float32)
        x[:, 0] = amax
        for i in range(1, k):  # near (j + 1/2) steps, by -1, 0, 1 places of the storage type
            j = i * 2
            v = amax.astype(np.float64) * (j + 0.5) / 127
            place = step * np.exp2(np.floor(np.log2(v)))
            x[:, i] = np.rint(v / place) * place + (i % 3 - 1) * place
        x[:, 63] = amax / 2
        x = rounded(x, storage)
        q, scale = quantize(x)
        X, Y, W = Matrix(x, storage), Matrix(None, "f32", 200, k), Matrix(None, "i8", 1, max(1, lin.workspace(200)))
        for rows, first in ((200, 0), (16, 3)):  # the row kernel, and the fused one
            print(f"[gpu] qlinear halves {storage} {rows}", flush=True)
            if storage == "f32":
                lin.run(X.ptr + first * k * 4, rows, Y.ptr, "f32", workspace=W.ptr, workspace_bytes=lin.workspace(200))
                got = Y.read()[:rows]
                assert np.array_equal(got, (q[first:first + rows] * scale[first:first + rows, None]).astype(np.float32))
            else:
                O = Matrix(None, storage, rows, k)
                lin.run(X.ptr + first * k * 2, rows, O.ptr, storage, workspace=W.ptr, workspace_bytes=lin.workspace(200))
                s32 = scale[first:first + rows].astype(np.float32)
                assert np.array_equal(O.read(), rounded(q[first:first + rows].astype(np.float32) * s32[:, None], storage))
                O.free()
        for m in (X, Y, W):
            m.free()
    lin.close()


def test_largest_sums(hip):
    """131071 products of -128 and -128: the largest sum 32 bits have to hold, in every way through the product."""
    k, n = 131071, 3
    w = np.full((k, n), -128, np.int8)
    lin = HipQuantLinear(hip, w, None, k, n, scales=np.full(n, 2.0 ** -20, np.float32))
    for rows in (2, 70):
        q = np.full((rows, k + 1), -128, np.int8)
        Q, S, Y = Matrix(q, "i8"), Matrix(np.ones((1, rows)), "f32"), Matrix(None, "f32", rows, n)
        print(f"[gpu] qlinear largest sums {rows}", flush=True)
        lin.run_quantized(Q.ptr, S.ptr, rows, Y.ptr, "f32", ldq=k + 1)
        assert (Y.read() == np.float32(k * 2.0 ** 14) * 2.0 ** -20).all()
        for m in (Q, S, Y):
            m.free()
    lin.close()


def test_weights_by_column(hip):
    """Floating weights are brought to 8 bits by column, exactly, a column of zeros included."""
    k, n, rows = 130, 50, 70
    w = synth.normal(8, 1, (k, n), 0.1) * np.exp2(np.arange(n) % 9 - 4).astype(np.float32)
    w[:, 7] = 0
    w[3, 9] = 2 * np.abs(w[:, 9]).max()
    w[4, 9] = w[3, 9] / 2  # a half
    wq, ws = quantize(w.T)
    x = rows_of(8, rows, k, "bf16")
    q, scale = quantize(x)
    want, tol = linear64(q, scale, wq.T, ws, None, None, "none", "bf16")
    lin = HipQuantLinear(hip, w, None, k, n)
    X, Y, W = Matrix(x, "bf16"), Matrix(None, "bf16", rows, n), Matrix(None, "i8", 1, max(1, lin.workspace(rows)))
    print("[gpu] qlinear float weights", flush=True)
    lin.run(X.ptr, rows, Y.ptr, "bf16", workspace=W.ptr, workspace_bytes=lin.workspace(rows))
    check(Y.read(), want, tol)
    for m in (X, Y, W):
        m.free()
    lin.close()


def test_columns_of_one_buffer(hip):
    """Input and output side by side in the rows of one buffer: disjoint elements, whatever their ranges."""
    rows, k, n = 100, 64, 48
    w, ws = weights8(9, k, n)
    x = rows_of(9, rows, k, "f16")
    q, scale = quantize(x)
    want, tol = linear64(q, scale, w, ws, None, None, "none", "f16")
    both = np.concatenate([x, np.zeros((rows, n), np.float32)], axis=1)
    lin = HipQuantLinear(hip, w, None, k, n, scales=ws)
    B, W = Matrix(both, "f16"), Matrix(None, "i8", 1, max(1, lin.workspace(rows)))
    print("[gpu] qlinear one buffer", flush=True)
    lin.run(B.ptr, rows, B.ptr + 2 * k, "f16", ldx=k + n, ldy=k + n, workspace=W.ptr, workspace_bytes=lin.workspace(rows))
    got = B.read()
    assert np.array_equal(got[:, :k], x)
    check(got[:, k:], want, tol)
    for m in (B, W):
        m.free()
    lin.close()


@pytest.mark.parametrize("rows", [6, 300])
def test_captured_calls_replay(hip, rows):
    """A call captured into a graph gives the eager bits on every replay, with new inputs and eager work in between;
    two graphs of one layer with workspaces of their own replay on two streams at once."""
    k, n = 192, 136
    w, ws = weights8(10, k, n)
    lin = HipQuantLinear(hip, w, None, k, n, scales=ws)
    T = N.thin()
    sides = []
    for i in range(2):
        st = N.c_void_p()
        N.check(T.sox_stream_create(ctypes.byref(st)), "stream")
        X, Y = Matrix(rows_of(20 + i, rows, k, "f16"), "f16"), Matrix(None, "f16", rows, n)
        W = Matrix(None, "i8", 1, max(1, lin.workspace(rows)))
        call = lambda X=X, Y=Y, W=W, st=st: lin.run(X.ptr, rows, Y.ptr, "f16", workspace=W.ptr,  # noqa: E731
                                                    workspace_bytes=lin.workspace(rows), stream=st)
        print(f"[gpu] qlinear capture {rows} side {i}", flush=True)
        N.check(T.sox_graph_begin(st), "capture")
        call()
        ex = N.c_void_p()
        N.check(T.sox_graph_end(st, ctypes.byref(ex)), "capture end")
        sides.append((st, X, Y, W, call, ex))
    for rep in range(3):
        want = []
        for i, (st, X, Y, W, call, ex) in enumerate(sides):
            x = rows_of(100 + 10 * rep + i, rows, k, "f16")
            X2 = Matrix(x, "f16")
            N.check(T.sox_memcpy_d2d(X.ptr, X2.ptr, x.size * 2, st), "new input")
            call()
            N.check(T.sox_stream_sync(st), "sync")
            X2.free()
            want.append(Y.read())
            Y.refill()
        for st, *_, ex in sides:
            N.check(T.sox_graph_launch(ex, st), "replay")
        for (st, X, Y, W, call, ex), e in zip(sides, want):
            N.check(T.sox_stream_sync(st), "sync")
            assert np.array_equal(Y.read(), e), rep
    for st, X, Y, W, call, ex in sides:
        T.sox_graph_destroy(ex)
        T.sox_stream_destroy(st)
        for m in (X, Y, W):
            m.free()
    lin.close()


def test_allocates_nothing(hip):
    k, n, rows = 64, 64, 100
    w, ws = weights8(11, k, n)
    lin = HipQuantLinear(hip, w, None, k, n, scales=ws)
    X, Y = Matrix(rows_of(11, rows, k, "f16"), "f16"), Matrix(None, "f16", rows, n)
    W = Matrix(None, "i8", 1, max(1, lin.workspace(rows)))
    before = N.thin().sox_alloc_count()
    lin.run(X.ptr, rows, Y.ptr, "f16", workspace=W.ptr, workspace_bytes=lin.workspace(rows))
    lin.run(X.ptr, 0, Y.ptr, "f16")
    assert N.thin().sox_alloc_count() == before
    Y.read()
    for m in (X, Y, W):
        m.free()
    lin.close()


def test_memory_of_the_host_is_refused(hip, monkeypatch):
    """Addresses that no GPU reads, and a tiling that there is not, are errors before anything is launched."""
    k, n, rows = 64, 64, 100
    w, ws = weights8(12, k, n)
    lin = HipQuantLinear(hip, w, None, k, n, scales=ws)
    X, Y = Matrix(rows_of(12, rows, k, "f16"), "f16"), Matrix(None, "f16", rows, n)
    W = Matrix(None, "i8", 1, 1024)
    host = np.zeros(rows * k * 2, np.uint8)
    given = dict(workspace=W.ptr, workspace_bytes=lin.workspace(rows))
    with pytest.raises(SoxError, match="x is not in memory the GPU reads"):
        lin.run(host.ctypes.data // 16 * 16 + 16, rows - 1, Y.ptr, "f16", **given)
    with pytest.raises(SoxError, match="y is not in memory the GPU reads"):
        lin.run(X.ptr, rows - 1, host.ctypes.data // 16 * 16 + 16, "f16", **given)
    monkeypatch.setenv("SIMDONNX_HIP_QGEMM", "1x1")
    with pytest.raises(SoxError, match="no tiling 1x1"):
        lin.run_quantized(X.ptr, W.ptr, rows, Y.ptr, "f16", ldq=64)
    Y.read()
    for m in (X, Y, W):
        m.free()
    lin.close()


def rows_apart(data, storage, pitch):
    """The rows of a matrix `pitch` bytes apart in an allocation that nothing else of is written or read: (address, read)."""
    bits = to_bits(data, storage)
    p = N.c_void_p()
    N.check(N.thin().sox_malloc(ctypes.byref(p), (len(bits) - 1) * pitch + bits[0].nbytes), "sox_malloc")
    for i, row in enumerate(bits):
        row = np.ascontiguousarray(row)
        N.check(N.thin().sox_memcpy_h2d(p.value + i * pitch, row.ctypes.data, row.nbytes, None), "h2d")
    N.check(N.thin().sox_stream_sync(None), "sync")

    def read():
        got = np.empty_like(bits)
        for i in range(len(got)):
            N.check(N.thin().sox_memcpy_d2h(got[i].ctypes.data, p.value + i * pitch, got[i].nbytes, None), "d2h")
        N.check(N.thin().sox_stream_sync(None), "sync")
        return from_bits(got, storage)
    return p, read


@pytest.mark.parametrize("rows,k", [(70, 1100), (40, 96), (12, 200)])
def test_rows_far_apart(hip, rows, k):
    """Offsets past 32 bits, in elements and in bytes, of the input, the 8-bit rows, the residual and the output."""
    n, pitch, st = 40, 1 << 28, "bf16"
    w, ws = weights8(13, k, n)
    x, r = rows_of(13, rows, k, st), rounded(synth.normal(13, 6, (rows, n), 1.0), st)
    q, scale = quantize(x)
    want, tol = linear64(q, scale, w, ws, None, r, "none", st)
    lin = HipQuantLinear(hip, w, None, k, n, scales=ws)
    (X, _), (Y, read), (R, _) = rows_apart(x, st, pitch), rows_apart(np.zeros((rows, n), np.float32), st, pitch), rows_apart(r, st, pitch)
    W = Matrix(None, "i8", 1, max(1, lin.workspace(rows)))
    print(f"[gpu] qlinear rows far apart {rows} x {k}", flush=True)
    lin.run(X.value, rows, Y.value, st, ldx=pitch // 2, ldy=pitch // 2, residual=R.value, ldr=pitch // 2, workspace=W.ptr,
            workspace_bytes=lin.workspace(rows))
    got = read()
    check(got, want, tol)
    q8 = np.zeros((rows, -(-k // 16) * 16), np.float32)
    q8[:, :k] = q
    S = Matrix(scale.astype(np.float32)[None], "f32")
    N.check(N.thin().sox_free(X), "free")
    p = N.c_void_p()
    N.check(N.thin().sox_malloc(ctypes.byref(p), (rows - 1) * pitch + q8.shape[1]), "sox_malloc")
    for i, row in enumerate(q8.astype(np.int8)):
        N.check(N.thin().sox_memcpy_h2d(p.value + i * pitch, row.ctypes.data, row.nbytes, None), "h2d")
    N.check(N.thin().sox_stream_sync(None), "sync")
    lin.run_quantized(p.value, S.ptr, rows, Y.value, st, ldq=pitch, ldy=pitch // 2, residual=R.value, ldr=pitch // 2)
    assert np.array_equal(read(), got)
    for m in (p, Y, R):
        N.thin().sox_free(m)
    for m in (W, S):
        m.free()
    lin.close()


def test_calls_from_threads(hip):
    """One layer called from four threads at once, each on a stream and with a workspace of its own."""
    k, n, rows, times = 1200, 136, 90, 20
    w, ws = weights8(14, k, n)
    lin = HipQuantLinear(hip, w, None, k, n, scales=ws)
    T = N.thin()
    sides, errors = [], []
    for i in range(4):
        st = N.c_void_p()
        N.check(T.sox_stream_create(ctypes.byref(st)), "stream")
        x = rows_of(30 + i, rows, k, "f16")
        X, Y = Matrix(x, "f16"), Matrix(None, "f16", rows, n)
        W = Matrix(None, "i8", 1, lin.workspace(rows))
        q, scale = quantize(x)
        sides.append((st, X, Y, W, linear64(q, scale, w, ws, None, None, "none", "f16")))

    def work(st, X, Y, W, want):
        try:
            for _ in range(times):
                lin.run(X.ptr, rows, Y.ptr, "f16", workspace=W.ptr, workspace_bytes=lin.workspace(rows), stream=st)
            N.check(T.sox_stream_sync(st), "sync")
        except Exception as e:  # noqa: BLE001 (reported by the test's own thread)
            errors.append(e)
    print("[gpu] qlinear from threads", flush=True)
    threads = [threading.Thread(target=work, args=s) for s in sides]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    for st, X, Y, W, want in sides:
        check(Y.read(), *want)
        T.sox_stream_destroy(st)
        for m in (X, Y, W):
            m.free()
    lin.close()


TORCH = """
import sys
import torch  # before the backend's libraries: both then share one HIP runtime
sys.path.insert(0, {root!r})
import numpy as np
from simdonnx_amd.backend import HipBackend, HipBlockNorm, HipQuantLinear
hip = HipBackend.default()
torch.manual_seed(1)
k, n = 320, 200
lin = HipQuantLinear(hip, torch.randint(-127, 128, (k, n)).numpy(), None, k, n, scales=np.full(n, 1e-3, np.float32))
norm = HipBlockNorm(hip, k, post="rms", pre="layer")
assert torch.zeros(3, device="cuda").add(1).sum().item() == 3  # no error of the backend's is left for torch to find
for rows in (5, 300):
    x, r = (torch.randn(rows, k, device="cuda", dtype=torch.float16) for _ in range(2))
    h, y = torch.zeros_like(x), torch.zeros(rows, n, device="cuda", dtype=torch.float16)
    q, s = torch.zeros(rows, lin.pitch, device="cuda", dtype=torch.int8), torch.zeros(rows, device="cuda")

    def step():
        st = torch.cuda.current_stream().cuda_stream
        norm.run_quantized(r.data_ptr(), rows, q.data_ptr(), s.data_ptr(), x=x.data_ptr(), h=h.data_ptr(), stream=st)
        lin.run_quantized(q.data_ptr(), s.data_ptr(), rows, y.data_ptr(), stream=st)
    print("[gpu] torch capture", rows, flush=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        step()
    for rep in range(3):
        x.normal_()
        step()
        torch.cuda.synchronize()
        want = [t.clone() for t in (h, y, q, s)]
        for t in (h, y, q, s):
            t.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, (h, y, q, s))), rep
        assert y.abs().max().item() > 0
print("torch ok", flush=True)
"""


def test_beside_torch():
    """torch's tensors and streams in, and a graph that torch captures: in a process that loads torch first."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-u", "-c", TORCH.format(root=root)], capture_output=True, text=True, timeout=110)
    assert r.returncode == 0 and "torch ok" in r.stdout, r.stdout + r.stderr[-3000:]
