"""The norms around a transformer block (sox_block_norm_*, HipBlockNorm) against the same in 64 bits, on its own, with
8-bit outputs, and in the run it is made for: norm, 8-bit product, product, norm. Tolerances: tests/layers.py."""
import ctypes

import numpy as np
import pytest

from simdonnx_amd import native as N
from simdonnx_amd import synth
from simdonnx_amd.backend import HipBlockNorm, HipInferenceSession, HipQuantLinear
from simdonnx_amd.plan import PlanBuilder
from tests.layers import SMALL, UNIT, Matrix, block64, linear64, quantize, rounded

pytestmark = pytest.mark.gpu


def params(seed, c, post, pre, scale=True, **more):
    p = dict(post=post, pre=pre, **more)
    for i, k in enumerate(("post", "pre")):
        if p[k] != "none":
            p[k + "_gamma"] = synth.uniform(seed, 10 + i, (c,), 0.5, 1.5)
        if p[k] == "layer":
            p[k + "_beta"] = synth.uniform(seed, 20 + i, (c,), -0.5, 0.5)
    if scale:
        p["scale"] = synth.uniform(seed, 30, (c,), -0.5, 1.0)
    return p


def values(seed, which, rows, c, storage, mean=0.0):
    v = synth.normal(seed, which, (rows, c), 1.0) * np.exp2(np.arange(rows) % 5 - 2)[:, None].astype(np.float32) + np.float32(mean)
    v[:, ::61] *= 8
    return rounded(v, storage)


def inside(got, want, err, storage):
    u = UNIT[storage]
    tol = u * np.abs(want) + SMALL[storage] + err * (1 + u)
    over = np.abs(got.astype(np.float64) - want) - tol
    assert (over <= 0).all(), f"{(over > 0).sum()} of {over.size} values, worst {over.max():.3g} over its tolerance"


def inside8(q, scales, want, err, c):
    """8-bit rows of values known up to err: within half a step and that, next to the exact scale."""
    amax = np.abs(want).max(axis=1)
    worst = err.max(axis=1)
    assert (np.abs(scales - amax / 127) <= (worst + 3 * 2.0 ** -24 * amax) / 127 + 2.0 ** -149).all()
    step = np.maximum(amax, 1e-300)[:, None] / 127
    near = np.abs(q[:, :c] - want / step)
    assert (near <= 0.5 + (err + worst[:, None]) / step + 127 * 4 * 2.0 ** -24).all(), near.max()
    assert (q[:, c:] == 0).all()


def run_case(hip, seed, rows, c, storage, p, gate_rows=0, x=True, res=True, h=True, y=True, pad=0, skip=0, mean=0.0):
    X = Matrix(values(seed, 1, rows, c, storage, mean), storage, ld=c + pad, skip=skip) if x else None
    R = Matrix(values(seed, 2, rows, c, storage, mean), storage, ld=c + pad, skip=skip) if res else None
    G = Matrix(rounded(synth.normal(seed, 3, (gate_rows, c), 1.0), storage), storage, ld=c + pad, skip=skip) if gate_rows else None
    f = lambda m: None if m is None else m.read().astype(np.float64)  # noqa: E731
    wh, wy, eh, ey = block64(f(R), f(X), f(G), p, storage)
    norm = HipBlockNorm(hip, c, **p)
    H = Matrix(None, storage, rows, c, ld=c + pad, skip=skip)
    Y = Matrix(None, storage, rows, c, ld=c + pad, skip=skip)
    c16 = -(-c // 16) * 16
    Q = Matrix(None, "i8", rows, c16, ld=c16 + 16 * (pad % 3))
    S = Matrix(None, "f32", 1, rows)
    given = dict(ldr=R.ld if R else None, x=X.ptr if X else None, ldx=X.ld if X else None, gate=G.ptr if G else None,
                 ldg=G.ld if G else None, gate_rows=gate_rows or 1)
    rp = R.ptr if R else None
    norm.run(rp, rows, storage, h=H.ptr if h else None, ldh=H.ld, y=Y.ptr if y else None, ldy=Y.ld, **given)
    if h:
        inside(H.read(), wh, eh, storage)
    if y:
        inside(Y.read(), wy, ey, storage)
    first = H.read()
    H.refill()
    norm.run_quantized(rp, rows, Q.ptr, S.ptr, storage, h=H.ptr if h else None, ldh=H.ld, ldq=Q.ld, **given)
    assert np.array_equal(H.read(), first, equal_nan=True)
    inside8(Q.read().astype(np.float64), S.read()[0].astype(np.float64), wy, ey, c)
    for m in (X, R, G, H, Y, Q, S):
        if m is not None:
            m.free()
    norm.close()


KINDS = [("none", "rms"), ("rms", "rms"), ("layer", "layer"), ("none", "layer"), ("rms", "none"), ("layer", "rms")]


@pytest.mark.parametrize("storage", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("rows,c,pad,skip", [(1, 1, 0, 0), (1, 768, 0, 0), (3, 8, 0, 0), (5, 192, 8, 0), (9, 513, 0, 1), (4, 1024, 0, 0),
                                             (6, 1111, 5, 0), (3, 2048, 0, 0), (5, 2056, 16, 0), (2, 4096, 0, 0), (3, 4099, 0, 0),
                                             (2, 8192, 0, 0), (3, 8200, 0, 0), (2, 16384, 0, 0), (2, 16383, 0, 3),
                                             (3, 2304, 0, 0), (4, 2559, 3, 1), (2, 2560, 0, 0), (3, 2561, 7, 0), (3, 3500, 0, 0),
                                             (3, 6000, 0, 0), (2, 6140, 5, 1), (2, 6152, 0, 0), (2, 7001, 2, 0)])
def test_sizes(hip, storage, rows, c, pad, skip):
    """Every instance at both ends of its range, on 16-byte boundaries and off them."""
    print(f"[gpu] block norm {storage} {rows} x {c}", flush=True)
    kinds = KINDS[c % len(KINDS)]
    run_case(hip, c, rows, c, storage, params(c, c, *kinds, res_scale=0.75), gate_rows=rows, pad=pad, skip=skip)


@pytest.mark.parametrize("kinds", KINDS + [("none", "none")])
@pytest.mark.parametrize("gate,act", [(0, "none"), (1, "sigmoid"), (4, "swish"), (12, "gelu"), (12, "relu"), (2, "hardswish")])
def test_forms(hip, kinds, gate, act):
    print(f"[gpu] block norm {kinds} gate {gate} {act}", flush=True)
    run_case(hip, 40 + gate, 12, 200, "bf16", params(7, 200, *kinds, gate_act=act, scale=gate != 4), gate_rows=gate)
    run_case(hip, 41 + gate, 12, 203, "f32", params(7, 203, *kinds, gate_act=act, res_scale=-1.5), gate_rows=gate)


@pytest.mark.parametrize("kw", [dict(x=False), dict(res=False), dict(h=False), dict(y=False)])
def test_parts_left_out(hip, kw):
    print(f"[gpu] block norm {kw}", flush=True)
    run_case(hip, 50, 7, 320, "f16", params(8, 320, "rms", "layer", res_scale=0.5), **kw)


def test_more_rows_than_workgroups(hip):
    """Rows walked by one workgroup: one wave a row, a workgroup a row, and the widest."""
    for rows, c in ((9000, 64), (2500, 1100), (1300, 4104), (700, 8200)):
        print(f"[gpu] block norm {rows} x {c}", flush=True)
        run_case(hip, 60, rows, c, "bf16", params(9, c, "layer", "layer"), gate_rows=rows // 10)


@pytest.mark.parametrize("rows,c,pad", [(13001, 192, 0), (13001, 190, 3), (7003, 512, 0), (7003, 391, 0), (5002, 768, 8), (5002, 1023, 0),
                                        (1207, 2304, 0), (1207, 2450, 1), (1100, 1536, 0), (701, 5000, 3), (601, 6500, 0), (601, 7003, 1)])
def test_rows_past_one_round(hip, rows, c, pad):
    """More rows than a launch holds at once, and not a multiple of a workgroup's."""
    print(f"[gpu] block norm {rows} x {c} + {pad}", flush=True)
    run_case(hip, rows, rows, c, "f16", params(c, c, "rms", "layer", gate_act="sigmoid"), gate_rows=1, pad=pad)


@pytest.mark.parametrize("storage", ["f32", "bf16"])
@pytest.mark.parametrize("rows,c,pad,skip", [(5003, 192, 0, 0), (5003, 256, 4, 0), (5003, 189, 0, 1), (3001, 257, 0, 0), (3001, 512, 0, 0),
                                             (3001, 391, 3, 0), (2050, 513, 0, 0), (2050, 768, 8, 0), (2050, 1023, 0, 1), (1024, 1024, 0, 0)])
def test_many_rows(hip, storage, rows, c, pad, skip):
    """The instances for many rows in the other types than fp16, at both ends of their ranges."""
    print(f"[gpu] block norm {storage} {rows} x {c} + {pad}", flush=True)
    kinds = KINDS[(rows + c) % len(KINDS)]
    run_case(hip, rows + c, rows, c, storage, params(c, c, *kinds, gate_act="swish"), gate_rows=rows if c % 2 else 1, pad=pad, skip=skip)


def test_hardswish_next_to_its_zero(hip):
    """v clip((v + 3) / 6, 0, 1) keeps its digits where it leaves zero: four roundings (the sum, the sixth, two products) of half
    a unit each, h being the gate alone; 5 units leave room for their products."""
    c = 2048
    g = np.concatenate([-3 + 2.0 ** -22 * np.arange(-100, 700), -3 + 2.0 ** -np.arange(1, 21.0), 3 + 2.0 ** -22 * np.arange(-200, 200),
                        np.linspace(-8, 8, 828)]).astype(np.float32)[None]
    assert g.size == c
    norm = HipBlockNorm(hip, c, pre="none", gate_act="hardswish")
    X, G, H = Matrix(np.ones((1, c)), "f32"), Matrix(g, "f32"), Matrix(None, "f32", 1, c)
    print("[gpu] block norm hardswish", flush=True)
    norm.run(None, 1, "f32", x=X.ptr, gate=G.ptr, h=H.ptr)
    v = g.astype(np.float64)
    want = v * np.clip((v + 3) / 6, 0, 1)
    assert (np.abs(H.read() - want) <= 5 * 2.0 ** -24 * np.abs(want)).all()
    for m in (X, G, H):
        m.free()
    norm.close()


def test_large_means(hip):
    """Rows far from zero: the variance comes from the deviations, not from a difference of squares."""
    print("[gpu] block norm large means", flush=True)
    run_case(hip, 70, 8, 768, "f32", params(10, 768, "layer", "layer", scale=False), mean=1000.0)
    run_case(hip, 71, 8, 2000, "f32", params(10, 2000, "none", "layer", scale=False), x=False, mean=-3000.0)


def test_quantizes_alone(hip):
    """Without norms, branch and scales: the residual's exact 8-bit rows."""
    for storage in ("f16", "bf16"):
        x = values(80, 1, 50, 333, storage)
        x[4] = 0
        norm = HipBlockNorm(hip, 333, pre="none")
        X, Q, S = Matrix(x, storage), Matrix(None, "i8", 50, 336), Matrix(None, "f32", 1, 50)
        print(f"[gpu] block norm to 8 bits {storage}", flush=True)
        norm.run_quantized(X.ptr, 50, Q.ptr, S.ptr, storage, ldq=336)
        q, scale = quantize(x)
        assert np.array_equal(Q.read()[:, :333], q) and np.array_equal(S.read()[0], scale.astype(np.float32))
        for m in (X, Q, S):
            m.free()
        norm.close()


def test_rows_that_are_not_finite(hip):
    """A NaN or an infinity stays in its row; zeros have a norm; 8-bit rows of it are zeros with a NaN scale."""
    c, rows = 300, 9
    x, r = values(90, 1, rows, c, "f32"), values(90, 2, rows, c, "f32")
    x[1, 7] = np.nan
    r[3, 299] = np.inf
    x[5] = r[5] = 0
    p = params(11, c, "rms", "layer")
    norm = HipBlockNorm(hip, c, **p)
    X, R, H, Y = Matrix(x, "f32"), Matrix(r, "f32"), Matrix(None, "f32", rows, c), Matrix(None, "f32", rows, c)
    Q, S = Matrix(None, "i8", rows, 304), Matrix(None, "f32", 1, rows)
    print("[gpu] block norm not finite", flush=True)
    norm.run(R.ptr, rows, "f32", x=X.ptr, h=H.ptr, y=Y.ptr)
    norm.run_quantized(R.ptr, rows, Q.ptr, S.ptr, "f32", x=X.ptr, ldq=304)
    h, y, q, s = H.read(), Y.read(), Q.read(), S.read()[0]
    bad = [1, 3]
    good = [i for i in range(rows) if i not in bad]
    assert np.isnan(h[1]).all() and h[3, 299] == np.inf and np.isfinite(h[3, :299]).all()
    assert np.isnan(y[bad]).all() and np.isnan(s[bad]).all() and (q[bad] == 0).all()
    wh, wy, eh, ey = block64(r[good].astype(np.float64), x[good].astype(np.float64), None, p, "f32")
    inside(h[good], wh, eh, "f32")
    inside(y[good], wy, ey, "f32")
    inside8(q[good].astype(np.float64), s[good].astype(np.float64), wy, ey, c)
    for m in (X, R, H, Y, Q, S):
        m.free()
    norm.close()


@pytest.mark.parametrize("rows,c", [(40, 192), (5, 3000), (600, 7000)])
def test_in_place(hip, rows, c):
    """The residual stream updated where it stands, and the branch's buffer taking y."""
    x, r = values(100, 1, rows, c, "bf16"), values(100, 2, rows, c, "bf16")
    p = params(12, c, "rms", "rms")
    wh, wy, eh, ey = block64(r.astype(np.float64), x.astype(np.float64), None, p, "bf16")
    norm = HipBlockNorm(hip, c, **p)
    X, R = Matrix(x, "bf16"), Matrix(r, "bf16")
    print(f"[gpu] block norm in place {rows} x {c}", flush=True)
    norm.run(R.ptr, rows, "bf16", x=X.ptr, h=R.ptr, y=X.ptr)
    inside(R.read(), wh, eh, "bf16")
    inside(X.read(), wy, ey, "bf16")
    for m in (X, R):
        m.free()
    norm.close()


def test_transformer_mlp_in_8_bits(hip):
    """A session's features through a block's second half as a model runs it, on the session's stream: residual, norm to
    8-bit rows, product with GELU, product, norm with gate and layer scale into the next block's 8-bit rows, and that
    block's projection. Each step against the 64-bit step of the inputs that the device had; captured into one graph, the
    run gives the same bits on three replays."""
    rows, c, hidden = 150, 192, 768
    storage = "f16"
    feats = rounded(synth.normal(200, 1, (rows, c), 1.0), storage)
    pb = PlanBuilder()
    v = pb.input(feats.shape, None, "features")
    out = pb.unary("Copy", v, name="copy")
    T = N.thin()
    with HipInferenceSession(hip.graph(pb.build(out), storage)) as session:
        session.set_input(feats)
        print("[gpu] 8-bit block: session", flush=True)
        session.run()
        stream = N.backend().sox_session_stream(session.h)
        p = N.c_void_p()
        N.check(N.backend().sox_session_value_ptr(session.h, out, ctypes.byref(p)), "value_ptr")
        residual = p.value
        attn = Matrix(values(201, 1, rows, c, storage), storage, stream=stream)
        gate = Matrix(rounded(synth.normal(201, 2, (3, c), 1.0), storage), storage, stream=stream)
        p1 = params(202, c, "none", "layer")
        p2 = params(203, c, "rms", "rms", gate_act="sigmoid")
        w1, w2, w3 = (synth.normal(204, i, s, 0.05) for i, s in enumerate([(c, hidden), (hidden, c), (c, 3 * c)]))
        b1, b2 = synth.uniform(205, 1, (hidden,), -0.2, 0.2), synth.uniform(205, 2, (c,), -0.2, 0.2)
        n1, n2 = HipBlockNorm(hip, c, **p1), HipBlockNorm(hip, c, **p2)
        fc1, fc2, qkv = HipQuantLinear(hip, w1, b1, c, hidden), HipQuantLinear(hip, w2, b2, hidden, c), HipQuantLinear(hip, w3, None, c, 3 * c)
        mk = lambda cols, st=storage, r=rows: Matrix(None, st, r, cols, stream=stream)  # noqa: E731
        H1, F1, F2, H2, Z = mk(c), mk(hidden), mk(c), mk(c), mk(3 * c)
        Q1, Q2, S1, S2 = mk(n1.channels, "i8"), mk(c, "i8"), mk(rows, "f32", 1), mk(rows, "f32", 1)
        W = Matrix(None, "i8", 1, max(1, fc2.workspace(rows)), stream=stream)

        def block():
            n1.run_quantized(residual, rows, Q1.ptr, S1.ptr, storage, x=attn.ptr, h=H1.ptr, ldq=Q1.ld, stream=stream)
            fc1.run_quantized(Q1.ptr, S1.ptr, rows, F1.ptr, storage, ldq=Q1.ld, act="gelu", stream=stream)
            fc2.run(F1.ptr, rows, F2.ptr, storage, workspace=W.ptr, workspace_bytes=fc2.workspace(rows), stream=stream)
            n2.run_quantized(H1.ptr, rows, Q2.ptr, S2.ptr, storage, x=F2.ptr, gate=gate.ptr, gate_rows=3, h=H2.ptr, ldq=Q2.ld,
                             stream=stream)
            qkv.run_quantized(Q2.ptr, S2.ptr, rows, Z.ptr, storage, ldq=Q2.ld, stream=stream)

        print("[gpu] 8-bit block: eager", flush=True)
        block()
        every = (H1, F1, F2, H2, Z, Q1, Q2, S1, S2)
        got = [m.read() for m in every]
        d = [g.astype(np.float64) for g in got]
        h1, f1, f2, h2, z, q1, q2, s1, s2 = d

        def linear(q, s, w, b, act, y):
            wq, ws = quantize(w.T)
            want, tol = linear64(q, s, wq.T, ws.astype(np.float32), b, None, act, storage)
            assert (np.abs(y - want) <= tol).all()

        wh, wy, eh, ey = block64(feats.astype(np.float64), attn.read().astype(np.float64), None, p1, storage)
        inside(got[0], wh, eh, storage)
        inside8(q1, s1[0], wy, ey, c)
        linear(q1, s1[0], w1, b1, "gelu", f1)
        linear(*quantize(f1), w2, b2, "none", f2)
        wh, wy, eh, ey = block64(h1, f2, gate.read().astype(np.float64), p2, storage)
        inside(got[3], wh, eh, storage)
        inside8(q2, s2[0], wy, ey, c)
        linear(q2, s2[0], w3, None, "none", z)

        print("[gpu] 8-bit block: captured", flush=True)
        N.check(T.sox_graph_begin(stream), "capture")
        block()
        ex = N.c_void_p()
        N.check(T.sox_graph_end(stream, ctypes.byref(ex)), "capture end")
        for rep in range(3):
            block()  # eager work between the replays
            for m in every:
                m.refill()
            N.check(T.sox_graph_launch(ex, stream), "replay")
            N.check(T.sox_stream_sync(stream), "sync")
            for m, g in zip(every, got):
                assert np.array_equal(m.read(), g), rep
        T.sox_graph_destroy(ex)
        for m in every + (attn, gate, W):
            m.free()
        for o in (n1, n2, fc1, fc2, qkv):
            o.close()
