"""The 8-bit layers as nodes of a plan: one product against 64 bits, and a gated transformer block against the same layers
called one by one, bit for bit (whole-number sums and per-row statistics do not depend on who launches them)."""
import numpy as np
import pytest

from simdonnx_amd.backend import HipBlockNorm, HipInferenceSession, HipQuantLinear, HipUnitRunner
from simdonnx_amd.native import SoxError
from simdonnx_amd.plan import PlanBuilder
from tests.layers import Matrix, linear64, quantize, rounded

pytestmark = pytest.mark.gpu
STORAGE = {"f32": False, "f16": True, "bf16": "bf16"}


def rng(seed):
    return np.random.default_rng(seed)


@pytest.mark.parametrize("storage", list(STORAGE))
@pytest.mark.parametrize("rows,k,n", [(1, 64, 48), (1, 1, 1), (7, 100, 33), (40, 1030, 130), (300, 192, 576), (2, 4100, 64)])
def test_product(hip, storage, rows, k, n):
    r = rng(rows * 31 + k)
    x = rounded(r.normal(size=(rows, k)), storage)
    res = rounded(r.normal(size=(rows, n)), storage)
    w, b = r.normal(size=(k, n)).astype(np.float32), r.normal(size=n).astype(np.float32)
    pb = PlanBuilder()
    xv, rv = pb.input((rows, k)), pb.input((rows, n))
    plan = pb.build(pb.quant_linear(xv, w, b, residual=rv, act="gelu"))
    print(f"[gpu] quant_linear {rows}x{k}x{n} {storage}", flush=True)
    q, s = quantize(x)
    wq, ws = quantize(w.T)
    want, tol = linear64(q, s, wq.T, ws, b.astype(np.float64), res.astype(np.float64), "gelu", storage)
    with HipInferenceSession(hip.graph(plan, STORAGE[storage])) as sess:
        for _ in range(3):
            sess.set_input(x, 0)
            sess.set_input(res, 1)
            got = sess.run().reshape(rows, n)
            assert (np.abs(got - want) <= tol).all()


class Block:
    """norm -> product, GELU -> product -> post norm, gate, residual, norm -> product with the residual."""

    def __init__(self, seed, b, t, c, f):
        r = rng(seed)
        g = lambda *s: r.normal(size=s).astype(np.float32)  # noqa: E731
        self.b, self.t, self.c = b, t, c
        self.w1, self.b1, self.w2, self.b2, self.w3 = g(c, f), g(f), g(f, c), g(c), g(c, c)
        self.first = dict(pre="layer", pre_gamma=1 + 0.1 * g(c), pre_beta=g(c))
        self.second = dict(post="rms", post_gamma=1 + 0.1 * g(c), scale=g(c), pre="rms", pre_gamma=1 + 0.1 * g(c),
                           res_scale=0.5, gate_act="sigmoid")

    def inputs(self, seed, storage):
        r = rng(seed)
        return (rounded(r.normal(size=(self.b * self.t, self.c)), storage), rounded(r.normal(size=(self.b, self.c)), storage))

    def plan(self):
        pb = PlanBuilder()
        x, gate = pb.input((self.b, self.t, self.c)), pb.input((self.b, 1, self.c))
        _, y = pb.block_norm(residual=x, h=False, **self.first)
        m = pb.quant_linear(pb.quant_linear(y, self.w1, self.b1, act="gelu"), self.w2, self.b2)
        h, y = pb.block_norm(residual=x, x=m, gate=gate, **self.second)
        return pb.build(pb.quant_linear(y, self.w3, residual=h, act="swish"))

    def by_calls(self, hip, x, gate, storage, handed):
        rows, c = x.shape
        f = self.w1.shape[1]
        n1, n2 = HipBlockNorm(hip, c, **self.first), HipBlockNorm(hip, c, **self.second)
        l1, l2, l3 = HipQuantLinear(hip, self.w1, self.b1, c, f), HipQuantLinear(hip, self.w2, self.b2, f, c), HipQuantLinear(hip, self.w3, None, c, c)
        need = max(lin.workspace(rows) for lin in (l1, l2, l3))
        m = lambda cols, kind=storage, n=rows: Matrix(storage=kind, rows=n, cols=cols)  # noqa: E731
        X, G, Y, A, B, H, Z = Matrix(x, storage), Matrix(gate, storage), m(c), m(f), m(c), m(c), m(c)
        Q, S, W = m(c, "i8"), m(rows, "f32", 1), m(max(need, 16), "i8", 1)
        st = storage
        ws = dict(workspace=W.ptr, workspace_bytes=need)
        if handed:
            n1.run_quantized(X.ptr, rows, Q.ptr, S.ptr, st, ldr=c, ldq=c)
            l1.run_quantized(Q.ptr, S.ptr, rows, A.ptr, st, c, f, act="gelu")
        else:
            n1.run(X.ptr, rows, st, c, y=Y.ptr, ldy=c)
            l1.run(Y.ptr, rows, A.ptr, st, c, f, act="gelu", **ws)
        l2.run(A.ptr, rows, B.ptr, st, f, c, **ws)
        tail = dict(x=B.ptr, ldx=c, gate=G.ptr, ldg=c, gate_rows=len(gate), h=H.ptr, ldh=c)
        if handed:
            n2.run_quantized(X.ptr, rows, Q.ptr, S.ptr, st, ldr=c, ldq=c, **tail)
            l3.run_quantized(Q.ptr, S.ptr, rows, Z.ptr, st, c, c, act="swish", residual=H.ptr, ldr=c)
        else:
            n2.run(X.ptr, rows, st, c, y=Y.ptr, ldy=c, **tail)
            l3.run(Y.ptr, rows, Z.ptr, st, c, c, act="swish", residual=H.ptr, ldr=c, **ws)
        got = Z.read()
        for o in (n1, n2, l1, l2, l3):
            o.close()
        for o in (X, G, Y, A, B, H, Z, Q, S, W):
            o.free()
        return got


@pytest.mark.parametrize("handed", [True, False], ids=["8-bit rows", "storage rows"])
@pytest.mark.parametrize("storage", list(STORAGE))
@pytest.mark.parametrize("b,t,c,f", [(1, 1, 64, 128), (2, 7, 192, 384), (3, 50, 96, 200), (1, 33, 1040, 72), (2, 400, 768, 2304)])
def test_block(hip, b, t, c, f, storage, handed, monkeypatch):
    if not handed:
        monkeypatch.setenv("SIMDONNX_HIP_NO_QUANT_NORM", "1")
    print(f"[gpu] block {b}x{t}x{c} {f} {storage} handed={handed}", flush=True)
    block = Block(b + t, b, t, c, f)
    with HipInferenceSession(hip.graph(block.plan(), STORAGE[storage])) as s:
        for seed in range(3):
            x, gate = block.inputs(seed, storage)
            s.set_input(x, 0)
            s.set_input(gate, 1)
            got = s.run().reshape(x.shape)
            assert np.array_equal(got, block.by_calls(hip, x, gate, storage, handed))


@pytest.mark.parametrize("b,t,c,f", [(2, 8, 4096, 64), (1, 30, 192, 384), (2, 300, 768, 520)])
def test_replayed_session(hip, b, t, c, f):
    """The captured list of dispatches gives each run's own results: tokens whose rows fill the LDS, panels, the ring."""
    print(f"[gpu] replay {b}x{t}x{c} {f}", flush=True)
    block = Block(b * t, b, t, c, f)
    with HipInferenceSession(hip.graph(block.plan(), True)) as s, HipInferenceSession(hip.graph(block.plan(), True)) as eager:
        s.set_replay(True)
        for seed in range(4):
            outs = []
            for sess in (s, eager):
                for i, v in enumerate(block.inputs(seed, "f16")):
                    sess.set_input(v, i)
                outs.append(sess.run().copy())
            assert np.array_equal(*outs)


def test_handed_rows_are_not_read_as_elements(hip, monkeypatch):
    """A session gives out a norm's y, but not where it holds 8-bit rows."""
    def session():
        pb = PlanBuilder()
        x = pb.input((20, 64))
        h, y = pb.block_norm(residual=x, pre="none")
        z = pb.quant_linear(y, np.eye(64, dtype=np.float32), residual=h)
        return HipInferenceSession(hip.graph(pb.build(z), True)), h, y

    x = rounded(rng(1).normal(size=(20, 64)), "f16")
    for kept in (False, True):
        if kept:
            monkeypatch.setenv("SIMDONNX_HIP_NO_QUANT_NORM", "1")
        s, h, y = session()
        with s:
            s.set_input(x, 0)
            s.run()
            assert np.array_equal(s.read_value(h).reshape(x.shape), x)
            if kept:
                assert np.array_equal(s.read_value(y).reshape(x.shape), x)
            else:
                with pytest.raises(SoxError, match="8-bit rows"):
                    s.read_value(y)


def test_odd_block(hip):
    """100 channels: not a multiple of 16, so the norm keeps storage rows."""
    block = Block(5, 2, 20, 100, 60)
    x, gate = block.inputs(1, "f16")
    with HipInferenceSession(hip.graph(block.plan(), True)) as s:
        s.set_input(x, 0)
        s.set_input(gate, 1)
        assert np.array_equal(s.run().reshape(x.shape), block.by_calls(hip, x, gate, "f16", False))


def test_outputs_over_operands(hip):
    """A plan that puts every output of the block's tail where its operands live."""
    r = rng(3)
    x, w = rounded(r.normal(size=(70, 64)), "f16"), r.normal(size=(64, 64)).astype(np.float32)

    def plan(over):
        pb = PlanBuilder()
        xv = pb.input((70, 64))
        h, y = pb.block_norm(residual=xv, x=xv, post="layer")
        z = pb.quant_linear(y, w, residual=h)
        p = pb.build(z)
        if over:
            for v in (h, y, z):
                p.buf_offset[p.values[v].buf] = p.buf_offset[p.values[xv].buf]
        return p

    out = []
    for over in (False, True):
        with HipInferenceSession(hip.graph(plan(over), True)) as s:
            s.set_input(x, 0)
            out.append(s.run().copy())
    assert np.array_equal(*out)


def test_units_side_by_side(hip):
    """Units of one wave, each with its own arena and scratch, on two streams."""
    r = rng(9)
    w = r.normal(size=(96, 80)).astype(np.float32)
    rows = [300, 1, 45, 700]
    xs = [rounded(r.normal(size=(n, 96)), "f16") for n in rows]
    graphs = []
    for n in rows:
        pb = PlanBuilder()
        xv = pb.input((n, 96))
        _, y = pb.block_norm(residual=xv, pre="rms", h=False)
        graphs.append(hip.graph(pb.build(pb.quant_linear(pb.quant_linear(y, w, act="relu"), w.T.copy())), True))
    alone = []
    for g, x in zip(graphs, xs):
        with HipInferenceSession(g) as s:
            s.set_input(x, 0)
            alone.append(s.run().copy().reshape(x.shape))
    run = HipUnitRunner(hip, streams=2)
    ids = [run.add(g) for g in graphs]
    run.cut()
    for _ in range(3):
        for i, x in zip(ids, xs):
            run.input(i)[:] = x.reshape(-1)
        run.submit()
        run.wait(0)
        for i, a in zip(ids, alone):
            assert np.array_equal(run.output(i).reshape(a.shape), a)
    run.close()


@pytest.mark.parametrize("tail", ["mlp residual", "projected", "projection residual"])
@pytest.mark.parametrize("storage", ["f16", "bf16"])
def test_norm_rows_in_fused_nodes(hip, tail, storage, monkeypatch):
    """A norm's y that a product reads and that a fused MLP's or projection's kernel reads as well: the bits of the norm,
    the product and the MLP as plans of their own."""
    r = rng(21)
    rows, c, hidden = 100, 192, 768
    g = lambda *s: (r.normal(size=s) / np.sqrt(s[0])).astype(np.float32)  # noqa: E731
    wq, w1, w2, wp, b1, b2 = g(c, c), g(c, hidden), g(hidden, c), g(c, c), g(hidden), g(c)
    x, s = (rounded(r.normal(size=(rows, c)), storage) for _ in range(2))

    def norm(pb, v):
        return pb.block_norm(residual=v, h=False)[1]

    def mlp(pb, y, v):
        res = y
        if tail != "mlp residual":
            res = v = pb.add(pb.gemm(y if tail == "projected" else v, wp, b2), v if tail == "projected" else y)
        m = pb.gemm(pb.layer_norm(v, np.ones(c, np.float32), np.zeros(c, np.float32)), w1, b1, act="gelu")
        return pb.add(pb.gemm(m, w2, b2), res)

    def run(build, *inputs):
        pb = PlanBuilder()
        plan = pb.build(build(pb, *[pb.input((rows, c)) for _ in inputs]))
        with HipInferenceSession(hip.graph(plan, STORAGE[storage])) as sess:
            for i, v in enumerate(inputs):
                sess.set_input(v, i)
            return sess.run().reshape(rows, c).copy()

    def whole(pb, xv, sv):
        y = norm(pb, xv)
        return pb.add(pb.quant_linear(y, wq), mlp(pb, y, sv))

    print(f"[gpu] norm beside a fused MLP, {tail} {storage}", flush=True)
    got = run(whole, x, s)
    y = run(norm, x)
    z, out = run(lambda pb, v: pb.quant_linear(v, wq), y), run(mlp, y, s)
    assert np.array_equal(got, rounded(z + out, storage))
    monkeypatch.setenv("SIMDONNX_HIP_NO_QUANT_NORM", "1")
    assert np.array_equal(run(whole, x, s), got)


@pytest.mark.parametrize("storage", list(STORAGE))
@pytest.mark.parametrize("off", [1, 4, 6])
def test_norm_rows_off_16_byte_boundaries(hip, storage, off):
    """A plan whose arena puts a norm's y on any element: the bits of the same plan on a boundary. The y are 16-bit values, in
    fp32 too, which norm and product bring to 8 bits alike, exactly."""
    r = rng(off)
    x, w = rounded(r.normal(size=(70, 64)), "bf16" if storage == "f32" else storage), r.normal(size=(64, 48)).astype(np.float32)

    def run(off):
        pb = PlanBuilder()
        _, y = pb.block_norm(residual=pb.input((70, 64)), pre="none", h=False)
        p = pb.build(pb.quant_linear(y, w, act="relu"))
        p.buf_offset[p.values[y].buf] = p.arena_floats + off
        p.arena_floats += 70 * 64 + off
        print(f"[gpu] norm at element {off} {storage}", flush=True)
        with HipInferenceSession(hip.graph(p, STORAGE[storage])) as s:
            s.set_input(x, 0)
            return s.run().copy()

    assert np.array_equal(run(off), run(0))


@pytest.mark.parametrize("fusion", ["residual add", "layer norm", "mlp"])
def test_views_of_fused_values(hip, fusion):
    """A product that reads a view of a value which a fusion would not store: the bits of two plans, one after the other."""
    r = rng(31)
    g = lambda *s: (r.normal(size=s) / np.sqrt(s[0])).astype(np.float32)  # noqa: E731
    rows, k, n = {"residual add": (128, 64, 64), "layer norm": (128, 64, 64), "mlp": (128, 192, 768)}[fusion]
    x = rounded(r.normal(size=(rows, k)), "f16")
    gamma, beta, w1, b1, w2, b2, wq = 1 + 0.1 * g(k), g(k), g(k, n), g(n), g(n, k), g(k), g(n, 48)

    def value(pb, v):
        if fusion == "residual add":
            y = pb.gemm(v, w1, b1)
            pb.add(y, v)
        elif fusion == "layer norm":
            y = pb.layer_norm(v, gamma, beta)
            pb.gemm(y, w1, b1)
        else:
            y = pb.gemm(pb.layer_norm(v, gamma, beta), w1, b1, act="gelu")
            pb.add(pb.gemm(y, w2, b2), v)
        return y

    def run(build, v):
        pb = PlanBuilder()
        plan = pb.build(build(pb, pb.input(v.shape)))
        with HipInferenceSession(hip.graph(plan, True)) as s:
            s.set_input(v, 0)
            return s.run().copy()

    print(f"[gpu] view of a fused value: {fusion}", flush=True)
    got = run(lambda pb, v: pb.quant_linear(pb.alias(value(pb, v), (2, rows // 2, n)), wq), x)
    y = run(value, x).reshape(rows, n)
    assert np.array_equal(got.reshape(rows, 48), run(lambda pb, v: pb.quant_linear(v, wq), y).reshape(rows, 48))
