"""The 8-bit layers as nodes of a plan, lowered by an offline backend: which dispatches a plan becomes, outputs that a plan
put over an operand, and the nodes that are refused."""
import ctypes
import os
import subprocess
import sys

import numpy as np
import pytest

from simdonnx_amd import native as N
from simdonnx_amd.backend import HipBackend
from simdonnx_amd.plan import NHWC, PlanBuilder
from tests.layers import PANELS

ROWS, C, K = 100, 64, 48


@pytest.fixture(scope="module")
def offline():
    b = HipBackend.offline()
    yield b
    b.close()


def weights(k=C, n=K):
    return np.linspace(-1, 1, k * n, dtype=np.float32).reshape(k, n)


def labels(backend, plan, storage=True):
    return [d[0] for d in backend.graph(plan, storage).dispatches]


def test_records():
    assert ctypes.sizeof(N.QuantLinearP) == 12 and ctypes.sizeof(N.BlockNormNodeP) == 4 * 8


@pytest.mark.parametrize("storage", [False, True, "bf16"])
def test_norm_hands_8_bit_rows(offline, storage, monkeypatch):
    """Two products of one norm: it rounds once for both; without the handing-over each rounds its rows itself."""
    def plan(c=C):
        pb = PlanBuilder()
        x = pb.input((ROWS, c))
        _, y = pb.block_norm(residual=x, h=False)
        a, b = pb.quant_linear(y, weights(c)), pb.quant_linear(y, weights(c))
        return pb.build(pb.add(a, b))

    def products(p):
        with_rows = labels(offline, p, storage)
        assert with_rows[0] == "block_norm" and with_rows.count("quant_linear") == 2
        return with_rows.count("quant_rows")

    monkeypatch.setenv("SIMDONNX_HIP_QGEMM", "64x64_w4k128s4")  # (a tiling: its floating rows need a launch of their own)
    assert products(plan()) == 0
    assert products(plan(56)) == 2  # not a multiple of 16
    monkeypatch.setenv("SIMDONNX_HIP_NO_QUANT_NORM", "1")
    assert products(plan()) == 2


def test_norm_keeps_its_rows_for_others(offline, monkeypatch):
    """A y that something else reads, as a residual, a view or the plan's output, stays in storage elements."""
    monkeypatch.setenv("SIMDONNX_HIP_QGEMM", "64x64_w4k128s4")

    def rows(use):
        pb = PlanBuilder()
        x = pb.input((ROWS, C))
        _, y = pb.block_norm(residual=x, h=False)
        return labels(offline, pb.build(use(pb, y))).count("quant_rows")

    w = weights(C, C)
    assert rows(lambda pb, y: pb.quant_linear(y, w)) == 0
    assert rows(lambda pb, y: pb.quant_linear(y, w, residual=y)) == 1
    assert rows(lambda pb, y: pb.add(pb.quant_linear(y, w), y)) == 1
    assert rows(lambda pb, y: pb.quant_linear(pb.alias(y, (2, ROWS // 2, C)), w)) == 1

    def output(pb, y):
        pb.quant_linear(y, w)
        return y
    assert rows(output) == 1


def mlp_after(pb, y, tail):
    """A transformer MLP that runs as one kernel, and where y comes into it."""
    ones, zeros = np.ones(192, np.float32), np.zeros(192, np.float32)

    def mlp(x, res):
        m = pb.gemm(pb.layer_norm(x, ones, zeros), weights(192, 768), np.zeros(768, np.float32), act="gelu")
        return pb.add(pb.gemm(m, weights(768, 192), zeros), res)

    s = pb.input((ROWS, 192))
    if tail == "mlp residual":
        return mlp(s, y)
    o, r = (y, s) if tail == "projected" else (s, y)
    x = pb.add(pb.gemm(o, weights(192, 192), zeros), r)
    return mlp(x, x)


@pytest.mark.parametrize("storage", [True, "bf16"])
@pytest.mark.parametrize("tail", ["mlp residual", "projected", "projection residual"])
def test_norm_keeps_its_rows_for_fused_nodes(offline, tail, storage, monkeypatch):
    """A y that a fused MLP's or projection's kernel reads, through nodes folded into it, stays in storage elements."""
    monkeypatch.setenv("SIMDONNX_HIP_QGEMM", "64x64_w4k128s4")  # (its floating rows need a launch of their own)

    pb = PlanBuilder()
    _, y = pb.block_norm(residual=pb.input((ROWS, 192)), h=False)
    z = pb.quant_linear(y, weights(192, 192))
    g = offline.graph(pb.build(pb.add(z, mlp_after(pb, y, tail))), storage)
    at, size = g.value_place(y)
    names = [d[0] for d in g.dispatches]
    reads = [(n, b[2]) for i, n in enumerate(names) for b in g.binds(i) if b[0] == N.SLOT_ARENA and b[1] == at]
    assert any(n.startswith("mlp") for n in names) and not any(n == "gemm" for n in names), names  # (folded)
    assert ("block_norm", size) in reads and ("quant_rows", size) in reads, reads
    assert len(reads) >= 3 and all(n == size for _, n in reads), reads


@pytest.mark.parametrize("storage", [False, True])
def test_norm_keeps_its_rows_off_16_byte_boundaries(offline, storage, monkeypatch):
    """8-bit rows are stored and read 8 and 16 bytes at a time: not in a buffer that the plan put off such a boundary."""
    monkeypatch.setenv("SIMDONNX_HIP_QGEMM", "64x64_w4k128s4")
    for off in range(9):
        pb = PlanBuilder()
        x = pb.input((ROWS, C))
        _, y = pb.block_norm(residual=x, h=False)
        p = pb.build(pb.quant_linear(y, weights(C, C)))
        p.buf_offset[p.values[y].buf] = p.arena_floats + off
        p.arena_floats += ROWS * C + off
        g = offline.graph(p, storage)
        boundary = g.value_place(y)[0] % 16 == 0
        assert boundary == (off % (8 if storage else 4) == 0)
        assert [d[0] for d in g.dispatches].count("quant_rows") == (0 if boundary else 1)


def test_handed_rows_are_not_bound_as_elements(offline, capsys):
    """An extension operator that names a norm's y outside of its node's inputs gets an error where it holds 8-bit rows."""
    seen = []

    def emit(g, node):
        seen.append(None)
        seen[-1] = g.bind(N.c_int32.from_buffer_copy(g.node(node)[1]).value)

    offline.register_ext("ReadsAnother", emit)

    def lower(named):
        pb = PlanBuilder()
        x = pb.input((ROWS, C))
        h, y = pb.block_norm(residual=x)
        z = pb.quant_linear(y, weights(C, C))
        e = pb.ext("ReadsAnother", [z], (ROWS, C), bytes(N.c_int32({"h": h, "y": y}[named])))
        return offline.graph(pb.build(e), True)

    lower("h")
    assert seen[-1].size == ROWS * C * 2
    with pytest.raises(N.SoxError, match="ReadsAnother emit failed"):
        lower("y")
    assert seen[-1] is None and "8-bit rows" in capsys.readouterr().out


@pytest.mark.parametrize("storage", ["f32", "f16", "bf16"])
def test_panels_take_moderate_numbers_of_rows(offline, storage):
    """The shapes by which the panel kernel is tested run on it, each instance among them."""
    taken = set()
    for rows, k, n in PANELS:
        pb = PlanBuilder()
        plan = pb.build(pb.quant_linear(pb.input((rows, k)), weights(k, n)))
        name = f"sox_qpanel_{storage}_c{-(-k // 256)}"
        assert offline.graph(plan, storage != "f32" and storage).kernels == [name], (rows, k, n)
        taken.add(name)
    assert len(taken) == 4


def plan_over(at, outs):
    """A plan whose arena puts the values `outs` where `at` says (elements)."""
    pb = PlanBuilder()
    x = pb.input((ROWS, C))
    h, y = pb.block_norm(residual=x, x=x)
    z = pb.quant_linear(y, weights(C, C), residual=h)
    p = pb.build(z)
    ids = dict(x=x, h=h, y=y, z=z)
    for name in outs:
        p.buf_offset[p.values[ids[name]].buf] = at
    return p, ids


@pytest.mark.parametrize("outs", ["h", "y", "z", "hy", "yz", "hyz"])
def test_outputs_over_operands_move(offline, outs):
    p, ids = plan_over(0, outs)
    g = offline.graph(p, True)
    assert [d[0] for d in g.dispatches][0] == "block_norm"
    place = {k: g.value_place(v) for k, v in ids.items()}  # (bytes, size)
    for out, others in (("h", "xy"), ("y", "xh"), ("z", "yh")):
        for o in others:
            a, b = place[out], place[o]
            assert a[0] + a[1] <= b[0] or b[0] + b[1] <= a[0], (out, o)
    assert max(a + n for a, n in place.values()) <= g.arena_bytes
    for i in range(len(g.dispatches)):
        for slot, off, size in g.binds(i):
            assert slot != N.SLOT_ARENA or off + size <= g.arena_bytes


def refused(match, backend, build, storage=True):
    pb = PlanBuilder()
    with pytest.raises(N.SoxError, match=match):
        backend.graph(pb.build(build(pb)), storage)


def test_refusals(offline):
    w = weights()

    def linear(shape=(ROWS, C), layout=None, **k):
        def build(pb):
            x = pb.input(shape, layout)
            ins = {key: pb.const(v) if isinstance(v, np.ndarray) else pb.input(v) for key, v in k.items()}
            return pb.quant_linear(x, ins.pop("w", None) or pb.const(w), ins.pop("b", None), **ins)
        return build

    refused("inner size", offline, linear((ROWS, C + 1)))
    refused("inner size", offline, linear((1, C, 5, 4), NHWC))
    refused("weights", offline, linear(w=np.ones((C, 2, 2), np.float32)))
    refused("finite", offline, linear(w=np.full((C, K), np.nan, np.float32)))
    refused("bias", offline, linear(b=np.ones(K + 1, np.float32)))
    refused("residual", offline, linear(residual=(ROWS, K + 1)))
    refused("131071", offline, linear((1, 131072), w=np.ones((131072, 1), np.float32)))

    def norm(shape=(ROWS, C), gate=None, **k):
        def build(pb):
            x = pb.input(shape)
            g = None if gate is None else pb.input(gate)
            h, y = pb.block_norm(residual=k.pop("res", x), x=x, gate=g, **k)
            return y
        return build

    refused("gate rows", offline, norm(gate=(3, C)))
    refused("gate rows", offline, norm(gate=(2 * ROWS, C)))
    refused("vector", offline, norm(pre_gamma=np.ones(C + 1, np.float32)))
    refused("16384", offline, norm((2, 16385)))
    refused("eps", offline, norm(pre_eps=-1.0))

    def operands(bits):
        def build(pb):
            x = pb.input((ROWS, C))
            p = N.BlockNormNodeP(N.BlockNormP(C, 0, 2, 0, 1e-5, 1e-5, 1.0), bits)
            return pb.ext("BlockNorm", [x], (ROWS, C), bytes(p))
        return build

    for bits in (0, 1, 512, 1 | 256 | 512, 1 | 2 | 512, 4 | 512, 1 | 512 | 1024):
        refused("operands|residual|branch|neither", offline, operands(bits))
    refused("too short", offline, lambda pb: pb.ext("BlockNorm", [pb.input((ROWS, C))], (ROWS, C), b"\0" * 8))
    refused("operands", offline, lambda pb: pb.ext("QuantLinear", [pb.input((ROWS, C))], (ROWS, C), bytes(12)))


def test_operand_in_the_outputs_buffer(offline):
    """Two values of one buffer that a node both reads and writes cannot be told apart: refused."""
    pb = PlanBuilder()
    x = pb.input((ROWS, C))
    a = pb.quant_linear(x, weights(C, C))
    y = pb.quant_linear(a, weights(C, C))
    pb.values[y].buf = pb.values[a].buf
    with pytest.raises(N.SoxError, match="operand's buffer"):
        offline.graph(pb.build(y), True)


def test_layers_under_sanitizers():
    """The layers' CPU tests again in a child process that loads the host code built under AddressSanitizer and
    UndefinedBehaviorSanitizer."""
    if os.environ.get("SIMDONNX_HIP_BACKEND_LIB"):
        pytest.skip("already the sanitizer child")
    from simdonnx_amd import build as B
    rt = B.sanitizer_runtime()
    if not rt:
        pytest.skip("the host compiler has no shared AddressSanitizer runtime")
    src = os.path.join(B.HDIR, "backend.cpp")
    if not os.path.exists(B.SAN_BACKEND) or os.path.getmtime(B.SAN_BACKEND) < os.path.getmtime(src):
        B.build_sanitized_backend()
    env = dict(os.environ, ASAN_OPTIONS="detect_leaks=0:halt_on_error=1", UBSAN_OPTIONS="halt_on_error=1:print_stacktrace=1",
               SIMDONNX_HIP_BACKEND_LIB=B.SAN_BACKEND)
    env["LD_PRELOAD"] = rt + (":" + env["LD_PRELOAD"] if env.get("LD_PRELOAD") else "")
    here = os.path.dirname(os.path.abspath(__file__))
    r = subprocess.run([sys.executable, "-m", "pytest", "-q", "-x", "-p", "no:cacheprovider", os.path.abspath(__file__),
                        os.path.join(here, "test_layer_refusals.py"), "-k", "not under_sanitizers"], cwd=os.path.dirname(here),
                       env=env, capture_output=True, text=True, timeout=600)
    assert r.returncode == 0 and "runtime error:" not in r.stdout + r.stderr, (r.stdout + r.stderr)[-6000:]
