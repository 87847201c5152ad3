"""A value that a fusion would not store any more, read through a zero-copy view as well (CValue.AliasOf, Engine/ExecPlan.cs:
207, 211) or given out as the plan's output through one: the fusion leaves it alone, on the CPU by the lowering."""
import numpy as np
import pytest

from simdonnx_amd import native as N
from simdonnx_amd.backend import HipBackend
from simdonnx_amd.plan import PlanBuilder

ROWS = 128


@pytest.fixture(scope="module")
def offline():
    b = HipBackend.offline()
    yield b
    b.close()


def f(*shape):
    return np.linspace(-1, 1, int(np.prod(shape)), dtype=np.float32).reshape(shape)


def residual_add(pb):
    x = pb.input((ROWS, 64))
    y = pb.gemm(x, f(64, 64), f(64))
    return y, pb.add(y, x)


def layer_norm(pb):
    y = pb.layer_norm(pb.input((ROWS, 64)), f(64) + 2, f(64))
    return y, pb.gemm(y, f(64, 128), f(128))


def mlp(pb):
    x = pb.input((ROWS, 192))
    h = pb.gemm(pb.layer_norm(x, f(192) + 2, f(192)), f(192, 768), f(768), act="gelu")
    return h, pb.add(pb.gemm(h, f(768, 192), f(192)), x)


def affine(pb):
    y = pb.conv_transpose(pb.input((1, 16, 8, 8), (0, 2, 3, 1)), f(16, 8, 2, 2), f(8))
    m = pb.mul(y, pb.const(f(1, 8, 1, 1)))
    return m, pb.add(m, pb.const(f(1, 8, 1, 1)))


def upsample_add(pb):
    x = pb.input((1, 16, 16, 16), (0, 2, 3, 1))
    u = pb.input((1, 32, 8, 8), (0, 2, 3, 1))
    a = pb.conv(x, f(32, 16, 1, 1), f(32), pad=0)
    return a, pb.resize_nearest(u, 2, add=a)


def gated(pb):
    x = pb.input((1, 16, 12, 12), (0, 2, 3, 1))
    s = pb.channel_gate(x, f(8, 16, 1, 1), f(8), f(16, 8, 1, 1), f(16))
    y = pb.mul(x, s)
    return y, pb.conv(y, f(24, 16, 1, 1), f(24), pad=0)


FUSIONS = [residual_add, layer_norm, mlp, affine, upsample_add, gated]


def lowered(backend, fusion, end):
    pb = PlanBuilder()
    y, out = fusion(pb)
    v = pb.values[y]
    view = pb.alias(y, v.shape, v.layout)
    if end == "output":
        out = view
    elif end == "reader":
        pb.unary("Tanh", view)
    elif end == "itself":
        pb.unary("Tanh", y)
    g = backend.graph(pb.build(out), True)
    place = g.value_place(y)[0]
    return g.kernels, [i for i in range(len(g.kernels)) if any(slot == 0 and at == place for slot, at, _ in g.binds(i))]


@pytest.mark.parametrize("end", ["reader", "output"])
@pytest.mark.parametrize("fusion", FUSIONS, ids=[x.__name__ for x in FUSIONS])
def test_view_of_a_value_keeps_it(offline, fusion, end):
    kernels, at = lowered(offline, fusion, end)
    plain, used = lowered(offline, fusion, "itself")
    if end == "reader":
        assert kernels == plain and at == used  # as where the value itself has a second reader
    assert at and (end == "output" or at[0] < len(kernels) - 1)
    assert lowered(offline, fusion, "nobody")[0] != [k for k in plain if "unary" not in k], "no fusion to be kept out"


@pytest.mark.parametrize("other", [True, False])
def test_concat_that_a_fused_mlp_adds(offline, other):
    """The concat of upsamples before a conv is stored where a fused MLP's kernel reads it as its residual."""
    pb = PlanBuilder()
    p, u = pb.input((1, 32, 16, 16), (0, 2, 3, 1)), pb.input((1, 32, 8, 8), (0, 2, 3, 1))
    x = pb.concat_channels([pb.resize_nearest(u, 2), p])
    s = pb.input((1, 16, 16, 64))
    h = pb.gemm(pb.layer_norm(s, f(64) + 2, f(64)), f(64, 256), f(256), act="gelu")
    pb.add(pb.gemm(h, f(256, 64), f(64)), x if other else s)
    g = offline.graph(pb.build(pb.conv(x, f(16, 64, 3, 3), f(16), pad=1)), True)
    assert any(k.startswith("sox_mlp") for k in g.kernels)
    assert any("upcat" in k for k in g.kernels) != other
    at, size = g.value_place(x)
    touch = [k for i, k in enumerate(g.kernels) if any(b[0] == 0 and b[1] < at + size and at < b[1] + b[2] for b in g.binds(i))]
    assert not other or not touch[0].startswith("sox_mlp"), touch  # (written before the MLP reads it)


@pytest.mark.parametrize("over", ["out", "residual", "clear"])
def test_slices_beside_a_fused_mlp(offline, over):
    """A conv does not write its slice of a concat ahead of a fused MLP whose output or residual the plan put there."""
    pb = PlanBuilder()
    layout = (0, 2, 3, 1)
    x = pb.input((1, 32, 16, 16), layout)
    s, r = pb.input((256, 64)), pb.input((256, 64))
    c = pb.conv(x, f(32, 32, 1, 1), f(32), pad=0)
    h = pb.gemm(pb.layer_norm(s, f(64) + 2, f(64)), f(64, 256), f(256), act="gelu")
    m = pb.add(pb.gemm(h, f(256, 64), f(64)), r)
    pb.unary("Tanh", m)
    cat = pb.concat_channels([c, x])
    p = pb.build(cat)
    place = p.arena_floats
    for v in (cat, {"out": m, "residual": r}.get(over, cat)):
        p.buf_offset[p.values[v].buf] = place
    p.arena_floats += 256 * 64
    g = offline.graph(p, True)
    assert any(k.startswith("sox_mlp") for k in g.kernels)
    at, size = g.value_place(cat)
    inside = [[b for b in g.binds(i) if b[0] == 0 and at <= b[1] < at + size] for i in range(len(g.kernels))]
    first = next(i for i, b in enumerate(inside) if b)
    assert ("conv" in g.kernels[first] or "gemm" in g.kernels[first]) == (over == "clear"), g.kernels


@pytest.mark.parametrize("wrong", [1000, 1 << 30, -1, -5])
@pytest.mark.parametrize("fusion", FUSIONS, ids=[x.__name__ for x in FUSIONS])
def test_readers_that_name_no_value(offline, fusion, wrong):
    """A node over an id that is no value's is refused, not looked up, by the fusions before it."""
    pb = PlanBuilder()
    _, out = fusion(pb)
    pb.unary("Tanh", out)
    p = pb.build(out)
    p.nodes[-1].ins = [wrong]
    with pytest.raises(N.SoxError, match="out of range"):
        offline.graph(p, True)
