"""What the 8-bit layers refuse, on the CPU: an offline backend's objects make every check of a call and then answer that
they have no device, so a call that reaches that answer was in order."""
import numpy as np
import pytest

from simdonnx_amd import native as N
from simdonnx_amd.backend import HipBackend, HipBlockNorm, HipQuantLinear
from simdonnx_amd.native import NotSupportedError, SoxError

K, C = 1100, 36  # inner, columns
ROWS = 2000  # (brought to 8 bits in a workspace)
BASE = 1 << 20  # addresses that nothing reads


@pytest.fixture(scope="module")
def offline():
    b = HipBackend.offline()
    yield b
    b.close()


@pytest.fixture
def linear(offline):
    lin = HipQuantLinear(offline, np.ones((K, C), np.int8), None, K, C, scales=np.ones(C, np.float32))
    yield lin
    lin.close()


@pytest.fixture
def norm(offline):
    n = HipBlockNorm(offline, C, post="rms", pre="layer", gate_act="sigmoid")
    yield n
    n.close()


def in_order(call, *a, **k):
    with pytest.raises(NotSupportedError, match="without a device"):
        call(*a, **k)


def refused(match, call, *a, **k):
    with pytest.raises(SoxError, match=match) as e:
        call(*a, **k)
    assert "without a device" not in str(e.value)


def at(i):
    return BASE + i * (1 << 24)


def run_args(**more):
    return dict(x=at(0), rows=ROWS, y=at(1), workspace=at(2), workspace_bytes=1 << 22) | more


def test_linear_checks(linear):
    run = linear.run
    in_order(run, **run_args())
    in_order(run, **run_args(ldx=K + 3, ldy=C + 5, residual=at(3), ldr=C + 1, storage="bf16", act="gelu"))
    in_order(run, **run_args(residual=at(1)))  # in place
    in_order(run, **run_args(rows=16, workspace=None, workspace_bytes=0))
    assert linear.workspace(0) == linear.workspace(16) == 0 and linear.workspace(ROWS) > ROWS * K
    linear.run(at(0), 0, at(1))  # no rows: nothing to do, nothing asked
    refused("x is null", run, **run_args(x=None))
    refused("y is null", run, **run_args(y=None))
    refused("rows", run, **run_args(rows=-1))
    refused("2\\^23 rows", run, **run_args(rows=(1 << 23) + 1))
    refused("x: rows of 1100 elements cannot be 1099 apart", run, **run_args(ldx=K - 1))
    refused("y: rows of 36", run, **run_args(ldy=C - 1))
    refused("y: rows of 36", run, **run_args(ldy=1 << 50))
    refused("residual: rows of 36", run, **run_args(residual=at(3), ldr=0))
    refused("x is not on 2-byte", run, **run_args(x=at(0) + 1))
    refused("y is not on 4-byte", run, **run_args(y=at(1) + 2, storage="f32"))
    refused("bytes of workspace, has 0", run, **run_args(workspace=None))
    refused("bytes of workspace, has 100", run, **run_args(workspace_bytes=100))
    refused("workspace is not on 16-byte", run, **run_args(workspace=at(2) + 8))
    refused("y overlaps x", run, **run_args(y=at(0) + ROWS * K * 2 - 2))
    refused("y overlaps workspace", run, **run_args(y=at(2) + 64))
    refused("workspace overlaps x", run, **run_args(workspace=at(0) + 16))
    refused("y overlaps residual without being it", run, **run_args(residual=at(1) + 2 * C))
    refused("y overlaps residual without being it", run, **run_args(residual=at(1), ldr=C + 2))
    with pytest.raises(KeyError):
        run(**run_args(storage="i8"))
    for storage in (-1, 3):
        assert N.backend().sox_qlinear_run(linear.h, None, storage, at(0), K, 100, None, 0, at(1), C, 0, at(2), 1 << 20) == N.SOX_E_INVALID
    for act in (-1, 6):
        assert N.backend().sox_qlinear_run(linear.h, None, 1, at(0), K, 100, None, 0, at(1), C, act, at(2), 1 << 20) == N.SOX_E_UNSUPPORTED
    assert N.backend().sox_qlinear_run(None, None, 1, at(0), K, 100, None, 0, at(1), C, 0, at(2), 1 << 20) == N.SOX_E_INVALID


def test_side_by_side_in_one_buffer(linear):
    """Columns of the same rows share a range of addresses, not elements."""
    ld = K + C
    in_order(linear.run, **run_args(ldx=ld, ldy=ld, y=at(0) + 2 * K))
    in_order(linear.run, **run_args(ldx=ld, ldy=ld, x=at(0) + 2 * C, y=at(0)))
    refused("y overlaps x", linear.run, **run_args(ldx=ld, ldy=ld, y=at(0) + 2 * K - 2))
    refused("y overlaps x", linear.run, **run_args(ldx=ld, ldy=ld, y=at(0) + 2 * K + 2))
    refused("y overlaps x", linear.run, **run_args(ldx=ld, ldy=ld + 2, y=at(0) + 2 * K))
    in_order(linear.run, **run_args(ldx=ld, ldy=ld, y=at(0) + 2 * ld * ROWS + 2 * K))


def test_linear_quantized_checks(linear):
    run = linear.run_quantized
    ok = dict(q=at(0), scales=at(1), rows=50, y=at(2))
    in_order(run, **ok)
    in_order(run, **ok | dict(ldq=1104))
    assert linear.pitch == 1152
    linear.run_quantized(at(0), at(1), 0, at(2))
    refused("q is null", run, **ok | dict(q=None))
    refused("scales is null", run, **ok | dict(scales=None))
    refused("q is not on 16-byte", run, **ok | dict(q=at(0) + 8))
    refused("q is not on 16-byte", run, **ok | dict(ldq=1112))
    refused("q: rows of 1104", run, **ok | dict(ldq=1088))
    refused("scales is not on 4-byte", run, **ok | dict(scales=at(1) + 2))
    refused("y overlaps q", run, **ok | dict(y=at(0) + 128))
    refused("y overlaps scales", run, **ok | dict(y=at(1) + 196))


def test_linear_creation(offline):
    w = np.ones((K, C), np.float32)
    HipQuantLinear(offline, w, np.zeros(C), K, C).close()
    for bad in (np.nan, np.inf):
        v = w.copy()
        v[3, 3] = bad
        refused("finite", HipQuantLinear, offline, v, None, K, C)
        s = np.ones(C, np.float32)
        s[0] = bad
        refused("finite", HipQuantLinear, offline, w.astype(np.int8), None, K, C, scales=s)
    refused("arguments", HipQuantLinear, offline, np.ones((0, C), np.float32), None, 0, C)
    refused("131071", HipQuantLinear, offline, np.zeros((131072, 1), np.int8), None, 131072, 1, scales=np.ones(1))
    for bad in (lambda: HipQuantLinear(offline, w, None, K, C + 1), lambda: HipQuantLinear(offline, w, np.zeros(C + 1), K, C),
                lambda: HipQuantLinear(offline, w * 0.5, None, K, C, scales=np.ones(C)),
                lambda: HipQuantLinear(offline, w * 300, None, K, C, scales=np.ones(C))):
        with pytest.raises(ValueError):
            bad()
    assert N.backend().sox_qlinear_create(offline.h, None, None, K, C, N.ctypes.byref(N.c_void_p())) == N.SOX_E_INVALID
    N.backend().sox_qlinear_destroy(None)
    assert N.backend().sox_qlinear_pitch(None) == 0 and N.backend().sox_qlinear_workspace(None, 5) == 0


def test_norm_checks(norm):
    run = norm.run
    ok = dict(residual=at(0), rows=60, x=at(1), h=at(2), y=at(3))
    in_order(run, **ok)
    in_order(run, **ok | dict(gate=at(4), gate_rows=20))
    in_order(run, **ok | dict(x=None))
    in_order(run, **ok | dict(residual=None))
    in_order(run, **ok | dict(h=None))
    in_order(run, **ok | dict(y=None))
    in_order(run, **ok | dict(h=at(0), y=at(1)))  # in place
    in_order(run, **ok | dict(h=at(1), y=at(0)))
    norm.run(at(0), 0, h=at(2))
    refused("neither a residual nor a branch", run, **ok | dict(residual=None, x=None))
    refused("neither h nor y", run, **ok | dict(h=None, y=None))
    refused("a gate without a branch", run, **ok | dict(x=None, gate=at(4)))
    refused("gate rows have to divide", run, **ok | dict(gate=at(4), gate_rows=7))
    refused("gate rows have to divide", run, **ok | dict(gate=at(4), gate_rows=0))
    refused("gate rows have to divide", run, **ok | dict(gate=at(4), gate_rows=120))
    refused("h overlaps y", run, **ok | dict(y=at(2)))
    refused("h overlaps gate", run, **ok | dict(gate=at(2)))
    refused("y overlaps gate", run, **ok | dict(gate=at(3)))
    refused("h overlaps residual without being it", run, **ok | dict(h=at(0) + 2 * C))
    refused("y overlaps x without being it", run, **ok | dict(y=at(1), ldy=C + 8))
    refused("x: rows of 36", run, **ok | dict(ldx=8))
    refused("h is not on 2-byte", run, **ok | dict(h=at(2) + 1))
    refused("rows", run, **ok | dict(rows=-5))
    q = dict(residual=at(0), rows=60, x=at(1), h=at(2), q=at(3), scales=at(4))
    in_order(norm.run_quantized, **q)
    in_order(norm.run_quantized, **q | dict(ldq=48, h=None))
    refused("q: rows of 48", norm.run_quantized, **q | dict(ldq=32))
    refused("q is not on 16-byte", norm.run_quantized, **q | dict(ldq=56))
    refused("q is null", norm.run_quantized, **q | dict(q=None))
    refused("scales is null", norm.run_quantized, **q | dict(scales=None))
    refused("q overlaps x", norm.run_quantized, **q | dict(q=at(1)))
    refused("h overlaps q", norm.run_quantized, **q | dict(q=at(2)))
    refused("scales overlaps residual", norm.run_quantized, **q | dict(scales=at(0)))
    refused("h overlaps scales", norm.run_quantized, **q | dict(scales=at(2)))


def test_norm_creation(offline):
    refused("arguments", HipBlockNorm, offline, 0)
    refused("16384", HipBlockNorm, offline, 16385)
    refused("eps", HipBlockNorm, offline, 8, pre_eps=-1.0)
    refused("eps", HipBlockNorm, offline, 8, post_eps=np.nan)
    refused("residual scale", HipBlockNorm, offline, 8, res_scale=np.inf)
    with pytest.raises(KeyError):
        HipBlockNorm(offline, 8, post="batch")
    with pytest.raises(ValueError):
        HipBlockNorm(offline, 8, pre_gamma=np.ones(9))
    for bad in (N.BlockNormP(8, 3, 0, 0, 0, 0, 1), N.BlockNormP(8, 0, -1, 0, 0, 0, 1)):
        assert N.backend().sox_block_norm_create(offline.h, N.ctypes.byref(bad), None, None, None, None, None,
                                                 N.ctypes.byref(N.c_void_p())) == N.SOX_E_INVALID
    bad = N.BlockNormP(8, 0, 0, 9, 0, 0, 1)
    assert N.backend().sox_block_norm_create(offline.h, N.ctypes.byref(bad), None, None, None, None, None,
                                             N.ctypes.byref(N.c_void_p())) == N.SOX_E_UNSUPPORTED
    N.backend().sox_block_norm_destroy(None)


@pytest.mark.parametrize("k,n", [(768, 768), (256, 4096), (512, 2048), (32, 16), (1024, 96), (1025, 40), (4096, 64), (4097, 64)])
def test_workspace_for_the_largest_call(offline, k, n):
    """A workspace taken for the largest number of rows is enough for every smaller call, whichever way each runs."""
    lin = HipQuantLinear(offline, np.ones((k, n), np.int8), None, k, n, scales=np.ones(n, np.float32))
    sizes = [lin.workspace(rows) for rows in range(2049)]
    assert sizes == sorted(sizes) and sizes[0] == 0
    assert (sizes[16] == 0) == (k <= 4096)
    far = [lin.workspace(rows) for rows in (1 << 14, 100003, 1 << 20, (1 << 20) + 1, 1 << 23)]
    assert far == sorted(far) and far[0] >= sizes[-1]
    for most in (2048, 1600, 1118, 21, 17):
        size = lin.workspace(most)
        for rows in {1, 15, 16, 17, 18, 20, 21, 64, 65, 1117, 1118, 1471, 1472, 1574, 1575, most}:
            if rows <= most:
                for storage in ("f16", "bf16", "f32"):
                    in_order(lin.run, x=at(0), rows=rows, y=at(4), storage=storage, workspace=at(8), workspace_bytes=size)
    lin.close()


def test_counts_past_32_bits(linear, norm):
    """Row counts whose lowest 32 bits are a count in order."""
    for rows in (1 << 32, (1 << 32) + 16, 1 << 31):
        refused("rows", linear.run, **run_args(rows=rows))
        refused("rows", linear.run_quantized, q=at(0), scales=at(1), rows=rows, y=at(2))
        refused("rows", norm.run, at(0), rows, h=at(2))
        refused("rows", norm.run_quantized, at(0), rows, at(2), at(3))
        refused("rows", norm.run, at(0), 16, x=at(1), gate=at(4), gate_rows=rows, h=at(2))
        assert linear.workspace(rows) == 0
