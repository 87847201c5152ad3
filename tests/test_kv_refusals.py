"""What rotary positions and the paged cache refuse, on the CPU: an offline backend's objects make every check of a call and
then answer that they have no device, so a call that reaches that answer was in order."""
import ctypes

import numpy as np
import pytest

from simdonnx_amd import native as N
from simdonnx_amd.backend import HipBackend, HipKvBatch, HipKvCache, HipRotary
from simdonnx_amd.native import NotSupportedError, SoxError
from test_layer_refusals import at, in_order, offline, refused  # noqa: F401

KV, D, PAGE = 2, 64, 16


@pytest.fixture
def rotary(offline):  # noqa: F811
    r = HipRotary(offline, D)
    yield r
    r.close()


@pytest.fixture
def cache(offline):  # noqa: F811
    c = HipKvCache(offline, KV, D, PAGE, "i8")
    yield c
    c.close()


def batch(**more):
    return HipKvBatch(**(dict(pool=at(20), pages=100, tables=at(30), table_pages=12, starts=at(31), lengths=at(32), sequences=3, rows=40) | more))


def test_rotary_checks(rotary):
    run, ok = rotary.run, dict(x=at(0), positions=at(1), rows=50, heads=4, y=at(2))
    in_order(run, **ok)
    in_order(run, **ok | dict(y=at(0)))  # in place
    in_order(run, **ok | dict(ldx=4 * D + 3, ldy=4 * D + 1, storage="f32"))
    in_order(run, **ok | dict(ldx=8 * D, ldy=8 * D, y=at(0) + 8 * D))  # heads side by side in one buffer
    rotary.run(at(0), at(1), 0, 4, at(2))
    refused("x is null", run, **ok | dict(x=None))
    refused("positions is null", run, **ok | dict(positions=None))
    refused("positions is not on 4-byte", run, **ok | dict(positions=at(1) + 2))
    refused("rows", run, **ok | dict(rows=-1))
    refused("rows", run, **ok | dict(rows=1 << 32))
    refused("2\\^23 rows", run, **ok | dict(rows=(1 << 23) + 1))
    refused("heads", run, **ok | dict(heads=0))
    refused("heads", run, **ok | dict(heads=1 << 32))
    refused("x: rows of 256 elements cannot be 255 apart", run, **ok | dict(ldx=255))
    refused("y overlaps x without being it", run, **ok | dict(y=at(0) + 2))
    refused("y overlaps x without being it", run, **ok | dict(y=at(0), ldy=5 * D))
    refused("y overlaps positions", run, **ok | dict(positions=at(2) + 8))
    with pytest.raises(KeyError):
        run(**ok | dict(storage="i8"))
    assert N.backend().sox_rotary_run(rotary.h, None, 3, at(1), at(0), 256, 1, 4, at(2), 256) == N.SOX_E_INVALID
    assert N.backend().sox_rotary_run(None, None, 1, at(1), at(0), 256, 1, 4, at(2), 256) == N.SOX_E_INVALID


def test_rotary_creation(offline):  # noqa: F811
    for dim in (8, 72, 256):
        HipRotary(offline, dim).close()
    refused("head_dim", HipRotary, offline, 0)
    for dim in (12, 264, 1024):
        with pytest.raises(NotSupportedError, match="head_dim"):
            HipRotary(offline, dim)
    for rotary in (0, 3, 66, -2):
        refused("rotary_dim", HipRotary, offline, 64, rotary_dim=rotary)
    for bad in (dict(base=0.0), dict(base=np.inf), dict(base=np.nan)):
        refused("base", HipRotary, offline, 64, **bad)
    for bad in (0.0, -1.0, np.nan):
        refused("factor", HipRotary, offline, 64, factor=bad)
    refused("amplitude", HipRotary, offline, 64, amplitude=np.nan)
    refused("original", HipRotary, offline, 64, original=-1)
    refused("low and high", HipRotary, offline, 64, original=100, low=4.0, high=4.0)
    refused("finite", HipRotary, offline, 64, frequencies=np.full(32, np.nan))
    with pytest.raises(ValueError):
        HipRotary(offline, 64, frequencies=np.ones(31))
    N.backend().sox_rotary_destroy(None)
    assert N.backend().sox_rotary_frequencies(None, at(0)) == N.SOX_E_INVALID
    assert N.backend().sox_rotary_create(offline.h, None, None, ctypes.byref(N.c_void_p())) == N.SOX_E_INVALID


def test_frequencies(offline):  # noqa: F811
    j = np.arange(32)
    f = 5e5 ** (-j / 32)
    close = lambda r, want: np.testing.assert_allclose(r.frequencies, want, rtol=1e-15)  # noqa: E731
    close(HipRotary(offline, 64, base=5e5), f)
    close(HipRotary(offline, 64, base=5e5, factor=4.0), f / 4)
    keep = np.clip((4096 * f / (2 * np.pi) - 1) / 3, 0, 1)
    assert 0 < ((keep > 0) & (keep < 1)).sum() and keep[0] == 1 and keep[-1] == 0
    np.testing.assert_allclose(HipRotary(offline, 64, base=5e5, factor=8.0, original=4096).frequencies, f * (keep + (1 - keep) / 8), rtol=1e-13)


def test_cache_creation(offline):  # noqa: F811
    sizes = {}
    for fmt in ("f16", "bf16", "f32", "i8"):
        c = HipKvCache(offline, 3, 40, 8, fmt)
        sizes[fmt] = c.page_bytes
        assert c.page_bytes % 256 == 0
        c.close()
    values = 2 * 3 * 8 * 40
    assert values * 2 <= sizes["f16"] == sizes["bf16"] < values * 2 + 256 and values * 4 <= sizes["f32"] < values * 4 + 256
    assert values + 2 * 3 * 8 * 4 <= sizes["i8"] < values + 2 * 3 * 8 * 4 + 256
    for page in (0, 3, 24, 8192, -16, 1 << 32):
        refused("page", HipKvCache, offline, 2, 64, page)
    refused("kv_heads", HipKvCache, offline, 0, 64)
    refused("kv_heads", HipKvCache, offline, 1025, 64)
    for dim in (4, 260, 512):
        with pytest.raises(NotSupportedError, match="head_dim"):
            HipKvCache(offline, 2, dim)
    with pytest.raises(KeyError):
        HipKvCache(offline, 2, 64, 16, "i4")
    bad = N.KvCacheP(2, 64, 16, 4)
    assert N.backend().sox_kv_cache_create(offline.h, ctypes.byref(bad), ctypes.byref(N.c_void_p())) == N.SOX_E_INVALID
    N.backend().sox_kv_cache_destroy(None)
    assert N.backend().sox_kv_cache_page_bytes(None) == 0 and N.backend().sox_kv_cache_workspace(None, 1, 1, 1) == 0


def test_batch_checks(cache):
    ok = dict(k=at(0), v=at(1))
    write, read = cache.write, cache.read
    for call in (write, read):
        in_order(call, batch(), **ok)
        in_order(call, batch(ldt=20), **ok)
        in_order(call, batch(), **ok | dict(ldk=KV * D + 1, ldv=KV * D + 7, storage="f32"))
        call(batch(rows=0), **ok)
        call(batch(sequences=0), **ok)
        refused("pool is null", call, batch(pool=None), **ok)
        refused("pool is not on 256-byte", call, batch(pool=at(20) + 128), **ok)
        refused("pages", call, batch(pages=0), **ok)
        refused("pages", call, batch(pages=1 << 32), **ok)
        refused("tables is null", call, batch(tables=None), **ok)
        refused("tables: rows of 12", call, batch(ldt=11), **ok)
        refused("table_pages", call, batch(table_pages=0), **ok)
        refused("table_pages", call, batch(table_pages=1 << 27), **ok)
        refused("starts is null", call, batch(starts=None), **ok)
        refused("starts is not on 4-byte", call, batch(starts=at(31) + 1), **ok)
        refused("lengths is null", call, batch(lengths=None), **ok)
        refused("sequences", call, batch(sequences=-1), **ok)
        refused("sequences", call, batch(sequences=1 << 32), **ok)
        refused("rows", call, batch(rows=-1), **ok)
        refused("rows", call, batch(rows=(1 << 32) + 4), **ok)
        refused("k is null", call, batch(), **ok | dict(k=None))
        refused("v: rows of 128", call, batch(), **ok | dict(ldv=127))
        refused("k is not on 2-byte", call, batch(), **ok | dict(k=at(0) + 1))
    for name, call in (("write", write), ("read", read)):
        refused("overlaps", call, batch(), **ok | dict(k=at(20) + 4096))
    refused("pool overlaps tables", write, batch(tables=at(20) + 512), **ok)
    refused("k overlaps v", read, batch(), **ok | dict(v=at(0)))
    refused("v overlaps lengths", read, batch(lengths=at(1) + 64), **ok)
    in_order(write, batch(), k=at(0), v=at(0))  # (two reads of the same rows)


def test_storage_of_the_cache(offline):  # noqa: F811
    c = HipKvCache(offline, KV, D, PAGE, "bf16")
    for call in (c.write, c.read):
        in_order(call, batch(), at(0), at(1), "bf16")
        refused("another storage", call, batch(), at(0), at(1), "f16")
    refused("another storage", c.attend, batch(), at(0), 4, at(1), "f32")
    c.close()


def test_write_with_queries(offline, cache, rotary):  # noqa: F811
    ok = dict(k=at(0), v=at(1), rotary=rotary, q=at(2), q_heads=4, y=at(3))
    in_order(cache.write, batch(), **ok)
    in_order(cache.write, batch(), **ok | dict(y=at(2)))  # in place
    ld = 8 * D
    in_order(cache.write, batch(), k=at(0) + 8 * D, v=at(0) + 12 * D, rotary=rotary, q=at(0), q_heads=4, y=at(0), ldk=ld, ldv=ld, ldq=ld, ldy=ld)
    in_order(cache.write, batch(), at(0), at(1), rotary=rotary)
    refused("q without a rotary", cache.write, batch(), **ok | dict(rotary=None))
    refused("q_heads", cache.write, batch(), **ok | dict(q_heads=0))
    refused("y is null", cache.write, batch(), **ok | dict(y=None))
    refused("y overlaps k", cache.write, batch(), **ok | dict(y=at(0)))
    refused("y overlaps q without being it", cache.write, batch(), **ok | dict(y=at(2) + 16))
    refused("pool overlaps y", cache.write, batch(), **ok | dict(y=at(20)))
    other = HipRotary(offline, 72)
    refused("another head_dim", cache.write, batch(), **ok | dict(rotary=other))
    other.close()


def test_attend_checks(cache):
    size = cache.workspace(40, 3, 4)
    ok = dict(q=at(0), q_heads=4, y=at(1), workspace=at(2), workspace_bytes=size)
    run = cache.attend
    in_order(run, batch(), **ok)
    in_order(run, batch(), **ok | dict(ldq=4 * D + 1, ldy=4 * D + 3, storage="f32", window=7, scale=0.3))
    run(batch(rows=0), **ok)
    run(batch(sequences=0), **ok)
    refused("q is null", run, batch(), **ok | dict(q=None))
    refused("multiple of kv_heads", run, batch(), **ok | dict(q_heads=3))
    refused("multiple of kv_heads", run, batch(), **ok | dict(q_heads=0))
    refused("multiple of kv_heads", run, batch(), **ok | dict(q_heads=1 << 32))
    for scale in (-1.0, np.nan, np.inf):
        refused("scale", run, batch(), **ok | dict(scale=scale))
    refused("window", run, batch(), **ok | dict(window=-1))
    refused("window", run, batch(), **ok | dict(window=1 << 32))
    refused("y overlaps q", run, batch(), **ok | dict(y=at(0)))
    refused("y overlaps pool", run, batch(), **ok | dict(y=at(20)))
    long = dict(sequences=1, rows=1, table_pages=1 << 13)
    refused("bytes of workspace, has 0", run, batch(**long), **ok | dict(workspace=None))
    refused("bytes of workspace, has 100", run, batch(**long), **ok | dict(workspace_bytes=100))
    refused("workspace is not on 16-byte", run, batch(**long), **ok | dict(workspace=at(2) + 8))
    refused("y overlaps workspace", run, batch(**long), **ok | dict(y=at(2) + 64))
    refused("workspace overlaps q", run, batch(**long), **ok | dict(workspace=at(0)))
    refused("rows", run, batch(rows=1 << 31), **ok)
    assert N.backend().sox_kv_cache_attend(None, None, batch().ref, 1, at(0), 256, 4, at(1), 256, 0.0, 0, at(2), size) == N.SOX_E_INVALID
    assert N.backend().sox_kv_cache_attend(cache.h, None, None, 1, at(0), 256, 4, at(1), 256, 0.0, 0, at(2), size) == N.SOX_E_INVALID


@pytest.mark.parametrize("kv,group,dim", [(1, 1, 64), (8, 4, 128), (2, 16, 256), (128, 1, 72)])
def test_workspace_for_the_largest_call(offline, kv, group, dim):  # noqa: F811
    """A workspace taken for the largest numbers of rows and sequences is enough for every smaller call, however long its tables."""
    c = HipKvCache(offline, kv, dim, 16, "f16")
    heads = kv * group
    sizes = [c.workspace(rows, 64, heads) for rows in (1, 2, 3, 63, 64, 65, 500, 4096, 100000, 1 << 23)]
    assert sizes == sorted(sizes) and sizes[0] > 0
    for most, sequences in ((1, 1), (64, 64), (700, 3), (5000, 32)):
        size = c.workspace(most, sequences, heads)
        for rows in {1, 2, 15, 16, 17, 64, 100, 128, 129, most}:
            for seq in {1, 2, sequences}:
                for pages in (1, 16, 1000, 1 << 16):
                    if rows <= most and seq <= sequences:
                        in_order(c.attend, batch(rows=rows, sequences=seq, table_pages=pages), q=at(0), q_heads=heads, y=at(8),
                                 workspace=at(64), workspace_bytes=size)
    assert c.workspace(0, 1, heads) == c.workspace(-1, 1, heads) == c.workspace(1 << 32, 1, heads) == c.workspace(1, 0, heads) == 0
    c.close()


def test_lost_objects():
    with pytest.raises(SoxError):
        N.check(N.backend().sox_kv_cache_write(None, None, None, 1, None, None, 0, None, 0, None, 0, 0, None, 0), "KvCache.Write")


def test_a_backend_of_its_own(offline, cache):  # noqa: F811
    """A rotary of another backend may stand on another device."""
    b = HipBackend.offline()
    r = HipRotary(b, D)
    refused("another head_dim or backend", cache.write, batch(), at(0), at(1), rotary=r)
    r.close()
    b.close()


def test_attend_too_large(offline):  # noqa: F811
    """More (row, query head)s than 32 bits count with their tiles, more workgroups than a launch holds."""
    c, q, y = HipKvCache(offline, 128, 8, 16, "f16"), at(0) + (1 << 40), at(0) + (1 << 41)
    far = dict(tables=at(0) + (1 << 42), starts=at(0) + (1 << 43), lengths=at(0) + (1 << 44))
    with pytest.raises(NotSupportedError, match="2\\^30 rows times q_heads"):
        c.attend(batch(rows=1 << 23), q, 256, y)
    in_order(c.attend, batch(sequences=1 << 16, rows=1 << 16, ldt=12, **far), q, 128, y)
    with pytest.raises(NotSupportedError, match="too many rows"):
        c.attend(batch(sequences=1 << 20, rows=1 << 20, ldt=12, **far), q, 128, y)
    c.close()
