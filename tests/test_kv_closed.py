"""Objects of the paged cache that are closed, on the CPU (an offline backend's)."""
import pytest

from simdonnx_amd.backend import HipKvCache, HipRotary
from test_kv_refusals import D, KV, PAGE, batch
from test_layer_refusals import at, in_order, offline, refused  # noqa: F401


def test_closed_objects(offline):  # noqa: F811
    """No call takes a closed object for one that was left out."""
    cache, rotary = HipKvCache(offline, KV, D, PAGE, "i8"), HipRotary(offline, D)
    in_order(cache.write, batch(), at(0), at(1), rotary=rotary)
    rotary.close()
    with pytest.raises(ValueError, match="rotary is closed"):
        cache.write(batch(), at(0), at(1), rotary=rotary)
    with pytest.raises(ValueError, match="rotary is closed"):
        cache.write(batch(), at(0), at(1), rotary=rotary, q=at(2), q_heads=4, y=at(3))
    refused("arguments", rotary.run, at(0), at(1), 50, 4, at(2))
    in_order(cache.write, batch(), at(0), at(1))
    size = cache.workspace(40, 3, 4)
    cache.close()
    refused("arguments", cache.write, batch(), at(0), at(1))
    refused("arguments", cache.read, batch(), at(0), at(1))
    refused("arguments", cache.attend, batch(), at(0), 4, at(1), workspace=at(2), workspace_bytes=size)
