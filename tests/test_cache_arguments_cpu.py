"""Arguments of the cache's C entry points at the edges; no GPU needed."""
import pytest

from delta_matching_b200 import _lib

from .test_cache_cpu import _append, _attn, _c


@pytest.mark.parametrize("scale", [float("inf"), 1e39])
def test_softmax_scale_is_finite(scale):
    assert _attn(_c(), scale=scale) == -1
    assert "softmax_scale" in _lib.last_error()
