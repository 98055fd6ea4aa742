"""Arguments of the cache's C entry points at the edges; no GPU needed."""
import pytest

from delta_matching_b200 import _lib

from .test_cache_cpu import _append, _attn, _c


@pytest.mark.parametrize("scale", [float("inf"), 1e39])
def test_softmax_scale_is_finite(scale):
    assert _attn(_c(), scale=scale) == -1
    assert "softmax_scale" in _lib.last_error()


def test_append_refuses_what_no_grid_holds():
    # 2^31 - 1 tokens are 2^26 + 1 blocks, of 16 sequences, 2 heads, K and V: above 2^32 items in CTAs of four
    assert _append(_c(), N=(1 << 31) - 1, B=16) == -1
    assert "too many tokens" in _lib.last_error()


@pytest.mark.parametrize("B, Nq, T", [(1, 131072, 2048), (8, 4096, 4096), (1, 1024, 1 << 20)])
def test_large_calls_of_many_rows_have_a_plan(B, Nq, T):
    """A whole prompt, and a chunk with a wide table: few enough steps for the tcgen05 form."""
    assert _lib.lib().dm_cache_attn_workspace_bytes(B, Nq, 32, 8, 128, T, 64, 0) > 0, _lib.last_error()
