"""Arguments of the cache functions at the edges: what cannot be served raises, on either route; shared block tables are served."""
import pytest
import torch

import delta_matching_b200 as dm
from delta_matching_b200 import _lib, ops

from .test_cache_gpu import _filled, _ints

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


@pytest.fixture(params=["native", "python"])
def route(request, monkeypatch):
    if request.param == "python":
        monkeypatch.setattr(_lib, "native_cache", lambda: _lib._NoCacheRoute)


def _call(B=2, lengths=(40, 33)):
    cache, _, table = _filled(list(lengths), 32, 2, 128, T=4)
    q, k = torch.randn(B, 1, 4, 128, device="cuda", dtype=BF), torch.randn(B, 1, 2, 128, device="cuda", dtype=BF)
    return cache, table.cuda(), _ints(list(lengths)).cuda(), q, k


@pytest.mark.parametrize("scale", [1e39, 1e-50, float("inf"), float("nan"), 0.0, -0.1])
def test_softmax_scale_in_32_bits(route, scale):
    cache, t, n, q, _ = _call()
    with pytest.raises(ValueError, match="softmax_scale"):
        dm.dm_cache_attn(q, cache, t, n, softmax_scale=scale)
    dm.dm_cache_attn(q, cache, t, n, softmax_scale=1e-30)
    ops.check_status("cuda")


def test_outputs_that_share_memory_are_refused(route):
    cache, t, n, q, k = _call()
    for w in (torch.zeros(1, 2, 128, device="cuda").expand(2, -1, -1), torch.zeros(2, 1, 128, device="cuda").expand(-1, 2, -1),
              torch.as_strided(torch.zeros(1000, device="cuda"), (2, 2, 128), (200, 100, 1))):
        with pytest.raises(ValueError, match="share memory"):
            dm.dm_cache_attn(q, cache, t, n, weights=w)
    # heads outside sequences, and gaps, are no sharing
    w = torch.zeros(2, 2, 130, device="cuda").transpose(0, 1)[:, :, :128]
    dm.dm_cache_attn(q, cache, t, n, weights=w)
    one = torch.ones(cache.ks.shape[0], 1, 1, device="cuda").expand(-1, 2, -1)
    shared = dm.KVCache8(cache.k8, cache.v8, one, one)
    dm.dm_cache_attn(q, shared, t, n)                            # to be read, scales may be shared
    with pytest.raises(ValueError, match="share memory"):
        dm.dm_cache_append(shared, k, k, t, n)
    with pytest.raises(ValueError, match="share memory"):
        dm.dm_cache_evict(shared, t, n, torch.zeros(2, 2, 128, device="cuda"), t, 32)
    ops.check_status("cuda")


def test_types(route):
    cache, t, n, q, k = _call()
    w = torch.zeros(2, 2, 128, device="cuda")
    for bad in (dict(budget=32.0), dict(budget=32.7), dict(budget=32, recent=1.5), dict(budget="32")):
        with pytest.raises(TypeError):
            dm.dm_cache_evict(cache, t[:, :2], n, w, t[:, 2:], **bad)
    for call in (lambda c: dm.dm_cache_append(c, k, k, t, n), lambda c: dm.dm_cache_attn(q, c, t, n), lambda c: dm.dm_cache_evict(c, t[:, :2], n, w, t[:, 2:], 8)):
        with pytest.raises(TypeError, match="KVCache8"):
            call(tuple(cache))
    ops.check_status("cuda")


@pytest.mark.parametrize("N", [1, 12])
def test_sequences_that_share_a_row_of_the_table(route, N):
    """Several sequences read one prefix, before any of them goes on: an expanded block table."""
    cache, t, n, _, _ = _call()
    q = torch.randn(3, N, 8, 128, device="cuda", dtype=BF)
    one, n3 = t[:1].expand(3, -1), n[:1].expand(3)
    o = dm.dm_cache_attn(q, cache, one, n3)
    ops.check_status("cuda")
    assert torch.equal(o, dm.dm_cache_attn(q, cache, one.contiguous(), n3.contiguous()))
