"""Refusals of the cache operators that need no GPU: the C ABI's checks before any CUDA call, the Python checks before the device check, and the
plan of a call's workspace."""
import ctypes

import pytest
import torch

import delta_matching_b200 as dm
from delta_matching_b200 import _lib
from delta_matching_b200.cache import _CCache

FINE = 0x10000


def _c(**kw):
    c = dict(k8=FINE, v8=FINE, ks=FINE, vs=FINE, code_page=2 * 64 * 128, code_head=64 * 128, code_slot=128, scale_page=4, scale_head=2,
             pages=8, heads=2, page_size=64, head_dim=128)
    c.update(kw)
    return _CCache(**c)


def _append(cache, k=FINE, v=FINE, B=2, N=3, table=FINE, T=4, lengths=FINE, new=FINE, st=(768, 256, 128)):
    return _lib.lib().dm_cache_append(ctypes.byref(cache), k, *st, v, *st, B, N, table, T, T, lengths, None, new, None, None)


def _attn(cache, q=FINE, B=2, Nq=1, H=4, table=FINE, T=4, lengths=FINE, scale=0.1, o=FINE, lse=FINE, w=None, W=0, ws=FINE, ws_bytes=1 << 40, st=(512, 512, 128)):
    return _lib.lib().dm_cache_attn(ctypes.byref(cache), q, *st, B, Nq, H, table, T, T, lengths, None, 1, scale, o, lse, w, 0, 0, W, 0, ws, ws_bytes, None, None)


def _evict(cache, B=2, table=FINE, T=4, lengths=FINE, w=FINE, table2=FINE, T2=2, budget=100, recent=10, new=FINE, kept=FINE, nw=FINE):
    return _lib.lib().dm_cache_evict(ctypes.byref(cache), B, table, T, T, lengths, w, 512, 256, table2, T2, T2, budget, recent, new, kept, nw, None, None)


@pytest.mark.parametrize("call", [_append, _attn, _evict])
@pytest.mark.parametrize("bad, says", [
    (dict(k8=None), " k8 "), (dict(v8=0x1008), " v8 "), (dict(ks=None), " ks "), (dict(vs=None), " vs "), (dict(head_dim=64), "head_dim"),
    (dict(page_size=48), "page size"), (dict(page_size=0), "page size"), (dict(pages=0), "empty"), (dict(heads=0), "empty"),
    (dict(code_slot=120), "multiples of 16"), (dict(code_page=0), "multiples of 16"), (dict(code_head=1 << 40), "multiples of 16")])
def test_bad_caches_are_refused(call, bad, says):
    assert call(_c(**bad)) == -1
    assert says in _lib.last_error()


@pytest.mark.parametrize("kw, says", [
    (dict(k=None), " k "), (dict(v=0x1008), " v "), (dict(table=None), "block table"), (dict(lengths=None), "lengths"), (dict(new=None), "new lengths"),
    (dict(B=0), "empty"), (dict(N=0), "empty"), (dict(T=0), "empty"), (dict(B=40000), "65535"), (dict(st=(768, 256, 100)), "16-byte aligned"),
    (dict(T=1 << 25), "2^30"), (dict(N=(1 << 31) - 1, B=30000), "too many")])
def test_append_refuses(kw, says):
    assert _append(_c(), **kw) == -1
    assert says in _lib.last_error()


@pytest.mark.parametrize("kw, says", [
    (dict(q=None), " q "), (dict(q=0x1008), " q "), (dict(o=None), " o "), (dict(lse=None), " lse "), (dict(ws=None), " workspace "), (dict(H=3), "nheads"),
    (dict(H=0), "empty"), (dict(Nq=0), "empty"), (dict(scale=0.0), "softmax_scale"), (dict(scale=float("nan")), "softmax_scale"),
    (dict(ws_bytes=16), "needed"), (dict(w=FINE, W=255), "weights"), (dict(Nq=1 << 21), "too many"), (dict(B=32000), "65535"),
    (dict(T=1 << 24, Nq=1 << 10), "too much")])
def test_attention_refuses(kw, says):
    assert _attn(_c(), **kw) == -1
    assert says in _lib.last_error()


@pytest.mark.parametrize("kw, says", [
    (dict(table2=None), "new block table"), (dict(w=None), "weights"), (dict(new=None), "new lengths"), (dict(kept=None), "kept"), (dict(nw=None), "new weights"),
    (dict(budget=0), "budget"), (dict(budget=129), "budget"), (dict(recent=101), "recent"), (dict(recent=-1), "recent"), (dict(T2=0), "empty")])
def test_eviction_refuses(kw, says):
    assert _evict(_c(), **kw) == -1
    assert says in _lib.last_error()


def test_null_cache():
    assert _lib.lib().dm_cache_append(None, *([FINE, 8, 8, 8] * 2), 1, 1, FINE, 1, 1, FINE, None, FINE, None, None) == -1
    assert "cache is NULL" in _lib.last_error()


def test_workspace_covers_every_slot():
    """Two slots of partial results per CTA of the main kernel, and a pair per row when the weights are wanted; 0 for what is refused."""
    L = _lib.lib()
    plain = L.dm_cache_attn_workspace_bytes(4, 1, 32, 8, 128, 64, 64, 0)
    assert plain > 0
    assert L.dm_cache_attn_workspace_bytes(4, 1, 32, 8, 128, 64, 64, 1) >= plain + 4 * 32 * 8
    assert L.dm_cache_attn_workspace_bytes(4, 1, 33, 8, 128, 64, 64, 0) == 0
    assert L.dm_cache_attn_workspace_bytes(4, 1, 32, 8, 64, 64, 64, 0) == 0
    assert L.dm_cache_attn_workspace_bytes(4, 1, 32, 8, 128, 64, 48, 0) == 0


def test_python_refusals_before_the_device():
    code = torch.zeros(2, 2, 64, 128, dtype=torch.float8_e4m3fn)
    scale = torch.ones(2, 2, 2)
    cache = dm.KVCache8(code, code, scale, scale)
    x, i = torch.zeros(1, 1, 2, 128, dtype=torch.bfloat16), torch.zeros(1, dtype=torch.int32)
    t = torch.zeros(1, 1, dtype=torch.int32)
    with pytest.raises(TypeError, match="KVCache8"):
        dm.dm_cache_append((code, code, scale, scale), x, x, t, i)
    with pytest.raises(ValueError, match="CUDA"):
        dm.dm_cache_append(cache, x, x, t, i)
    with pytest.raises(ValueError, match="CUDA"):
        dm.dm_cache_attn(x, cache, t, i)
    with pytest.raises(ValueError, match="CUDA"):
        dm.dm_cache_evict(cache, t, i, torch.zeros(1, 2, 64), t, 4)
    with pytest.raises(ValueError, match="4-D"):
        dm.dm_cache_attn(x, dm.KVCache8(code[0], code, scale, scale), t, i)
    with pytest.raises(ValueError, match="page_size"):
        dm.KVCache8.empty(4, 40, 2, 128, device="cpu")


def test_registered_ops_state_their_layout():
    from torch._subclasses.fake_tensor import FakeTensorMode
    ns = torch.ops.delta_matching_b200
    B, N, H, Hk, D, P, T = 3, 5, 8, 2, 128, 64, 7
    with FakeTensorMode():
        new = lambda *s, d=torch.float32: torch.empty(*s, device="cuda", dtype=d)
        pools = (new(9, Hk, P, D, d=torch.float8_e4m3fn), new(9, Hk, P, D, d=torch.float8_e4m3fn), new(9, Hk, P // 32), new(9, Hk, P // 32))
        k, q = new(B, N, Hk, D, d=torch.bfloat16), new(B, N, H, D, d=torch.bfloat16)
        table, lengths, w = new(B, T, d=torch.int32), new(B, d=torch.int32), new(B, Hk, T * P)
        got = ns.cache_append(*pools, k, k, table, lengths, None)
        assert got.shape == (B,) and got.dtype == torch.int32
        for o, lse in (ns.cache_attn(q, *pools, table, lengths, lengths, True, None), ns.cache_attn_weights(q, *pools, table, lengths, None, True, 0.1, w, False)):
            assert o.shape == q.shape and o.dtype == torch.bfloat16 and lse.shape == (B, H, N) and lse.dtype == torch.float32
        n, kept, nw = ns.cache_evict(*pools, table, lengths, w, new(B, 2, d=torch.int32), 100, 10)
        assert n.shape == (B,) and kept.shape == (B, Hk, 100) and kept.dtype == torch.int32 and nw.shape == (B, Hk, 2 * P) and nw.dtype == torch.float32
