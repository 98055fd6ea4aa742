"""Refusals of the functions for drafted tokens that need no GPU: the C ABI's checks before any CUDA call, the Python checks before the device check, and
what the registered ops say of their results."""
import ctypes

import pytest
import torch

import delta_matching_b200 as dm
from delta_matching_b200 import _lib

from .test_cache_cpu import FINE, _c


def _tree(parents=FINE, row=5, B=2, N=5, depth=FINE, seen=FINE):
    return _lib.lib().dm_draft_tree(parents, row, None, B, N, depth, seen, None, None)


def _append(cache, q=FINE, k=FINE, v=FINE, B=2, N=3, H=4, freqs=FINE, F=64, table=FINE, T=4, lengths=FINE, offsets=None, o_row=3, out=FINE, new=FINE, st=(768, 256, 128)):
    return _lib.lib().dm_cache_append_rotary(ctypes.byref(cache), q, *st, k, *st, v, *st, B, N, H, freqs, F, 0, table, T, T, lengths, offsets, o_row, None, out, new, None, None)


def _attn(cache, q=FINE, B=2, N=5, H=4, table=FINE, T=4, lengths=FINE, seen=FINE, s_sb=5, s_sn=1, scale=0.1, o=FINE, lse=FINE, ws=FINE, ws_bytes=1 << 40, st=(2560, 512, 128)):
    return _lib.lib().dm_cache_attn_tree(ctypes.byref(cache), q, *st, B, N, H, table, T, T, lengths, None, seen, s_sb, s_sn, scale, o, lse, ws, ws_bytes, None, None)


def _keep(cache, B=2, table=FINE, T=4, before=FINE, lengths=FINE, path=FINE, row=3, M=3, counts=FINE, new=FINE):
    return _lib.lib().dm_cache_keep(ctypes.byref(cache), B, table, T, T, before, lengths, path, row, M, counts, new, None, None)


@pytest.mark.parametrize("call", [_append, _attn, _keep])
@pytest.mark.parametrize("bad, says", [
    (dict(k8=None), " k8 "), (dict(v8=0x1008), " v8 "), (dict(ks=None), " ks "), (dict(vs=None), " vs "), (dict(head_dim=64), "head_dim"),
    (dict(page_size=48), "page size"), (dict(pages=0), "empty"), (dict(heads=0), "empty"), (dict(code_slot=120), "multiples of 16")])
def test_bad_caches_are_refused(call, bad, says):
    assert call(_c(**bad)) == -1
    assert says in _lib.last_error()


@pytest.mark.parametrize("kw, says", [
    (dict(parents=None), "parents"), (dict(depth=None), "depth"), (dict(seen=None), "seen"), (dict(B=0), "empty"), (dict(N=0), "empty"), (dict(N=1025), "1024"),
    (dict(row=-1), "apart")])
def test_tree_refuses(kw, says):
    assert _tree(**kw) == -1
    assert says in _lib.last_error()


@pytest.mark.parametrize("kw, says", [
    (dict(q=None), " q "), (dict(k=0x1008), " k "), (dict(v=None), " v "), (dict(out=0x1008), "rotated q"), (dict(table=None), "block table"), (dict(lengths=None), "lengths"),
    (dict(new=None), "new lengths"), (dict(freqs=None), "freqs"), (dict(F=0), "multiple of 8"), (dict(F=12), "multiple of 8"), (dict(F=72), "multiple of 8"), (dict(B=0), "empty"),
    (dict(N=0), "empty"), (dict(H=0), "empty"), (dict(H=3), "nheads"), (dict(T=0), "empty"), (dict(B=40000), "65535"), (dict(st=(768, 256, 100)), "16-byte aligned"),
    (dict(offsets=FINE, o_row=-1), "apart"), (dict(N=(1 << 28) + 1), "too many")])
def test_append_refuses(kw, says):
    assert _append(_c(), **kw) == -1
    assert says in _lib.last_error()


@pytest.mark.parametrize("kw, says", [
    (dict(q=None), " q "), (dict(q=0x1008), " q "), (dict(o=None), " o "), (dict(lse=None), " lse "), (dict(ws=None), " workspace "), (dict(seen=None), "seen"),
    (dict(s_sn=-1), "strides of seen"), (dict(H=3), "nheads"), (dict(H=0), "empty"), (dict(N=0), "empty"), (dict(N=1025), "1024"), (dict(scale=0.0), "softmax_scale"),
    (dict(scale=float("inf")), "softmax_scale"), (dict(ws_bytes=8), "needed"), (dict(B=32000), "65535"), (dict(T=1 << 25), "2^30"), (dict(table=None), "block table")])
def test_attention_refuses(kw, says):
    assert _attn(_c(), **kw) == -1
    assert says in _lib.last_error()


@pytest.mark.parametrize("kw, says", [
    (dict(before=None), "before"), (dict(lengths=None), "lengths"), (dict(path=None), "path"), (dict(counts=None), "counts"), (dict(new=None), "new lengths"), (dict(M=0), "empty"),
    (dict(M=1025), "1024"), (dict(row=-1), "apart"), (dict(B=0), "empty"), (dict(T=0), "empty")])
def test_keep_refuses(kw, says):
    assert _keep(_c(), **kw) == -1
    assert says in _lib.last_error()


def test_workspace():
    L = _lib.lib()
    assert L.dm_cache_attn_tree_workspace_bytes(4, 16, 32, 8, 128, 64, 64) > 0
    for bad in ((4, 16, 33, 8, 128, 64, 64), (4, 16, 32, 8, 64, 64, 64), (4, 16, 32, 8, 128, 64, 48), (4, 1025, 32, 8, 128, 64, 64), (0, 16, 32, 8, 128, 64, 64)):
        assert L.dm_cache_attn_tree_workspace_bytes(*bad) == 0


def test_python_refusals_before_the_device():
    code, scale = torch.zeros(2, 2, 64, 128, dtype=torch.float8_e4m3fn), torch.ones(2, 2, 2)
    cache = dm.KVCache8(code, code, scale, scale)
    x, i, t = torch.zeros(1, 1, 2, 128, dtype=torch.bfloat16), torch.zeros(1, dtype=torch.int32), torch.zeros(1, 1, dtype=torch.int32)
    tree = dm.DraftTree(t, t[..., None])
    with pytest.raises(ValueError, match="CUDA"):
        dm.dm_draft_tree(t)
    for bad in (cache, (code, code, scale, scale)):
        error, says = (ValueError, "CUDA") if bad is cache else (TypeError, "KVCache8")
        with pytest.raises(error, match=says):
            dm.dm_cache_append_rotary(bad, x, x, x, t, i, torch.zeros(64))
        with pytest.raises(error, match=says):
            dm.dm_cache_attn_tree(x, bad, t, i, tree)
        with pytest.raises(error, match=says):
            dm.dm_cache_keep(bad, t, i, i, t, i)


def test_registered_ops_state_their_layout():
    from torch._subclasses.fake_tensor import FakeTensorMode
    ns = torch.ops.delta_matching_b200
    B, N, H, Hk, D, P, T = 3, 37, 8, 2, 128, 64, 7
    with FakeTensorMode():
        new = lambda *s, d=torch.float32: torch.empty(*s, device="cuda", dtype=d)
        pools = (new(9, Hk, P, D, d=torch.float8_e4m3fn), new(9, Hk, P, D, d=torch.float8_e4m3fn), new(9, Hk, P // 32), new(9, Hk, P // 32))
        k, q = new(B, N, Hk, D, d=torch.bfloat16), new(B, N, H, D, d=torch.bfloat16)
        table, lengths = new(B, T, d=torch.int32), new(B, d=torch.int32)
        depth, seen = ns.draft_tree(new(B, N, d=torch.int32), None)
        assert depth.shape == (B, N) and seen.shape == (B, N, 2) and depth.dtype == seen.dtype == torch.int32
        out, n = ns.cache_append_rotary(*pools, q, k, k, table, lengths, new(64), depth, None, False)
        assert out.shape == q.shape and out.dtype == torch.bfloat16 and n.shape == (B,) and n.dtype == torch.int32
        o, lse = ns.cache_attn_tree(q, *pools, table, lengths, seen, lengths, None)
        assert o.shape == q.shape and o.dtype == torch.bfloat16 and lse.shape == (B, H, N) and lse.dtype == torch.float32
        n = ns.cache_keep(*pools, table, lengths, lengths, depth, lengths)
        assert n.shape == (B,) and n.dtype == torch.int32
