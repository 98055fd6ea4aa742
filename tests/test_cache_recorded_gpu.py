"""Calls of the cache functions that something records: torch.jit.trace and make_fx give, replayed on other inputs, what the functions give; a forward-mode tangent is
refused."""
import pytest
import torch

import delta_matching_b200 as dm
from delta_matching_b200 import ops

from . import cache_ref as ref
from .test_cache_gpu import _filled, _ints

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def _step(k8, v8, ks, vs, q, k, v, table, lengths, w):
    """Append, attend with weights added up, attend without, evict: everything a call can return or write."""
    cache = dm.KVCache8(k8, v8, ks, vs)
    lengths = dm.dm_cache_append(cache, k, v, table[:, :3], lengths)
    o, lse = dm.dm_cache_attn(q, cache, table[:, :3], lengths, weights=w, accumulate=True, return_lse=True)
    o2 = dm.dm_cache_attn(q, cache, table[:, :3], lengths, causal=False)
    n, kept, nw = dm.dm_cache_evict(cache, table[:, :3], lengths, w, table[:, 3:], 40, 8)
    return 2.0 * o, lse, o2, n, kept, nw


def _inputs(seed):
    cache, _, table = _filled([40, 61], 32, 2, 128, seed=seed, T=5)
    g = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda", dtype=torch.float32)
    return [*cache, rand(2, 3, 4, 128).to(BF), rand(2, 3, 2, 128).to(BF), rand(2, 3, 2, 128).to(BF), table.cuda(), _ints([40, 61]).cuda(), rand(2, 2, 96).abs()]


def _copy(xs):
    return [x.view(torch.uint8).clone().view(x.dtype) if x.dtype == torch.float8_e4m3fn else x.clone() for x in xs]


def _bits(t):
    return t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t.view(torch.int32) if t.dtype == torch.float32 else t


@pytest.mark.parametrize("record", ["jit.trace", "make_fx"])
def test_recorded_calls_replay(record):
    one, two = _inputs(1), _inputs(2)
    if record == "jit.trace":
        again = torch.jit.trace(_step, tuple(_copy(one)), check_trace=False)
    else:
        from torch.fx.experimental.proxy_tensor import make_fx
        again = make_fx(_step)(*_copy(one))
    a, b = _copy(two), _copy(two)
    torch.full((1 << 24,), float("nan"), device="cuda")          # what an uninitialised output would hold
    got, want = again(*a), _step(*b)
    ops.check_status("cuda")
    for i, (x, y) in enumerate(zip((*got, *a), (*want, *b))):
        assert torch.equal(_bits(x), _bits(y)), i


def test_dispatch_mode_sees_the_calls():
    from torch.utils._python_dispatch import TorchDispatchMode
    seen = []

    class Log(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            seen.append(func.name())
            return func(*args, **(kwargs or {}))

    a, b = _inputs(3), _inputs(3)
    with Log():
        got = _step(*a)
    want = _step(*b)
    assert [n.split("::")[1] for n in seen if n.startswith("delta_matching_b200::")] == ["cache_append", "cache_attn_weights", "cache_attn", "cache_evict"]
    for x, y in zip(got, want):
        assert torch.equal(_bits(x), _bits(y))


def test_tangents_are_refused():
    from torch.autograd import forward_ad
    k8, v8, ks, vs, q, k, v, table, lengths, w = _inputs(4)
    cache = dm.KVCache8(k8, v8, ks, vs)
    with forward_ad.dual_level():
        dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))
        with pytest.raises(NotImplementedError, match="q carries a forward-mode tangent"):
            dm.dm_cache_attn(dual(q), cache, table, lengths)
        with pytest.raises(NotImplementedError, match="v carries a forward-mode tangent"):
            dm.dm_cache_append(cache, k, dual(v), table, lengths)
        with pytest.raises(NotImplementedError, match="weights carries a forward-mode tangent"):
            dm.dm_cache_evict(cache, table[:, :3], lengths, dual(w), table[:, 3:], 40)
        dm.dm_cache_attn(q, cache, table, lengths)               # the level alone is no reason
    ops.check_status("cuda")
