"""examples/decode_with_cache.py: the operators together, step by step against exact attention over what was put in, and the cache's bookkeeping."""
import importlib.util
import os

import pytest
import torch

from .conftest import ROOT

pytestmark = pytest.mark.gpu


def _example():
    spec = importlib.util.spec_from_file_location("decode_with_cache", os.path.join(ROOT, "examples", "decode_with_cache.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def _prompts(lengths):
    g = torch.Generator(device="cuda").manual_seed(1)
    return [torch.randn(n, 256, generator=g, device="cuda").to(torch.bfloat16) for n in lengths]


def test_every_step_is_attention_over_the_history():
    """Without evictions: each step's output against fp32 attention on the bf16 keys and values.  The cache holds them in e4m3: half of the last of
    four significant bits, 2^-4 of a value at most, about 0.027 of the norm for evenly spread ones; the weights shift by as much again."""
    m = _example()
    layer = m.Layer(256, 8, 2, 128)
    history, worst = None, []

    def record(k, v, q, o, lengths):
        nonlocal history
        if history is None:
            history = [(k[b, :n], v[b, :n]) for b, n in enumerate(lengths)]
            first = [0] * len(lengths)
        else:
            history = [(torch.cat([hk, k[b]]), torch.cat([hv, v[b]])) for b, (hk, hv) in enumerate(history)]
            first = [n - 1 for n in lengths]
        for b, n in enumerate(lengths):
            kk, vv = (t.float().repeat_interleave(4, 1).transpose(0, 1) for t in history[b])
            qq = q[b, :n - first[b]].float().transpose(0, 1)
            s = qq @ kk.transpose(1, 2) * 128 ** -0.5
            s = s.masked_fill(torch.arange(n, device="cuda")[None] > torch.arange(first[b], n, device="cuda")[:, None], -torch.inf)
            want = (torch.softmax(s, -1) @ vv).transpose(0, 1)
            worst.append(float((o[b, :n - first[b]].float() - want).norm() / want.norm()))

    made, held, evictions = m.generate(layer, _prompts([1, 33, 70]), 20, 1000, 500, 100, record=record)
    assert evictions == 0 and held == [21, 53, 90] and bool(made.isfinite().all())
    assert max(worst) < 0.08, max(worst)                          # the bound of the framework's own e4m3 attention


def test_evictions_bound_the_cache():
    m = _example()
    layer = m.Layer(256, 4, 2, 128)
    made, held, evictions = m.generate(layer, _prompts([5, 40, 64]), 150, 80, 48, 16)
    assert evictions > 2 and max(held) <= 80 and bool(made.isfinite().all())
    again, _, _ = m.generate(layer, _prompts([5, 40, 64]), 150, 80, 48, 16)
    assert torch.equal(made, again)


def test_compiled_step_equals_eager():
    """append, attention with weights and eviction under torch.compile, without a graph break."""
    import delta_matching_b200 as dm
    g = torch.Generator(device="cuda").manual_seed(2)
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda").to(torch.bfloat16)
    k, v, q = rand(2, 40, 2, 128), rand(2, 40, 2, 128), rand(2, 40, 4, 128)
    table = torch.tensor([[0, 1], [2, 3]], dtype=torch.int32, device="cuda")
    new_table = torch.tensor([[4], [5]], dtype=torch.int32, device="cuda")

    def step(cache, k, v, q, weights):
        lengths = dm.dm_cache_append(cache, k, v, table, torch.zeros(2, dtype=torch.int32, device="cuda"))
        o, lse = dm.dm_cache_attn(q, cache, table, lengths, weights=weights, return_lse=True)
        plain = dm.dm_cache_attn(q, cache, table, lengths)
        return (o, lse, plain) + dm.dm_cache_evict(cache, table, lengths, weights, new_table, 20, recent=4)

    out = []
    for fn in (step, torch.compile(step, fullgraph=True, backend="aot_eager")):
        cache = dm.KVCache8(*(torch.zeros(6, 2, 32, 128, device="cuda", dtype=torch.uint8).view(torch.float8_e4m3fn) for _ in range(2)),
                            *(torch.zeros(6, 2, 1, device="cuda") for _ in range(2)))
        w = torch.zeros(2, 2, 64, device="cuda")
        out.append(fn(cache, k, v, q, w) + (w, cache.k8.view(torch.uint8), cache.v8.view(torch.uint8), cache.ks, cache.vs))
    for a, b in zip(*out):
        assert torch.equal(a, b)


def test_native_route_equals_python_route(monkeypatch):
    """The C++ route and the Python route around the same entry points: the same bits."""
    import delta_matching_b200 as dm
    from delta_matching_b200 import _lib
    m = _example()
    layer = m.Layer(256, 4, 2, 128)
    native = m.generate(layer, _prompts([5, 40, 64]), 60, 80, 48, 16)
    monkeypatch.setattr(_lib, "_CACHE_ROUTE", _lib._NoCacheRoute)
    python = m.generate(layer, _prompts([5, 40, 64]), 60, 80, 48, 16)
    assert torch.equal(native[0], python[0]) and native[1:] == python[1:]
    with pytest.raises(ValueError, match="CUDA"):
        dm.dm_cache_attn(torch.zeros(1, 1, 2, 128, dtype=torch.bfloat16), dm.KVCache8(*(t.cpu() for t in dm.KVCache8.empty(1, 32, 2, 128))),
                         torch.zeros(1, 1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32))
