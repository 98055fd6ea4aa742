"""The cache functions under a fake-tensor mode: the registered ops' shapes, with no GPU and no kernel."""
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import delta_matching_b200 as dm


def test_functions_under_a_fake_mode():
    B, N, H, Hk, D, P, T = 3, 5, 8, 2, 128, 64, 7
    with FakeTensorMode():
        new = lambda *s, d=torch.float32: torch.empty(*s, device="cuda", dtype=d)
        cache = dm.KVCache8(new(9, Hk, P, D, d=torch.float8_e4m3fn), new(9, Hk, P, D, d=torch.float8_e4m3fn), new(9, Hk, P // 32), new(9, Hk, P // 32))
        q, k = new(B, N, H, D, d=torch.bfloat16), new(B, N, Hk, D, d=torch.bfloat16)
        table, lengths, w = new(B, T, d=torch.int32), new(B, d=torch.int32), new(B, Hk, T * P)
        lengths = dm.dm_cache_append(cache, k, k, table, lengths)
        assert lengths.shape == (B,) and lengths.dtype == torch.int32
        o, lse = dm.dm_cache_attn(q, cache, table, lengths, weights=w, accumulate=True, return_lse=True)
        assert o.shape == q.shape and o.dtype == torch.bfloat16 and lse.shape == (B, H, N)
        assert dm.dm_cache_attn(q, cache, table, lengths).shape == q.shape
        n, kept, nw = dm.dm_cache_evict(cache, table, lengths, w, new(B, 2, d=torch.int32), 100, 10)
        assert n.shape == (B,) and kept.shape == (B, Hk, 100) and nw.shape == (B, Hk, 2 * P)
