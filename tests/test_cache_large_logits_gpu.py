"""Attention where logits are so large that fp32 no longer counts in ones: a row whose best key is ahead by more than the logits' rounding gets that key's value and
weight, and nothing is ever infinite, out of the values' range, or a weight above one."""
import pytest
import torch

import delta_matching_b200 as dm
from delta_matching_b200 import ops

from . import cache_ref as ref
from .test_cache_gpu import _ints

pytestmark = pytest.mark.gpu
BF = torch.bfloat16
ROWS = {128: [(1, 3), (3, 5), (10, 2), (9, 4), (70, 4)], 256: [(1, 5), (4, 4), (9, 2), (45, 3)]}


@pytest.mark.parametrize("D, N, rep", [(D, N, rep) for D in ROWS for N, rep in ROWS[D]])
@pytest.mark.parametrize("size", [2.0 ** 20, 2.0 ** 23, 2.0 ** 25, 2.0 ** 27, 2.0 ** 34, 2.0 ** 60])
@pytest.mark.parametrize("sign", [1, -1])
def test_the_best_key_takes_all(size, sign, D, N, rep):
    B, Hk, n = 2, 2, 32 * 13 + N
    g = torch.Generator().manual_seed(N)
    k, v, q = torch.zeros(B, n, Hk, D), torch.randn(B, n, Hk, D, generator=g), torch.zeros(B, N, rep * Hk, D)
    best = [37, 290]                                             # of sequence b; seen by every row
    # the logit of key j is (its element 0) * q's: from -1 to -2 (or 1 to 2) times `size`, the best one's -0.5 (4)
    q[..., 0] = size * D ** 0.5 / 1.4426950408889634
    k[..., 0] = sign * (1 + torch.arange(n) % 7 / 7.0)[None, :, None]
    for b in range(B):
        k[b, best[b], :, 0] = 4.0 if sign > 0 else -0.5
        v[b, 32 * 5:32 * 6] *= 2.0 ** (30 * b)                   # and one block's values are far larger
    T, P = -(-n // 64), 64
    cache = ref.make_cache(B * T, P, Hk, D)
    table = ref.make_table(B, T, B * T)
    lengths = dm.dm_cache_append(cache, k.to(BF).cuda(), v.to(BF).cuda(), table.cuda(), _ints([0] * B).cuda())
    w = torch.zeros(B, Hk, T * P, device="cuda")
    o, lse = dm.dm_cache_attn(q.to(BF).cuda(), cache, table.cuda(), lengths, weights=w, return_lse=True)
    ops.check_status("cuda")
    for b in range(B):
        at = best[b]
        page = int(table[b, at // P])
        want = cache.v8[page, :, at % P].float() * cache.vs[page, :, at % P // 32][:, None]
        want = want.repeat_interleave(rep, 0).to(BF)[None].expand(N, -1, -1)
        assert torch.equal(o[b], want)                           # the others' weights are below 2^-2^19
        top = q.to(BF).double() [b, 0, 0, 0] * (4.0 if sign > 0 else -0.5) * D ** -0.5
        assert bool(((lse[b].double().cpu() - top).abs() <= 2.0 ** -18 * top.abs()).all())
        others = w[b].clone()
        others[:, at] = 0
        assert not bool(others.any())
        assert bool((w[b, :, at] > 0).all()) and bool((w[b, :, at] <= N * rep * (1 + 2.0 ** -10)).all())
        if size <= 2.0 ** 20:                                    # beyond, the second kernel of many rows makes the logit itself a second time, a rounding off
            assert torch.allclose(w[b, :, at], torch.tensor(float(N * rep), device="cuda"), rtol=0.25)


@pytest.mark.parametrize("D, N, rep", [(D, N, rep) for D in ROWS for N, rep in ROWS[D]])
@pytest.mark.parametrize("size", [2.0 ** 22, 2.0 ** 26, 2.0 ** 33, 2.0 ** 70])
def test_close_ones_stay_a_mean(size, D, N, rep):
    """Logits that differ by a few roundings: whatever they come to, the result is a mean of what is seen."""
    B, Hk, n = 2, 1, 32 * 9 + N
    g = torch.Generator().manual_seed(N)
    k, v, q = torch.randn(B, n, Hk, D, generator=g) * 2.0 ** -20, torch.rand(B, n, Hk, D, generator=g) + 0.5, torch.randn(B, N, rep * Hk, D, generator=g)
    k[..., 0] = 1.0
    q[..., 0] = size
    T, P = -(-n // 32), 32
    cache = ref.make_cache(B * T, P, Hk, D)
    table = ref.make_table(B, T, B * T)
    lengths = dm.dm_cache_append(cache, k.to(BF).cuda(), v.to(BF).cuda(), table.cuda(), _ints([0] * B).cuda())
    w = torch.zeros(B, Hk, T * P, device="cuda")
    o = dm.dm_cache_attn(q.to(BF).cuda(), cache, table.cuda(), lengths, weights=w)
    ops.check_status("cuda")
    held = cache.v8.float() * cache.vs.repeat_interleave(32, 2)[..., None]
    low, high = 0.4, float(held[held.isfinite()].max())
    assert bool((o.float() >= low * (1 - 2.0 ** -7)).all()) and bool((o.float() <= high * (1 + 2.0 ** -7)).all())
    assert bool(w.isfinite().all()) and bool((w >= 0).all()) and bool((w <= N * rep * (1 + 2.0 ** -10)).all())
