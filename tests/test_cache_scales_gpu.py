"""Attention over blocks whose V scales lie far apart: a row's result has the bits of what it sees and weighs, whatever the scale of other blocks.

Bound of an element of o, against 64 bits: bf16's rounding, 2^-8 of the value; a logit off by at most eps = 2^-19 of the sum of its terms' sizes, a probability
by twice that, exp2 and the sums by 2^-19, p in f16 by 2^-11 of itself: (2^-11 + 2 eps + 2^-19) sum p |v|; and f16's smallest step: products of a
probability and its V scale are held below 2^16 with the row's largest at 2^11 or more, values off by up to 2^-25, so each by 2^-36 of the
largest, times a code of up to 448, summed over the keys that the row sees."""
import math

import pytest
import torch

import delta_matching_b200 as dm
from delta_matching_b200 import ops

from . import cache_ref as ref
from .test_cache_gpu import _ints

pytestmark = pytest.mark.gpu
BF = torch.bfloat16

# rows of a call (new tokens, heads of the group): the forms for few and many rows
ROWS = {128: [(1, 3), (3, 5), (10, 2), (9, 4), (70, 4)], 256: [(1, 5), (4, 4), (9, 2), (45, 3)]}
CASES = [(D, N, rep) for D in ROWS for N, rep in ROWS[D]]


def _cache(k, v, P, seed):
    """Pools with the tokens k, v (B, n, Hk, D)."""
    B, n, Hk, D = k.shape
    T = -(-n // P)
    cache = ref.make_cache(B * T + 1, P, Hk, D)
    table = ref.make_table(B, T, B * T + 1, seed)
    dm.dm_cache_append(cache, k.cuda(), v.cuda(), table.cuda(), torch.zeros(B, dtype=torch.int32, device="cuda"))
    ops.check_status("cuda")
    return cache, table


def _check(q, cache, table, n, causal=True):
    """All rows of one sequence after the other against 64 bits."""
    B, N, H, D = q.shape
    Hk, P = cache.k8.shape[1:3]
    o, lse = dm.dm_cache_attn(q.cuda(), cache, table.cuda(), _ints([n] * B).cuda(), causal=causal, return_lse=True)
    ops.check_status("cuda")
    at = torch.arange(n, device="cuda")
    worst = 0.0
    for b in range(B):
        page = table[b].cuda().long()[at // P]
        limit = (n - N + 1 + torch.arange(N, device="cuda")).clamp(min=0) if causal else torch.full((N,), n, device="cuda")
        see = at[None] < limit[:, None]
        for h in range(H):
            hk = h * Hk // H
            (k, _), (v, vs) = ((c[page, hk, at % P].double(), s[page, hk, at % P // 32].double()[:, None]) for c, s in ((cache.k8.float(), cache.ks), (cache.v8.float(), cache.vs)))
            k, v = k * cache.ks[page, hk, at % P // 32].double()[:, None], v * vs
            qi = q[b, :, h].cuda().double()
            s = ((qi @ k.T) * D ** -0.5).masked_fill(~see, -math.inf)
            eps = ((qi.abs() @ k.abs().T) * D ** -0.5).masked_fill(~see, 0.0).amax(1) * 2.0 ** -19
            p = torch.nan_to_num(torch.softmax(s, 1))
            want = p @ v
            off = 2.0 ** -8 * want.abs() + (2.0 ** -11 + 2 * eps + 2.0 ** -19)[:, None] * (p @ v.abs()) + (2.0 ** -36 * see.sum(1) * 448 * (p * vs.T).amax(1))[:, None] + 1e-37
            err = (o[b, :, h].double() - want).abs()
            assert bool((err <= off).all()), (b, h, float((err / off).max()), (err > off).nonzero()[0].tolist())
            worst = max(worst, float((err / off).max()))
    return o


@pytest.mark.parametrize("D, N, rep", CASES)
@pytest.mark.parametrize("far", [12, 33, 41, 70, 110])
def test_a_coarse_block_without_weight_costs_nothing(far, D, N, rep):
    """Blocks 3 and 7 have values 2^far of the others' and keys that no query looks at."""
    n, Hk = 32 * 10 + 3 + N, 2
    g = torch.Generator().manual_seed(far)
    k, v, q = (torch.randn(2, m, h, D, generator=g) for m, h in ((n, Hk), (n, Hk), (N, rep * Hk)))
    k[..., 0] = 0.0
    q[..., 0] = 60.0
    for blk in (3, 7):
        k[:, 32 * blk:32 * blk + 32, :, 0] = -60.0               # logits 3600 / sqrt(D) below the others'
        v[0, 32 * blk:32 * blk + 32] *= 2.0 ** far
    v *= 2.0 ** -60
    cache, table = _cache(k.to(BF), v.to(BF), 64, far)
    _check(q.to(BF), cache, table, n)


@pytest.mark.parametrize("D, N, rep", [c for c in CASES if c[1] > 1])
@pytest.mark.parametrize("far", [12, 33, 41, 70, 110])
def test_a_coarse_block_that_a_row_does_not_see_costs_nothing(far, D, N, rep):
    """The last new token, alone in its block, has a V of 2^far of the others': earlier rows are as they are without it."""
    n, Hk = 32 * 9 + 1, 1
    g = torch.Generator().manual_seed(far)
    k, v, q = (torch.randn(2, m, h, D, generator=g) for m, h in ((n, Hk), (n, Hk), (N, rep * Hk)))
    v *= 2.0 ** -60
    small = _cache(k.to(BF), v.to(BF), 32, far)
    v[:, n - 1] *= 2.0 ** far
    large = _cache(k.to(BF), v.to(BF), 32, far)
    a, b = (_check(q.to(BF), *c, n) for c in (small, large))
    assert torch.allclose(a[:, :-1].double(), b[:, :-1].double(), rtol=2.0 ** -6, atol=2.0 ** -66)


@pytest.mark.parametrize("D, N, rep", CASES)
@pytest.mark.parametrize("causal", [True, False])
def test_scales_in_any_order(D, N, rep, causal):
    """Scales that jump between 2^-100 and 2^90 from block to block, with weight that favours fine blocks, coarse ones, or neither."""
    Hk, n = 1, 32 * 21 + 5
    g = torch.Generator().manual_seed(8)
    B = 3
    k, v, q = (torch.randn(B, m, h, D, generator=g) for m, h in ((n, Hk), (n, Hk), (N, rep * Hk)))
    k[..., 0] = 0.0
    q[..., 0] = 4.0
    for j, e in enumerate((0, -100, 3, 90, -3, -40, 40, 0, 20, -20, 89, 1, -99, 0, 7, -7, 30, -30, 2, 60, -60, 88)):
        v[:, 32 * j:32 * j + 32] *= 2.0 ** e
        k[0, 32 * j:32 * j + 32, :, 0] = -0.17 * e * D ** 0.5    # logits fall by log 2 for every power of two that V rises: products alike
        k[1, 32 * j:32 * j + 32, :, 0] = -0.3 * e * D ** 0.5
    cache, table = _cache(k.to(BF), v.to(BF), 32, 5)
    _check(q.to(BF), cache, table, n, causal)
    _check(q.to(BF), cache, table, 32 * 6 + 1, causal)


@pytest.mark.parametrize("D, N, rep", CASES)
def test_a_coarse_block_of_tiny_weight_counts(D, N, rep):
    """Its probability times its scale is what the others' are, though its probability is 2^-45 of theirs."""
    n, Hk = 32 * 10 + N, 1
    g = torch.Generator().manual_seed(3)
    k, v, q = (torch.randn(1, m, h, D, generator=g) * 0.1 for m, h in ((n, Hk), (n, Hk), (N, rep * Hk)))
    k[..., 0], q[..., 0] = 0.0, 1.0
    k[:, 96:128, :, 0] = -45 * math.log(2.0) * D ** 0.5
    v[:, 96:128] *= 2.0 ** 45
    cache, table = _cache(k.to(BF), v.to(BF), 64, 3)
    _check(q.to(BF), cache, table, n)
