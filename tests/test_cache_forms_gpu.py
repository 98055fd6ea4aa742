"""Attention and weights over the whole range of calls: sums that go on in every form, more sequences than the divisions of the work have entries, and random calls.  Against
64 bits on the GPU, with the bounds of tests/cache_ref.py (attention)."""
import math
import random

import pytest
import torch

import delta_matching_b200 as dm
from delta_matching_b200 import ops

from .test_cache_gpu import _filled, _ints, _rand

pytestmark = pytest.mark.gpu


def _reference(q, cache, table, lengths, counts, causal, scale):
    """-> (o, lse, weights) and bounds; weights (B, Hk, T * page)."""
    B, N, H, D = q.shape
    Hk, P = cache.k8.shape[1:3]
    rep = H // Hk
    new = lambda *s, fill=0.0: torch.full(s, fill, dtype=torch.float64, device="cuda")
    o, do, lse, dlse = new(B, N, H, D), new(B, N, H, D), new(B, H, N, fill=-math.inf), new(B, H, N)
    w, dw = new(B, Hk, table.shape[1] * P), new(B, Hk, table.shape[1] * P)
    for b in range(B):
        n, count = int(lengths[b]), int(counts[b])
        if n == 0 or count == 0:
            continue
        at = torch.arange(n, device="cuda")
        page, slot = table[b].cuda().long()[at // P], at % P
        see = (at[None] < ((n - count + 1 + torch.arange(count, device="cuda")).clamp(min=0)[:, None] if causal else n)).expand(count, n)
        for h in range(Hk):
            k, v = (c[page, h, slot].float().double() * s[page, h, slot // 32].double()[:, None] for c, s in ((cache.k8, cache.ks), (cache.v8, cache.vs)))
            coarsest = float(cache.vs[page, h, slot // 32].max())
            qi = q[b, :count, h * rep:(h + 1) * rep].double().transpose(0, 1)                # (rep, count, D)
            s = (qi @ k.T * scale).masked_fill(~see, -math.inf)
            eps = ((qi.abs() @ k.abs().T) * scale).masked_fill(~see, 0.0).amax(2) * 2.0 ** -19
            l = torch.logsumexp(s, 2)
            p = torch.nan_to_num(torch.softmax(s, 2))
            heads = slice(h * rep, (h + 1) * rep)
            lse[b, heads, :count] = l
            off = torch.where(see.any(1), 2.0 ** -19 + 2.0 ** -22 * l.nan_to_num(neginf=0.0).abs(), 0.0)
            dlse[b, heads, :count] = torch.where(see.any(1), eps, 0.0) + off
            x = p @ v
            o[b, :count, heads] = x.transpose(0, 1)
            do[b, :count, heads] = (2.0 ** -8 * x.abs() + (2.0 ** -11 + 2 * eps + 2.0 ** -19)[..., None] * (p @ v.abs()) + (2.0 ** -40 * see.sum(1) * 448 * coarsest + 1e-37)[None, :, None]).transpose(0, 1)
            w[b, h, :n] = p.sum((0, 1))
            dw[b, h, :n] = ((2 * eps + off)[..., None] * p + 1e-37).sum((0, 1))
    return (o, lse, w), (do, dlse, dw)


def _check(q, cache, table, lengths, counts, causal, weights, accumulate=False, strided=False, wide=0, scale=None):
    """One call against 64 bits.  weights: wanted; strided: as a view of a larger tensor; wide: further entries."""
    B, N, H, D = q.shape
    Hk, P = cache.k8.shape[1:3]
    W = table.shape[1] * P + wide
    g = torch.Generator(device="cuda").manual_seed(N)
    store = torch.rand(B, Hk, 2, W, generator=g, device="cuda") if strided else torch.rand(B, Hk, 1, W, generator=g, device="cuda")
    before, view = store.clone(), store[:, :, -1]
    if not accumulate:
        view.fill_(math.nan)
    o, lse = dm.dm_cache_attn(q, cache, table.cuda(), _ints(lengths).cuda(), q_counts=_ints(counts).cuda(), causal=causal, softmax_scale=scale,
                              weights=view if weights else None, accumulate=accumulate and weights, return_lse=True)
    ops.check_status("cuda")
    want, off = _reference(q, cache, table, lengths, counts, causal, scale or D ** -0.5)
    seen = want[1] > -math.inf
    assert bool(((o.double() - want[0]).abs() <= off[0]).all()), float(((o.double() - want[0]).abs() / off[0].clamp(min=1e-300)).max())
    assert torch.equal(lse > -math.inf, seen) and bool(((lse.double() - want[1]).abs()[seen] <= off[1][seen]).all())
    if weights:
        add, bound = (torch.nn.functional.pad(t, (0, wide)) for t in (want[2], off[2]))
        base = before[:, :, -1].double() if accumulate else torch.zeros_like(add)
        # the sum in fp32, rounded once more where it is added
        assert bool(((view.double() - base - add).abs() <= bound + 2.0 ** -23 * (base + add)).all())
        held = torch.arange(W, device="cuda")[None] < _ints(lengths).cuda()[:, None]
        assert torch.equal(view.masked_select(~held[:, None].expand(-1, Hk, -1)), (before[:, :, -1] if accumulate else torch.zeros_like(before[:, :, -1])).masked_select(~held[:, None].expand(-1, Hk, -1)))
        if strided:
            assert torch.equal(store[:, :, 0], before[:, :, 0])


@pytest.mark.parametrize("D, N, rep", [(128, 1, 4), (128, 5, 1), (128, 5, 4), (128, 9, 4), (128, 60, 5), (256, 5, 1), (256, 17, 1), (256, 60, 5)])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("accumulate", [False, True])
def test_weights_of_every_form(accumulate, causal, D, N, rep):
    """5, 20, 36 and 300 rows and more: set and added to, in a part of a wider tensor, with idle and empty sequences, lengths off a tile's edge."""
    lengths, counts = [333, 0, 130, 127, 40, 64], [N, N, 0, max(1, N // 2), N, 1]
    cache, _, table = _filled(lengths, 32, 2, D, seed=N)
    q = _rand(torch.Generator().manual_seed(N), len(lengths), N, 2 * rep, D).cuda()
    _check(q, cache, table, lengths, counts, causal, True, accumulate, strided=True, wide=77)


@pytest.mark.parametrize("B", [129, 150, 300])
@pytest.mark.parametrize("D, N, rep, most", [(128, 1, 2, 90), (128, 1, 2, 2600), (128, 9, 4, 200), (128, 7, 3, 90), (256, 9, 2, 200)])
def test_more_sequences_than_entries(B, D, N, rep, most):
    """Both divisions of the work group sequences from 129 on; lengths of all sizes beside one another, empty ones among them."""
    rng = random.Random(B)
    lengths = [rng.choice([0, 1, 31, 32, 33, rng.randint(0, most), rng.randint(0, most)]) for _ in range(B)]
    lengths[B // 2] = most
    counts = [rng.choice([N, N, 0, rng.randint(0, N)]) for _ in range(B)]
    cache, _, table = _filled(lengths, 32, 1, D, seed=B)
    q = _rand(torch.Generator().manual_seed(B), B, N, rep, D).cuda()
    _check(q, cache, table, lengths, counts, True, weights=True)


@pytest.mark.parametrize("seed", range(24))
def test_random_calls(seed):
    rng = random.Random(seed)
    D, Hk, P = rng.choice([128, 128, 256]), rng.randint(1, 3), rng.choice([32, 64, 96, 160])
    rep = rng.choice([1, 2, 3, 4, 5, 8, 17])
    N = rng.choice([1, 1, 2, 3, rng.randint(2, 12), rng.randint(9, 150)])
    B, most = rng.randint(1, 9), rng.choice([40, 300, 2500])
    lengths = [rng.choice([0, 1, rng.randint(0, most), rng.randint(0, most), most]) for _ in range(B)]
    counts = [rng.choice([N, N, rng.randint(0, N)]) for _ in range(B)]
    cache, _, table = _filled(lengths, P, Hk, D, seed=seed, layout=rng.choice(["dense", "joint", "slots"]), T=max(1, -(-max(lengths) // P)) + rng.choice([0, 0, 3]))
    q = (_rand(torch.Generator().manual_seed(seed), B, N, Hk * rep, D) * rng.choice([1.0, 1.0, 4.0])).cuda()
    _check(q, cache, table, lengths, counts, rng.random() < 0.7, rng.random() < 0.6, rng.random() < 0.5, rng.random() < 0.5, rng.choice([0, 0, 5, 200]), rng.choice([None, None, 0.3]))
