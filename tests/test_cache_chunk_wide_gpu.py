"""Attention over the cache for many new tokens at once at head_dim 256 (the tcgen05 form: units of 128 rows, the keys of a tile shared by two groups of
warps) against its definition in 64 bits.  The bounds are those of tests/cache_ref.py."""
import pytest
import torch

import delta_matching_b200 as dm
from delta_matching_b200 import ops

from . import cache_ref as ref
from .test_cache_gpu import _check, _filled, _ints, _rand

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("N, rep, P", [(33, 1, 32), (48, 8, 64), (128, 1, 96), (9, 4, 160), (43, 3, 128)])
def test_units(N, rep, P, causal):
    """33 and more rows: part of a row tile, whole ones, several; lengths below, at and above the counts."""
    lengths = [700, N, 400, N + 129, 5]
    counts = [N, N, N // 2, N - 1, N]
    cache, pools, table = _filled(lengths, P, 2, 256, seed=N)
    q = _rand(torch.Generator().manual_seed(N), len(lengths), N, 2 * rep, 256)
    _check(q, cache, pools, table, lengths, counts, causal, weights=N != 128)


@pytest.mark.parametrize("n", [65, 1999])
def test_one_sequence_is_cut(n):
    """One head's keys divided over many CTAs: every row joined from pieces, some of which a row does not see."""
    cache, pools, table = _filled([n], 64, 1, 256, seed=n)
    q = _rand(torch.Generator().manual_seed(n), 1, 64, 1, 256)
    _check(q, cache, pools, table, [n])


@pytest.mark.parametrize("kscale, vscale, qscale, scale", [(1e-20, 1.0, 1e20, None), (1.0, 1e-30, 1.0, None), (1.0, 1e30, 1.0, None), (30.0, 1.0, 30.0, None),
                                                           (1.0, 1.0, 1.0, 3.0), (1.0, 1.0, 1e-30, None)])
def test_ranges(kscale, vscale, qscale, scale):
    lengths = [450, 97]
    cache, pools, table = _filled(lengths, 32, 1, 256, kscale=kscale, vscale=vscale)
    q = _rand(torch.Generator().manual_seed(1), 2, 14, 3, 256, scale=qscale)
    q[0, 0, 1] = 0                                               # a query of zeros sees all keys alike
    _check(q, cache, pools, table, lengths, scale=scale, weights=True)


def test_blocks_of_very_different_size():
    """V blocks 2^-100 ... 2^100 of one another and blocks of zeros, in an order that makes the running scale jump; a key that takes all; maxima that
    rise from tile to tile, and in one half of a tile alone."""
    B, Hk, D, P, n = 4, 1, 256, 32, 32 * 21 + 5
    cache = ref.make_cache(B * 22, P, Hk, D)
    table = ref.make_table(B, 22, B * 22)
    g = torch.Generator().manual_seed(8)
    k, v, q = _rand(g, B, n, Hk, D), _rand(g, B, n, Hk, D), _rand(g, B, 10, 4, D)
    for j, e in enumerate((0, -100, 3, 100, -3, -40, 40, 0, 20, -20, 99, 1, -99, 0, 7, -7, 30, -30, 2, 60, -60, 101)):
        v[0, 32 * j:32 * j + 32] *= 2.0 ** e
    v[1, 64:300] = 0
    k[1, 96:160] = 0
    k[1, 400] *= 40
    k[2] *= torch.linspace(0.1, 6.0, n)[:, None, None].to(k.dtype)
    for t in range(5):                                           # keys 64 ... 127 of even tiles, 0 ... 63 of odd ones
        k[3, 128 * t + (64 if t % 2 == 0 else 0):128 * t + (128 if t % 2 == 0 else 64)] *= t + 2
    dm.dm_cache_append(cache, k.cuda(), v.cuda(), table.cuda(), _ints([0] * B).cuda())
    _check(q, cache, ref.Pools(cache), table, [n] * B)
    _check(q, cache, ref.Pools(cache), table, [32 * 3, 32 * 6 + 1, 400, 520])


def test_nan_inputs():
    """A NaN among the held values or in a query reaches the rows that see it and no others."""
    lengths, N, rep = [300, 300], 24, 2
    cache, pools, table = _filled(lengths, 32, 1, 256)
    q = _rand(torch.Generator().manual_seed(2), 2, N, rep, 256).cuda()
    clean = dm.dm_cache_attn(q, cache, table.cuda(), _ints(lengths).cuda())
    bad = q.clone()
    bad[0, 3, 1, 200] = float("nan")
    o = dm.dm_cache_attn(bad, cache, table.cuda(), _ints(lengths).cuda())
    want = torch.zeros_like(o, dtype=torch.bool)
    want[0, 3, 1] = True
    assert torch.equal(o.isnan(), want) and torch.equal(o[~want], clean[~want])
    for j in (280, 200):                                         # keys of a tile's first half and of another's second
        cache.k8.view(torch.uint8)[int(table[1, j // 32]), 0, j % 32, 3] = 0x7F
        o = dm.dm_cache_attn(q, cache, table.cuda(), _ints(lengths).cuda())
        assert torch.equal(o[0], clean[0])
        seen = torch.arange(N) + 300 - N >= j                    # the tokens whose causal view reaches it
        assert torch.equal(o[1].isnan().all(-1).all(-1).cpu(), seen) and torch.equal(o[1].isnan().any(-1).any(-1).cpu(), seen)


def test_repeats_bit_for_bit():
    lengths = [1900, 117, 833]
    cache, pools, table = _filled(lengths, 64, 2, 256)
    q = _rand(torch.Generator().manual_seed(4), 3, 70, 8, 256).cuda()
    t, n = table.cuda(), _ints(lengths).cuda()

    def call():
        w = torch.full((3, 2, table.shape[1] * 64), 7.0, device="cuda")
        return (*dm.dm_cache_attn(q, cache, t, n, weights=w, return_lse=True), w)

    first = call()
    for _ in range(10):
        assert all(torch.equal(a, b) for a, b in zip(call(), first))
    ops.check_status("cuda")


def test_bad_device_values_are_reported():
    cache, pools, table = _filled([40, 40], 32, 1, 256)
    q = torch.randn(2, 20, 2, 256, device="cuda", dtype=torch.bfloat16)
    n = _ints([40, 40]).cuda()
    for bad_table, bad_n, counts, says in ((_ints([[0, 99], [1, 2]]), n, None, "page"), (_ints([[0, -1], [1, 2]]), n, None, "page"),
                                           (table, _ints([40, 1000]).cuda(), None, "length"), (table, n, _ints([1, 70]).cuda(), "length")):
        dm.dm_cache_attn(q, cache, bad_table.cuda(), bad_n, q_counts=counts)
        with pytest.raises(RuntimeError, match=says):
            ops.check_status("cuda")


@pytest.mark.parametrize("B, Hk, rep, N, lo, hi", [(6, 8, 4, 9, 3000, 4100), (5, 8, 3, 43, 2900, 4097)])
def test_long_pieces(B, Hk, rep, N, lo, hi):
    lengths = [lo + (hi - lo) * b // (B - 1) for b in range(B)]
    counts = [N - b % 3 for b in range(B)]
    cache, pools, table = _filled(lengths, 64, Hk, 256, seed=N)
    q = _rand(torch.Generator().manual_seed(N), B, N, Hk * rep, 256).cuda()
    o, lse = dm.dm_cache_attn(q, cache, table.cuda(), _ints(lengths).cuda(), q_counts=_ints(counts).cuda(), return_lse=True)
    ops.check_status("cuda")
    want, off = ref.attention_on_device(q, cache, table, lengths, counts, True, 256 ** -0.5)
    assert bool(((o.double() - want[0]).abs() <= off[0]).all())
    seen = want[1] > -torch.inf
    assert torch.equal(lse > -torch.inf, seen) and bool(((lse.double() - want[1])[seen].abs() <= off[1][seen]).all())
