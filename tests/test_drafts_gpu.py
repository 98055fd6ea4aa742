"""The functions for drafted tokens against their definitions in 64 bits (tests/drafts_ref.py)."""
import math
import os
import subprocess
import sys

import pytest
import torch

import delta_matching_b200 as dm
from delta_matching_b200 import _lib, ops

from . import cache_ref as ref
from . import drafts_ref as dref
from .test_cache_gpu import _filled, _ints, _rand

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


@pytest.fixture(params=["native", "python"])
def route(request, monkeypatch):
    if request.param == "python":
        monkeypatch.setattr(_lib, "native_cache", lambda: _lib._NoCacheRoute)


# ------------------------------------------------------------------------------------------------------------------ tree
@pytest.mark.parametrize("kind", ["chain", "star", "roots", "near", "any"])
@pytest.mark.parametrize("N", [1, 2, 31, 32, 33, 63, 100, 255, 511, 1024])
def test_tree(N, kind):
    B = 3
    parents = dref.make_parents(kind, B, N, seed=N)
    for counts in (None, _ints([N, N // 2, 0])):
        got = dm.dm_draft_tree(parents.cuda(), None if counts is None else counts.cuda())
        ops.check_status("cuda")
        depth, see = dref.tree(parents, [N] * B if counts is None else counts)
        assert torch.equal(got.depth.cpu(), depth) and torch.equal(got.seen.cpu(), dref.pack(see))
        assert (got.counts is None) == (counts is None)


def test_tree_of_a_part(route):
    """Parents that are a part of a wider tensor, and one row for all."""
    parents = dref.make_parents("any", 4, 70, seed=1)
    wide = torch.full((4, 90), 99, dtype=torch.int32)
    wide[:, 7:77] = parents
    one = dref.make_parents("near", 1, 70).cuda()
    for got, of in ((dm.dm_draft_tree(wide.cuda()[:, 7:77]), parents), (dm.dm_draft_tree(parents.t().contiguous().cuda().t()), parents),
                    (dm.dm_draft_tree(one.expand(4, -1)), one.cpu().expand(4, -1))):
        depth, see = dref.tree(of, [70] * 4)
        assert torch.equal(got.depth.cpu(), depth) and torch.equal(got.seen.cpu(), dref.pack(see))
    ops.check_status("cuda")


def test_bad_parents_are_reported():
    for at, parent in ((3, 3), (3, 4), (0, 0), (5, -2), (2, 1 << 30)):
        parents = dref.make_parents("chain", 2, 9)
        parents[1, at] = parent
        got = dm.dm_draft_tree(parents.cuda())
        with pytest.raises(RuntimeError, match="parent"):
            ops.check_status("cuda")
        parents[1, at] = -1
        assert torch.equal(got.depth.cpu(), dref.tree(parents, [9, 9])[0])
    parents = dref.make_parents("chain", 2, 9)
    parents[1, 6] = 77                                           # behind the count: not looked at
    dm.dm_draft_tree(parents.cuda(), _ints([9, 6]).cuda())
    ops.check_status("cuda")


# ---------------------------------------------------------------------------------------------------------------- append
def _appended(cache, pools, table, q, k, v, lengths, freqs, offsets, counts, interleaved):
    """One call against the definition: the bits of values and untouched slots, the rotated within half a step of their format."""
    B, N, Hk, D = k.shape
    P = cache.k8.shape[2]
    before = ref.Pools(cache)
    all_ = _ints([N] * B) if counts is None else counts
    out, new = dm.dm_cache_append_rotary(cache, q.cuda(), k.cuda(), v.cuda(), table.cuda(), lengths.cuda(), freqs.cuda(), None if offsets is None else offsets.cuda(),
                                         None if counts is None else counts.cuda(), interleaved)
    ops.check_status("cuda")
    assert torch.equal(new.cpu(), lengths + all_)
    positions = lengths[:, None].long() + (torch.arange(N) if offsets is None else offsets.long())
    want, off = dref.rotate(q, positions, freqs, interleaved)
    real = (torch.arange(N) < all_[:, None])[..., None, None]
    want, off = want * real, off * real
    got = out.cpu().double()
    assert bool(((got - want).abs() <= 2.0 ** -8 * want.abs() + off * 1.01).all())
    # values, and what is not written: as the plain append; keys: within half a step of e4m3, on the scale of their exact values
    ref.append(before, (k, v), table, lengths, all_)
    now = ref.Pools(cache)
    assert torch.equal(now.codes[1], before.codes[1]) or ref.same_values(dm.KVCache8(cache.v8, cache.v8, cache.vs, cache.vs), _twice(before, 1))
    turned, key_off = dref.rotate(k, positions, freqs, interleaved)
    for b in range(B):
        for h in range(Hk):
            j, end = int(lengths[b]), int(lengths[b]) + int(all_[b])
            while j < end:
                stop = min(end, j - j % 32 + 32)
                page, slot, blk = int(table[b, j // P]), j % P, j % P // 32
                y, y_off = (x[b, j - int(lengths[b]):stop - int(lengths[b]), h] for x in (turned, key_off))
                s = ref.scale_of(float(y.abs().max()))
                if j % 32:
                    old = float(pools.scales[0][page, h, blk])
                    s = max(s, old)
                    rows = slice(blk * 32, slot)
                    was = pools.codes[0][page, h, rows].view(torch.float8_e4m3fn).double() * (old / s)
                    kept = now.codes[0][page, h, rows].view(torch.float8_e4m3fn).double()
                    assert bool(((kept == ref.grid(was)) | (kept.isnan() & was.isnan())).all())
                assert float(now.scales[0][page, h, blk]) == s
                got = now.codes[0][page, h, slot:slot + stop - j].view(torch.float8_e4m3fn).double() * s
                step = torch.exp2(torch.floor(torch.log2((y.abs() / s).clamp(min=2.0 ** -6))) - 3) * s
                assert bool(((got - y).abs() <= step / 2 + y_off * 1.01).all())
                j = stop
    return out, new


def _twice(pools, which):
    """Pools whose K and V are both one of theirs."""
    x = object.__new__(ref.Pools)
    x.codes, x.scales = [pools.codes[which]] * 2, [pools.scales[which]] * 2
    return x


def _freqs(F, base=10000.0):
    return (base ** (-torch.arange(F, dtype=torch.float64) / F)).float()


@pytest.mark.parametrize("D, F, interleaved", [(128, 64, False), (128, 32, True), (128, 8, False), (128, 56, True), (256, 128, False), (256, 128, True), (256, 40, False)])
@pytest.mark.parametrize("N, P, layout", [(1, 32, "dense"), (33, 96, "joint"), (70, 64, "slots")])
def test_append_rotary(N, P, layout, D, F, interleaved):
    """Starts on, before and behind a block's edge, whole and ragged, positions by index and by tree."""
    B, Hk, H = 4, 2, 6
    lengths = _ints([0, 1, 31, 40])
    T = -(-(40 + N) // P)
    for offsets, ragged in ((None, False), ("tree", True)):
        cache, pools, table = _filled(lengths.tolist(), P, Hk, D, seed=N, layout=layout, T=T)
        g = torch.Generator().manual_seed(N)
        q, k, v = _rand(g, B, N, H, D), _rand(g, B, N, Hk, D, scale=3.0), _rand(g, B, N, Hk, D)
        off = None if offsets is None else dref.tree(dref.make_parents("any", B, N), [N] * B)[0]
        _appended(cache, pools, table, q, k, v, lengths, _freqs(F), off, _ints([N, max(0, N - 1), N // 2, 0]) if ragged else None, interleaved)


@pytest.mark.parametrize("D, F, interleaved", [(128, 64, False), (256, 96, True)])
@pytest.mark.parametrize("B, N", [(1, 4099), (2, 2100)])
def test_append_rotary_of_prompts(B, N, D, F, interleaved):
    """From 4096 tokens on more rows are in flight; ragged, behind a start inside a block."""
    lengths = _ints([17, 0][:B])
    cache, pools, table = _filled(lengths.tolist(), 64, 2, D, T=-(-(17 + N) // 64))
    g = torch.Generator().manual_seed(N)
    _appended(cache, pools, table, _rand(g, B, N, 4, D), _rand(g, B, N, 2, D, scale=3.0), _rand(g, B, N, 2, D), lengths, _freqs(F), None, _ints([N - 5, N][:B]), interleaved)


@pytest.mark.parametrize("start", [100003, (1 << 24) + 1])
def test_append_rotary_far_positions(start):
    """Angles of far positions, where 32 bits would have lost them: the pages before are one and the same."""
    pages = 2
    cache = ref.make_cache(pages, 32, 1, 128)
    table = torch.zeros(1, -(-(start + 40) // 32), dtype=torch.int32)
    table[0, start // 32:] = _ints([1, 0, 1])[:table.shape[1] - start // 32]
    g = torch.Generator().manual_seed(5)
    q, k, v = _rand(g, 1, 3, 2, 128), _rand(g, 1, 3, 1, 128), _rand(g, 1, 3, 1, 128)
    cache.ks.fill_(2.0 ** -20), cache.vs.fill_(2.0 ** -20)
    _appended(cache, ref.Pools(cache), table, q, k, v, _ints([start]), _freqs(64, 1e6), _ints([[0, 1 << 20, -5]]), None, False)


def test_append_rotary_again_and_strided(route):
    """The same call leaves the same cache; strided inputs, a part of a table and of offsets."""
    B, N, H, Hk, D = 2, 37, 4, 2, 128
    lengths = _ints([13, 64])
    g = torch.Generator().manual_seed(2)
    qkv = _rand(g, B, N, H + 2 * Hk, D, scale=5.0)
    off = dref.tree(dref.make_parents("near", B, N), [N] * B)[0]
    wide_t, wide_o = torch.full((B, 9), 99, dtype=torch.int32), torch.full((B, 50), 99, dtype=torch.int32)
    wide_o[:, 3:3 + N] = off
    cache, pools, table = _filled(lengths.tolist(), 32, Hk, D, T=6)
    wide_t[:, 2:8] = table
    x = qkv.cuda()
    args = (cache, x[:, :, :H], x[:, :, H:H + Hk], x[:, :, H + Hk:], wide_t.cuda()[:, 2:8], lengths.cuda(), _freqs(64).cuda(), wide_o.cuda()[:, 3:3 + N])
    once = dm.dm_cache_append_rotary(*args)
    kept = ref.Pools(cache)
    again = dm.dm_cache_append_rotary(*args)
    assert ref.same_values(cache, kept) and torch.equal(once[0], again[0]) and torch.equal(once[1], again[1])
    other, _, _ = _filled(lengths.tolist(), 32, Hk, D, T=6)
    out, _ = _appended(other, pools, table, qkv[:, :, :H], qkv[:, :, H:H + Hk], qkv[:, :, H + Hk:], lengths, _freqs(64), off, None, False)
    assert torch.equal(out, once[0]) and ref.same_values(other, kept)
    odd = torch.nn.functional.pad(x, (3, 2))[..., 3:3 + D]       # rows that are not aligned: copied
    third, _, _ = _filled(lengths.tolist(), 32, Hk, D, T=6)
    out3, _ = dm.dm_cache_append_rotary(third, odd[:, :, :H], odd[:, :, H:H + Hk], odd[:, :, H + Hk:], *args[4:])
    assert torch.equal(out3, out) and ref.same_values(third, kept)
    ops.check_status("cuda")


def test_append_rotary_by_nothing_is_append():
    """Frequencies of zero turn nothing: the cache of dm_cache_append, bit for bit, and q as it is; NaN and infinities too."""
    lengths = _ints([5, 40])
    g = torch.Generator().manual_seed(4)
    q, k, v = _rand(g, 2, 50, 4, 128), _rand(g, 2, 50, 2, 128, scale=9.0), _rand(g, 2, 50, 2, 128)
    k[0, 3, 0, 70], k[0, 4, 1, 127], v[1, 9, 1, 3], v[1, 8, 1, 3] = float("nan"), float("inf"), float("nan"), float("-inf")
    one, _, table = _filled(lengths.tolist(), 32, 2, 128, T=4)
    two, _, _ = _filled(lengths.tolist(), 32, 2, 128, T=4)
    dm.dm_cache_append(one, k.cuda(), v.cuda(), table.cuda(), lengths.cuda())
    out, _ = dm.dm_cache_append_rotary(two, q.cuda(), k.cuda(), v.cuda(), table.cuda(), lengths.cuda(), torch.zeros(8, device="cuda"))
    assert torch.equal(out.cpu(), q) and ref.same_values(two, ref.Pools(one))
    ops.check_status("cuda")


# ------------------------------------------------------------------------------------------------------------- attention
def _attended(q, cache, table, lengths, counts, parents, scale=None, part=None):
    """A call against the definition."""
    B, N, H, D = q.shape
    all_ = [N] * B if counts is None else counts.tolist()
    tree = dm.dm_draft_tree(parents.cuda(), None if counts is None else counts.cuda())
    o, lse = dm.dm_cache_attn_tree(q.cuda(), cache, table.cuda(), lengths.cuda(), tree, softmax_scale=scale, return_lse=True)
    ops.check_status("cuda")
    see = dref.tree(parents, all_)[1]
    want, off = dref.attention(q, cache, table, lengths, all_, see, D ** -0.5 if scale is None else scale)
    for got, w, d in ((o, want[0], off[0]), (lse, want[1], off[1])):
        same = (got.double() == w) | (got.isnan() & w.isnan())
        assert bool((same | ((got.double() - w).abs() <= d)).all()), float(((got.double() - w).abs() / d).nan_to_num(0.0).max())
    return o, lse


@pytest.mark.parametrize("D", [128, 256])
@pytest.mark.parametrize("H, Hk", [(4, 4), (6, 2), (15, 3), (16, 1)])
@pytest.mark.parametrize("N", [1, 5, 16, 33, 64, 100])
def test_attention(N, H, Hk, D):
    """Nothing before the drafts, one token, ends before, on and behind the edges of blocks, tiles and pages; whole and ragged."""
    P = 96
    before = [0, 1, 31, 96, 127, 300]
    B = len(before)
    lengths = [n + N for n in before]
    cache, _, table = _filled(lengths, P, Hk, D, seed=N + H)
    g = torch.Generator().manual_seed(N)
    q = _rand(g, B, N, H, D, scale=1.5)
    _attended(q, cache, table, _ints(lengths), None, dref.make_parents("any", B, N, seed=N))
    counts = _ints([N, max(1, N // 2), N, 1, N - 1, 0])
    full = [n + int(c) for n, c in zip(before, counts)]
    cache, _, table = _filled(full, P, Hk, D, seed=N + H, T=table.shape[1])
    o, lse = _attended(q, cache, table, _ints(full), counts, dref.make_parents("near", B, N, seed=N))
    behind = torch.arange(N) >= counts[:, None]
    assert not bool(o.cpu()[behind].any()) and bool((lse.cpu().transpose(1, 2)[behind] == -math.inf).all())


@pytest.mark.parametrize("kind", ["chain", "star", "roots"])
def test_attention_of_a_chain_is_causal(kind):
    """A chain sees what the causal attention of as many new tokens sees; the definition holds for the other extremes."""
    lengths = _ints([70, 300, 1100])
    cache, _, table = _filled(lengths.tolist(), 64, 2, 128)
    g = torch.Generator().manual_seed(1)
    q = _rand(g, 3, 24, 8, 128)
    o, lse = _attended(q, cache, table, lengths, None, dref.make_parents(kind, 3, 24))
    if kind == "chain":
        o2, lse2 = dm.dm_cache_attn(q.cuda(), cache, table.cuda(), lengths.cuda(), return_lse=True)
        assert bool(((lse - lse2).abs() < 1e-4).all()) and bool(((o.float() - o2.float()).abs() < 0.02 * o2.float().abs().amax()).all())


@pytest.mark.parametrize("N, H, Hk, D, lengths", [(7, 8, 2, 128, [5000, 9, 2500]), (40, 8, 2, 128, [6007, 41, 3333]), (256, 4, 1, 128, [3500, 257]), (64, 16, 2, 128, [4100, 64]),
                                                 (1024, 2, 1, 128, [1024, 2100]), (20, 4, 2, 256, [5003, 20, 1999]), (300, 2, 1, 256, [2000, 333]), (3, 16, 16, 256, [3001, 70])])
def test_attention_long(N, H, Hk, D, lengths):
    """Cut into many pieces; trees of up to 1024 nodes."""
    cache, _, table = _filled(lengths, 64, Hk, D, seed=N)
    g = torch.Generator().manual_seed(N)
    B = len(lengths)
    _attended(_rand(g, B, N, H, D), cache, table, _ints(lengths), None, dref.make_parents("near", B, N, seed=3))


@pytest.mark.parametrize("D", [128, 256])
@pytest.mark.parametrize("N", [3, 17, 48])
def test_attention_sees_nothing_else(N, D):
    """Drafted tokens that are NaN, huge or on other scales, NaN queries behind the counts, junk behind the lengths, bits that mean nothing: rows that do not see
    them are not touched, bit for bit."""
    H, Hk, before = 8, 2, [37, 130]
    counts = _ints([N, N - 1])
    lengths = _ints([n + int(c) for n, c in zip(before, counts)])
    parents = dref.make_parents("any", 2, N, seed=7)
    see = dref.tree(parents, counts)[1]
    g = torch.Generator().manual_seed(N)
    q, k, v = _rand(g, 2, N, H, D), _rand(g, 2, N, Hk, D), _rand(g, 2, N, Hk, D)
    k[:, 1, :, 5], v[:, 1] = 0.0, 0.0                            # (neither zeros nor NaN set a block's scale)
    outs = []
    for bad in (False, True):
        cache, _, table = _filled(before, 64, Hk, D, T=4, seed=1)
        k2, v2, q2 = k.clone(), v.clone(), q.clone()
        if bad:
            k2[:, 1, :, 5], v2[:, 1] = float("nan"), float("nan")
            q2[1, N - 1] = float("nan")
        dm.dm_cache_append(cache, k2.cuda(), v2.cuda(), table.cuda(), _ints(before).cuda(), counts=counts.cuda())
        tree = dm.dm_draft_tree(parents.cuda(), counts.cuda())
        seen = tree.seen.clone()
        if bad:                                                  # later nodes' bits, and no own ones
            words = dref.pack(torch.triu(torch.ones(N, N, dtype=torch.bool), 1).expand(2, N, N)).cuda()
            own = dref.pack(torch.eye(N, dtype=torch.bool).expand(2, N, N)).cuda()
            seen = (seen | words) & ~own
        o, lse = dm.dm_cache_attn_tree(q2.cuda(), cache, table.cuda(), lengths.cuda(), tree._replace(seen=seen), return_lse=True)
        ops.check_status("cuda")
        outs.append((o.cpu(), lse.cpu().transpose(1, 2)))
    sees = see[:, :, 1]
    for x, y in zip(*outs):
        assert torch.equal(x[~sees], y[~sees])
        real = sees & (torch.arange(N) < counts[:, None])
        assert bool(y[real].isnan().all())


def test_attention_scales_and_sizes():
    """V scales far apart, one key that outweighs all, logits in the hundreds, a long tail that carries the weight of its number, q with large and small channels."""
    H, Hk, N, D = 8, 2, 12, 128
    lengths = _ints([3000 + N, 100 + N])
    cache, _, table = _filled(lengths.tolist(), 64, Hk, D, kscale=0.05, vscale=1.0)
    cache.vs.mul_(torch.exp2(torch.randint(-30, 30, cache.vs.shape, device="cuda").float()))
    g = torch.Generator().manual_seed(3)
    parents = dref.make_parents("any", 2, N, seed=1)
    q = _rand(g, 2, N, H, D)
    _attended(q, cache, table, lengths, None, parents)
    cache, _, table = _filled(lengths.tolist(), 64, Hk, D, kscale=0.05)
    page = int(table[0, 0])
    cache.ks[page, :, 0] *= 2.0 ** 9                             # 32 keys far larger than the rest
    _attended(q, cache, table, lengths, None, parents)
    wide = (q.float() * torch.exp2(torch.randint(-9, 6, (D,), generator=g).float())).to(BF)
    cache, _, table = _filled(lengths.tolist(), 64, Hk, D)
    _attended(wide, cache, table, lengths, None, parents)
    _attended(q, cache, table, lengths, None, parents, scale=3.0)
    _attended(q, cache, table, lengths, None, parents, scale=1e-6)
    _attended(torch.zeros_like(q), cache, table, lengths, None, parents)


@pytest.mark.parametrize("N", [4, 40])
def test_attention_large_logits(N):
    """Logits beyond what fp32 adds whole numbers to: still the definition, whose bound grows with them."""
    lengths = _ints([500 + N])
    cache, _, table = _filled(lengths.tolist(), 64, 1, 128)
    g = torch.Generator().manual_seed(3)
    q = _rand(g, 1, N, 2, 128, scale=1e5)
    for scale in (1.0, 1e4):
        o, lse = _attended(q, cache, table, lengths, None, dref.make_parents("any", 1, N, seed=1), scale=scale)
        assert bool(torch.isfinite(o).all())


@pytest.mark.parametrize("D", [128, 256])
@pytest.mark.parametrize("N", [2, 8, 33, 65])
def test_attention_of_products_far_apart(N, D):
    """V scales up to 2^120 apart and logits in the hundreds: what the first blocks, a part of the keys or another copy of the row hold may be nothing to the largest product, and the
    other way round."""
    for seed in range(4):
        lengths = _ints([N, N + 190, N + 1270, N + 700])
        cache, _, table = _filled(lengths.tolist(), 64, 3, D, seed=seed, kscale=0.05)
        g = torch.Generator(device="cuda").manual_seed(seed)
        cache.vs.mul_(torch.exp2(torch.randint(-60, 60, cache.vs.shape, generator=g, device="cuda").float()))
        g = torch.Generator().manual_seed(seed)
        q = (_rand(g, 4, N, 9, D, scale=4.0).float() * torch.exp2(torch.randint(-8, 6, (D,), generator=g).float())).to(BF)
        _attended(q, cache, table, lengths, None, dref.make_parents("any", 4, N, seed=seed), scale=(None, 1.0, 0.01, 0.1)[seed])


@pytest.mark.parametrize("B, Hk", [(5, 3), (4, 4), (11, 3), (17, 2), (37, 2), (25, 3), (37, 4), (149, 1)])
@pytest.mark.parametrize("N, D", [(9, 128), (70, 128), (9, 256)])
def test_attention_of_many_sequences(B, Hk, N, D):
    """Every size of a cluster, and one unit more than the chip holds of them."""
    lengths = [N + (37 * b) % 900 for b in range(B)]
    cache, _, table = _filled(lengths, 64, Hk, D, seed=B)
    g = torch.Generator().manual_seed(B)
    _attended(_rand(g, B, N, 2 * Hk, D), cache, table, _ints(lengths), None, dref.make_parents("near", B, N, seed=1))


@pytest.mark.parametrize("D", [128, 256])
@pytest.mark.parametrize("scale", [1.0, 40.0, -1.0, -40.0])
@pytest.mark.parametrize("N", [3, 25, 40])
def test_attention_far_from_zero(N, scale, D):
    """All logits far below or above zero, in sequences that end inside the first block, the first tile and later ones: parts of a row's keys are none."""
    H, Hk, lengths = 2, 1, _ints([N, N + 20, N + 70, N + 300])
    cache, _, table = _filled(lengths.tolist(), 64, Hk, D)
    keys = cache.k8.view(torch.uint8)
    keys.copy_(keys | 0x80)                                      # the signs of the codes: keys of negative values
    g = torch.Generator().manual_seed(N)
    q = (_rand(g, 4, N, H, D).abs() * (1.0 if scale > 0 else -1.0)).to(BF)
    _attended(q, cache, table, lengths, None, dref.make_parents("any", 4, N, seed=1), scale=abs(scale))


@pytest.mark.parametrize("layout, P", [("joint", 32), ("slots", 128), ("dense", 256)])
def test_attention_layouts_and_strides(layout, P, route):
    """Pools in other layouts, q as a part of a packed tensor, seen as a part of a wider one, and one tree for all sequences."""
    N, H, Hk, D = 21, 6, 3, 128
    lengths = _ints([150, 333])
    cache, _, table = _filled(lengths.tolist(), P, Hk, D, layout=layout)
    g = torch.Generator().manual_seed(9)
    packed = _rand(g, 2, N, H + 4, D).cuda()
    parents = dref.make_parents("any", 1, N, seed=2)
    tree = dm.dm_draft_tree(parents.cuda())
    wide = torch.full((1, N, 5), -1, dtype=torch.int32, device="cuda")
    wide[:, :, 2:3] = tree.seen
    seen = wide[:, :, 2:3].expand(2, -1, -1)
    o = dm.dm_cache_attn_tree(packed[:, :, 2:2 + H], cache, table.cuda(), lengths.cuda(), dm.DraftTree(tree.depth, seen))
    ops.check_status("cuda")
    want, off = dref.attention(packed[:, :, 2:2 + H].cpu(), cache, table, lengths, [N, N], dref.tree(parents, [N])[1].expand(2, -1, -1), D ** -0.5)
    assert bool(((o.double() - want[0]).abs() <= off[0]).all())
    odd = torch.nn.functional.pad(packed, (1, 2))[:, :, 2:2 + H, 1:1 + D]
    assert torch.equal(o, dm.dm_cache_attn_tree(odd, cache, table.cuda(), lengths.cuda(), dm.DraftTree(tree.depth, seen)))


def test_attention_repeats_bit_for_bit():
    for N, H, Hk, D, lengths in ((9, 8, 2, 128, [5000, 17, 900]), (60, 8, 1, 128, [9000, 100, 77]), (40, 4, 2, 256, [3000, 45, 2222])):
        cache, _, table = _filled(lengths, 64, Hk, D)
        q = torch.randn(3, N, H, D, device="cuda", dtype=BF)
        tree = dm.dm_draft_tree(dref.make_parents("any", 3, N).cuda(), _ints([N, min(N, 17), N // 2]).cuda())
        args = (q, cache, table.cuda(), _ints(lengths).cuda(), tree)
        first = dm.dm_cache_attn_tree(*args, return_lse=True)
        for _ in range(5):
            assert all(torch.equal(a, b) for a, b in zip(first, dm.dm_cache_attn_tree(*args, return_lse=True)))
    ops.check_status("cuda")


# ------------------------------------------------------------------------------------------------------------------ keep
def _paths(before, drafts, kind, seed=0):
    g = torch.Generator().manual_seed(seed)
    B, M = len(before), max(max(drafts), 1)
    path, counts = torch.zeros(B, M, dtype=torch.int32), torch.zeros(B, dtype=torch.int32)
    for b, d in enumerate(drafts):
        if kind == "all":
            nodes = torch.arange(d)
        elif kind == "last":
            nodes = torch.arange(max(0, d - 1), d)
        else:
            nodes = (torch.rand(d, generator=g) < (0.3 if kind == "few" else 0.85)).nonzero()[:, 0]
        path[b, :len(nodes)], counts[b] = nodes.to(torch.int32), len(nodes)
    return path, counts


@pytest.mark.parametrize("D", [128, 256])
@pytest.mark.parametrize("kind", ["few", "most", "all", "last"])
@pytest.mark.parametrize("P, layout, most", [(32, "dense", 5), (96, "joint", 40), (64, "slots", 300)])
def test_keep(P, layout, most, kind, D):
    before = [0, 1, 31, 32, 90]
    drafts = [most, most // 2, 1, 0, most]
    lengths = [a + d for a, d in zip(before, drafts)]
    cache, pools, table = _filled(lengths, P, 2, D, seed=most, layout=layout)
    path, counts = _paths(before, drafts, kind)
    new = dm.dm_cache_keep(cache, table.cuda(), _ints(before).cuda(), _ints(lengths).cuda(), path.cuda(), counts.cuda())
    ops.check_status("cuda")
    assert torch.equal(new.cpu(), dref.keep(pools, table, before, path, counts))
    assert ref.same_values(cache, pools)


def test_keep_all_1024(route):
    before, drafts = [40], [1024]
    cache, pools, table = _filled([1064], 64, 1, 128, vscale=4.0)
    path, counts = _paths(before, drafts, "most", seed=5)
    wide = torch.full((1, 1100), -9, dtype=torch.int32)
    wide[:, 50:1074] = path
    new = dm.dm_cache_keep(cache, table.cuda(), _ints(before).cuda(), _ints([1064]).cuda(), wide.cuda()[:, 50:1074], counts.cuda())
    ops.check_status("cuda")
    assert torch.equal(new.cpu(), dref.keep(pools, table, before, path, counts)) and ref.same_values(cache, pools)


def test_keep_scales_far_apart():
    """Zeros of a coarse block beside tiny tokens, NaN codes, a rejected token whose size the scale need not hold any longer."""
    for sizes in ((1e30, 1e-30), (1e-30, 1e30), (1.0, 1e3)):
        cache = ref.make_cache(4, 32, 1, 128)
        table = _ints([[2, 0, 1]])
        g = torch.Generator().manual_seed(1)
        k = torch.zeros(1, 80, 1, 128, dtype=BF)
        k[0, :10] = _rand(g, 10, 1, 128, scale=sizes[0])
        k[0, 20] = 100 * sizes[1]
        k[0, 33:60] = _rand(g, 27, 1, 128, scale=sizes[1])
        k[0, 40, 0, 9], k[0, 41, 0, 9], k[0, 5, 0, 0] = float("nan"), float("inf"), float("nan")
        for before, path in ((9, [5, 25, 30, 31, 40]), (0, [0, 11, 40, 41]), (32, [1, 2, 8, 9]), (12, [8, 21, 22])):
            now = ref.make_cache(4, 32, 1, 128)
            dm.dm_cache_append(now, k.cuda(), k.cuda(), table.cuda(), _ints([0]).cuda())
            pools = ref.Pools(now)
            dm.dm_cache_keep(now, table.cuda(), _ints([before]).cuda(), _ints([80]).cuda(), _ints([path]).cuda(), _ints([len(path)]).cuda())
            dref.keep(pools, table, [before], _ints([path]), [len(path)])
            assert ref.same_values(now, pools)
    ops.check_status("cuda")


def test_bad_paths_are_reported():
    """A path that repeats, falls or leaves the drafted tokens: its sequence stays as it is, the others are served."""
    before, lengths = _ints([40, 33]), _ints([50, 43])
    for bad in ([3, 3], [4, 2], [-1, 2], [2, 10]):
        cache, pools, table = _filled(lengths.tolist(), 32, 2, 128)
        path, counts = _ints([bad, [1, 9]]), _ints([2, 2])
        new = dm.dm_cache_keep(cache, table.cuda(), before.cuda(), lengths.cuda(), path.cuda(), counts.cuda())
        with pytest.raises(RuntimeError, match="path"):
            ops.check_status("cuda")
        assert new.tolist() == [40, 35]
        dref.keep(pools, table, [40, 33], path, [0, 2])
        assert ref.same_values(cache, pools)


def test_bad_device_values_are_reported():
    cache, _, table = _filled([40, 40], 32, 1, 128)
    q, k = torch.randn(2, 3, 2, 128, device="cuda", dtype=BF), torch.randn(2, 3, 1, 128, device="cuda", dtype=BF)
    n, before, f = _ints([40, 40]).cuda(), _ints([37, 37]).cuda(), _freqs(64).cuda()
    tree = dm.dm_draft_tree(dref.make_parents("chain", 2, 3).cuda())
    path, two = _ints([[0, 2, 0], [1, 2, 0]]).cuda(), _ints([2, 2]).cuda()
    for bad_table, bad_n, counts, says in ((_ints([[0, 99], [1, 2]]), n, None, "page"), (_ints([[0, -1], [1, 2]]), n, None, "page"), (table, _ints([40, 1000]).cuda(), None, "length"),
                                           (table, _ints([-3, 40]).cuda(), None, "length"), (table, n, _ints([1, 7]).cuda(), "length"), (table, n, _ints([-1, 1]).cuda(), "length")):
        dm.dm_cache_attn_tree(q, cache, bad_table.cuda(), bad_n, tree._replace(counts=counts))
        with pytest.raises(RuntimeError, match=says):
            ops.check_status("cuda")
        dm.dm_cache_append_rotary(cache, q, k, k, bad_table.cuda(), bad_n, f, counts=counts)
        with pytest.raises(RuntimeError, match=says):
            ops.check_status("cuda")
        if counts is None:
            dm.dm_cache_keep(cache, bad_table.cuda(), before, bad_n, path, two)
            with pytest.raises(RuntimeError):
                ops.check_status("cuda")
    dm.dm_cache_attn_tree(q, cache, table.cuda(), _ints([40, 2]).cuda(), tree)       # more drafted tokens than tokens
    with pytest.raises(RuntimeError, match="length"):
        ops.check_status("cuda")
    dm.dm_cache_keep(cache, table.cuda(), _ints([41, 37]).cuda(), n, path, two)
    with pytest.raises(RuntimeError, match="length|path"):
        ops.check_status("cuda")


# ------------------------------------------------------------------------------------------------------------- arguments
def test_refusals(route):
    cache, _, table = _filled([40], 32, 2, 128)
    t, n, f = table.cuda(), _ints([40]).cuda(), _freqs(64).cuda()
    q, k = torch.zeros(1, 3, 4, 128, device="cuda", dtype=BF), torch.zeros(1, 3, 2, 128, device="cuda", dtype=BF)
    tree = dm.dm_draft_tree(dref.make_parents("chain", 1, 3).cuda())
    path = _ints([[0, 1]]).cuda()
    for args, error, says in (((torch.zeros(1, 3),), ValueError, "CUDA"), ((torch.zeros(1, 3, device="cuda"),), TypeError, "int32"),
                              ((torch.zeros(3, device="cuda", dtype=torch.int32),), ValueError, "shape"), ((torch.zeros(1, 1025, device="cuda", dtype=torch.int32),), ValueError, "1024"),
                              ((torch.zeros(1, 0, device="cuda", dtype=torch.int32),), ValueError, "1024"), ((torch.zeros(0, 4, device="cuda", dtype=torch.int32),), ValueError, "empty"),
                              ((tree.depth, n.repeat(2)), ValueError, "shape"), ((tree.depth, n.long()), TypeError, "int32"), ((tree.depth, n.cpu()), ValueError, "must be on")):
        with pytest.raises(error, match=says):
            dm.dm_draft_tree(*args)
    base = dict(cache=cache, q=q, k=k, v=k, block_table=t, lengths=n, freqs=f)
    for kw, error, says in ((dict(q=q[:, :, :3]), ValueError, "nheads"), (dict(q=q[:, :2]), ValueError, "same tokens"), (dict(v=k[:, :2]), ValueError, "same shape"),
                            (dict(q=q.half()), TypeError, "bfloat16"), (dict(freqs=f.double()), TypeError, "float32"), (dict(freqs=f[:12]), ValueError, "multiple of 8"),
                            (dict(freqs=f.repeat(2)), ValueError, "multiple of 8"), (dict(freqs=f[:0]), ValueError, "multiple of 8"), (dict(freqs=f[None]), ValueError, "multiple of 8"),
                            (dict(freqs=f.cpu()), ValueError, "must be on"), (dict(offsets=tree.depth[:, :2]), ValueError, "shape"), (dict(offsets=tree.depth.long()), TypeError, "int32"),
                            (dict(counts=n.repeat(2)), ValueError, "shape"), (dict(lengths=n[:0]), ValueError, "shape"), (dict(k=k[:, :, :1]), ValueError, "heads"),
                            (dict(cache=dm.KVCache8(cache.k8, cache.v8, *(torch.ones(cache.ks.shape[0], 1, 1, device="cuda").expand(-1, 2, -1),) * 2)), ValueError, "share memory")):
        with pytest.raises(error, match=says):
            dm.dm_cache_append_rotary(**{**base, **kw})
    base = dict(q=q, cache=cache, block_table=t, lengths=n, tree=tree)
    for kw, error, says in ((dict(tree=tuple(tree)), TypeError, "DraftTree"), (dict(tree=tree._replace(seen=None)), TypeError, "DraftTree"), (dict(tree=tree._replace(seen=tree.seen.long())), TypeError, "int32"),
                            (dict(tree=tree._replace(seen=tree.seen[:, :2])), ValueError, "shape"), (dict(tree=tree._replace(counts=n.repeat(2))), ValueError, "shape"),
                            (dict(tree=tree._replace(seen=tree.seen.cpu())), ValueError, "must be on"), (dict(q=q[:, :, :3]), ValueError, "nheads"), (dict(softmax_scale=0.0), ValueError, "softmax_scale"),
                            (dict(softmax_scale=1e39), ValueError, "softmax_scale"), (dict(q=q.float()), TypeError, "bfloat16"), (dict(block_table=t[:, :0]), ValueError, "no pages"),
                            (dict(cache=tuple(cache)), TypeError, "KVCache8")):
        with pytest.raises(error, match=says):
            dm.dm_cache_attn_tree(**{**base, **kw})
    base = dict(cache=cache, block_table=t, before=n, lengths=n, path=path, counts=n)
    for kw, error, says in ((dict(path=path.long()), TypeError, "int32"), (dict(path=path[:, :0]), ValueError, "1024"), (dict(before=n.repeat(2)), ValueError, "shape"), (dict(counts=None), TypeError, "int32"),
                            (dict(path=path.cpu()), ValueError, "must be on"), (dict(block_table=t.long()), TypeError, "int32")):
        with pytest.raises(error, match=says):
            dm.dm_cache_keep(**{**base, **kw})
    ops.check_status("cuda")


def test_tangents_are_refused():
    from torch.autograd import forward_ad
    cache, _, table = _filled([40], 32, 2, 128)
    t, n, f = table.cuda(), _ints([40]).cuda(), _freqs(64).cuda()
    q, k = torch.zeros(1, 3, 4, 128, device="cuda", dtype=BF), torch.zeros(1, 3, 2, 128, device="cuda", dtype=BF)
    tree = dm.dm_draft_tree(dref.make_parents("chain", 1, 3).cuda())
    with forward_ad.dual_level():
        dual = lambda x: forward_ad.make_dual(x, torch.ones_like(x))
        with pytest.raises(NotImplementedError, match="q carries a forward-mode tangent"):
            dm.dm_cache_attn_tree(dual(q), cache, t, n, tree)
        for name in ("q", "k", "v", "freqs"):
            kw = dict(q=q, k=k, v=k, freqs=f)
            with pytest.raises(NotImplementedError, match=f"{name} carries a forward-mode tangent"):
                dm.dm_cache_append_rotary(cache, block_table=t, lengths=n, **{**kw, name: dual(kw[name])})
    ops.check_status("cuda")


# --------------------------------------------------------------------------------------------------------------- together
def _step(k8, v8, ks, vs, q, k, v, parents, counts, path, kept, table, lengths, freqs):
    """A step: tree, append, attention, the path kept, and attention of one more token."""
    cache = dm.KVCache8(k8, v8, ks, vs)
    tree = dm.dm_draft_tree(parents, counts)
    turned, now = dm.dm_cache_append_rotary(cache, q, k, v, table, lengths, freqs, offsets=tree.depth, counts=counts)
    o, lse = dm.dm_cache_attn_tree(turned, cache, table, now, tree, return_lse=True)
    after = dm.dm_cache_keep(cache, table, lengths, now, path, kept)
    o2 = dm.dm_cache_attn(turned[:, :1], cache, table, after)
    return 2.0 * o, lse, after, o2, tree.depth, turned


def _inputs(seed, N=19):
    before = [40, 61]
    cache, _, table = _filled(before, 32, 2, 128, seed=seed, T=4)
    g = torch.Generator().manual_seed(seed)
    parents, counts = dref.make_parents("any", 2, N, seed=seed), _ints([N, N - 6])
    path, kept = _paths(before, counts.tolist(), "few", seed)
    return [*cache, _rand(g, 2, N, 4, 128).cuda(), _rand(g, 2, N, 2, 128).cuda(), _rand(g, 2, N, 2, 128).cuda(), parents.cuda(), counts.cuda(),
            torch.nn.functional.pad(path, (0, N - path.shape[1])).cuda(), kept.cuda(), table.cuda(), _ints(before).cuda(), _freqs(64).cuda()]


def _copy(xs):
    return [x.view(torch.uint8).clone().view(x.dtype) if x.dtype == torch.float8_e4m3fn else x.clone() for x in xs]


def _bits(t):
    return t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t.view(torch.int32) if t.dtype == torch.float32 else t


def test_step_by_the_definition():
    xs = _inputs(5)
    k8, v8, ks, vs, q, k, v, parents, counts, path, kept, table, lengths, freqs = xs
    one = _copy(xs)
    got = _step(*one)
    ops.check_status("cuda")
    cache, at = dm.KVCache8(k8, v8, ks, vs), lengths.cpu()
    depth, see = dref.tree(parents.cpu(), counts.cpu())
    turned, now = _appended(cache, ref.Pools(cache), table.cpu(), q.cpu(), k.cpu(), v.cpu(), at, freqs.cpu(), depth, counts.cpu(), False)
    want, off = dref.attention(turned.cpu(), cache, table.cpu(), now.cpu(), counts.tolist(), see, 128 ** -0.5)
    assert torch.equal(got[5], turned) and torch.equal(got[4].cpu(), depth)
    assert bool(((got[0].double() / 2 - want[0]).abs() <= off[0]).all())
    pools = ref.Pools(cache)
    after = dref.keep(pools, table.cpu(), at, path.cpu(), kept.cpu())
    assert torch.equal(got[2].cpu(), after) and ref.same_values(dm.KVCache8(*one[:4]), pools)
    last, off2 = ref.attention(turned[:, :1].cpu(), pools, table.cpu(), after, [1, 1], True, 128 ** -0.5)
    assert bool(((got[3].cpu().double() - last[0]).abs() <= off2[0]).all())


def test_step_as_one_graph():
    """Captured once, replayed with other trees, counts, paths and lengths: the bits of the eager calls."""
    xs = _inputs(1)
    static = _copy(xs)
    warm = torch.cuda.Stream()
    warm.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(warm):
        _step(*static)
    warm.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _step(*static)
    for seed in (2, 3, 4):
        fresh = _inputs(seed)
        for a, b in zip(static, fresh):
            _bits(a).copy_(_bits(b))
        graph.replay()
        want = _step(*fresh)
        ops.check_status("cuda")
        for i, (x, y) in enumerate(zip((*out, *static[:4]), (*want, *fresh[:4]))):
            assert torch.equal(_bits(x), _bits(y)), (seed, i)


@pytest.mark.parametrize("record", ["jit.trace", "make_fx", "compile"])
def test_recorded_steps_replay(record):
    one, two = _inputs(1), _inputs(2)
    if record == "jit.trace":
        again = torch.jit.trace(_step, tuple(_copy(one)), check_trace=False)
    elif record == "make_fx":
        from torch.fx.experimental.proxy_tensor import make_fx
        again = make_fx(_step)(*_copy(one))
    else:
        again = torch.compile(_step, fullgraph=True, backend="aot_eager")
    a, b = _copy(two), _copy(two)
    got, want = again(*a), _step(*b)
    ops.check_status("cuda")
    for i, (x, y) in enumerate(zip((*got, *a), (*want, *b))):
        assert torch.equal(_bits(x), _bits(y)), i


def test_routes_agree(monkeypatch):
    a, b = _inputs(6), _inputs(6)
    want = _step(*a)
    monkeypatch.setattr(_lib, "native_cache", lambda: _lib._NoCacheRoute)
    for x, y in zip((*_step(*b), *b), (*want, *a)):
        assert torch.equal(_bits(x), _bits(y))


def test_two_streams_at_once():
    """Calls on two streams, each with its own cache: the bits of the calls one after the other."""
    a, b = _inputs(7, 40), _inputs(8, 40)
    want = [_step(*_copy(x)) for x in (a, b)]
    xs = [[_copy(x) for _ in range(8)] for x in (a, b)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = [[], []]
    for i in range(8):
        for s in (0, 1):
            with torch.cuda.stream(streams[s]):
                outs[s].append(_step(*xs[s][i]))
    torch.cuda.synchronize()
    ops.check_status("cuda")
    for s in (0, 1):
        for got in outs[s]:
            assert all(torch.equal(_bits(x), _bits(y)) for x, y in zip(got, want[s]))


def test_first_call_of_a_process_is_captured():
    """What the library asks the device for once does not disturb a capture."""
    code = """
import torch, delta_matching_b200 as dm
from delta_matching_b200 import ops
ints = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")
cache, table, parents, freqs = dm.KVCache8.empty(8, 64, 2, 128), ints(*range(8)).view(2, 4), ints([-1, 0, 0], [-1, 0, 1]), torch.ones(8, device="cuda")
q, k, v = (torch.ones(2, 3, h, 128, device="cuda", dtype=torch.bfloat16) for h in (4, 2, 2))
lengths, path, kept = ints(40, 90), ints([0, 2], [0, 1]), ints(2, 1)
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    tree = dm.dm_draft_tree(parents)
    turned, now = dm.dm_cache_append_rotary(cache, q, k, v, table, lengths, freqs, offsets=tree.depth)
    o = dm.dm_cache_attn_tree(turned, cache, table, now, tree)
    new = dm.dm_cache_keep(cache, table, lengths, now, path, kept)
graph.replay()
ops.check_status("cuda")
assert new.tolist() == [42, 91] and bool(o.isfinite().all())
print("captured")
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=200)
    assert r.returncode == 0 and "captured" in r.stdout, r.stderr[-2000:]


def test_pools_beyond_two_gigabytes():
    """Pages whose codes lie more than 2^31 bytes into the pools: the bits of the same step in small ones."""
    B, N, H, Hk, D, P = 2, 9, 8, 8, 128, 64
    outs = []
    for pages, first in ((8, 0), (40000, 39990)):
        cache = dm.KVCache8(*(torch.empty(pages, Hk, P, D, device="cuda", dtype=torch.uint8).view(torch.float8_e4m3fn) for _ in range(2)),
                            *(torch.empty(pages, Hk, P // 32, device="cuda") for _ in range(2)))
        table = (torch.arange(8, dtype=torch.int32).view(B, 4) + first).cuda()
        g = torch.Generator().manual_seed(1)
        lengths = torch.zeros(B, dtype=torch.int32, device="cuda")
        for n in (100, N):
            q, k, v = (_rand(g, B, n, h, D).cuda() for h in (H, Hk, Hk))
            before = lengths
            turned, lengths = dm.dm_cache_append_rotary(cache, q, k, v, table, before, _freqs(64).cuda())
        tree = dm.dm_draft_tree(dref.make_parents("near", B, N, seed=1).cuda())
        o, lse = dm.dm_cache_attn_tree(turned, cache, table, lengths, tree, return_lse=True)
        new = dm.dm_cache_keep(cache, table, before, lengths, _ints([[0, 3, 8], [2, 4, 5]]).cuda(), _ints([3, 2]).cuda())
        assert new.tolist() == [103, 102]
        held = [c.view(torch.uint8)[first:first + 8, :, :32].flatten(1) if c.dtype != torch.float32 else c[first:first + 8, :, 0] for c in cache]
        outs.append([turned, o, lse] + [x[[0, 4]] for x in held])
        ops.check_status("cuda")
    for x, y in zip(*outs):
        assert torch.equal(x, y)


def test_thousands_of_sequences():
    """As many as a call takes; a node alone is what the causal attention makes of one token: both are within 2^-8 of the sum of weights times values (which is less than twice the
    largest output here) and 2^-8 of rounding, their LSE within 2^-17."""
    B, H, Hk, D = 8191, 8, 1, 128
    lengths = (torch.arange(B) * 7 % 64 + 1).to(torch.int32)
    cache, _, table = _filled([64] * 4, 32, Hk, D)
    table = table[torch.arange(B) % 4].contiguous().cuda()
    g = torch.Generator().manual_seed(1)
    q = _rand(g, B, 1, H, D).cuda()
    tree = dm.dm_draft_tree(torch.full((B, 1), -1, dtype=torch.int32, device="cuda"))
    o, lse = dm.dm_cache_attn_tree(q, cache, table, lengths.cuda(), tree, return_lse=True)
    want, lse2 = dm.dm_cache_attn(q, cache, table, lengths.cuda(), return_lse=True)
    ops.check_status("cuda")
    assert bool(((lse - lse2).abs() < 1e-4).all()) and bool(((o.float() - want.float()).abs() < 0.02 * want.float().abs().amax()).all())
