"""dm_cache_attn_tree where the key tiles of all units are divided evenly over the CTAs and the pieces of cut units are joined by a second kernel: what long tables and full batches take.

A table with room for 97 key tiles and more is divided however short the sequences are; which form a call takes is asserted, so that these tests stay on theirs."""
import math

import pytest
import torch

import delta_matching_b200 as dm
from delta_matching_b200 import _lib, ops

from . import drafts_ref as dref
from .test_cache_gpu import _filled, _ints, _rand
from .test_drafts_gpu import _attended

pytestmark = pytest.mark.gpu
BF = torch.bfloat16
SHAPES = [(4, 8, 2, 128, 32), (9, 12, 2, 128, 64), (40, 8, 2, 128, 128), (5, 6, 3, 256, 32), (33, 2, 2, 256, 64), (70, 4, 2, 256, 128)]      # N, H, Hk, D, rows of a unit


def _wide(table, P, tiles=100):
    """The same pages in a table that has room for so many key tiles of 128 tokens."""
    return torch.nn.functional.pad(table, (0, max(0, tiles * 128 // P - table.shape[1])))


def _plan(B, N, H, Hk, D, table, P):
    """(CTAs of a cluster, CTAs, rows of a unit)"""
    return tuple(_lib.lib().dm_dbg_cache_tree_plan(B, N, H, Hk, D, table.shape[1], P, what) for what in range(3))


def _divided(B, N, H, Hk, D, table, P, rows=None):
    cluster, ctas, row_tile = _plan(B, N, H, Hk, D, table, P)
    assert cluster == 0 and ctas > 1 and rows in (None, row_tile)
    return ctas


def _held(n, N, Hk, D, P=64, seed=0, **kw):
    """A cache of sequences of n[b] tokens, the last N of them drafted, with a wide table."""
    cache, pools, table = _filled(n, P, Hk, D, seed=seed, **kw)
    return cache, _wide(table, P)


def test_plan_refuses():
    plan = _lib.lib().dm_dbg_cache_tree_plan
    assert plan(2, 0, 8, 2, 128, 4, 64, 0) < 0 and plan(2, 5, 8, 3, 128, 4, 64, 0) < 0 and plan(2, 5, 8, 2, 128, 4, 64, 4) < 0
    assert plan(2, 5, 8, 2, 128, 4, 64, 2) == 32 and plan(2, 9, 8, 2, 128, 4, 64, 2) == 64 and plan(2, 30, 8, 2, 128, 4, 64, 2) == 128


@pytest.mark.parametrize("N, H, Hk, D, rows", SHAPES)
def test_pieces(N, H, Hk, D, rows):
    """Few units, each cut into many pieces: ends on and around the edges of blocks and tiles, sequences without drafts, whole and ragged."""
    before = [0, 1, 31, 127, 128, 700, 2500]
    B = len(before)
    for counts in (None, _ints([N, max(1, N // 2), N, 1, N, 0, N - 1])):
        n = [a + (N if counts is None else int(counts[b])) for b, a in enumerate(before)]
        cache, table = _held(n, N, Hk, D, seed=N)
        _divided(B, N, H, Hk, D, table, 64, rows)
        g = torch.Generator().manual_seed(N)
        o, lse = _attended(_rand(g, B, N, H, D, scale=1.5), cache, table, _ints(n), counts, dref.make_parents("any", B, N, seed=N))
        if counts is not None:
            behind = torch.arange(N) >= counts[:, None]
            assert not bool(o.cpu()[behind].any()) and bool((lse.cpu().transpose(1, 2)[behind] == -math.inf).all())


@pytest.mark.parametrize("N, H, Hk, D, rows", [(4, 16, 4, 128, 32), (9, 24, 4, 128, 64), (40, 16, 4, 128, 128), (5, 8, 4, 256, 32), (33, 4, 4, 256, 64), (70, 8, 4, 256, 128)])
def test_whole_units(N, H, Hk, D, rows):
    """More units than three for each SM: most are whole, one behind the other in a CTA."""
    B = 120
    n = [N + (53 * b) % 400 for b in range(B)]
    counts = _ints([N - b % N if b % 7 else 0 for b in range(B)])
    n = [a - N + int(c) for a, c in zip(n, counts)]
    cache, table = _held(n, N, Hk, D, seed=B)
    _divided(B, N, H, Hk, D, table, 64, rows)
    g = torch.Generator().manual_seed(B)
    _attended(_rand(g, B, N, H, D), cache, table, _ints(n), counts, dref.make_parents("near", B, N, seed=1))


@pytest.mark.parametrize("D", [128, 256])
def test_more_pieces_than_lanes(D):
    """A unit over all SMs: the join takes several rounds of 32 pieces; rows that are made by themselves too."""
    N, H, n = 6, 2, [140 * 4 * 128 + 77]
    cache, _, table = _filled(n, 256, 1, D)
    assert _divided(1, N, H, 1, D, table, 256) > 96
    g = torch.Generator().manual_seed(D)
    q = _rand(g, 1, N, H, D, scale=1.5)
    parents = dref.make_parents("any", 1, N, seed=1)
    _attended(q, cache, table, _ints(n), None, parents)
    at = n[0] - N + 2                                            # a drafted token's value: NaN
    cache.v8.view(torch.uint8)[int(table[0, at // 256]), 0, at % 256, 5] = 0x7F
    _attended(q, cache, table, _ints(n), None, parents)


def _forms(N, H, Hk, D, rows):
    """Lengths before the drafts of few sequences, whose units are cut, and of many, whose units are whole."""
    return [130, 37, 900], [130, 37, 260] + [20 + b % 90 for b in range(600 // Hk)]


@pytest.mark.parametrize("many", [False, True])
@pytest.mark.parametrize("N, H, Hk, D, rows", SHAPES)
def test_sees_nothing_else(N, H, Hk, D, rows, many):
    """Drafted tokens that are NaN, NaN queries behind the counts: rows that do not see them are not touched, bit for bit; the others are NaN where they have to be."""
    before = _forms(N, H, Hk, D, rows)[many]
    B = len(before)
    counts = _ints([N] + [N - 1] * (B - 1))
    lengths = [n + int(c) for n, c in zip(before, counts)]
    parents = dref.make_parents("any", B, N, seed=7)
    see = dref.tree(parents, counts)[1]
    g = torch.Generator().manual_seed(N)
    q, k, v = _rand(g, B, N, H, D), _rand(g, B, N, Hk, D), _rand(g, B, N, Hk, D)
    k[:, 1, :, 5], v[:, 1, :, 7] = 0.0, 0.0                      # (neither zeros nor NaN set a block's scale)
    outs = []
    for bad in (0, 1, 2):                                        # nothing, NaN in a key, NaN in one channel of a value
        cache, table = _held(before, N, Hk, D, T=-(-(max(before) + N) // 64), seed=1)
        _divided(B, N, H, Hk, D, table, 64, rows)
        k2, v2, q2 = k.clone(), v.clone(), q.clone()
        if bad:
            (k2 if bad == 1 else v2)[:3, 1, :, 5 if bad == 1 else 7] = float("nan")
            q2[1, N - 1] = float("nan")
        dm.dm_cache_append(cache, k2.cuda(), v2.cuda(), table.cuda(), _ints(before).cuda(), counts=counts.cuda())
        tree = dm.dm_draft_tree(parents.cuda(), counts.cuda())
        o, lse = dm.dm_cache_attn_tree(q2.cuda(), cache, table.cuda(), _ints(lengths).cuda(), tree, return_lse=True)
        ops.check_status("cuda")
        outs.append((o.cpu(), lse.cpu().transpose(1, 2)))
    sees = see[:, :, 1].clone()
    sees[3:] = False
    real = sees & (torch.arange(N) < counts[:, None])
    assert bool(real.any())
    for got in outs[1:]:
        for x, y in zip(outs[0], got):
            assert torch.equal(x[~sees], y[~sees])
    assert bool(outs[1][0][real].isnan().all()) and bool(outs[1][1][real].isnan().all())
    o, lse = outs[2]
    assert bool(o[real][..., 7].isnan().all()) and not bool(o[real][..., :7].isnan().any()) and not bool(o[real][..., 8:].isnan().any()) and bool(lse[real].isfinite().all())
    (w, wl), (d, dl) = dref.attention(q, cache, table, lengths, counts.tolist(), see, D ** -0.5)
    for got, want, off in ((o, w.cpu(), d.cpu()), (lse, wl.cpu().transpose(1, 2), dl.cpu().transpose(1, 2))):
        same = (got == want) | (got.isnan() & want.isnan())
        assert bool((same | ((got.double() - want).abs() <= off)).all())


@pytest.mark.parametrize("many", [False, True])
@pytest.mark.parametrize("N, H, Hk, D, rows", SHAPES)
def test_large_logits(N, H, Hk, D, rows, many):
    """Logits beyond what fp32 adds whole numbers to: every row is made by itself."""
    n = [a + N for a in _forms(N, H, Hk, D, rows)[many]]
    cache, table = _held(n, N, Hk, D)
    _divided(len(n), N, H, Hk, D, table, 64, rows)
    g = torch.Generator().manual_seed(3)
    o, lse = _attended(_rand(g, len(n), N, H, D, scale=1e5), cache, table, _ints(n), None, dref.make_parents("any", len(n), N, seed=1), scale=100.0)
    assert bool(torch.isfinite(o).all())


@pytest.mark.parametrize("seed", [0, 1, 2, 3])
@pytest.mark.parametrize("N, H, Hk, D, rows", SHAPES)
def test_products_far_apart(N, H, Hk, D, rows, seed):
    """V scales up to 2^120 apart and logits in the hundreds: a piece's reference may be anywhere beside another's."""
    n = [N, N + 190, N + 1270, N + 700, N + 2600]
    cache, table = _held(n, N, Hk, D, seed=seed, kscale=0.05)
    _divided(len(n), N, H, Hk, D, table, 64, rows)
    g = torch.Generator(device="cuda").manual_seed(seed)
    cache.vs.mul_(torch.exp2(torch.randint(-60, 60, cache.vs.shape, generator=g, device="cuda").float()))
    g = torch.Generator().manual_seed(seed)
    q = (_rand(g, len(n), N, H, D, scale=4.0).float() * torch.exp2(torch.randint(-8, 6, (D,), generator=g).float())).to(BF)
    _attended(q, cache, table, _ints(n), None, dref.make_parents("any", len(n), N, seed=seed), scale=(None, 1.0, 0.01, 0.1)[seed])


@pytest.mark.parametrize("scale", [1.0, 40.0, -1.0, -40.0])
@pytest.mark.parametrize("N, H, Hk, D, rows", SHAPES)
def test_far_from_zero(N, H, Hk, D, rows, scale):
    """All logits far below or above zero: pieces, and parts of a tile, in which a row sees nothing."""
    n = _ints([N, N + 20, N + 70, N + 300, N + 1500])
    cache, table = _held(n.tolist(), N, Hk, D)
    _divided(len(n), N, H, Hk, D, table, 64, rows)
    keys = cache.k8.view(torch.uint8)
    keys.copy_(keys | 0x80)                                      # the signs of the codes: keys of negative values
    g = torch.Generator().manual_seed(N)
    q = (_rand(g, len(n), N, H, D).abs() * (1.0 if scale > 0 else -1.0)).to(BF)
    _attended(q, cache, table, n, None, dref.make_parents("any", len(n), N, seed=1), scale=abs(scale))


@pytest.mark.parametrize("many", [False, True])
@pytest.mark.parametrize("N, H, Hk, D, rows", SHAPES)
def test_repeats_and_replays(N, H, Hk, D, rows, many):
    """The same bits each time, on two streams, and from a graph that is replayed with other lengths, counts and queries."""
    before = _forms(N, H, Hk, D, rows)[many]
    B = len(before)
    counts = _ints([N - b % N for b in range(B)])
    lengths = _ints([a + int(c) for a, c in zip(before, counts)])
    cache, table = _held(lengths.tolist(), N, Hk, D)
    _divided(B, N, H, Hk, D, table, 64, rows)
    q = torch.randn(B, N, H, D, device="cuda", dtype=BF)
    tree = dm.dm_draft_tree(dref.make_parents("any", B, N).cuda(), counts.cuda())
    args = [q, cache, table.cuda(), lengths.cuda(), tree]
    first = dm.dm_cache_attn_tree(*args, return_lse=True)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = []
    for i in range(6):
        with torch.cuda.stream(streams[i % 2]):
            outs.append(dm.dm_cache_attn_tree(*args, return_lse=True))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for out in outs for a, b in zip(first, out))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = dm.dm_cache_attn_tree(*args, return_lse=True)
    for turn in range(2):
        if turn:                                                 # a prefix of what is held, and other trees
            args[3].copy_((lengths - counts // 2).cuda())
            tree.counts.copy_((counts - counts // 2).cuda())
            q.copy_(torch.randn_like(q))
        graph.replay()
        want = dm.dm_cache_attn_tree(*args, return_lse=True)
        ops.check_status("cuda")
        assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_bad_device_values_are_reported():
    """Entries, lengths and counts out of range: reported, and nothing outside the buffers is read."""
    N, Hk, P = 3, 2, 32
    cache, table = _held([40, 40], N, Hk, 128, P=P)
    _divided(2, N, 4, Hk, 128, table, P)
    q = torch.randn(2, N, 4, 128, device="cuda", dtype=BF)
    n = _ints([40, 40])
    tree = dm.dm_draft_tree(dref.make_parents("chain", 2, N).cuda())
    high, low = table.clone(), table.clone()
    high[0, 1], low[0, 1] = 99, -1
    for bad_table, bad_n, counts, says in ((high, n, None, "page"), (low, n, None, "page"), (table, _ints([40, 1 << 30]), None, "length"), (table, _ints([-3, 40]), None, "length"),
                                           (table, n, _ints([1, 7]), "length"), (table, n, _ints([-1, 1]), "length"), (table, _ints([40, 2]), None, "length")):
        dm.dm_cache_attn_tree(q, cache, bad_table.cuda(), bad_n.cuda(), tree._replace(counts=None if counts is None else counts.cuda()))
        with pytest.raises(RuntimeError, match=says):
            ops.check_status("cuda")


def _long_whole_units():
    """Three hundred sequences of 131072 tokens, all of the same pages but the last one; whole units come first in each CTA's share."""
    B, N, H, Hk, D, P, n = 300, 8, 4, 1, 128, 256, 131072
    last = (n + N) // P
    g = torch.Generator(device="cuda").manual_seed(0)
    pages = last + B
    code = lambda: (torch.randn(pages, Hk, P, D, generator=g, device="cuda") * 40).to(torch.float8_e4m3fn)
    cache = dm.KVCache8(code(), code(), *(torch.full((pages, Hk, P // 32), 2.0 ** -5, device="cuda") for _ in range(2)))
    table = torch.arange(last + 1, dtype=torch.int32).expand(B, -1).clone()
    table[:, last] = last + torch.arange(B)
    assert _divided(B, N, H, Hk, D, table, P, 32) == 148
    lengths = _ints([n + N] * B)
    q = torch.randn(B, N, H, D, generator=g, device="cuda").to(BF)
    parents = dref.make_parents("chain", B, N)
    tree = dm.dm_draft_tree(parents.cuda())
    return q, cache, table, lengths, tree, parents


@pytest.mark.parametrize("kind", ["nan", "large"])
def test_marked_rows_of_long_whole_units(kind):
    """One sequence of many has a NaN in its first draft's value, or logits for which its rows are made by themselves, a key after the other over 131072 tokens: its unit's CTA goes on with the
    next unit meanwhile, and no wait runs out."""
    q, cache, table, lengths, tree, parents = _long_whole_units()
    N, H, D = q.shape[1:]
    args = (q, cache, table.cuda(), lengths.cuda(), tree)
    whole = dm.dm_cache_attn_tree(*args, return_lse=True)
    if kind == "nan":
        at = int(lengths[0]) - N
        cache.v8.view(torch.uint8)[int(table[0, at // 256]), 0, at % 256, 9] = 0x7F
    else:
        q[0] *= 1e6
    got = dm.dm_cache_attn_tree(*args, return_lse=True)
    torch.cuda.synchronize()
    ops.check_status("cuda")
    assert all(torch.equal(a[1:], b[1:]) for a, b in zip(whole, got))
    assert int(got[0].isnan().sum()) == (N * H if kind == "nan" else 0) == int(got[0][0, ..., 9].isnan().sum())
    (w, wl), (d, dl) = dref.attention(q[:1].cpu(), cache, table[:1], lengths[:1], [N], dref.tree(parents[:1], [N])[1], D ** -0.5)
    for x, want, off in ((got[0][:1], w, d), (got[1][:1], wl, dl)):
        same = x.isnan() & want.isnan()
        assert bool((same | ((x.double() - want).abs() <= off)).all())


@pytest.mark.parametrize("before, B", [(1000, 64), (3000, 4), (6000, 8)])
def test_a_nan_value_costs_little(before, B):
    """NaN in one channel of the values of a sequence's first draft, which all its rows see: nothing is summed anew, the call takes at most twenty times as long (a few hundred times if
    those rows were made a key after the other).  Sequences whose units are whole, cut, and a cluster's."""
    N, H, Hk, D, P = 25, 32, 8, 128, 64
    n = [before + N] * B
    T = -(-n[0] // P)
    g = torch.Generator(device="cuda").manual_seed(0)
    code = lambda: (torch.randn(B * T, Hk, P, D, generator=g, device="cuda") * 40).to(torch.float8_e4m3fn)
    cache = dm.KVCache8(code(), code(), *(torch.full((B * T, Hk, P // 32), 2.0 ** -5, device="cuda") for _ in range(2)))
    table = torch.arange(B * T, dtype=torch.int32).view(B, T)
    tree = dm.dm_draft_tree(dref.make_parents("chain", B, N).cuda())
    q = torch.randn(B, N, H, D, generator=g, device="cuda").to(BF)
    args = (q, cache, table.cuda(), _ints(n).cuda(), tree)

    def took():
        best = math.inf
        for _ in range(4):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            out = dm.dm_cache_attn_tree(*args)
            b.record()
            b.synchronize()
            best = min(best, a.elapsed_time(b))
        return best, out

    base, plain = took()
    cache.v8.view(torch.uint8)[int(table[0, before // P]), :, before % P, 3] = 0x7F
    with_nan, out = took()
    ops.check_status("cuda")
    assert bool(out[0, ..., 3].isnan().all()) and int(out.isnan().sum()) == N * H
    keep = torch.ones(D, dtype=torch.bool, device="cuda")
    keep[3] = False
    assert torch.equal(out[..., keep], plain[..., keep]) and torch.equal(out[1:], plain[1:])
    assert with_nan < 20 * base, (with_nan, base)


@pytest.mark.parametrize("divided", [False, True])
@pytest.mark.parametrize("N, H, Hk, D, rows", SHAPES)
def test_nan_values_and_large_logits(N, H, Hk, D, rows, divided):
    """Both at once, in different channels of two drafted tokens: what a row sees of them, and nothing else, is NaN; some rows have large logits, others not."""
    n = [N + 130, N + 37, N + 700]
    cache, _, table = _filled(n, 64, Hk, D, seed=2)
    if divided:
        table = _wide(table, 64)
    assert (_plan(3, N, H, Hk, D, table, 64)[0] == 0) == divided
    v = cache.v8.view(torch.uint8)
    for b in range(3):
        for node, channel in ((0, 3), (min(2, N - 1), D - 2)):
            at = n[b] - N + node
            v[int(table[b, at // 64]), :, at % 64, channel] = 0xFF
    g = torch.Generator().manual_seed(3)
    q = _rand(g, 3, N, H, D)
    q[:, ::3] *= 1e6
    _attended(q, cache, table, _ints(n), None, dref.make_parents("any", 3, N, seed=1), scale=10.0)
