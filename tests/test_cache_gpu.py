"""The cache operators against their definitions in 64 bits (tests/cache_ref.py)."""
import math

import pytest
import torch

import delta_matching_b200 as dm
from delta_matching_b200 import ops

from . import cache_ref as ref

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def _rand(g, *shape, scale=1.0):
    return (torch.randn(*shape, generator=g) * scale).to(BF)


def _filled(lengths, P, Hk, D, seed=0, layout="dense", kscale=1.0, vscale=1.0, T=None):
    """A cache that holds lengths[b] random tokens of each sequence (all else: NaN codes and scales), its CPU copy and its table."""
    B = len(lengths)
    T = T or max(1, -(-max(lengths) // P))
    pages = B * T + 2
    cache = ref.make_cache(pages, P, Hk, D, layout=layout)
    table = ref.make_table(B, T, pages, seed)
    g = torch.Generator().manual_seed(seed)
    N = max(1, max(lengths))
    # the size of K and V varies from token to token, so that neighbouring blocks have different scales
    size = torch.exp(torch.randn(B, N, 1, 1, generator=g))
    k, v = (_rand(g, B, N, Hk, D) * size * kscale).to(BF), (_rand(g, B, N, Hk, D) * size.flip(1) * vscale).to(BF)
    got = dm.dm_cache_append(cache, k.cuda(), v.cuda(), table.cuda(), torch.zeros(B, dtype=torch.int32, device="cuda"),
                             counts=torch.tensor(lengths, dtype=torch.int32, device="cuda"))
    assert got.tolist() == list(lengths)
    ops.check_status("cuda")
    return cache, ref.Pools(cache), table


def _ints(x):
    return torch.tensor(x, dtype=torch.int32)


# ---------------------------------------------------------------------------------------------------------------- append
@pytest.mark.parametrize("D", [128, 256])
@pytest.mark.parametrize("P, layout", [(32, "dense"), (96, "joint"), (64, "slots")])
@pytest.mark.parametrize("N", [1, 31, 33, 70])
def test_append_in_steps(N, P, layout, D):
    """Three calls, one behind the other, with starts on, before and behind a block's edge; sizes that make scales grow and not."""
    B, Hk, T = 4, 3, -(-(40 + 3 * N) // P)
    cache = ref.make_cache(B * T + 1, P, Hk, D, layout=layout)
    table = ref.make_table(B, T, B * T + 1, seed=N)
    pools = ref.Pools(cache)
    g = torch.Generator().manual_seed(N)
    lengths = _ints([0, 0, 0, 0])
    first = _ints([0, 1, 31, 40])                                # the starts of the second call
    for step in range(4):
        n = 40 if step == 0 else N
        counts = first if step == 0 else _ints([N, max(0, N - 1), N // 2, N])
        k, v = (_rand(g, B, n, Hk, D, scale=s) for s in (4.0 ** (step - 2), 3.0 ** (1 - step)))
        whole = torch.equal(counts, _ints([n] * B))
        new = dm.dm_cache_append(cache, k.cuda(), v.cuda(), table.cuda(), lengths.cuda(), counts=None if whole else counts.cuda())
        ref.append(pools, (k, v), table, lengths, counts)
        lengths = lengths + counts
        assert torch.equal(new.cpu(), lengths)
        assert ref.same_values(cache, pools), step
    ops.check_status("cuda")


def test_append_again_leaves_the_same_cache():
    cache, pools, table = _filled([13, 64, 95], 32, 2, 128, T=6)
    k, v = (torch.randn(3, 50, 2, 128, device="cuda", dtype=BF) * 30 for _ in range(2))
    args = (cache, k, v, table.cuda(), _ints([13, 64, 95]).cuda())
    dm.dm_cache_append(*args)
    once = ref.Pools(cache)
    dm.dm_cache_append(*args)
    assert ref.same_values(cache, once) and not ref.same_values(cache, pools)


def test_append_zeros_then_small_values():
    """A block that begins with zeros takes the scale of what follows."""
    cache = ref.make_cache(2, 32, 1, 128)
    pools, table = ref.Pools(cache), _ints([[1]])
    for n, size in ((3, 0.0), (2, 1e-6), (1, 1e-30)):
        x = (torch.randn(1, n, 1, 128) * size).to(BF)
        at = _ints([0 if size == 0.0 else 3 if size == 1e-6 else 5])
        dm.dm_cache_append(cache, x.cuda(), x.cuda(), table.cuda(), at.cuda())
        ref.append(pools, (x, x), table, at, _ints([n]))
    assert ref.same_values(cache, pools)
    assert float(pools.scales[0][1, 0, 0]) < 1e-7


def test_append_special_values():
    """NaN stays NaN and does not set the scale, infinities saturate, tiny and huge values keep their scales, powers of two at the edge of one."""
    for fill, want_scale in ((1.0, 2.0 ** -8), (448.0, 1.0), (450.0, 2.0), (2.0 ** -126, 2.0 ** -126), (3.0e38, 2.0 ** 120), (448 * 2.0 ** 110, 2.0 ** 110)):
        cache = ref.make_cache(1, 32, 1, 128, fill=0)
        x = torch.full((1, 2, 1, 128), fill, dtype=BF)
        x[0, 0, 0, 5] = float("nan")
        dm.dm_cache_append(cache, x.cuda(), x.cuda(), _ints([[0]]).cuda(), _ints([0]).cuda())
        scale = float(cache.ks[0, 0, 0])
        got = cache.k8[0, 0, :2].cpu().float() * scale
        assert scale == ref.scale_of(float(x.nan_to_num(0.0).double().max())) and (want_scale == scale)
        assert got[0, 5].isnan() and int(got.isnan().sum()) == 1
        assert torch.allclose(got[1], x[0, 1, 0].float(), rtol=2.0 ** -4)
    cache = ref.make_cache(1, 32, 1, 128, fill=0)
    x = torch.ones(1, 1, 1, 128, dtype=BF)
    x[..., 0], x[..., 1] = float("inf"), float("-inf")
    dm.dm_cache_append(cache, x.cuda(), x.cuda(), _ints([[0]]).cuda(), _ints([0]).cuda())
    assert cache.k8[0, 0, 0, :3].cpu().float().tolist() == [448.0, -448.0, 0.0]


@pytest.mark.parametrize("how", ["packed", "odd offset", "head-major"])
def test_append_strided_inputs(how):
    g = torch.Generator().manual_seed(3)
    B, N, Hk, D = 2, 37, 2, 128
    k, v = _rand(g, B, N, Hk, D), _rand(g, B, N, Hk, D)
    if how == "packed":
        both = torch.cat([k, v], 2).cuda()
        kd, vd = both[:, :, :Hk], both[:, :, Hk:]
    elif how == "odd offset":
        kd, vd = (torch.nn.functional.pad(t, (3, 2)).cuda()[..., 3:3 + D] for t in (k, v))
    else:
        kd, vd = (t.transpose(1, 2).contiguous().cuda().transpose(1, 2) for t in (k, v))
    cache = ref.make_cache(5, 32, Hk, D)
    pools, table, at = ref.Pools(cache), _ints([[4, 0, 1], [2, 3, 4]])[:, :2], _ints([5, 20])
    cache.ks.fill_(2.0 ** -10), cache.vs.fill_(2.0 ** -10)
    [t.fill_(2.0 ** -10) for t in pools.scales]
    wide = torch.full((B, 7), 99, dtype=torch.int32)             # the table a part of a wider one
    wide[:, 2:4] = table
    dm.dm_cache_append(cache, kd, vd, wide.cuda()[:, 2:4], at.cuda())
    ref.append(pools, (k, v), table, at, _ints([N, N]))
    assert ref.same_values(cache, pools)
    ops.check_status("cuda")


# ------------------------------------------------------------------------------------------------------------- attention
def _check(q, cache, pools, table, lengths, counts=None, causal=True, scale=None, weights=False, wide=0):
    B, N, H, D = q.shape
    Hk, P = cache.k8.shape[1:3]
    W = table.shape[1] * P + wide
    w = torch.full((B, Hk, W), float("nan"), device="cuda") if weights else None
    o, lse = dm.dm_cache_attn(q.cuda(), cache, table.cuda(), _ints(lengths).cuda(), q_counts=None if counts is None else _ints(counts).cuda(),
                              causal=causal, softmax_scale=scale, weights=w, return_lse=True)
    ops.check_status("cuda")
    want, off = ref.attention(q, pools, table, lengths, counts or [N] * B, causal, scale or D ** -0.5)
    got = [o.cpu().double(), lse.cpu().double()] + ([w.cpu().double()] if weights else [])
    assert o.dtype == BF and o.is_contiguous() and lse.dtype == torch.float32
    assert torch.equal(got[1] == -math.inf, want[1] == -math.inf)
    got[1], want_lse = torch.where(want[1] == -math.inf, 0.0, got[1]), torch.where(want[1] == -math.inf, 0.0, want[1])
    for name, x, y, d in zip(("o", "lse", "weights"), got, (want[0], want_lse, torch.nn.functional.pad(want[2], (0, wide))),
                             (off[0], off[1], torch.nn.functional.pad(off[2], (0, wide)))):
        bad = ~((x - y).abs() <= d)
        assert not bool(bad.any()), (name, int(bad.sum()), float((x - y)[bad].abs().max()), bad.nonzero()[0].tolist())
    return o, lse, w


@pytest.mark.parametrize("D", [128, 256])
@pytest.mark.parametrize("rep", [1, 3, 8, 16, 17])
def test_attention_one_token(rep, D):
    """Lengths around the blocks and warps of a CTA, one new token each; rows in one and several tiles."""
    lengths = [1, 2, 31, 32, 33, 127, 129, 300]
    cache, pools, table = _filled(lengths, 64, 2, D, seed=rep)
    q = _rand(torch.Generator().manual_seed(rep), len(lengths), 1, 2 * rep, D)
    _check(q, cache, pools, table, lengths, weights=rep in (1, 8, 17))


@pytest.mark.parametrize("D", [128, 256])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("N, rep", [(2, 1), (5, 3), (7, 1), (33, 2), (130, 3)])
def test_attention_several_tokens(N, rep, causal, D):
    """New tokens fewer and more than what is held, ragged counts down to none, rows that see nothing."""
    lengths = [0, 1, N - 1, N, N + 31, 200]
    counts = [N, N, N, N // 2, 0, N]
    cache, pools, table = _filled(lengths, 96, 2, D, seed=N)
    q = _rand(torch.Generator().manual_seed(N), len(lengths), N, 2 * rep, D)
    _check(q, cache, pools, table, lengths, counts, causal, weights=N in (5, 33))


@pytest.mark.parametrize("layout, P", [("joint", 32), ("slots", 128)])
def test_attention_layouts_and_long_lengths(layout, P):
    """More blocks than CTAs take in one piece: units are cut and joined; strided q and weights."""
    lengths = [2500, 0, 700]
    cache, pools, table = _filled(lengths, P, 2, 128, seed=P, layout=layout)
    g = torch.Generator().manual_seed(P)
    q = _rand(g, 3, 1, 10, 128)
    o, lse, w = _check(q, cache, pools, table, lengths, weights=True, wide=5)
    packed = torch.cat([q, _rand(g, 3, 1, 4, 128)], 2).cuda()
    again = dm.dm_cache_attn(packed[:, :, :10], cache, table.cuda(), _ints(lengths).cuda())
    assert torch.equal(o, again)
    # weights of a strided tensor, added to what is there
    room = torch.rand(3, 2, 2, w.shape[2], device="cuda")
    before, view = room.clone(), room[:, :, 1]
    dm.dm_cache_attn(q.cuda(), cache, table.cuda(), _ints(lengths).cuda(), weights=view, accumulate=True)
    held = (torch.arange(w.shape[2])[None, None] < _ints(lengths)[:, None, None]).cuda()
    assert torch.equal(view, torch.where(held, before[:, :, 1] + w, before[:, :, 1])) and torch.equal(room[:, :, 0], before[:, :, 0])


@pytest.mark.parametrize("kscale, vscale, qscale, scale", [(1e-20, 1.0, 1e20, None), (1.0, 1e-30, 1.0, None), (1.0, 1e30, 1.0, None), (30.0, 1.0, 30.0, None),
                                                           (1.0, 1.0, 1.0, 3.0), (1.0, 1.0, 1e-30, None)])
def test_attention_ranges(kscale, vscale, qscale, scale):
    lengths = [150, 33]
    cache, pools, table = _filled(lengths, 32, 1, 128, kscale=kscale, vscale=vscale)
    q = _rand(torch.Generator().manual_seed(1), 2, 2, 3, 128, scale=qscale)
    q[0, 0, 1] = 0                                               # a query of zeros sees all keys alike
    _check(q, cache, pools, table, lengths, scale=scale, weights=True)


def test_attention_blocks_of_very_different_size():
    """V blocks 2^-100 ... 2^100 of one another and blocks of zeros, in an order that makes the running scale jump; and a key that takes all."""
    B, Hk, D, P, n = 2, 1, 128, 32, 32 * 12 + 5
    cache = ref.make_cache(B * 13, P, Hk, D)
    table = ref.make_table(B, 13, B * 13)
    g = torch.Generator().manual_seed(8)
    k, v = _rand(g, B, n, Hk, D), _rand(g, B, n, Hk, D)
    for j, e in enumerate((0, -100, 3, 100, -3, -40, 40, 0, 20, -20, 99, 1, -99)):
        v[0, 32 * j:32 * j + 32] *= 2.0 ** e
    v[1, 64:128] = 0
    k[1, 96:160] = 0
    k[1, 200] *= 40
    dm.dm_cache_append(cache, k.cuda(), v.cuda(), table.cuda(), _ints([0, 0]).cuda())
    q = _rand(g, B, 1, 4, D)
    _check(q, cache, ref.Pools(cache), table, [n, n])
    _check(q, cache, ref.Pools(cache), table, [32 * 3, 32 * 6 + 1])


def test_attention_nan_and_inf_inputs():
    """A NaN among the held values or in a query reaches the rows that see it and no others."""
    lengths = [100, 100]
    cache, pools, table = _filled(lengths, 32, 1, 128)
    q = _rand(torch.Generator().manual_seed(2), 2, 1, 2, 128).cuda()
    clean = dm.dm_cache_attn(q, cache, table.cuda(), _ints(lengths).cuda())
    bad = q.clone()
    bad[0, 0, 1, 7] = float("nan")
    o = dm.dm_cache_attn(bad, cache, table.cuda(), _ints(lengths).cuda())
    assert bool(o[0, 0, 1].isnan().all()) and torch.equal(o[0, 0, 0], clean[0, 0, 0]) and torch.equal(o[1], clean[1])
    cache.k8.view(torch.uint8)[int(table[1, 70 // 32]), 0, 70 % 32, 3] = 0x7F
    o = dm.dm_cache_attn(q, cache, table.cuda(), _ints(lengths).cuda())
    assert bool(o[1].isnan().all()) and torch.equal(o[0], clean[0])
    o = dm.dm_cache_attn(q, cache, table.cuda(), _ints([100, 70]).cuda())
    assert bool(o[1].isfinite().all())


def test_attention_repeats_bit_for_bit_and_on_another_stream():
    lengths = [900, 17, 333, 64]
    cache, pools, table = _filled(lengths, 64, 4, 128)
    q = _rand(torch.Generator().manual_seed(4), 4, 3, 20, 128).cuda()
    t, n = table.cuda(), _ints(lengths).cuda()
    w = torch.zeros(4, 4, t.shape[1] * 64, device="cuda")
    first = dm.dm_cache_attn(q, cache, t, n, weights=w, return_lse=True)
    w0 = w.clone()
    for _ in range(5):
        again = dm.dm_cache_attn(q, cache, t, n, weights=w, return_lse=True)
        assert torch.equal(again[0], first[0]) and torch.equal(again[1], first[1]) and torch.equal(w, w0)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        on_side = dm.dm_cache_attn(q, cache, t, n)
    side.synchronize()
    assert torch.equal(on_side, first[0])


def test_offsets_beyond_32_bits():
    """Pages more than 4 GiB apart."""
    gap, P, Hk, D = (5 << 30) + 4096, 32, 2, 128
    try:
        room = torch.zeros(2, gap + P * Hk * D, dtype=torch.uint8, device="cuda")
    except torch.OutOfMemoryError:
        pytest.skip("not enough free device memory")
    cache = dm.KVCache8(*(torch.as_strided(r, (2, Hk, P, D), (gap, P * D, D, 1)).view(torch.float8_e4m3fn) for r in room),
                        *(torch.zeros(2, Hk, 1, device="cuda") for _ in range(2)))
    g = torch.Generator().manual_seed(5)
    k, v, q = _rand(g, 1, 64, Hk, D), _rand(g, 1, 64, Hk, D), _rand(g, 1, 1, 4, D)
    near = ref.make_cache(2, P, Hk, D)
    out = []
    for c in (cache, near):
        n = dm.dm_cache_append(c, k.cuda(), v.cuda(), _ints([[1, 0]]).cuda(), _ints([0]).cuda())
        out.append(dm.dm_cache_attn(q.cuda(), c, _ints([[1, 0]]).cuda(), n))
    assert torch.equal(*out)
    assert torch.equal(cache.k8[1].view(torch.uint8), near.k8[1].view(torch.uint8))


# -------------------------------------------------------------------------------------------------------------- eviction
@pytest.mark.parametrize("D, P, P_layout", [(128, 32, "dense"), (256, 64, "joint"), (128, 96, "slots")])
@pytest.mark.parametrize("budget, recent", [(1, 0), (1, 1), (40, 7), (64, 64), (96, 0), (192, 33)])
def test_evict(budget, recent, D, P, P_layout):
    lengths = [0, 1, 40, 150, 191]
    T, T2, Hk = -(-191 // P), -(-budget // P), 2
    B = len(lengths)
    pages = B * (T + T2)
    cache = ref.make_cache(pages, P, Hk, D, layout=P_layout)
    tables = ref.make_table(1, pages, pages, seed=budget)[0]
    table, new_table = tables[:B * T].view(B, T), tables[B * T:].view(B, T2)
    g = torch.Generator().manual_seed(budget)
    size = torch.exp(2 * torch.randn(B, 191, 1, 1, generator=g))
    k, v = (_rand(g, B, 191, Hk, D) * size).to(BF), (_rand(g, B, 191, Hk, D) * size).to(BF)
    k[:, 64:100] = 0
    dm.dm_cache_append(cache, k.cuda(), v.cuda(), table.cuda(), torch.zeros(B, dtype=torch.int32, device="cuda"), counts=_ints(lengths).cuda())
    pools = ref.Pools(cache)
    weights = torch.rand(B, Hk, T * P + 3, generator=g)
    weights[:, :, ::3] = weights[:, :, ::3].round(decimals=1)    # ties, zeros of both signs, negative and not finite ones
    weights[:, 0, 5:90:7], weights[:, 1, 2:60:5], weights[:, :, 33], weights[:, :, 34], weights[:, :, 35] = 0.0, -0.0, float("nan"), float("inf"), -1.0
    got = dm.dm_cache_evict(cache, table.cuda(), _ints(lengths).cuda(), weights.cuda(), new_table.cuda(), budget, recent=recent)
    ops.check_status("cuda")
    want = ref.evict(pools, table, new_table, lengths, weights, budget, recent)
    assert torch.equal(got[0].cpu(), want[0]) and torch.equal(got[1].cpu(), want[1])
    assert torch.equal(got[2].cpu().nan_to_num(-7.0), want[2].nan_to_num(-7.0))
    assert ref.same_values(cache, pools)


@pytest.mark.parametrize("n, budget, recent, kind", [(50000, 20000, 64, "random"), (50000, 20000, 0, "few values"), (33333, 33332, 5, "equal"), (40001, 17, 1, "random"),
                                                    (70000, 69999, 0, "few values")])
def test_evict_long_rows(n, budget, recent, kind):
    """Rows that a cluster of CTAs shares: what is kept against a stable sort."""
    Hk, P, D = 3, 64, 128
    T, T2 = -(-n // P), -(-budget // P)
    pages = T + T2
    cache = dm.KVCache8(*(torch.randint(0, 127, (pages, Hk, P, D), device="cuda", dtype=torch.uint8).view(torch.float8_e4m3fn) for _ in range(2)),
                        *(torch.ones(pages, Hk, P // 32, device="cuda") for _ in range(2)))
    table = torch.arange(T, device="cuda", dtype=torch.int32)[None]
    new_table = torch.arange(T, pages, device="cuda", dtype=torch.int32)[None]
    g = torch.Generator().manual_seed(n)
    w = torch.rand(1, Hk, T * P, generator=g)
    w = w if kind == "random" else (w * 4).floor() if kind == "few values" else torch.ones_like(w)
    new, kept, nw = dm.dm_cache_evict(cache, table, _ints([n]).cuda(), w.cuda(), new_table, budget, recent=recent)
    order = torch.sort(w[0, :, :n - recent], dim=-1, descending=True, stable=True).indices[:, :budget - recent].sort(-1).values
    want = torch.cat([order, torch.arange(n - recent, n).expand(Hk, -1)], 1)
    assert torch.equal(kept[0].cpu().long(), want) and new.tolist() == [budget]
    assert torch.equal(nw[0, :, :budget].cpu(), w[0].gather(1, want)) and not bool(nw[0, :, budget:].any())
    h = torch.arange(Hk)[:, None]
    moved = cache.k8.view(torch.uint8).cpu()
    to = torch.arange(budget)
    got = moved.view(torch.float8_e4m3fn)[new_table.cpu()[0, to // P].long(), :, to % P].float().transpose(0, 1) * cache.ks.cpu()[
        new_table.cpu()[0, to // P].long(), :, to % P // 32].T[..., None]
    assert torch.equal(got, moved.view(torch.float8_e4m3fn)[want // P, h, want % P].float())


@pytest.mark.parametrize("n, budget, recent, kind", [(150001, 50000, 64, "random"), (150001, 149000, 3, "few values"), (340003, 1001, 1, "random"),
                                                    (340003, 340001, 0, "few values")])
def test_evict_longest_rows(n, budget, recent, kind):
    """Slices of a row that a CTA takes in several turns, and that its shared memory does not hold."""
    test_evict_long_rows(n, budget, recent, kind)


def test_evict_scales_far_apart():
    """Zero rows on a coarse scale beside tiny rows; NaN codes move and do not set the scale."""
    cache = ref.make_cache(4, 32, 1, 128)
    table, new_table = _ints([[2, 0]]), _ints([[3]])
    g = torch.Generator().manual_seed(1)
    k = torch.zeros(1, 64, 1, 128, dtype=BF)
    k[0, 0] = 1e30
    k[0, 33:40] = _rand(g, 7, 1, 128, scale=1e-30)
    k[0, 35, 0, 9] = float("nan")
    dm.dm_cache_append(cache, k.cuda(), k.cuda(), table.cuda(), _ints([0]).cuda())
    pools = ref.Pools(cache)
    w = torch.zeros(1, 1, 64)
    w[0, 0, 5:21] = 1.0                                          # zeros of the first block, and the last sixteen of the second
    w[0, 0, 32:48] = 2.0
    dm.dm_cache_evict(cache, table.cuda(), _ints([64]).cuda(), w.cuda(), new_table.cuda(), 32)
    ref.evict(pools, table, new_table, [64], w, 32, 0)
    assert ref.same_values(cache, pools)


# ------------------------------------------------------------------------------------------- together; what the host cannot see
def test_decode_as_one_graph():
    """Append and attention captured once, replayed while the lengths grow on the device."""
    B, Hk, H, D, P, T = 2, 2, 6, 128, 32, 5
    cache = ref.make_cache(B * T, P, Hk, D)
    table = ref.make_table(B, T, B * T)
    g = torch.Generator().manual_seed(6)
    ks, vs, qs = (_rand(g, 70, B, 1, h, D).cuda() for h in (Hk, Hk, H))
    k, v, q = ks[0].clone(), vs[0].clone(), qs[0].clone()
    lengths, t, w = torch.zeros(B, dtype=torch.int32, device="cuda"), table.cuda(), torch.zeros(B, Hk, T * P, device="cuda")

    def step():
        lengths.copy_(dm.dm_cache_append(cache, k, v, t, lengths))
        return dm.dm_cache_attn(q, cache, t, lengths, weights=w, accumulate=True)

    warm = torch.cuda.Stream()
    with torch.cuda.stream(warm):
        step()
    warm.synchronize()
    lengths.zero_(), w.zero_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = step()
    for i in range(70):
        k.copy_(ks[i]), v.copy_(vs[i]), q.copy_(qs[i])
        graph.replay()
        if i in (0, 31, 32, 69):
            want, off = ref.attention(qs[i].cpu(), ref.Pools(cache), table, [i + 1] * B, [1] * B, True, D ** -0.5)
            assert bool(((o.cpu().double() - want[0]).abs() <= off[0]).all())
    assert lengths.tolist() == [70, 70]
    # every token has given away a weight of one per head of the group
    assert abs(float(w.double().sum()) - 70 * B * H) < 1e-3
    ops.check_status("cuda")


def test_bad_device_values_are_reported():
    """Page numbers and lengths out of range touch nothing outside the pools; the next call, or check_status, raises."""
    cache, pools, table = _filled([40, 40], 32, 1, 128)
    q = torch.randn(2, 1, 2, 128, device="cuda", dtype=BF)
    k = torch.randn(2, 3, 1, 128, device="cuda", dtype=BF)
    n = _ints([40, 40]).cuda()
    for bad_table, bad_n, counts, says in ((_ints([[0, 99], [1, 2]]), n, None, "page"), (_ints([[0, -1], [1, 2]]), n, None, "page"),
                                           (table, _ints([40, 1000]).cuda(), None, "length"), (table, _ints([-3, 40]).cuda(), None, "length"),
                                           (table, n, _ints([1, 7]).cuda(), "length"), (table, n, _ints([-1, 1]).cuda(), "length")):
        dm.dm_cache_attn(q, cache, bad_table.cuda(), bad_n, q_counts=counts)
        with pytest.raises(RuntimeError, match=says):
            ops.check_status("cuda")
        dm.dm_cache_append(cache, k, k, bad_table.cuda(), bad_n, counts=counts)
        with pytest.raises(RuntimeError, match=says):
            ops.check_status("cuda")
    dm.dm_cache_append(cache, k, k, table.cuda(), _ints([40, 62]).cuda())      # the last token does not fit
    with pytest.raises(RuntimeError, match="length"):
        ops.check_status("cuda")
    w = torch.zeros(2, 1, 64, device="cuda")
    for bad, says in ((_ints([[99], [1]]), "page"), (_ints([[-5], [1]]), "page")):
        dm.dm_cache_evict(cache, table.cuda(), n, w, bad.cuda(), 8)
        torch.cuda.synchronize()
        with pytest.raises(RuntimeError, match=says):
            dm.dm_cache_attn(q, cache, table.cuda(), n)
    dm.dm_cache_attn(q, cache, table.cuda(), n)
    ops.check_status("cuda")


def test_refusals_on_the_device():
    cache, pools, table = _filled([40], 32, 2, 128)
    t, n = table.cuda(), _ints([40]).cuda()
    q, k = torch.zeros(1, 1, 4, 128, device="cuda", dtype=BF), torch.zeros(1, 1, 2, 128, device="cuda", dtype=BF)
    w = torch.zeros(1, 2, 64, device="cuda")
    with pytest.raises(TypeError, match="bfloat16"):
        dm.dm_cache_attn(q.half(), cache, t, n)
    with pytest.raises(TypeError, match="int32"):
        dm.dm_cache_attn(q, cache, t.long(), n)
    with pytest.raises(TypeError, match="int32"):
        dm.dm_cache_append(cache, k, k, t, n.long())
    with pytest.raises(TypeError, match="float32"):
        dm.dm_cache_attn(q, cache, t, n, weights=w.half())
    with pytest.raises(TypeError, match="e4m3"):
        dm.dm_cache_attn(q, dm.KVCache8(cache.k8.view(torch.uint8), *cache[1:]), t, n)
    for kw, says in ((dict(q=q[:, :, :3]), "nheads"), (dict(q=q[0]), "4-D"), (dict(q=q[:, :0]), "empty"), (dict(t=t[:, :0]), "no pages"), (dict(n=n[:0]), "shape"),
                     (dict(n=n.cpu()), "must be on"), (dict(t=t.repeat(2, 1)), "shape"), (dict(softmax_scale=-1.0), "softmax_scale"), (dict(accumulate=True), "accumulate"),
                     (dict(weights=w[:, :, :63]), "weights"), (dict(weights=w.expand(1, 2, 64).transpose(1, 2).contiguous().transpose(1, 2)), "adjacent"),
                     (dict(q_counts=n.repeat(2)), "shape"), (dict(q=torch.zeros(1, 1, 4, 256, device="cuda", dtype=BF)), "head_dim")):
        kw = dict(dict(q=q, cache=cache, t=t, n=n), **kw)
        with pytest.raises(ValueError, match=says):
            dm.dm_cache_attn(kw.pop("q"), kw.pop("cache"), kw.pop("t"), kw.pop("n"), **kw)
    with pytest.raises(ValueError, match="same shape"):
        dm.dm_cache_append(cache, k, k.repeat(1, 2, 1, 1), t, n)
    with pytest.raises(ValueError, match="heads"):
        dm.dm_cache_append(cache, k.repeat(1, 1, 2, 1), k.repeat(1, 1, 2, 1), t, n)
    with pytest.raises(ValueError, match="strides"):
        dm.dm_cache_attn(q, dm.KVCache8(cache.k8, cache.v8.transpose(0, 1).contiguous().transpose(0, 1), *cache[2:]), t, n)
    with pytest.raises(ValueError, match="adjacent"):
        dm.dm_cache_attn(q, dm.KVCache8(*(x.transpose(2, 3).contiguous().transpose(2, 3) for x in cache[:2]), *cache[2:]), t, n)
    with pytest.raises(ValueError, match="budget"):
        dm.dm_cache_evict(cache, t, n, w, t[:, :1], 33)
    with pytest.raises(ValueError, match="budget"):
        dm.dm_cache_evict(cache, t, n, w, t[:, :1], 0)
    with pytest.raises(ValueError, match="recent"):
        dm.dm_cache_evict(cache, t, n, w, t[:, :1], 8, recent=9)
    with pytest.raises(ValueError, match="weights"):
        dm.dm_cache_evict(cache, t, n, w[:, :1], t[:, :1], 8)
