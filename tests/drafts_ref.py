"""The functions for drafted tokens from their definitions, in 64 bits, a sequence and a head at a time, beside cache_ref.py; and their error bounds."""
import math

import torch

from . import cache_ref as ref

BLK = ref.BLK


def make_parents(kind, B, N, seed=0):
    """(B, N) int32: a chain, all children of the first node, all roots, or any earlier node or none."""
    g = torch.Generator().manual_seed(seed)
    i = torch.arange(N).expand(B, N)
    if kind == "chain":
        p = i - 1
    elif kind == "star":
        p = torch.where(i == 0, -1, 0)
    elif kind == "roots":
        p = torch.full((B, N), -1)
    elif kind == "near":                                         # one of the five nodes before
        p = (i - 1 - (torch.rand(B, N, generator=g) * 5).long()).clamp(min=-1)
    else:
        p = (torch.rand(B, N, generator=g) * (i + 1)).long() - 1
    return p.to(torch.int32)


def tree(parents, counts):
    """-> depth (B, N) int32, truth values (B, N, N), by walking."""
    B, N = parents.shape
    depth, see = torch.zeros(B, N, dtype=torch.int32), torch.zeros(B, N, N, dtype=torch.bool)
    for b in range(B):
        for i in range(int(counts[b])):
            at = int(parents[b, i])
            see[b, i, i] = True
            while at >= 0:
                see[b, i, at] = True
                depth[b, i] += 1
                at = int(parents[b, at])
    return depth, see


def pack(see):
    """Truth values (B, N, M) as words of 32 bits, int32."""
    B, N, M = see.shape
    W = -(-M // 32)
    bits = torch.nn.functional.pad(see.long(), (0, 32 * W - M)).view(B, N, W, 32) << torch.arange(32)
    return bits.sum(-1).to(torch.int32)                          # (wraps: the bits are what counts)


def rotate(x, positions, freqs, interleaved):
    """x (..., N, heads, D) bf16, positions (..., N) -> the rotated values in fp64 and a bound of what fp32 makes of them: the angle is reduced in 64 bits and
    rounded to 32 (2^-23 for angles up to pi), sine and cosine are off by 2 units at most (2^-23), products and their sum by half a unit each
    (2^-24 of |x| + |y| three times): less than 2^-21 of |x| + |y| in all."""
    F = freqs.numel()
    a = torch.arange(F) * 2 if interleaved else torch.arange(F)
    b = a + 1 if interleaved else a + F
    angle = positions.double()[..., None] * freqs.double()
    cos, sin = torch.cos(angle)[..., None, :], torch.sin(angle)[..., None, :]
    y, off = x.double().clone(), torch.zeros(x.shape, dtype=torch.float64)
    u, v = x.double()[..., a], x.double()[..., b]
    y[..., a], y[..., b] = u * cos - v * sin, v * cos + u * sin
    off[..., a] = off[..., b] = (u.abs() + v.abs()) * 2.0 ** -21
    return y, off


def held_tokens(pools, which, table, b, n):
    """The first n tokens of sequence b: (Hk, n, D) fp64."""
    return torch.stack([pools.values(which, table, b, h, n) for h in range(pools.codes[0].shape[1])])


def keep(pools, table, before, path, counts):
    """Changes `pools` as dm_cache_keep does; -> new lengths."""
    Hk, P = pools.codes[0].shape[1:3]
    for b in range(len(before)):
        n, count = int(before[b]), int(counts[b])
        if count == 0:
            continue
        top = n + int(path[b, count - 1]) + 1
        for which in (0, 1):
            for h in range(Hk):
                all_ = pools.values(which, table, b, h, top)
                begin = n - n % BLK
                kept = torch.cat([all_[begin:n], all_[n + path[b, :count].long()]])
                for j in range(0, kept.shape[0], BLK):
                    part = kept[j:j + BLK]
                    at = begin + j
                    page, slot = int(table[b, at // P]), at % P
                    s = ref.scale_of(float(part.abs().nan_to_num(0.0).max()))
                    pools.codes[which][page, h, slot:slot + part.shape[0]] = ref.bytes_of(torch.where(part.isnan(), part, ref.grid(part / s)))
                    pools.scales[which][page, h, slot // BLK] = s
    return torch.tensor([int(a) + int(c) for a, c in zip(before, counts)], dtype=torch.int32)


def attention(q, cache, table, lengths, counts, see, scale):
    """-> (o, lse) in fp64 and bounds of their errors, on the GPU.

    Bounds.  A logit is an fp32 sum of D products in any order: 2^-19 of the sum of their sizes, as in cache_ref.py.  q is held as two codes per element,
    its row's largest brought to 2^7 ... 2^8: e4m3 (4 bits; a step of 2^-9 below 2^-6) and what that leaves in e5m2 (3 bits).  What is left of an element of at least 2^-6 is at
    most 8 times its eighth bit, which 3 bits hold; below, at most 2^-10 is left, on steps of 2^-13: off by 2^-14, 2^-21 of the largest element.  That times the sum of the
    sizes of the key's channels.  Both move a probability by twice as much relatively; exp2 and the fp32 sums by 2^-19.  A probability is held in the output product
    with the largest of its block of 32 keys brought to 2^7 ... 2^8 as an e4m3 code of its first four bits (below 2^(e-3) is left, for 2^e ... 2^(e+1)) and an e4m3 code of
    the rest, off by 2^(e-8): 2^-8 of itself.  Where either is below 2^-6 its code is off by up to 2^-10: together 2^-9, 2^-16 of the block's largest.  o is rounded to bf16 (2^-8).

    The codes of a block count in powers of two from 2^-127 of 2^u on, u fixed: 40 above the largest product 2^t of a probability and a V scale in the first blocks, or 40 where the row
    sees nothing in these (then it is made by itself if all its products are below 2^-40).  A smaller product counts as that: a key's value is off by up to 2^8 448 2^(u - 127), 2^(u - 110).  That
    is 2^-69 of the largest product (2^(u - 41) at least), or 2^-29 where u was not taken from it: times the number of keys."""
    B, N, H, D = q.shape
    Hk, P = cache.k8.shape[1:3]
    dev = "cuda"
    o, do = torch.zeros(B, N, H, D, dtype=torch.float64, device=dev), torch.zeros(B, N, H, D, dtype=torch.float64, device=dev)
    lse, dlse = torch.full((B, H, N), -math.inf, dtype=torch.float64, device=dev), torch.zeros(B, H, N, dtype=torch.float64, device=dev)
    k32, v32 = cache.k8.float(), cache.v8.float()
    for b in range(B):
        n, count = int(lengths[b]), int(counts[b])
        if count == 0:
            continue
        at = torch.arange(n, device=dev)
        page = table[b].to(dev).long()[at // P]
        sees = torch.ones(count, n, dtype=torch.bool, device=dev)
        sees[:, n - count:] = see[b, :count, :count].to(dev)
        for h in range(Hk):
            k, v = (c[page, h, at % P].double() * s[page, h, at % P // BLK].double()[:, None] for c, s in ((k32, cache.ks), (v32, cache.vs)))
            vs = cache.vs[page, h, at % P // BLK].double()
            for hh in range(h * H // Hk, (h + 1) * H // Hk):
                qi = q[b, :count, hh].to(dev).double()
                zero = lambda x: x.masked_fill(~sees, 0.0)       # (what is not seen may be anything)
                s = (qi @ k.T * scale).masked_fill(~sees, -math.inf)
                eps = (zero(qi.abs() @ k.abs().T * scale).amax(1) * 2.0 ** -19
                       + 2.0 ** -21 * qi.abs().amax(1) * (zero(k.abs().sum(1).expand(count, n)).amax(1) * scale))
                lse[b, hh, :count] = torch.logsumexp(s, 1)
                p = torch.softmax(s, 1)
                pad = -n % BLK
                top = torch.nn.functional.pad(p, (0, pad)).view(count, -1, BLK).amax(2).repeat_interleave(BLK, 1)[:, :n]       # of the key's block
                if bool(torch.isfinite(v).all()):
                    pv, pav, tav = p @ v, p @ v.abs(), zero(top) @ v.abs()
                else:                                            # each row over what it sees
                    rows = [[x[i, sees[i]] @ y[sees[i]] for x, y in ((p, v), (p, v.abs()), (top, v.abs()))] for i in range(count)]
                    pv, pav, tav = (torch.stack(x) for x in zip(*rows))
                o[b, :count, hh] = pv
                do[b, :count, hh] = 2.0 ** -8 * pv.abs() + (2.0 ** -8 + 2 * eps + 2.0 ** -19)[:, None] * pav + 2.0 ** -16 * tav + (n * 2.0 ** -29 * (p * vs).amax(1))[:, None] + 1e-37
                dlse[b, hh, :count] = eps + 2.0 ** -19 + 2.0 ** -22 * lse[b, hh, :count].abs()
    return (o, lse), (do, dlse)
