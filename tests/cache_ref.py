"""The cache operators from their definitions, in 64 bits on the CPU, one sequence and one head at a time; and the error bounds of the attention.

A cache is held here as the tokens of each sequence: `tokens(cache, table, b, n)` reads values through the block table."""
import math

import torch

BLK = 32


def make_cache(pages, P, Hk, D, seed=0, layout="dense", fill=0xFF):
    """Pools whose every byte is `fill` (0xFF: NaN codes), in one of the layouts that a program may keep."""
    import delta_matching_b200 as dm
    dev = "cuda"
    if layout == "dense":
        raw = [torch.full((pages, Hk, P, D), fill, dtype=torch.uint8, device=dev) for _ in range(2)]
        scales = [torch.full((pages, Hk, P // BLK), float("nan"), device=dev) for _ in range(2)]
    elif layout == "joint":                                      # K and V of a page in one allocation
        both = torch.full((pages, 2, Hk, P, D), fill, dtype=torch.uint8, device=dev)
        sc = torch.full((pages, 2, Hk, P // BLK), float("nan"), device=dev)
        raw, scales = [both[:, 0], both[:, 1]], [sc[:, 0], sc[:, 1]]
    else:                                                        # slot-major storage, seen head-major
        raw = [torch.full((pages, P, Hk, D), fill, dtype=torch.uint8, device=dev).transpose(1, 2) for _ in range(2)]
        scales = [torch.full((pages, Hk, P // BLK), float("nan"), device=dev) for _ in range(2)]
    return dm.KVCache8(*(t.view(torch.float8_e4m3fn) for t in raw), *scales)


def make_table(B, T, pages, seed=0, first=0):
    g = torch.Generator().manual_seed(seed)
    order = torch.randperm(pages, generator=g)[first:first + B * T]
    return order.view(B, T).to(torch.int32)


def scale_of(amax):
    """Smallest power of two s >= 2^-126 with amax <= 448 s, by trial."""
    s = 2.0 ** -126
    while amax > 448.0 * s:
        s *= 2.0
    return s


def grid(x):
    """fp64 values on the grid of e4m3, ties to even, at most 448 in size."""
    a = x.abs()
    e = torch.floor(torch.log2(torch.where(a > 0, a, torch.ones_like(a)))).clamp(min=-6)
    step = torch.exp2(e - 3)
    return torch.sign(x) * (torch.round(a / step) * step).clamp(max=448.0)


def bytes_of(x):
    """e4m3 bytes of values that are on its grid."""
    return x.to(torch.float32).to(torch.float8_e4m3fn).view(torch.uint8)


class Pools:
    """CPU copy of a cache: code bytes and scales."""

    def __init__(self, cache):
        self.codes = [t.view(torch.uint8).cpu().clone() for t in (cache.k8, cache.v8)]
        self.scales = [t.cpu().clone() for t in (cache.ks, cache.vs)]

    def values(self, which, table, b, h, n):
        P = self.codes[0].shape[2]
        out = torch.zeros(n, self.codes[0].shape[3], dtype=torch.float64)
        for j in range(n):
            page, slot = int(table[b, j // P]), j % P
            out[j] = self.codes[which][page, h, slot].view(torch.float8_e4m3fn).double() * float(self.scales[which][page, h, slot // BLK])
        return out


def append(pools, xs, table, lengths, counts):
    """xs = (k, v) (B, N, Hk, D) CPU bf16; changes `pools`."""
    P = pools.codes[0].shape[2]
    for which, x in enumerate(xs):
        for b in range(x.shape[0]):
            for h in range(x.shape[2]):
                j, end = int(lengths[b]), int(lengths[b]) + int(counts[b])
                while j < end:
                    stop = min(end, j - j % BLK + BLK)
                    page, slot, blk = int(table[b, j // P]), j % P, j % P // BLK
                    new = x[b, j - int(lengths[b]):stop - int(lengths[b]), h].double()
                    s = scale_of(float(new.abs().max()))
                    code, scale = pools.codes[which], pools.scales[which]
                    if j % BLK:
                        old = float(scale[page, h, blk])
                        s = max(s, old)
                        rows = slice(blk * BLK, slot)
                        code[page, h, rows] = bytes_of(grid(code[page, h, rows].view(torch.float8_e4m3fn).double() * (old / s)))
                    code[page, h, slot:slot + stop - j] = bytes_of(grid(new / s))
                    scale[page, h, blk] = s
                    j = stop
    return pools


def attention(q, pools, table, lengths, counts, causal, scale):
    """-> o, lse, weights (B, Hk, T * P) in fp64 and bounds of their errors (same shapes).  Bounds: a logit is an fp32 sum of D exact products in an
    unspecified order, off by at most 2^-19 of the sum of their sizes (D 2^-24 and the products with the scales); that moves a probability by
    twice its size relatively, exp2 and the fp32 sums by 2^-19; in the output product a probability, with V's scale, is held in f16 below 2^15 for the row's
    largest: 11 bits (2^-11), and never closer than half of f16's smallest step, 2^-25, which is 2^-40 of the largest; o is rounded to bf16, whose
    eight significant bits err by up to 2^-8 of the value."""
    B, N, H, D = q.shape
    Hk, P = pools.codes[0].shape[1:3]
    W = table.shape[1] * P
    o, lse = torch.zeros(B, N, H, D, dtype=torch.float64), torch.full((B, H, N), -math.inf, dtype=torch.float64)
    w = torch.zeros(B, Hk, W, dtype=torch.float64)
    do, dlse, dw = torch.zeros_like(o), torch.zeros_like(lse), torch.zeros_like(w)
    for b in range(B):
        n, count = int(lengths[b]), int(counts[b])
        if n == 0:
            continue
        for h in range(Hk):
            k, v = pools.values(0, table, b, h, n), pools.values(1, table, b, h, n)
            coarsest = max(float(pools.scales[1][int(table[b, j // P]), h, j % P // BLK]) for j in range(0, n, BLK))
            for hh in range(h * H // Hk, (h + 1) * H // Hk):
                for i in range(count):
                    see = max(0, n - count + i + 1) if causal else n
                    if see == 0:
                        continue
                    qi = q[b, i, hh].double()
                    s = (k[:see] @ qi) * scale
                    eps = float(((k[:see].abs() @ qi.abs()) * scale).max()) * 2.0 ** -19
                    lse[b, hh, i] = torch.logsumexp(s, 0)
                    p = torch.exp(s - lse[b, hh, i])
                    o[b, i, hh] = p @ v[:see]
                    do[b, i, hh] = 2.0 ** -8 * o[b, i, hh].abs() + (2.0 ** -11 + 2 * eps + 2.0 ** -19) * (p @ v[:see].abs()) + 2.0 ** -40 * see * 448 * coarsest + 1e-37
                    dlse[b, hh, i] = eps + 2.0 ** -19 + 2.0 ** -22 * float(lse[b, hh, i].abs())
                    w[b, h, :see] += p
                    dw[b, h, :see] += (2 * eps + 2.0 ** -19 + 2.0 ** -22 * float(lse[b, hh, i].abs())) * p + 1e-37
    return (o, lse, w), (do, dlse, dw)


def evict(pools, table, new_table, lengths, weights, budget, recent):
    """Changes `pools`; -> new lengths, kept, new weights."""
    Hk, P = pools.codes[0].shape[1:3]
    B, T2 = new_table.shape
    kept = torch.full((B, Hk, budget), -1, dtype=torch.int32)
    out = torch.zeros(B, Hk, T2 * P, dtype=torch.float32)
    for b in range(B):
        n = int(lengths[b])
        for h in range(Hk):
            if n <= budget:
                idx = list(range(n))
            else:
                rank = lambda j: -math.inf if math.isnan(float(weights[b, h, j])) else float(weights[b, h, j])
                early = sorted(range(n - recent), key=lambda j: (-rank(j), j))[:budget - recent]
                idx = sorted(early) + list(range(n - recent, n))
            kept[b, h, :len(idx)] = torch.tensor(idx, dtype=torch.int32)
            out[b, h, :len(idx)] = weights[b, h, idx]
            for which in (0, 1):
                x = pools.values(which, table, b, h, n)[idx]
                for j in range(0, len(idx), BLK):
                    part = x[j:j + BLK]
                    page, blk = int(new_table[b, j // P]), j % P // BLK
                    s = scale_of(float(part.abs().nan_to_num(0.0).max()))
                    rows = torch.zeros(BLK, x.shape[1], dtype=torch.uint8)
                    rows[:part.shape[0]] = bytes_of(torch.where(part.isnan(), part, grid(part / s)))
                    pools.codes[which][page, h, blk * BLK:(blk + 1) * BLK] = rows
                    pools.scales[which][page, h, blk] = s
    return torch.tensor([min(int(n), budget) for n in lengths], dtype=torch.int32), kept, out


def same_values(cache, pools):
    """Codes bit for bit up to the sign of zero, scales bit for bit (NaN where never written)."""
    for got, want in zip((cache.k8, cache.v8), pools.codes):
        a, b = got.view(torch.uint8).cpu(), want
        if not bool(((a == b) | (((a | b) & 0x7F) == 0) | (((a & 0x7F) == 0x7F) & ((b & 0x7F) == 0x7F))).all()):
            return False
    return all(torch.equal(a.cpu().view(torch.int32), b.view(torch.int32)) for a, b in zip((cache.ks, cache.vs), pools.scales))


def attention_on_device(q, cache, table, lengths, counts, causal, scale):
    """attention() for sizes that take the CPU too long: the same formulas and bounds, in fp64 on the GPU, one (sequence, kv head) at a time.  -> o, lse and
    bounds; rows that see nothing are 0 and -inf."""
    B, N, H, D = q.shape
    Hk, P = cache.k8.shape[1:3]
    rep = H // Hk
    o, do = torch.zeros(B, N, H, D, dtype=torch.float64, device="cuda"), torch.zeros(B, N, H, D, dtype=torch.float64, device="cuda")
    lse, dlse = torch.full((B, H, N), -math.inf, dtype=torch.float64, device="cuda"), torch.zeros(B, H, N, dtype=torch.float64, device="cuda")
    for b in range(B):
        n, count = int(lengths[b]), int(counts[b])
        if n == 0 or count == 0:
            continue
        at = torch.arange(n, device="cuda")
        page = table[b].to("cuda").long()[at // P]
        see = at[None] < ((n - count + 1 + torch.arange(count, device="cuda")).clamp(min=0)[:, None] if causal else n)
        for h in range(Hk):
            k, v = (c[page, h, at % P].double() * s[page, h, at % P // BLK].double()[:, None] for c, s in ((cache.k8.float(), cache.ks), (cache.v8.float(), cache.vs)))
            coarsest = float(cache.vs[page, h, at % P // BLK].max())
            for hh in range(h * rep, (h + 1) * rep):
                qi = q[b, :count, hh].cuda().double()
                s = (qi @ k.T * scale).masked_fill(~see, -math.inf)
                eps = (qi.abs() @ k.abs().T * scale).masked_fill(~see, 0.0).amax(1) * 2.0 ** -19
                some = see.any(1)
                lse[b, hh, :count] = torch.logsumexp(s, 1)
                p = torch.nan_to_num(torch.softmax(s, 1))
                o[b, :count, hh] = p @ v
                do[b, :count, hh] = (2.0 ** -8 * o[b, :count, hh].abs() + (2.0 ** -11 + 2 * eps + 2.0 ** -19)[:, None] * (p @ v.abs())
                                     + (2.0 ** -40 * see.sum(1) * 448 * coarsest + 1e-37)[:, None])
                dlse[b, hh, :count] = torch.where(some, eps + 2.0 ** -19 + 2.0 ** -22 * lse[b, hh, :count].abs(), 0.0)
    return (o, lse), (do, dlse)
