"""The operators of the 8-bit key/value cache, over the range of calls that a serving loop makes of them.

The cache: pools of pages `k8`, `v8` (pages, Hk, page, D) in e4m3 and their scales `ks`, `vs` (pages, Hk, page // 32), a power of two for each
block of 32 slots and head; a block table (B, T) of page numbers.  A case is one call:
    attn    few or many new queries (B, nq, H, D) over what each sequence holds; `weights`: with the attention weight that each held token got
    append  new tokens (B, new, Hk, D) quantised into the cache behind what it holds
    evict   each sequence cut to `budget` tokens a head: the last `recent` ones and those of greatest accumulated weight
Lengths are spread evenly from `lo` to `hi` over the B sequences, and so are the counts of new tokens (from 1 to all) where a case is `ragged`.
`qk_scale` widens the range of the logits.
"""
import math

import torch

own = False

BLK = 32
E4M3 = torch.float8_e4m3fn


def _case(op, name=None, **kw):
    c = dict(op=op, B=1, Hk=8, D=128, page=64, lo=4096, hi=4096)
    if op == "attn":
        c.update(H=32, nq=1, causal=True, ragged=False, weights=False, qk_scale=1.0)
    elif op == "append":
        c.update(new=1, ragged=False)
    else:
        c.update(budget=2048, recent=256)
    c.update(kw)
    return c if name is None else dict(c, name=name)


def listed():
    return [
        # one short conversation on a toy model: latency is all there is
        _case("attn", "decode tiny", H=8, Hk=2, lo=255, hi=255),
        # one token a sequence at the benchmark's grouped-query layer, a small batch near its training length
        _case("attn", "decode layer", B=4, lo=3601, hi=4096),
        # the same layer in a full serving batch: new and old conversations side by side
        _case("attn", "decode batch ragged", B=64, lo=17, hi=8191),
        # one long document at the long-context configuration's heads (rep = 8)
        _case("attn", "decode long", H=64, page=128, lo=131071, hi=131071),
        # head_dim 256 without groups: a query row a head, the configuration's heads, pages of one block
        _case("attn", "decode wide head", B=8, H=16, Hk=16, D=256, page=32, lo=4001, hi=8192),
        # drafted tokens to be verified, odd head counts, ragged everywhere
        _case("attn", "drafts odd heads", B=3, H=15, Hk=5, nq=5, page=96, lo=611, hi=1792, ragged=True, qk_scale=2.0),
        # decoding that also keeps the books for eviction
        _case("attn", "decode weights", B=16, lo=2049, hi=4096, weights=True),
        # a chunk of a prompt against what came before it
        _case("attn", "prompt chunk", B=2, nq=512, lo=4096, hi=8192),
        # what one decoding step writes for a full batch
        _case("append", "append token", B=64, lo=17, hi=8191),
        # prompts of a small batch, behind prefixes that end inside a block
        _case("append", "append prompts", B=4, new=4096, lo=3, hi=1001, ragged=True),
        # the layer's cache halved
        _case("evict", "evict layer", B=4, lo=3001, hi=4096),
        # a long document cut to a quarter
        _case("evict", "evict long", page=128, lo=131071, hi=131071, budget=32768, recent=1024),
    ]


def _spread(lo, hi, n):
    return [hi] if n == 1 else [round(lo + (hi - lo) * i / (n - 1)) for i in range(n)]


def _counts(most, ragged, n):
    return _spread(1, most, n) if ragged else [most] * n


def _tokens(c):
    """Lengths and new tokens of each sequence, shortest first."""
    return _spread(c["lo"], c["hi"], c["B"]), _counts(c["nq"] if c["op"] == "attn" else c.get("new", 0), c.get("ragged", False), c["B"])


def _table_width(c):
    """Pages a sequence's row of the table has room for."""
    return max(1, -(-(c["hi"] + c.get("new", 0)) // c["page"]))


def work(case):
    c = case
    n, new = _tokens(c)
    held = 2 * (c["D"] + 4 / BLK) * c["Hk"]                      # bytes of a token's K and V
    if c["op"] == "attn":
        rows = c["B"] * c["nq"] * c["H"]
        keys = sum(sum(max(0, a - m + i + 1) if c["causal"] else a for i in range(m)) for a, m in zip(n, new))
        b = sum(n) * held + rows * (4 * c["D"] + 4)
        if c["weights"]:
            b += 4.0 * c["B"] * c["Hk"] * _table_width(c) * c["page"]
        return {"bytes": b, "flops": 4.0 * keys * c["H"] * c["D"]}
    if c["op"] == "append":
        return {"bytes": sum(new) * (held + 4.0 * c["D"] * c["Hk"]), "flops": 2.0 * 2 * sum(new) * c["Hk"] * c["D"]}
    kept = sum(min(a, c["budget"]) for a in n)
    return {"bytes": kept * (2 * held + 8.0 * c["Hk"]) + 4.0 * sum(n) * c["Hk"], "flops": 2.0 * 2 * kept * c["Hk"] * c["D"]}


_MOST = {k: max(work(c)[k] for c in listed()) for k in ("bytes", "flops")}


def _log_uniform(rng, lo, hi):
    return round(math.exp(rng.uniform(math.log(lo), math.log(hi))))


def draw(rng):
    while True:
        op = rng.choice(["attn", "attn", "attn", "append", "evict"])
        hi = _log_uniform(rng, 8, 131072)
        c = _case(op, B=_log_uniform(rng, 1, 64), Hk=_log_uniform(rng, 1, 16), D=rng.choice([128, 128, 256]), page=rng.choice([32, 64, 64, 96, 128, 256]),
                  lo=rng.choice([0, 1, hi // 3, hi]), hi=hi, ragged=rng.random() < 0.4)
        if op == "attn":
            c["H"] = c["Hk"] * rng.choice([1, 2, 3, 4, 4, 5, 7, 8, 8, 16])
            c["nq"] = rng.choice([1, 1, 1, rng.randint(2, 8), _log_uniform(rng, 9, 512)])
            c["causal"], c["weights"], c["qk_scale"] = rng.random() < 0.85, rng.random() < 0.3, rng.choice([1.0, 1.0, 3.0])
        elif op == "append":
            c["new"] = rng.choice([1, rng.randint(2, 40), _log_uniform(rng, 33, 8192)])
        else:
            del c["ragged"]
            c["budget"] = max(1, round(hi * rng.uniform(0.1, 1.1)))
            c["recent"] = rng.randint(0, c["budget"])
        w = work(c)
        padded = c["B"] * (_table_width(c) + 1) * c["page"] * c["Hk"] * c["D"]
        if c.get("H", 1) <= 64 and 0 < w["bytes"] <= _MOST["bytes"] and w["flops"] <= _MOST["flops"] and padded <= 6e8:
            return c


# ---------------------------------------------------------------------------------------------------------------- inputs
def _pow2(amax):
    """Smallest power of two s with amax <= 448 s, at least 2^-126 (fp32)."""
    m, e = torch.frexp(amax / 448.0)
    e = torch.where(amax > 0, e.int() - (m == 0.5).int(), -126).clamp(min=-126)
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _quantised(x):
    """x (..., page, D) fp32 -> codes, scales (..., page // 32)."""
    y = x.view(*x.shape[:-2], x.shape[-2] // BLK, BLK, x.shape[-1])
    s = _pow2(y.abs().amax((-1, -2)))
    return (y / s[..., None, None]).to(E4M3).view(x.shape), s


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda").manual_seed(seed)
    host = torch.Generator().manual_seed(seed)
    B, Hk, D, P = c["B"], c["Hk"], c["D"], c["page"]
    T = _table_width(c)
    T2 = -(-c["budget"] // P) if c["op"] == "evict" else 0
    pages = B * (T + T2) + 3
    order = torch.randperm(pages, generator=host, dtype=torch.int64)
    lengths, new = (torch.tensor(v, dtype=torch.int32) for v in _tokens(c))
    mix = torch.randperm(B, generator=host)

    def rand(*shape):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)

    # keys have channels of a large mean and of a large spread, as the keys of trained layers do
    mean, gain = rand(Hk, 1, D), torch.exp(0.4 * rand(Hk, 1, D))
    k8 = torch.empty(pages, Hk, P, D, device="cuda", dtype=E4M3)
    v8, ks, vs = torch.empty_like(k8), torch.empty(pages, Hk, P // BLK, device="cuda"), torch.empty(pages, Hk, P // BLK, device="cuda")
    step = max(1, (1 << 27) // (Hk * P * D))
    for at in range(0, pages, step):                             # a bounded part of the pools at a time in 32 bits
        part = slice(at, min(pages, at + step))
        n = part.stop - part.start
        k8[part], ks[part] = _quantised(rand(n, Hk, P, D) * gain + mean)
        v8[part], vs[part] = _quantised(rand(n, Hk, P, D))
    s = {"case": dict(c), "k8": k8, "v8": v8, "ks": ks, "vs": vs, "table": order[:B * T].view(B, T).to("cuda", torch.int32),
         "lengths": lengths[mix].cuda(), "new": new[mix].cuda()}
    if c["op"] == "attn":
        # a page is taken into use as it is: what lies behind a sequence's last token may be anything, NaN codes too
        behind = torch.arange(T * P, device="cuda")[None] >= s["lengths"][:, None]
        b, at = behind.nonzero(as_tuple=True)
        page = s["table"].long()[b, at // P]
        junk = torch.randint(0, 256, (at.numel(), 1, 1), generator=g, device="cuda", dtype=torch.uint8)
        for pool in (k8, v8):
            pool.view(torch.uint8)[page, :, at % P] = junk.expand(-1, Hk, D)
        s["q"] = (rand(B, c["nq"], c["H"], D) * c["qk_scale"]).to(torch.bfloat16)
        s["weights"] = torch.zeros(B, Hk, T * P, device="cuda") if c["weights"] else None
    elif c["op"] == "append":
        s["k"] = (rand(B, c["new"], Hk, D) * gain.transpose(0, 1) + mean.transpose(0, 1)).to(torch.bfloat16)
        s["v"] = rand(B, c["new"], Hk, D).to(torch.bfloat16)
    else:
        # sums of attention weights: few heavy tokens (the first ones among them), a long tail, and tokens nobody has looked at
        w = torch.exp(2.0 * rand(B, Hk, T * P))
        w[..., :4] += 100.0
        s["weights"] = w * (torch.rand(B, Hk, T * P, generator=g, device="cuda") > 0.1)
        s["new_table"] = order[B * T:B * (T + T2)].view(B, T2).to("cuda", torch.int32)
    return s


# --------------------------------------------------------------------------------------------------------------- passes
def run(state):
    c = state["case"]
    if not own:
        return _PLAIN[c["op"]](state)
    import delta_matching_b200 as dm
    s = state
    cache = dm.KVCache8(s["k8"], s["v8"], s["ks"], s["vs"])
    if c["op"] == "attn":
        o, lse = dm.dm_cache_attn(s["q"], cache, s["table"], s["lengths"], q_counts=s["new"] if c["ragged"] else None, causal=c["causal"],
                                  weights=s["weights"], return_lse=True)
        return {"o": o, "lse": lse} if s["weights"] is None else {"o": o, "lse": lse, "weights": s["weights"]}
    if c["op"] == "append":
        lengths = dm.dm_cache_append(cache, s["k"], s["v"], s["table"], s["lengths"], counts=s["new"] if c["ragged"] else None)
        return {"lengths": lengths, "k8": s["k8"], "v8": s["v8"], "ks": s["ks"], "vs": s["vs"]}
    lengths, kept, weights = dm.dm_cache_evict(cache, s["table"], s["lengths"], s["weights"], s["new_table"], c["budget"], recent=c["recent"])
    return {"lengths": lengths, "kept": kept, "weights": weights, "k8": s["k8"], "v8": s["v8"], "ks": s["ks"], "vs": s["vs"]}


def _held(codes, scales, table):
    """What the table's pages hold, in token order: (B, Hk, T * page, D) fp32."""
    B, T = table.shape
    _, Hk, P, D = codes.shape
    x = codes.view(torch.uint8)[table.long()].view(E4M3).float().view(B, T, Hk, P // BLK, BLK, D)
    x = x * scales[table.long()][..., None, None]
    return x.view(B, T, Hk, P, D).transpose(1, 2).reshape(B, Hk, T * P, D)


def _plain_attn(s):
    c = s["case"]
    B, nq, H, Hk, D = c["B"], c["nq"], c["H"], c["Hk"], c["D"]
    k, v = _held(s["k8"], s["ks"], s["table"]), _held(s["v8"], s["vs"], s["table"])
    L = k.shape[2]
    pos = torch.arange(L, device="cuda")
    n = s["lengths"].long()
    v = torch.where((pos[None] < n[:, None])[:, None, :, None], v, 0.0)
    i = torch.arange(nq, device="cuda")[None]
    count = s["new"].long()[:, None]
    last = (n[:, None] - count + i + 1) if c["causal"] else n[:, None].expand(B, nq)
    see = pos < torch.where(i < count, last, 0)[..., None]                                  # (B, nq, L)
    q = s["q"].float().view(B, nq, Hk, H // Hk, D).permute(0, 2, 3, 1, 4).reshape(B, Hk, -1, D)
    x = ((q @ k.transpose(2, 3)) * D ** -0.5).view(B, Hk, -1, nq, L)
    x = torch.where(see[:, None, None], x, -math.inf)
    m = x.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, 0.0, m)
    p = torch.exp(x - m)
    del x
    l = p.sum(-1, keepdim=True)
    some = torch.where(l > 0, l, 1.0)
    o = (p.view(B, Hk, -1, L) @ v).view(B, Hk, -1, nq, D) / some
    out = {"o": o.permute(0, 3, 1, 2, 4).reshape(B, nq, H, D).to(torch.bfloat16),
           "lse": torch.where(l > 0, m + torch.log(some), -math.inf).view(B, H, nq)}
    if c["weights"]:
        s["weights"].copy_((p / some).sum((2, 3)))
        out["weights"] = s["weights"]
    return out


def _plain_append(s):
    c = s["case"]
    B, new, Hk, D, P = c["B"], c["new"], c["Hk"], c["D"], c["page"]
    start, count = s["lengths"].long(), s["new"].long()
    blocks = (new + BLK - 2) // BLK + 1                                                     # that new tokens of one sequence can touch
    block = start[:, None] // BLK + torch.arange(blocks, device="cuda")                     # (B, blocks)
    pos = block[..., None] * BLK + torch.arange(BLK, device="cuda")
    i = pos - start[:, None, None]
    is_new, is_old = (i >= 0) & (i < count[:, None, None]), (i < 0)
    touched = is_new.any(-1)
    bs = torch.arange(B, device="cuda")[:, None].expand_as(block)[touched]
    page, sub = s["table"].long()[bs, (block // (P // BLK))[touched]], (block % (P // BLK))[touched]
    is_new, is_old, i = is_new[touched], is_old[touched], i[touched]
    for x, codes, scales in ((s["k"], s["k8"], s["ks"]), (s["v"], s["v8"], s["vs"])):
        pool = codes.view(torch.uint8).view(-1, Hk, P // BLK, BLK, D)
        x = x[bs[:, None], i.clamp(0, new - 1)].float().transpose(1, 2)                     # (touched, Hk, 32, D)
        before, old_scale = pool[page, :, sub], scales[page, :, sub]
        some_new, some_old = is_new[:, None, :, None], is_old[:, None, :, None]
        scale = _pow2(torch.where(some_new, x, 0.0).abs().amax((-1, -2)))
        scale = torch.where(is_old.any(-1)[:, None], torch.maximum(scale, old_scale), scale)
        y = torch.where(some_new, x / scale[..., None, None], before.view(E4M3).float() * (old_scale / scale)[..., None, None])
        pool[page, :, sub] = torch.where(some_new | some_old, y.to(E4M3).view(torch.uint8), before)
        scales[page, :, sub] = scale
    return {"lengths": s["lengths"] + s["new"], "k8": s["k8"], "v8": s["v8"], "ks": s["ks"], "vs": s["vs"]}


def _plain_evict(s):
    c = s["case"]
    B, Hk, D, P, m = c["B"], c["Hk"], c["D"], c["page"], c["budget"]
    w, n = s["weights"], s["lengths"].long()[:, None, None]
    L, T2 = w.shape[2], s["new_table"].shape[1]
    pos = torch.arange(L, device="cuda").expand(B, Hk, L)
    by_weight = torch.sort(torch.where(torch.isnan(w), -math.inf, w), dim=-1, descending=True, stable=True).indices
    kind = torch.where(pos >= n, 0, torch.where(pos >= n - c["recent"], 2, 1)).gather(2, by_weight)
    order = by_weight.gather(2, torch.sort(kind, dim=-1, descending=True, stable=True).indices)
    order = torch.cat([order, order.new_full((B, Hk, max(0, T2 * P - L)), L)], 2)[..., :T2 * P]
    rank = torch.arange(T2 * P, device="cuda")
    left = n.clamp(max=m)
    kept = torch.sort(torch.where(rank < left, order, L), dim=-1).values
    valid = rank < left
    at = torch.where(valid, kept, 0)
    h = torch.arange(Hk, device="cuda")[None, :, None]
    page = s["table"].long().gather(1, (at // P).view(B, -1)).view(B, Hk, -1)
    block = torch.arange(T2 * P // BLK, device="cuda")
    touched = (block * BLK < left[:, 0]).nonzero(as_tuple=True)                             # (sequence, new block)
    to, sub = s["new_table"].long()[touched[0], touched[1] // (P // BLK)], touched[1] % (P // BLK)
    for codes, scales in ((s["k8"], s["ks"]), (s["v8"], s["vs"])):
        bytes_ = codes.view(torch.uint8)
        x = bytes_[page, h, at % P].view(E4M3).float() * scales[page, h, at % P // BLK][..., None]
        x = torch.where(valid[..., None], x, 0.0).view(B, Hk, -1, BLK, D)
        scale = _pow2(x.abs().amax((-1, -2)))
        y = (x / scale[..., None, None]).to(E4M3).view(torch.uint8)
        bytes_.view(-1, Hk, P // BLK, BLK, D)[to, :, sub] = y[touched[0], :, touched[1]]
        scales[to, :, sub] = scale[touched[0], :, touched[1]]
    return {"lengths": s["lengths"].clamp(max=m), "kept": torch.where(valid, kept, -1)[..., :m].to(torch.int32),
            "weights": torch.where(valid, w.gather(2, at), 0.0), "k8": s["k8"], "v8": s["v8"], "ks": s["ks"], "vs": s["vs"]}


_PLAIN = {"attn": _plain_attn, "append": _plain_append, "evict": _plain_evict}


# ---------------------------------------------------------------------------------------------------------------- exact
def _e4m3_grid(x):
    """x (fp64, at most 448 in size) on the grid of e4m3, ties to even."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(x / step) * step


def _scale64(amax):
    """2^max(-126, ceil(log2(amax / 448))), by counting powers of two that are too small."""
    s = torch.full_like(amax, 2.0 ** -126)
    for e in (128, 64, 32, 16, 8, 4, 2, 1):
        s = torch.where(amax > 448 * s * 2.0 ** (e - 1), s * 2.0 ** e, s)
    return s


def _rows64(s, b, n, codes, scales):
    """The first n tokens of sequence b: (Hk, n, D) fp64."""
    P = s["case"]["page"]
    at = torch.arange(n, device="cuda")
    page = s["table"][b].long()[at // P]
    return (codes[page, :, at % P].double() * scales[page, :, at % P // BLK].double()[..., None]).transpose(0, 1)


def _exact_attn(s):
    c = s["case"]
    H, Hk, D = c["H"], c["Hk"], c["D"]
    o, lse = torch.zeros(s["q"].shape, device="cuda", dtype=torch.float64), torch.full((c["B"], H, c["nq"]), -math.inf, device="cuda", dtype=torch.float64)
    weights = torch.zeros_like(s["weights"], dtype=torch.float64) if c["weights"] else None
    for b, (n, count) in enumerate(zip(s["lengths"].tolist(), s["new"].tolist())):
        if n == 0 or count == 0:
            continue
        k, v = _rows64(s, b, n, s["k8"].float(), s["ks"]), _rows64(s, b, n, s["v8"].float(), s["vs"])
        for h in range(H):
            x = s["q"][b, :count, h].double() @ k[h * Hk // H].T / math.sqrt(D)
            if c["causal"]:
                hidden = torch.arange(n, device="cuda")[None] > torch.arange(count, device="cuda")[:, None] + n - count
                x = x.masked_fill(hidden, -math.inf)
            lse[b, h, :count] = torch.logsumexp(x, -1)
            p = torch.nan_to_num(torch.softmax(x, -1))
            o[b, :count, h] = p @ v[h * Hk // H]
            if c["weights"]:
                weights[b, h * Hk // H, :n] += p.sum(0)
    return {"o": o, "lse": lse, "weights": weights} if c["weights"] else {"o": o, "lse": lse}


def _exact_append(s):
    c = s["case"]
    P, out = c["page"], {"lengths": s["lengths"] + s["new"]}
    for name, x, codes, scales in (("k", s["k"], s["k8"], s["ks"]), ("v", s["v"], s["v8"], s["vs"])):
        codes, scales = codes.double(), scales.double()
        for b, (n, count) in enumerate(zip(s["lengths"].tolist(), s["new"].tolist())):
            i = 0
            while i < count:
                slot, take = (n + i) % P, min(BLK - (n + i) % BLK, count - i)
                page, blk, first = int(s["table"][b, (n + i) // P]), slot // BLK, slot - slot % BLK
                y = x[b, i:i + take].double().transpose(0, 1)
                scale = _scale64(y.abs().amax((1, 2)))
                if slot % BLK:
                    scale = torch.maximum(scale, scales[page, :, blk])
                    codes[page, :, first:slot] = _e4m3_grid(codes[page, :, first:slot] * (scales[page, :, blk] / scale)[:, None, None])
                codes[page, :, slot:slot + take], scales[page, :, blk] = _e4m3_grid(y / scale[:, None, None]), scale
                i += take
        out.update({name + "8": codes, name + "s": scales})
    return out


def _exact_evict(s):
    c = s["case"]
    B, Hk, P, m = c["B"], c["Hk"], c["page"], c["budget"]
    T2 = s["new_table"].shape[1]
    kept = torch.full((B, Hk, m), -1, device="cuda", dtype=torch.int32)
    weights = torch.zeros(B, Hk, T2 * P, device="cuda", dtype=torch.float64)
    new = {"k8": s["k8"].double(), "v8": s["v8"].double(), "ks": s["ks"].double(), "vs": s["vs"].double()}
    for b, n in enumerate(s["lengths"].tolist()):
        left = min(n, m)
        if left == 0:
            continue
        late = min(c["recent"], n) if n > m else n
        recent = torch.arange(n - late, n, device="cuda")
        idx = torch.empty(Hk, left, device="cuda", dtype=torch.int64)
        for h in range(Hk):
            idx[h, left - late:] = recent
            if left > late:                                      # of the least weight kept, the lowest indices
                w = s["weights"][b, h, :n - late]
                least = torch.sort(w, descending=True).values[left - late - 1]
                above, equal = (w > least).nonzero()[:, 0], (w == least).nonzero()[:, 0]
                idx[h, :left - late] = torch.cat([above, equal[:left - late - above.numel()]]).sort().values
        kept[b, :, :left], weights[b, :, :left] = idx.int(), s["weights"][b].double().gather(1, idx)
        full = -(-left // BLK)
        for name in "kv":
            x = _rows64(s, b, n, s[name + "8"].float(), s[name + "s"]).gather(1, idx[..., None].expand(-1, -1, c["D"]))
            x = torch.nn.functional.pad(x, (0, 0, 0, full * BLK - left)).view(Hk, full, BLK, c["D"])
            scale = _scale64(x.abs().amax((2, 3)))
            y = _e4m3_grid(x / scale[..., None, None])
            for j in range(full):
                page, blk = int(s["new_table"][b, j * BLK // P]), j % (P // BLK)
                new[name + "8"][page, :, blk * BLK:(blk + 1) * BLK], new[name + "s"][page, :, blk] = y[:, j], scale[:, j]
    return {"lengths": s["lengths"].clamp(max=m), "kept": kept, "weights": weights, **new}


def exact(case, seed):
    return {"attn": _exact_attn, "append": _exact_append, "evict": _exact_evict}[case["op"]](prepare(case, seed))
