"""The operators of drafted tokens over the 8-bit key/value cache, over the range of calls that a serving loop makes of them.

A step of such a loop: a small model drafts a tree of tokens behind each sequence; their queries and keys get their position's rotation and the keys
and values go into the cache; every drafted token attends to the sequence and to its own ancestors; and of the tree one path is kept.  The cache is
that of operators.py: pools of pages `k8`, `v8` (pages, Hk, page, D) in e4m3, their scales `ks`, `vs` (pages, Hk, page // 32), a power of two for each
block of 32 slots and head, and a block table (B, T) of page numbers.  A case is one call:
    tree    parents (B, nodes) -> depths and, as bits, which nodes each node sees: itself and its ancestors
    append  new tokens: q and k rotated by position (angle = position x frequency), k and v quantised into the cache behind what it holds
    attn    the queries of `nodes` drafted tokens over what is held before them (all of it) and over the drafted tokens that they see
    keep    the tokens of a path through the tree moved together behind what was held before it
Lengths (before the new tokens) are spread evenly from `lo` to `hi` over the B sequences, and so are the counts of new tokens (from 1 to all) where a case
is `ragged`.  `span`: how far back a node's parent may lie; `roots`: whether the first node is the only one without a parent.
"""
import math

import torch

own = False

BLK = 32
E4M3 = torch.float8_e4m3fn


def _case(op, name=None, **kw):
    c = dict(op=op, B=1, new=16, ragged=False)
    if op != "tree":
        c.update(Hk=8, D=128, page=64, lo=4096, hi=4096)
    if op != "append":
        c.update(span=8, roots=False)
    if op == "attn":
        c.update(H=32, qk_scale=1.0)
    elif op == "append":
        c.update(H=32, tree=False, rotary=128, interleaved=False)
    c.update(kw)
    return c if name is None else dict(c, name=name)


def listed():
    return [
        # a few short trees: latency is all there is
        _case("tree", "tree small batch", B=4, new=17),
        # long drafts, mostly chains, for a full batch, ragged
        _case("tree", "tree long drafts", B=64, new=509, span=3, roots=True, ragged=True),
        # what one decoding step writes for a full batch
        _case("append", "rotate token", B=64, new=1, lo=17, hi=8190),
        # drafted trees far into their documents: half of head_dim rotated, in neighbouring pairs; odd counts
        _case("append", "rotate drafts", B=16, new=23, tree=True, ragged=True, rotary=64, interleaved=True, lo=30001, hi=120000, page=96, H=20, Hk=5),
        # prompts of a small batch behind prefixes that end inside a block
        _case("append", "rotate prompts", B=4, new=4096, lo=3, hi=1001, ragged=True),
        # one short conversation on a toy model, odd head counts
        _case("attn", "verify tiny", H=15, Hk=5, new=7, lo=255, hi=255, page=96, qk_scale=2.0),
        # trees of 16 at the benchmark's grouped-query layer, a small batch near its training length
        _case("attn", "verify layer", B=4, lo=3585, hi=4080),
        # the same layer in a full serving batch, new and old conversations side by side, trees of all sizes
        _case("attn", "verify batch ragged", B=64, new=25, lo=17, hi=8166, ragged=True, roots=True),
        # one long document at the long-context configuration's heads (rep = 8) and a large tree
        _case("attn", "verify long", H=64, new=60, page=128, lo=131011, hi=131011),
        # head_dim 256 without groups, pages of one block
        _case("attn", "verify wide head", B=8, H=16, Hk=16, D=256, new=33, page=32, lo=3968, hi=8159),
        # a path of a small tree kept, for the layer's batch
        _case("keep", "keep layer", B=4, lo=3585, hi=4080),
        # long drafts of a full batch of which most is kept, across blocks
        _case("keep", "keep long drafts", B=64, new=250, span=2, lo=33, hi=2041, page=96, ragged=True),
    ]


def _spread(lo, hi, n):
    return [hi] if n == 1 else [round(lo + (hi - lo) * i / (n - 1)) for i in range(n)]


def _tokens(c):
    """Lengths before the call and new tokens of each sequence, shortest first."""
    n = _spread(c["lo"], c["hi"], c["B"]) if "hi" in c else [0] * c["B"]
    return n, _spread(1, c["new"], c["B"]) if c["ragged"] else [c["new"]] * c["B"]


def _words(c):
    return -(-c["new"] // 32)


def work(case):
    c = case
    n, new = _tokens(c)
    nodes = c["B"] * c["new"]
    if c["op"] == "tree":
        return {"bytes": 4.0 * nodes * (2 + _words(c)), "flops": 1.0 * nodes * _words(c)}
    held = 2 * (c["D"] + 4 / BLK) * c["Hk"]                      # bytes of a token's K and V
    if c["op"] == "attn":
        rows = nodes * c["H"]
        keys = sum(a * m + m for a, m in zip(n, new))            # each drafted token sees itself at least
        return {"bytes": (sum(n) + sum(new)) * held + rows * (4.0 * c["D"] + 4) + 4.0 * nodes * _words(c), "flops": 4.0 * keys * c["H"] * c["D"]}
    if c["op"] == "append":
        q = c["B"] * c["new"] * c["H"] * c["D"]
        return {"bytes": sum(new) * (held + 4.0 * c["D"] * c["Hk"]) + 4.0 * q, "flops": 3.0 * sum(new) * c["rotary"] * (c["H"] + c["Hk"]) + 4.0 * sum(new) * c["Hk"] * c["D"]}
    # a path that is not the tree's first nodes is read and written once
    return {"bytes": 2.0 * sum(new) * held / 2 + 4.0 * sum(new), "flops": 2.0 * sum(new) * c["Hk"] * c["D"]}


_MOST = {k: max(work(c)[k] for c in listed()) for k in ("bytes", "flops")}


def _log_uniform(rng, lo, hi):
    return round(math.exp(rng.uniform(math.log(lo), math.log(hi))))


def draw(rng):
    while True:
        op = rng.choice(["attn", "attn", "attn", "append", "append", "tree", "keep"])
        c = _case(op, B=_log_uniform(rng, 1, 64), ragged=rng.random() < 0.4)
        if op == "append":
            c["tree"] = rng.random() < 0.4
            c["new"] = rng.choice([1, rng.randint(2, 40), _log_uniform(rng, 33, 8192)]) if not c["tree"] else _log_uniform(rng, 1, 256)
        else:
            # a tree has some nodes and a choice of parents: a chain is the same whatever the seed
            c["new"] = _log_uniform(rng, 16 if op == "tree" else 1, {"tree": 1024, "attn": 256, "keep": 512}[op])
            c["span"], c["roots"] = rng.choice([2, 3, 8, 64] if op == "tree" else [1, 2, 8, 64]), rng.random() < 0.3
        if op != "tree":
            hi = _log_uniform(rng, 8, 131072)
            c.update(Hk=_log_uniform(rng, 1, 16), D=rng.choice([128, 128, 256]), page=rng.choice([32, 64, 64, 96, 128, 256]), lo=rng.choice([0, 1, hi // 3, hi]), hi=hi)
        if op in ("attn", "append"):
            c["H"] = c["Hk"] * rng.choice([1, 2, 3, 4, 4, 5, 7, 8, 8, 16])
        if op == "attn":
            c["qk_scale"] = rng.choice([1.0, 1.0, 3.0])
        elif op == "append":
            c["rotary"], c["interleaved"] = rng.choice([c["D"], c["D"], c["D"] // 2, 16 * rng.randint(1, c["D"] // 16)]), rng.random() < 0.4
        w = work(c)
        padded = c["B"] * (_table_width(c) + 1) * c["page"] * c["Hk"] * c["D"] if op != "tree" else 0
        scores = c["B"] * c["H"] * c["new"] * (c["hi"] + c["new"]) if op == "attn" else c["B"] * c["new"] ** 2 if op == "tree" else 0
        if c.get("H", 1) <= 64 and w["bytes"] <= _MOST["bytes"] and w["flops"] <= _MOST["flops"] and padded <= 6e8 and scores <= 1.2e9:
            return c


def _table_width(c):
    """Pages a sequence's row of the table has room for."""
    return max(1, -(-(c["hi"] + c["new"]) // c["page"]))


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


def _parents(c, g):
    """Parents (B, new) int64 on the host: a node's parent is one of the `span` nodes before it, or none."""
    i = torch.arange(c["new"])
    back = 1 + (torch.rand(c["B"], c["new"], generator=g) * c["span"]).long().clamp(max=c["span"] - 1)
    parents = i - back
    return parents.clamp(min=-1) if c["roots"] else torch.where(i == 0, -1, parents.clamp(min=0))


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda").manual_seed(seed)
    host = torch.Generator().manual_seed(seed)
    B, N = c["B"], c["new"]
    lengths, new = (torch.tensor(v, dtype=torch.int32) for v in _tokens(c))
    mix = torch.randperm(B, generator=host)
    s = {"case": dict(c), "new": new[mix].cuda()}
    if c["op"] == "tree":
        return dict(s, parents=_parents(c, host).to("cuda", torch.int32))
    Hk, D, P = c["Hk"], c["D"], c["page"]
    T = _table_width(c)
    pages = B * T + 3
    order = torch.randperm(pages, generator=host, dtype=torch.int64)

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
    s.update(k8=k8, v8=v8, ks=ks, vs=vs, table=order[:B * T].view(B, T).to("cuda", torch.int32), before=lengths[mix].cuda())
    s["lengths"] = s["before"] + s["new"]                        # with the drafted tokens
    if c["op"] != "append":
        # a page is taken into use as it is: what lies behind a sequence's last token may be anything, NaN codes too
        behind = torch.arange(T * P, device="cuda")[None] >= s["lengths"][:, None]
        b, at = behind.nonzero(as_tuple=True)
        page = s["table"].long()[b, at // P]
        junk = torch.randint(0, 256, (at.numel(), 1, 1), generator=g, device="cuda", dtype=torch.uint8)
        for pool in (k8, v8):
            pool.view(torch.uint8)[page, :, at % P] = junk.expand(-1, Hk, D)
    if c["op"] == "attn":
        s["q"] = (rand(B, N, c["H"], D) * c["qk_scale"]).to(torch.bfloat16)
        s["depth"], s["seen"] = _plain_tree(_parents(c, host).cuda(), s["new"])
    elif c["op"] == "append":
        s["q"] = rand(B, N, c["H"], D).to(torch.bfloat16)
        s["k"] = (rand(B, N, Hk, D) * gain.transpose(0, 1) + mean.transpose(0, 1)).to(torch.bfloat16)
        s["v"] = rand(B, N, Hk, D).to(torch.bfloat16)
        half = c["rotary"] // 2
        s["freqs"] = (500000.0 ** (-torch.arange(half, dtype=torch.float64) / half)).float().cuda()
        s["offsets"] = _plain_tree(_parents(dict(c, span=8, roots=False), host).cuda(), s["new"])[0] if c["tree"] else None
    else:
        # the path to a node in the later part of the tree (the nodes are in topological order, and so is the path)
        parents, to = _parents(c, host), (new[mix].double() * (0.6 + 0.4 * torch.rand(B, generator=host, dtype=torch.float64))).long()
        path, kept = torch.zeros(B, N, dtype=torch.int32), torch.zeros(B, dtype=torch.int32)
        for b in range(B):
            at, nodes = min(int(to[b]), int(new[mix][b]) - 1), []
            while at >= 0:
                nodes.append(at)
                at = int(parents[b, at])
            path[b, :len(nodes)], kept[b] = torch.tensor(nodes[::-1], dtype=torch.int32), len(nodes)
        s["path"], s["kept"] = path.cuda(), kept.cuda()
    return s


# --------------------------------------------------------------------------------------------------------------- passes
def run(state):
    s, c = state, state["case"]
    if not own:
        return _PLAIN[c["op"]](state)
    import delta_matching_b200 as dm
    counts = s["new"] if c["ragged"] else None
    if c["op"] == "tree":
        tree = dm.dm_draft_tree(s["parents"], counts=counts)
        return {"depth": tree.depth, "seen": tree.seen}
    cache = dm.KVCache8(s["k8"], s["v8"], s["ks"], s["vs"])
    if c["op"] == "attn":
        o, lse = dm.dm_cache_attn_tree(s["q"], cache, s["table"], s["lengths"], dm.DraftTree(s["depth"], s["seen"], counts), return_lse=True)
        return {"o": o, "lse": lse}
    if c["op"] == "append":
        q, lengths = dm.dm_cache_append_rotary(cache, s["q"], s["k"], s["v"], s["table"], s["before"], s["freqs"], offsets=s["offsets"], counts=counts,
                                               interleaved=c["interleaved"])
        return {"q": q, "lengths": lengths, "k8": s["k8"], "v8": s["v8"], "ks": s["ks"], "vs": s["vs"]}
    lengths = dm.dm_cache_keep(cache, s["table"], s["before"], s["lengths"], s["path"], s["kept"])
    return {"lengths": lengths, "k8": s["k8"], "v8": s["v8"], "ks": s["ks"], "vs": s["vs"]}


def _plain_tree(parents, counts):
    B, N = parents.shape
    i = torch.arange(N, device=parents.device)
    real = i < counts[:, None]
    # ancestors by doubling: paths of up to 1, 3, 7, ... steps
    see = ((parents[:, :, None] == i) | (i[:, None] == i)).float()
    for _ in range(max(1, (N - 1).bit_length())):
        see = torch.minimum(see @ see, see.new_ones(()))
    see = see * real[:, :, None]
    depth = torch.where(real, see.sum(-1) - 1, 0.0).to(torch.int32)
    W = -(-N // 32)
    bits = torch.nn.functional.pad(see, (0, 32 * W - N)).view(B, N, W, 32).long() << torch.arange(32, device=parents.device)
    word = bits.sum(-1)
    return depth, torch.where(word >= 2 ** 31, word - 2 ** 32, word).to(torch.int32)


def _seen_nodes(seen, N):
    """Bits (B, N, W) -> (B, N, N) truth values."""
    return ((seen[..., None] >> torch.arange(32, device=seen.device)) & 1).flatten(2)[..., :N] != 0


def _held(codes, scales, table):
    """What the table's pages hold, in token order: (B, Hk, T * page, D) fp32."""
    B, T = table.shape
    _, Hk, P, D = codes.shape
    x = codes.view(torch.uint8)[table.long()].view(E4M3).float().view(B, T, Hk, P // BLK, BLK, D)
    x = x * scales[table.long()][..., None, None]
    return x.view(B, T, Hk, P, D).transpose(1, 2).reshape(B, Hk, T * P, D)


def _plain_attn(s):
    c = s["case"]
    B, N, H, Hk, D = c["B"], c["new"], c["H"], c["Hk"], c["D"]
    k, v = _held(s["k8"], s["ks"], s["table"]), _held(s["v8"], s["vs"], s["table"])
    L = k.shape[2]
    pos = torch.arange(L, device="cuda")
    n, count = s["lengths"].long()[:, None], s["new"].long()[:, None]
    v = torch.where((pos < n)[:, None, :, None], v, 0.0)
    at = pos - (n - count)                                                                  # (B, L): index among the drafted tokens
    among = torch.gather(_seen_nodes(s["seen"], N), 2, at.clamp(0, N - 1)[:, None].expand(B, N, L)) & (at >= 0)[:, None] & (pos < n)[:, None]
    see = ((at < 0)[:, None] | among) & (torch.arange(N, device="cuda") < count)[..., None]         # (B, N, L)
    q = s["q"].float().view(B, N, Hk, H // Hk, D).permute(0, 2, 3, 1, 4).reshape(B, Hk, -1, D)
    x = ((q @ k.transpose(2, 3)) * D ** -0.5).view(B, Hk, -1, N, L)
    x = torch.where(see[:, None, None], x, -math.inf)
    m = x.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, 0.0, m)
    p = torch.exp(x - m)
    del x
    l = p.sum(-1, keepdim=True)
    some = torch.where(l > 0, l, 1.0)
    o = (p.view(B, Hk, -1, L) @ v).view(B, Hk, -1, N, D) / some
    return {"o": o.permute(0, 3, 1, 2, 4).reshape(B, N, H, D).to(torch.bfloat16), "lse": torch.where(l > 0, m + torch.log(some), -math.inf).view(B, H, N)}


def _rotated(x, s, positions):
    """x (B, N, heads, D) bf16 -> fp32, its first 2 len(freqs) channels rotated: pairs (j, j + half), or (2 j, 2 j + 1) where interleaved."""
    angle = positions[..., None].double() * s["freqs"].double()
    cos, sin = torch.cos(angle).float()[:, :, None], torch.sin(angle).float()[:, :, None]
    half = s["freqs"].numel()
    x = x.float()
    if s["case"]["interleaved"]:
        a, b = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = x[..., :half], x[..., half:2 * half]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([turned, x[..., 2 * half:]], -1)


def _plain_append(s):
    c = s["case"]
    B, new, Hk, D, P = c["B"], c["new"], c["Hk"], c["D"], c["page"]
    start, count = s["before"].long(), s["new"].long()
    i = torch.arange(new, device="cuda")
    positions = start[:, None] + (i if s["offsets"] is None else s["offsets"].long())
    q = torch.where((i < count[:, None])[..., None, None], _rotated(s["q"], s, positions), 0.0).to(torch.bfloat16)
    blocks = (new + BLK - 2) // BLK + 1                                                     # that new tokens of one sequence can touch
    block = start[:, None] // BLK + torch.arange(blocks, device="cuda")                     # (B, blocks)
    pos = block[..., None] * BLK + torch.arange(BLK, device="cuda")
    i = pos - start[:, None, None]
    is_new, is_old = (i >= 0) & (i < count[:, None, None]), (i < 0)
    touched = is_new.any(-1)
    bs = torch.arange(B, device="cuda")[:, None].expand_as(block)[touched]
    page, sub = s["table"].long()[bs, (block // (P // BLK))[touched]], (block % (P // BLK))[touched]
    is_new, is_old, i = is_new[touched], is_old[touched], i[touched]

    def write(x, codes, scales):
        pool = codes.view(torch.uint8).view(-1, Hk, P // BLK, BLK, D)
        x = x[bs[:, None], i.clamp(0, new - 1)].transpose(1, 2)                             # (touched, Hk, 32, D)
        before, old_scale = pool[page, :, sub], scales[page, :, sub]
        some_new, some_old = is_new[:, None, :, None], is_old[:, None, :, None]
        scale = _pow2(torch.where(some_new, x, 0.0).abs().amax((-1, -2)))
        scale = torch.where(is_old.any(-1)[:, None], torch.maximum(scale, old_scale), scale)
        y = torch.where(some_new, x / scale[..., None, None], before.view(E4M3).float() * (old_scale / scale)[..., None, None])
        pool[page, :, sub] = torch.where(some_new | some_old, y.to(E4M3).view(torch.uint8), before)
        scales[page, :, sub] = scale

    write(_rotated(s["k"], s, positions), s["k8"], s["ks"])
    write(s["v"].float(), s["v8"], s["vs"])
    return {"q": q, "lengths": s["before"] + s["new"], "k8": s["k8"], "v8": s["v8"], "ks": s["ks"], "vs": s["vs"]}


def _plain_keep(s):
    c = s["case"]
    B, N, Hk, D, P = c["B"], c["new"], c["Hk"], c["D"], c["page"]
    start, count, table = s["before"].long(), s["kept"].long(), s["table"].long()
    blocks = (N + BLK - 2) // BLK + 1
    block = start[:, None] // BLK + torch.arange(blocks, device="cuda")                     # (B, blocks)
    pos = block[..., None] * BLK + torch.arange(BLK, device="cuda")
    i = pos - start[:, None, None]
    moved, old = (i >= 0) & (i < count[:, None, None]), (i < 0)
    touched = moved.any(-1)
    bs = torch.arange(B, device="cuda")[:, None].expand_as(block)[touched]
    moved, old, i, pos = moved[touched], old[touched], i[touched], pos[touched]
    held = moved | old
    source = torch.where(moved, start[bs][:, None] + s["path"].long()[bs[:, None], i.clamp(0, N - 1)], pos)
    source = torch.where(held, source, 0)
    from_page, to, sub = table[bs[:, None], source // P], table[bs, (block // (P // BLK))[touched]], (block % (P // BLK))[touched]

    def move(codes, scales):
        x = codes.view(torch.uint8)[from_page, :, source % P].view(E4M3).float() * scales[from_page, :, source % P // BLK][..., None]        # (touched, 32, Hk, D)
        x = x.transpose(1, 2)
        scale = _pow2(torch.where(held[:, None, :, None], x, 0.0).abs().amax((-1, -2)))
        pool = codes.view(torch.uint8).view(-1, Hk, P // BLK, BLK, D)
        pool[to, :, sub] = torch.where(held[:, None, :, None], (x / scale[..., None, None]).to(E4M3).view(torch.uint8), pool[to, :, sub])
        scales[to, :, sub] = scale

    move(s["k8"], s["ks"])
    move(s["v8"], s["vs"])
    return {"lengths": s["before"] + s["kept"], "k8": s["k8"], "v8": s["v8"], "ks": s["ks"], "vs": s["vs"]}


_PLAIN = {"tree": lambda s: dict(zip(("depth", "seen"), _plain_tree(s["parents"].long(), s["new"]))), "append": _plain_append, "attn": _plain_attn, "keep": _plain_keep}


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


def _exact_tree(s):
    parents, (B, N) = s["parents"].cpu(), s["parents"].shape
    depth, seen = torch.zeros(B, N, dtype=torch.int32), torch.zeros(B, N, -(-N // 32), dtype=torch.int64)
    for b, count in enumerate(s["new"].tolist()):
        of = parents[b].tolist()
        for i in range(count):
            if of[i] >= 0:
                depth[b, i] = depth[b, of[i]] + 1
                seen[b, i] = seen[b, of[i]]
            seen[b, i, i // 32] += 1 << (i % 32)
    return {"depth": depth.cuda(), "seen": torch.where(seen >= 2 ** 31, seen - 2 ** 32, seen).to("cuda", torch.int32)}


def _rows64(s, b, n, codes, scales):
    """The first n tokens of sequence b: (Hk, n, D) fp64."""
    P = s["case"]["page"]
    at = torch.arange(n, device="cuda")
    page = s["table"][b].long()[at // P]
    return (codes[page, :, at % P].double() * scales[page, :, at % P // BLK].double()[..., None]).transpose(0, 1)


def _exact_attn(s):
    c = s["case"]
    H, Hk, D, N = c["H"], c["Hk"], c["D"], c["new"]
    o, lse = torch.zeros(s["q"].shape, device="cuda", dtype=torch.float64), torch.full((c["B"], H, N), -math.inf, device="cuda", dtype=torch.float64)
    k8, v8 = s["k8"].float(), s["v8"].float()
    for b, (n, count) in enumerate(zip(s["lengths"].tolist(), s["new"].tolist())):
        k, v = _rows64(s, b, n, k8, s["ks"]), _rows64(s, b, n, v8, s["vs"])
        hidden = torch.zeros(count, n, device="cuda", dtype=torch.bool)
        hidden[:, n - count:] = ~_seen_nodes(s["seen"][b:b + 1, :count], N)[0, :, :count]
        for h in range(H):
            x = (s["q"][b, :count, h].double() @ k[h * Hk // H].T / math.sqrt(D)).masked_fill(hidden, -math.inf)
            lse[b, h, :count] = torch.logsumexp(x, -1)
            o[b, :count, h] = torch.softmax(x, -1) @ v[h * Hk // H]
    return {"o": o, "lse": lse}


def _exact_append(s):
    c = s["case"]
    P, half = c["page"], c["rotary"] // 2
    first = torch.arange(half, device="cuda") * (2 if c["interleaved"] else 1)
    second = first + (1 if c["interleaved"] else half)
    k8, v8, ks, vs = (s[name].double() for name in ("k8", "v8", "ks", "vs"))
    q = torch.zeros(s["q"].shape, device="cuda", dtype=torch.float64)

    def turned(x, positions):                                    # (tokens, heads, D) as complex numbers times exp(i angle)
        x = x.double()
        z = torch.complex(x[..., first], x[..., second]) * torch.polar(torch.ones((), device="cuda", dtype=torch.float64), positions[:, None, None].double() * s["freqs"].double())
        x[..., first], x[..., second] = z.real, z.imag
        return x

    for b, (n, count) in enumerate(zip(s["before"].tolist(), s["new"].tolist())):
        at = torch.arange(count, device="cuda")
        positions = n + (at if s["offsets"] is None else s["offsets"][b, :count])
        q[b, :count] = turned(s["q"][b, :count], positions)
        for x, codes, scales in ((turned(s["k"][b, :count], positions), k8, ks), (s["v"][b, :count].double(), v8, vs)):
            i = 0
            while i < count:
                slot, take = (n + i) % P, min(BLK - (n + i) % BLK, count - i)
                page, blk, begin = int(s["table"][b, (n + i) // P]), slot // BLK, slot - slot % BLK
                y = x[i:i + take].transpose(0, 1)
                scale = _scale64(y.abs().amax((1, 2)))
                if slot % BLK:
                    scale = torch.maximum(scale, scales[page, :, blk])
                    codes[page, :, begin:slot] = _e4m3_grid(codes[page, :, begin:slot] * (scales[page, :, blk] / scale)[:, None, None])
                codes[page, :, slot:slot + take], scales[page, :, blk] = _e4m3_grid(y / scale[:, None, None]), scale
                i += take
    return {"q": q, "lengths": s["before"] + s["new"], "k8": k8, "v8": v8, "ks": ks, "vs": vs}


def _exact_keep(s):
    c = s["case"]
    P, out = c["page"], {"lengths": s["before"] + s["kept"]}
    for name in "kv":
        codes, scales = s[name + "8"].double(), s[name + "s"].double()
        for b, (n, count) in enumerate(zip(s["before"].tolist(), s["kept"].tolist())):
            if count == 0:
                continue
            begin, end = n - n % BLK, n + count
            source = torch.cat([torch.arange(begin, n, device="cuda"), n + s["path"][b, :count].long()])
            page = s["table"][b].long()[source // P]
            x = (codes[page, :, source % P] * scales[page, :, source % P // BLK][..., None]).transpose(0, 1)         # (Hk, tokens, D)
            for at in range(begin, end, BLK):
                y = x[:, at - begin:min(at + BLK, end) - begin]
                page, blk = int(s["table"][b, at // P]), at % P // BLK
                scale = _scale64(y.abs().amax((1, 2)))
                codes[page, :, at % P:at % P + y.shape[1]], scales[page, :, blk] = _e4m3_grid(y / scale[:, None, None]), scale
        out.update({name + "8": codes, name + "s": scales})
    return {"lengths": out["lengths"], "k8": out["k8"], "v8": out["v8"], "ks": out["ks"], "vs": out["vs"]}


def exact(case, seed):
    return {"tree": _exact_tree, "append": _exact_append, "attn": _exact_attn, "keep": _exact_keep}[case["op"]](prepare(case, seed))
