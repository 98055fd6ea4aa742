"""Answering with a grouped-query attention layer over the 8-bit key/value cache: prompts in, tokens out one at a time, the cache cut to the tokens
that matter whenever a sequence has outgrown it.

    python examples/decode_with_cache.py [--steps 200] [--limit 160] [--budget 96]

The layer is a toy (random projections, its output is the next input); what is real is how the operators are used together: pages handed out from
a free list, one append and one attention call a step for the whole batch, attention weights kept per token and head, eviction into fresh
pages.  Everything the kernels need stays on the device; the host only counts tokens."""
from __future__ import annotations

import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from delta_matching_b200 import KVCache8, dm_cache_append, dm_cache_attn, dm_cache_evict, ops  # noqa: E402


class Pages:
    """The cache's pages and who has them.  Tables are (sequences, `width`) int32; entries a sequence has no page for are 0 and never read."""

    def __init__(self, count, page_size, nheads_k, head_dim):
        self.cache = KVCache8.empty(count, page_size, nheads_k, head_dim)
        self.page_size, self.free = page_size, list(range(count))[::-1]

    def take(self, tokens):
        return [self.free.pop() for _ in range(-(-tokens // self.page_size))]

    def give_back(self, pages):
        self.free.extend(pages)

    def table(self, owned, width):
        return torch.tensor([p + [0] * (width - len(p)) for p in owned], dtype=torch.int32).cuda()


class Layer:
    """Projections of a grouped-query attention layer, bf16."""

    def __init__(self, dim, nheads, nheads_k, head_dim, seed=0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        w = lambda *s: (torch.randn(*s, generator=g, device="cuda") * s[0] ** -0.5).to(torch.bfloat16)
        self.h, self.hk, self.d = nheads, nheads_k, head_dim
        self.w_in, self.w_out = w(dim, (nheads + 2 * nheads_k) * head_dim), w(nheads * head_dim, dim)

    def qkv(self, x):
        """x (B, N, dim) -> q (B, N, H, D), k, v (B, N, Hk, D): slices of one tensor, which the operators read in place."""
        packed = (x @ self.w_in).view(*x.shape[:2], self.h + 2 * self.hk, self.d)
        return packed.split([self.h, self.hk, self.hk], dim=2)

    def out(self, o):
        y = o.flatten(2) @ self.w_out
        return y * torch.rsqrt(y.float().square().mean(-1, keepdim=True) + 1e-6).to(y.dtype)


def generate(layer, prompts, steps, limit, budget, recent, page_size=32, record=None):
    """prompts: (n_b, dim) bf16 tensors.  -> the generated inputs (B, steps, dim), tokens held at the end, evictions.  `limit`: tokens at which the
    sequences are cut to `budget`.  record(k, v, q, o, lengths) is called after every attention call."""
    B, dim = len(prompts), prompts[0].shape[1]
    width = -(-(max(limit, max(p.shape[0] for p in prompts)) + 1) // page_size)
    pages = Pages(2 * B * width, page_size, layer.hk, layer.d)
    counts = [p.shape[0] for p in prompts]
    owned = [pages.take(width * page_size) for _ in range(B)]
    table, lengths = pages.table(owned, width), torch.zeros(B, dtype=torch.int32, device="cuda")
    weights = torch.zeros(B, layer.hk, width * page_size, device="cuda")

    # the prompts, all of them in one call each: shorter ones are padded, and the counts say by how much
    x = torch.nn.utils.rnn.pad_sequence(prompts, batch_first=True)
    new = torch.tensor(counts, dtype=torch.int32, device="cuda")
    q, k, v = layer.qkv(x)
    lengths = dm_cache_append(pages.cache, k, v, table, lengths, counts=new)
    o = dm_cache_attn(q, pages.cache, table, lengths, q_counts=new, weights=weights)
    if record:
        record(k, v, q, o, counts)
    x = layer.out(o)[torch.arange(B), new.long() - 1][:, None]

    held, made, evictions = list(counts), [], 0
    for _ in range(steps):
        if max(held) >= limit:
            fresh = [pages.take(width * page_size) for _ in range(B)]
            new_table = pages.table(fresh, width)
            lengths, _, weights = dm_cache_evict(pages.cache, table, lengths, weights, new_table, budget, recent=recent)
            for p in owned:
                pages.give_back(p)
            owned, table, held, evictions = fresh, new_table, [min(n, budget) for n in held], evictions + 1
        made.append(x)
        q, k, v = layer.qkv(x)
        lengths = dm_cache_append(pages.cache, k, v, table, lengths)
        o = dm_cache_attn(q, pages.cache, table, lengths, weights=weights, accumulate=True)
        held = [n + 1 for n in held]
        if record:
            record(k, v, q, o, held)
        x = layer.out(o)
    ops.check_status()
    assert lengths.tolist() == held
    return torch.cat(made, 1), held, evictions


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--steps", type=int, default=200)
    ap.add_argument("--limit", type=int, default=160)
    ap.add_argument("--budget", type=int, default=96)
    a = ap.parse_args()
    layer = Layer(512, 8, 2, 128)
    g = torch.Generator(device="cuda").manual_seed(1)
    prompts = [torch.randn(n, 512, generator=g, device="cuda").to(torch.bfloat16) for n in (3, 57, 120, 31)]
    begin, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    begin.record()
    made, held, evictions = generate(layer, prompts, a.steps, a.limit, a.budget, a.budget // 4)
    end.record()
    torch.cuda.synchronize()
    print(f"{made.shape[0]} sequences, {a.steps} tokens each, {evictions} evictions, tokens held at the end {held}, "
          f"{begin.elapsed_time(end) / a.steps:.3f} ms a step")


if __name__ == "__main__":
    main()
