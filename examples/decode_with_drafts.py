"""Speculative decoding over the 8-bit key/value cache: a tree of drafted tokens a step, one pass of the model over all of them, one path kept.

    python examples/decode_with_drafts.py [--tokens 400] [--depth 6]

The model is a toy (random weights, greedy answers), and so is what drafts: each sequence's own last two successors of a token, the first in a chain, the second beside
it.  What is real is how the operators are used together: prompts and drafts appended with their positions' rotation, attention of the tree, the path that
agrees with the model moved together in every layer's cache.  A step is device work alone, captured once in a CUDA graph; the host only reads how many tokens came out."""
from __future__ import annotations

import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from delta_matching_b200 import KVCache8, dm_cache_append_rotary, dm_cache_attn, dm_cache_attn_tree, dm_cache_keep, dm_draft_tree, ops  # noqa: E402


class Model:
    """Grouped-query attention layers with residuals over an embedding that is also the output's, bf16."""

    def __init__(self, vocab=512, dim=256, layers=2, nheads=8, nheads_k=2, head_dim=128, seed=0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        w = lambda *s: (torch.randn(*s, generator=g, device="cuda") * s[0] ** -0.5).to(torch.bfloat16)
        self.h, self.hk, self.d = nheads, nheads_k, head_dim
        self.embedding = w(dim, vocab).T.contiguous()
        self.layers = [(w(dim, (nheads + 2 * nheads_k) * head_dim), w(nheads * head_dim, dim)) for _ in range(layers)]
        self.freqs = (10000.0 ** (-torch.arange(head_dim // 2, device="cuda").double() / (head_dim // 2))).float()

    def __call__(self, tokens, caches, table, lengths, attend, offsets=None, counts=None, record=None):
        """tokens (B, N) -> the answers (B, N) and the new lengths; attend(q, cache, lengths) is the attention that the tokens take."""
        x = self.embedding[tokens] * 16.0
        now = lengths
        for (w_in, w_out), cache in zip(self.layers, caches):
            norm = x * torch.rsqrt(x.float().square().mean(-1, keepdim=True) + 1e-6).to(x.dtype)
            q, k, v = (norm @ w_in).view(*x.shape[:2], self.h + 2 * self.hk, self.d).split([self.h, self.hk, self.hk], dim=2)
            turned, now = dm_cache_append_rotary(cache, q, k, v, table, lengths, self.freqs, offsets=offsets, counts=counts)
            o = attend(turned, cache, now)
            if record and cache is caches[0]:
                record(q, k, v, o)
            x = x + o.flatten(2) @ w_out
        return (x.float() @ self.embedding.float().T).argmax(-1), now


class Decoder:
    """A batch of sequences: the model's caches, the tokens held, and what drafts the next ones."""

    def __init__(self, model, prompts, room, depth, page_size=64):
        B, dev = len(prompts), "cuda"
        self.model, self.depth = model, depth
        width = -(-(max(map(len, prompts)) + room + 2 * depth + 1) // page_size)
        self.caches = [KVCache8.empty(B * width, page_size, model.hk, model.d) for _ in model.layers]
        self.table = torch.randperm(B * width).to(torch.int32).view(B, width).cuda()
        # node 0 is the last answer; 2 d - 1 and 2 d are the guesses at depth d, both behind the first guess before them
        parents = [-1] + [max(0, 2 * (d - 1) - 1) for d in range(1, depth + 1) for _ in (0, 1)]
        self.tree = dm_draft_tree(torch.tensor([parents] * B, dtype=torch.int32, device=dev))
        self.rows = torch.arange(B, device=dev)
        counts = torch.tensor([len(p) for p in prompts], dtype=torch.int32, device=dev)
        tokens = torch.nn.utils.rnn.pad_sequence([torch.as_tensor(p) for p in prompts], batch_first=True).cuda()
        answers, self.lengths = model(tokens, self.caches, self.table, torch.zeros(B, dtype=torch.int32, device=dev),
                                      lambda q, cache, n: dm_cache_attn(q, cache, self.table, n, q_counts=counts), counts=counts)
        self.last = answers[self.rows, counts.long() - 1]
        self.next_ones = torch.zeros(B, model.embedding.shape[0], 2, dtype=torch.long, device=dev)      # a token's last two successors

    def draft(self):
        tokens = [self.last]
        at = self.last
        for _ in range(self.depth):
            guesses = self.next_ones[self.rows, at]
            tokens += [guesses[:, 0], guesses[:, 1]]
            at = guesses[:, 0]
        return torch.stack(tokens, 1)

    def step(self, record=None):
        """-> the tokens that came out (B, depth + 1), of which the first counts[b] count, and counts.  Updates the decoder's tensors in place."""
        tokens = self.draft()
        answers, now = self.model(tokens, self.caches, self.table, self.lengths, lambda q, cache, n: dm_cache_attn_tree(q, cache, self.table, n, self.tree),
                                  offsets=self.tree.depth, record=record)
        # down the tree, as long as a guess is what the model answers
        at, going = torch.zeros_like(self.rows), torch.ones_like(self.rows, dtype=torch.bool)
        path, counts = [at], torch.ones_like(self.lengths)
        for d in range(1, self.depth + 1):
            want = answers[self.rows, at]
            first = going & (tokens[:, 2 * d - 1] == want)
            second = going & ~first & (tokens[:, 2 * d] == want)
            path.append(torch.where(first, 2 * d - 1, 2 * d))
            counts += first | second
            at = torch.where(first | second, path[-1], at)
            going = first
        path = torch.stack(path, 1)
        for cache in self.caches:
            lengths = dm_cache_keep(cache, self.table, self.lengths, now, path.to(torch.int32), counts)
        out = answers.gather(1, path)
        for d in range(self.depth + 1):                       # what came behind what
            token, got = tokens[self.rows, path[:, d]], out[:, d]
            old = self.next_ones[self.rows, token]
            new = torch.stack([got, torch.where(old[:, 0] == got, old[:, 1], old[:, 0])], 1)
            self.next_ones[self.rows, token] = torch.where((d < counts)[:, None], new, old)
        self.last.copy_(answers[self.rows, at])
        self.lengths.copy_(lengths)
        return out, counts


def generate(model, prompts, tokens, depth, graph=True, record=None):
    """At least `tokens` tokens behind each prompt -> their lists, and the number of passes of the model."""
    # (a sequence may be done before another: each goes on until all are)
    decoder = Decoder(model, prompts, (tokens + depth + 1) * (depth + 1), depth)
    made, passes = [[t] for t in decoder.last.tolist()], 0
    step = lambda: decoder.step(record)
    while min(map(len, made)) < tokens:
        out, counts = step()
        passes += 1
        for sequence, row, n in zip(made, out.tolist(), counts.tolist()):
            sequence += row[:n]
        if graph and passes == 2:
            captured = torch.cuda.CUDAGraph()
            with torch.cuda.graph(captured):
                held = decoder.step()
            step = lambda: captured.replay() or held
    ops.check_status()
    assert [len(p) + len(m) - 1 for p, m in zip(prompts, made)] == decoder.lengths.tolist()
    return made, passes


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--tokens", type=int, default=400)
    ap.add_argument("--depth", type=int, default=6)
    a = ap.parse_args()
    model = Model()
    g = torch.Generator().manual_seed(1)
    prompts = [torch.randint(512, (n,), generator=g).tolist() for n in (3, 57, 120, 31)]
    for depth in (0, a.depth):
        generate(model, prompts, 8, depth)
        begin, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        begin.record()
        made, passes = generate(model, prompts, a.tokens, depth)
        end.record()
        torch.cuda.synchronize()
        print(f"{len(prompts)} sequences, drafts of depth {depth}: {sum(map(len, made))} tokens in {passes} passes, {sum(map(len, made)) / passes / len(made):.2f} a pass and sequence, "
              f"{begin.elapsed_time(end) / passes:.3f} ms a pass")


if __name__ == "__main__":
    main()
