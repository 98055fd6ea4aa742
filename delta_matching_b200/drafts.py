"""Drafted tokens over the 8-bit key/value cache: a step of speculative decoding.

A small model drafts a tree of tokens behind each sequence, the large one looks at all of them in one pass, and one path of the tree is kept.

    from delta_matching_b200 import dm_draft_tree, dm_cache_append_rotary, dm_cache_attn_tree, dm_cache_keep
    tree = dm_draft_tree(parents)                                       # parents (B, N) int32: an earlier node, or -1
    q, now = dm_cache_append_rotary(cache, q, k, v, block_table, lengths, freqs, offsets=tree.depth)        # once a layer
    o = dm_cache_attn_tree(q, cache, block_table, now, tree)            # once a layer
    lengths = dm_cache_keep(cache, block_table, lengths, now, path, kept)                                   # once a layer, with the path that won

dm_cache_append_rotary is also what a prompt or a single token takes whose keys carry their position's rotation.  As in cache.py everything is a device
tensor that the host never reads, so that a step is captured in a CUDA graph as it stands; what the kernels find out of range is reported by RuntimeError
from the next call, or from ops.check_status, and nothing outside the buffers is touched.  Input errors raise ValueError / TypeError; no autograd graph is
recorded, a forward-mode tangent raises NotImplementedError.  Under torch.compile, torch.jit.trace and dispatch modes the functions are registered ops
without a graph break.  examples/decode_with_drafts.py runs them together.  The reference package has no counterpart.
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple, Optional

import torch

from . import _lib, ops
from .cache import (_OPS, _c_cache, _check_cache, _check_ints, _check_lengths, _check_rows, _check_table, _check_written, _recorded, _refuse_tangents)

MAX_NODES = 1024


class DraftTree(NamedTuple):
    """What dm_draft_tree makes of a tree's parents: depth (B, N) int32, a node's ancestors; seen (B, N, (N + 31) // 32) int32, bit j % 32 of word j // 32 of
    node i: node i sees node j (itself and its ancestors); counts (B) int32 or None: the nodes of each sequence, None: N each.  A program with a tree that
    does not change may keep one, or make it itself: bits of later nodes are not looked at, and a node sees itself whatever its bit says."""
    depth: torch.Tensor
    seen: torch.Tensor
    counts: Optional[torch.Tensor] = None


def _check_nodes(what, N):
    if not 0 < N <= MAX_NODES:
        raise ValueError(f"delta_matching: {what} must have 1 to {MAX_NODES} drafted tokens (got {N})")


def _row(t):
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def dm_draft_tree(parents, counts=None):
    """parents (B, N) int32 on CUDA, N <= 1024: each drafted token's parent, an earlier one, or -1 for the sequence's last token (several may have that).
    counts (B) int32: sequence b has the first counts[b] of them; the others' depths and bits are 0.  -> DraftTree.  A parent that is no earlier node is
    reported, and -1 in its place."""
    if not torch.compiler.is_compiling():
        out = _lib.native_cache().draft_tree(parents, counts)
        if out is not None:
            return DraftTree(*out, counts)
    if _recorded():
        return DraftTree(*_OPS.draft_tree(parents, counts), counts)
    return DraftTree(*tree_now(parents, counts), counts)


def tree_now(parents, counts):
    """dm_draft_tree by the Python route, whatever records: what the registered op comes to where the native route does not take it."""
    if not isinstance(parents, torch.Tensor) or not parents.is_cuda:
        raise ValueError("delta_matching: parents must be a CUDA tensor")
    dev = parents.device
    parents = _check_ints("parents", parents, (None, None), dev)
    B, N = parents.shape
    if B == 0:
        raise ValueError(f"delta_matching: empty tensor parents {tuple(parents.shape)}")
    _check_nodes("parents", N)
    counts = None if counts is None else _check_lengths("counts", counts, B, dev)
    ops._enter(dev)
    with torch.cuda.device(dev):
        depth = torch.empty(B, N, device=dev, dtype=torch.int32)
        seen = torch.empty(B, N, (N + 31) // 32, device=dev, dtype=torch.int32)
        _lib.check(_lib.lib().dm_draft_tree(parents.data_ptr(), _row(parents), ops._ptr(counts), B, N, depth.data_ptr(), seen.data_ptr(),
                                            ops.status_word(dev).data_ptr(), ops._stream(parents)))
        ops._after(dev)
    return depth, seen


def dm_cache_append_rotary(cache, q, k, v, block_table, lengths, freqs, offsets=None, counts=None, interleaved=False):
    """dm_cache_append of keys that are rotated by position on the way, and the rotated queries: q (B, N, H, D), k, v (B, N, Hk, D) bf16 (any strides).  New
    token i of sequence b stands at position t = lengths[b] + offsets[b, i] (offsets (B, N) int32, a tree's depths; None: i), and channels (j, j + F) of q
    and k, or (2 j, 2 j + 1) where interleaved, turn by the angle t freqs[j]: (x cos - y sin, y cos + x sin).  freqs (F) fp32 on the device, F a multiple of 8,
    at most D / 2: further channels stay as they are.  Angles are reduced in 64 bits, products are fp32; keys are rounded once, to their codes.

    As in dm_cache_append, a block that already holds tokens keeps the larger scale and its older codes are rounded anew when that grows: also for drafted tokens that are rejected later.

    Returns (q rotated (B, N, H, D) bf16, 0 for tokens beyond counts, and the new lengths (B) int32)."""
    if not torch.compiler.is_compiling():
        out = _lib.native_cache().cache_append_rotary(cache, q, k, v, block_table, lengths, freqs, offsets, counts, interleaved)
        if out is not None:
            return out
    if _recorded():
        return _OPS.cache_append_rotary(*cache, q, k, v, block_table, lengths, freqs, offsets, counts, bool(interleaved))
    return append_rotary_now(cache, q, k, v, block_table, lengths, freqs, offsets, counts, interleaved)


def append_rotary_now(cache, q, k, v, block_table, lengths, freqs, offsets, counts, interleaved):
    """dm_cache_append_rotary by the Python route, whatever records."""
    pages, Hk, P, D = _check_cache(cache)
    _check_written(cache)
    _refuse_tangents(q=q, k=k, v=v, freqs=freqs, ks=cache.ks, vs=cache.vs)
    dev = cache.k8.device
    q, k, v = _check_rows("q", q, None, D, dev), _check_rows("k", k, Hk, D, dev), _check_rows("v", v, Hk, D, dev)
    if k.shape != v.shape:
        raise ValueError(f"delta_matching: k and v must have the same shape (got {tuple(k.shape)} and {tuple(v.shape)})")
    B, N, H = q.shape[:3]
    if k.shape[:2] != (B, N):
        raise ValueError(f"delta_matching: q and k must have the same tokens (got {tuple(q.shape)} and {tuple(k.shape)})")
    if H % Hk:
        raise ValueError(f"delta_matching: nheads ({H}) must be a positive multiple of nheads_k ({Hk})")
    if not isinstance(freqs, torch.Tensor) or freqs.dtype != torch.float32:
        raise TypeError("delta_matching: freqs must be a float32 tensor")
    if freqs.dim() != 1 or freqs.shape[0] == 0 or freqs.shape[0] % 8 or 2 * freqs.shape[0] > D:
        raise ValueError(f"delta_matching: freqs must be a multiple of 8 frequencies, for at most the {D} channels of a head (got {tuple(freqs.shape)})")
    if freqs.device != dev:
        raise ValueError(f"delta_matching: freqs must be on {dev} (got {freqs.device})")
    freqs = freqs.contiguous()
    table, row = _check_table("block_table", block_table, B, dev)
    lengths = _check_lengths("lengths", lengths, B, dev)
    offsets = None if offsets is None else _check_ints("offsets", offsets, (B, N), dev)
    counts = None if counts is None else _check_lengths("counts", counts, B, dev)
    ops._enter(dev)
    with torch.cuda.device(dev):
        out = torch.empty(B, N, H, D, device=dev, dtype=torch.bfloat16)
        new = torch.empty(B, device=dev, dtype=torch.int32)
        _lib.check(_lib.lib().dm_cache_append_rotary(
            ctypes.byref(_c_cache(cache, pages, Hk, P, D)), q.data_ptr(), q.stride(0), q.stride(1), q.stride(2), k.data_ptr(), k.stride(0), k.stride(1),
            k.stride(2), v.data_ptr(), v.stride(0), v.stride(1), v.stride(2), B, N, H, freqs.data_ptr(), freqs.shape[0], int(bool(interleaved)),
            table.data_ptr(), row, table.shape[1], lengths.data_ptr(), ops._ptr(offsets), 0 if offsets is None else _row(offsets), ops._ptr(counts),
            out.data_ptr(), new.data_ptr(), ops.status_word(dev).data_ptr(), ops._stream(q)))
        ops._after(dev)
    return out, new


def _check_tree(tree):
    if not isinstance(tree, DraftTree) or not all(isinstance(t, torch.Tensor) for t in tree[:2]):
        raise TypeError("delta_matching: tree must be a DraftTree of torch tensors")
    return tree.seen, tree.counts


def dm_cache_attn_tree(q, cache, block_table, lengths, tree, softmax_scale=None, return_lse=False):
    """Attention of a tree of drafted tokens over what the cache holds: q (B, N, H, D) bf16 (any strides; H a multiple of the cache's heads) -> o (B, N, H, D)
    bf16.  The N drafted tokens of a sequence (tree.counts[b] of them) are the last of the lengths[b] that it holds: append first.  Each sees all tokens
    before the drafted ones, its ancestors and itself (tree.seen).  Rows beyond the counts are 0, their LSE -inf.  return_lse=True also returns the LSE
    (B, H, N) fp32, natural log.

    q keeps its 8 bits down to 2^-13 of the row's largest element, smaller ones are off by 2^-21 of that; sums and statistics are fp32.  In the second product a probability is off by 2^-9 of itself
    (dm_cache_attn: 2^-11) and by 2^-16 of the largest one of its block of 32 keys.  Rows with logits beyond 2^22, or whose later logits are above the
    first 32 to 64 keys' by 90 (by 38 where these have values of zero), are served one key after the other, about 0.6 us each."""
    if not torch.compiler.is_compiling():
        out = _lib.native_cache().cache_attn_tree(q, cache, block_table, lengths, tree, softmax_scale, return_lse)
        if out is not None:
            return out
    if _recorded():
        seen, counts = _check_tree(tree)
        o, lse = _OPS.cache_attn_tree(q, *cache, block_table, lengths, seen, counts, softmax_scale)
        return (o, lse) if return_lse else o
    return attn_tree_now(q, cache, block_table, lengths, tree, softmax_scale, return_lse)


def attn_tree_now(q, cache, block_table, lengths, tree, softmax_scale, return_lse):
    """dm_cache_attn_tree by the Python route, whatever records."""
    pages, Hk, P, D = _check_cache(cache)
    _refuse_tangents(q=q, ks=cache.ks, vs=cache.vs)
    dev = cache.k8.device
    q = _check_rows("q", q, None, D, dev)
    B, N, H = q.shape[:3]
    if H % Hk:
        raise ValueError(f"delta_matching: nheads ({H}) must be a positive multiple of nheads_k ({Hk})")
    _check_nodes("q", N)
    seen, counts = _check_tree(tree)
    seen = _check_ints("tree.seen", seen, (B, N, (N + 31) // 32), dev)
    counts = None if counts is None else _check_lengths("tree.counts", counts, B, dev)
    table, row = _check_table("block_table", block_table, B, dev)
    T = table.shape[1]
    lengths = _check_lengths("lengths", lengths, B, dev)
    scale = D ** -0.5 if softmax_scale is None else float(softmax_scale)
    if not 0.0 < ctypes.c_float(scale).value < float("inf"):
        raise ValueError(f"delta_matching: softmax_scale must be positive and finite in 32 bits (got {softmax_scale!r})")
    ops._enter(dev)
    L = _lib.lib()
    with torch.cuda.device(dev):
        o = torch.empty(B, N, H, D, device=dev, dtype=torch.bfloat16)
        lse = torch.empty(B, H, N, device=dev, dtype=torch.float32)
        bytes_ = L.dm_cache_attn_tree_workspace_bytes(B, N, H, Hk, D, T, P)
        if bytes_ == 0:
            raise ValueError(_lib.last_error())
        ws = torch.empty(bytes_, device=dev, dtype=torch.uint8)
        _lib.check(L.dm_cache_attn_tree(
            ctypes.byref(_c_cache(cache, pages, Hk, P, D)), q.data_ptr(), q.stride(0), q.stride(1), q.stride(2), B, N, H, table.data_ptr(), row, T,
            lengths.data_ptr(), ops._ptr(counts), seen.data_ptr(), seen.stride(0), seen.stride(1), scale, o.data_ptr(), lse.data_ptr(), ws.data_ptr(), bytes_,
            ops.status_word(dev).data_ptr(), ops._stream(q)))
        ops._after(dev)
    return (o, lse) if return_lse else o


def dm_cache_keep(cache, block_table, before, lengths, path, counts):
    """Keep one path of the drafted tokens: those that `lengths` (B) int32 counts and `before` (B) int32 does not.  path (B, M) int32, M <= 1024: indexes of
    drafted tokens, strictly increasing, of which the first counts[b] (int32) are kept; they become the tokens before[b], before[b] + 1, ...  Returns the new
    lengths before + counts.  The tokens move within the sequences' own pages; each block of 32 slots that is written gets the smallest power-of-two scale
    that holds its tokens (codes whose block's scale stays are not changed).  Where a rejected token had made the scale of a block of older tokens grow, it falls again, but what
    that rounded away of them (elements below 2^-14 of the block's largest) does not come back.  A path that does not increase, or leaves the drafted tokens, is reported; nothing of its sequence
    moves, and its new length is before[b]."""
    if not torch.compiler.is_compiling():
        new = _lib.native_cache().cache_keep(cache, block_table, before, lengths, path, counts)
        if new is not None:
            return new
    if _recorded():
        return _OPS.cache_keep(*cache, block_table, before, lengths, path, counts)
    return keep_now(cache, block_table, before, lengths, path, counts)


def keep_now(cache, block_table, before, lengths, path, counts):
    """dm_cache_keep by the Python route, whatever records."""
    pages, Hk, P, D = _check_cache(cache)
    _check_written(cache)
    _refuse_tangents(ks=cache.ks, vs=cache.vs)
    dev = cache.k8.device
    path = _check_ints("path", path, (None, None), dev)
    B, M = path.shape
    if B == 0:
        raise ValueError(f"delta_matching: empty tensor path {tuple(path.shape)}")
    _check_nodes("path", M)
    table, row = _check_table("block_table", block_table, B, dev)
    before, lengths, counts = (_check_lengths(name, t, B, dev) for name, t in (("before", before), ("lengths", lengths), ("counts", counts)))
    ops._enter(dev)
    with torch.cuda.device(dev):
        new = torch.empty(B, device=dev, dtype=torch.int32)
        _lib.check(_lib.lib().dm_cache_keep(
            ctypes.byref(_c_cache(cache, pages, Hk, P, D)), B, table.data_ptr(), row, table.shape[1], before.data_ptr(), lengths.data_ptr(),
            path.data_ptr(), _row(path), M, counts.data_ptr(), new.data_ptr(), ops.status_word(dev).data_ptr(), ops._stream(path)))
        ops._after(dev)
    return new
