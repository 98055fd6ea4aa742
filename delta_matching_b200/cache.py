"""The 8-bit key/value cache: writing it, attending to it, bounding it.

A cache is pools of pages, shared by all sequences, and what is held has the form of the training kernels' operands: e4m3 codes with one
power-of-two scale per 32 tokens and kv head.

    from delta_matching_b200 import KVCache8, dm_cache_append, dm_cache_attn, dm_cache_evict
    cache = KVCache8.empty(pages=512, page_size=64, nheads_k=8, head_dim=128, device="cuda")
    lengths = dm_cache_append(cache, k, v, block_table, lengths)       # k, v (B, N, Hk, D) bf16: N new tokens a sequence
    o = dm_cache_attn(q, cache, block_table, lengths)                  # q (B, N, H, D) bf16: their queries
    o = dm_cache_attn(q, cache, block_table, lengths, weights=w, accumulate=True)
    lengths, kept, w = dm_cache_evict(cache, block_table, lengths, w, new_block_table, budget=2048, recent=256)

`block_table` (B, T) int32 names each sequence's pages: its token j is slot j % page_size of page block_table[b, j // page_size]; `lengths` (B)
int32 is what each sequence holds.  Both are device tensors and are never copied to the host: every call can be captured in a CUDA graph and
replayed with other lengths.  An entry or length out of range is therefore reported like a kernel that gave up (RuntimeError from the next
call, or from ops.check_status), and nothing outside the buffers is touched.

Input errors raise ValueError / TypeError.  These are serving operators: no autograd graph is recorded, a forward-mode tangent raises
NotImplementedError.  Under torch.compile, torch.jit.trace and dispatch modes they are registered ops without a graph break.  examples/decode_with_cache.py runs the three together.  The reference package has no counterpart.
"""
from __future__ import annotations

import ctypes
import operator
from typing import NamedTuple

import torch

from . import _lib, ops
from . import torch_ops as _torch_ops  # noqa: F401  (registers torch.ops.delta_matching_b200.*)

E4M3 = torch.float8_e4m3fn
_OPS = torch.ops.delta_matching_b200


def _recorded():
    """Whether something outside records this call or takes its place: a compiler, torch.jit.trace, a dispatch mode (make_fx, fake tensors).  It sees
    the registered ops and not what the functions below do through ctypes."""
    return torch.compiler.is_compiling() or torch.jit.is_tracing() or torch._C._len_torch_dispatch_stack() > 0


def _refuse_tangents(**tensors):
    for name, t in tensors.items():
        if isinstance(t, torch.Tensor) and t.is_floating_point() and torch.autograd.forward_ad.unpack_dual(t).tangent is not None:
            raise NotImplementedError(f"delta_matching: {name} carries a forward-mode tangent; the cache functions have no derivatives")


class _CCache(ctypes.Structure):
    """dm_kv_cache of include/dm_b200.h."""
    _fields_ = [("k8", ctypes.c_void_p), ("v8", ctypes.c_void_p), ("ks", ctypes.c_void_p), ("vs", ctypes.c_void_p),
                ("code_page", ctypes.c_int64), ("code_head", ctypes.c_int64), ("code_slot", ctypes.c_int64),
                ("scale_page", ctypes.c_int64), ("scale_head", ctypes.c_int64),
                ("pages", ctypes.c_int), ("heads", ctypes.c_int), ("page_size", ctypes.c_int), ("head_dim", ctypes.c_int)]


class KVCache8(NamedTuple):
    """Pools of pages: k8, v8 (pages, Hk, page_size, D) float8_e4m3fn, ks, vs (pages, Hk, page_size // 32) fp32 powers of two; a value is its
    code times the scale of its block of 32 slots.  Any strides with adjacent elements of a slot (multiples of 16 otherwise) and adjacent
    scales of a head, the same for K and V: also views of one tensor, or (pages, page_size, Hk, D) storage transposed."""
    k8: torch.Tensor
    v8: torch.Tensor
    ks: torch.Tensor
    vs: torch.Tensor

    @classmethod
    def empty(cls, pages: int, page_size: int, nheads_k: int, head_dim: int, device="cuda") -> "KVCache8":
        """Pools of uninitialised codes and scales (what has not been appended is never used)."""
        if page_size <= 0 or page_size % ops.BLK:
            raise ValueError(f"delta_matching: page_size must be a positive multiple of {ops.BLK} (got {page_size})")
        code = lambda: torch.empty(pages, nheads_k, page_size, head_dim, device=device, dtype=E4M3)
        scale = lambda: torch.empty(pages, nheads_k, page_size // ops.BLK, device=device, dtype=torch.float32)
        return cls(code(), code(), scale(), scale())


def _overlaps(t):
    """Whether two elements of t may share an address: a dimension's stride is below what the dimensions of smaller strides span."""
    reach = 1
    for stride, n in sorted(zip(t.stride(), t.shape)):
        if n > 1:
            if stride < reach:
                return True
            reach += (n - 1) * stride
    return False


def _check_written(cache):
    if _overlaps(cache.k8) or _overlaps(cache.ks):
        raise ValueError("delta_matching: slots or scales of the cache share memory (an expanded tensor?): they cannot be written")


def _check_cache(cache):
    if not isinstance(cache, KVCache8) or not all(isinstance(t, torch.Tensor) for t in cache):
        raise TypeError("delta_matching: cache must be a KVCache8 of torch tensors")
    k8, v8, ks, vs = cache
    if k8.dim() != 4 or ks.dim() != 3:
        raise ValueError(f"delta_matching: k8 / v8 must be 4-D (pages, nheads_k, page_size, head_dim) and ks / vs 3-D (got {k8.dim()}-D, {ks.dim()}-D)")
    if not all(t.is_cuda for t in cache):
        raise ValueError("delta_matching: the cache must be CUDA tensors")
    if k8.dtype != E4M3 or v8.dtype != E4M3 or ks.dtype != torch.float32 or vs.dtype != torch.float32:
        raise TypeError(f"delta_matching: k8 / v8 must be float8_e4m3fn and ks / vs float32 (got {k8.dtype}, {v8.dtype}, {ks.dtype}, {vs.dtype})")
    pages, Hk, P, D = k8.shape
    if D not in (128, 256):
        raise ValueError(f"delta_matching: head_dim must be 128 or 256 (got {D})")
    if P == 0 or P % ops.BLK:
        raise ValueError(f"delta_matching: page_size must be a positive multiple of {ops.BLK} (got {P})")
    if pages == 0 or Hk == 0:
        raise ValueError(f"delta_matching: empty cache {tuple(k8.shape)}")
    if v8.shape != k8.shape or ks.shape != (pages, Hk, P // ops.BLK) or vs.shape != ks.shape:
        raise ValueError("delta_matching: k8 and v8 must have one shape and ks, vs (pages, nheads_k, page_size // 32) "
                         f"(got {tuple(k8.shape)}, {tuple(v8.shape)}, {tuple(ks.shape)}, {tuple(vs.shape)})")
    if k8.stride() != v8.stride() or ks.stride() != vs.stride():
        raise ValueError("delta_matching: k8 and v8, and ks and vs, must have equal strides")
    if k8.stride(3) != 1 or any(s % 16 for s in k8.stride()[:3]) or k8.data_ptr() % 16 or v8.data_ptr() % 16:
        raise ValueError("delta_matching: the codes of a slot must be adjacent and start at multiples of 16 bytes")
    if P // ops.BLK > 1 and ks.stride(2) != 1:
        raise ValueError("delta_matching: the scales of a head must be adjacent")
    if len({t.device for t in cache}) != 1:
        raise ValueError("delta_matching: the cache must be on one device")
    return pages, Hk, P, D


def _c_cache(cache, pages, Hk, P, D):
    k8, v8, ks, vs = cache
    # a dimension of size one may carry any stride: give it one that a tensor map takes
    s = [st if n > 1 else 16 for st, n in zip(k8.stride(), k8.shape)]
    return _CCache(k8.data_ptr(), v8.data_ptr(), ks.data_ptr(), vs.data_ptr(), s[0], s[1], s[2], ks.stride(0), ks.stride(1), pages, Hk, P, D)


def _check_ints(name, t, shape, device):
    if not isinstance(t, torch.Tensor) or t.dtype != torch.int32:
        raise TypeError(f"delta_matching: {name} must be an int32 tensor")
    if t.dim() != len(shape) or any(want not in (None, have) for want, have in zip(shape, t.shape)):
        raise ValueError(f"delta_matching: {name} must have shape {tuple('any' if s is None else s for s in shape)} (got {tuple(t.shape)})")
    if t.device != device:
        raise ValueError(f"delta_matching: {name} must be on {device} (got {t.device})")
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _check_table(name, t, B, device):
    t = _check_ints(name, t, (B, None), device)
    if t.shape[1] == 0:
        raise ValueError(f"delta_matching: {name} has no pages")
    return t, t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _check_lengths(name, t, B, device):
    return _check_ints(name, t, (B,), device).contiguous()


def _check_rows(name, t, heads, D, device):
    """A (B, N, heads, D) bf16 tensor as the kernels read it (copied where its rows are not 16-byte aligned)."""
    if not isinstance(t, torch.Tensor) or t.dim() != 4:
        raise ValueError(f"delta_matching: {name} must be a 4-D tensor (batch, seqlen, nheads, headdim)")
    if t.dtype != torch.bfloat16:
        raise TypeError(f"delta_matching: {name} must be torch.bfloat16 (got {t.dtype})")
    if t.device != device:
        raise ValueError(f"delta_matching: {name} must be on the cache's device {device} (got {t.device})")
    if t.numel() == 0:
        raise ValueError(f"delta_matching: empty tensor {name} {tuple(t.shape)}")
    if (heads is not None and t.shape[2] != heads) or t.shape[3] != D:
        raise ValueError(f"delta_matching: {name} must match the cache's heads and head_dim ({heads}, {D}) (got {tuple(t.shape)})")
    return ops._rows(t)


def _check_weights(t, B, Hk, room, device):
    if not isinstance(t, torch.Tensor) or t.dtype != torch.float32:
        raise TypeError("delta_matching: weights must be a float32 tensor")
    if t.dim() != 3 or t.shape[0] != B or t.shape[1] != Hk or t.shape[2] < room:
        raise ValueError(f"delta_matching: weights must be ({B}, {Hk}, at least {room}) for this block table (got {tuple(t.shape)})")
    if t.device != device:
        raise ValueError(f"delta_matching: weights must be on {device} (got {t.device})")
    if t.stride(2) != 1 and t.shape[2] > 1:
        raise ValueError("delta_matching: the weights of a head must be adjacent")


def dm_cache_append(cache, k, v, block_table, lengths, counts=None):
    """Write new tokens into the cache: k, v (B, N, Hk, D) bf16 (any strides) go to positions lengths[b], lengths[b] + 1, ... of each sequence,
    the first counts[b] of them where counts (B) int32 is given.  Returns the new lengths (B) int32; `lengths` itself stays as it is, so the
    same call again leaves the same cache.

    Each block of 32 slots and head gets the smallest power-of-two scale that holds its new values; a block that already holds tokens keeps
    the larger of the two scales, and its codes are rounded anew when that grows.  A page that is written belongs to one sequence: shared
    prefixes end at a page's edge."""
    if not torch.compiler.is_compiling():
        new = _lib.native_cache().cache_append(cache, k, v, block_table, lengths, counts)
        if new is not None:
            return new
    if _recorded():
        return _OPS.cache_append(*cache, k, v, block_table, lengths, counts)
    return append_now(cache, k, v, block_table, lengths, counts)


def append_now(cache, k, v, block_table, lengths, counts):
    """dm_cache_append by the Python route, whatever records: what the registered op comes to where the native route does not take it."""
    pages, Hk, P, D = _check_cache(cache)
    _check_written(cache)
    _refuse_tangents(k=k, v=v, ks=cache.ks, vs=cache.vs)
    dev = cache.k8.device
    k, v = _check_rows("k", k, Hk, D, dev), _check_rows("v", v, Hk, D, dev)
    if k.shape != v.shape:
        raise ValueError(f"delta_matching: k and v must have the same shape (got {tuple(k.shape)} and {tuple(v.shape)})")
    B, N = k.shape[:2]
    table, row = _check_table("block_table", block_table, B, dev)
    lengths = _check_lengths("lengths", lengths, B, dev)
    counts = None if counts is None else _check_lengths("counts", counts, B, dev)
    ops._enter(dev)
    with torch.cuda.device(dev):
        new = torch.empty(B, device=dev, dtype=torch.int32)
        _lib.check(_lib.lib().dm_cache_append(
            ctypes.byref(_c_cache(cache, pages, Hk, P, D)), k.data_ptr(), k.stride(0), k.stride(1), k.stride(2),
            v.data_ptr(), v.stride(0), v.stride(1), v.stride(2), B, N, table.data_ptr(), row, table.shape[1], lengths.data_ptr(),
            ops._ptr(counts), new.data_ptr(), ops.status_word(dev).data_ptr(), ops._stream(k)))
        ops._after(dev)
    return new


def dm_cache_attn(q, cache, block_table, lengths, q_counts=None, causal=True, softmax_scale=None, weights=None, accumulate=False,
                  return_lse=False):
    """Attention of new tokens over what the cache holds: q (B, N, H, D) bf16 (any strides; H a multiple of the cache's heads) -> o (B, N, H, D)
    bf16.  `lengths` counts the new tokens in (append first): with causal=True new token i of sequence b sees the first lengths[b] - N + i + 1
    tokens, otherwise all lengths[b].  q_counts (B) int32: sequence b has only its first q_counts[b] new tokens (they take the place of N
    above; the others' rows are 0).  A row that sees nothing is 0, its LSE -inf.

    weights: an fp32 (B, Hk, W) tensor, W >= T * page_size, that receives for every held token the softmax weight it got, summed over the new
    tokens and over the query heads of its kv head; accumulate=True adds it to what is there.  return_lse=True also returns the LSE (B, H, N)
    fp32, natural log.  The logits and the softmax are those of the codes' exact values: q keeps its 8 bits (elements below 2^-28 of the row's
    largest lose some), sums and statistics are fp32.  In the second product a probability times the scale of its V block keeps 11 bits down to
    2^-25 of the largest such product that the row sees; smaller ones are off by up to 2^-36 of that."""
    if not torch.compiler.is_compiling():
        out = _lib.native_cache().cache_attn(q, cache, block_table, lengths, q_counts, causal, softmax_scale, weights, accumulate, return_lse)
        if out is not None:
            return out
    if _recorded():
        args = (q, *cache, block_table, lengths, q_counts, bool(causal), softmax_scale)
        o, lse = _OPS.cache_attn(*args) if weights is None else _OPS.cache_attn_weights(*args, weights, bool(accumulate))
        return (o, lse) if return_lse else o
    return attn_now(q, cache, block_table, lengths, q_counts, causal, softmax_scale, weights, accumulate, return_lse)


def attn_now(q, cache, block_table, lengths, q_counts, causal, softmax_scale, weights, accumulate, return_lse):
    """dm_cache_attn by the Python route, whatever records: what the registered ops come to where the native route does not take them."""
    pages, Hk, P, D = _check_cache(cache)
    _refuse_tangents(q=q, ks=cache.ks, vs=cache.vs, weights=weights)
    dev = cache.k8.device
    q = _check_rows("q", q, None, D, dev)
    B, N, H = q.shape[:3]
    if H % Hk:
        raise ValueError(f"delta_matching: nheads ({H}) must be a positive multiple of nheads_k ({Hk})")
    table, row = _check_table("block_table", block_table, B, dev)
    T = table.shape[1]
    lengths = _check_lengths("lengths", lengths, B, dev)
    q_counts = None if q_counts is None else _check_lengths("q_counts", q_counts, B, dev)
    scale = D ** -0.5 if softmax_scale is None else float(softmax_scale)
    if not 0.0 < ctypes.c_float(scale).value < float("inf"):
        raise ValueError(f"delta_matching: softmax_scale must be positive and finite in 32 bits (got {softmax_scale!r})")
    if weights is not None:
        _check_weights(weights, B, Hk, T * P, dev)
        if _overlaps(weights):
            raise ValueError("delta_matching: weights share memory (an expanded tensor?): they cannot be written")
    elif accumulate:
        raise ValueError("delta_matching: accumulate=True needs weights")
    ops._enter(dev)
    L = _lib.lib()
    with torch.cuda.device(dev):
        o = torch.empty(B, N, H, D, device=dev, dtype=torch.bfloat16)
        lse = torch.empty(B, H, N, device=dev, dtype=torch.float32)
        bytes_ = L.dm_cache_attn_workspace_bytes(B, N, H, Hk, D, T, P, int(weights is not None))
        if bytes_ == 0:
            raise ValueError(_lib.last_error())
        ws = torch.empty(bytes_, device=dev, dtype=torch.uint8)
        w = (0, 0, 0, 0) if weights is None else (weights.data_ptr(), weights.stride(0), weights.stride(1), weights.shape[2])
        _lib.check(L.dm_cache_attn(
            ctypes.byref(_c_cache(cache, pages, Hk, P, D)), q.data_ptr(), q.stride(0), q.stride(1), q.stride(2), B, N, H,
            table.data_ptr(), row, T, lengths.data_ptr(), ops._ptr(q_counts), int(bool(causal)), scale, o.data_ptr(), lse.data_ptr(),
            *w, int(bool(accumulate)), ws.data_ptr(), bytes_, ops.status_word(dev).data_ptr(), ops._stream(q)))
        ops._after(dev)
    return (o, lse) if return_lse else o


def dm_cache_evict(cache, block_table, lengths, weights, new_block_table, budget, recent=0):
    """Cut every sequence to at most `budget` tokens a kv head: the last `recent` and, of the others, those of greatest weight (weights (B, Hk, W)
    fp32 as dm_cache_attn accumulates them; equal ones: the lowest positions; NaN is least), in their order.  The kept tokens are written,
    requantised to the scales of their new blocks, to the pages of new_block_table (B, T2) int32, which must not hold any of the sequences'
    tokens; the old pages are not changed and are the caller's to free.  Sequences within the budget are copied.

    Returns (new lengths (B) int32, kept (B, Hk, budget) int32: the old positions in order, -1 beyond, new weights (B, Hk, T2 * page_size) fp32: those of the
    kept tokens, 0 beyond).  The heads of a sequence keep different tokens but equally many."""
    if not torch.compiler.is_compiling():
        out = _lib.native_cache().cache_evict(cache, block_table, lengths, weights, new_block_table, budget, recent)
        if out is not None:
            return out
    if _recorded():
        return _OPS.cache_evict(*cache, block_table, lengths, weights, new_block_table, budget, recent)
    return evict_now(cache, block_table, lengths, weights, new_block_table, budget, recent)


def evict_now(cache, block_table, lengths, weights, new_block_table, budget, recent):
    """dm_cache_evict by the Python route, whatever records: what the registered op comes to where the native route does not take it."""
    pages, Hk, P, D = _check_cache(cache)
    _check_written(cache)
    _refuse_tangents(ks=cache.ks, vs=cache.vs, weights=weights)
    dev = cache.k8.device
    if not isinstance(lengths, torch.Tensor) or lengths.dim() != 1 or lengths.numel() == 0:
        raise ValueError("delta_matching: lengths must be a 1-D tensor, one entry per sequence")
    B = lengths.shape[0]
    lengths = _check_lengths("lengths", lengths, B, dev)
    table, row = _check_table("block_table", block_table, B, dev)
    new_table, new_row = _check_table("new_block_table", new_block_table, B, dev)
    T, T2 = table.shape[1], new_table.shape[1]
    _check_weights(weights, B, Hk, T * P, dev)
    budget, recent = operator.index(budget), operator.index(recent)
    if not 0 < budget <= T2 * P:
        raise ValueError(f"delta_matching: budget must be between 1 and the {T2 * P} tokens of a row of new_block_table (got {budget})")
    if not 0 <= recent <= budget:
        raise ValueError(f"delta_matching: recent must be between 0 and the budget (got {recent})")
    ops._enter(dev)
    with torch.cuda.device(dev):
        new = torch.empty(B, device=dev, dtype=torch.int32)
        kept = torch.empty(B, Hk, budget, device=dev, dtype=torch.int32)
        new_weights = torch.empty(B, Hk, T2 * P, device=dev, dtype=torch.float32)
        _lib.check(_lib.lib().dm_cache_evict(
            ctypes.byref(_c_cache(cache, pages, Hk, P, D)), B, table.data_ptr(), row, T, lengths.data_ptr(), weights.data_ptr(),
            weights.stride(0), weights.stride(1), new_table.data_ptr(), new_row, T2, budget, recent, new.data_ptr(), kept.data_ptr(),
            new_weights.data_ptr(), ops.status_word(dev).data_ptr(), ops._stream(lengths)))
        ops._after(dev)
    return new, kept, new_weights
