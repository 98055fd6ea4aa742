"""The op layer registered with torch.library, so that a tracing compiler sees opaque ops with known output shapes
instead of ctypes calls it cannot look into.

    torch.ops.delta_matching_b200.quant_qkv(q, k, v)                     -> q8, qs, k8, ks, v8, vs, kmean
    torch.ops.delta_matching_b200.fwd_fp8(q8, k8, v8, qs, ks, vs, causal) -> O, LSE
    torch.ops.delta_matching_b200.quant_do(do, o, with_o)                -> do8, dos, delta
    torch.ops.delta_matching_b200.delta_fp8(q8, k8, v8, do8, qs, ks, vs, dos, lse, causal, norm) -> delta
    torch.ops.delta_matching_b200.bwd_fp8(q8, k8, v8, do8, qs, ks, vs, dos, lse, delta, causal, ds32) -> dq, dk, dv
    torch.ops.delta_matching_b200.cache_append(k8!, v8!, ks!, vs!, k, v, block_table, lengths, counts) -> new lengths
    torch.ops.delta_matching_b200.cache_attn(q, k8, v8, ks, vs, block_table, lengths, q_counts, causal, softmax_scale) -> O, LSE
    torch.ops.delta_matching_b200.cache_attn_weights(..., weights!, accumulate) -> O, LSE
    torch.ops.delta_matching_b200.cache_evict(k8!, v8!, ks!, vs!, block_table, lengths, weights, new_block_table, budget, recent)
        -> new lengths, kept, new weights

The reference registers the same roles as real ops (csrc/delta_matching_api.cpp:683-715: fwd_fp8, delta_fp8, bwd_fp8_t)
and its autograd function calls them through torch.ops (delta_matching/attn.py:37-118), which is what lets its API run
under torch.compile without a graph break (tests/test_api.py:304-317).  The implementations are the functions of
delta_matching_b200.ops (CUDA only; there is no CPU implementation to fall back to); the fake implementations only
state shapes, dtypes and devices.  Tensors are in the op layer's layout: inputs (B, H, N, D) views, codes (B, H, N, D)
e4m3, scales (B, H, N // 32) fp32, O / dQ (B, N, H, D), dK / dV (B, N, Hk, D) bf16.  The cache's ops take its four pools one by one (those
marked ! are written in place) and are what the functions of cache.py call while something records: a compiler, torch.jit.trace, a dispatch mode.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch
from torch import Tensor

from . import ops

NS = "delta_matching_b200"
E4M3 = torch.float8_e4m3fn
F32 = torch.float32
BF16 = torch.bfloat16


def _quant_qkv(q: Tensor, k: Tensor, v: Tensor) -> Tuple[Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor]:
    return ops.quant_qkv(q, k, v)


quant_qkv = torch.library.custom_op(f"{NS}::quant_qkv", _quant_qkv, mutates_args=(), device_types="cuda")


@quant_qkv.register_fake
def _(q, k, v):
    B, H, N, D = q.shape
    Hk = k.shape[1]
    code = lambda h: q.new_empty((B, h, N, D), dtype=E4M3)
    scale = lambda h: q.new_empty((B, h, N // ops.BLK), dtype=F32)
    return code(H), scale(H), code(Hk), scale(Hk), code(Hk), scale(Hk), q.new_empty((B, Hk, D), dtype=F32)


def _fwd_fp8(q8: Tensor, k8: Tensor, v8: Tensor, qs: Tensor, ks: Tensor, vs: Tensor, causal: bool) -> Tuple[Tensor, Tensor]:
    return ops.fwd_fp8(q8, k8, v8, qs, ks, vs, causal)


fwd_fp8 = torch.library.custom_op(f"{NS}::fwd_fp8", _fwd_fp8, mutates_args=(), device_types="cuda")


@fwd_fp8.register_fake
def _(q8, k8, v8, qs, ks, vs, causal):
    B, H, N, D = q8.shape
    return q8.new_empty((B, N, H, D), dtype=BF16), q8.new_empty((B, H, N), dtype=F32)


def _quant_do(do: Tensor, o: Tensor, with_o: bool) -> Tuple[Tensor, Tensor, Tensor]:
    """with_o: also return the stale delta rowsum(dO * O); otherwise `o` is not read and delta comes back empty."""
    do8, dos, delta = ops.quant_do(do, o if with_o else None)
    if delta is None:
        delta = do.new_empty((0,), dtype=F32)
    return do8, dos, delta


quant_do = torch.library.custom_op(f"{NS}::quant_do", _quant_do, mutates_args=(), device_types="cuda")


@quant_do.register_fake
def _(do, o, with_o):
    B, H, N, D = do.shape
    delta = do.new_empty((B, H, N) if with_o else (0,), dtype=F32)
    return do.new_empty((B, H, N, D), dtype=E4M3), do.new_empty((B, H, N // ops.BLK), dtype=F32), delta


def _delta_fp8(q8: Tensor, k8: Tensor, v8: Tensor, do8: Tensor, qs: Tensor, ks: Tensor, vs: Tensor, dos: Tensor,
               lse: Tensor, causal: bool, norm: bool) -> Tensor:
    return ops.delta_fp8(q8, k8, v8, do8, qs, ks, vs, dos, lse, causal, norm)


delta_fp8 = torch.library.custom_op(f"{NS}::delta_fp8", _delta_fp8, mutates_args=(), device_types="cuda")


@delta_fp8.register_fake
def _(q8, k8, v8, do8, qs, ks, vs, dos, lse, causal, norm):
    return torch.empty_like(lse)


def _bwd_fp8(q8: Tensor, k8: Tensor, v8: Tensor, do8: Tensor, qs: Tensor, ks: Tensor, vs: Tensor, dos: Tensor,
             lse: Tensor, delta: Tensor, causal: bool, ds32: bool) -> Tuple[Tensor, Tensor, Tensor]:
    return ops.bwd_fp8(q8, k8, v8, do8, qs, ks, vs, dos, lse, delta, causal, ds32=ds32)


bwd_fp8 = torch.library.custom_op(f"{NS}::bwd_fp8", _bwd_fp8, mutates_args=(), device_types="cuda")


@bwd_fp8.register_fake
def _(q8, k8, v8, do8, qs, ks, vs, dos, lse, delta, causal, ds32):
    B, H, N, D = q8.shape
    Hk = k8.shape[1]
    return (q8.new_empty((B, N, H, D), dtype=BF16), q8.new_empty((B, N, Hk, D), dtype=BF16),
            q8.new_empty((B, N, Hk, D), dtype=BF16))


def _cache_call(native, python, *args):
    """What the functions of cache.py do at once: the native route, or the Python one where that takes the call."""
    from . import _lib, cache
    out = getattr(_lib.native_cache(), native)(*args)
    return getattr(cache, python)(*args) if out is None else out


def _cache_append(k8: Tensor, v8: Tensor, ks: Tensor, vs: Tensor, k: Tensor, v: Tensor, block_table: Tensor, lengths: Tensor,
                  counts: Optional[Tensor]) -> Tensor:
    from . import cache
    return _cache_call("cache_append", "append_now", cache.KVCache8(k8, v8, ks, vs), k, v, block_table, lengths, counts)


cache_append = torch.library.custom_op(f"{NS}::cache_append", _cache_append, mutates_args=("k8", "v8", "ks", "vs"), device_types="cuda")


@cache_append.register_fake
def _(k8, v8, ks, vs, k, v, block_table, lengths, counts):
    return lengths.new_empty(lengths.shape)


def _cache_attn(q: Tensor, k8: Tensor, v8: Tensor, ks: Tensor, vs: Tensor, block_table: Tensor, lengths: Tensor, q_counts: Optional[Tensor],
                causal: bool, softmax_scale: Optional[float]) -> Tuple[Tensor, Tensor]:
    from . import cache
    return _cache_call("cache_attn", "attn_now", q, cache.KVCache8(k8, v8, ks, vs), block_table, lengths, q_counts, causal, softmax_scale, None, False, True)


cache_attn = torch.library.custom_op(f"{NS}::cache_attn", _cache_attn, mutates_args=(), device_types="cuda")


@cache_attn.register_fake
def _(q, k8, v8, ks, vs, block_table, lengths, q_counts, causal, softmax_scale):
    B, N, H, D = q.shape
    return q.new_empty((B, N, H, D)), q.new_empty((B, H, N), dtype=F32)


def _cache_attn_weights(q: Tensor, k8: Tensor, v8: Tensor, ks: Tensor, vs: Tensor, block_table: Tensor, lengths: Tensor, q_counts: Optional[Tensor],
                        causal: bool, softmax_scale: Optional[float], weights: Tensor, accumulate: bool) -> Tuple[Tensor, Tensor]:
    from . import cache
    return _cache_call("cache_attn", "attn_now", q, cache.KVCache8(k8, v8, ks, vs), block_table, lengths, q_counts, causal, softmax_scale, weights, accumulate, True)


cache_attn_weights = torch.library.custom_op(f"{NS}::cache_attn_weights", _cache_attn_weights, mutates_args=("weights",), device_types="cuda")


@cache_attn_weights.register_fake
def _(q, k8, v8, ks, vs, block_table, lengths, q_counts, causal, softmax_scale, weights, accumulate):
    B, N, H, D = q.shape
    return q.new_empty((B, N, H, D)), q.new_empty((B, H, N), dtype=F32)


def _cache_evict(k8: Tensor, v8: Tensor, ks: Tensor, vs: Tensor, block_table: Tensor, lengths: Tensor, weights: Tensor, new_block_table: Tensor,
                 budget: int, recent: int) -> Tuple[Tensor, Tensor, Tensor]:
    from . import cache
    return _cache_call("cache_evict", "evict_now", cache.KVCache8(k8, v8, ks, vs), block_table, lengths, weights, new_block_table, budget, recent)


cache_evict = torch.library.custom_op(f"{NS}::cache_evict", _cache_evict, mutates_args=("k8", "v8", "ks", "vs"), device_types="cuda")


@cache_evict.register_fake
def _(k8, v8, ks, vs, block_table, lengths, weights, new_block_table, budget, recent):
    B, Hk = weights.shape[:2]
    return (lengths.new_empty((B,)), lengths.new_empty((B, Hk, budget)), weights.new_empty((B, Hk, new_block_table.shape[1] * k8.shape[2])))


class _Direct:
    """The attention's five calls without the dispatcher in between: what the eager path uses (a registered op costs tens of
    microseconds of host time per call, which shows once the kernels of a step take about two milliseconds)."""
    quant_qkv = staticmethod(_quant_qkv)
    fwd_fp8 = staticmethod(_fwd_fp8)
    quant_do = staticmethod(_quant_do)
    delta_fp8 = staticmethod(_delta_fp8)
    bwd_fp8 = staticmethod(_bwd_fp8)


DIRECT = _Direct
