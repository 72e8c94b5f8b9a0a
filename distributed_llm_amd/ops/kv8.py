"""The paged K/V cache in 8 bits: e4m3 codes with one f32 scale a token and head (csrc/kernels/kv8.hip).

Half the bytes of the bf16 cache (and 4 a vector), so half the time of a decode step's attention and twice the tokens of a pool.  Layouts and slots are
the bf16 cache's: K [num_blocks, nkv, 16, d], V [num_blocks, nkv, d, 16], scales [num_blocks, nkv, 16], slot = block * 16 + offset, negative slots
(padding rows) are not written.  Attention over it: ``draft.tree_attention`` with the scales, for single tokens, drafted trees and the rows of a prompt.

A vector's scale is its largest magnitude / 448 (2^-100 / 448 at least) and its codes are e4m3(448 x / largest), rounded to nearest even: code times scale,
which is what attention computes with, is off by at most 2^-4 of the value, or 2^-10 / 448 of the vector's largest where that is more; ``read`` rounds it to
bf16 once more.  A vector with an infinity or NaN reads back as NaN.
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Tuple

import torch

from . import BLOCK_SIZE, _native, reference as ref


class Cache(NamedTuple):
    k: torch.Tensor         # float8_e4m3fn [num_blocks, nkv, 16, d]
    v: torch.Tensor         # float8_e4m3fn [num_blocks, nkv, d, 16]
    k_scale: torch.Tensor   # float32 [num_blocks, nkv, 16]
    v_scale: torch.Tensor


def alloc(num_blocks: int, nkv: int, d: int, device=None) -> Cache:
    """An empty pool (codes of zero)."""
    codes = [torch.zeros(s, dtype=torch.uint8, device=device).view(torch.float8_e4m3fn) for s in ((num_blocks, nkv, BLOCK_SIZE, d), (num_blocks, nkv, d, BLOCK_SIZE))]
    return Cache(*codes, *(torch.zeros((num_blocks, nkv, BLOCK_SIZE), dtype=torch.float32, device=device) for _ in range(2)))


def need(cond: bool, what: str) -> None:
    if not cond:
        raise ValueError(what)


def need_device(t: torch.Tensor, name: str, like: torch.Tensor) -> None:
    need(t.device == like.device, f"{name} is on another device")


def overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two tensors of at least one value lie in common bytes (from their first to their last)."""
    ends = [(t.data_ptr(), t.data_ptr() + (1 + sum((n - 1) * m for n, m in zip(t.shape, t.stride()))) * t.element_size()) for t in (a, b)]
    return ends[0][0] < ends[1][1] and ends[1][0] < ends[0][1]


def need_vec(t: torch.Tensor, name: str, n: int, like: torch.Tensor) -> None:
    need_device(t, name, like)
    need(t.dtype == torch.int32 and t.shape == (n,) and t.is_contiguous(), f"{name}: contiguous int32 [{n}]")


def need_cache(k, v, ks, vs, like: torch.Tensor, lead: int = 0) -> Tuple[int, int, int]:
    """(blocks, nkv, d) of a bf16 cache, or of an 8-bit one with its scales."""
    for t in (k, v):
        need(t.device == like.device, "the cache is on another device")
    need(k.dim() == 4 + lead and v.dim() == 4 + lead and k.is_contiguous() and v.is_contiguous() and k.shape[-2] == BLOCK_SIZE and
         v.shape[-1] == BLOCK_SIZE and v.shape[-2] == k.shape[-1] and v.shape[:-2] == k.shape[:-2],
         "cache layout: contiguous K [blocks, nkv, 16, d], V [blocks, nkv, d, 16]")
    need((ks is None) == (vs is None), "k_scale and v_scale come together")
    if ks is None:
        need(k.dtype == torch.bfloat16 and v.dtype == torch.bfloat16, "a cache without scales is bfloat16")
    else:
        need(k.dtype == torch.float8_e4m3fn and v.dtype == torch.float8_e4m3fn, "a cache with scales is float8_e4m3fn")
        for t in (ks, vs):
            need(t.device == like.device, "scales is on another device")
            need(t.dtype == torch.float32 and t.is_contiguous() and t.shape == k.shape[:-1], "scales: contiguous f32 [blocks, nkv, 16]")
    return k.shape[lead], k.shape[lead + 1], k.shape[-1]


def _need_kv8(cache: Cache, like: torch.Tensor) -> Tuple[int, int, int]:
    blocks, nkv, d = need_cache(*cache, like)
    need(16 <= d <= 128 and d % 16 == 0, "head_dim must be a multiple of 16, at most 128")
    return blocks, nkv, d


def rope_and_cache(qkv: torch.Tensor, positions: torch.Tensor, cos_sin: torch.Tensor, slots: torch.Tensor, cache: Cache, nq: int, nkv: int, d: int,
                   q_out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Rotate q and k, write k and v into the 8-bit cache, return q as bf16 [T, nq, d] (``ops.rope_and_cache`` for this cache).  k is quantised from
    the rotated f32 values, without a rounding to bf16 between.  Slots must differ; positions are those of ``cos_sin``'s rows."""
    ext = _native(qkv)
    if ext is not None:
        return ext.kv8_rope(qkv, positions, cos_sin, slots, *cache, nq, nkv, d, q_out)
    need(qkv.dim() == 2 and qkv.dtype == torch.bfloat16 and qkv.stride(1) == 1 and qkv.stride(0) % 8 == 0,
         "qkv: bfloat16 [T, (nq + 2 nkv) d] with rows of 16-byte alignment")
    blocks, n, dim = _need_kv8(cache, qkv)
    T = qkv.shape[0]
    need(n == nkv and dim == d and nq >= 0 and nkv >= 1 and qkv.shape[1] >= (nq + 2 * nkv) * d, "qkv and cache disagree on heads or head_dim")
    need_vec(positions, "positions", T, qkv)
    need_vec(slots, "slots", T, qkv)
    need_device(cos_sin, "cos_sin", qkv)
    need(cos_sin.dim() == 2 and cos_sin.dtype == torch.float32 and cos_sin.is_contiguous() and cos_sin.shape[1] == d and cos_sin.shape[0] >= 1,
         "cos_sin: contiguous float32 [max_pos, d]")
    if q_out is not None:
        need_device(q_out, "q_out", qkv)
        need(q_out.shape == (T, nq, d) and q_out.dtype == torch.bfloat16 and q_out.is_contiguous(), "q_out: contiguous bfloat16 [T, nq, d], 16-byte aligned")
        need(q_out.numel() == 0 or not overlap(q_out, qkv), "q_out overlaps qkv")
    need(T == 0 or blocks >= 1, "the cache has no blocks")
    q = ref.kv8_rope(qkv, positions, cos_sin, slots, cache, nq, nkv, d)
    return q if q_out is None else q_out.copy_(q)


def write(k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, cache: Cache) -> None:
    """bf16 [T, nkv, d] rows into the cache (``ops.kv_write`` for this cache)."""
    ext = _native(k)
    if ext is not None:
        return ext.kv8_write(k, v, slots, *cache)
    for t in (k, v):
        need(t.dim() == 3 and t.dtype == torch.bfloat16 and t.shape == k.shape and t.stride(2) == 1 and (t.stride(1) == t.shape[2] or t.shape[1] == 1) and
             t.stride(0) % 8 == 0, "k, v: bfloat16 [T, nkv, d] with rows of 16-byte alignment")
    need_device(v, "v", k)
    blocks, nkv, d = _need_kv8(cache, k)
    need(nkv == k.shape[1] and d == k.shape[2] and nkv >= 1, "k, v and cache disagree on heads or head_dim")
    need_vec(slots, "slots", k.shape[0], k)
    need(k.shape[0] == 0 or blocks >= 1, "the cache has no blocks")
    ref.kv8_write(k, v, slots, cache)


def read(cache: Cache, slots: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """Tokens of the cache as bf16 rows (k, v), each [T, nkv, d]: a conversation handed to another pool, or to a model's bf16 cache.  A slot outside the
    pool gives zeros."""
    ext = _native(cache.k)
    if ext is not None:
        return ext.kv8_read(*cache, slots)
    blocks, _, _ = _need_kv8(cache, cache.k)
    need(slots.dim() == 1, "slots: contiguous int32 [T]")
    need_vec(slots, "slots", slots.shape[0], cache.k)
    need(slots.shape[0] == 0 or blocks >= 1, "the cache has no blocks")
    k, v = ref.kv8_read(cache, slots)
    return k, v
