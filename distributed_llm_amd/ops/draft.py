"""Drafted tokens: attention for a tree of them over the paged cache, their verification, and what a step keeps of them.

A speculative step asks the target model about several tokens of a sequence at once.  Its nodes are the sequence's rows ``seq_qstart .. seq_qstart +
seq_qlen - 1`` of the step: the root, which is the last committed token, and the drafted tokens behind it, every node behind its parent (``parents``: the
place within the sequence, -1 at the root).  Their K and V go to the cache as any new tokens' do (``ops.rope_and_cache``, ``kv8.rope_and_cache``), node i at
place ``seq_ctx - seq_qlen + i``; their positions are the root's plus ``depth``.

    mask, depth = draft.tree_mask(parents, qstart, qlen, max_nodes)          # a chain needs none
    out = draft.tree_attention(q, k_cache, v_cache, tables, qstart, qlen, ctx, mask)          # in every layer
    accepted, token, path = draft.verify(probabilities, tokens, uniform, qstart, qlen, max_nodes, parents=parents)
    draft.keep(k_caches, v_caches, tables, qlen, ctx, path, accepted)          # the sequence now has ctx - qlen + accepted + 1 tokens in the cache

No call looks at lengths on the host or waits, so a captured graph takes new trees and lengths.
"""
from __future__ import annotations

import math
from typing import Optional, Tuple

import torch

from . import _native, reference as ref
from .kv8 import need, need_cache, need_device, need_vec, overlap

MAX_NODES = 1024    # of a tree


def tree_mask(parents: torch.Tensor, seq_qstart: torch.Tensor, seq_qlen: torch.Tensor, max_nodes: int) -> Tuple[torch.Tensor, torch.Tensor]:
    """What each node sees of its tree, for ``tree_attention``: int32 [T, ceil(max_nodes / 32)], bit i % 32 of word i / 32 where node i is itself or an
    ancestor; and each node's depth, int32 [T].  Trees have at most ``max_nodes`` nodes; rows of no sequence are zero."""
    ext = _native(parents)
    if ext is not None:
        return ext.tree_mask(parents, seq_qstart, seq_qlen, max_nodes)
    need(parents.dim() == 1 and parents.dtype == torch.int32 and parents.is_contiguous(), "parents: contiguous int32 [T]")
    need(1 <= max_nodes <= MAX_NODES, f"max_nodes must be 1 to {MAX_NODES}")
    for t, name in ((seq_qstart, "seq_qstart"), (seq_qlen, "seq_qlen")):
        need_vec(t, name, seq_qstart.numel(), parents)
    return ref.tree_mask(parents, seq_qstart, seq_qlen, max_nodes)


def tree_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_tables: torch.Tensor, seq_qstart: torch.Tensor,
                   seq_qlen: torch.Tensor, seq_ctx: torch.Tensor, mask: Optional[torch.Tensor] = None, scale: Optional[float] = None,
                   k_scale: Optional[torch.Tensor] = None, v_scale: Optional[torch.Tensor] = None, max_qlen: int = 0, max_ctx: int = 0,
                   out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of new tokens ``q`` [T, nq, d] (bf16, head_dim 64, 96 or 128) over the paged cache, bf16 or, with its scales, 8-bit.

    A token sees the ``seq_ctx - seq_qlen`` keys before its sequence's new ones, and of those the ones that ``mask`` (``tree_mask``) names; without a mask
    itself and those before it (a chain, a prompt's rows, a single token).  A row that sees nothing, or scores of minus infinity alone, is zero; what a row does not
    see does not reach it, NaN and infinities included, nor do keys of pages outside the pool.  Any number of query heads a kv head.  Rows of ``q`` that belong to no sequence are
    not written.  ``max_qlen``, ``max_ctx``: the longest, where the host knows them (0: it does not); they pick the launch, never the result's rows."""
    scale = (1.0 / math.sqrt(q.shape[-1])) if scale is None else scale
    ext = _native(q)
    if ext is not None:
        return ext.tree_attention(q, k_cache, v_cache, block_tables, seq_qstart, seq_qlen, seq_ctx, mask, scale, k_scale, v_scale, max_qlen, max_ctx, out)
    need(q.dim() == 3 and q.dtype == torch.bfloat16 and q.stride(2) == 1 and q.stride(0) % 8 == 0 and q.stride(1) % 8 == 0,
         "q: bfloat16 [T, nq, d] with rows of 16-byte alignment")
    T, nq, d = q.shape
    _, nkv, dim = need_cache(k_cache, v_cache, k_scale, v_scale, q)
    need(dim == d and d in (64, 96, 128), "head_dim must be 64, 96 or 128, and the cache's")
    need(nkv >= 1 and nq >= 1 and nq % nkv == 0, "query heads must be a multiple of the cache's")
    need_device(block_tables, "block_tables", q)
    need(block_tables.dim() == 2 and block_tables.dtype == torch.int32 and block_tables.is_contiguous(),
         "block_tables: contiguous int32 [num_seqs, max_blocks]")
    for t, name in ((seq_qstart, "seq_qstart"), (seq_qlen, "seq_qlen"), (seq_ctx, "seq_ctx")):
        need_vec(t, name, block_tables.shape[0], q)
    need(max_qlen >= 0 and max_ctx >= 0, "max_qlen and max_ctx: 0 (unknown) or more")
    if mask is not None:
        need_device(mask, "mask", q)
        need(mask.dim() == 2 and mask.dtype == torch.int32 and mask.is_contiguous() and mask.shape[0] == T and mask.shape[1] >= 1,
             "mask: contiguous int32 [T, words]")
    if out is not None:
        need_device(out, "out", q)
        need(out.shape == q.shape and out.dtype == torch.bfloat16 and out.is_contiguous(), "out: contiguous bfloat16 like q, 16-byte aligned")
        need(T == 0 or not overlap(out, q), "out overlaps q")
    o = ref.tree_attention(q, k_cache, v_cache, block_tables, seq_qstart, seq_qlen, seq_ctx, mask, scale, k_scale, v_scale)
    if out is None:
        return o
    for q0, n in zip(seq_qstart.tolist(), seq_qlen.tolist()):
        out[max(q0, 0):max(q0 + n, 0)] = o[max(q0, 0):max(q0 + n, 0)]
    return out


def verify(target: torch.Tensor, tokens: torch.Tensor, uniform: torch.Tensor, seq_qstart: torch.Tensor, seq_qlen: torch.Tensor, max_nodes: int,
           parents: Optional[torch.Tensor] = None, draft: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Which drafted tokens the target keeps, and the token after them: (accepted [S], token [S], path [S, max_nodes]), int32.

    ``target`` [T, V] (f32 or bf16): row i holds the target's probabilities after node i.  ``tokens`` [T]: the nodes' tokens.  ``uniform`` [T]: numbers
    of [0, 1), one a node: the root's draws the token after the last accepted node, the others accept.  With these the tokens are distributed as the
    target's own.
      ``draft`` given: a chain (node i behind node i - 1) whose tokens were drawn, node i's from row i of ``draft``.  It is accepted where
      u draft < target, and the last draw is from max(target - draft, 0) of the refused node, or from the target behind the last one.
      no ``draft``: given candidates, a tree by ``parents`` or a chain.  A node's children are tried in order, each against what the earlier ones left
      of the target: u (1 - what they held) < target; the last draw leaves the refused children's tokens out.
    A NaN accepts nothing, nor do candidates behind it, of whose parent it leaves no number; the last draw takes it for 0.
    ``path``: the root and the accepted nodes, -1 behind them.  A sequence without nodes gets 0 accepted and token -1.  Sums and products are of 64
    bits."""
    ext = _native(target)
    if ext is not None:
        return ext.verify_drafts(target, tokens, uniform, seq_qstart, seq_qlen, max_nodes, parents, draft)
    need(target.dim() == 2 and target.dtype in (torch.float32, torch.bfloat16) and target.shape[1] >= 1 and (target.stride(1) == 1 or target.shape[1] == 1),
         "target: float32 or bfloat16 [T, vocab]")
    T, S = target.shape[0], seq_qstart.numel()
    need_vec(tokens, "tokens", T, target)
    need_device(uniform, "uniform", target)
    need(uniform.dtype == torch.float32 and uniform.shape == (T,) and uniform.is_contiguous(), "uniform: contiguous float32 [T]")
    need_vec(seq_qstart, "seq_qstart", S, target)
    need_vec(seq_qlen, "seq_qlen", S, target)
    need(1 <= max_nodes <= MAX_NODES, f"max_nodes must be 1 to {MAX_NODES}")
    need(parents is None or draft is None, "a tree's candidates are given, not drawn: parents or draft, not both")
    if parents is not None:
        need_vec(parents, "parents", T, target)
    if draft is not None:
        need_device(draft, "draft", target)
        need(draft.shape == target.shape and draft.dtype == target.dtype and (draft.stride(1) == 1 or draft.shape[1] == 1), "draft: like target")
    need(S <= 65535, "at most 65535 sequences")
    return ref.verify_drafts(target, tokens, uniform, seq_qstart, seq_qlen, max_nodes, parents, draft)


def keep(k_cache: torch.Tensor, v_cache: torch.Tensor, block_tables: torch.Tensor, seq_qlen: torch.Tensor, seq_ctx: torch.Tensor, path: torch.Tensor,
         accepted: torch.Tensor, k_scale: Optional[torch.Tensor] = None, v_scale: Optional[torch.Tensor] = None) -> None:
    """Move K and V of the accepted nodes to the places behind the root, in place: node ``path[s, j]`` to place ``seq_ctx - seq_qlen + j``, j up to
    ``accepted[s]``.  Caches of one layer, or of all of them with a leading dimension; scales with an 8-bit one.  A chain's accepted nodes are in place
    already.  The blocks that hold a sequence's drafted tokens must be its own."""
    ext = _native(k_cache)
    if ext is not None:
        return ext.keep_drafts(k_cache, v_cache, block_tables, seq_qlen, seq_ctx, path, accepted, k_scale, v_scale)
    need(k_cache.dim() in (4, 5), "caches: one layer's or [layers, ...]")
    _, _, d = need_cache(k_cache, v_cache, k_scale, v_scale, k_cache, k_cache.dim() - 4)
    need(16 <= d <= 128 and d % 16 == 0, "head_dim must be a multiple of 16, at most 128")
    need_device(block_tables, "block_tables", k_cache)
    need(block_tables.dim() == 2 and block_tables.dtype == torch.int32 and block_tables.is_contiguous(), "block_tables: contiguous int32 [num_seqs, max_blocks]")
    S = block_tables.shape[0]
    for t, name in ((seq_qlen, "seq_qlen"), (seq_ctx, "seq_ctx"), (accepted, "accepted")):
        need_vec(t, name, S, k_cache)
    need_device(path, "path", k_cache)
    need(path.dim() == 2 and path.dtype == torch.int32 and path.is_contiguous() and path.shape[0] == S and path.shape[1] >= 1,
         "path: contiguous int32 [num_seqs, max_nodes]")
    need(S <= 65535, "at most 65535 sequences")
    ref.keep_drafts(k_cache, v_cache, block_tables, seq_qlen, seq_ctx, path, accepted, k_scale, v_scale)
