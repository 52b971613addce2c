"""Paged-cache operators for serving many samples of a few prompts: kv_append_rope and
attention_shared_prefix (no reference counterparts; attention_block_tkg, nki_kernels/attention/
attention_block_tkg.py:83, appends one row per sequence inside its fused block and reads a shared
prompt once per sequence).

Paged caches are [num_blocks, block_len, kv_heads, d] as in attention_block_tkg (d = 64 or 128),
contiguous in d; the block, row and head strides are free, so K and V may be views of one pool.
They are bf16, or float8 e4m3 (torch.float8_e4m3fn, or uint8 tensors of the codes).

The checks of arguments and the calls are native (csrc/torch_ops.cpp).
"""
from __future__ import annotations

from typing import Optional

import torch

from . import _lib as L

def kv_append_rope(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cos: Optional[torch.Tensor],
                   sin: Optional[torch.Tensor], positions: Optional[torch.Tensor], K_cache: torch.Tensor,
                   V_cache: torch.Tensor, slots: torch.Tensor, q_norm: Optional[torch.Tensor] = None,
                   k_norm: Optional[torch.Tensor] = None, eps: float = 1e-6, k_scale: Optional[torch.Tensor] = None,
                   v_scale: Optional[torch.Tensor] = None, output: Optional[torch.Tensor] = None):
    """Appends new tokens to a paged KV cache, their heads normed and rotated on the way; returns
    (q, K_cache, V_cache), q bf16 and the caches updated in place.

    q [T, q_heads, d], k and v [T, kv_heads, d]: bf16 or fp32, T >= 0 tokens of any sequences (a
    prompt, a decode batch, or both); views of one QKV projection are read where they lie.  In fp32:
    with q_norm / k_norm ([d]) each head becomes x * rsqrt(mean(x^2) + eps) * norm; then its first
    r elements are rotated by row positions[t] of cos / sin ([rows, r / 2] fp32, the halves layout:
    element i pairs with i + r / 2; r a multiple of 8, at most d; cos = sin = positions = None: no
    rotation).  slots [T] (int32 / int64) holds each token's cache row, block * block_len + row.  A
    slot outside the pool (-1, UINT32_MAX: padding) stores nothing; a position outside the tables
    stores nothing and gives a zero q row.  The slots that store must be distinct: a row that two
    tokens name is left undefined.  bf16 caches get one rounding from fp32; FP8 caches (k_scale and v_scale, as in
    attention_block_tkg) e4m3(clip(x * scale, +-240)).  `output`: a bf16 [T, q_heads, d] tensor for
    q, which may be q itself.
    """
    return L.native().kv_append_rope(q, k, v, cos, sin, positions, K_cache, V_cache, slots, q_norm, k_norm, eps, k_scale,
                                     v_scale, output)


def attention_shared_prefix(q: torch.Tensor, K_cache: torch.Tensor, V_cache: torch.Tensor,
                            prefix_tables: Optional[torch.Tensor], prefix_lens: Optional[torch.Tensor],
                            prefix_starts: Optional[torch.Tensor], tables: torch.Tensor, lens: torch.Tensor,
                            softmax_scale: Optional[float] = None, sink: Optional[torch.Tensor] = None,
                            output: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Decode attention over a paged cache in which groups of sequences share a prefix; the prefix
    is read once for all of a group's query rows.  Returns a tensor of q's shape, bf16.

    q [B, q_heads, d], or [B, S_tkg, q_heads, d] with S_tkg <= 8 new tokens per sequence: bf16,
    rotated, the new tokens' keys and values already in the cache (kv_append_rope).  Group g holds
    the sequences prefix_starts[g] .. prefix_starts[g + 1] - 1 (prefix_starts [G + 1], ascending;
    sequences outside of it belong to no group) and its prefix is the first prefix_lens[g] positions
    of prefix_tables[g] ([G, blocks]).  All three None: no prefixes.  Sequence b's own positions, its
    new tokens last, are the first lens[b] of tables[b] ([B, blocks]); they start in a block of their
    own whatever the prefix's length.  New token i sees the prefix and the own positions up to its
    own, lens[b] - S_tkg + i.  All four index tensors are int32 in device memory and are not read on
    the host (the call can be captured); a length is clamped to what its table holds, a block id
    outside the pool reads as rows of zeros.

    softmax_scale: 1 / sqrt(d) by default.  sink [q_heads]: a logit that joins each head's
    normaliser.  A query that sees nothing gets zeros.  FP8 caches are attended as stored (as in
    attention_block_tkg: fold k_scale into softmax_scale, v_scale into what follows).
    """
    return L.native().attention_shared_prefix(q, K_cache, V_cache, prefix_tables, prefix_lens, prefix_starts, tables, lens,
                                              softmax_scale, sink, output)
