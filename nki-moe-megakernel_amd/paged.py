"""Paged-cache operators for serving many samples of a few prompts: kv_append_rope and
attention_shared_prefix (no reference counterparts; attention_block_tkg, nki_kernels/attention/
attention_block_tkg.py:83, appends one row per sequence inside its fused block and reads a shared
prompt once per sequence).

Paged caches are [num_blocks, block_len, kv_heads, d] as in attention_block_tkg (d = 64 or 128),
contiguous in d; the block, row and head strides are free, so K and V may be views of one pool.
They are bf16, or float8 e4m3 (torch.float8_e4m3fn, or uint8 tensors of the codes).
"""
from __future__ import annotations

from typing import Optional

import torch

from . import _lib as L

_FP8 = (torch.float8_e4m3fn, torch.uint8)
_INT = (torch.int32, torch.int64)


def _read(t: torch.Tensor, mask: int, bytes_mask: int):
    """(t, its strides) for reading, or of a copy where a row does not start on the boundary that
    the kernels' loads need: strides and address free of the masks' bits."""
    st = t.stride()
    if st[-1] != 1 or (st[0] | st[1] | st[-2]) & mask or t.data_ptr() & bytes_mask:
        t = t.clone(memory_format=torch.contiguous_format)
        st = t.stride()
    return t, st


def _written(t: torch.Tensor, what: str, mask: int, bytes_mask: int):
    """The strides of a tensor that is used in place (0 where there is nothing to step over)."""
    st = t.stride()
    if st[-1] == 1 and all(st) and not ((st[0] | st[1] | st[-2]) & mask or t.data_ptr() & bytes_mask):
        return st
    st = tuple(0 if n == 1 else s for s, n in zip(st[:-1], t.shape))
    if t.numel() and (t.stride(-1) != 1 or any(s == 0 < n - 1 or s & mask for s, n in zip(st, t.shape))
                      or t.data_ptr() & bytes_mask):
        raise ValueError(f"{what} is used in place: its last dimension must be contiguous and its rows distinct, "
                         f"starting on multiples of {mask + 1} elements")
    return st


def _index(t: torch.Tensor, n: int, name: str, types=_INT) -> torch.Tensor:
    if t.dtype not in types:
        raise ValueError(f"{name} must be {' or '.join(str(x).split('.')[1] for x in types)}, got {t.dtype}")
    if t.shape != (n,):
        raise ValueError(f"{name} must be [{n}], got {tuple(t.shape)}")
    return t.contiguous()


def _caches(K_cache, V_cache, d: int):
    """(num_blocks, block_len, kv_heads, fp8) of a pair of paged caches."""
    shape, dtype = K_cache.shape, K_cache.dtype
    if len(shape) != 4 or shape != V_cache.shape:
        raise ValueError("K_cache and V_cache must both be [num_blocks, block_len, kv_heads, d], got "
                         f"{tuple(K_cache.shape)} and {tuple(V_cache.shape)}")
    if shape[3] != d:
        raise ValueError(f"the caches hold heads of {shape[3]}, the inputs of {d}")
    if d not in (64, 128):
        raise NotImplementedError(f"d must be 64 or 128, got {d}")
    if V_cache.dtype != dtype or (dtype != torch.bfloat16 and dtype not in _FP8):
        raise ValueError(f"the KV caches must both be bfloat16 or float8_e4m3, got {dtype} / {V_cache.dtype}")
    return shape[0], shape[1], shape[2], dtype != torch.bfloat16


def _scale(t: torch.Tensor, name: str) -> torch.Tensor:
    if t.dim() != 2 or t.shape[1] != 1 or t.numel() < 1:
        raise ValueError(f"{name} must be (1, 1) or (PMAX, 1), got {tuple(t.shape)}")
    if t.dtype not in (torch.float32, torch.float16, torch.bfloat16):
        raise ValueError(f"{name} dtype must be float32 / float16 / bfloat16, got {t.dtype}")
    return t if t.dtype == torch.float32 else t[:1].float()


def _norm(t: torch.Tensor, name: str, d: int) -> torch.Tensor:
    if t.numel() != d:
        raise ValueError(f"{name} must have {d} elements, got {tuple(t.shape)}")
    if t.dim() == 1 and t.dtype == torch.bfloat16 and t.stride(0) == 1 and not t.data_ptr() & 7:
        return t
    return t.reshape(-1).to(torch.bfloat16).clone(memory_format=torch.contiguous_format)


def _table(t: torch.Tensor) -> torch.Tensor:
    if t.dtype != torch.float32:
        if t.dtype != torch.bfloat16:
            raise ValueError(f"cos and sin must be float32 or bfloat16, got {t.dtype}")
        t = t.float()
    t = t.contiguous()
    return t.clone() if t.data_ptr() & 15 else t


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
    dev = L.gpu_index(q=q, k=k, v=v, cos=cos, sin=sin, positions=positions, K_cache=K_cache, V_cache=V_cache,
                      slots=slots, q_norm=q_norm, k_norm=k_norm, k_scale=k_scale, v_scale=v_scale, output=output)
    shape, kshape = q.shape, k.shape
    if len(shape) != 3 or len(kshape) != 3 or kshape != v.shape or kshape[0] != shape[0] or kshape[2] != shape[2]:
        raise ValueError("q must be [T, q_heads, d], k and v [T, kv_heads, d], got "
                         f"{tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}")
    T, nq, d = shape
    num_blocks, block_len, nkv, fp8 = _caches(K_cache, V_cache, d)
    if nkv != kshape[1]:
        raise ValueError(f"the caches hold {nkv} kv heads, k and v {kshape[1]}")
    dtype = q.dtype
    if (dtype != torch.bfloat16 and dtype != torch.float32) or k.dtype != dtype or v.dtype != dtype:
        raise ValueError(f"q, k and v must all be bfloat16 or float32, got {q.dtype}, {k.dtype}, {v.dtype}")
    if (k_scale is None) != (v_scale is None) or fp8 == (k_scale is None):
        raise ValueError("float8_e4m3 caches need k_scale and v_scale, bfloat16 caches neither")
    if (cos is None) != (sin is None) or (cos is None) != (positions is None):
        raise ValueError("cos, sin and positions must be given together")
    rot = rows = cos_p = sin_p = pos_p = pos_64 = 0
    if cos is not None:
        if cos.dim() != 2 or cos.shape != sin.shape or cos.shape[0] < 1:
            raise ValueError(f"cos and sin must be [rows, r / 2], got {tuple(cos.shape)} and {tuple(sin.shape)}")
        rows, rot = cos.shape
        rot *= 2
        if rot & 7 or not 8 <= rot <= d:
            raise ValueError(f"the rotated part must be a multiple of 8 from 8 to d = {d}, got {rot}")
        cos, sin, positions = _table(cos), _table(sin), _index(positions, T, "positions")
        cos_p, sin_p, pos_p, pos_64 = cos.data_ptr(), sin.data_ptr(), positions.data_ptr(), positions.dtype == torch.int64
    slots = _index(slots, T, "slots")
    if q_norm is not None:
        q_norm = _norm(q_norm, "q_norm", d)
    if k_norm is not None:
        k_norm = _norm(k_norm, "k_norm", d)
    quad = 3 if fp8 else 7
    ks, vs = _written(K_cache, "K_cache", 3, quad), _written(V_cache, "V_cache", 3, quad)
    if output is None:
        output = torch.empty(shape, dtype=torch.bfloat16, device=q.device)
    elif output.shape != shape or output.dtype != torch.bfloat16:
        raise ValueError(f"output must be bfloat16 [{T}, {nq}, {d}], got {output.dtype} {tuple(output.shape)}")
    os_ = _written(output, "output", 3, 7)
    if T == 0:
        return output, K_cache, V_cache
    f32 = dtype == torch.float32
    quad = 15 if f32 else 7
    (q, q_st), (k, k_st), (v, v_st) = _read(q, 3, quad), _read(k, 3, quad), _read(v, 3, quad)
    if fp8:
        k_scale, v_scale = _scale(k_scale, "k_scale"), _scale(v_scale, "v_scale")
    args = L.KvAppendArgs(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), f32, q_st[0], q_st[1], k_st[0], k_st[1], v_st[0], v_st[1],
        output.data_ptr(), os_[0], os_[1], L.ptr(q_norm), L.ptr(k_norm), eps, cos_p, sin_p, rows, rot, pos_p, pos_64,
        K_cache.data_ptr(), V_cache.data_ptr(), ks[0], ks[1], ks[2], vs[0], vs[1], vs[2], num_blocks, block_len,
        fp8, L.ptr(k_scale), L.ptr(v_scale), slots.data_ptr(), slots.dtype == torch.int64, T, nq, nkv, d)
    L.call(L.load().mkd_kv_append_rope, "kv_append_rope", dev, args)
    return output, K_cache, V_cache


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
    dev = L.gpu_index(q=q, K_cache=K_cache, V_cache=V_cache, prefix_tables=prefix_tables, prefix_lens=prefix_lens,
                      prefix_starts=prefix_starts, tables=tables, lens=lens, sink=sink, output=output)
    shape = q.shape
    if len(shape) not in (3, 4) or q.dtype != torch.bfloat16:
        raise ValueError(f"q must be bfloat16 [B, (S_tkg,) q_heads, d], got {q.dtype} {tuple(q.shape)}")
    B, nq, d, S_tkg = shape[0], shape[-2], shape[-1], shape[1] if len(shape) == 4 else 1
    if not 1 <= S_tkg <= 8:
        raise ValueError(f"S_tkg must be in [1, 8], got {S_tkg}")
    num_blocks, block_len, nkv, fp8 = _caches(K_cache, V_cache, d)
    if nkv < 1 or nq % nkv or nq < 1:
        raise ValueError(f"{nq} query heads do not share {nkv} kv heads evenly")
    i32 = (torch.int32,)
    if tables.dim() != 2 or tables.shape[0] != B or tables.dtype != torch.int32:
        raise ValueError(f"tables must be int32 [B={B}, blocks], got {tables.dtype} {tuple(tables.shape)}")
    lens = _index(lens, B, "lens", i32)
    if (prefix_tables is None) != (prefix_lens is None) or (prefix_tables is None) != (prefix_starts is None):
        raise ValueError("prefix_tables, prefix_lens and prefix_starts must be given together")
    G = wide = 0
    if prefix_tables is not None:
        if prefix_tables.dim() != 2 or prefix_tables.dtype != torch.int32:
            raise ValueError(f"prefix_tables must be int32 [G, blocks], got {prefix_tables.dtype} {tuple(prefix_tables.shape)}")
        G, wide = prefix_tables.shape
        prefix_lens = _index(prefix_lens, G, "prefix_lens", i32)
        prefix_starts = _index(prefix_starts, G + 1, "prefix_starts", i32)
        prefix_tables = prefix_tables.contiguous()
    if sink is not None:
        if sink.numel() != nq:
            raise ValueError(f"sink must have {nq} elements, got {tuple(sink.shape)}")
        if sink.dim() != 1 or sink.dtype != torch.float32 or sink.stride(0) != 1:
            sink = sink.reshape(-1).float().contiguous()
    row = 15 if fp8 else 7                      # 16 bytes
    ks, vs = _written(K_cache, "K_cache", row, 15), _written(V_cache, "V_cache", row, 15)
    if output is None:
        output = torch.empty(shape, dtype=torch.bfloat16, device=q.device)
    elif output.shape != shape or output.dtype != torch.bfloat16:
        raise ValueError(f"output must be bfloat16 {tuple(shape)}, got {output.dtype} {tuple(output.shape)}")
    os_ = _written(output, "output", 1, 3)
    if B == 0:
        return output
    q, qs = _read(q, 7, 15)
    tables = tables.contiguous()
    args = L.SharedPrefixArgs(
        q.data_ptr(), qs[0], qs[1] if S_tkg > 1 else 0, qs[-2], output.data_ptr(), os_[0], os_[1] if S_tkg > 1 else 0,
        os_[len(shape) - 2], K_cache.data_ptr(), V_cache.data_ptr(), ks[0], ks[1], ks[2], vs[0], vs[1], vs[2],
        num_blocks, block_len, fp8, L.ptr(prefix_tables), L.ptr(prefix_lens), L.ptr(prefix_starts), tables.data_ptr(),
        lens.data_ptr(), G, wide, tables.shape[1], softmax_scale if softmax_scale is not None else d ** -0.5,
        L.ptr(sink), B, S_tkg, nq, nkv, d)
    lib = L.load()
    n = lib.mkd_shared_prefix_workspace_bytes(args)
    ws = torch.empty(n, dtype=torch.uint8, device=q.device)
    L.call(lib.mkd_attention_shared_prefix, "attention_shared_prefix", dev, args, ws.data_ptr(), n)
    return output
