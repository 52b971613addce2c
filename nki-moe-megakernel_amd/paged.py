"""Paged-cache operators for serving many samples of a few prompts: kv_append_rope and
attention_shared_prefix (no reference counterparts; attention_block_tkg, nki_kernels/attention/
attention_block_tkg.py:83, appends one row per sequence inside its fused block and reads a shared
prompt once per sequence).

Paged caches are [num_blocks, block_len, kv_heads, d] as in attention_block_tkg (d = 64 or 128),
contiguous in d; the block, row and head strides are free, so K and V may be views of one pool.
They are bf16, or float8 e4m3 (torch.float8_e4m3fn, or uint8 tensors of the codes).
"""
from __future__ import annotations

import math
from typing import Optional

import torch

from . import _lib as L

_FP8 = (torch.float8_e4m3fn, torch.uint8)


def _strides(t: torch.Tensor, n: int):
    """Strides of the first n dimensions, 0 where there is nothing to step over."""
    return tuple(0 if t.shape[i] == 1 else t.stride(i) for i in range(n))


def _rows(t: torch.Tensor, quantum: int) -> torch.Tensor:
    """t, or a contiguous copy where its rows do not start on multiples of `quantum` elements."""
    n = t.dim() - 1
    if (t.stride(n) == 1 or t.shape[n] == 1) and not t.data_ptr() % (quantum * t.element_size()) \
            and not any(s % quantum for s in _strides(t, n)):
        return t
    t = t.contiguous()
    return t if not t.data_ptr() % 16 else t.clone()


def _written(t: torch.Tensor, what: str, quantum: int):
    """Checks a tensor that is written in place."""
    n = t.dim() - 1
    if t.numel() and (t.stride(n) != 1 or any(t.shape[i] > 1 and t.stride(i) == 0 for i in range(n))
                      or t.data_ptr() % (quantum * t.element_size()) or any(s % quantum for s in _strides(t, n))):
        raise ValueError(f"{what} is written in place: its last dimension must be contiguous and its rows distinct, "
                         f"on multiples of {quantum} elements")


def _same_device(dev, **tensors):
    for name, t in tensors.items():
        if t is not None and t.device != dev:
            raise ValueError(f"{name} is on {t.device}, the operator's inputs on {dev}")


def _index(t: torch.Tensor, n: int, name: str, types=(torch.int32, torch.int64)) -> torch.Tensor:
    if t.dtype not in types:
        raise ValueError(f"{name} must be {' or '.join(str(x).split('.')[1] for x in types)}, got {t.dtype}")
    if t.numel() != n or t.dim() != 1:
        raise ValueError(f"{name} must be [{n}], got {tuple(t.shape)}")
    return t.contiguous()


def _caches(K_cache, V_cache, d: int):
    """(num_blocks, block_len, kv_heads, fp8) of a pair of paged caches."""
    if K_cache.dim() != 4 or K_cache.shape != V_cache.shape:
        raise ValueError("K_cache and V_cache must both be [num_blocks, block_len, kv_heads, d], got "
                         f"{tuple(K_cache.shape)} and {tuple(V_cache.shape)}")
    if K_cache.shape[3] != d:
        raise ValueError(f"the caches hold heads of {K_cache.shape[3]}, the inputs of {d}")
    if d not in (64, 128):
        raise NotImplementedError(f"d must be 64 or 128, got {d}")
    if K_cache.dtype != V_cache.dtype or K_cache.dtype not in (torch.bfloat16, *_FP8):
        raise ValueError(f"the KV caches must both be bfloat16 or float8_e4m3, got {K_cache.dtype} / {V_cache.dtype}")
    return (*K_cache.shape[:3], K_cache.dtype in _FP8)


def _scale(t: torch.Tensor, name: str) -> torch.Tensor:
    if t.dim() != 2 or t.shape[1] != 1 or t.numel() < 1:
        raise ValueError(f"{name} must be (1, 1) or (PMAX, 1), got {tuple(t.shape)}")
    if t.dtype not in (torch.float32, torch.float16, torch.bfloat16):
        raise ValueError(f"{name} dtype must be float32 / float16 / bfloat16, got {t.dtype}")
    return t if t.dtype == torch.float32 else t[:1].float()


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
    L.require_gpu(q, k, v, cos, sin, positions, K_cache, V_cache, slots, q_norm, k_norm, k_scale, v_scale, output)
    dev = q.device
    _same_device(dev, k=k, v=v, cos=cos, sin=sin, positions=positions, K_cache=K_cache, V_cache=V_cache, slots=slots,
                 q_norm=q_norm, k_norm=k_norm, k_scale=k_scale, v_scale=v_scale, output=output)
    if q.dim() != 3 or k.dim() != 3 or k.shape != v.shape or k.shape[0] != q.shape[0] or k.shape[2] != q.shape[2]:
        raise ValueError("q must be [T, q_heads, d], k and v [T, kv_heads, d], got "
                         f"{tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}")
    T, nq, d = q.shape
    num_blocks, block_len, nkv, fp8 = _caches(K_cache, V_cache, d)
    if nkv != k.shape[1]:
        raise ValueError(f"the caches hold {nkv} kv heads, k and v {k.shape[1]}")
    if q.dtype not in (torch.bfloat16, torch.float32) or k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError(f"q, k and v must all be bfloat16 or float32, got {q.dtype}, {k.dtype}, {v.dtype}")
    if fp8 != (k_scale is not None and v_scale is not None) or (k_scale is None) != (v_scale is None):
        raise ValueError("float8_e4m3 caches need k_scale and v_scale, bfloat16 caches neither")
    if (cos is None) != (sin is None) or (cos is None) != (positions is None):
        raise ValueError("cos, sin and positions must be given together")
    rot = 0
    if cos is not None:
        if cos.dim() != 2 or cos.shape != sin.shape or cos.shape[0] < 1:
            raise ValueError(f"cos and sin must be [rows, r / 2], got {tuple(cos.shape)} and {tuple(sin.shape)}")
        rot = 2 * cos.shape[1]
        if rot % 8 or not 8 <= rot <= d:
            raise ValueError(f"the rotated part must be a multiple of 8 from 8 to d = {d}, got {rot}")
        if any(t.dtype not in (torch.float32, torch.bfloat16) for t in (cos, sin)):
            raise ValueError(f"cos and sin must be float32 or bfloat16, got {cos.dtype} and {sin.dtype}")
        cos, sin = (t.float().contiguous() for t in (cos, sin))
        cos, sin = (t if not t.data_ptr() % 16 else t.clone() for t in (cos, sin))
        positions = _index(positions, T, "positions")
    slots = _index(slots, T, "slots")
    norms = []
    for name, t in (("q_norm", q_norm), ("k_norm", k_norm)):
        if t is not None:
            if t.numel() != d:
                raise ValueError(f"{name} must have {d} elements, got {tuple(t.shape)}")
            t = _rows(t.reshape(-1).to(torch.bfloat16), 4)
        norms.append(t)
    _written(K_cache, "K_cache", 4)
    _written(V_cache, "V_cache", 4)
    if output is None:
        output = torch.empty(T, nq, d, dtype=torch.bfloat16, device=dev)
    elif tuple(output.shape) != (T, nq, d) or output.dtype != torch.bfloat16:
        raise ValueError(f"output must be bfloat16 [{T}, {nq}, {d}], got {output.dtype} {tuple(output.shape)}")
    else:
        _written(output, "output", 4)
    if T == 0:
        return output, K_cache, V_cache
    q, k, v = _rows(q, 4), _rows(k, 4), _rows(v, 4)
    ks, vs = (_scale(k_scale, "k_scale"), _scale(v_scale, "v_scale")) if fp8 else (None, None)
    args = L.KvAppendArgs(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), L.DT_F32 if q.dtype == torch.float32 else L.DT_BF16,
        _strides(q, 2), _strides(k, 2), _strides(v, 2), output.data_ptr(), _strides(output, 2),
        L.ptr(norms[0]), L.ptr(norms[1]), float(eps), L.ptr(cos), L.ptr(sin), cos.shape[0] if rot else 0, rot,
        L.ptr(positions), int(rot > 0 and positions.dtype == torch.int64), K_cache.data_ptr(), V_cache.data_ptr(),
        _strides(K_cache, 3), _strides(V_cache, 3), num_blocks, block_len, L.KV_FP8 if fp8 else 0, L.ptr(ks), L.ptr(vs),
        slots.data_ptr(), int(slots.dtype == torch.int64), T, nq, nkv, d)
    with L.on_device(dev):
        L.check(L.load().mkd_kv_append_rope(args, L.stream_ptr(dev)), "kv_append_rope")
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
    L.require_gpu(q, K_cache, V_cache, prefix_tables, prefix_lens, prefix_starts, tables, lens, sink, output)
    dev = q.device
    _same_device(dev, K_cache=K_cache, V_cache=V_cache, prefix_tables=prefix_tables, prefix_lens=prefix_lens,
                 prefix_starts=prefix_starts, tables=tables, lens=lens, sink=sink, output=output)
    if q.dim() not in (3, 4) or q.dtype != torch.bfloat16:
        raise ValueError(f"q must be bfloat16 [B, (S_tkg,) q_heads, d], got {q.dtype} {tuple(q.shape)}")
    shape = q.shape
    q4 = q if q.dim() == 4 else q.unsqueeze(1)
    B, S_tkg, nq, d = q4.shape
    if not 1 <= S_tkg <= 8:
        raise ValueError(f"S_tkg must be in [1, 8], got {S_tkg}")
    num_blocks, block_len, nkv, fp8 = _caches(K_cache, V_cache, d)
    if nkv < 1 or nq % nkv or nq < 1:
        raise ValueError(f"{nq} query heads do not share {nkv} kv heads evenly")
    i32 = (torch.int32,)
    if tables.dim() != 2 or tables.shape[0] != B or tables.dtype != torch.int32:
        raise ValueError(f"tables must be int32 [B={B}, blocks], got {tables.dtype} {tuple(tables.shape)}")
    lens = _index(lens, B, "lens", i32)
    given = [t is not None for t in (prefix_tables, prefix_lens, prefix_starts)]
    if any(given) != all(given):
        raise ValueError("prefix_tables, prefix_lens and prefix_starts must be given together")
    G = 0
    if given[0]:
        if prefix_tables.dim() != 2 or prefix_tables.dtype != torch.int32:
            raise ValueError(f"prefix_tables must be int32 [G, blocks], got {prefix_tables.dtype} {tuple(prefix_tables.shape)}")
        G = prefix_tables.shape[0]
        prefix_lens = _index(prefix_lens, G, "prefix_lens", i32)
        prefix_starts = _index(prefix_starts, G + 1, "prefix_starts", i32)
        prefix_tables = prefix_tables.contiguous()
    if sink is not None:
        if sink.numel() != nq:
            raise ValueError(f"sink must have {nq} elements, got {tuple(sink.shape)}")
        sink = sink.reshape(-1).float().contiguous()
    for name, t in (("K_cache", K_cache), ("V_cache", V_cache)):
        if t.stride(3) != 1 or t.data_ptr() % 16 or any(s * t.element_size() % 16 for s in _strides(t, 3)):
            raise ValueError(f"{name}'s rows must be contiguous and start on 16-byte boundaries")
    if output is None:
        output = torch.empty(shape, dtype=torch.bfloat16, device=dev)
    elif output.shape != shape or output.dtype != torch.bfloat16:
        raise ValueError(f"output must be bfloat16 {tuple(shape)}, got {output.dtype} {tuple(output.shape)}")
    else:
        _written(output, "output", 2)
    if B == 0:
        return output
    q4, tables = _rows(q4, 8), tables.contiguous()
    out4 = output if output.dim() == 4 else output.unsqueeze(1)
    args = L.SharedPrefixArgs(
        q4.data_ptr(), _strides(q4, 3), output.data_ptr(), _strides(out4, 3), K_cache.data_ptr(), V_cache.data_ptr(),
        _strides(K_cache, 3), _strides(V_cache, 3), num_blocks, block_len, L.KV_FP8 if fp8 else 0,
        L.ptr(prefix_tables), L.ptr(prefix_lens), L.ptr(prefix_starts), tables.data_ptr(), lens.data_ptr(),
        G, prefix_tables.shape[1] if G else 0, tables.shape[1],
        float(softmax_scale) if softmax_scale is not None else 1.0 / math.sqrt(d), L.ptr(sink), B, S_tkg, nq, nkv, d)
    lib = L.load()
    with L.on_device(dev):
        ws = torch.empty(lib.mkd_shared_prefix_workspace_bytes(args), dtype=torch.uint8, device=dev)
        rc = lib.mkd_attention_shared_prefix(args, ws.data_ptr(), ws.numel(), L.stream_ptr(dev))
        L.check(rc, "attention_shared_prefix")
    return output
