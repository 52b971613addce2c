"""sample_tokens: the next tokens from logits and given random numbers (beside the greedy choice
of the decode step's epilogue; the reference samples greedily, main.py:390-398)."""
from __future__ import annotations

import math
from typing import Optional, Union

import torch

from . import _lib as L

Setting = Union[float, int, torch.Tensor]


def _setting(x: Setting, name: str, B: int, dev, lo: float, hi: float):
    """(value for all rows, [B] tensor or None)"""
    if isinstance(x, torch.Tensor):
        if x.device != dev or x.dim() != 1 or x.numel() != B:
            raise ValueError(f"{name} must be a number or [B={B}] on {dev}, got {tuple(x.shape)} on {x.device}")
        if name == "top_k":
            if x.dtype not in (torch.int32, torch.int64):
                raise ValueError(f"top_k must be int32 or int64, got {x.dtype}")
            x = x if x.dtype == torch.int32 else x.clamp(0, 2 ** 31 - 1).to(torch.int32)
        elif not x.is_floating_point():
            raise ValueError(f"{name} must be floating point, got {x.dtype}")
        else:
            x = x.float()
        return 0, x.contiguous()
    if not lo <= x <= hi:      # (a NaN too)
        raise ValueError(f"{name} must be in [{lo}, {hi}], got {x}")
    return (min(int(x), 2 ** 31 - 1) if name == "top_k" else float(x)), None


def sample_tokens(logits: torch.Tensor, uniforms: torch.Tensor, temperature: Setting = 1.0, top_k: Setting = 0,
                  top_p: Setting = 1.0, min_p: Setting = 0.0, output: Optional[torch.Tensor] = None):
    """One token per row of logits [B, V] (bf16 or fp32, V <= 2^20); returns (tokens [B] int32,
    logprobs [B] fp32).

    A row's tokens in order of falling logit, ties with the lowest index first, have the masses
    e_j = exp((l_j - l_0) / temperature).  top_k > 0 keeps the first top_k; top_p < 1 keeps, of those,
    the tokens before which less than top_p of their mass lies; min_p keeps the ones with e_j >= min_p;
    the first token always stays.  The row's token is the first kept one whose cumulative mass exceeds
    uniforms[b] (fp32 in [0, 1), the caller's random number) times the kept mass, its logprob the
    logarithm of its share of it.  temperature 0 takes the first token.  Each setting is a number, or
    a [B] tensor in device memory (read there: the call can be captured).  -inf and NaN logits are
    never chosen; a row with nothing to choose gives -1 and -inf.  The result does not depend on the
    order of any addition: equal inputs give equal tokens.  `output`: an int32 [B] tensor for the tokens.
    """
    index = L.gpu_index(logits=logits, uniforms=uniforms, output=output)
    dev = logits.device
    if logits.dim() != 2 or logits.dtype not in (torch.bfloat16, torch.float32):
        raise ValueError(f"logits must be bfloat16 or float32 [B, V], got {logits.dtype} {tuple(logits.shape)}")
    B, V = logits.shape
    if not 1 <= V <= 1 << 20:
        raise ValueError(f"V must be in [1, 2^20], got {V}")
    if uniforms.dtype != torch.float32 or uniforms.dim() != 1 or uniforms.numel() != B:
        raise ValueError(f"uniforms must be float32 [B={B}], got {uniforms.dtype} {tuple(uniforms.shape)}")
    t, t_rows = _setting(temperature, "temperature", B, dev, 0.0, 3.4e38)
    k, k_rows = _setting(top_k, "top_k", B, dev, 0, math.inf)
    p, p_rows = _setting(top_p, "top_p", B, dev, 0.0, 1.0)
    m, m_rows = _setting(min_p, "min_p", B, dev, 0.0, 1.0)
    if output is None:
        output = torch.empty(B, dtype=torch.int32, device=dev)
    elif output.dtype != torch.int32 or tuple(output.shape) != (B,) or not output.is_contiguous():
        raise ValueError(f"output must be a contiguous int32 [{B}] tensor")
    logprobs = torch.empty(B, dtype=torch.float32, device=dev)
    if B == 0:
        return output, logprobs
    if V > 1 and logits.stride(1) != 1:
        logits = logits.contiguous()
    uniforms = uniforms.contiguous()
    args = L.SampleArgs(
        logits.data_ptr(), L.DT_F32 if logits.dtype == torch.float32 else L.DT_BF16, logits.stride(0) if B > 1 else 0,
        uniforms.data_ptr(), t, p, m, k, L.ptr(t_rows), L.ptr(p_rows), L.ptr(m_rows), L.ptr(k_rows),
        output.data_ptr(), logprobs.data_ptr(), B, V)
    lib = L.load()
    n = lib.mkd_sample_workspace_bytes(B, V)
    ws = torch.empty(n, dtype=torch.uint8, device=dev)
    L.call(lib.mkd_sample_tokens, "sample_tokens", index, args, ws.data_ptr(), n)
    return output, logprobs
