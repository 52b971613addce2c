"""Float64 restatements (CPU) of the operators for serving many samples of a few prompts."""
from __future__ import annotations

import math

import numpy as np
import torch

F64 = torch.float64


def kv_append_rope(q, k, v, cos, sin, positions, K_cache, V_cache, slots, q_norm=None, k_norm=None, eps=1e-6,
                   k_scale=None, v_scale=None):
    """(q, K, V) in float64: the values before their rounding to bf16 / e4m3, on copies of the caches."""
    T, nq, d = q.shape
    K, V = K_cache.to(F64).clone(), V_cache.to(F64).clone()
    num_blocks, block_len = K.shape[:2]
    out = torch.zeros(T, nq, d, dtype=F64)

    def head(x, weight, t):
        x = x.to(F64).clone()
        if weight is not None:
            x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * weight.reshape(-1).to(F64)
        if cos is not None:
            h = cos.shape[1]
            c, s = cos[t].to(F64), sin[t].to(F64)
            a, b = x[..., :h].clone(), x[..., h:2 * h].clone()
            x[..., :h], x[..., h:2 * h] = a * c - b * s, b * c + a * s
        return x

    for t in range(T):
        p = int(positions[t]) if cos is not None else 0
        if cos is not None and not 0 <= p < cos.shape[0]:
            continue
        out[t] = head(q[t], q_norm, p)
        r = int(slots[t])
        if 0 <= r < num_blocks * block_len:
            kt, vt = head(k[t], k_norm, p), v[t].to(F64)
            if k_scale is not None:
                kt, vt = (kt * k_scale).clamp(-240, 240), (vt * v_scale).clamp(-240, 240)
            K[r // block_len, r % block_len], V[r // block_len, r % block_len] = kt, vt
    return out, K, V


def attention_shared_prefix(q, K_cache, V_cache, prefix_tables, prefix_lens, prefix_starts, tables, lens, scale,
                            sink=None):
    """(out, mean |v| under each row's weights), float64 [B, S, nq, d]; q [B, S, nq, d]."""
    B, S, nq, d = q.shape
    num_blocks, block_len, nkv = K_cache.shape[:3]
    gqa = nq // nkv

    def rows(cache, table, n):
        n = max(0, min(n, len(table) * block_len))
        out = torch.zeros(n, nkv, d, dtype=F64)
        for t in range(n):
            blk = int(table[t // block_len])
            if 0 <= blk < num_blocks:
                out[t] = cache[blk, t % block_len].to(F64)
        return out

    out, mean = torch.zeros(B, S, nq, d, dtype=F64), torch.zeros(B, S, nq, d, dtype=F64)
    kept = {}
    for b in range(B):
        k, v = rows(K_cache, tables[b], int(lens[b])), rows(V_cache, tables[b], int(lens[b]))
        own = k.shape[0]
        for g in range(0 if prefix_lens is None else len(prefix_lens)):
            if int(prefix_starts[g]) <= b < int(prefix_starts[g + 1]):
                if g not in kept:
                    kept[g] = (rows(K_cache, prefix_tables[g], int(prefix_lens[g])),
                               rows(V_cache, prefix_tables[g], int(prefix_lens[g])))
                k, v = torch.cat([kept[g][0], k]), torch.cat([kept[g][1], v])
                break
        for s in range(S):
            n = k.shape[0] - own + max(0, own - (S - 1 - s))
            for h in range(nq):
                kk, vv = k[:n, h // gqa], v[:n, h // gqa]
                z = kk @ q[b, s, h].to(F64) * scale
                top = max([float(z.max())] if n else [-math.inf], default=-math.inf)
                if sink is not None:
                    top = max(top, float(sink[h]))
                if top == -math.inf:
                    continue
                e = torch.exp(z - top)
                total = e.sum() + (math.exp(float(sink[h]) - top) if sink is not None else 0.0)
                out[b, s, h], mean[b, s, h] = e @ vv / total, e @ vv.abs() / total
    return out, mean


def sample_tokens(logits, uniforms, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(tokens, logprobs) as numpy arrays; settings are numbers or sequences per row."""
    x = logits.to(F64).numpy()
    B = x.shape[0]
    f32 = lambda v: np.asarray(np.broadcast_to(np.asarray(v, np.float32), (B,)), np.float64)
    temp, pp, mp, u = f32(temperature), f32(top_p), f32(min_p), f32(uniforms)
    kk = np.broadcast_to(np.asarray(top_k), (B,))
    tokens, logprobs = np.full(B, -1, np.int64), np.full(B, -np.inf)
    for b in range(B):
        live = np.flatnonzero(x[b] > -np.inf)            # (NaN compares false)
        if not live.size:
            continue
        order = live[np.argsort(-x[b][live], kind="stable")]
        if not temp[b] > 0:
            tokens[b], logprobs[b] = order[0], 0.0
            continue
        if kk[b] > 0:
            order = order[:kk[b]]
        y, top = x[b][order], x[b][order[0]]
        e = np.where(y == top, 1.0, np.exp(np.where(y == top, 0.0, (y - top) / temp[b]))) if np.isfinite(top) \
            else (y == top).astype(np.float64)
        if pp[b] < 1:
            before = np.concatenate([[0.0], np.cumsum(e)[:-1]])
            keep = before < pp[b] * e.sum()
            keep[0] = True
            e = e[:np.count_nonzero(keep)]
        e = e[:max(1, np.count_nonzero(e >= mp[b]))]
        cum = np.cumsum(e)
        j = min(int(np.searchsorted(cum, u[b] * cum[-1], side="right")), e.size - 1)
        tokens[b], logprobs[b] = order[j], math.log(e[j] / cum[-1])
    return tokens, logprobs
