"""sample_tokens: the next tokens from logits and given random numbers (beside the greedy choice
of the decode step's epilogue; the reference samples greedily, main.py:390-398)."""
from __future__ import annotations

from typing import Optional, Union

import torch

from . import _lib as L

Setting = Union[float, int, torch.Tensor]


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
    return L.native().sample_tokens(logits, uniforms, temperature, top_k, top_p, min_p, output)
