"""Attention over whole prompts: what stands between the rotary embedding and the output projection while a prompt is
taken in.  (The reference calls a library's attention there, modeling/llama/llama_qblocks.py:104-150.)  For single tokens, over
the 4-bit cache: quantize.quant_kv_cache."""
from __future__ import annotations

import torch

from . import ops


def prompt_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_q: torch.Tensor, cu_k: torch.Tensor | None = None, *,
                     causal: bool = True, scale: float | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """softmax(scale q k^T) v within each of several sequences packed behind each other.

    q [tokens, q heads, d], k [tokens, kv heads, d], v [tokens, kv heads, e]: fp16, d and e from 1 to 128 (pruned heads
    included, e may differ from d), any strides but a unit one along the width, so that the column ranges of a fused
    projection's output are taken as they are: `qkv(x)` of a W4A16FusedLinear, each result viewed as [tokens, heads, width].
    cu_q int32 [sequences + 1] on the GPU: sequence i has the rows cu_q[i] .. cu_q[i + 1] (KVStep.cu is such a tensor).
    cu_k: the same for k and v where they differ, as when a prompt's earlier pieces come from W4KVCache.load; the causal mask is then
    aligned at the ends.  A row that sees nothing is 0.  Nothing is recorded for autograd."""
    return ops.prompt_attention(q, k, v, cu_q, cu_k, causal=causal, scale=scale, out=out)
