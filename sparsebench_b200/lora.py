"""Projections beside the layer (its router's among them) with the low-rank adapters of many requests at once."""

from __future__ import annotations

import torch

from sparsebench_b200 import _C


def lora_linear(
    x: torch.Tensor,
    weight: torch.Tensor,
    lora_a: torch.Tensor,
    lora_b: torch.Tensor,
    adapter_idx: torch.Tensor,
    scale: torch.Tensor | None = None,
    out_dtype: torch.dtype | None = None,
) -> torch.Tensor:
    """out[t] = x[t] @ weight + scale[a] * (x[t] @ lora_a[a].T) @ lora_b[a], a = adapter_idx[t].

    x [T, D] and weight [D, N] bf16; lora_a [L, r, D] and lora_b [L, r, N] bf16, the r directions of an adapter as
    rows (pad a smaller rank with zero rows); adapter_idx [T] int32 or int64, a token whose id is outside [0, L)
    has no adapter; scale [L] fp32 or None (1). D, N and r are multiples of 8, r at most 128. out_dtype bfloat16
    (default) or float32, e.g. for router logits that go into route(). Tokens may come in any order; a batch of whole
    requests is the fast case. A token's output depends on its own adapter alone, also where another one holds
    infinities or NaN. No host sync; no gradient (adapters are served, not trained, here)."""
    return _C.lora_linear_cuda(x, weight, lora_a, lora_b, adapter_idx, scale,
                               torch.bfloat16 if out_dtype is None else out_dtype)
