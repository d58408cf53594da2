"""A projection with per-token low-rank adapters from its definition in 64 bits, with the error bound of a kernel that
accumulates in fp32 and holds x A^T as one bf16 (bf16 results) or as three of them (fp32 results)."""

from __future__ import annotations

import torch

HALF_FP32 = 2.0**-24


def lora_reference(x, weight, lora_a, lora_b, adapter_idx, scale=None, fp32: bool = False):
    """(value, bound) [T, N] in float64; the bound leaves out the last rounding."""
    x, weight = x.double(), weight.double()
    d_model, rank = x.shape[1], lora_a.shape[1]
    out = x @ weight
    bound = (d_model + 3 * rank) * HALF_FP32 * (x.abs() @ weight.abs())
    # Half a bf16 step of x A^T, or of what is left over the second time.
    held = 2.0**-24 if fp32 else 2.0**-8
    for a in range(lora_a.shape[0]):
        rows = torch.nonzero(adapter_idx == a).flatten()
        if not rows.numel():
            continue
        s = 1.0 if scale is None else float(scale[a])
        la, lb = lora_a[a].double(), lora_b[a].double()
        v = s * (x[rows] @ la.T)
        v_abs = abs(s) * (x[rows].abs() @ la.abs().T)
        v_bound = (d_model + 2) * HALF_FP32 * v_abs + held * v.abs()
        out[rows] += v @ lb
        bound[rows] += v_bound @ lb.abs() + (d_model + 3 * rank) * HALF_FP32 * (v.abs() @ lb.abs())
    return out, bound
