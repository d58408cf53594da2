"""The gated MoE layer and its gradients from their definitions in 64 bits, with error bounds for a bf16 kernel.

`gated_layer` is the definition (differentiable). `gated_reference` restates forward and backward stage by stage and
carries, next to every value, how far a computation may be off that accumulates in fp32 and rounds to bf16 where the
kernels do: a rounding is off by at most half a step (bf16: 2^-8 of the value), a sum of n products in fp32 by at most
n 2^-24 of the sum of their magnitudes, and errors travel through products by the magnitudes they are multiplied with.
"""

from __future__ import annotations

import math

import torch

HALF_BF16 = 2.0**-8
HALF_FP32 = 2.0**-24
# The kernels evaluate exp, the reciprocal and erf (absolute error 1.5e-7) approximately: at most this much of |v| off.
ACT_ERROR = 1e-6
CURVATURE = 0.8  # |act''| is at most 0.5 (SiLU) and 2 phi(0) = 0.798 (GELU)


def activation(v: torch.Tensor, name: str) -> torch.Tensor:
    if name == "silu":
        return v / (1 + torch.exp(-v))
    return 0.5 * v * (1 + torch.erf(v / math.sqrt(2)))


def slope(v: torch.Tensor, name: str) -> torch.Tensor:
    if name == "silu":
        s = 1 / (1 + torch.exp(-v))
        return s * (1 + v * (1 - s))
    return 0.5 * (1 + torch.erf(v / math.sqrt(2))) + v * torch.exp(-0.5 * v * v) / math.sqrt(2 * math.pi)


def gated_layer(x, expert_idx, gate, w_gate, w_up, w_down, act: str = "silu") -> torch.Tensor:
    """out[t] = sum_j gate[t, j] (act(x Wg) * (x Wu)) Wd with the weights of expert_idx[t, j]; ids outside the
    experts are skipped. In the type of its inputs."""
    out = torch.zeros_like(x)
    for e in range(w_gate.shape[0]):
        t, j = torch.nonzero(expert_idx == e, as_tuple=True)
        if t.numel():
            h = activation(x[t] @ w_gate[e], act) * (x[t] @ w_up[e])
            out = out.index_add(0, t, gate[t, j, None] * (h @ w_down[e]))
    return out


def gated_reference(x, expert_idx, gate, w_gate, w_up, w_down, act: str = "silu", grad_out=None) -> dict:
    """{name: (value, bound)} in float64 for out and, with grad_out, dx, dgate, dw_gate, dw_up, dw_down. Bounds leave
    out the last rounding (to the output's type): the caller adds it."""
    x, gate, w_gate, w_up, w_down = (t.double() for t in (x, gate, w_gate, w_up, w_down))
    num_experts, d_model, ffn_dim = w_gate.shape

    def zeros(*shape):
        return torch.zeros(*shape, dtype=torch.float64, device=x.device)

    out, out_b = zeros(*x.shape), zeros(*x.shape)
    if grad_out is not None:
        go = grad_out.double()
        names = {"dx": x, "dgate": gate, "dw_gate": w_gate, "dw_up": w_up, "dw_down": w_down}
        val = {n: torch.zeros_like(t) for n, t in names.items()}
        bnd = {n: torch.zeros_like(t) for n, t in names.items()}
    for e in range(num_experts):
        t, j = torch.nonzero(expert_idx == e, as_tuple=True)
        if not t.numel():
            continue
        xs, wg, wu, wd, w = x[t], w_gate[e], w_up[e], w_down[e], gate[t, j, None]
        g, u = xs @ wg, xs @ wu
        g_b, u_b = (d_model * HALF_FP32 * (xs.abs() @ m.abs()) for m in (wg, wu))
        a, s = activation(g, act), slope(g, act)
        h = a * u
        a_b = 1.13 * g_b + ACT_ERROR * g.abs()  # |act'| <= 1.13
        h_b = a_b * u.abs() + a.abs() * u_b + HALF_BF16 * h.abs()
        y = h @ wd
        y_b = h_b @ wd.abs() + ffn_dim * HALF_FP32 * (h.abs() @ wd.abs())
        out.index_add_(0, t, w * y)
        out_b.index_add_(0, t, w.abs() * (y_b + 4 * HALF_FP32 * y.abs()))
        if grad_out is None:
            continue
        # G and U are read back as bf16.
        g_b, u_b = g_b + HALF_BF16 * g.abs(), u_b + HALF_BF16 * u.abs()
        a_b = 1.13 * g_b + ACT_ERROR * g.abs()
        s_b = CURVATURE * g_b + ACT_ERROR * (1 + g.abs())
        do = go[t]
        val["dgate"][t, j] = (do * y).sum(1)
        bnd["dgate"][t, j] = (do.abs() * y_b + d_model * HALF_FP32 * (do * y).abs()).sum(1)
        wdo = w * do  # held as bf16 for dw_down; dh takes the unscaled rows and w in fp32
        dh = wdo @ wd.T
        dh_b = (d_model + 1) * HALF_FP32 * (wdo.abs() @ wd.abs().T)
        du, dg = dh * a, dh * u * s
        du_b = dh_b * a.abs() + dh.abs() * a_b + HALF_BF16 * du.abs()
        dg_b = dh_b * (u * s).abs() + dh.abs() * (u_b * s.abs() + u.abs() * s_b) + HALF_BF16 * dg.abs()
        n = t.numel()
        val["dw_down"][e] = h.T @ wdo
        bnd["dw_down"][e] = h_b.T @ wdo.abs() + (HALF_BF16 + n * HALF_FP32) * (h.abs().T @ wdo.abs())
        for name, d, d_b, wt in (("dw_gate", dg, dg_b, wg), ("dw_up", du, du_b, wu)):
            val[name][e] = xs.T @ d
            bnd[name][e] = xs.abs().T @ d_b + n * HALF_FP32 * (xs.abs().T @ d.abs())
        row = dg @ wg.T + du @ wu.T
        row_b = (dg_b @ wg.abs().T + du_b @ wu.abs().T
                 + 2 * ffn_dim * HALF_FP32 * (dg.abs() @ wg.abs().T + du.abs() @ wu.abs().T))
        val["dx"].index_add_(0, t, row)
        bnd["dx"].index_add_(0, t, row_b + 4 * HALF_FP32 * row.abs())
    result = {"out": (out, out_b)}
    if grad_out is not None:
        result.update({n: (val[n], bnd[n]) for n in val})
    return result
