"""The MoE layer with gated experts, for serving and for training.

    out[t] = sum over the token's picks of gate * (act(x w_gate[e]) * (x w_up[e])) w_down[e]

Routing, the gated SDD, DSD and the combine as in moe_forward; a decoding step (at most 128 token copies) streams the picked
experts' weights without a layout. The backward pass is a call of its own (moe_backward_gated), so that a training step can
be captured into a CUDA graph as it is; moe_gated() wraps the two for torch.autograd. No host sync anywhere.
"""

from __future__ import annotations

from dataclasses import dataclass
from typing import NamedTuple

import torch
from torch.autograd import forward_ad

from sparsebench_b200 import _C


@dataclass(frozen=True)
class GatedSaved:
    """What moe_forward_gated_saved keeps for moe_backward_gated: the inputs by reference (the gates and
    weights must still hold the same values then) and, in one buffer, the layout, x and Y in its order and the blocks of
    H, G and U (rows * (6 D + 6 F) bytes). state is None for an empty batch; stream is the raw handle of the stream that it
    was made on (None: not known)."""

    x: torch.Tensor
    expert_weight: torch.Tensor
    w_gate: torch.Tensor
    w_up: torch.Tensor
    w_down: torch.Tensor
    activation: str
    state: torch.Tensor | None
    stream: int | None = None


class GatedGrads(NamedTuple):
    x: torch.Tensor  # [T, D]
    expert_weight: torch.Tensor  # [T, k], in expert_weight's type
    w_gate: torch.Tensor  # [E, D, F]
    w_up: torch.Tensor  # [E, D, F]
    w_down: torch.Tensor  # [E, F, D]


def _check_shapes(x, expert_idx, expert_weight, w_gate, w_up, w_down) -> None:
    shape = w_gate.shape
    if len(shape) != 3 or w_up.shape != shape:
        raise ValueError(f"w_gate and w_up must be [E, D, F], got {tuple(shape)} and {tuple(w_up.shape)}")
    num_experts, d_model, ffn_dim = shape
    if tuple(w_down.shape) != (num_experts, ffn_dim, d_model):
        raise ValueError(f"w_down must be {(num_experts, ffn_dim, d_model)}, got {tuple(w_down.shape)}")
    x_shape, idx_shape = x.shape, expert_idx.shape
    if (len(x_shape) != 2 or x_shape[1] != d_model or len(idx_shape) != 2 or idx_shape != expert_weight.shape
            or idx_shape[0] != x_shape[0]):
        raise ValueError("x must be [T, D] and expert_idx / expert_weight [T, k]")


def _forward(x, expert_idx, expert_weight, w_gate, w_up, w_down, activation, keep):
    _check_shapes(x, expert_idx, expert_weight, w_gate, w_up, w_down)
    if expert_idx.numel() == 0:  # host-known size: nothing routed anywhere
        _C.check_gated_inputs(x, expert_idx, expert_weight, w_gate, w_up, w_down, activation)
        return torch.zeros_like(x), None
    return _C.moe_gated_forward_cuda(x, expert_idx, expert_weight, w_gate, w_up, w_down, activation, keep)


def moe_forward_gated(
    x: torch.Tensor,
    expert_idx: torch.Tensor,
    expert_weight: torch.Tensor,
    w_gate: torch.Tensor,
    w_up: torch.Tensor,
    w_down: torch.Tensor,
    activation: str = "silu",
) -> torch.Tensor:
    """x [T, D], expert_idx / expert_weight [T, k], w_gate and w_up [E, D, F], w_down [E, F, D] -> [T, D]; bf16 (gates
    bf16 or fp32), fp32 accumulation inside the kernels, D and F multiples of 128. activation: "silu" (SwiGLU experts)
    or "gelu" (erf form). An expert id outside [0, E) is skipped, as in moe_forward. Keeps
    nothing for a gradient: see moe_gated."""
    return _forward(x, expert_idx, expert_weight, w_gate, w_up, w_down, activation, False)[0]


def moe_forward_gated_saved(
    x: torch.Tensor,
    expert_idx: torch.Tensor,
    expert_weight: torch.Tensor,
    w_gate: torch.Tensor,
    w_up: torch.Tensor,
    w_down: torch.Tensor,
    activation: str = "silu",
) -> tuple[torch.Tensor, GatedSaved]:
    """moe_forward_gated that also returns what moe_backward_gated needs."""
    out, state = _forward(x, expert_idx, expert_weight, w_gate, w_up, w_down, activation, True)
    stream = None if state is None else _C._raw_stream(x.get_device())
    return out, GatedSaved(x, expert_weight, w_gate, w_up, w_down, activation, state, stream)


def moe_backward_gated(grad_out: torch.Tensor, saved: GatedSaved) -> GatedGrads:
    """The gradients of everything moe_forward_gated_saved took, from the gradient of its output [T, D] (bf16). May be
    called more than once, and on another stream than the forward call's after waiting for it. Sums over rows are in a
    fixed order: the same inputs give the same bits."""
    s = saved
    _check_shapes(s.x, s.expert_weight, s.expert_weight, s.w_gate, s.w_up, s.w_down)
    if grad_out.shape != s.x.shape:
        raise ValueError(f"grad_out must be {tuple(s.x.shape)}, got {tuple(grad_out.shape)}")
    if s.state is None:
        return GatedGrads(*(torch.zeros_like(t) for t in (s.x, s.expert_weight, s.w_gate, s.w_up, s.w_down)))
    return GatedGrads(*_C.moe_gated_backward_cuda(grad_out, s.x, s.expert_weight, s.w_gate, s.w_up, s.w_down, s.state,
                                                  s.activation, s.stream))


class _GatedMoE(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, expert_idx, expert_weight, w_gate, w_up, w_down, activation):
        out, saved = moe_forward_gated_saved(x, expert_idx, expert_weight, w_gate, w_up, w_down, activation)
        # Autograd checks the inputs for in-place changes; the state, most of the layer's memory, goes with them: freed
        # by the backward pass, and in the hands of saved_tensors_hooks (offloading, checkpointing).
        ctx.save_for_backward(x, expert_weight, w_gate, w_up, w_down, saved.state)
        ctx.activation, ctx.stream = activation, saved.stream
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_out):
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("the autograd form of the gated layer cannot be captured into a CUDA graph: "
                               "capture moe_forward_gated_saved and moe_backward_gated")
        *inputs, state = ctx.saved_tensors
        grad_out = grad_out.contiguous()
        if grad_out.data_ptr() % 16 != 0:  # a view of a larger gradient, as torch.cat's backward pass hands out
            grad_out = grad_out.clone()
        grads = moe_backward_gated(grad_out, GatedSaved(*inputs, ctx.activation, state, ctx.stream))
        return grads.x, None, grads.expert_weight, grads.w_gate, grads.w_up, grads.w_down, None


def moe_gated(
    x: torch.Tensor,
    expert_idx: torch.Tensor,
    expert_weight: torch.Tensor,
    w_gate: torch.Tensor,
    w_up: torch.Tensor,
    w_down: torch.Tensor,
    activation: str = "silu",
) -> torch.Tensor:
    """moe_forward_gated for torch.autograd: differentiable in x, expert_weight and the three weights (once, and by
    backward passes: an input that carries a forward-mode tangent is refused). Its backward pass refuses to run under CUDA graph capture: capture the two explicit calls instead."""
    leaves = (x, expert_weight, w_gate, w_up, w_down)
    if any(forward_ad.unpack_dual(t).tangent is not None for t in leaves):  # of any dual level; requires_grad is not set there
        raise NotImplementedError("moe_gated has no forward-mode derivative (make_dual, func.jvp): it is differentiable by "
                                  "backward passes only")
    if not torch.is_grad_enabled() or not any(t.requires_grad for t in leaves):
        return moe_forward_gated(x, expert_idx, expert_weight, w_gate, w_up, w_down, activation)  # nothing to keep
    return _GatedMoE.apply(x, expert_idx, expert_weight, w_gate, w_up, w_down, activation)
