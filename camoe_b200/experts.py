"""The expert layer that follows the time mix: tokens to their experts and back.

CaMoE sends each token to its top-2 experts (camoe/system.py:263-297, by
boolean masks over every expert) and each RWKV expert is a squared-ReLU
feed-forward product (camoe/experts.py).  Here the tokens' slots are sorted by
expert once, every expert works on its own contiguous rows, and the rows go
back to their tokens with their weights:

    xs, plan = expert_dispatch(x, index, n_experts)   # x [N, C], index [N, k]
    ys = expert_ffn(xs, w_up, w_down, plan.offsets)   # w_up [E, F, C], w_down [E, C, F]
    out = expert_combine(ys, weight, plan)            # weight [N, k] fp32

All three are differentiable once, in reverse mode (the index is not), and launch
on the current CUDA stream without synchronising.  A slot whose index is outside [0, n_experts) is
unused: it reads nothing and contributes nothing, and a token without used
slots gets zeros.  ``ExpertLayer`` is the module over them.  The C ABI is
include/camoe_experts.h.
"""
from __future__ import annotations

from typing import NamedTuple

import torch
import torch.nn as nn

from ._lib import ERR_ALIGNMENT, check, torch_ops
from .ops import dtype_code

_torch_ops = torch_ops()

MAX_EXPERTS, MAX_SLOTS = 1024, 64


class ExpertPlan(NamedTuple):
    """Where each slot's row stands (int32).  ``offsets`` [E + 1]: expert e owns
    rows [offsets[e], offsets[e + 1]); ``position`` [N, k]: the row of each
    slot, -1 for an unused one; ``source`` [N k]: the slot n k + j of each row,
    -1 behind offsets[E]."""
    offsets: torch.Tensor
    position: torch.Tensor
    source: torch.Tensor


def _check(t: torch.Tensor, name: str, shape, dtype, device) -> None:
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor (the op has no CPU path)")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, expected {device}")
    if t.dtype != dtype:
        raise TypeError(f"{name} has dtype {t.dtype}, expected {dtype}")
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {tuple(shape)}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")


def _check_aligned(*ts: torch.Tensor) -> None:
    if any(t.data_ptr() % 16 for t in ts):
        check(ERR_ALIGNMENT)


# The calls check their arguments, allocate, launch and make the autograd nodes
# in csrc/torch_ops.cpp; where that refuses, the functions named _refuse_* here
# raise what is wrong.


def _refuse_dispatch(x, index, E):
    if x.dim() != 2 or index.dim() != 2:
        raise ValueError(f"expected x [N, C] and index [N, k], got {tuple(x.shape)} and {tuple(index.shape)}")
    dtype_code(x.dtype)
    _check(x, "x", x.shape, x.dtype, x.device)
    if index.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"index must be int32 or int64, got {index.dtype}")
    _check(index, "index", (x.shape[0], index.shape[1]), index.dtype, x.device)
    raise ValueError(f"1 to {MAX_EXPERTS} experts and 1 to {MAX_SLOTS} slots per token, got {E} and {index.shape[1]}")


def expert_dispatch(x: torch.Tensor, index: torch.Tensor, n_experts: int):
    """Tokens sorted by expert: x [N, C] (bf16 or fp32), index [N, k] (int32 or
    int64; anything outside [0, n_experts) is an unused slot).  Returns (xs
    [N k, C], plan): the used slots' rows in the order of their experts, a
    slot's own order within an expert, and zeros in the rows of the unused ones
    behind them.  Differentiable in x."""
    out = _torch_ops.dispatch(x, index, n_experts)
    if out is None:
        _refuse_dispatch(x, index, n_experts)
    xs, offsets, position, source = out
    return xs, ExpertPlan(offsets, position, source)


def _refuse_combine(ys, weight, plan):
    dtype_code(ys.dtype)
    if ys.dim() != 2:
        raise ValueError(f"expected ys [N k, C], got {tuple(ys.shape)}")
    if plan.position.dim() != 2 or plan.offsets.dim() != 1 or plan.offsets.shape[0] < 2:
        raise ValueError("a plan has offsets [E + 1], position [N, k] and source [N k]")
    N, k = plan.position.shape
    _check(ys, "ys", (N * k, ys.shape[1]), ys.dtype, ys.device)
    _check(weight, "weight", (N, k), torch.float32, ys.device)
    for name, shape in (("offsets", plan.offsets.shape), ("position", (N, k)), ("source", (N * k,))):
        _check(getattr(plan, name), f"plan.{name}", shape, torch.int32, ys.device)
    raise ValueError(f"1 to {MAX_EXPERTS} experts and 1 to {MAX_SLOTS} slots per token, got {plan.offsets.shape[0] - 1} and {k}")


def expert_combine(ys: torch.Tensor, weight: torch.Tensor, plan: ExpertPlan) -> torch.Tensor:
    """The experts' rows back to their tokens: out[n] = sum over j of weight[n, j]
    ys[position[n, j]], summed in fp32 and rounded once.  ys [N k, C] (bf16 or
    fp32), weight [N, k] fp32.  Differentiable in ys and weight."""
    out = _torch_ops.combine(ys, weight, *plan)
    if out is None:
        _refuse_combine(ys, weight, plan)
    return out


def _refuse_ffn(xs, w_up, w_down, offsets):
    if xs.dim() != 2 or w_up.dim() != 3:
        raise ValueError(f"expected xs [R, C] and w_up [E, F, C], got {tuple(xs.shape)} and {tuple(w_up.shape)}")
    R, C = xs.shape
    E, F, _ = w_up.shape
    dev, bf = xs.device, torch.bfloat16
    _check(xs, "xs", (R, C), bf, dev)
    _check(w_up, "w_up", (E, F, C), bf, dev)
    _check(w_down, "w_down", (E, C, F), bf, dev)
    _check(offsets, "offsets", (E + 1,), torch.int32, dev)
    _check_aligned(xs, w_up, w_down)
    raise ValueError(f"1 to {MAX_EXPERTS} experts and widths that are positive multiples of 8, got E = {E}, "
                     f"C = {C}, F = {F}")


def expert_ffn(xs: torch.Tensor, w_up: torch.Tensor, w_down: torch.Tensor, offsets: torch.Tensor) -> torch.Tensor:
    """Each expert's squared-ReLU product over its own rows:
    ys[p] = w_down[e] relu(w_up[e] xs[p])^2 for p in [offsets[e], offsets[e + 1]),
    zeros behind offsets[E].  xs [R, C], w_up [E, F, C], w_down [E, C, F], all
    bf16 (C and F multiples of 8); offsets [E + 1] int32, non-decreasing from 0.
    Sums are fp32; the hidden rows and, in the backward, the gradient before
    the activation are rounded to bf16, the type of the tensor cores' operands.
    Differentiable in xs, w_up and w_down."""
    out = _torch_ops.ffn(xs, w_up, w_down, offsets)
    if out is None:
        _refuse_ffn(xs, w_up, w_down, offsets)
    return out


class ExpertLayer(nn.Module):
    """E squared-ReLU experts of width C and hidden width F behind a router's choice.

    ``forward(x, index, weight)``: x [..., C], index [..., k] the chosen experts
    (anything outside [0, E) is an unused slot) and weight [..., k] fp32; returns
    the weighted sum of the chosen experts' outputs in x's dtype.  The products
    run in bf16: fp32 parameters are cast per call, as ``RWKV7TimeMix`` casts
    its own (gradients arrive in fp32); convert the module with ``.bfloat16()``
    to serve without that (the same outputs, bit for bit, where bf16 holds the
    values)."""

    def __init__(self, n_embd: int, n_experts: int, hidden: int | None = None):
        super().__init__()
        hidden = 4 * n_embd if hidden is None else hidden
        if n_embd % 8 or hidden % 8 or min(n_embd, hidden) <= 0:
            raise ValueError(f"widths must be positive multiples of 8, got {n_embd} and {hidden}")
        if not 1 <= n_experts <= MAX_EXPERTS:
            raise ValueError(f"1 to {MAX_EXPERTS} experts, got {n_experts}")
        self.n_experts = n_experts
        self.w_up = nn.Parameter(torch.empty(n_experts, hidden, n_embd).uniform_(-0.5 * n_embd ** -0.5,
                                                                                 0.5 * n_embd ** -0.5))
        self.w_down = nn.Parameter(torch.zeros(n_experts, n_embd, hidden))

    def forward(self, x: torch.Tensor, index: torch.Tensor, weight: torch.Tensor) -> torch.Tensor:
        bf = torch.bfloat16
        rows = x.reshape(-1, x.shape[-1]).to(bf).contiguous()
        k = index.shape[-1]
        xs, plan = expert_dispatch(rows, index.reshape(-1, k).contiguous(), self.n_experts)
        ys = expert_ffn(xs, self.w_up.to(bf), self.w_down.to(bf), plan.offsets)
        out = expert_combine(ys, weight.reshape(-1, k).float().contiguous(), plan)
        return out.view(x.shape).to(x.dtype)
