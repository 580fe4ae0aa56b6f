"""The expert layer that follows the time mix: tokens to their experts and back.

CaMoE sends each token to its top-2 experts (camoe/system.py:263-297, by
boolean masks over every expert) and each RWKV expert is a squared-ReLU
feed-forward product (camoe/experts.py).  Here the tokens' slots are sorted by
expert once, every expert works on its own contiguous rows, and the rows go
back to their tokens with their weights:

    xs, plan = expert_dispatch(x, index, n_experts)   # x [N, C], index [N, k]
    ys = expert_ffn(xs, w_up, w_down, plan.offsets)   # w_up [E, F, C], w_down [E, C, F]
    out = expert_combine(ys, weight, plan)            # weight [N, k] fp32

All three are differentiable (the index is not) and launch on the current CUDA
stream without synchronising.  A slot whose index is outside [0, n_experts) is
unused: it reads nothing and contributes nothing, and a token without used
slots gets zeros.  ``ExpertLayer`` is the module over them.  The C ABI is
include/camoe_experts.h.
"""
from __future__ import annotations

from typing import NamedTuple

import torch
import torch.nn as nn

from . import _lib
from ._lib import check
from .ops import dtype_code

MAX_EXPERTS, MAX_SLOTS = 1024, 64


class ExpertPlan(NamedTuple):
    """Where each slot's row stands (int32).  ``offsets`` [E + 1]: expert e owns
    rows [offsets[e], offsets[e + 1]); ``position`` [N, k]: the row of each
    slot, -1 for an unused one; ``source`` [N k]: the slot n k + j of each row,
    -1 behind offsets[E]."""
    offsets: torch.Tensor
    position: torch.Tensor
    source: torch.Tensor


def _stream(t: torch.Tensor) -> int:
    """The current stream of t's device; a tenth of the host time of
    torch.cuda.current_stream(t.device).cuda_stream (0.1 against 2.3 us), which
    counts where a call is one small kernel."""
    return torch._C._cuda_getCurrentRawStream(t.get_device())


def _check(t: torch.Tensor, name: str, shape, dtype, device) -> None:
    if t.shape == shape and t.dtype is dtype and t.is_cuda and t.device == device and t.is_contiguous():
        return
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


def _check_plan(plan: ExpertPlan, device):
    if plan.position.dim() != 2 or plan.offsets.dim() != 1 or plan.offsets.shape[0] < 2:
        raise ValueError("a plan has offsets [E + 1], position [N, k] and source [N k]")
    N, k = plan.position.shape
    E = plan.offsets.shape[0] - 1
    _check(plan.offsets, "plan.offsets", (E + 1,), torch.int32, device)
    _check(plan.position, "plan.position", (N, k), torch.int32, device)
    _check(plan.source, "plan.source", (N * k,), torch.int32, device)
    return N, k, E


def _dispatch(x, index, E):
    N, C = x.shape
    k = index.shape[1]
    dev = x.device
    xs = torch.empty(N * k, C, dtype=x.dtype, device=dev)
    offsets = torch.empty(E + 1, dtype=torch.int32, device=dev)
    position = torch.empty(N, k, dtype=torch.int32, device=dev)
    source = torch.empty(N * k, dtype=torch.int32, device=dev)
    lib = _lib.lib()
    need = lib.camoe_ex_dispatch_work_bytes(N, k, E)
    work = torch.empty(need, dtype=torch.uint8, device=dev) if need else None  # none for few tokens
    check(lib.camoe_ex_dispatch(x.data_ptr(), dtype_code(x.dtype), index.data_ptr(), index.element_size(),
                                xs.data_ptr(), offsets.data_ptr(), position.data_ptr(), source.data_ptr(),
                                None if work is None else work.data_ptr(), need, N, k, E, C, _stream(x)))
    return xs, offsets, position, source


def _combine(rows, weight, position, C):
    N, k = position.shape
    out = torch.empty(N, C, dtype=rows.dtype, device=rows.device)
    check(_lib.lib().camoe_ex_combine(rows.data_ptr(), dtype_code(rows.dtype),
                                      None if weight is None else weight.data_ptr(), position.data_ptr(),
                                      out.data_ptr(), N, k, C, _stream(rows)))
    return out


class _DispatchFn(torch.autograd.Function):
    """The sorted rows; the plan, which has no gradient, goes out by ``plan`` (one
    output instead of four spares the engine's work on the other three)."""

    @staticmethod
    def forward(ctx, x, index, E, plan):
        xs, *ints = _dispatch(x, index, E)
        plan.extend(ints)
        ctx.save_for_backward(ints[1])
        return xs

    @staticmethod
    def backward(ctx, dxs):
        position, = ctx.saved_tensors
        return _combine(dxs.contiguous(), None, position, dxs.shape[1]), None, None, None


def expert_dispatch(x: torch.Tensor, index: torch.Tensor, n_experts: int):
    """Tokens sorted by expert: x [N, C] (bf16 or fp32), index [N, k] (int32 or
    int64; anything outside [0, n_experts) is an unused slot).  Returns (xs
    [N k, C], plan): the used slots' rows in the order of their experts, a
    slot's own order within an expert, and zeros in the rows of the unused ones
    behind them."""
    if x.dim() != 2 or index.dim() != 2:
        raise ValueError(f"expected x [N, C] and index [N, k], got {tuple(x.shape)} and {tuple(index.shape)}")
    N, C = x.shape
    k, E = index.shape[1], int(n_experts)
    dtype_code(x.dtype)
    _check(x, "x", (N, C), x.dtype, x.device)
    if index.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"index must be int32 or int64, got {index.dtype}")
    _check(index, "index", (N, k), index.dtype, x.device)
    if not 1 <= E <= MAX_EXPERTS or not 1 <= k <= MAX_SLOTS:
        raise ValueError(f"1 to {MAX_EXPERTS} experts and 1 to {MAX_SLOTS} slots per token, got {E} and {k}")
    if torch.is_grad_enabled() and x.requires_grad:
        plan = []
        xs = _DispatchFn.apply(x, index, E, plan)
    else:
        xs, *plan = _dispatch(x, index, E)
    return xs, ExpertPlan(*plan)


class _CombineFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ys, weight, offsets, position):
        ctx.save_for_backward(ys, weight, offsets, position)
        return _combine(ys, weight, position, ys.shape[1])

    @staticmethod
    def backward(ctx, dout):
        ys, weight, offsets, position = ctx.saved_tensors
        dout = dout.contiguous()
        N, k = position.shape
        C = ys.shape[1]
        dys = torch.empty_like(ys) if ctx.needs_input_grad[0] else None
        dw = torch.empty_like(weight) if ctx.needs_input_grad[1] else None
        check(_lib.lib().camoe_ex_combine_bwd(
            dout.data_ptr(), dtype_code(ys.dtype), ys.data_ptr(), weight.data_ptr(), offsets.data_ptr(),
            position.data_ptr(), None if dys is None else dys.data_ptr(), None if dw is None else dw.data_ptr(),
            N, k, offsets.shape[0] - 1, C, _stream(ys)))
        return dys, dw, None, None


def expert_combine(ys: torch.Tensor, weight: torch.Tensor, plan: ExpertPlan) -> torch.Tensor:
    """The experts' rows back to their tokens: out[n] = sum over j of weight[n, j]
    ys[position[n, j]], summed in fp32 and rounded once.  ys [N k, C] (bf16 or
    fp32), weight [N, k] fp32.  Differentiable in ys and weight."""
    dtype_code(ys.dtype)
    if ys.dim() != 2:
        raise ValueError(f"expected ys [N k, C], got {tuple(ys.shape)}")
    N, k, _ = _check_plan(plan, ys.device)
    _check(ys, "ys", (N * k, ys.shape[1]), ys.dtype, ys.device)
    _check(weight, "weight", (N, k), torch.float32, ys.device)
    if torch.is_grad_enabled() and (ys.requires_grad or weight.requires_grad):
        return _CombineFn.apply(ys, weight, plan.offsets, plan.position)
    return _combine(ys, weight, plan.position, ys.shape[1])


def _ffn(xs, w_up, w_down, offsets, low: bool):
    R, C = xs.shape
    E, F, _ = w_up.shape
    h = torch.empty(R, F, dtype=xs.dtype, device=xs.device)
    h_low = torch.empty(R, (F + 15) // 16 * 16, dtype=torch.int8, device=xs.device) if low else None
    ys = torch.empty(R, C, dtype=xs.dtype, device=xs.device)
    check(_lib.lib().camoe_ex_ffn_fwd(xs.data_ptr(), w_up.data_ptr(), w_down.data_ptr(), offsets.data_ptr(),
                                      h.data_ptr(), None if h_low is None else h_low.data_ptr(), ys.data_ptr(), R, E, C, F,
                                      _stream(xs)))
    return ys, h, h_low


class _FfnFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, xs, w_up, w_down, offsets):
        # h to 8 bits below bf16 where the backward takes its root
        ys, h, h_low = _ffn(xs, w_up, w_down, offsets, ctx.needs_input_grad[0] or ctx.needs_input_grad[1])
        ctx.save_for_backward(xs, w_up, w_down, offsets, h, h_low)
        return ys

    @staticmethod
    def backward(ctx, dys):
        xs, w_up, w_down, offsets, h, h_low = ctx.saved_tensors
        dys = dys.contiguous()
        R, C = xs.shape
        E, F, _ = w_up.shape
        need = ctx.needs_input_grad
        dxs, dw_up, dw_down = (torch.empty_like(t) if n else None for t, n in zip((xs, w_up, w_down), need))
        dpre = torch.empty_like(h) if need[0] or need[1] else None
        ptr = (lambda t: None if t is None else t.data_ptr())
        check(_lib.lib().camoe_ex_ffn_bwd(
            dys.data_ptr(), xs.data_ptr(), w_up.data_ptr(), w_down.data_ptr(), offsets.data_ptr(), h.data_ptr(),
            ptr(h_low), ptr(dpre), ptr(dxs), ptr(dw_up), ptr(dw_down), R, E, C, F, _stream(xs)))
        return dxs, dw_up, dw_down, None


def expert_ffn(xs: torch.Tensor, w_up: torch.Tensor, w_down: torch.Tensor, offsets: torch.Tensor) -> torch.Tensor:
    """Each expert's squared-ReLU product over its own rows:
    ys[p] = w_down[e] relu(w_up[e] xs[p])^2 for p in [offsets[e], offsets[e + 1]),
    zeros behind offsets[E].  xs [R, C], w_up [E, F, C], w_down [E, C, F], all
    bf16 (C and F multiples of 8); offsets [E + 1] int32, non-decreasing from 0.
    Sums are fp32; the hidden rows and, in the backward, the gradient before
    the activation are rounded to bf16, the type of the tensor cores' operands.
    Differentiable in xs, w_up and w_down."""
    if xs.dim() != 2 or w_up.dim() != 3:
        raise ValueError(f"expected xs [R, C] and w_up [E, F, C], got {tuple(xs.shape)} and {tuple(w_up.shape)}")
    R, C = xs.shape
    E, F, _ = w_up.shape
    dev, bf = xs.device, torch.bfloat16
    _check(xs, "xs", (R, C), bf, dev)
    _check(w_up, "w_up", (E, F, C), bf, dev)
    _check(w_down, "w_down", (E, C, F), bf, dev)
    _check(offsets, "offsets", (E + 1,), torch.int32, dev)
    if not 1 <= E <= MAX_EXPERTS:
        raise ValueError(f"1 to {MAX_EXPERTS} experts, got {E}")
    if C % 8 or F % 8 or C == 0 or F == 0:
        raise ValueError(f"the widths must be positive multiples of 8, got C = {C} and F = {F}")
    if torch.is_grad_enabled() and (xs.requires_grad or w_up.requires_grad or w_down.requires_grad):
        return _FfnFn.apply(xs, w_up, w_down, offsets)
    return _ffn(xs, w_up, w_down, offsets, False)[0]
