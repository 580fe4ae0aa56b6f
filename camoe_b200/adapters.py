"""A projection shared by all rows with the low-rank adapter of each row's
request beside it, for serving one model to many requests.

    y[n] = weight x[n] + scale[a] up[a] (down[a] x[n]),   a = adapter[n]

Rows of different adapters, and rows of none, go through one call.  It has no
backward (adapters are served, not trained, here).  The C ABI is
camoe_ad_linear in include/camoe_experts.h.
"""
from __future__ import annotations

import torch

from .experts import _check, _check_aligned, _torch_ops

MAX_RANK, MAX_ADAPTERS = 256, 1024


def _refuse(x, weight, down, up, adapter, scale):
    if x.dim() != 2 or weight.dim() != 2 or down.dim() != 3:
        raise ValueError(f"expected x [N, C], weight [M, C] and down [L, D, C], got {tuple(x.shape)}, "
                         f"{tuple(weight.shape)} and {tuple(down.shape)}")
    N, C = x.shape
    M = weight.shape[0]
    L, D, _ = down.shape
    dev, bf = x.device, torch.bfloat16
    _check(x, "x", (N, C), bf, dev)
    _check(weight, "weight", (M, C), bf, dev)
    _check(down, "down", (L, D, C), bf, dev)
    _check(up, "up", (L, M, D), bf, dev)
    _check(adapter, "adapter", (N,), torch.int32, dev)
    if scale is not None:
        _check(scale, "scale", (L,), torch.float32, dev)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, down, up, scale)):
        raise RuntimeError("adapter_linear has no backward: call it under torch.no_grad()")
    _check_aligned(x, weight, down, up)
    raise ValueError(f"C, M and D must be positive multiples of 8, D at most {MAX_RANK}, 1 to {MAX_ADAPTERS} "
                     f"adapters, got C = {C}, M = {M}, D = {D}, L = {L}")


def adapter_linear(x: torch.Tensor, weight: torch.Tensor, down: torch.Tensor, up: torch.Tensor,
                   adapter: torch.Tensor, scale: torch.Tensor | None = None) -> torch.Tensor:
    """x [N, C], weight [M, C] (``F.linear``'s layout), down [L, D, C], up
    [L, M, D], all bf16, C, M and D multiples of 8 and D at most 256 (adapters
    of a smaller rank are padded with zeros); adapter [N] int32, a row outside
    [0, L) has none; scale [L] fp32, ones when not given.  Returns y [N, M].

    Sums are fp32 and y is rounded once.  With many rows (above 128, or above 512
    where the adapters are little work) scale down x is rounded to bf16 before its
    product with up, the type of the tensor cores' operands: a row of a large call
    has that rounding more than the same row in a small one (2.0e-3 against 1.7e-3
    of y in the 2-norm).  A row has its own adapter's values alone: infinities and
    NaN of the others do not reach it.  No input may require a gradient outside
    torch.no_grad(), or carry a forward-mode tangent."""
    y = _torch_ops.adapter_linear(x, weight, down, up, adapter, scale)
    if y is None:
        _refuse(x, weight, down, up, adapter, scale)
    return y


class AdapterSet:
    """The low-rank adapters of L requests for some of a module's projections:
    ``add("key", down [L, D, C], up [L, M, D], scale [L])`` per projection;
    ``linear("key", x [..., C], weight [M, C], adapter [rows])`` runs that
    projection, with its adapters where it has any."""

    def __init__(self):
        self._of = {}

    def add(self, name: str, down: torch.Tensor, up: torch.Tensor, scale: torch.Tensor | None = None) -> "AdapterSet":
        bf = torch.bfloat16
        self._of[name] = (down.to(bf).contiguous(), up.to(bf).contiguous(),
                          None if scale is None else scale.float().contiguous())
        return self

    def linear(self, name: str, x: torch.Tensor, weight: torch.Tensor, adapter: torch.Tensor) -> torch.Tensor:
        if name not in self._of:
            return torch.nn.functional.linear(x, weight)
        down, up, scale = self._of[name]
        y = adapter_linear(x.reshape(-1, x.shape[-1]).contiguous(), weight, down, up, adapter, scale)
        return y.view(*x.shape[:-1], weight.shape[0])
