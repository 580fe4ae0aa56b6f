"""A projection shared by all rows with the low-rank adapter of each row's
request beside it, for serving one model to many requests.

    y[n] = weight x[n] + scale[a] up[a] (down[a] x[n]),   a = adapter[n]

Rows of different adapters, and rows of none, go through one call.  It has no
backward (adapters are served, not trained, here).  The C ABI is
camoe_ad_linear in include/camoe_experts.h.
"""
from __future__ import annotations

import torch

from . import _lib
from ._lib import check
from .experts import _check, _stream

MAX_RANK, MAX_ADAPTERS = 256, 1024


def adapter_linear(x: torch.Tensor, weight: torch.Tensor, down: torch.Tensor, up: torch.Tensor,
                   adapter: torch.Tensor, scale: torch.Tensor | None = None) -> torch.Tensor:
    """x [N, C], weight [M, C] (``F.linear``'s layout), down [L, D, C], up
    [L, M, D], all bf16, C, M and D multiples of 8 and D at most 256 (adapters
    of a smaller rank are padded with zeros); adapter [N] int32, a row outside
    [0, L) has none; scale [L] fp32, ones when not given.  Returns y [N, M]."""
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
    if C % 8 or M % 8 or D % 8 or min(C, M, D) == 0 or D > MAX_RANK or not 1 <= L <= MAX_ADAPTERS:
        raise ValueError(f"C, M and D must be positive multiples of 8, D at most {MAX_RANK}, 1 to {MAX_ADAPTERS} "
                         f"adapters, got C = {C}, M = {M}, D = {D}, L = {L}")
    if torch.is_grad_enabled() and any(t.requires_grad for t in (x, weight, down, up)):
        raise RuntimeError("adapter_linear has no backward: call it under torch.no_grad()")
    lib = _lib.lib()
    y = torch.empty(N, M, dtype=bf, device=dev)
    need = lib.camoe_ad_work_bytes(N, C, M, D, L)
    work = torch.empty(need, dtype=torch.uint8, device=dev)
    check(lib.camoe_ad_linear(x.data_ptr(), weight.data_ptr(), down.data_ptr(), up.data_ptr(), adapter.data_ptr(),
                              None if scale is None else scale.data_ptr(), y.data_ptr(), work.data_ptr(), need,
                              N, C, M, D, L, _stream(x)))
    return y
