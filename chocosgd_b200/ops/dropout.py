"""Dropout whose mask is a function of a key and is never stored (``csrc/dropout.cu``).

``dropout(x, p, key, site=0, residual=None)``: element ``i`` (in row-major order) is dropped iff its 16-bit draw from
Philox4x32-10 under ``key`` is below ``q * 65536``, where ``q`` is ``p`` rounded to a multiple of 2^-16; kept elements are
scaled by ``1 / (1 - q)``; ``residual`` is added in the same pass.  The backward pass computes the mask again from the key.

``key`` is a 64-bit device word, so a captured CUDA graph draws a new mask whenever the word changes: ``new_key(device)``
draws one from PyTorch's generator (``torch.manual_seed``, checkpointed generator states and graph replays then act as for
the library's dropout).  Layers that share a key give different ``site`` numbers."""
from __future__ import annotations

import torch

from . import _lib
from .norm import DT, ptr


def new_key(device) -> torch.Tensor:
    """A 64-bit key on ``device``, drawn from PyTorch's generator of that device."""
    return torch.randint(-(1 << 63), (1 << 63) - 1, (1,), dtype=torch.int64, device=device)


def drop_steps(p: float) -> int:
    """The drop probability in steps of 2^-16."""
    return int(round(p * 65536))


def _apply(x, residual, key, drop, site):
    if not x.is_contiguous():
        x = x.contiguous()
    y = torch.empty_like(x)
    n = x.numel()
    if n:
        _lib.check(_lib.packed("dropout_apply", "9q")(x.data_ptr(), ptr(residual), y.data_ptr(), n, key.data_ptr(), site, drop,
                                                      DT[x.dtype], _lib.raw_stream(x.device)), "dropout_apply")
        _lib.count(1)
    return y


class _DropoutFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, key, drop, site):
        ctx.save_for_backward(key)
        ctx.drop, ctx.site, ctx.has_residual = drop, site, residual is not None
        return _apply(x, residual.contiguous() if residual is not None else None, key, drop, site)

    @staticmethod
    def backward(ctx, dy):
        (key,) = ctx.saved_tensors
        dx = None
        if ctx.needs_input_grad[0]:
            # the gradient's gradient is the same function again
            dx = (_DropoutFn.apply if torch.is_grad_enabled() else _apply)(dy, None, key, ctx.drop, ctx.site)
        return dx, dy if ctx.has_residual else None, None, None, None


def dropout_supported(x) -> bool:
    return x.is_cuda and x.dtype in DT


def dropout(x, p: float, key, site: int = 0, residual=None):
    if not dropout_supported(x):
        raise ValueError(f"dropout: needs a CUDA tensor of fp32, bf16 or fp16, got {x.dtype} on {x.device}")
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"dropout: the probability has to lie in [0, 1], got {p}")
    if not (key.dtype == torch.int64 and key.numel() == 1 and key.device == x.device):
        raise ValueError("dropout: the key is one 64-bit integer on the input's device (new_key)")
    if not 0 <= site < 1 << 32:
        raise ValueError(f"dropout: site has to fit into 32 bits, got {site}")
    if residual is not None and not (residual.shape == x.shape and residual.dtype == x.dtype and residual.device == x.device):
        raise ValueError("dropout: the residual has the input's shape, type and device")
    drop = drop_steps(p)
    if drop == 65536:                      # everything is dropped
        y = torch.where(torch.ones((), dtype=torch.bool, device=x.device), torch.zeros_like(x), x)
        return y if residual is None else residual + y
    return _lib.on_device(x.device, _DropoutFn.apply, x, residual, key, drop, site)
