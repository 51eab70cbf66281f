"""Dropout whose mask is a function of a key and is never stored (``csrc/dropout.cu``; autograd
node and checks: ``csrc/autograd.cpp``).

``dropout(x, p, key, site=0, residual=None)``: element ``i`` (in row-major order) is dropped iff its 16-bit draw from
Philox4x32-10 under ``key`` is below ``q * 65536``, where ``q`` is ``p`` rounded to a multiple of 2^-16; kept elements are
scaled by ``1 / (1 - q)``; ``residual`` is added in the same pass.  The backward pass computes the mask again from the key.
There is no forward-mode derivative: a dual tensor is refused.

``key`` is a 64-bit device word, so a captured CUDA graph draws a new mask whenever the word changes: ``new_key(device)``
draws one from PyTorch's generator (``torch.manual_seed``, checkpointed generator states and graph replays then act as for
the library's dropout).  Layers that share a key give different ``site`` numbers."""
from __future__ import annotations

import torch

from . import _lib


def new_key(device) -> torch.Tensor:
    """A 64-bit key on ``device``, drawn from PyTorch's generator of that device."""
    return torch.randint(-(1 << 63), (1 << 63) - 1, (1,), dtype=torch.int64, device=device)


def drop_steps(p: float) -> int:
    """The drop probability in steps of 2^-16."""
    return int(round(p * 65536))


def dropout_supported(x, residual=None) -> bool:
    return (x.is_cuda and x.dtype in (torch.float32, torch.bfloat16, torch.float16) and not _lib.nodes().has_tangent(x)
            and (residual is None or not _lib.nodes().has_tangent(residual)))


def dropout(x, p: float, key, site: int = 0, residual=None):
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"dropout: the probability has to lie in [0, 1], got {p}")
    if not 0 <= site < 1 << 32:
        raise ValueError(f"dropout: site has to fit into 32 bits, got {site}")
    return _lib.nodes().dropout(x, drop_steps(p), key, site, residual)
