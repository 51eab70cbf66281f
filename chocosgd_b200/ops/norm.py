"""Layer normalisation over the last dimension, forward and backward (``csrc/layer_norm.cu``; its autograd node and the
checks of the arguments: ``csrc/autograd.cpp``).

``layer_norm(x, weight, bias, eps)`` is ``torch.nn.functional.layer_norm`` for one normalised dimension: ``x`` fp32, bf16
or fp16 of any leading shape (rows may be strided, the last dimension has to be contiguous), ``weight`` / ``bias`` of ``x``'s
type or fp32, either of them may be ``None``.  Statistics and sums are fp32.  The parameters' gradients are summed in a fixed
order: the same inputs give the same bits.  The backward pass has no derivative of its own and says so; there is
no forward-mode derivative, a dual tensor is refused (the layer class takes the library's path for it)."""
from __future__ import annotations

from . import _lib


def last_error() -> int:
    """Non-zero if a bounded wait of one of the kernels on the current device ran out since the last call (synchronises); the
    optimizers' ``check`` reads it in a training loop."""
    return _lib.load().layer_norm_last_error()


def layer_norm_supported(x, weight=None, bias=None) -> bool:
    return x.is_cuda and _lib.nodes().layer_norm_supported(x, weight, bias)


def layer_norm(x, weight=None, bias=None, eps: float = 1e-5):
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over the last dimension."""
    return _lib.nodes().layer_norm(x, weight, bias, eps)
