"""Layer normalisation over the last dimension, forward and backward (``csrc/layer_norm.cu``).

``layer_norm(x, weight, bias, eps)`` is ``torch.nn.functional.layer_norm`` for one normalised dimension: ``x`` fp32, bf16
or fp16 of any leading shape (rows may be strided, the last dimension has to be contiguous), ``weight`` / ``bias`` of ``x``'s
type or fp32, either of them may be ``None``.  Statistics and sums are fp32.  The parameters' gradients are summed in a fixed
order: the same inputs give the same bits."""
from __future__ import annotations

import ctypes

import torch

from . import _lib

DT = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def _partial_floats(d: int) -> int:
    lib = _lib.load()
    if not getattr(lib, "_ln_declared", False):
        lib.layer_norm_partial_floats.argtypes = [ctypes.c_int]
        lib.layer_norm_partial_floats.restype = ctypes.c_longlong
        lib.layer_norm_last_error.restype = ctypes.c_int
        lib._ln_declared = True
    return lib.layer_norm_partial_floats(d)


def last_error() -> int:
    """Non-zero after a bounded wait of the backward kernel on the current device ran out (synchronises)."""
    _partial_floats(1)
    return _lib.load().layer_norm_last_error()


def rows_of(x: torch.Tensor) -> torch.Tensor:
    """``x`` as ``[rows, last]`` with a contiguous last dimension: a view where the strides allow it."""
    x2 = x if x.dim() == 2 else x.reshape(-1, x.shape[-1])
    return x2 if x2.stride(1) == 1 and x2.stride(0) >= x2.shape[1] else x2.contiguous()


def ptr(t) -> int:
    return t.data_ptr() if t is not None else 0


def pitch(x2: torch.Tensor) -> int:
    """Elements from row to row of a matrix from ``rows_of`` (a single row's stride says nothing)."""
    return x2.stride(0) if x2.shape[0] > 1 else max(1, x2.shape[1])


class _LayerNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        x2 = rows_of(x)
        n, d = x2.shape
        dev = x.device
        y = torch.empty_like(x, memory_format=torch.contiguous_format)
        p = weight if weight is not None else bias
        ctx.p_dtype = p_dtype = p.dtype if p is not None else x.dtype
        stats = torch.empty(2 * n, dtype=torch.float32, device=dev) if any(ctx.needs_input_grad) else None
        if n:
            _lib.check(_lib.packed("layer_norm_forward", "10qdq")(
                x2.data_ptr(), pitch(x2), ptr(weight), ptr(bias), y.data_ptr(), ptr(stats), n, d, DT[x.dtype], DT[p_dtype], eps,
                _lib.raw_stream(dev)), "layer_norm_forward")
            _lib.count(1)
        if stats is not None:
            ctx.save_for_backward(x2, weight, stats)
        return y

    @staticmethod
    def backward(ctx, dy):
        _lib.no_second_derivative("layer_norm")
        x2, weight, stats = ctx.saved_tensors
        n, d = x2.shape
        dev, (need_x, need_w, need_b, _) = x2.device, ctx.needs_input_grad
        dx = torch.empty_like(dy, memory_format=torch.contiguous_format) if need_x else None
        make = torch.empty if n else torch.zeros
        dw = make(d, dtype=ctx.p_dtype, device=dev) if need_w else None
        db = make(d, dtype=ctx.p_dtype, device=dev) if need_b else None
        if n:
            dy2 = rows_of(dy)
            partial = None
            if need_w or need_b:
                partial = torch.empty(_partial_floats(d), dtype=torch.float32, device=dev)
            _lib.check(_lib.packed("layer_norm_backward", "15q")(
                x2.data_ptr(), pitch(x2), dy2.data_ptr(), pitch(dy2), ptr(weight), stats.data_ptr(), ptr(dx), ptr(dw),
                ptr(db), ptr(partial), n, d, DT[x2.dtype], DT[ctx.p_dtype], _lib.raw_stream(dev)), "layer_norm_backward")
            _lib.count(2 if partial is not None else 1)
        return dx, dw, db, None


def layer_norm_supported(x, weight=None, bias=None) -> bool:
    if not (x.is_cuda and x.dtype in DT and x.dim() >= 1 and 0 < x.shape[-1] < 1 << 24):
        return False
    for p in (weight, bias):
        if p is not None and not (p.dim() == 1 and p.shape[0] == x.shape[-1] and p.device == x.device
                                  and (p.dtype is x.dtype or p.dtype is torch.float32)):
            return False
    return weight is None or bias is None or weight.dtype is bias.dtype


def layer_norm(x, weight=None, bias=None, eps: float = 1e-5):
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over the last dimension."""
    if not layer_norm_supported(x, weight, bias):
        raise ValueError("layer_norm: needs a CUDA tensor of fp32, bf16 or fp16 and, where given, weight and bias of its last "
                         "dimension's length on its device, both of its type or both fp32: got "
                         f"{tuple(x.shape)} {x.dtype} {x.device}, "
                         + ", ".join("None" if p is None else f"{tuple(p.shape)} {p.dtype} {p.device}" for p in (weight, bias)))
    if weight is not None and not weight.is_contiguous():
        weight = weight.contiguous()
    if bias is not None and not bias.is_contiguous():
        bias = bias.contiguous()
    return _lib.on_device(x.device, _LayerNormFn.apply, x, weight, bias, eps)
