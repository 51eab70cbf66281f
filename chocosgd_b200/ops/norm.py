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


def _declare():
    lib = _lib.load()
    if not getattr(lib, "_ln_declared", False):
        vp, i, ll = ctypes.c_void_p, ctypes.c_int, ctypes.c_longlong
        lib.layer_norm_forward.argtypes = [vp, ll, vp, vp, vp, vp, vp, ll, i, ctypes.c_float, i, i, vp]
        lib.layer_norm_backward.argtypes = [vp, ll, vp, ll, vp, vp, vp, vp, vp, vp, vp, ll, i, i, i, vp]
        lib.layer_norm_partial_floats.argtypes = [i]
        lib.layer_norm_partial_floats.restype = ll
        lib.layer_norm_forward.restype = lib.layer_norm_backward.restype = i
        lib._ln_declared = True
    return lib


def rows_of(x: torch.Tensor) -> torch.Tensor:
    """``x`` as ``[rows, last]`` with a contiguous last dimension: a view where the strides allow it."""
    x2 = x if x.dim() == 2 else x.reshape(-1, x.shape[-1])
    return x2 if x2.stride(1) == 1 and x2.stride(0) >= x2.shape[1] else x2.contiguous()


class _LayerNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        lib = _declare()
        x2 = rows_of(x)
        n, d = x2.shape
        y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        p = weight if weight is not None else bias
        ctx.p_dtype = p.dtype if p is not None else x.dtype
        train = any(ctx.needs_input_grad)
        stats = torch.empty((2, n), dtype=torch.float32, device=x.device) if train else None
        if n:
            sp = stats.data_ptr() if train else 0
            _lib.check(lib.layer_norm_forward(x2.data_ptr(), x2.stride(0), _lib.ptr(weight), _lib.ptr(bias), y.data_ptr(),
                                              sp, sp + 4 * n if train else 0, n, d, eps, DT[x.dtype], DT[ctx.p_dtype],
                                              _lib.stream_ptr()), "layer_norm_forward")
            _lib.count(1)
        if train:
            ctx.save_for_backward(x2, weight, stats)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        lib = _declare()
        x2, weight, stats = ctx.saved_tensors
        n, d = x2.shape
        dev, need = x2.device, ctx.needs_input_grad
        dx = torch.empty(dy.shape, dtype=x2.dtype, device=dev) if need[0] else None
        make = torch.empty if n else torch.zeros
        dw = make(d, dtype=ctx.p_dtype, device=dev) if need[1] else None
        db = make(d, dtype=ctx.p_dtype, device=dev) if need[2] else None
        if n:
            dy2 = rows_of(dy)
            partial = None
            if need[1] or need[2]:
                partial = torch.empty(lib.layer_norm_partial_floats(d), dtype=torch.float32, device=dev)
            sp = stats.data_ptr()
            _lib.check(lib.layer_norm_backward(x2.data_ptr(), x2.stride(0), dy2.data_ptr(), dy2.stride(0), _lib.ptr(weight),
                                               sp, sp + 4 * n, _lib.ptr(dx), _lib.ptr(dw), _lib.ptr(db), _lib.ptr(partial),
                                               n, d, DT[x2.dtype], DT[ctx.p_dtype], _lib.stream_ptr()),
                       "layer_norm_backward")
            _lib.count(2 if partial is not None else 1)
        return dx, dw, db, None


def layer_norm_supported(x, weight=None, bias=None) -> bool:
    return (x.is_cuda and x.dtype in DT and x.dim() >= 1 and 0 < x.shape[-1] < 1 << 24
            and all(p is None or (p.is_cuda and p.device == x.device and p.dim() == 1 and p.shape[0] == x.shape[-1]
                                  and p.dtype in (x.dtype, torch.float32)) for p in (weight, bias))
            and (weight is None or bias is None or weight.dtype == bias.dtype))


def layer_norm(x, weight=None, bias=None, eps: float = 1e-5):
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over the last dimension."""
    if not layer_norm_supported(x, weight, bias):
        raise ValueError("layer_norm: needs a CUDA tensor of fp32, bf16 or fp16 and, where given, weight and bias of its last "
                         "dimension's length on its device, both of its type or both fp32: got "
                         f"{tuple(x.shape)} {x.dtype} {x.device}, "
                         + ", ".join("None" if p is None else f"{tuple(p.shape)} {p.dtype} {p.device}" for p in (weight, bias)))
    weight = weight.contiguous() if weight is not None else None
    bias = bias.contiguous() if bias is not None else None
    return _lib.on_device(x.device, _LayerNormFn.apply, x, weight, bias, eps)
