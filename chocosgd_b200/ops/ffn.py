"""Gated feed-forward block, forward and backward (``csrc/gated_ffn.cu``).

``gated_ffn(x, w_in, w_out, act="silu")`` computes ``(act(x Wg^T) * (x Wu^T)) Wout^T`` with ``w_in = [Wg; Wu]`` of shape
``[2 F, D]`` (gate rows first) and ``w_out`` of shape ``[N, F]``; ``x`` has any leading shape.  All three are bf16, fp16 or fp32 and of
one type.  16-bit operands are multiplied as they are with fp32 accumulators, the hidden activation is rounded once to their type;
fp32 operands are split into three bf16 parts each and keep fp32 accuracy (a row that holds an infinity gives
non-finite results, not always the infinity itself; so does a hidden value above fp16's range with fp16 operands).  Rows that do not start on 16-byte boundaries (and
fp32 operands) are re-laid into an image of the operand first; the backward pass uses the forward pass' images.  Without a gradient
and for few tokens (up to 4, fp32: 32) the weights are read once as they are, without tensor cores."""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from .norm import DT, pitch, ptr, rows_of

ACTIVATIONS = {"silu": 0, "gelu": 1, "relu": 2, "sigmoid": 3}


def _declare():
    lib = _lib.load()
    if not getattr(lib, "_ffn_declared", False):
        i, ll = ctypes.c_int, ctypes.c_longlong
        lib.gated_ffn_last_error.restype = i
        lib.gated_ffn_few_tokens.argtypes = [i]
        lib.gated_ffn_few_tokens.restype = i
        lib.gated_ffn_partial_floats.argtypes = [i] * 6
        lib.gated_ffn_partial_floats.restype = ll
        lib._ffn_declared = True
    return lib


def last_error() -> int:
    """Non-zero after a bounded wait of one of the kernels on the current device ran out (synchronises)."""
    return _declare().gated_ffn_last_error()


def _pad16(n: int) -> int:
    return (n + 15) // 16 * 16


def _pad32(n: int) -> int:
    return (n + 31) // 32 * 32


def _aligned(t: torch.Tensor) -> bool:
    return t.dtype != torch.float32 and t.data_ptr() % 16 == 0 and pitch(t) % 8 == 0


class _Layout:
    """Byte offsets of several buffers inside one allocation."""

    def __init__(self):
        self.size = 0

    def add(self, nbytes: int) -> int:
        at = self.size
        self.size += (nbytes + 255) // 256 * 256
        return at

    def image(self, t: torch.Tensor):
        """Room for the operand image of a matrix, or None where it is read as it is."""
        if _aligned(t):
            return None
        return self.add(t.shape[0] * _pad16(t.shape[1]) * (6 if t.dtype == torch.float32 else 2))


def _at(base, offset):
    return 0 if offset is None else base + offset


class _GatedFfnFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w_in, w_out, act):
        lib = _declare()
        x2, wi, wo = rows_of(x), rows_of(w_in), rows_of(w_out)
        (m, d), f, n = x2.shape, w_in.shape[0] // 2, w_out.shape[0]
        train = any(ctx.needs_input_grad)
        y = torch.empty((*x.shape[:-1], n), dtype=x.dtype, device=x.device)
        dt = DT[x.dtype]
        few = not train and m <= lib.gated_ffn_few_tokens(dt)
        lay = _Layout()
        if few:
            img, z, partial, h = (None, None, None), None, None, lay.add(4 * m * _pad16(f))
        else:
            img = [lay.image(t) for t in (x2, wi, wo)]
            h = lay.add((3 if x.dtype == torch.float32 else 1) * m * _pad16(f) * 2)
            z = lay.add(2 * _pad32(m) * _pad16(f) * 4) if train else None
            floats = lib.gated_ffn_partial_floats(m, d, f, n, dt, 0)
            partial = torch.empty(floats, dtype=torch.float32, device=x.device) if floats else None
        buf = torch.empty(lay.size, dtype=torch.uint8, device=x.device)
        if m:
            b = buf.data_ptr()
            rc = _lib.packed("gated_ffn_forward", "21q")(
                x2.data_ptr(), pitch(x2), _at(b, img[0]), wi.data_ptr(), pitch(wi), _at(b, img[1]),
                wo.data_ptr(), pitch(wo), _at(b, img[2]), b + h, _at(b, z), ptr(partial),
                y.data_ptr(), m, d, f, n, act, dt, int(few), _lib.raw_stream(x2.device))
            if rc:
                raise RuntimeError(f"gated_ffn_forward failed with code {rc}")
            _lib.count(2 + int(any(i is not None for i in img)) + int(partial is not None))
        if train:
            ctx.save_for_backward(x2, wi, wo, buf)
            ctx.layout, ctx.act, ctx.x_shape = (img, h, z), act, x.shape
        return y

    @staticmethod
    def backward(ctx, dy):
        _lib.no_second_derivative("gated_ffn")
        lib = _declare()
        x2, wi, wo, buf = ctx.saved_tensors
        img, h, z = ctx.layout
        (m, d), f, n = x2.shape, wi.shape[0] // 2, wo.shape[0]
        need = ctx.needs_input_grad
        make = torch.empty if m else torch.zeros
        dx = torch.empty(ctx.x_shape, dtype=x2.dtype, device=x2.device) if need[0] else None
        dwi = make(2 * f, d, dtype=x2.dtype, device=x2.device) if need[1] else None
        dwo = make(n, f, dtype=x2.dtype, device=x2.device) if need[2] else None
        if m:
            dy2 = rows_of(dy)
            lay = _Layout()
            dy_img = lay.image(dy2)
            dz = lay.add((3 if x2.dtype == torch.float32 else 1) * 2 * m * _pad16(f) * 2)
            floats = lib.gated_ffn_partial_floats(m, d, f, n, DT[x2.dtype], 1)
            partial = lay.add(4 * floats) if floats else None
            scratch = torch.empty(lay.size, dtype=torch.uint8, device=x2.device)
            b, s = buf.data_ptr(), scratch.data_ptr()
            rc = _lib.packed("gated_ffn_backward", "26q")(
                x2.data_ptr(), pitch(x2), _at(b, img[0]), wi.data_ptr(), pitch(wi), _at(b, img[1]),
                wo.data_ptr(), pitch(wo), _at(b, img[2]), dy2.data_ptr(), pitch(dy2),
                _at(s, dy_img), b + h, b + z, s + dz, _at(s, partial), ptr(dx), ptr(dwi),
                ptr(dwo), m, d, f, n, ctx.act, DT[x2.dtype], _lib.raw_stream(x2.device))
            if rc:
                raise RuntimeError(f"gated_ffn_backward failed with code {rc}")
            _lib.count(1 + int(need[0] or need[1]) + int(dy_img is not None) + int(partial is not None))
        return dx, dwi, dwo, None


def gated_ffn_supported(x, w_in, w_out) -> bool:
    return (x.is_cuda and x.dtype in DT and x.dim() >= 1 and w_in.dim() == 2 and w_out.dim() == 2
            and w_in.dtype == x.dtype and w_out.dtype == x.dtype and w_in.device == x.device and w_out.device == x.device
            and x.shape[-1] == w_in.shape[1] and w_in.shape[0] == 2 * w_out.shape[1]
            and min(w_in.shape[0], w_in.shape[1], w_out.shape[0]) > 0
            and max(x.numel() // x.shape[-1], w_in.shape[0], w_in.shape[1], w_out.shape[0]) < 1 << 30)


def gated_ffn(x, w_in, w_out, act: str = "silu"):
    """``(act(x Wg^T) * (x Wu^T)) Wout^T``; ``act``: silu, gelu (the exact one), relu or sigmoid."""
    if act not in ACTIVATIONS:
        raise ValueError(f"gated_ffn: activation {act!r} is none of {', '.join(ACTIVATIONS)}")
    if not gated_ffn_supported(x, w_in, w_out):
        raise ValueError("gated_ffn: needs x [..., D], w_in [2 F, D] and w_out [N, F] on one CUDA device and of one type (fp32, "
                         "bf16 or fp16): got "
                         + ", ".join(f"{tuple(t.shape)} {t.dtype} {t.device}" for t in (x, w_in, w_out)))
    return _lib.on_device(x.device, _GatedFfnFn.apply, x, w_in, w_out, ACTIVATIONS[act])
