"""Gated feed-forward block, forward and backward (``csrc/gated_ffn.cu``, for few tokens
``csrc/gated_ffn_few.cu``; autograd node and checks: ``csrc/autograd.cpp``).

``gated_ffn(x, w_in, w_out, act="silu")`` computes ``(act(x Wg^T) * (x Wu^T)) Wout^T`` with ``w_in = [Wg; Wu]`` of shape
``[2 F, D]`` (gate rows first) and ``w_out`` of shape ``[N, F]``; ``x`` has any leading shape.  All three are bf16, fp16 or fp32 and of
one type.  16-bit operands are multiplied as they are with fp32 accumulators, the hidden activation is rounded once to their type;
fp32 operands are split into three bf16 parts each and keep fp32 accuracy (a row that holds an infinity gives
non-finite results, not always the infinity itself; so does a hidden value above fp16's range with fp16 operands).  Rows that do not start on 16-byte boundaries (and
fp32 operands) are re-laid into an image of the operand first; the backward pass uses the forward pass' images.  Without a gradient
and for few tokens (up to 4, fp32: 32) the weights are read once as they are, without tensor cores.  Neither the backward pass' own derivative nor a forward-mode one exists;
both are refused."""
from __future__ import annotations

from . import _lib

ACTIVATIONS = {"silu": 0, "gelu": 1, "relu": 2, "sigmoid": 3}


def last_error() -> int:
    """Non-zero if a bounded wait of one of the kernels on the current device ran out since the last call (synchronises); the
    optimizers' ``check`` reads it in a training loop."""
    return _lib.load().gated_ffn_last_error()


def gated_ffn_supported(x, w_in, w_out) -> bool:
    return x.is_cuda and _lib.nodes().gated_ffn_supported(x, w_in, w_out)


def gated_ffn(x, w_in, w_out, act: str = "silu"):
    """``(act(x Wg^T) * (x Wu^T)) Wout^T``; ``act``: silu, gelu (the exact one), relu or sigmoid."""
    code = ACTIVATIONS.get(act)
    if code is None:
        raise ValueError(f"gated_ffn: activation {act!r} is none of {', '.join(ACTIVATIONS)}")
    return _lib.nodes().gated_ffn(x, w_in, w_out, code)
