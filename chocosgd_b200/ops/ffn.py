"""Gated feed-forward block, forward and backward (``csrc/gated_ffn.cu``, for few tokens
``csrc/gated_ffn_few.cu``; autograd node and checks: ``csrc/autograd.cpp``).

``gated_ffn(x, w_in, w_out, act="silu")`` computes ``(act(x Wg^T) * (x Wu^T)) Wout^T`` with ``w_in = [Wg; Wu]`` of shape
``[2 F, D]`` (gate rows first) and ``w_out`` of shape ``[N, F]``; ``x`` has any leading shape.  All three are bf16, fp16 or fp32 and of
one type.  16-bit operands are multiplied as they are with fp32 accumulators.  What a product hands to the next one is rounded once to
their type, because the tensor core takes operands of one type: the hidden values ``H = act(G) U`` and, in the backward pass, the
gradients of ``G`` and ``U`` (with fp16 operands any of the three above fp16's range becomes an infinity); ``G`` and ``U`` themselves are
kept in fp32.  fp32 operands are split into three bf16 parts each and keep fp32 accuracy (a row that holds an infinity gives
non-finite results, not always the infinity itself).  Rows that do not start on 16-byte boundaries (and fp32 operands) are re-laid into
an image of the operand first; the backward pass uses the forward pass' images.

Without a gradient and for few tokens the weights are read once as they are: fp32 up to 32 tokens; 16 bits up to 4 tokens, and up to 16
where the weights have at most 2^25 elements.  Up to 8 (fp32) or 4 tokens (16 bits) that is done with fp32 multiply-adds, above with the
warps' matrix instruction.  ``H`` stays in fp32 up to 4 16-bit tokens and is rounded as above from 5 on, so outputs of the same token
in an evaluation call and in a training call, or in calls of 4 and of 5 tokens, need not be equal to the last bit.

The same inputs give the same bits.  Neither the backward pass' own derivative nor a forward-mode one exists; both are refused."""
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
