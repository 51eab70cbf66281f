"""Layer classes used by the model zoo.

Each class is a drop-in subclass of the ``torch.nn`` layer (same parameters, same
``state_dict`` keys).  ``set_native(True)`` routes the forward/backward of supported
shapes on CUDA tensors to the hand-written kernels; everything else (CPU, unsupported
shapes, ``set_native(False)``) runs the stock PyTorch op, which also serves as the numerics
reference in the tests."""
from __future__ import annotations

import torch
import torch.nn as nn
import torch.nn.functional as F

_NATIVE = {"linear": False, "conv": False, "lstm": False, "bn": False, "wgrad": False, "ce": False, "pool": False, "embed": False,
           "norm": False, "ffn": False, "dropout": False}


def set_native(enabled: bool = True, which=("linear", "conv", "lstm", "bn")):
    for k in which:
        _NATIVE[k] = bool(enabled)


def available_kinds():
    """Kinds of layers whose native kernels are built into this tree."""
    import importlib.util

    kinds = ["bn", "linear", "wgrad", "ce", "pool", "embed", "norm", "ffn"]
    for kind, mod in (("conv", "conv"), ("lstm", "lstm")):
        if importlib.util.find_spec(f"{__package__}.{mod}") is not None:
            kinds.append(kind)
    return tuple(kinds)


#: kinds switched on by ``auto``: the ones measured faster than the library op inside a training
#: step.  ``linear`` takes only layers large enough to fill the machine (the language model's
#: decoder: fp32-grade products on the TF32 tensor cores against the library's fp32 FMA GEMM);
#: ``lstm`` (persistent recurrence kernels) is opt-in through ``set_native`` / ``--native_layers all``.
#: ``dropout`` (masks from a counter-based generator instead of the library's) is no part of ``all``: it draws other masks from the
#: same seed, so it is switched on by itself (``--counter_dropout``).
AUTO_KINDS = ("bn", "conv", "wgrad", "ce", "linear", "pool", "embed", "norm", "ffn")


def configure_native(mode: str = "auto"):
    """Apply a ``--native_layers`` choice: auto = batch-norm + 3x3 convolution forward / input /
    weight gradient, large linear layers, layer norm, gated feed-forward, all = every kind built
    into the tree, bn = batch-norm + linear, conv = bn + convolution forward / input gradient,
    off = library ops only."""
    set_native(False, which=tuple(_NATIVE))
    if mode in ("off", None) or not torch.cuda.is_available():
        return
    if mode == "bn":
        set_native(True, which=("bn", "linear", "ce"))
    elif mode == "conv":
        set_native(True, which=("bn", "linear", "conv", "ce"))
    elif mode == "all":
        set_native(True, which=available_kinds())
    else:
        set_native(True, which=tuple(k for k in AUTO_KINDS if k in available_kinds()))


def native_enabled(kind: str) -> bool:
    return _NATIVE[kind]


class Linear(nn.Linear):
    def forward(self, x):
        if _NATIVE["linear"] and x.is_cuda and x.dtype == torch.float32 and not torch.is_autocast_enabled():
            from .gemm import linear_native, linear_supported

            if linear_supported(x, self.weight):
                return linear_native(x, self.weight, self.bias)
        return F.linear(x, self.weight, self.bias)


class Conv2d(nn.Conv2d):
    def forward(self, x):
        if _NATIVE["conv"] and x.is_cuda:
            from .conv import any_conv_supported, conv2d_native, conv_stem_native, stem_conv_supported

            if any_conv_supported(self, x):
                return conv2d_native(self, x)
            if self.in_channels == 3 and stem_conv_supported(self, x):
                return conv_stem_native(self, x)
        return super().forward(x)


class Embedding(nn.Embedding):
    """``tie_to_other_gradient()``: the weight is shared with a layer that produces a dense gradient of it in
    every backward pass (tied decoder); the look-ups' gradient is then added into that gradient in place."""

    def tie_to_other_gradient(self):
        self._wants_deferred = True

    def forward(self, idx):
        if _NATIVE["embed"] and idx.is_cuda and torch.is_grad_enabled() == self.weight.requires_grad:
            from .embedding import embedding_native, embedding_supported, enable_deferred_grad

            if embedding_supported(self, idx):
                if getattr(self, "_wants_deferred", False) and self.training and not getattr(self, "deferred_grad", False):
                    enable_deferred_grad(self)
                return embedding_native(self, idx)
        return super().forward(idx)


class MaxPool2d(nn.MaxPool2d):
    def forward(self, x):
        if _NATIVE["pool"] and x.is_cuda:
            from .pool import maxpool_native, maxpool_supported

            if maxpool_supported(self, x):
                return maxpool_native(x)
        return super().forward(x)


class BatchNorm2d(nn.BatchNorm2d):
    def forward(self, x):
        from .bn import bn_act, stock_forward

        if _NATIVE["bn"] and x.is_cuda:
            return bn_act(self, x, None, relu=False)
        return stock_forward(self, x)


class LSTM(nn.LSTM):
    def forward(self, input, hx=None):
        if _NATIVE["lstm"] and input.is_cuda and input.dtype == torch.float32:
            from .lstm import lstm_native, lstm_supported

            if lstm_supported(self, input):
                return lstm_native(self, input, hx)
        if input.is_cuda:
            self.flatten_parameters()
        return super().forward(input, hx)


class LayerNorm(nn.LayerNorm):
    """``torch.nn.LayerNorm``; over one dimension on the native path, which keeps the input's type."""

    def forward(self, x):
        if _NATIVE["norm"] and x.is_cuda and len(self.normalized_shape) == 1 and x.shape[-1] == self.normalized_shape[0]:
            from .norm import layer_norm, layer_norm_supported

            if layer_norm_supported(x, self.weight, self.bias):
                return layer_norm(x, self.weight, self.bias, self.eps)
        if self.weight is not None and x.dtype != self.weight.dtype:
            return super().forward(x.to(self.weight.dtype)).to(x.dtype)
        return super().forward(x).to(x.dtype)


class Dropout(nn.Dropout):
    """``torch.nn.Dropout``.  With the native kind ``dropout`` (or ``counter=True``, for layers that never had the library's masks)
    the mask comes from a counter-based generator under a key drawn from PyTorch's generator, and is never stored.
    ``forward(x, residual)`` returns ``residual + dropout(x)``, in one pass on the native path."""

    def __init__(self, p: float = 0.5, inplace: bool = False, counter: bool = False):
        super().__init__(p, inplace)
        self.counter = counter

    def forward(self, x, residual=None):
        on = _NATIVE["dropout"] or (self.counter and _NATIVE["ffn"])
        if on and self.training and self.p > 0 and not self.inplace and x.is_cuda:
            from .dropout import dropout, dropout_supported, new_key

            if dropout_supported(x, residual):
                if residual is not None and (residual.dtype != x.dtype or residual.shape != x.shape):
                    return residual + dropout(x, self.p, new_key(x.device))
                return dropout(x, self.p, new_key(x.device), residual=residual)
        y = super().forward(x)
        return y if residual is None else residual + y


class GatedFeedForward(nn.Module):
    """``(act(x Wg^T) * (x Wu^T)) Wout^T`` with ``weight_in = [Wg; Wu]`` of shape ``[2 hidden, dim]`` and ``weight_out``
    ``[dim, hidden]``, no biases; ``act``: silu, gelu, relu or sigmoid.  Under autocast input and weights are cast as for a
    linear layer."""

    def __init__(self, dim: int, hidden: int, act: str = "silu"):
        super().__init__()
        from .ffn import ACTIVATIONS

        if act not in ACTIVATIONS:
            raise ValueError(f"GatedFeedForward: activation {act!r} is none of {', '.join(ACTIVATIONS)}")
        self.dim, self.hidden, self.act = dim, hidden, act
        self.weight_in = nn.Parameter(torch.empty(2 * hidden, dim))
        self.weight_out = nn.Parameter(torch.empty(dim, hidden))
        self.reset_parameters()

    def reset_parameters(self):
        nn.init.uniform_(self.weight_in, -(self.dim ** -0.5), self.dim ** -0.5)
        nn.init.uniform_(self.weight_out, -(self.hidden ** -0.5), self.hidden ** -0.5)

    def extra_repr(self):
        return f"{self.dim}, hidden={self.hidden}, act={self.act!r}"

    def forward(self, x):
        w_in, w_out = self.weight_in, self.weight_out
        if _NATIVE["ffn"] and x.is_cuda:
            from .ffn import gated_ffn, gated_ffn_supported

            if torch.is_autocast_enabled("cuda"):
                dt = torch.get_autocast_dtype("cuda")
                x, w_in, w_out = x.to(dt), w_in.to(dt), w_out.to(dt)
            if gated_ffn_supported(x, w_in, w_out):
                return gated_ffn(x, w_in, w_out, self.act)
        gate, up = F.linear(x, w_in).chunk(2, dim=-1)
        act = {"silu": F.silu, "gelu": F.gelu, "relu": F.relu, "sigmoid": torch.sigmoid}[self.act]
        return F.linear(act(gate) * up, w_out)
