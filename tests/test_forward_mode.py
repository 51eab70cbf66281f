"""Tangents of forward-mode differentiation: refused by the kernels, carried by the layers (which take the library's path)."""
import pytest
import torch
import torch.autograd.forward_ad as fwAD


def test_tangents_are_seen():
    from chocosgd_b200.ops import _lib

    x, v = torch.randn(3), torch.randn(3)
    with fwAD.dual_level():
        d = fwAD.make_dual(x, v)
        assert _lib.nodes().has_tangent(d) and not _lib.nodes().has_tangent(x) and _lib.nodes().has_tangent(d * 2)
    assert not _lib.nodes().has_tangent(x)


@pytest.mark.gpu
def test_entry_points_refuse_a_tangent_in_any_input():
    from chocosgd_b200.ops.dropout import dropout, dropout_supported
    from chocosgd_b200.ops.ffn import gated_ffn, gated_ffn_supported
    from chocosgd_b200.ops.norm import layer_norm, layer_norm_supported

    key = torch.tensor([3], device="cuda")
    calls = ((lambda *a: layer_norm(*a), layer_norm_supported, ((6, 8), (8,), (8,))),
             (lambda x, r: dropout(x, 0.5, key, residual=r), dropout_supported, ((6, 8), (6, 8))),
             (lambda x, r: dropout(x, 1.0, key, residual=r), dropout_supported, ((6, 8), (6, 8))),
             (lambda *a: gated_ffn(*a), gated_ffn_supported, ((6, 8), (24, 8), (8, 12))))
    for call, supported, shapes in calls:
        for which in range(len(shapes)):
            for grad in (False, True):
                args = [torch.randn(*s, device="cuda", requires_grad=grad) for s in shapes]
                with fwAD.dual_level():
                    args[which] = fwAD.make_dual(args[which], torch.randn_like(args[which]))
                    assert not supported(*args)
                    with pytest.raises(NotImplementedError, match="forward-mode"):
                        call(*args)
                    args[which] = torch.randn(*shapes[which], device="cuda")
                    call(*args)


@pytest.mark.gpu
def test_backward_passes_refuse_a_tangent_in_the_gradient():
    """Forward over reverse where only what follows the operator is differentiated forwards."""
    from chocosgd_b200.ops.dropout import dropout
    from chocosgd_b200.ops.ffn import gated_ffn
    from chocosgd_b200.ops.norm import layer_norm

    key = torch.tensor([3], device="cuda")
    w_in, w_out = torch.randn(24, 8, device="cuda"), torch.randn(8, 12, device="cuda")
    for call in (layer_norm, lambda x: dropout(x, 0.5, key), lambda x: gated_ffn(x, w_in, w_out)):
        x = torch.randn(6, 8, device="cuda", requires_grad=True)
        with fwAD.dual_level():
            scale = fwAD.make_dual(torch.randn(6, 8, device="cuda"), torch.randn(6, 8, device="cuda"))
            with pytest.raises(NotImplementedError, match="forward-mode"):
                torch.autograd.grad((call(x) * scale).sum(), x)
            torch.autograd.grad(call(x).sum(), x)


@pytest.mark.gpu
def test_layers_carry_the_tangent():
    from chocosgd_b200.models import layers as L
    from chocosgd_b200.ops import nn as nnn

    torch.manual_seed(0)
    block = L.FeedForwardBlock(16, 24, "silu", 0.0).cuda()
    x, v = torch.randn(5, 16, device="cuda"), torch.randn(5, 16, device="cuda")
    try:
        nnn.set_native(True, which=("norm", "ffn", "dropout"))
        with fwAD.dual_level():
            t = fwAD.unpack_dual(block(fwAD.make_dual(x, v))).tangent
            drop = L.Dropout(0.5)
            assert fwAD.unpack_dual(drop(fwAD.make_dual(x, v), x)).tangent is not None
            assert fwAD.unpack_dual(drop(x, fwAD.make_dual(x, v))).tangent is not None
        nnn.set_native(False, which=("norm", "ffn", "dropout"))
        with fwAD.dual_level():
            want = fwAD.unpack_dual(block(fwAD.make_dual(x, v))).tangent
    finally:
        nnn.set_native(False, which=("norm", "ffn", "dropout"))
    assert t is not None and torch.equal(t, want)
