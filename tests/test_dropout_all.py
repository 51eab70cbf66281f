"""Dropout that drops everything (p = 1): the rules of every other p."""
import pytest
import torch


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n", [1, 9, 4096, 1003])
def test_values_and_gradients(n, dtype):
    from chocosgd_b200.ops.dropout import dropout

    key = torch.tensor([3], device="cuda")
    x = torch.randn(n, device="cuda").to(dtype)
    x[0] = float("nan")
    x.requires_grad_()
    r, dy = torch.randn(n, device="cuda").to(dtype).requires_grad_(), torch.randn(n, device="cuda").to(dtype)
    y = dropout(x, 1.0, key)
    assert y.dtype == dtype and torch.equal(y, torch.zeros_like(x))
    assert torch.equal(torch.autograd.grad(y, x, dy)[0], torch.zeros_like(x))
    y = dropout(x, 1.0, key, residual=r)
    dx, dr = torch.autograd.grad(y, (x, r), dy)
    assert torch.equal(y, r) and not dx.any() and torch.equal(dr, dy)
    assert torch.equal(dropout(x[1:], 1.0, key, residual=r[1:]), r[1:])       # off 16-byte boundaries


@pytest.mark.gpu
def test_a_residual_of_another_shape_type_or_device_is_refused():
    from chocosgd_b200.ops.dropout import dropout

    key = torch.tensor([3], device="cuda")
    x = torch.randn(6, 8, device="cuda")
    for p in (0.5, 1.0, 1 - 2.0 ** -18):
        for r in (torch.randn(8, device="cuda"), torch.randn(6, 8, device="cuda").half(), torch.randn(6, 8), torch.randn(2, 6, 8, device="cuda")):
            with pytest.raises(ValueError):
                dropout(x, p, key, residual=r)


@pytest.mark.gpu
def test_one_launch():
    from chocosgd_b200.ops import _lib
    from chocosgd_b200.ops.dropout import dropout

    key, x = torch.tensor([3], device="cuda"), torch.randn(100, device="cuda")
    n0 = _lib.LAUNCHES[0]
    dropout(x, 1.0, key, residual=x)
    assert _lib.LAUNCHES[0] - n0 == 1
