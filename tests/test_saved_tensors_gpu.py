"""Backward passes whose saved tensors come back through hooks, or whose leaves were given other storage in between: the same values
with other strides and another alignment give the same bits, another size, type or device is refused."""
import pytest
import torch

DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def _off(t):
    """The same values off every 16-byte boundary: odd row stride, odd first element."""
    if t.dim() == 0 or t.numel() == 0:
        return t.clone()
    if t.dim() == 1:
        wide = torch.zeros(t.numel() + 3, dtype=t.dtype, device=t.device)
        wide[3:] = t
        return wide[3:]
    wide = torch.zeros(*t.shape[:-1], t.shape[-1] // 2 * 2 + 5, dtype=t.dtype, device=t.device)
    wide[..., 3:3 + t.shape[-1]] = t
    return wide[..., 3:3 + t.shape[-1]]


def _aligned(t):
    """The same values with rows on 16-byte boundaries (a stride of 64 elements more than needed)."""
    if t.dim() != 2:
        return t.clone()
    wide = torch.zeros(t.shape[0], (t.shape[1] + 63) // 64 * 64 + 64, dtype=t.dtype, device=t.device)
    wide[:, :t.shape[1]] = t
    return wide[:, :t.shape[1]]


def _last_first(t):
    """The same values stored with the last dimension outermost."""
    return t.t().contiguous().t() if t.dim() == 2 else t.clone()


def _every_other(t):
    wide = torch.zeros(*t.shape, 2, dtype=t.dtype, device=t.device)
    wide[..., 0] = t
    return wide[..., 0]


UNPACK = {"clone": torch.clone, "contiguous": lambda t: t.clone(memory_format=torch.contiguous_format), "off": _off, "aligned": _aligned,
          "transposed": _last_first, "every_other": _every_other}
VIEWS = {"contiguous": lambda t: t.clone(), "off": _off, "aligned": _aligned}


def _hooks(name):
    if name == "cpu":
        return torch.autograd.graph.save_on_cpu()
    return torch.autograd.graph.saved_tensors_hooks(lambda t: t, UNPACK[name])


def _ffn_inputs(dtype, rows, d, f, n, view):
    g = torch.Generator(device="cuda").manual_seed(rows + d)
    shapes = ((rows, d), (2 * f, d), (n, f))
    leaves = [VIEWS[view](torch.randn(*s, device="cuda", generator=g).mul_(s[1] ** -0.5).to(dtype)).requires_grad_() for s in shapes]
    return leaves, torch.randn(rows, n, device="cuda", generator=g).to(dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("view", sorted(VIEWS))
@pytest.mark.parametrize("sizes", [(77, 111, 57, 43), (130, 72, 136, 40), (1, 70, 33, 9)])
def test_gated_ffn(sizes, view, dtype):
    """Operand images are made where the forward pass needs them; what comes back decides nothing about where they lie."""
    from chocosgd_b200.ops.ffn import gated_ffn

    leaves, dy = _ffn_inputs(dtype, *sizes, view)
    want = torch.autograd.grad(gated_ffn(*leaves), leaves, dy)
    for name in ("cpu", *sorted(UNPACK)):
        with _hooks(name):
            y = gated_ffn(*leaves)
        for a, b in zip(torch.autograd.grad(y, leaves, dy), want):
            assert torch.equal(a, b), name


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_gated_ffn_of_a_strided_input_with_packed_hooks(dtype):
    """An input of row stride 1112 whose packed copy has row stride 1111."""
    from chocosgd_b200.ops.ffn import gated_ffn

    g = torch.Generator(device="cuda").manual_seed(0)
    wide = torch.randn(97, 1112, device="cuda", generator=g).to(dtype)
    x = wide[:, :1111].requires_grad_()
    wi = (torch.randn(300, 1111, device="cuda", generator=g) * 0.03).to(dtype).requires_grad_()
    wo = (torch.randn(64, 150, device="cuda", generator=g) * 0.08).to(dtype).requires_grad_()
    dy = torch.randn(97, 64, device="cuda", generator=g).to(dtype)
    want = torch.autograd.grad(gated_ffn(x, wi, wo), (x, wi, wo), dy)
    with torch.autograd.graph.save_on_cpu():
        y = gated_ffn(x, wi, wo)
    for a, b in zip(torch.autograd.grad(y, (x, wi, wo), dy), want):
        assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_gated_ffn_whose_weights_moved(dtype):
    """.data of a leaf assigned between the passes (the flat parameter arena does it): same values, other storage."""
    from chocosgd_b200.ops.ffn import gated_ffn

    for before, after in (("contiguous", _off), ("off", _aligned), ("aligned", torch.Tensor.contiguous)):
        leaves, dy = _ffn_inputs(dtype, 60, 71, 40, 56, before)
        want = torch.autograd.grad(gated_ffn(*leaves), leaves, dy)
        y = gated_ffn(*leaves)
        for t in leaves:
            t.data = after(t.detach())
        for a, b in zip(torch.autograd.grad(y, leaves, dy), want):
            assert torch.equal(a, b)


@pytest.mark.gpu
def test_gated_ffn_refuses_other_sizes_types_and_devices():
    from chocosgd_b200.ops.ffn import gated_ffn

    for which in range(4):                                   # x, w_in, w_out, the workspace
        for change in (lambda t: t[:-1], lambda t: t.cpu(), lambda t: t.double()):
            leaves, dy = _ffn_inputs(torch.bfloat16, 33, 72, 40, 56, "contiguous")
            count = [0]

            def unpack(t):
                count[0] += 1
                return change(t) if count[0] == which + 1 else t

            with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
                y = gated_ffn(*leaves)
            with pytest.raises(RuntimeError, match="saved tensor came back"):
                torch.autograd.grad(y, leaves, dy)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gated_ffn_in_a_checkpoint(dtype):
    from torch.utils.checkpoint import checkpoint

    from chocosgd_b200.ops.ffn import gated_ffn

    leaves, dy = _ffn_inputs(dtype, 60, 71, 40, 71, "contiguous")
    want = torch.autograd.grad(gated_ffn(gated_ffn(*leaves), *leaves[1:]), leaves, dy)
    for reentrant in (False, True):
        y = checkpoint(lambda *a: gated_ffn(gated_ffn(*a), *a[1:]), *leaves, use_reentrant=reentrant)
        for t in leaves:
            t.grad = None
        y.backward(dy)
        for t, b in zip(leaves, want):
            assert torch.equal(t.grad, b)
