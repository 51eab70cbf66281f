"""Backward passes whose saved tensors come back through hooks, or whose leaves were given other storage in between: the same values
with other strides and another alignment give the same bits, another size, type or device is refused."""
import pytest
import torch

from test_norm_gpu import U, _plain

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


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,w_dtype", [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.float16, torch.float32)])
@pytest.mark.parametrize("view", sorted(VIEWS))
@pytest.mark.parametrize("shape", [(41, 131), (300, 256), (2, 3, 65), (3, 16385)])
def test_layer_norm(shape, view, dtype, w_dtype):
    from chocosgd_b200.ops.norm import layer_norm

    g = torch.Generator(device="cuda").manual_seed(sum(shape))
    x = VIEWS[view](torch.randn(*shape, device="cuda", generator=g).to(dtype)).requires_grad_()
    w = VIEWS["off"](torch.randn(shape[-1], device="cuda", generator=g).to(w_dtype)).requires_grad_()
    b = torch.randn(shape[-1], device="cuda", generator=g).to(w_dtype).requires_grad_()
    dy = torch.randn(*shape, device="cuda", generator=g).to(dtype)
    want = torch.autograd.grad(layer_norm(x, w, b), (x, w, b), dy)
    # Another alignment may take the kernel of another access width, which adds up in another order.  Twice the bound of either side
    # against 64 bits: z within zerr, the two means within 32 roundings of their terms, sums over rows of at most depth additions.
    rdx, rdw, rdb, z, rs, gw, zerr = _plain(x.detach(), w, b, 1e-5, dy)[1:8]
    dyd, lead = dy.double().abs(), tuple(range(len(shape) - 1))
    u, uw, depth = U[dtype], U[w_dtype], 162
    gm, gz = gw.abs().mean(-1, keepdim=True), (gw * z).abs().mean(-1, keepdim=True)
    tol = (rs * (32 * 2.0 ** -24 * (gw.abs() + gm + z.abs() * gz) + zerr * gz + z.abs() * (gw.abs() * zerr).mean(-1, keepdim=True))
           + u * rdx.abs() + 1e-7,
           depth * 2.0 ** -24 * (dyd * z.abs()).sum(lead) + (dyd * zerr).sum(lead) + uw * rdw.abs() + 1e-7,
           depth * 2.0 ** -24 * dyd.sum(lead) + uw * rdb.abs() + 1e-7)
    for name in ("cpu", *sorted(UNPACK)):
        with _hooks(name):
            y = layer_norm(x, w, b)
        for p, q, t in zip(torch.autograd.grad(y, (x, w, b), dy), want, tol):
            assert ((p.double() - q.double()).abs() <= 2 * t).all(), name


@pytest.mark.gpu
def test_layer_norm_and_dropout_refuse_other_sizes_types_and_devices():
    from chocosgd_b200.ops.dropout import dropout
    from chocosgd_b200.ops.norm import layer_norm

    w = torch.ones(64, device="cuda")
    key = torch.tensor([3], device="cuda")
    for call, saved in ((lambda x: layer_norm(x, w), 3), (lambda x: dropout(x, 0.5, key), 1)):
        for which in range(saved):
            for change in (lambda t: t[:-1], lambda t: t.repeat_interleave(2, 0), lambda t: t.cpu(), lambda t: t.to(torch.float64)):
                x = torch.randn(30, 64, device="cuda").requires_grad_()
                count = [0]

                def unpack(t):
                    count[0] += 1
                    return change(t) if count[0] == which + 1 else t

                with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
                    y = call(x)
                with pytest.raises(RuntimeError, match="saved tensor came back"):
                    torch.autograd.grad(y, x, torch.ones_like(y))


@pytest.mark.gpu
def test_dropout():
    from chocosgd_b200.ops.dropout import dropout

    key = torch.tensor([41], device="cuda")
    x, dy = torch.randn(1003, device="cuda").requires_grad_(), torch.randn(1003, device="cuda")
    want = torch.autograd.grad(dropout(x, 0.4, key), x, dy)[0]
    for name in ("cpu", *sorted(UNPACK)):
        with _hooks(name):
            y = dropout(x, 0.4, key)
        assert torch.equal(torch.autograd.grad(y, x, dy)[0], want), name
