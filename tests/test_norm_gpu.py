"""Layer-norm kernels against a plain implementation in 64 bits.

Tolerances, per element, from the arithmetic: z is computed from x, mu and rs with at most 4 roundings of 2^-24 relative to
|x| + |mu| (the sum behind mu adds log2-depth trees: below 24 roundings), so |dz| <= 32 * 2^-24 * (|x| + |mu|) * rs; the output is
rounded once to its type (half a step).  Sums over rows of n terms are held in fp32 in at most n / 148 + 148 sequential additions."""
import pytest
import torch

U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def _plain(x, w, b, eps, dy):
    x, dy = x.double(), dy.double()
    d = x.shape[-1]
    w = torch.ones(d, dtype=torch.float64, device=x.device) if w is None else w.double()
    b = torch.zeros(d, dtype=torch.float64, device=x.device) if b is None else b.double()
    mu = x.mean(-1, keepdim=True)
    rs = 1 / torch.sqrt(((x - mu) ** 2).mean(-1, keepdim=True) + eps)
    z = (x - mu) * rs
    g = dy * w
    dx = rs * (g - g.mean(-1, keepdim=True) - z * (g * z).mean(-1, keepdim=True))
    lead = tuple(range(x.dim() - 1))
    # size of the error of z: roundings of x - mu
    zerr = 32 * 2.0 ** -24 * (x.abs() + mu.abs()) * rs + 8 * 2.0 ** -24 * z.abs()
    return z * w + b, dx, (dy * z).sum(lead), dy.sum(lead), z, rs, g, zerr, w


def _check(shape, dtype, w_dtype, has_w=True, has_b=True, pitch=0, offset=0.0, seed=0):
    from chocosgd_b200.ops.norm import layer_norm

    gen = torch.Generator(device="cuda").manual_seed(seed + sum(shape))
    d = shape[-1]
    base = torch.randn(*shape[:-1], d + pitch, device="cuda", generator=gen) * 1.7 + offset
    x = base.to(dtype)[..., :d].detach().requires_grad_()
    w = (torch.randn(d, device="cuda", generator=gen) * 0.3 + 1).to(w_dtype).requires_grad_() if has_w else None
    b = (torch.randn(d, device="cuda", generator=gen) * 0.3).to(w_dtype).requires_grad_() if has_b else None
    dy = torch.randn(*shape, device="cuda", generator=gen).to(dtype)
    y = layer_norm(x, w, b, 1e-5)
    leaves = [t for t in (x, w, b) if t is not None]
    grads = dict(zip([id(t) for t in leaves], torch.autograd.grad(y, leaves, dy)))
    again = torch.autograd.grad(layer_norm(x, w, b, 1e-5), leaves, dy)
    ry, rdx, rdw, rdb, z, rs, g, zerr, wd = _plain(x.detach(), w, b, 1e-5, dy)
    assert y.dtype == dtype and y.shape == x.shape
    assert ((y.double() - ry).abs() <= zerr * wd.abs() + 2 * 2.0 ** -24 * ry.abs() + U[dtype] * ry.abs() + 1e-7).all()
    dx = grads[id(x)]
    assert dx.dtype == dtype and dx.shape == x.shape
    # the two means carry the mean error of their terms; each term below a few roundings
    gm, gz = g.abs().mean(-1, keepdim=True), (g * z).abs().mean(-1, keepdim=True)
    bound = rs * (32 * 2.0 ** -24 * (g.abs() + gm + z.abs() * gz) + zerr * gz
                  + z.abs() * (g.abs() * zerr).mean(-1, keepdim=True)) + U[dtype] * rdx.abs() + 1e-7
    assert ((dx.double() - rdx).abs() <= bound).all()
    lead = tuple(range(len(shape) - 1))
    n = max(1, y.numel() // d)
    depth = n / 148 + 160
    if has_w:
        dw = grads[id(w)]
        assert dw.dtype == w_dtype
        tol = depth * 2.0 ** -24 * (dy.double() * z).abs().sum(lead) + (dy.double().abs() * zerr).sum(lead) \
            + U[w_dtype] * rdw.abs() + 1e-7
        assert ((dw.double() - rdw).abs() <= tol).all()
    if has_b:
        db = grads[id(b)]
        tol = depth * 2.0 ** -24 * dy.double().abs().sum(lead) + U[w_dtype] * rdb.abs() + 1e-7
        assert ((db.double() - rdb).abs() <= tol).all()
    for p, q in zip(grads.values(), again):
        assert torch.equal(p, q)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", [(1, 1), (1, 2), (3, 7), (5, 33), (2, 3, 65), (32, 650), (300, 256), (7, 1027), (9, 4096), (2, 8190),
                                   (3, 8193), (2, 16384), (3, 16385), (2, 40000)])
def test_matches_64_bits(shape, dtype):
    _check(shape, dtype, dtype)


@pytest.mark.gpu
def test_many_rows_and_wide_parameters():
    _check((4999, 650), torch.float32, torch.float32)
    _check((20000, 64), torch.bfloat16, torch.float32)
    _check((3001, 1027), torch.float16, torch.float32)
    _check((700, 32), torch.float16, torch.float16)


@pytest.mark.gpu
@pytest.mark.parametrize("has_w,has_b", [(False, False), (True, False), (False, True)])
def test_without_parameters(has_w, has_b):
    _check((65, 130), torch.float32, torch.float32, has_w, has_b)
    _check((4, 20000), torch.bfloat16, torch.float32, has_w, has_b)


@pytest.mark.gpu
def test_strided_rows_and_large_offsets():
    _check((40, 72), torch.float32, torch.float32, pitch=8)
    _check((40, 72), torch.bfloat16, torch.bfloat16, pitch=3)
    _check((40, 640), torch.float32, torch.float32, offset=300.0)     # the variance is taken about the mean


@pytest.mark.gpu
def test_constant_rows_empty_input_and_non_finite_rows():
    from chocosgd_b200.ops.norm import layer_norm

    w, b = torch.randn(96, device="cuda"), torch.randn(96, device="cuda")
    y = layer_norm(torch.full((4, 96), 3.25, device="cuda"), w, b)
    assert torch.equal(y, b.expand(4, 96))                            # x - mean is exactly zero
    e = torch.empty(0, 96, device="cuda", requires_grad=True)
    w.requires_grad_()
    ge, gw = torch.autograd.grad(layer_norm(e, w, b), (e, w), torch.empty(0, 96, device="cuda"))
    assert ge.shape == (0, 96) and not gw.any()
    x = torch.randn(3, 96, device="cuda")
    x[1, 5] = float("nan")
    y = layer_norm(x, w.detach(), b)
    assert torch.isnan(y[1]).all() and torch.isfinite(y[0]).all() and torch.isfinite(y[2]).all()


@pytest.mark.gpu
def test_gradient_against_differences():
    from chocosgd_b200.ops.norm import layer_norm

    torch.manual_seed(3)
    x = torch.randn(4, 20, device="cuda", requires_grad=True)
    w = torch.randn(20, device="cuda", requires_grad=True)
    b = torch.randn(20, device="cuda", requires_grad=True)
    c = torch.randn(4, 20, device="cuda")
    grads = torch.autograd.grad((layer_norm(x, w, b) * c).sum(), (x, w, b))
    for t, g in zip((x, w, b), grads):
        v = torch.randn_like(t)
        h = 2.0 ** -7
        with torch.no_grad():
            f = []
            for s in (h, -h):
                args = [(p + s * v if p is t else p) for p in (x, w, b)]
                f.append((layer_norm(*args).double() * c.double()).sum())
        # central difference: h^2 / 6 of a third derivative of order 10, and 80 terms of 2^-22 over 2 h
        assert abs(float((f[0] - f[1]) / (2 * h)) - float((g * v).sum())) < 2e-2 * max(1.0, float((g * v).abs().sum()))


@pytest.mark.gpu
def test_side_stream_and_captured_graph():
    from chocosgd_b200.ops.norm import layer_norm

    torch.manual_seed(5)
    x = torch.randn(130, 650, device="cuda", requires_grad=True)
    w = torch.randn(650, device="cuda", requires_grad=True)
    b = torch.randn(650, device="cuda", requires_grad=True)
    dy = torch.randn(130, 650, device="cuda")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(2):
            out = [layer_norm(x, w, b).detach(), *torch.autograd.grad(layer_norm(x, w, b), (x, w, b), dy)]
    s.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = layer_norm(x, w, b)
        grads = torch.autograd.grad(y, (x, w, b), dy)
        y = y.detach()
    with torch.no_grad():
        x.mul_(2).add_(1)
    g.replay()
    want = [layer_norm(x, w, b).detach(), *torch.autograd.grad(layer_norm(x, w, b), (x, w, b), dy)]
    torch.cuda.synchronize()
    assert not torch.equal(out[1], want[1])
    for a, r in zip((y, *grads), want):
        assert torch.equal(a, r)


@pytest.mark.gpu
@pytest.mark.parametrize("shape,dtype", [((5000, 1024), torch.bfloat16), ((2500, 4104), torch.float16), ((2400, 8192), torch.bfloat16),
                                         ((2400, 2048), torch.float32), ((3000, 9000), torch.bfloat16), ((2401, 12000), torch.float16),
                                         ((3000, 650), torch.float32), ((2500, 1030), torch.bfloat16), ((2400, 10240), torch.float32)])
def test_rows_for_every_sm(shape, dtype):
    """Enough rows for the ring of bulk copies, and widths on each side of its limits."""
    from chocosgd_b200.ops.norm import last_error

    _check(shape, dtype, dtype)
    assert last_error() == 0


@pytest.mark.gpu
def test_more_than_32_bits_of_elements_single_rows_and_second_derivatives():
    from chocosgd_b200.ops.norm import layer_norm

    n, d = (1 << 21) + 3, 1024
    x = torch.randn(1 << 10, d, device="cuda").bfloat16().repeat((1 << 11) + 1, 1)[:n].requires_grad_()
    w = torch.randn(d, device="cuda")
    y = layer_norm(x, w)
    # equal rows through the same kernel give equal bits (a call with fewer rows may take another one)
    assert torch.equal(y[-1027:-3], y[:1024]) and torch.equal(y[-3:], y[:3])
    (dx,) = torch.autograd.grad(y, x, torch.ones_like(y))
    assert torch.equal(dx[:1024], dx[-1027:-3])
    del y, dx, x
    v = torch.randn(1, 64, device="cuda")
    for stride in (0, 1, 7):
        assert torch.equal(layer_norm(v.as_strided((1, 64), (stride, 1))), layer_norm(v))
    v.requires_grad_()
    with pytest.raises(RuntimeError):
        torch.autograd.grad(layer_norm(v).sum(), v, create_graph=True)


def test_refusals():
    from chocosgd_b200.ops.norm import layer_norm, layer_norm_supported

    x = torch.randn(4, 8)
    with pytest.raises(ValueError):
        layer_norm(x)                                                 # CPU tensor: the layer class runs the library there
    assert not layer_norm_supported(x.double())


@pytest.mark.gpu
def test_refusals_on_the_device():
    from chocosgd_b200.ops.norm import layer_norm

    x = torch.randn(4, 8, device="cuda")
    for args in ((x.double(),), (x, torch.ones(7, device="cuda")), (x, torch.ones(8)),
                 (x.bfloat16(), torch.ones(8, device="cuda", dtype=torch.float16)),
                 (x.bfloat16(), torch.ones(8, device="cuda", dtype=torch.float32), torch.ones(8, device="cuda", dtype=torch.bfloat16)),
                 (x[:, :0],)):
        with pytest.raises(ValueError):
            layer_norm(*args)


@pytest.mark.gpu
def test_allocation_failure_is_pytorchs_exception():
    """An expanded input whose copy (a tebibyte) no device holds: the error is the one that callers catch, and the next call works."""
    from chocosgd_b200.ops.norm import layer_norm

    row = torch.ones(1, 1024, device="cuda")
    with pytest.raises(torch.cuda.OutOfMemoryError):
        layer_norm(row.expand(1 << 28, 1024))
    assert torch.equal(layer_norm(row.expand(3, 1024)), torch.zeros(3, 1024, device="cuda"))
