"""Counter-based dropout kernels against a plain implementation of the generator and of the operator in 64 bits."""
import numpy as np
import pytest
import torch

U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
# below the smallest normal number (fp16: 2^-14) a type's spacing is constant: half of it is smallest_normal * eps / 2 (fp16: 2^-25)
TINY = {t: torch.finfo(t).smallest_normal * torch.finfo(t).eps / 2 for t in U}


def philox(counter, key):
    """Philox4x32-10 on Python integers."""
    c, k = list(counter), list(key)
    for _ in range(10):
        p0, p1 = 0xD2511F53 * c[0], 0xCD9E8D57 * c[2]
        c = [(p1 >> 32) ^ c[1] ^ k[0], p1 & 0xFFFFFFFF, (p0 >> 32) ^ c[3] ^ k[1], p0 & 0xFFFFFFFF]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return c


def draws(n, key, site):
    out = []
    for i in range((n + 7) // 8):
        for w in philox((i & 0xFFFFFFFF, i >> 32, site, 0), (key & 0xFFFFFFFF, (key >> 32) & 0xFFFFFFFF)):
            out += [w & 0xFFFF, w >> 16]
    return np.array(out[:n])


def plain(x, p, key, site, residual):
    q = round(p * 65536) / 65536
    keep = torch.from_numpy(draws(x.numel(), key, site) >= q * 65536).to(x.device).view(x.shape)
    y = torch.where(keep, x.double() / (1 - q), 0.0)
    return (y if residual is None else y + residual.double()), keep, q


def test_generator_known_answers():
    """Known answers of Philox4x32-10 published with the generator."""
    assert philox((0, 0, 0, 0), (0, 0)) == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    assert philox((0xFFFFFFFF,) * 4, (0xFFFFFFFF,) * 2) == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,p,site", [(1, 0.5, 0), (7, 0.3, 1), (8, 0.3, 2), (9, 0.9, 3), (1003, 0.4, 0xFFFFFFFF), (8192, 0.1, 5),
                                      (40001, 0.65, 7)])
@pytest.mark.parametrize("residual", [False, True])
def test_matches_64_bits(n, p, site, dtype, residual):
    from chocosgd_b200.ops.dropout import dropout

    g = torch.Generator(device="cuda").manual_seed(n)
    x = torch.randn(n, device="cuda", generator=g).to(dtype).requires_grad_()
    r = torch.randn(n, device="cuda", generator=g).to(dtype).requires_grad_() if residual else None
    dy = torch.randn(n, device="cuda", generator=g).to(dtype)
    key = -0x123456789ABCDEF1 + n
    k = torch.tensor([key], device="cuda")
    y = dropout(x, p, k, site=site, residual=r)
    ref, keep, q = plain(x.detach(), p, key, site, r.detach() if residual else None)
    # one rounding of the product's factor and one fused multiply-add in fp32, one rounding of the result
    scaled = (x.double() / (1 - q)).abs()
    assert ((y.double() - ref).abs() <= 2 * 2.0 ** -24 * (scaled + ref.abs()) + U[dtype] * ref.abs() + TINY[dtype]).all()
    grads = torch.autograd.grad(y, (x, r) if residual else (x,), dy)
    want = torch.where(keep, dy.double() / (1 - q), 0.0)
    assert ((grads[0].double() - want).abs() <= (2 * 2.0 ** -24 + U[dtype]) * want.abs() + TINY[dtype]).all()
    assert ((grads[0] != 0) <= keep).all()
    if residual:
        assert torch.equal(grads[1], dy)


@pytest.mark.gpu
def test_unaligned_and_strided_inputs_draw_the_same_mask():
    from chocosgd_b200.ops.dropout import dropout

    k = torch.tensor([77], device="cuda")
    base = torch.randn(1025, device="cuda")
    x = base[1:]                                    # 4-byte aligned
    assert torch.equal(dropout(x, 0.5, k), dropout(x.clone(), 0.5, k))
    m = torch.randn(48, 33, device="cuda")
    assert torch.equal(dropout(m.t(), 0.5, k), dropout(m.t().contiguous(), 0.5, k))
    r = torch.randn(33, 48, device="cuda")
    assert torch.equal(dropout(m.t(), 0.5, k, residual=r), dropout(m.t().contiguous(), 0.5, k, residual=r))
    e = torch.randn(1, 48, device="cuda").expand(33, 48)
    assert torch.equal(dropout(e, 0.5, k, residual=e), dropout(e.contiguous(), 0.5, k, residual=e.contiguous()))


@pytest.mark.gpu
def test_rates_keys_and_sites():
    """Kept share within six standard deviations of 1 - q over 2^22 elements; other keys and sites give other masks."""
    from chocosgd_b200.ops.dropout import dropout, new_key

    n = 1 << 22
    x = torch.ones(n, device="cuda")
    torch.manual_seed(11)
    k = new_key(x.device)
    torch.manual_seed(11)
    assert torch.equal(k, new_key(x.device))
    k2 = new_key(x.device)
    for p in (0.1, 0.4, 0.5):
        y = dropout(x, p, k)
        kept = float((y != 0).double().mean())
        assert abs(kept - (1 - p)) < 6 * (p * (1 - p) / n) ** 0.5 + 2.0 ** -16
        for other in (dropout(x, p, k2), dropout(x, p, k, site=1)):
            both = float(((y != 0) & (other != 0)).double().mean())
            assert abs(both - (1 - p) ** 2) < 6 * (0.25 / n) ** 0.5 + 2.0 ** -15
    assert torch.equal(dropout(x, 0.0, k), x)
    assert not dropout(x, 1.0, k).any()
    r = torch.randn(n, device="cuda")
    assert torch.equal(dropout(x, 1.0, k, residual=r), r)


@pytest.mark.gpu
def test_dropped_places_hide_non_finite_values():
    from chocosgd_b200.ops.dropout import dropout

    k = torch.tensor([5], device="cuda")
    x = torch.full((4096,), float("nan"), device="cuda")
    x[::2] = float("inf")
    ones = dropout(torch.ones(4096, device="cuda"), 0.5, k)
    y = dropout(x, 0.5, k, residual=torch.ones(4096, device="cuda"))
    assert torch.equal(y[ones == 0], torch.ones_like(y[ones == 0]))
    assert not torch.isfinite(y[ones != 0]).any()
    z = torch.full((9,), float("nan"), device="cuda", requires_grad=True)
    out = dropout(z, 1.0, k)
    assert torch.equal(out, torch.zeros_like(out))
    assert torch.equal(torch.autograd.grad(out.sum(), z)[0], torch.zeros(9, device="cuda"))


@pytest.mark.gpu
def test_empty_second_derivative_and_captured_graph():
    from chocosgd_b200.ops.dropout import dropout

    k = torch.tensor([123], device="cuda")
    e = torch.empty(0, 5, device="cuda", requires_grad=True)
    assert torch.autograd.grad(dropout(e, 0.5, k).sum(), e)[0].shape == (0, 5)
    x = torch.randn(1000, device="cuda", requires_grad=True)
    (g1,) = torch.autograd.grad((dropout(x, 0.5, k) ** 2).sum(), x, create_graph=True)
    (g2,) = torch.autograd.grad(g1.sum(), x)
    m = dropout(torch.ones_like(x), 0.5, k)
    torch.testing.assert_close(g2, 2 * m * m)
    x = x.detach().clone().requires_grad_()           # a leaf without a live eager graph, as a capture needs
    dy = torch.randn(1000, device="cuda")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        torch.autograd.grad(dropout(x, 0.5, k), x, dy)
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = dropout(x, 0.5, k)
        (dx,) = torch.autograd.grad(y, x, dy)
        y = y.detach()
    for key in (9, 10):
        k.fill_(key)
        g.replay()
        assert torch.equal(y, dropout(x, 0.5, k))
        assert torch.equal(dx, torch.autograd.grad(dropout(x, 0.5, k), x, dy)[0])


@pytest.mark.gpu
def test_more_than_32_bits_of_elements():
    from chocosgd_b200.ops.dropout import dropout

    n = (1 << 32) + 21                                # 8.6 GB; draws of the runs around element 2^32 and of the last ones
    x = torch.ones(n, dtype=torch.bfloat16, device="cuda")
    key = 0x0123456789ABCDEF
    y = dropout(x, 0.5, torch.tensor([key], device="cuda"), site=6)
    for run in ((1 << 29) - 1, 1 << 29, (1 << 29) + 1, n // 8):
        want = []
        for w in philox((run & 0xFFFFFFFF, run >> 32, 6, 0), (key & 0xFFFFFFFF, key >> 32)):
            want += [(w & 0xFFFF) >= 32768, (w >> 16) >= 32768]
        got = (y[run * 8:run * 8 + 8] != 0).tolist()
        assert got == want[:len(got)], run


def test_refusals():
    from chocosgd_b200.ops.dropout import dropout

    k = torch.zeros(1, dtype=torch.int64)
    with pytest.raises(ValueError):
        dropout(torch.randn(4), 0.5, k)               # CPU tensor


@pytest.mark.gpu
def test_refusals_on_the_device():
    from chocosgd_b200.ops.dropout import dropout

    k = torch.zeros(1, dtype=torch.int64, device="cuda")
    x = torch.randn(4, device="cuda")
    for args, kw in (((x.double(), 0.5, k), {}), ((x, 1.5, k), {}), ((x, -0.1, k), {}), ((x, 0.5, k.int()), {}),
                     ((x, 0.5, k.cpu()), {}), ((x, 0.5, torch.zeros(2, dtype=torch.int64, device="cuda")), {}),
                     ((x, 0.5, k), {"site": -1}), ((x, 0.5, k), {"site": 1 << 32}),
                     ((x, 0.5, k), {"residual": x[:2]}), ((x, 0.5, k), {"residual": x.half()}), ((x, 0.5, k), {"residual": x.cpu()})):
        with pytest.raises(ValueError):
            dropout(*args, **kw)


@pytest.mark.gpu
def test_layer_with_a_residual_of_another_shape_or_type():
    from chocosgd_b200.ops.nn import Dropout, set_native

    x, bias = torch.ones(64, 96, device="cuda"), torch.full((96,), 3.0, device="cuda")
    layer = Dropout(0.5)
    try:
        set_native(True, which=("dropout",))
        for r in (bias, torch.full((64, 96), 3.0, device="cuda", dtype=torch.bfloat16)):
            y = layer(x, r)
            assert y.shape == x.shape and set(y.unique().tolist()) == {3.0, 5.0}
    finally:
        set_native(False, which=("dropout",))
