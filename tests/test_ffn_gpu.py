"""Gated feed-forward kernels against a plain implementation in 64 bits.

Tolerances.  Every product's error is measured against S = the same product of absolute values.  16-bit operands: exact
products, accumulated in fp32 with truncation: at most one step of 2^-23 of the running sum per 16 terms, so K / 16 * 2^-23 * S
(K the length of the sum); fp32 operands (three bf16 parts): the terms left out are below 2^-23 of each product, an
accumulator holds 32 k (12 tensor-core steps of at most 2^-23) and is added up in fp32 (K / 32 roundings).  What the
operator rounds in between (H, dG, dU to the operands' type u) enters the next product as u * |value|.  All of these are worst cases
over signs, so no term is random."""
import math

import pytest
import torch

U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {t: torch.finfo(t).smallest_normal * torch.finfo(t).eps / 2 for t in U}


def _act(name, z):
    if name == "silu":
        s = torch.sigmoid(z)
        return z * s, s * (1 + z * (1 - s)), 1.1 + 0 * z, 0.5 + 0 * z
    if name == "gelu":
        c = torch.special.ndtr(z)
        return z * c, c + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi), 1.13 + 0 * z, 0.8 + 0 * z
    if name == "relu":
        return z.clamp(min=0), (z > 0).double(), 1 + 0 * z, 0 * z
    s = torch.sigmoid(z)
    return s, s * (1 - s), 0.25 + 0 * z, 0.1 + 0 * z


def _plain(x, wi, wo, dy, act, dtype):
    """Outputs and bounds of their errors, all in 64 bits."""
    x, wi, wo, dy = (t.double() for t in (x, wi, wo, dy))
    f = wo.shape[1]
    u = U[dtype]

    def acc(k):
        """Accumulation and products, relative to the product of absolute values."""
        if dtype == torch.float32:
            return 14 * 2.0 ** -23 + (k / 32 + 2) * 2.0 ** -24
        return (k / 16 + 2) * 2.0 ** -23

    def prod(a, b, ea, eb, k):
        """a b^T with element errors ea, eb of the operands."""
        return a @ b.t(), (a.abs() + ea) @ (eb.t()) + ea @ b.abs().t() + acc(k) * (a.abs() @ b.abs().t())

    zero = torch.zeros_like
    d, n, m = x.shape[1], wo.shape[0], x.shape[0]
    z, ez = prod(x, wi, zero(x), zero(wi), d)
    g, up = z[:, :f], z[:, f:]
    eg, eu = ez[:, :f], ez[:, f:]
    a, da, l1, l2 = _act(act, g)                     # value, slope, Lipschitz bounds of both
    fn = 16 * 2.0 ** -24                             # exp, erf and division in fp32
    ea, eda = l1 * eg + fn * (a.abs() + 1e-3 * g.abs()), l2 * eg + fn * (1 + g.abs())
    kink = (g.abs() <= eg) if act == "relu" else torch.zeros_like(g, dtype=torch.bool)
    eda = torch.where(kink, torch.ones_like(eda), eda)
    h = a * up
    op = u if dtype != torch.float32 else 2.0 ** -23
    eh = (ea * (up.abs() + eu) + a.abs() * eu)
    eh = eh + op * (h.abs() + eh) + TINY[dtype]
    y, ey = prod(h, wo, eh, zero(wo), f)
    dh, edh = prod(dy, wo.t(), zero(dy), zero(wo.t()), n)
    dg, du = dh * up * da, dh * a
    edg = edh * (up.abs() + eu) * (da.abs() + eda) + dh.abs() * (eu * (da.abs() + eda) + up.abs() * eda)
    edu = edh * (a.abs() + ea) + dh.abs() * ea
    edg, edu = edg + op * (dg.abs() + edg) + TINY[dtype], edu + op * (du.abs() + edu) + TINY[dtype]
    dz, edz = torch.cat((dg, du), 1), torch.cat((edg, edu), 1)
    dx, edx = prod(dz, wi.t(), edz, zero(wi.t()), 2 * f)
    dwi, edwi = prod(dz.t(), x.t(), edz.t(), zero(x.t()), m)
    dwo, edwo = prod(dy.t(), h.t(), zero(dy.t()), eh.t(), m)
    outs = []
    for v, e in ((y, ey), (dx, edx), (dwi, edwi), (dwo, edwo)):
        outs.append((v, e + u * (v.abs() + e) + TINY[dtype]))
    return outs


def _inputs(m, d, f, n, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + m + 3 * d + 5 * f + 7 * n)

    def r(*s, scale=1.0):
        return (torch.randn(*s, device="cuda", generator=g) * scale).to(dtype)

    return r(m, d), r(2 * f, d, scale=d ** -0.5), r(n, f, scale=f ** -0.5), r(m, n)


def _compare(got, want, what):
    for name, t, (ref, tol) in zip(("y", "dx", "dw_in", "dw_out"), got, want):
        assert t.shape == ref.shape
        bad = (t.double() - ref).abs() > tol
        assert not bad.any(), (what, name, int(bad.sum()), float(((t.double() - ref).abs() / tol).max()))


def _check(m, d, f, n, dtype, act="silu", seed=0):
    from chocosgd_b200.ops.ffn import gated_ffn, last_error

    x, wi, wo, dy = _inputs(m, d, f, n, dtype, seed)
    for t in (x, wi, wo):
        t.requires_grad_()
    with torch.no_grad():
        y0 = gated_ffn(x, wi, wo, act)
    y = gated_ffn(x, wi, wo, act)
    grads = torch.autograd.grad(y, (x, wi, wo), dy)
    y = y.detach()
    torch.cuda.synchronize()
    assert last_error() == 0
    assert y.dtype == dtype and all(t.dtype == dtype and t.is_contiguous() for t in grads)
    want = _plain(x.detach(), wi.detach(), wo.detach(), dy, act, dtype)
    _compare((y, *grads), want, (m, d, f, n, dtype, act))
    _compare((y0,), want[:1], (m, d, f, n, dtype, act, "evaluation"))
    again = torch.autograd.grad(gated_ffn(x, wi, wo, act), (x, wi, wo), dy)
    for p, q in zip(grads, again):
        assert torch.equal(p, q)                     # fixed summation order


DTYPES = [torch.bfloat16, torch.float16, torch.float32]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,d,f,n", [(128, 64, 64, 64), (128, 128, 256, 128), (256, 192, 384, 320)])
def test_whole_tiles(m, d, f, n, dtype):
    _check(m, d, f, n, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,d,f,n", [(1, 1, 1, 1), (1, 8, 8, 8), (2, 3, 5, 7), (1, 65, 33, 129), (5, 200, 100, 200), (17, 72, 136, 40),
                                     (129, 63, 65, 31), (131, 650, 260, 650), (300, 1111, 333, 257)])
def test_ragged_sizes(m, d, f, n, dtype):
    _check(m, d, f, n, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["silu", "gelu", "relu", "sigmoid"])
@pytest.mark.parametrize("dtype", DTYPES)
def test_activations(act, dtype):
    _check(70, 136, 200, 136, dtype, act)


@pytest.mark.gpu
def test_tile_widths_and_several_tiles_per_block():
    """Sizes that reach every tile width, with more tiles than SMs and a ragged last wave."""
    _check(1500, 320, 1900, 640, torch.bfloat16)
    _check(2100, 264, 2600, 1000, torch.float16)
    _check(700, 128, 1300, 256, torch.bfloat16)
    _check(1120, 650, 1300, 650, torch.float32)
    _check(2000, 96, 640, 1600, torch.float32)


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 2, 3, 4, 5, 7, 8, 9, 15, 16, 17, 31, 32, 33, 63, 64, 65])
@pytest.mark.parametrize("dtype", DTYPES)
def test_few_tokens(m, dtype):
    _check(m, 520, 1032, 520, dtype)
    _check(m, 131, 77, 53, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,d,f,n", [(12, 4096, 24, 40), (16, 40, 4100, 24), (30, 2002, 31, 33), (13, 1, 1, 1), (16, 31, 700, 650), (9, 650, 2600, 650)])
def test_few_tokens_long_and_short_sums(m, d, f, n, dtype):
    """One block or a cluster of eight for the sum over k, less than a step of it, rows that fill no tile."""
    _check(m, d, f, n, dtype, "gelu")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m", [2, 7, 12, 24])
def test_few_tokens_in_graphs_on_streams_and_with_non_finite_rows(m, dtype):
    from chocosgd_b200.ops.ffn import gated_ffn

    x, wi, wo, _ = _inputs(m, 650, 1300, 650, dtype)
    want = gated_ffn(x, wi, wo)
    torch.cuda.synchronize()
    outs = []
    for _ in range(5):
        for s in (torch.cuda.Stream(), torch.cuda.Stream()):
            with torch.cuda.stream(s):
                outs.append(gated_ffn(x, wi, wo))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):                                 # two calls in a row, the second on the first one's result
        y = gated_ffn(gated_ffn(x, wi, wo), wi, wo)
    x.mul_(-1)
    wo.mul_(2)
    g.replay()
    assert torch.equal(y, gated_ffn(gated_ffn(x, wi, wo), wi, wo))
    clean = gated_ffn(x, wi, wo)
    x[0, 7], x[m - 1] = float("nan"), float("inf")
    y = gated_ffn(x, wi, wo)
    assert torch.equal(y[1:m - 1], clean[1:m - 1]) and torch.isnan(y[0]).all() and not torch.isfinite(y[m - 1]).any()


@pytest.mark.gpu
def test_few_tokens_do_not_touch_what_lies_beside_the_result():
    """Rows of a view whose neighbours are not finite: neither read into the sums nor written."""
    from chocosgd_b200.ops.ffn import gated_ffn

    for dtype in DTYPES:
        for m in (3, 13, 29):
            x, wi, wo, _ = _inputs(m, 70, 90, 50, dtype)
            want = gated_ffn(x, wi, wo)
            views = []
            for t in (x, wi, wo):
                wide = torch.full((t.size(0) + 2, t.size(1) + 10), float("nan"), dtype=dtype, device="cuda")
                wide[1:-1, 2:-8] = t
                views.append(wide[1:-1, 2:-8])
            assert torch.equal(gated_ffn(*views), want)


@pytest.mark.gpu
def test_leading_dimensions_strides_and_broadcast_gradients():
    from chocosgd_b200.ops.ffn import gated_ffn

    x, wi, wo, _ = _inputs(24, 72, 40, 56, torch.bfloat16)
    y = gated_ffn(x, wi, wo)
    assert torch.equal(gated_ffn(x.view(2, 3, 4, 72), wi, wo), y.view(2, 3, 4, 56))
    assert torch.equal(gated_ffn(x[5], wi, wo), gated_ffn(x[5:6], wi, wo)[0])
    wide = torch.zeros(24, 80, dtype=x.dtype, device="cuda")
    wide[:, 3:75] = x
    assert torch.equal(gated_ffn(wide[:, 3:75], wi, wo), y)          # rows that start off a 16-byte boundary
    assert torch.equal(gated_ffn(x.t().contiguous().t(), wi, wo), y)  # transposed storage
    assert torch.equal(gated_ffn(x, wi.t().contiguous().t(), wo.t().contiguous().t()), y)
    leaves = [t.requires_grad_() for t in (x, wi, wo)]
    a = torch.autograd.grad(gated_ffn(x, wi, wo).sum(), leaves)       # an expanded gradient (strides 0)
    b = torch.autograd.grad(gated_ffn(x, wi, wo), leaves, torch.ones(24, 56, dtype=x.dtype, device="cuda"))
    for p, q in zip(a, b):
        assert torch.equal(p, q)


@pytest.mark.gpu
def test_partial_gradients_and_empty_batches():
    from chocosgd_b200.ops.ffn import gated_ffn

    x, wi, wo, dy = _inputs(33, 72, 40, 56, torch.float32)
    for t in (x, wi, wo):
        t.requires_grad_()
    full = torch.autograd.grad(gated_ffn(x, wi, wo), (x, wi, wo), dy)
    for i in range(3):
        args = [t if j == i else t.detach() for j, t in enumerate((x, wi, wo))]
        (g,) = torch.autograd.grad(gated_ffn(*args), args[i], dy)
        assert torch.equal(g, full[i])
    e = torch.empty(0, 72, device="cuda", requires_grad=True)
    ge, gi, go = torch.autograd.grad(gated_ffn(e, wi, wo), (e, wi, wo), torch.empty(0, 56, device="cuda"))
    assert ge.shape == (0, 72) and not gi.any() and not go.any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_non_finite_rows_stay_in_their_rows(dtype):
    from chocosgd_b200.ops.ffn import gated_ffn

    x, wi, wo, dy = _inputs(140, 72, 40, 56, dtype)
    clean = gated_ffn(x, wi, wo)
    x[3, 7] = float("nan")
    x[130] = float("inf")
    y = gated_ffn(x, wi, wo)
    ok = torch.ones(140, dtype=torch.bool, device="cuda")
    ok[3] = ok[130] = False
    assert torch.equal(y[ok], clean[ok]) and torch.isnan(y[3]).all() and not torch.isfinite(y[130]).any()


@pytest.mark.gpu
def test_large_and_small_fp32_values_keep_their_bits():
    """Powers of two through relu: every product is exact, so is the result, from 2^-60 to 2^60."""
    from chocosgd_b200.ops.ffn import gated_ffn

    for e in (-60, -10, 0, 10, 60):
        x = torch.full((3, 64), 2.0 ** e, device="cuda")
        wi = torch.full((2 * 64, 64), 2.0 ** (-e / 2 if e % 2 == 0 else 0), device="cuda")
        wo = torch.full((64, 64), 1.0, device="cuda")
        y = gated_ffn(x, wi, wo, "relu")
        s = 64.0 * 2.0 ** e * 2.0 ** (-e / 2)
        assert torch.equal(y, torch.full_like(y, s * s * 64))


@pytest.mark.gpu
def test_gradient_against_differences():
    from chocosgd_b200.ops.ffn import gated_ffn

    x, wi, wo, c = _inputs(6, 24, 40, 16, torch.float32)
    leaves = [t.requires_grad_() for t in (x, wi, wo)]
    for act in ("silu", "gelu", "sigmoid"):
        grads = torch.autograd.grad((gated_ffn(*leaves, act) * c).sum(), leaves)
        for i, g in enumerate(grads):
            v = torch.randn_like(leaves[i])
            h = 2.0 ** -6
            with torch.no_grad():
                f = []
                for s in (h, -h):
                    args = [t + s * v if j == i else t for j, t in enumerate(leaves)]
                    f.append(float((gated_ffn(*args, act).double() * c.double()).sum()))
            # h^2 / 6 of a third derivative, relative to the terms of the directional derivative
            assert abs((f[0] - f[1]) / (2 * h) - float((g * v).sum())) < 2e-2 * float((g * v).abs().sum())


@pytest.mark.gpu
def test_side_stream_two_at_once_and_captured_graphs():
    from chocosgd_b200.ops.ffn import gated_ffn

    x, wi, wo, dy = _inputs(96, 72, 136, 72, torch.bfloat16)
    leaves = [t.requires_grad_() for t in (x, wi, wo)]

    def step():
        y = gated_ffn(*leaves)
        g = torch.autograd.grad(y, leaves, dy)
        return (y.detach(), *g)

    want = step()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    outs = []
    for _ in range(5):
        for s in (s1, s2):
            with torch.cuda.stream(s):
                outs.append(step())
    torch.cuda.synchronize()
    for o in outs:
        for a, b in zip(o, want):
            assert torch.equal(a, b)
    del outs
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            r = step()
        graphs.append((g, r))
    with torch.no_grad():
        x.mul_(-1)
    for g, _ in graphs:
        g.replay()
    want = step()
    torch.cuda.synchronize()
    for _, r in graphs:
        for a, b in zip(r, want):
            assert torch.equal(a, b)


@pytest.mark.gpu
def test_single_rows_with_odd_strides_and_second_derivatives():
    from chocosgd_b200.ops.ffn import gated_ffn

    x, wi, wo, dy = _inputs(1, 72, 40, 56, torch.bfloat16)
    want = gated_ffn(x, wi, wo)
    for stride in (0, 1, 3, 8):
        assert torch.equal(gated_ffn(x.as_strided((1, 72), (stride, 1)), wi, wo), want)
        v = x.as_strided((1, 72), (stride, 1)).detach().requires_grad_()
        w = x.detach().clone().requires_grad_()
        assert torch.equal(torch.autograd.grad(gated_ffn(v, wi, wo), v, dy)[0], torch.autograd.grad(gated_ffn(w, wi, wo), w, dy)[0])
    x.requires_grad_()
    with pytest.raises(RuntimeError):
        torch.autograd.grad(gated_ffn(x, wi, wo).float().sum(), x, create_graph=True)


@pytest.mark.gpu
def test_hidden_buffer_above_32_bit_offsets():
    from chocosgd_b200.ops.ffn import gated_ffn

    m, d, f = (1 << 18) + 5, 64, 8200                         # 2.15e9 hidden values
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(m, d, device="cuda", generator=g).bfloat16()
    wi = (torch.randn(2 * f, d, device="cuda", generator=g) * d ** -0.5).bfloat16()
    wo = (torch.randn(d, f, device="cuda", generator=g) * f ** -0.5).bfloat16()
    y = gated_ffn(x, wi, wo)
    tail = gated_ffn(x[-300:], wi, wo)
    # another tile may cut k elsewhere: 8200 products of order 1 / 90 summed in another order, rounded to eight bits
    assert (y[-300:].float() - tail.float()).abs().max() <= 2 * 2.0 ** -8 * tail.float().abs().max()
    assert torch.isfinite(y.float().sum())


def test_refusals():
    from chocosgd_b200.ops.ffn import gated_ffn

    with pytest.raises(ValueError):
        gated_ffn(torch.randn(2, 8), torch.randn(8, 8), torch.randn(8, 4))       # CPU tensors
    with pytest.raises(ValueError):
        gated_ffn(torch.randn(2, 8), torch.randn(8, 8), torch.randn(8, 4), act="tanh")


@pytest.mark.gpu
def test_refusals_on_the_device():
    from chocosgd_b200.ops.ffn import gated_ffn

    x, wi, wo, _ = _inputs(4, 8, 16, 8, torch.float32)
    for args in ((x.double(), wi.double(), wo.double()), (x.half(), wi, wo), (x[:, :7], wi, wo), (x, wi[:-1], wo), (x, wi, wo[:, :8]),
                 (x, wi.cpu(), wo), (x, wi[:0], wo[:, :0]), (x[:, :0], wi[:, :0], wo), (x, wi.view(2, 16, 8), wo)):
        with pytest.raises(ValueError):
            gated_ffn(*args)
