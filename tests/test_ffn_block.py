"""Layer norm, dropout and the gated feed-forward layer as layers of the language model: the library's path on the CPU, and on a
GPU the native path, alone, together in the residual block, in the model, and in a captured training step."""
import pytest
import torch
import torch.nn.functional as F


def _all(names=("norm", "ffn")):
    from chocosgd_b200.ops import nn as nnn

    nnn.set_native(True, which=names)


def _off():
    from chocosgd_b200.ops import nn as nnn

    nnn.set_native(False, which=("norm", "ffn", "dropout", "linear", "ce", "lstm", "embed"))


def test_layers_on_the_cpu_are_the_library_compositions():
    from chocosgd_b200.models import layers as L

    torch.manual_seed(0)
    x = torch.randn(5, 3, 12)
    ln = L.LayerNorm(12)
    torch.testing.assert_close(ln(x), F.layer_norm(x, (12,), ln.weight, ln.bias, ln.eps))
    assert ln(x.bfloat16()).dtype == torch.bfloat16
    for act, f in (("silu", F.silu), ("gelu", F.gelu), ("relu", F.relu), ("sigmoid", torch.sigmoid)):
        m = L.GatedFeedForward(12, 20, act)
        g, u = m.weight_in[:20], m.weight_in[20:]
        torch.testing.assert_close(m(x), (f(x @ g.t()) * (x @ u.t())) @ m.weight_out.t())
    b = L.FeedForwardBlock(12, 20, "silu", 0.5).eval()
    torch.testing.assert_close(b(x), x + b.ffn(b.norm(x)))
    b.train()
    torch.manual_seed(1)
    y = b(x)
    torch.manual_seed(1)
    torch.testing.assert_close(y, x + F.dropout(b.ffn(b.norm(x)), 0.5, True))
    with pytest.raises(ValueError):
        L.GatedFeedForward(12, 20, "tanh")
    d = L.Dropout(0.25)
    assert isinstance(d, torch.nn.Dropout) and torch.equal(d.eval()(x), x)


def test_language_model_with_and_without_the_block():
    from chocosgd_b200.config import get_args, validate
    from chocosgd_b200.models import define_nlp_model
    from chocosgd_b200.models.rnn_lm import RNNLM

    conf = get_args(["--arch", "rnn_lm", "--rnn_n_hidden", "24"])
    assert conf.rnn_n_ffn == 0 and conf.counter_dropout is False
    plain = define_nlp_model(conf, 50)
    assert plain.ffn is None and not any(k.startswith("ffn") for k in plain.state_dict())
    torch.manual_seed(3)
    a = RNNLM(50, 24, 24, 2, dropout=0.3)
    torch.manual_seed(3)
    b = define_nlp_model(get_args(["--arch", "rnn_lm", "--rnn_n_hidden", "24", "--drop_rate", "0.3", "--rnn_tie_weights", "False"]), 50)
    for p, q in zip(a.parameters(), b.parameters()):
        assert torch.equal(p, q)                           # no draw of the generator is spent on a block that is not there
    conf = get_args(["--arch", "rnn_lm", "--rnn_n_hidden", "24", "--rnn_n_ffn", "40", "--rnn_ffn_act", "gelu"])
    m = define_nlp_model(conf, 50)
    assert m.ffn.ffn.weight_in.shape == (80, 24) and m.ffn.ffn.act == "gelu"
    out, h = m(torch.randint(0, 50, (7, 4)), m.init_hidden(4))
    assert out.shape == (7, 4, 50)
    out.sum().backward()
    assert all(p.grad is not None for p in m.parameters())
    conf.rnn_n_ffn = -1
    with pytest.raises(ValueError):
        validate(conf)


def test_kinds():
    from chocosgd_b200.ops import nn as nnn

    assert {"norm", "ffn"} <= set(nnn.AUTO_KINDS) and "dropout" not in nnn.available_kinds()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_the_operators_together(dtype):
    """norm -> feed-forward -> dropout and residual sum, forward and backward, against the same formulas in 64 bits with the mask
    that the dropout drew.  Rounding to the type u after each of the three operators: the output is x + v / (1 - q) with v rounded
    twice on the way (H, Y) and z once, each at most u of a value whose sum of absolute values over the product is S."""
    from chocosgd_b200.ops.dropout import dropout
    from chocosgd_b200.ops.ffn import gated_ffn
    from chocosgd_b200.ops.norm import layer_norm

    u = {torch.float32: 2.0 ** -21, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}[dtype]
    g = torch.Generator(device="cuda").manual_seed(0)
    m, d, f, p = 210, 130, 264, 0.4
    x = torch.randn(m, d, device="cuda", generator=g).to(dtype).requires_grad_()
    w = (1 + 0.2 * torch.randn(d, device="cuda", generator=g)).to(dtype).requires_grad_()
    b = (0.2 * torch.randn(d, device="cuda", generator=g)).to(dtype).requires_grad_()
    wi = (torch.randn(2 * f, d, device="cuda", generator=g) * d ** -0.5).to(dtype).requires_grad_()
    wo = (torch.randn(d, f, device="cuda", generator=g) * f ** -0.5).to(dtype).requires_grad_()
    dy = torch.randn(m, d, device="cuda", generator=g).to(dtype)
    key = torch.tensor([99], device="cuda")
    leaves = (x, w, b, wi, wo)
    y = dropout(gated_ffn(layer_norm(x, w, b), wi, wo), p, key, site=4, residual=x)
    got = (y.detach(), *torch.autograd.grad(y, leaves, dy))
    keep = dropout(torch.ones(m, d, device="cuda"), p, key, site=4).double()
    ref = [t.detach().double().requires_grad_() for t in leaves]
    n = F.layer_norm(ref[0], (d,), ref[1], ref[2], 1e-5)
    gate, up = (n @ ref[3].t()).chunk(2, -1)
    yr = ref[0] + (F.silu(gate) * up) @ ref[4].t() * keep
    want = (yr.detach(), *torch.autograd.grad(yr, ref, dy.double()))
    for name, a, r in zip(("y", "dx", "dw", "db", "dw_in", "dw_out"), got, want):
        # in the 2-norm: five roundings of at most u each enter along the way, none of them grows on average
        err = float((a.double() - r).norm() / r.norm())
        assert err < 5 * u, (name, err)


@pytest.mark.gpu
def test_layers_match_the_library_on_the_device():
    from chocosgd_b200.models import layers as L

    torch.manual_seed(0)
    torch.backends.cuda.matmul.allow_tf32 = False
    block = L.FeedForwardBlock(200, 333, "gelu", 0.0).cuda()
    x = torch.randn(6, 9, 200, device="cuda", requires_grad=True)
    dy = torch.randn(6, 9, 200, device="cuda")
    params = (x, *block.parameters())
    try:
        ref = block(x)
        g_ref = torch.autograd.grad(ref, params, dy)
        _all()
        out = block(x)
        g = torch.autograd.grad(out, params, dy)
        with torch.no_grad():
            torch.testing.assert_close(block(x), ref, rtol=1e-5, atol=1e-5)
        with torch.autocast("cuda", dtype=torch.bfloat16):
            low = block(x)
        assert low.dtype == torch.float32
        torch.testing.assert_close(low, ref, rtol=3e-2, atol=3e-2)      # eight bits of the hidden values
    finally:
        _off()
        torch.backends.cuda.matmul.allow_tf32 = True
    # sums of 200 to 333 products of order one in fp32
    torch.testing.assert_close(out, ref, rtol=1e-5, atol=1e-5)
    for a, r in zip(g, g_ref):
        assert (a - r).abs().max() < 2e-5 * r.abs().max()


@pytest.mark.gpu
def test_dropout_layer_native():
    from chocosgd_b200.models import layers as L

    d = L.Dropout(0.4)
    x = torch.randn(1000, 64, device="cuda")
    try:
        torch.manual_seed(5)
        stock = d(x)
        _all(("dropout",))
        torch.manual_seed(5)
        a = d(x)
        torch.manual_seed(5)
        b = d(x)
        c = d(x)
        assert torch.equal(a, b) and not torch.equal(a, c) and not torch.equal(a, stock)
        kept = a != 0
        torch.testing.assert_close(a[kept], x[kept] / (1 - round(0.4 * 65536) / 65536))
        assert torch.equal(d.eval()(x), x)
        d.train()
        r = torch.randn_like(x)
        torch.manual_seed(5)
        torch.testing.assert_close(d(x, r), a + r)
    finally:
        _off()


@pytest.mark.gpu
@pytest.mark.parametrize("native", [("norm", "ffn"), ("norm", "ffn", "dropout", "lstm", "embed", "ce")])
def test_training_step_of_the_model_with_the_block(native):
    """Eager and captured steps of the language model with the block: same kernels, no dropout, so the same losses; the loss of
    the first step is the library's."""
    from chocosgd_b200.config import get_args
    from chocosgd_b200.models import define_model
    from chocosgd_b200.optim import define_optimizer
    from chocosgd_b200.parallel.topology import Graph
    from chocosgd_b200.train.engine import TrainStep
    from chocosgd_b200.train.metrics import Metrics

    def run(kinds, use_graph, rate="0.0"):
        if kinds:
            _all(kinds)
        try:
            conf = get_args(["--arch", "rnn_lm", "--optimizer", "parallel_choco_v", "--comm_op", "sign", "--graph_topology", "ring", "--lr",
                             "0.5", "--momentum_factor", "0.0", "--consensus_stepsize", "0.3", "--gossip_impl", "fused", "--drop_rate", rate,
                             "--rnn_n_hidden", "64", "--rnn_n_ffn", "160"])
            graph = Graph("ring", 1, 0)
            torch.manual_seed(0)
            model = define_model(conf, graph, data_loader={"n_tokens": 300}, device=torch.device("cuda", 0), consistent=False, verbose=False)
            opt = define_optimizer(conf, model, graph)
            g = torch.Generator().manual_seed(2)
            x = torch.randint(0, 300, (8, 4), generator=g).pin_memory()
            y = torch.randint(0, 300, (8, 4), generator=g).pin_memory()
            hidden = tuple(h.cuda() for h in model.init_hidden(4))
            step = TrainStep(model, torch.nn.CrossEntropyLoss(), opt, x, y, metrics=Metrics(model, "language_modeling"),
                             use_cuda_graph=use_graph, clip_grad_norm=0.4, hidden=hidden, warmup_iters=1)
            model.train()
            losses = [float(step(x, y)) for _ in range(3)]
            opt.finalize()
            opt.engine.check()
            return losses, opt.arena.x.clone()
        finally:
            _off()

    l_ref, _ = run((), False)
    l_e, x_e = run(native, False)
    l_g, x_g = run(native, True)
    assert abs(l_e[0] - l_ref[0]) < 1e-4 * l_ref[0]
    for a, b in zip(l_e, l_g):
        assert abs(a - b) < 1e-3 * a
    assert (x_e - x_g).abs().max() < 1e-3 * x_e.abs().max()
    losses, _ = run(native, True, "0.5")                     # with masks: every replay draws its own
    assert all(l == l for l in losses) and len(set(losses)) == 3


def _block(x, w, b, wi, wo, key, p=0.25):
    from chocosgd_b200.ops.dropout import dropout
    from chocosgd_b200.ops.ffn import gated_ffn
    from chocosgd_b200.ops.norm import layer_norm

    return dropout(gated_ffn(layer_norm(x, w, b), wi, wo), p, key, site=2, residual=x)


def _block_inputs(rows, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dim, hidden = 136, 272
    shapes = ((rows, dim), (dim,), (dim,), (2 * hidden, dim), (dim, hidden))
    leaves = [torch.randn(*s, device="cuda", generator=g).mul_(0.3).to(dtype).requires_grad_() for s in shapes]
    return leaves, torch.randn(rows, dim, device="cuda", generator=g).to(dtype), torch.tensor([seed * 7919 + 1], device="cuda")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_graph_that_is_kept_gives_the_same_gradients_again(dtype):
    leaves, dy, key = _block_inputs(150, dtype, 1)
    y = _block(*leaves, key)
    first = torch.autograd.grad(y, leaves, dy, retain_graph=True)
    for p, q in zip(first, torch.autograd.grad(y, leaves, dy)):
        assert torch.equal(p, q)


@pytest.mark.gpu
def test_parameters_changed_in_place_are_refused_in_the_backward_pass():
    for which in range(1, 5):
        if which == 2:
            continue                                        # the bias is no part of any derivative
        leaves, dy, key = _block_inputs(9, torch.float32, 2)
        y = _block(*leaves, key)
        with torch.no_grad():
            leaves[which].mul_(2.0)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            torch.autograd.grad(y, leaves, dy)


@pytest.mark.gpu
def test_two_threads_on_streams_of_their_own():
    """Forward and backward passes of two threads at once, of different sizes and types: each as if it were alone."""
    import threading

    work = [_block_inputs(150, torch.float32, 3), _block_inputs(70, torch.bfloat16, 4)]
    alone = [torch.autograd.grad(_block(*leaves, key), leaves, dy) for leaves, dy, key in work]
    torch.cuda.synchronize()
    got, errors = [None, None], []

    def run(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                leaves, dy, key = work[i]
                for _ in range(20):
                    got[i] = torch.autograd.grad(_block(*leaves, key), leaves, dy)
        except Exception as e:                              # reported by the main thread
            errors.append(e)

    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(60)
    torch.cuda.synchronize()
    assert not errors, errors
    for a, b in zip(alone, got):
        for p, q in zip(a, b):
            assert torch.equal(p, q)


@pytest.mark.gpu
def test_launches_of_the_nodes_are_counted():
    from chocosgd_b200.ops import _lib

    leaves, dy, key = _block_inputs(40, torch.bfloat16, 5)
    n0 = _lib.LAUNCHES[0]
    y = _block(*leaves, key)
    n1 = _lib.LAUNCHES[0]
    torch.autograd.grad(y, leaves, dy)
    assert n1 - n0 >= 4 and _lib.LAUNCHES[0] - n1 >= 5      # norm, gate, output, dropout; their gradients
