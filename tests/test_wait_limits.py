"""What a kernel does when one of its bounded waits runs out: it leaves in order, waits for its copies in flight, and says so."""
import random

import pytest
import torch


@pytest.mark.parametrize("depth,ahead", [(2, 2), (3, 3), (5, 5), (8, 8), (3, 2)])
def test_layer_norm_ring_drains_what_is_in_flight(depth, ahead):
    """The ring's bookkeeping restated: row i of a group uses stage i % depth and the parity of i // depth.  The copies of ``ahead`` rows
    are started first, then one more per finished row; a wait that runs out at row i leaves rows i .. i + ahead - 1 in flight."""
    for rows in range(1, 3 * depth + 2):
        for fails_at in range(rows):
            issued = list(range(min(ahead, rows)))
            k = phase = 0
            for i in range(fails_at):
                assert (k, phase) == (i % depth, i // depth & 1)
                if i + ahead < rows:
                    issued.append(i + ahead)
                k += 1
                if k == depth:
                    k, phase = 0, phase ^ 1
            drained = [((k + j) % depth, phase ^ (k + j >= depth)) for j in range(ahead) if fails_at + j < rows]
            assert drained == [(q % depth, q // depth & 1) for q in issued if q >= fails_at]


@pytest.mark.gpu
@pytest.mark.parametrize("shape,dtype", [((5000, 1024), torch.bfloat16), ((2400, 8192), torch.bfloat16), ((2401, 9000), torch.float16),
                                         ((2400, 2048), torch.float32), ((40, 256), torch.float32)])
def test_layer_norm_ring_whose_waits_run_out(shape, dtype):
    """Every row group takes its first wait for one that ran out, with copies in flight.  The calls return, the error word says so once, the results are NaN,
    and the next calls are right."""
    from chocosgd_b200.ops import _lib
    from chocosgd_b200.ops.norm import last_error, layer_norm

    lib = _lib.load()
    torch.manual_seed(0)
    x = torch.randn(*shape, device="cuda").to(dtype).requires_grad_()
    w = torch.randn(shape[1], device="cuda").to(dtype).requires_grad_()
    b = torch.randn(shape[1], device="cuda").to(dtype).requires_grad_()
    dy = torch.randn(*shape, device="cuda").to(dtype)
    want = layer_norm(x, w, b)
    grads = torch.autograd.grad(want, (x, w, b), dy, retain_graph=True)
    assert last_error() == 0
    ring_forward = shape[0] >= 16 * 148
    lib.layer_norm_give_up(1)
    try:
        y = layer_norm(x, w, b)
        assert last_error() == int(ring_forward) and last_error() == 0
        assert torch.isnan(y).all() if ring_forward else torch.equal(y, want)
        late = torch.autograd.grad(want, (x, w, b), dy, retain_graph=True)
        assert last_error() == 1 and last_error() == 0
        assert all(torch.isnan(t).all() for t in late)
    finally:
        assert lib.layer_norm_give_up(0) == 1
    assert torch.equal(layer_norm(x, w, b), want)
    for p, q in zip(torch.autograd.grad(want, (x, w, b), dy), grads):
        assert torch.equal(p, q)
    assert last_error() == 0


# ---- gated feed-forward: what a pair of CTAs has in flight, restated ------------------------------------------------------
class _Stage:
    """An mbarrier with one arrival per phase and a byte count (in halves of a pair's stage)."""

    def __init__(self):
        self.phase, self.arrivals, self.tx = 0, 1, 0

    def update(self, arrivals=0, tx=0):
        self.arrivals -= arrivals
        self.tx += tx
        assert self.arrivals >= 0
        if self.arrivals == 0 and self.tx == 0:
            self.phase, self.arrivals = self.phase + 1, 1


@pytest.mark.parametrize("ranks", [1, 2])
@pytest.mark.parametrize("stages", [2, 3, 8])
def test_gated_ffn_drains_what_both_ctas_have_in_flight(stages, ranks):
    """Either CTA may stop at any stage.  The drain's waits all end, each only when the copies it stands for have landed, and nothing is
    in flight behind it."""
    rng = random.Random(stages)
    for _ in range(400):
        full = [_Stage() for _ in range(stages)]
        stop = [rng.randrange(0, 3 * stages) for _ in range(ranks)]
        issued, consumed, flying = [0] * ranks, 0, []

        def land():
            j = flying.pop(rng.randrange(len(flying)))
            full[j % stages].update(tx=-1)

        consume_to = rng.randrange(0, 3 * stages)
        for _ in range(40 * stages):
            r = rng.randrange(ranks + 2)
            if r < ranks and issued[r] < stop[r] and issued[r] < consumed + stages:
                j = issued[r]
                if r == 0:
                    full[j % stages].update(arrivals=1, tx=ranks)
                flying.append(j)
                issued[r] += 1
            elif r == ranks and flying:
                land()
            elif r == ranks + 1 and consumed < consume_to and consumed < min(issued) and full[consumed % stages].phase > consumed // stages:
                consumed += 1
        mine, peer = issued[0], issued[-1]
        end = max(mine, peer)
        for j in range(max(0, end - stages), end):
            bar, phase = full[j % stages], j // stages
            assert bar.phase in (phase, phase + 1)           # a wait for the phase's parity means this phase
            if ranks == 2:
                if j >= mine:
                    bar.update(arrivals=1, tx=1)
                if j >= peer:
                    bar.update(tx=-1)
            while bar.phase == phase:
                assert flying, "the wait would run out"
                land()
            assert j not in flying
        assert not flying


@pytest.mark.gpu
@pytest.mark.parametrize("m,d,f,n,dtype", [(2000, 1024, 2048, 1024, torch.bfloat16), (700, 520, 1304, 512, torch.float16),
                                           (300, 200, 520, 200, torch.bfloat16), (33, 72, 136, 72, torch.bfloat16),
                                           (1120, 650, 1300, 650, torch.float32), (70, 136, 200, 136, torch.float32)])
def test_gated_ffn_whose_waits_run_out(m, d, f, n, dtype):
    """One CTA of a pair, or both, give up some time into the kernel, with copies and multiplications in flight: the calls return, the error word
    says so once, and the next calls are right."""
    from chocosgd_b200.ops import _lib
    from chocosgd_b200.ops.ffn import gated_ffn, last_error

    lib = _lib.load()
    torch.manual_seed(0)
    leaves = [(torch.randn(*s, device="cuda") * s[1] ** -0.5).to(dtype).requires_grad_() for s in ((m, d), (2 * f, d), (n, f))]
    dy = torch.randn(m, n, device="cuda").to(dtype)
    y = gated_ffn(*leaves)
    grads = torch.autograd.grad(y, leaves, dy, retain_graph=True)
    assert last_error() == 0
    for ranks in (1, 2, 3):
        for ns in (0, 500, 2000, 5000, 20000):
            assert lib.gated_ffn_give_up(ns << 2 | ranks) == 0
            try:
                gated_ffn(*leaves)
                late = last_error()
                torch.autograd.grad(y, leaves, dy, retain_graph=True)
                late_backward = last_error()
            finally:
                lib.gated_ffn_give_up(0)
            if ranks != 2:                                  # rank 1 exists in launches of pairs only
                assert late == 1 and late_backward == 1
            assert last_error() == 0
        assert torch.equal(gated_ffn(*leaves), y)
        for p, q in zip(torch.autograd.grad(y, leaves, dy, retain_graph=True), grads):
            assert torch.equal(p, q)
        assert last_error() == 0


# ---- the host's side ---------------------------------------------------------------------------------------------------------
class _FakeLib:
    def __init__(self, **words):
        self.words, self.reads = words, 0

    def __getattr__(self, name):
        def read():
            self.reads += 1
            return self.words.pop(name, 0)                 # reading a word resets it

        return read


def test_error_words_end_in_an_exception(monkeypatch):
    from chocosgd_b200.ops import _lib
    from chocosgd_b200.utils.error_handler import KernelTimeout

    for words, named in (({}, []), ({"layer_norm_last_error": 1}, ["layer_norm"]), ({"gated_ffn_last_error": -1}, ["gated_ffn"]),
                         ({"layer_norm_last_error": 1, "gated_ffn_last_error": 1}, ["layer_norm", "gated_ffn"])):
        lib = _FakeLib(**words)
        monkeypatch.setattr(_lib, "load", lambda: lib)
        monkeypatch.setattr(_lib, "_NODES", object())
        if named:
            with pytest.raises(KernelTimeout) as e:
                _lib.check_waits()
            assert e.value.kernels == named
        _lib.check_waits()
        monkeypatch.setattr(_lib, "_NODES", None)
        reads = lib.reads
        _lib.check_waits()                                 # none of the kernels has run in this process
        assert lib.reads == reads


def test_optimizers_read_the_error_words(monkeypatch):
    import contextlib
    import types

    from chocosgd_b200.ops import _lib
    from chocosgd_b200.optim.base import DistributedOptimizer
    from chocosgd_b200.utils.error_handler import KernelTimeout

    calls = []

    def late():
        calls.append(1)
        raise KernelTimeout(["layer_norm"])

    monkeypatch.setattr(_lib, "check_waits", late)
    monkeypatch.setattr(torch.cuda, "device", lambda d: contextlib.nullcontext())
    for kind, n in (("cpu", 0), ("cuda", 1)):
        stub = types.SimpleNamespace(engine=None, _exchange=None, _gather=False, device=torch.device(kind))
        stub.check_kernels = lambda stub=stub: DistributedOptimizer.check_kernels(stub)
        if n:
            with pytest.raises(KernelTimeout):
                DistributedOptimizer.check(stub)
        else:
            DistributedOptimizer.check(stub)
        assert len(calls) == n


def test_a_validation_is_not_used_before_the_error_words_are_read(monkeypatch):
    import types

    from chocosgd_b200.train import loops
    from chocosgd_b200.utils.error_handler import KernelTimeout

    def late():
        raise KernelTimeout(["layer_norm"])

    monkeypatch.setattr(loops, "validate", lambda *a, **k: [0.0])
    optimizer = types.SimpleNamespace(finalize=lambda: None, check_kernels=late)
    tracker = types.SimpleNamespace(best_tracker=None)       # not reached
    with pytest.raises(KernelTimeout):
        loops.do_validate(None, None, None, None, optimizer, None, tracker, None, None, None)


@pytest.mark.gpu
def test_a_training_step_with_a_late_kernel_is_reported():
    from chocosgd_b200.config import get_args
    from chocosgd_b200.models import define_model
    from chocosgd_b200.ops import _lib
    from chocosgd_b200.ops import nn as nnn
    from chocosgd_b200.optim import define_optimizer
    from chocosgd_b200.parallel.topology import Graph
    from chocosgd_b200.utils.error_handler import KernelTimeout

    conf = get_args(["--arch", "rnn_lm", "--optimizer", "parallel_choco_v", "--comm_op", "sign", "--graph_topology", "ring", "--lr", "0.5",
                     "--drop_rate", "0.0", "--rnn_n_hidden", "64", "--rnn_n_ffn", "160", "--gossip_impl", "fused"])
    graph = Graph("ring", 1, 0)
    model = define_model(conf, graph, data_loader={"n_tokens": 300}, device=torch.device("cuda", 0), consistent=False, verbose=False)
    opt = define_optimizer(conf, model, graph)
    lib = _lib.load()
    words = torch.randint(0, 300, (8, 40), device="cuda")
    hidden = tuple(h.cuda() for h in model.init_hidden(40))
    try:
        nnn.set_native(True, which=("norm", "ffn"))
        model(words, hidden)[0].sum().backward()
        opt.check()
        lib.gated_ffn_give_up(3)
        model(words, hidden)[0].sum().backward()
        lib.gated_ffn_give_up(0)
        with pytest.raises(KernelTimeout, match="gated_ffn"):
            opt.check()
        opt.check()                                        # reported once
        opt.finalize()
    finally:
        lib.gated_ffn_give_up(0)
        nnn.set_native(False, which=("norm", "ffn"))
