"""What a kernel does when one of its bounded waits runs out: it leaves in order, waits for its copies in flight, and says so."""
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
