"""The launches that the nodes of layer norm, dropout and gated feed-forward count are the kernel nodes of a captured graph."""
import ctypes

import pytest
import torch

KERNEL_NODE = 0                                             # cudaGraphNodeTypeKernel


def _kernel_nodes(call):
    from chocosgd_b200.ops import _lib

    call()                                                  # allocations, first use
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    n0 = _lib.LAUNCHES[0]
    with torch.cuda.graph(graph):
        kept = call()
    counted = _lib.LAUNCHES[0] - n0
    rt = ctypes.CDLL("libcudart.so.12")
    n = ctypes.c_size_t(0)
    raw = ctypes.c_void_p(graph.raw_cuda_graph())
    assert rt.cudaGraphGetNodes(raw, None, ctypes.byref(n)) == 0
    nodes = (ctypes.c_void_p * n.value)()
    assert rt.cudaGraphGetNodes(raw, nodes, ctypes.byref(n)) == 0
    types = []
    for node in nodes:
        t = ctypes.c_int(-1)
        assert rt.cudaGraphNodeGetType(ctypes.c_void_p(node), ctypes.byref(t)) == 0
        types.append(t.value)
    del kept
    return counted, types.count(KERNEL_NODE)


def _leaves(shapes, dtype):
    return [torch.randn(*s, device="cuda").mul_(0.1).to(dtype).requires_grad_() for s in shapes]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("m,d,f,n", [(1, 64, 64, 64), (12, 72, 136, 72), (40, 70, 90, 50), (300, 1111, 333, 257), (2000, 320, 1900, 640),
                                     (1120, 650, 2600, 650), (120, 1024, 4096, 1024)])
def test_gated_ffn(m, d, f, n, dtype):
    from chocosgd_b200.ops.ffn import gated_ffn

    for wanted in ((), (0, 1, 2), (0,), (1,), (2,), (0, 2)):
        leaves = _leaves(((m, d), (2 * f, d), (n, f)), dtype)
        dy = torch.randn(m, n, device="cuda").to(dtype)
        args = [t if i in wanted else t.detach() for i, t in enumerate(leaves)]

        def call():
            y = gated_ffn(*args)
            return torch.autograd.grad(y, [args[i] for i in wanted], dy) if wanted else y

        counted, nodes = _kernel_nodes(call)
        assert counted == nodes and counted >= 2, (wanted, counted, nodes)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("n,d", [(3, 65), (5000, 1024), (3, 16385)])
def test_layer_norm_and_dropout(n, d, dtype):
    from chocosgd_b200.ops.dropout import dropout
    from chocosgd_b200.ops.norm import layer_norm

    key = torch.tensor([5], device="cuda")
    dy = torch.randn(n, d, device="cuda").to(dtype)
    for wanted in ((), (0, 1, 2), (0,), (1,), (2,)):
        leaves = _leaves(((n, d), (d,), (d,)), dtype)
        args = [t if i in wanted else t.detach() for i, t in enumerate(leaves)]

        def call():
            y = layer_norm(*args)
            return torch.autograd.grad(y, [args[i] for i in wanted], dy) if wanted else y

        counted, nodes = _kernel_nodes(call)
        assert counted == nodes and counted >= 1, (wanted, counted, nodes)
    (x,) = _leaves(((n, d),), dtype)
    assert _kernel_nodes(lambda: torch.autograd.grad(dropout(x, 0.5, key), x, dy)) == (2, 2)
