"""Layer norm of rows whose mean is far from zero, in every kernel: z comes from x - mean."""
import pytest
import torch

from test_norm_gpu import U, _check, _plain

@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape,pitch", [((5, 64), 0), ((5, 1024), 0), ((2400, 1024), 0), ((2400, 4096), 0), ((2400, 8192), 0),
                                         ((2400, 1024), 1), ((3, 16392), 0)])
def test_rows_of_one_value_give_the_bias(shape, pitch, dtype):
    """Few rows (registers), rows for every SM (the ring of bulk copies), rows off 16-byte boundaries, rows above 16384 elements.  The sums
    of these values are exact in fp32 and the widths are powers of two (the last kernel divides): so is the mean, and x - mean is zero."""
    from chocosgd_b200.ops.norm import layer_norm

    w, b = torch.randn(shape[1], device="cuda").to(dtype).requires_grad_(), torch.randn(shape[1], device="cuda").to(dtype)
    for value in (3.25, 1000.0, -0.40625, 57344.0):         # eight bits or fewer
        x = torch.full((shape[0], shape[1] + pitch), value, device="cuda", dtype=dtype)[:, :shape[1]]
        y = layer_norm(x, w, b)
        assert torch.equal(y, b.expand(shape)), value
        (dw,) = torch.autograd.grad(y, w, torch.randn(*shape, device="cuda").to(dtype))
        assert not dw.any()                                 # sums of dy z with z = 0


@pytest.mark.gpu
@pytest.mark.parametrize("shape,dtype", [((2400, 2048), torch.float32), ((2400, 4096), torch.bfloat16), ((2400, 1032), torch.float16),
                                         ((40, 640), torch.float32), ((2400, 1027), torch.float32)])
def test_large_offsets_against_64_bits(shape, dtype):
    _check(shape, dtype, dtype, offset=300.0)


@pytest.mark.gpu
def test_error_at_a_large_offset_is_that_of_the_mean():
    """fp32, mean / deviation 300.  x - mean is exact here (both within a factor of two, or the difference has no more bits than x); what
    is left is the mean's own error: sums in trees and runs of at most 32 additions, half a unit of the last place each, never all of one
    sign, and the rounding of the quotient."""
    from chocosgd_b200.ops.norm import layer_norm

    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(2400, 2048, device="cuda", generator=g) + 300
    z = layer_norm(x)
    ref = _plain(x, None, None, 1e-5, torch.zeros_like(x))[4]
    off = (z.double() - ref).abs().max(1).values            # per row: dominated by the mean's error
    assert float(off.max()) < 33 * U[torch.float32] * 300
