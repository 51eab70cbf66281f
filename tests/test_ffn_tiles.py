"""Every tile that the feed-forward products can run with (accumulator columns, CTAs per tile, whole or cut along k), against 64 bits."""
import ctypes

import pytest
import torch

from test_ffn_gpu import _check

# sizes that reach all tiles between them, then some as models have them
SIZES = {
    torch.float32: [(38, 83, 364, 97), (35, 74, 11236, 114), (8076, 70, 139, 157), (157, 399, 5593, 416), (151, 180, 10840, 889),
                    (37, 88, 2000, 1804), (1287, 96, 69, 1596), (794, 152, 71, 2790),
                    (1120, 650, 2600, 650), (2000, 1024, 2048, 1024)],
    torch.bfloat16: [(44, 68, 1038, 72), (36, 66, 15615, 243), (8579, 81, 218, 137), (179, 392, 13473, 93), (1287, 96, 69, 1596),
                     (5704, 102, 578, 445), (36, 71, 2821, 2607), (137, 169, 7474, 1567),
                     (2000, 1024, 2048, 1024), (120, 1024, 4096, 1024), (400, 1024, 2048, 1024), (1111, 520, 4104, 520)],
}
SIZES[torch.float16] = SIZES[torch.bfloat16]
ACTS = ("silu", "gelu", "relu", "sigmoid")


def _tiles(m, d, f, n, dtype):
    """{(launch, accumulator columns, CTAs, cut)} of a training pass."""
    from chocosgd_b200.ops import _lib

    out = (ctypes.c_int * 20)()
    _lib.load().gated_ffn_plan(m, d, f, n, {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}[dtype], out)
    tiles = set()
    for i, launch in enumerate(("gate", "y", "dgate", "gradients")):
        columns, ctas, *slices = out[5 * i:5 * i + 5]
        for q in slices[:3 if launch == "gradients" else 1]:
            tiles.add((launch, columns, ctas, q > 1))
    return tiles


@pytest.mark.parametrize("dtype", sorted(SIZES, key=str))
def test_the_sizes_reach_every_tile(dtype):
    """On 148 SMs.  Gate and dgate are never cut."""
    if torch.cuda.is_available() and torch.cuda.get_device_properties(0).multi_processor_count != 148:
        pytest.skip("the choice depends on the number of SMs")
    reached = set().union(*(_tiles(*s, dtype) for s in SIZES[dtype]))
    want = {(launch, columns, ctas, cut) for launch in ("gate", "y", "dgate", "gradients") for columns, ctas in ((256, 2), (128, 2), (128, 1), (64, 1))
            for cut in ((False, True) if launch in ("y", "gradients") else (False,))}
    assert reached == want, (want - reached, reached - want)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,size", [(t, s) for t in SIZES for s in SIZES[t]])
def test_against_64_bits(dtype, size):
    _check(*size, dtype, ACTS[SIZES[dtype].index(size) % 4])
