"""The encoder operators where small shapes do not lead: large tiles, operands in parts, long tables.

Which kernels a shape takes is held by tests/test_encoder_launches.py, on the CPU; the bounds and their derivation are
those of test_encoder_gpu.py.
"""

import pytest

import quiver_amd as quiver
from test_encoder_gpu import TYPES, _gpu, _say

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows,dim", [(30, 50), (300_000, 100), (250_000, 128), (1_000_000, 1)])
def test_embed_grad_without_tokens(dtype, rows, dim):
    """All rows become zero, also in memory that held something else before."""
    _say("embed_grad without tokens", dtype, rows, dim)
    dev = _gpu()
    stale = [torch.full((rows, dim), 7.0, dtype=TYPES[dtype], device=dev) for _ in range(2)]
    del stale  # the allocator hands this memory to the result
    for index in (torch.int64, torch.int32):
        got = quiver.embed_grad(torch.empty((0, dim), dtype=TYPES[dtype], device=dev),
                                torch.empty((0,), dtype=index, device=dev), rows)
        assert got.shape == (rows, dim) and not got.any()
