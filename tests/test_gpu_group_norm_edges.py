"""Group norm (``engine.group_norm``) on features of a few channels, over many rows and beyond 2^31 values, against the definitions
in 64 bits.  A thread sums up to 512 rows of a chunk, then come at most 8 steps over the block, 33 over the chunks and 32 over
the graphs: 585 additions of 2^-24 each at most, of which test_gpu_group_norm.py grants 320, enough for chunks of 1792 rows at 8 a step
(224, 8, 33 and 32)."""
import ctypes as C

import pytest

from mask_b200 import _lib
from tests.test_gpu_group_norm import U, _both, _check_backward, _inputs, _norm

gpu = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("channels", [4, 8, 16, 20, 24, 32, 48])
def test_threads_are_as_many_as_there_are_vectors(channels, dtype):
    """A chunk is 8 rows for each of the block's threads along the rows: 256 by the vectors of four channels of a row.  The
    scratch has two numbers for each channel of a chunk."""
    L = _lib.lib()
    rows = 255
    for backward in (0, 1):
        norm, buffer, at = _norm(dtype=dtype, rows=rows, channels=channels, groups=1, x_stride=channels, y_stride=channels, grad_stride=channels)
        vectors = channels // 4
        chunks = rows // (8 * (256 // vectors)) + 1
        up = lambda b: (b + 255) // 256 * 256   # noqa: E731
        assert L.mask_group_norm_scratch_bytes(C.byref(norm), backward) == up(chunks * channels * 8) + (up(channels * 8) if backward else 0)


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,channels,groups", [(3, 4, 1), (2047, 4, 2), (2049, 4, 4), (20000, 4, 1), (9000, 8, 2), (5000, 16, 4), (70001, 16, 1), (30000, 20, 5),
                                                  (4000, 24, 3), (2708, 32, 8), (40000, 32, 4), (20001, 48, 6), (5000, 1, 1), (9000, 3, 3), (6000, 7, 1)])
def test_few_channels(rows, channels, groups, dtype):
    for activation in ("relu", "silu"):
        _both(rows, channels, groups, dtype, activation=activation, seed=rows)
    _both(rows, channels, groups, dtype, [0, 0, rows // 3, rows // 3 + 1, rows], "none", seed=rows)
