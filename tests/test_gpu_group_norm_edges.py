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


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_many_rows(dtype):
    """The hidden layer of a full graph, as it is trained."""
    _both(1 << 18, 512, 32, dtype, activation="relu", seed=41)


@gpu
def test_gradients_of_features_beyond_32_bits():
    """2.5 thousand million values; the sums in 64 bits by pieces of rows."""
    import torch
    from mask_b200 import engine
    rows, channels, groups = (1 << 22) + 3, 600, 30
    g = torch.Generator(device="cuda").manual_seed(32)
    x = torch.empty(rows, channels, device="cuda", dtype=torch.bfloat16)
    for part in x.split(1 << 20):
        part.copy_(torch.randn(part.shape, generator=g, device="cuda"))
    offsets = [0, rows - 1000, rows]
    off = torch.tensor(offsets, dtype=torch.int32, device="cuda")
    y, m, r = engine.group_norm(x, groups, offsets=off, activation="silu")
    dx, dw, db = engine.group_norm_backward(y, x, m, r, groups, offsets=off, activation="silu")
    want, size = torch.zeros(2, channels, dtype=torch.float64, device="cuda"), torch.zeros(2, channels, dtype=torch.float64, device="cuda")
    for lo in range(0, rows, 1 << 17):
        hi = min(lo + (1 << 17), rows)
        graph = (torch.arange(lo, hi, device="cuda") >= offsets[1]).long()
        per = lambda t: t.double()[graph].repeat_interleave(channels // groups, 1)   # noqa: E731
        u = (x[lo:hi].double() - per(m)) * per(r)
        s = torch.sigmoid(u)
        du = y[lo:hi].double() * s * (1 + u * (1 - s))
        for i, t in enumerate((du * u, du)):
            want[i] += t.sum(0)
            size[i] += t.abs().sum(0)
    # 585 additions of 2^-24; the activation's derivative is good to 2^-18 of (1 + |u|)
    for got, w, a in zip((dw, db), want, size):
        assert bool(((got.double() - w).abs() <= a * (585 * 2.0 ** -24 + 2.0 ** -16)).all())
        assert float(w.abs().min()) > 0.1 * float(a.min())         # no cancellation that would hide rows from another place
    # the last graph, behind 2^31 values, against the definition; its own sums from a call of it alone
    tail = slice(rows - 1000, rows)
    alone = engine.group_norm_backward(y[tail], x[tail], m[1:], r[1:], groups, activation="silu")
    _check_backward(y[tail], x[tail], m[1:], r[1:], groups, None, None, activation="silu", got=(dx[tail], alone[1], alone[2]))
