"""Group norm with an activation (``engine.group_norm``) and its gradients against their definitions in 64 bits.

Tolerances are sums of what each step may be off by.  A sum of float32 values passes through fewer than 160 additions one
after the other (at most 128 rows a thread, then the block's), each off by 2^-24 of what has been summed; means are joined
in fewer than 32 steps.  The exponential is good to 2^-20.  What the oracle uses of the kernel's own outputs is its
statistics, for the gradients, since they are their inputs.
"""
import ctypes as C

import pytest

from mask_b200 import _lib

gpu = pytest.mark.gpu
U = 2.0 ** -23


def _dtype(name):
    import torch
    return {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[name]


def _inputs(rows, channels, dtype, seed=0, mean=1.0):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = (torch.randn(rows, channels, generator=g, device="cuda") + mean * torch.randn(channels, generator=g, device="cuda")).to(_dtype(dtype))
    grad = torch.randn(rows, channels, generator=g, device="cuda").to(_dtype(dtype))
    weight = 1.0 + 0.3 * torch.randn(channels, generator=g, device="cuda")
    return x, grad, weight, 0.3 * torch.randn(channels, generator=g, device="cuda")


def _bounds(offsets, rows):
    return list(zip(offsets, offsets[1:])) if offsets is not None else [(0, rows)]


def _act(u, name):
    import torch
    return {"none": lambda v: v, "relu": torch.relu, "silu": torch.nn.functional.silu}[name](u)


def _ulp(t, dtype):
    import torch
    return t.abs() * (torch.finfo(dtype).eps / 2) + (2.0 ** -25 if dtype == torch.float16 else 2.0 ** -134)


def _within(got, want, tolerance, what):
    import torch
    assert got.shape == want.shape, what
    off = (got.double() - want).abs() - tolerance
    assert bool((off <= 0).all()), (what, float(off.max()), float(tolerance.max()), int((off > 0).sum()), torch.nonzero(off > 0)[:4].tolist())


def _check_forward(x, groups, weight, bias, offsets=None, eps=1e-5, activation="none", got=None):
    import torch
    from mask_b200 import engine
    rows, channels = x.shape
    w, b = (t.double() if t is not None else torch.full((channels,), v, device="cuda", dtype=torch.float64) for t, v in ((weight, 1.0), (bias, 0.0)))
    off = None if offsets is None else torch.tensor(offsets, dtype=torch.int32, device="cuda")
    if got is None:
        got = engine.group_norm(x, groups, weight, bias, off, eps, activation)
    y, mean, rstd = got
    for i, (lo, hi) in enumerate(_bounds(offsets, rows)):
        per = x[lo:hi].double().reshape(hi - lo, groups, channels // groups)
        if hi == lo:
            assert bool((mean[i] == 0).all())
            _within(rstd[i], torch.full((groups,), eps ** -0.5, device="cuda", dtype=torch.float64), eps ** -0.5 * U, "rstd of no rows")
            continue
        m, var = per.mean((0, 2)), per.var((0, 2), unbiased=False)
        largest = per.abs().amax((0, 2))
        em = 32 * U * largest
        ev = 64 * U * var + 2 * var.sqrt() * em + em * em
        r = (var + eps).rsqrt()
        er = 0.6 * r ** 3 * ev + 2 * U * r
        _within(mean[i], m, em, "mean")
        _within(rstd[i], r, er, "rstd")
        d = per - m[:, None]
        wg, bg = w.reshape(groups, -1), b.reshape(groups, -1)
        u = d * r[:, None] * wg + bg
        eu = wg.abs() * (em[:, None] * r[:, None] + d.abs() * er[:, None]) + 4 * U * ((d * r[:, None] * wg).abs() + u.abs())
        want = _act(u, activation)
        ey = 1.1 * eu + (2.0 ** -19 * want.abs() if activation == "silu" else 0.0)
        want, ey = want.reshape(hi - lo, -1), ey.reshape(hi - lo, -1)
        _within(y[lo:hi], want, ey + _ulp(want.abs() + ey, x.dtype), "y")
    return got


def _check_backward(grad, x, mean, rstd, groups, weight, bias, offsets=None, activation="none", got=None):
    import torch
    from mask_b200 import engine
    rows, channels = x.shape
    w, b = (t.double() if t is not None else torch.full((channels,), v, device="cuda", dtype=torch.float64) for t, v in ((weight, 1.0), (bias, 0.0)))
    off = None if offsets is None else torch.tensor(offsets, dtype=torch.int32, device="cuda")
    if got is None:
        got = engine.group_norm_backward(grad, x, mean, rstd, groups, weight, bias, off, activation)
    dx, dweight, dbias = got
    sums = [torch.zeros(channels, dtype=torch.float64, device="cuda") for _ in range(4)]      # dweight, dbias and their tolerances
    wg = w.reshape(groups, -1)
    for i, (lo, hi) in enumerate(_bounds(offsets, rows)):
        if hi == lo:
            continue
        shape = (hi - lo, groups, channels // groups)
        d = x[lo:hi].double().reshape(shape) - mean[i].double()[:, None]
        r = rstd[i].double()[:, None]
        xhat = d * r
        u = xhat * wg + b.reshape(groups, -1)
        eu = 4 * U * ((xhat * wg).abs() + u.abs())
        dy = grad[lo:hi].double().reshape(shape)
        if activation == "none":
            du, edu = dy, torch.zeros_like(dy)
        elif activation == "relu":      # the gate is the sign of a rounded value
            du, edu = dy * (u > 0), dy.abs() * (u.abs() <= eu)
        else:
            s = torch.sigmoid(u)
            du, edu = dy * s * (1 + u * (1 - s)), dy.abs() * (0.6 * eu + 2.0 ** -18 * (1 + u.abs() * s))
        edu = edu + U * du.abs()
        p2, ep2 = du * xhat, edu * xhat.abs() + 3 * U * (du * xhat).abs()
        s1, s2 = du.sum(0), p2.sum(0)
        e1, e2 = edu.sum(0) + 160 * U * du.abs().sum(0), ep2.sum(0) + 160 * U * p2.abs().sum(0)
        for t, v in zip(sums, (s2, s1, e2, e1)):
            t += v.reshape(-1)
        n = (hi - lo) * (channels // groups)
        m1, m2 = ((v * wg).sum(1, keepdim=True) / n for v in (s1, s2))
        steps = (channels // groups / 32 + 12) * U
        em1, em2 = (((e + steps * v.abs()) * wg.abs()).sum(1, keepdim=True) / n for e, v in ((e1, s1), (e2, s2)))
        want = r * (du * wg - m1 - xhat * m2)
        tolerance = r * (edu * wg.abs() + em1 + xhat.abs() * em2 + 6 * U * ((du * wg).abs() + m1.abs() + (xhat * m2).abs()))
        want, tolerance = want.reshape(hi - lo, -1), tolerance.reshape(hi - lo, -1)
        _within(dx[lo:hi], want, tolerance + _ulp(want.abs() + tolerance, x.dtype), "dx")
    graphs = len(_bounds(offsets, rows))
    _within(dweight, sums[0], sums[2] + (graphs + 10) * U * sums[0].abs() + graphs * U * sums[2], "dweight")
    _within(dbias, sums[1], sums[3] + (graphs + 10) * U * sums[1].abs() + graphs * U * sums[3], "dbias")
    return got


def _both(rows, channels, groups, dtype, offsets=None, activation="none", seed=0, affine=True, mean=1.0):
    x, grad, weight, bias = _inputs(rows, channels, dtype, seed, mean)
    if not affine:
        weight = bias = None
    _, m, r = _check_forward(x, groups, weight, bias, offsets, 1e-5, activation)
    _check_backward(grad, x, m, r, groups, weight, bias, offsets, activation)


SIZES = [(1, 1, 1), (1, 8, 2), (7, 5, 5), (33, 48, 6), (300, 64, 8), (2708, 64, 8), (1000, 320, 32), (50, 1030, 10), (4099, 16, 1), (70001, 24, 3),
         (9, 2048, 4), (513, 768, 768)]


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,channels,groups", SIZES)
def test_sizes(rows, channels, groups, dtype):
    _both(rows, channels, groups, dtype, activation="silu" if rows % 2 else "none", seed=rows)


@gpu
@pytest.mark.parametrize("rows,channels,groups", [(4, 194, 1), (2, 328, 1), (30, 1000, 2), (40, 592, 16), (900, 129, 1), (900, 132, 1), (2000, 320, 32), (64, 4096, 1),
                                                  (1500, 66, 22), (5, 3, 3), (2700, 12, 2), (130, 160, 32)])
def test_groups_and_slabs(rows, channels, groups):
    """Groups wider than what a block takes of a row, groups that do not divide it, and the sizes of graph between the ways of
    taking one."""
    for dtype in ("f32", "bf16"):
        _both(rows, channels, groups, dtype, activation="silu", seed=21)
        _both(rows, channels, groups, dtype, [0, 0, rows // 3, rows], "none", seed=22)


@gpu
@pytest.mark.parametrize("activation", ["none", "relu", "silu"])
@pytest.mark.parametrize("affine", [True, False])
def test_activations(activation, affine):
    for dtype in ("f32", "bf16"):
        _both(700, 96, 12, dtype, activation=activation, seed=2, affine=affine)


BATCHES = {"ragged": [0, 1, 1, 40, 41, 300, 300, 1011, 1200], "empty": [0, 0, 0], "inside": [5, 17, 17, 600, 900], "singles": list(range(0, 257)),
           "one": [0, 1200], "long-last": [0, 3, 1200], "long-first": [0, 1199, 1200]}


@gpu
@pytest.mark.parametrize("batch", sorted(BATCHES))
@pytest.mark.parametrize("dtype,channels,groups", [("f32", 40, 5), ("bf16", 128, 16), ("f32", 7, 1)])
def test_batches(batch, dtype, channels, groups):
    # a group of one or two values has a gradient that is all cancellation, which the tolerance knows
    _both(1200, channels, groups, dtype, BATCHES[batch], "silu", seed=4)


@gpu
def test_many_graphs():
    import torch
    sizes = torch.randint(0, 9, (5000,), generator=torch.Generator().manual_seed(5))
    offsets = [0] + torch.cumsum(sizes, 0).tolist()
    x, grad, weight, bias = _inputs(offsets[-1] + 3, 64, "f32", 5)
    from mask_b200 import engine
    off = torch.tensor(offsets, dtype=torch.int32, device="cuda")
    y, m, r = engine.group_norm(x, 4, weight, bias, off, 1e-5, "relu")
    graph = torch.repeat_interleave(torch.arange(5000), sizes).cuda()
    v = x[:-3].double().reshape(-1, 4, 16)
    n = sizes.double().cuda()[:, None].clamp(min=1) * 16
    mean = torch.zeros(5000, 4, dtype=torch.float64, device="cuda").index_add_(0, graph, v.sum(2)) / n
    var = torch.zeros_like(mean).index_add_(0, graph, (v - mean[graph][:, :, None]).square().sum(2)) / n
    assert float((m - mean).abs().max()) < 32 * U * float(x.abs().max())
    want = torch.relu(((v - mean[graph][:, :, None]) * (var + 1e-5).rsqrt()[graph][:, :, None]).reshape(-1, 64) * weight.double() + bias.double())
    # at least 16 values to a group: rstd below 3 or so here, checked rather than assumed
    top = float((var + 1e-5).rsqrt()[sizes.cuda() > 0].max())
    assert float((y[:-3] - want).abs().max()) < 2 * top * 200 * U * float(x.abs().max())
    _check_backward(grad[:offsets[300]], x[:offsets[300]], m[:300], r[:300], 4, weight, bias, offsets[:301], "relu")


@gpu
@pytest.mark.parametrize("channels,groups", [(64, 64), (96, 3)])
def test_a_few_long_graphs_among_many_short_ones(channels, groups):
    """Graphs of several chunks, whose sums are joined, between graphs that are finished at once and graphs without rows."""
    import torch
    sizes = torch.randint(0, 6, (400,), generator=torch.Generator().manual_seed(9))
    for at, n in ((0, 3000), (37, 1500), (38, 2600), (399, 4000)):
        sizes[at] = n
    offsets = [0] + torch.cumsum(sizes, 0).tolist()
    _both(offsets[-1], channels, groups, "f32", offsets, "silu", seed=9)


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_far_from_zero_and_outliers(dtype):
    """Means a thousand times the deviation; a first row far from the rest."""
    _both(3000, 32, 4, dtype, mean=1000.0, seed=6)
    x, grad, weight, bias = _inputs(3000, 32, dtype, 7)
    x[0] = 1e4
    _, m, r = _check_forward(x, 4, weight, bias)
    _check_backward(grad, x, m, r, 4, weight, bias)


@gpu
def test_constant_values():
    """Variance 0: the output is the bias, the gradient that of the centred values."""
    import torch
    x = torch.full((64, 16), 3.0, device="cuda")
    _, _, weight, bias = _inputs(64, 16, "f32")
    y, m, r = _check_forward(x, 4, weight, bias)
    assert torch.equal(y, bias.expand(64, 16)) and bool((m == 3.0).all())


@gpu
def test_rows_outside_every_graph_are_left_alone():
    import torch
    from mask_b200 import engine
    x, grad, weight, bias = _inputs(1200, 48, "f32", 8)
    off = torch.tensor(BATCHES["inside"], dtype=torch.int32, device="cuda")
    want = engine.group_norm(x, 6, weight, bias, off)
    grads = engine.group_norm_backward(grad, x, want[1], want[2], 6, weight, bias, off)
    for bad in (float("nan"), float("inf")):
        dirty, dirty_grad = x.clone(), grad.clone()
        for t in (dirty, dirty_grad):
            t[:5] = bad
            t[900:] = bad
        out = torch.full_like(x, 7.0)
        y, m, r = engine.group_norm(dirty, 6, weight, bias, off, out=out)
        assert y is out and torch.equal(y[5:900], want[0][5:900]) and torch.equal(m, want[1]) and torch.equal(r, want[2])
        assert bool((y[:5] == 7).all()) and bool((y[900:] == 7).all())
        out = torch.full_like(x, 7.0)
        dx, dw, db = engine.group_norm_backward(dirty_grad, dirty, m, r, 6, weight, bias, off, out=out)
        assert dx is out and torch.equal(dx[5:900], grads[0][5:900]) and torch.equal(dw, grads[1]) and torch.equal(db, grads[2])
        assert bool((dx[:5] == 7).all()) and bool((dx[900:] == 7).all())


@gpu
def test_offsets_that_do_not_ascend_touch_nothing_outside():
    """Wrong results at worst: everything next to the arrays stays what it was."""
    import torch
    from mask_b200 import engine
    guard = torch.full((1200 + 200, 48), 5.0, device="cuda")
    inner = guard[100:1300]
    x, grad, weight, bias = _inputs(1200, 48, "f32", 9)
    for offsets in ([900, 100, 2 ** 31 - 1, -5, 700], [2 ** 31 - 1, 2 ** 31 - 1, 0], [-2 ** 31, -1, -1]):
        off = torch.tensor(offsets, dtype=torch.int32, device="cuda")
        _, m, r = engine.group_norm(x, 6, weight, bias, off, out=inner)
        engine.group_norm_backward(grad, x, m, r, 6, weight, bias, off, out=inner)
        torch.cuda.synchronize()
        assert bool((guard[:100] == 5).all()) and bool((guard[1300:] == 5).all())


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_strides_and_in_place(dtype):
    import torch
    from mask_b200 import engine
    rows, channels = 500, 64
    x, grad, weight, bias = _inputs(rows, channels, dtype, 10)
    want = engine.group_norm(x, 8, weight, bias, activation="silu")
    grads = engine.group_norm_backward(grad, x, want[1], want[2], 8, weight, bias, activation="silu")
    for pad, shift in ((16, 8), (3, 1)):
        wide = [torch.full((rows, channels + pad), float("nan"), device="cuda", dtype=x.dtype) for _ in range(3)]
        xs, gs, out = (t[:, shift:shift + channels] for t in wide)
        xs.copy_(x)
        gs.copy_(grad)
        y, m, r = engine.group_norm(xs, 8, weight, bias, activation="silu", out=out)
        _check_forward(x, 8, weight, bias, activation="silu", got=(y, m, r))
        assert bool(wide[2][:, :shift].isnan().all()) and bool(wide[2][:, shift + channels:].isnan().all())
        got = engine.group_norm_backward(gs, xs, want[1], want[2], 8, weight, bias, activation="silu", out=out)
        _check_backward(grad, x, want[1], want[2], 8, weight, bias, activation="silu", got=got)
    for which in (0, 1):
        a, b = x.clone(), grad.clone()
        dx = engine.group_norm_backward(b, a, want[1], want[2], 8, weight, bias, activation="silu", out=(a, b)[which])[0]
        assert torch.equal(dx, grads[0])
    a = x.clone()
    assert torch.equal(engine.group_norm(a, 8, weight, bias, activation="silu", out=a)[0], want[0])


@gpu
def test_no_rows():
    import torch
    from mask_b200 import engine
    x = torch.empty(0, 12, device="cuda")
    y, m, r = engine.group_norm(x, 3)
    assert y.shape == (0, 12) and bool((m == 0).all()) and m.shape == (1, 3)
    dx, dw, db = engine.group_norm_backward(x, x, m, r, 3)
    assert dx.shape == (0, 12) and bool((dw == 0).all()) and bool((db == 0).all())


@gpu
@pytest.mark.parametrize("rows,batch", [(1200, "ragged"), (1000, None), (60, None), (9000, None)])
def test_another_stream_captured_graphs_and_repeats(rows, batch):
    import torch
    from mask_b200 import engine
    x, grad, weight, bias = _inputs(rows, 80, "bf16", 11)
    other = _inputs(rows, 80, "bf16", 12)[:2]
    off = None if batch is None else torch.tensor(BATCHES[batch], dtype=torch.int32, device="cuda")

    def step(a, g):
        y, m, r = engine.group_norm(a, 10, weight, bias, off, activation="relu")
        return (y, m, r, *engine.group_norm_backward(g, a, m, r, 10, weight, bias, off, activation="relu"))
    want, want_other = step(x, grad), step(*other)
    for _ in range(3):
        for a, b in zip(step(x, grad), want):
            assert torch.equal(a, b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(x, grad)
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    static, graphs, outs = [x.clone(), grad.clone()], [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(*static))
        graphs.append(g)
    for source, expected in ((other, want_other), ((x, grad), want)):
        for s, t in zip(static, source):
            s.copy_(t)
        for g in graphs:
            g.replay()
        eager = step(*source)
        for got in (*outs, eager):
            for a, b in zip(got, expected):
                assert torch.equal(a, b)


@gpu
def test_gradients_against_differences():
    import torch
    from mask_b200 import engine
    x, grad, weight, bias = _inputs(40, 12, "f32", 13)
    offsets = [0, 15, 40]
    off = torch.tensor(offsets, dtype=torch.int32, device="cuda")
    _, m, r = engine.group_norm(x, 3, weight, bias, off, activation="silu")
    got = engine.group_norm_backward(grad, x, m, r, 3, weight, bias, off, activation="silu")

    def loss(x, w, b):
        out = [torch.nn.functional.group_norm(x[lo:hi].t()[None], 3, w, b, 1e-5)[0].t() for lo, hi in zip(offsets, offsets[1:])]
        return (torch.nn.functional.silu(torch.cat(out)) * grad.double()).sum()
    step = 1e-6
    for which, at in ((0, (3, 5)), (0, (39, 11)), (1, (4,)), (2, (9,))):
        ends = []
        for sign in (1, -1):
            v = [t.double().clone() for t in (x, weight, bias)]
            v[which][at] += sign * step
            ends.append(float(loss(*v)))
        slope = (ends[0] - ends[1]) / (2 * step)
        # differences: 2^-52 of a loss below 100 over the step; float32 sums of at most 500 terms of size about 1
        assert abs(float(got[which][at]) - slope) < 1e-7 + 200 * U * (abs(slope) + 1)


# ---- refusals ------------------------------------------------------------------------------------------------
def _norm(**changes):
    buffer = (C.c_char * 4096).from_buffer(bytearray(4096))
    at = (C.addressof(buffer) + 255) // 256 * 256
    norm = _lib.Norm(dtype=0, activation=0, rows=4, channels=8, groups=2, graphs=1, eps=1e-5, x=at, x_stride=8, y=at, y_stride=8, mean=at, rstd=at,
                     grad=at, grad_stride=8)
    for k, v in changes.items():
        setattr(norm, k, v)
    return norm, buffer, at


@pytest.mark.parametrize("changes,says", [
    (dict(dtype=3), b"dtype"), (dict(activation=3), b"activation"), (dict(rows=-1), b"rows"), (dict(rows=2 ** 31), b"rows"), (dict(channels=0), b"channels"),
    (dict(channels=2 ** 20 + 2), b"channels"), (dict(groups=3), b"multiple"), (dict(groups=0), b"multiple"), (dict(graphs=0), b"graphs"),
    (dict(graphs=2), b"offsets"), (dict(eps=-1.0), b"eps"), (dict(eps=float("nan")), b"eps"), (dict(x=None), b"NULL"), (dict(mean=None), b"NULL"),
    (dict(x_stride=-8), b"strides"), (dict(y_stride=7), b"overlap"),
])
@pytest.mark.parametrize("backward", [0, 1])
def test_bad_arguments_are_refused_before_anything_is_launched(changes, says, backward):
    L = _lib.lib()
    norm, buffer, at = _norm(**changes)
    assert L.mask_group_norm_scratch_bytes(C.byref(norm), backward) == 0
    assert (L.mask_group_norm_backward if backward else L.mask_group_norm)(C.byref(norm), at, 1 << 40, None) == 1
    assert says in L.mask_last_error()


def test_scratch_and_alignment_are_checked():
    L = _lib.lib()
    norm, buffer, at = _norm()
    for backward, call in ((0, L.mask_group_norm), (1, L.mask_group_norm_backward)):
        need = L.mask_group_norm_scratch_bytes(C.byref(norm), backward)
        assert need > 0
        assert call(C.byref(norm), at, need - 1, None) == 4
        assert call(C.byref(norm), at + 16, need, None) == 1
        assert call(None, at, need, None) == 1
        for name in ("x", "y", "mean", "rstd", "weight", "bias", "offsets") + (("grad", "dweight", "dbias") if backward else ()):
            bad, buffer2, at2 = _norm()
            setattr(bad, name, at2 + 2)
            assert call(C.byref(bad), at2, need, None) == 1 and b"aligned" in L.mask_last_error(), name
    norm, buffer, at = _norm(grad=None)
    assert L.mask_group_norm_scratch_bytes(C.byref(norm), 0) > 0 and L.mask_group_norm_scratch_bytes(C.byref(norm), 1) == 0
    norm, buffer, at = _norm(y=None)
    assert L.mask_group_norm_scratch_bytes(C.byref(norm), 0) == 0 and L.mask_group_norm_scratch_bytes(C.byref(norm), 1) > 0


def test_engine_refuses_tensors_that_are_not_on_the_gpu():
    import torch
    from mask_b200 import engine
    x = torch.zeros(4, 8)
    with pytest.raises(RuntimeError, match="x must be a CUDA tensor"):
        engine.group_norm(x, 2)
    with pytest.raises(RuntimeError, match="x must be a CUDA tensor"):
        engine.group_norm_backward(x, x, x, x, 2)
    with pytest.raises(RuntimeError, match="activation must be one of"):
        engine.group_norm(x, 2, activation="tanh")


@gpu
def test_engine_refusals():
    import torch
    from mask_b200 import engine
    x, grad, weight, bias = _inputs(20, 24, "f32")
    off = torch.tensor([0, 20], dtype=torch.int32, device="cuda")
    for args, more, says in (((x, 5), {}, "24 channels are not a multiple of 5"), ((x, 0), {}, "multiple"), ((x.double(), 4), {}, "x must be float32"),
                             ((x[0], 4), {}, "dense 2-D"), ((x.t(), 4), {}, "rows of x"), ((x, 4, weight[:23]), {}, "weight must be contiguous float32"),
                             ((x, 4, weight, bias.bfloat16()), {}, "bias must be contiguous float32"), ((x, 4, weight.cpu()), {}, "weight must be a CUDA"),
                             ((x, 4), dict(offsets=off.long()), "offsets must be"), ((x, 4), dict(offsets=off[:1]), "offsets must be"),
                             ((x, 4), dict(eps=-1.0), "eps"), ((x, 4), dict(out=torch.empty(20, 23, device="cuda")), "out must have"),
                             ((x, 4), dict(out=x.bfloat16()), "out must have"), ((x, 4), dict(out=x[:1].expand(20, 24)), "rows of out")):
        with pytest.raises(RuntimeError, match=says):
            engine.group_norm(*args, **more)
    _, m, r = engine.group_norm(x, 4)
    for args, says in (((grad[:19], x, m, r, 4), "grad must have"), ((grad.bfloat16(), x, m, r, 4), "grad must have"), ((grad, x, m[:, :3], r, 4), "mean must be"),
                       ((grad, x, m, r.double(), 4), "rstd must be"), ((grad, x, m, r, 8), "mean must be"), ((grad.cpu(), x, m, r, 4), "grad must be a CUDA")):
        with pytest.raises(RuntimeError, match=says):
            engine.group_norm_backward(*args)


@gpu
def test_offsets_beyond_32_bits():
    """2.5 thousand million values: the last graph's rows lie behind 2^31 elements."""
    import torch
    from mask_b200 import engine
    rows, channels = (1 << 22) + 3, 600
    g = torch.Generator(device="cuda").manual_seed(31)
    x = torch.empty(rows, channels, device="cuda", dtype=torch.bfloat16)
    for part in x.split(1 << 20):
        part.copy_(torch.randn(part.shape, generator=g, device="cuda"))
    offsets = [0, rows - 1000, rows]
    off = torch.tensor(offsets, dtype=torch.int32, device="cuda")
    y, m, r = engine.group_norm(x, 30, offsets=off, activation="silu")
    _check_forward(x[-1000:], 30, None, None, activation="silu", got=(y[-1000:], m[1:], r[1:]))
    # a mean over 84 million values of unit variance is within 1e-3 of 0, the deviation within 1e-3 of 1
    assert float(m[0].abs().max()) < 1e-3 and float((r[0] - 1).abs().max()) < 1e-3
    want = torch.nn.functional.silu((x[-2000:-1000].double().reshape(1000, 30, 20) - m[0].double()[:, None]) * r[0].double()[:, None]).reshape(1000, 600)
    assert float((y[-2000:-1000].double() - want).abs().max()) < 0.03        # half a step of bfloat16 at 5 or so
    dx, dw, db = engine.group_norm_backward(y, x, m, r, 30, offsets=off, activation="silu")
    part = engine.group_norm_backward(y[-1000:].contiguous(), x[-1000:].contiguous(), m[1:].contiguous(), r[1:].contiguous(), 30, activation="silu")
    assert float((dx[-1000:].double() - part[0].double()).abs().max()) < 0.03
    assert bool(torch.isfinite(dw).all()) and bool(torch.isfinite(db).all())
