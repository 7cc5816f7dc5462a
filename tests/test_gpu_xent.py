"""The classifier head (``engine.linear_cross_entropy``) against its definition in 64 bits.

Tolerances are sums of what each step may be off by:
  * float32 operands are scaled by a power of two and taken as two float16 parts: x = hi + lo + e with |e| <= 2^-22 |x| or
    2^-40 of the largest |x|, and of the four products of parts lo lo (2^-22) is dropped: 2^-20 |x y| in all, and 2^-39 of the
    largest; 16-bit operands are multiplied exactly;
  * float32 sums: at most one unit in the last place (2^-23 of what has been summed) for each step of 16 products -- with
    float32 operands 48 such steps at most, then one for each 256 of the contraction -- and one for each part, of 64 of the contraction at least, of at most 600;
  * the gradient of the logits: its logit's and log sum's errors (each the largest of a row's logits'), the exponential's
    (2^-20) and, between the products, one rounding (2^-8 bfloat16; 2^-11 float16, or 2^-25 below its normal range; 2^-22 or
    2^-40 for two parts);
  * the results' own rounding.
"""
import ctypes as C
import itertools

import pytest

from mask_b200 import _lib

gpu = pytest.mark.gpu


def _dtype(name):
    import torch
    return {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[name]


def _inputs(rows, dim, classes, dtype, layout="dim", labelled="all", seed=0):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    hidden = torch.randn(rows, dim, generator=g, device="cuda").to(_dtype(dtype))
    weight = (torch.randn(classes, dim, generator=g, device="cuda") * (2.0 / dim ** 0.5)).to(_dtype(dtype))
    weight = weight.t() if layout == "dim" else weight.t().contiguous()
    labels = torch.randint(0, classes, (rows,), generator=g, device="cuda")
    if labelled == "none":
        labels.fill_(-1)
    elif labelled == "last":
        labels[:-1] = -1
    elif labelled == "some":
        labels[torch.rand(rows, generator=g, device="cuda") < 0.6] = -100
        labels[::7] = classes                   # one past the last class
    return hidden, weight, labels


def _want(hidden, weight, labels, reduction="mean", scale=1.0):
    """(loss, its tolerance), (dhidden, ...), (dweight, ...) in 64 bits."""
    import torch
    f32, dim, classes = hidden.dtype == torch.float32, weight.shape[0], weight.shape[1]
    keep = (labels >= 0) & (labels < classes)
    h, w = hidden[keep].double(), weight.double()
    y, n = labels[keep], int(keep.sum())
    rel, least = (2.0 ** -20, 2.0 ** -39) if f32 else (0.0, 0.0)
    steps = lambda k: 2.0 ** -23 * ((min(3 * (k / 16 + 1), 48) + k / 256 if f32 else k / 16 + 1) + min(k / 64 + 1, 600))   # noqa: E731
    most = lambda x: float(x.abs().max()) if x.numel() else 0.0   # noqa: E731
    logits = h @ w
    elogit = (h.abs() @ w.abs()).mul_(rel + steps(dim)) + least * (most(h) * w.abs().sum(0) + most(w) * h.abs().sum(1, keepdim=True))
    erow = elogit.amax(1, keepdim=True) if n else elogit.sum(1, keepdim=True)
    lse = torch.logsumexp(logits, 1, keepdim=True)
    rows = (lse - logits.gather(1, y[:, None])).squeeze(1)
    erows = (2 * erow + 2.0 ** -20 * (1 + lse.abs())).squeeze(1)
    p = (logits - lse).exp()
    hot = torch.zeros_like(p).scatter_(1, y[:, None], 1.0)
    g = p - hot
    # the exponent's argument is rounded too: 2^-23 of the logit and of the log sum
    eg = p * (2 * erow + 2.0 ** -20 + 2.0 ** -22 * (logits.abs() + lse.abs())).expm1() + 2.0 ** -23 * hot
    eg += g.abs() * (2.0 ** -22 if f32 else 2.0 ** -8 if hidden.dtype == torch.bfloat16 else 2.0 ** -11)
    eg += 2.0 ** -40 if f32 else 0.0 if hidden.dtype == torch.bfloat16 else 2.0 ** -25
    if reduction == "mean" and n:
        scale = scale / n
    out = 2.0 ** -23 if f32 else torch.finfo(hidden.dtype).eps / 2
    tiny = 2.0 ** -25 if hidden.dtype == torch.float16 else 2.0 ** -134
    dh = torch.zeros(hidden.shape, dtype=torch.float64, device="cuda")
    eh = torch.zeros_like(dh)
    dh[keep] = scale * (g @ w.t())
    eh[keep] = abs(scale) * (eg @ w.abs().t() + (g.abs() @ w.abs().t()) * (rel + steps(classes)) + least * most(w) * g.abs().sum(1, keepdim=True))
    dw = scale * (h.t() @ g)
    ew = abs(scale) * (h.abs().t() @ eg + (h.abs().t() @ g.abs()) * (rel + steps(n)) + least * most(h) * g.abs().sum(0))
    eh, ew = eh * 1.01 + out * dh.abs() + tiny * keep[:, None], ew * 1.01 + out * dw.abs() + tiny
    if reduction == "none":
        loss, eloss = torch.zeros(len(labels), dtype=torch.float64, device="cuda"), torch.zeros(len(labels), dtype=torch.float64, device="cuda")
        loss[keep], eloss[keep] = rows, erows
    else:
        over = n if reduction == "mean" and n else 1
        loss, eloss = rows.sum() / over, erows.sum() / over + 2.0 ** -23 * rows.sum() / over
    return (loss, eloss), (dh, eh), (dw, ew)


def _check(got, want, what):
    import torch
    value, tolerance = want
    assert got.shape == value.shape, what
    off = (got.double() - value).abs() - tolerance
    assert bool((off <= 0).all()), (what, float(off.max()), float(tolerance.max()), int((off > 0).sum()), torch.nonzero(off > 0)[:4].tolist())


def _both(hidden, weight, labels, reduction="mean", scale=1.0):
    from mask_b200 import engine
    want = _want(hidden, weight, labels, reduction, scale)
    got = engine.linear_cross_entropy(hidden, weight, labels, reduction=reduction, grads=True, grad_scale=scale)
    for g, w, what in zip(got, want, ("loss", "dhidden", "dweight")):
        _check(g, w, what)
    _check(engine.linear_cross_entropy(hidden, weight, labels, reduction=reduction), want[0], "loss alone")
    return got


SIZES = [(1, 1, 1), (1, 16, 7), (5, 3, 2), (128, 64, 64), (129, 65, 65), (127, 200, 128), (300, 33, 129), (257, 128, 256), (300, 72, 257),
         (1000, 200, 1000), (64, 512, 5003), (2000, 1024, 300), (40, 1100, 40), (17, 320, 513)]


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,dim,classes", SIZES)
def test_sizes(rows, dim, classes, dtype):
    layout = "dim" if (rows + classes) % 2 else "class"
    _both(*_inputs(rows, dim, classes, dtype, layout), scale=1024.0 if dtype == "f16" else 1.0)


@gpu
@pytest.mark.parametrize("classes", [47, 700])
@pytest.mark.parametrize("labelled", ["none", "last", "some"])
@pytest.mark.parametrize("reduction", ["none", "mean", "sum"])
def test_labels(reduction, labelled, classes):
    for dtype, layout in (("f32", "class"), ("bf16", "dim")):
        hidden, weight, labels = _inputs(517, 96, classes, dtype, layout, labelled, seed=3)
        loss, dhidden, dweight = _both(hidden, weight, labels, reduction, 0.5)
        out = (labels < 0) | (labels >= classes)
        assert bool((dhidden[out] == 0).all())
        if labelled == "none":
            assert bool((loss == 0).all()) and bool((dweight == 0).all())


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,dim,classes", [(2708, 16, 7), (512, 64, 16), (512, 16, 64), (512, 1024, 1), (1, 1, 1024), (4096, 2, 64), (4097, 2, 60), (700, 5, 150)])
def test_few_products(rows, dim, classes, dtype):
    """Around the sizes up to which one block takes the whole head."""
    for labelled in ("some", "all"):
        _both(*_inputs(rows, dim, classes, dtype, "class" if labelled == "some" else "dim", labelled, seed=6), scale=256.0 if dtype == "f16" else 1.0)


@gpu
@pytest.mark.parametrize("rows", [3000, 70001])
def test_many_chunks_of_labels(rows):
    """More rows than one block numbers, in unequal chunks."""
    _both(*_inputs(rows, 24, 19, "f32", "class", "some", seed=5))


@gpu
def test_no_rows():
    import torch
    from mask_b200 import engine
    for dtype in ("f32", "bf16"):
        hidden, weight, labels = _inputs(0, 40, 300, dtype)
        for reduction in ("mean", "sum", "none"):
            loss, dhidden, dweight = engine.linear_cross_entropy(hidden, weight, labels, reduction=reduction, grads=True)
            assert loss.numel() == (0 if reduction == "none" else 1) and bool((loss == 0).all())
            assert dhidden.shape == (0, 40) and torch.equal(dweight, torch.zeros_like(weight))


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("classes", [33, 400])
def test_what_unlabelled_rows_hold_reaches_nothing(dtype, classes):
    import torch
    from mask_b200 import engine
    hidden, weight, labels = _inputs(400, 70, classes, dtype, labelled="some", seed=7)
    want = engine.linear_cross_entropy(hidden, weight, labels, grads=True)
    out = (labels < 0) | (labels >= classes)
    for bad in (float("nan"), float("inf"), torch.finfo(hidden.dtype).min):
        dirty = hidden.clone()
        dirty[out] = bad
        for a, b in zip(engine.linear_cross_entropy(dirty, weight, labels, grads=True), want):
            assert torch.equal(a, b)


@gpu
@pytest.mark.parametrize("classes", [33, 400])
def test_nan_in_a_labelled_row(classes):
    """Its loss is NaN; the other rows' losses and gradients of hidden are what they were."""
    import torch
    from mask_b200 import engine
    hidden, weight, labels = _inputs(200, 64, classes, "f32", seed=8)
    want = engine.linear_cross_entropy(hidden, weight, labels, reduction="none", grads=True)
    hidden[77, 5] = float("nan")
    loss, dhidden, dweight = engine.linear_cross_entropy(hidden, weight, labels, reduction="none", grads=True)
    other = torch.arange(200, device="cuda") != 77
    assert bool(loss[77].isnan()) and bool(dhidden[77].isnan().all()) and bool(dweight.isnan().any())
    assert torch.equal(loss[other], want[0][other]) and torch.equal(dhidden[other], want[1][other])


@gpu
def test_large_and_small_logits():
    """Logits of some thousands beside rows of zeros, and rows whose label is certain or out of the question."""
    import torch
    for classes in (50, 600):
        hidden, weight, labels = _inputs(150, 64, classes, "f32", seed=9)
        hidden[:50] *= 300.0
        hidden[50:100] = 8.0 * weight.t()[labels[50:100]]
        hidden[100:120] = -8.0 * weight.t()[labels[100:120]]
        hidden[120] = 0.0
        got = _both(hidden, weight, labels, "none")
        assert bool(torch.isfinite(got[0]).all())


@gpu
@pytest.mark.parametrize("classes", [50, 600])
@pytest.mark.parametrize("scale_h,scale_w", [(1e-30, 1e30), (1e25, 1e-26), (3e-39, 1.0), (1e-3, 1e3)])
def test_operands_of_any_magnitude(scale_h, scale_w, classes):
    """float32 operands far from 1, subnormal ones among them."""
    hidden, weight, labels = _inputs(150, 64, classes, "f32", "dim", "some", seed=10)
    _both(hidden * scale_h, weight * scale_w, labels, scale=1e-6)


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_strides(dtype):
    """Rows apart from one another, addresses off 16 bytes, a weight contiguous along neither axis."""
    import torch
    from mask_b200 import engine
    rows, dim, classes = 200, 61, 300
    hidden, weight, labels = _inputs(rows, dim, classes, dtype, "class", "some", seed=11)
    want = engine.linear_cross_entropy(hidden, weight, labels, grads=True)
    wide = torch.full((rows, dim + 9), float("nan"), device="cuda", dtype=hidden.dtype)
    wide[:, 3:3 + dim] = hidden
    table = torch.full((classes, dim + 3), float("nan"), device="cuda", dtype=hidden.dtype)
    table[:, 1:1 + dim] = weight.t()
    spread = torch.full((dim, classes, 2), float("nan"), device="cuda", dtype=hidden.dtype)
    spread[:, :, 1] = weight
    for w in (weight, weight.t().contiguous().t(), table[:, 1:1 + dim].t(), spread[:, :, 1]):
        got = engine.linear_cross_entropy(wide[:, 3:3 + dim], w, labels, grads=True)
        for a, b in zip(got, want):
            assert torch.equal(a, b)


@gpu
@pytest.mark.parametrize("classes,dim", [(47, 80), (1500, 80), (1500, 600), (200, 256)])
def test_another_stream_and_a_captured_graph(classes, dim):
    """Captured, and replayed with other contents in the same buffers while eager calls run beside it."""
    import torch
    from mask_b200 import engine
    hidden, weight, labels = _inputs(700, dim, classes, "f32", "class", "some", seed=13)
    other = _inputs(700, dim, classes, "f32", "class", "all", seed=14)
    want, want_other = (engine.linear_cross_entropy(*x, grads=True) for x in ((hidden, weight, labels), other))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = engine.linear_cross_entropy(hidden, weight, labels, grads=True)
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    static = [t.clone() for t in (hidden, weight, labels)]
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(engine.linear_cross_entropy(*static, grads=True))
        graphs.append(g)
    for source, expected in ((other, want_other), ((hidden, weight, labels), want)):
        for s, t in zip(static, source):
            s.copy_(t)
        for g in graphs:
            g.replay()
        eager = engine.linear_cross_entropy(*source, grads=True)
        for got in (*outs, eager):
            for a, b in zip(got, expected):
                assert torch.equal(a, b)


@gpu
def test_two_streams_at_once():
    """Heads of every kind of tile on two streams, none waiting for the other, against the same one after the other."""
    import torch
    from mask_b200 import engine
    sides = [torch.cuda.Stream() for _ in range(2)]
    problems = [[_inputs(rows, dim, classes, dtype, "class", "some", seed=s + k) for k, (rows, dim, classes, dtype) in
                 enumerate(((2000, 512, 3000, "bf16"), (5000, 64, 40, "f32"), (1500, 300, 700, "f32"), (9000, 640, 500, "f16"), (100, 16, 7, "f32")))]
                for s in (41, 51)]
    wants = [[engine.linear_cross_entropy(*x, grads=True) for x in ps] for ps in problems]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i in range(len(problems[0])):
            for side, ps, out in zip(sides, problems, got):
                with torch.cuda.stream(side):
                    out.append(engine.linear_cross_entropy(*ps[i], grads=True))
    torch.cuda.synchronize()
    for out, want in zip(got, wants):
        for i, result in enumerate(out):
            for a, b in zip(result, want[i % len(want)]):
                assert torch.equal(a, b), i


@gpu
def test_pieces_of_the_classes():
    """More classes than one piece of the gradient of the logits holds (2 GB); long sums on both sides."""
    for dtype, rows in (("f32", 12000), ("bf16", 24000)):
        _both(*_inputs(rows, 48, 50001, dtype, "dim", "some", seed=17))


@gpu
def test_sums_of_many_classes_do_not_drift():
    """A loss is formed from numbers below 32 in bits, rounded twice: 2^-20 ln 2 each.  The sums behind it take thousands of
    steps, none of which may leave a trace of its own: root mean square below 2^-19, small logits that are exact to 2^-22."""
    import torch
    from mask_b200 import engine
    for classes in (20000, 53055):
        hidden, weight, labels = _inputs(95, 18, classes, "f32", seed=27)
        got = engine.linear_cross_entropy(hidden, weight, labels, reduction="none")
        off = got.double() - _want(hidden, weight, labels, "none")[0][0]
        assert float(off.square().mean().sqrt()) < 2.0 ** -19


@gpu
def test_same_call_same_bits():
    import torch
    from mask_b200 import engine
    for rows, dim, classes in ((4000, 64, 47), (900, 128, 5000)):
        x = _inputs(rows, dim, classes, "bf16", labelled="some", seed=19)
        first = engine.linear_cross_entropy(*x, grads=True)
        for _ in range(3):
            for a, b in zip(engine.linear_cross_entropy(*x, grads=True), first):
                assert torch.equal(a, b)


@gpu
def test_gradients_against_differences():
    """Central differences of the definition in 64 bits, for a few entries."""
    import torch
    from mask_b200 import engine
    for classes in (9, 300):
        hidden, weight, labels = _inputs(60, 20, classes, "f32", "class", "some", seed=23)
        _, dhidden, dweight = engine.linear_cross_entropy(hidden, weight, labels, grads=True)
        keep = (labels >= 0) & (labels < classes)

        def loss(h, w):
            return torch.nn.functional.cross_entropy((h @ w)[keep], labels[keep])
        step = 1e-5
        for tensor, grad, which in ((hidden, dhidden, 0), (weight, dweight, 1)):
            for i, j in itertools.product((0, 2, 19), (1, 8)):
                ends = []
                for sign in (1, -1):
                    x = [hidden.double().clone(), weight.double().clone()]
                    x[which][i, j] += sign * step
                    ends.append(float(loss(*x)))
                slope = (ends[0] - ends[1]) / (2 * step)
                # differences: step^2 times the third derivative (below 1) and 2^-53 / step; the kernel: float32 products
                assert abs(float(grad[i, j]) - slope) < 1e-9 + 1e-10 + 2.0 ** -12 * (abs(slope) + 1e-2)


# ---- refusals --------------------------------------------------------------------------------------------
def _head(**changes):
    buffer = (C.c_char * 4096).from_buffer(bytearray(4096))
    at = (C.addressof(buffer) + 255) // 256 * 256
    head = _lib.Head(dtype=0, reduction=1, rows=4, dim=4, classes=4, hidden=at, hidden_stride=4, weight=at, weight_dim_stride=4,
                     weight_class_stride=1, labels=at, loss=at, grad_scale=1.0, dhidden=at, dhidden_stride=4, dweight=at,
                     dweight_dim_stride=4, dweight_class_stride=1)
    for k, v in changes.items():
        setattr(head, k, v)
    return head, buffer, at


@pytest.mark.parametrize("changes,says", [
    (dict(dtype=3), b"dtype"), (dict(dtype=-1), b"dtype"), (dict(reduction=7), b"reduction"), (dict(rows=-1), b"rows"), (dict(rows=2 ** 31 - 256), b"rows"),
    (dict(dim=0), b"dim"), (dict(classes=0), b"classes"), (dict(classes=2 ** 31 - 256), b"classes"), (dict(hidden=None), b"NULL"), (dict(weight=None), b"NULL"),
    (dict(labels=None), b"NULL"), (dict(loss=None), b"loss"), (dict(hidden_stride=-1), b"strides"), (dict(dweight_dim_stride=-4), b"strides"),
    (dict(dhidden_stride=3), b"overlap"),
])
def test_bad_arguments_are_refused_before_anything_is_launched(changes, says):
    L = _lib.lib()
    head, buffer, at = _head(**changes)
    assert L.mask_linear_xent_scratch_bytes(C.byref(head)) == 0
    assert L.mask_linear_xent(C.byref(head), at, 1 << 40, None) == 1
    assert says in L.mask_last_error()


def test_misaligned_operands_and_small_scratch_are_refused():
    L = _lib.lib()
    head, buffer, at = _head()
    need = L.mask_linear_xent_scratch_bytes(C.byref(head))
    assert need > 0
    assert L.mask_linear_xent(C.byref(head), at, need - 1, None) == 4
    assert L.mask_linear_xent(C.byref(head), at + 16, need, None) == 1 and b"scratch" in L.mask_last_error()
    assert L.mask_linear_xent(C.byref(head), None, need, None) == 1
    assert L.mask_linear_xent(None, at, need, None) == 1 and L.mask_linear_xent_scratch_bytes(None) == 0
    for name, by in (("hidden", 2), ("weight", 1), ("dhidden", 2), ("dweight", 2), ("loss", 2), ("labels", 4)):
        head, buffer, at = _head()
        setattr(head, name, at + by)
        assert L.mask_linear_xent(C.byref(head), at, need, None) == 1 and b"aligned" in L.mask_last_error(), name


def test_scratch_is_bounded_by_the_pieces_not_by_the_logits():
    L = _lib.lib()
    head, buffer, at = _head(dtype=1, rows=1 << 17, dim=512, classes=1 << 20, weight_dim_stride=1, weight_class_stride=512,
                              hidden_stride=512, dhidden_stride=512, dweight_dim_stride=1, dweight_class_stride=512)
    logits = (1 << 17) * (1 << 20) * 2
    assert 0 < L.mask_linear_xent_scratch_bytes(C.byref(head)) < logits // 100


def test_engine_refuses_tensors_that_are_not_on_the_gpu():
    import torch
    from mask_b200 import engine
    with pytest.raises(RuntimeError, match="hidden must be a CUDA tensor"):
        engine.linear_cross_entropy(torch.zeros(2, 2), torch.zeros(2, 2), torch.zeros(2, dtype=torch.int64))
    with pytest.raises(RuntimeError, match="reduction must be one of"):
        engine.linear_cross_entropy(torch.zeros(2, 2), torch.zeros(2, 2), torch.zeros(2, dtype=torch.int64), reduction="median")


@gpu
def test_engine_refusals():
    import torch
    from mask_b200 import engine
    hidden, weight, labels = _inputs(6, 8, 5, "f32")
    call = engine.linear_cross_entropy
    for args, says in (((hidden.cpu(), weight, labels), "hidden must be a CUDA tensor"), ((hidden, weight.cpu(), labels), "weight must be a CUDA"),
                       ((hidden, weight, labels.cpu()), "labels must be a CUDA"), ((hidden[0], weight, labels), "hidden must be a dense 2-D"),
                       ((hidden, weight[0], labels), "weight must be a dense 2-D"), ((hidden, weight, labels[:, None]), "labels must be a dense 1-D"),
                       ((hidden.double(), weight, labels), "hidden must be float32"), ((hidden.bfloat16(), weight, labels), "weight must have hidden's dtype"),
                       ((hidden, weight, labels.int()), "labels must be int64"), ((hidden, weight[:7], labels), "weight has 7 rows"),
                       ((hidden, weight, labels[:5]), "5 labels for 6 rows"), ((hidden.t().contiguous().t(), weight, labels), "rows of hidden"),
                       ((hidden, weight, labels.repeat_interleave(2)[::2]), "labels must be contiguous"), ((hidden, weight[:, :0], labels), "at least one"),
                       ((hidden.to_sparse(), weight, labels), "hidden must be a dense")):
        with pytest.raises(RuntimeError, match=says):
            call(*args)
    assert torch.isfinite(call(hidden, weight, labels))


@gpu
@pytest.mark.parametrize("classes", [16, 300])
def test_offsets_beyond_32_bits(classes):
    """2.2 thousand million features: rows behind 2^31 elements, every other one labelled; rows do not depend on one another."""
    import torch
    from mask_b200 import engine
    rows, dim = (1 << 22) + 5, 520
    g = torch.Generator(device="cuda").manual_seed(37)
    hidden = torch.empty(rows, dim, device="cuda", dtype=torch.bfloat16)
    for part in hidden.split(1 << 20):
        part.copy_(torch.randn(part.shape, generator=g, device="cuda"))
    weight = (torch.randn(classes, dim, generator=g, device="cuda") * (2.0 / dim ** 0.5)).bfloat16().t()
    labels = torch.randint(0, classes, (rows,), generator=g, device="cuda")
    labels[::2] = -1
    loss, dhidden, dweight = engine.linear_cross_entropy(hidden, weight, labels, reduction="none", grads=True)
    tail = slice(rows - 1000, rows)
    want = _want(hidden[tail], weight, labels[tail], "none")
    _check(loss[tail], want[0], "loss")
    _check(dhidden[tail], want[1], "dhidden")
    assert bool(torch.isfinite(dweight).all()) and bool((loss[::2] == 0).all())
