"""The classifier head (``engine.linear_cross_entropy``) where its numbers leave the ordinary range: logits that vanish or pass
what a float32 holds, infinite weights, probabilities below float16's range, contractions of many rows, and features beyond 2^31
values, against the definition in 64 bits.  What each step may be off by is in test_gpu_xent.py, whose oracle is used here."""
import math

import pytest

from tests.test_gpu_xent import _both, _check, _inputs, _want

gpu = pytest.mark.gpu


@gpu
@pytest.mark.parametrize("classes", [12, 50, 600])
@pytest.mark.parametrize("scale_h,scale_w", [(0.0, 0.0), (1e-10, 0.0), (0.0, 1.0), (1e-20, 1e-20), (1e-38, 1e-30), (1e-38, 1e-38)])
def test_logits_that_vanish(scale_h, scale_w, classes):
    """Every class alike: the loss is log(classes), whatever way the sizes take."""
    import torch
    hidden, weight, labels = _inputs(150, 64, classes, "f32", "dim", "some", seed=10)
    loss, dhidden, dweight = _both(hidden * scale_h, weight * scale_w, labels)
    assert abs(float(loss) - math.log(classes)) < 2.0 ** -20 * (1 + math.log(classes))
    assert bool(torch.isfinite(dhidden).all()) and bool(torch.isfinite(dweight).all())


def _far_operands(classes):
    """Logits of row 0: 2^180 for class 0, else 0; of the others: 2^120 for odd classes, else 0."""
    import torch
    hidden = torch.zeros(70, 64, device="cuda")
    weight = torch.zeros(64, classes, device="cuda")
    hidden[0, 0], hidden[1:, 1] = 2.0 ** 120, 2.0 ** 90
    weight[0, 0], weight[1, 1::2] = 2.0 ** 60, 2.0 ** 30
    return hidden, weight, torch.arange(70, device="cuda") % classes


@gpu
@pytest.mark.parametrize("classes", [50, 600])
def test_logits_beyond_a_float(classes):
    """Infinite ones are their row's alone; a label's that is far below the largest keeps its size."""
    import torch
    from mask_b200 import engine
    hidden, weight, labels = _far_operands(classes)
    loss = engine.linear_cross_entropy(hidden, weight, labels, reduction="none")
    assert bool(loss[0].isnan())
    # largest logit 0, the label's -2^120 with the same operands' scales
    hidden[1:, 1] *= -1
    loss, dhidden, dweight = engine.linear_cross_entropy(hidden, weight, labels, reduction="none", grads=True)
    assert bool(loss[0].isnan()) and bool(dhidden[0].isnan().any())
    odd = labels[1:] % 2 == 1
    even = (classes + 1) // 2
    assert float((loss[1:][odd] / 2.0 ** 120 - 1).abs().max()) < 2.0 ** -20
    assert float((loss[1:][~odd] - math.log(even)).abs().max()) < 2.0 ** -20 * 8


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("classes", [50, 600])
def test_logits_that_no_exponent_tells_apart(classes, dtype):
    """Beyond 2^31 a row's loss and gradients are NaN, not any number; the other rows' are theirs.  Logits of a million
    are taken."""
    import torch
    from mask_b200 import engine
    hidden, weight, labels = _inputs(90, 64, classes, dtype, seed=12)
    hidden[40:] *= 2.0 ** 36
    loss, dhidden, dweight = engine.linear_cross_entropy(hidden, weight, labels, reduction="none", grads=True)
    far = (hidden.double() @ weight.double()).amax(1).abs() > 2.0 ** 31
    assert bool(far[40:].any()) and not bool(far[:40].any())
    assert bool(loss[far].isnan().all()) and bool(dhidden[far].isnan().all()) and bool(torch.isfinite(loss[:40]).all())
    if dtype == "bf16":         # operands are what they are; float32 ones are exact to 2^-40 of the largest
        want = _want(hidden[:40], weight, labels[:40], "none")
        _check(loss[:40], want[0], "loss")
        _check(dhidden[:40], want[1], "dhidden")
    hidden, weight, labels = _inputs(90, 64, classes, dtype, seed=12)
    hidden[:40] *= 2.0 ** 20
    got = engine.linear_cross_entropy(hidden, weight, labels, reduction="none")
    _check(got, _want(hidden, weight, labels, "none")[0], "loss")


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_small_heads_take_logits_of_any_size(dtype):
    """They subtract logits before anything is rounded to bits: any finite one has its loss."""
    import torch
    from mask_b200 import engine
    hidden, weight, labels = _inputs(90, 64, 12, dtype, seed=12)
    hidden[40:] *= 2.0 ** 36 if dtype != "f16" else 2.0 ** 12
    loss, dhidden, dweight = engine.linear_cross_entropy(hidden, weight, labels, reduction="none", grads=True)
    _check(loss, _want(hidden, weight, labels, "none")[0], "loss")
    assert bool(torch.isfinite(dhidden).all()) and bool(torch.isfinite(dweight.float()).all() or dtype == "f16")


MASKED = [(100, 16, 20), (150, 64, 50), (300, 64, 600), (129, 200, 300)]


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,dim,classes", MASKED)
@pytest.mark.parametrize("layout", ["dim", "class"])
def test_classes_masked_by_minus_infinity(rows, dim, classes, dtype, layout):
    """A feature that is 1 and whose weight is -inf takes classes out: probability 0, whatever way the sizes take.  What is
    multiplied with that weight, the feature's own gradient, is 0 times infinity."""
    import torch
    from mask_b200 import engine
    hidden, weight, labels = _inputs(rows, dim, classes, dtype, "dim", "some", seed=15)
    hidden[:, dim - 1] = 1.0
    masked = torch.arange(classes, device="cuda") % 3 == 1
    labels[(labels >= 0) & (labels < classes) & (labels % 3 == 1)] = 0
    out = weight.clone()
    out[dim - 1, masked] = -math.inf
    out = out.t().contiguous().t() if layout == "dim" else out.contiguous()
    kept = torch.nonzero(~masked).squeeze(1)
    place = torch.full((classes,), -1, dtype=torch.int64, device="cuda")
    place[kept] = torch.arange(len(kept), device="cuda")
    real = (labels >= 0) & (labels < classes)
    fewer = torch.where(real, place[labels.clamp(0, classes - 1)], -1)
    want = _want(hidden, weight[:, kept], fewer, "sum")
    for got in (engine.linear_cross_entropy(hidden, out, labels, reduction="sum"),
                engine.linear_cross_entropy(hidden, out, labels, reduction="sum", grads=True)[0]):
        _check(got, want[0], "loss")
    _, dhidden, dweight = engine.linear_cross_entropy(hidden, out, labels, reduction="sum", grads=True)
    _check(dweight[:, kept], want[2], "dweight")
    assert bool((dweight[:, masked] == 0).all())
    _check(dhidden[:, :dim - 1], tuple(t[:, :dim - 1] for t in want[1]), "dhidden")
    assert bool(dhidden[real, dim - 1].isnan().all()) and bool((dhidden[~real] == 0).all())
    # a label that is masked: the loss is infinite
    at = int(torch.nonzero(real)[0])
    labels[at] = 1
    loss = engine.linear_cross_entropy(hidden, out, labels, reduction="none")
    assert float(loss[at]) == math.inf


@gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("rows,dim,classes", MASKED)
def test_classes_masked_by_the_lowest_value(rows, dim, classes, dtype):
    """In 16 bits the lowest value is as good: products with it are exact."""
    import torch
    hidden, weight, labels = _inputs(rows, dim, classes, dtype, "dim", "some", seed=16)
    hidden[:, dim - 1] = 1.0
    masked = torch.arange(classes, device="cuda") % 3 == 1
    labels[(labels >= 0) & (labels < classes) & (labels % 3 == 1)] = 0
    weight = weight.clone()
    weight[dim - 1, masked] = torch.finfo(weight.dtype).min
    from mask_b200 import engine
    loss, dhidden, dweight = engine.linear_cross_entropy(hidden, weight, labels, grads=True)
    kept = torch.nonzero(~masked).squeeze(1)
    real = (labels >= 0) & (labels < classes)
    logits = hidden[real].double() @ weight.double()
    want = torch.nn.functional.cross_entropy(logits, labels[real])
    assert abs(float(loss) - float(want)) < 2.0 ** -16 * (1 + float(want))
    assert bool(torch.isfinite(dhidden).all()) and bool((dweight[:, masked] == 0).all())
    g = torch.softmax(logits, 1)
    g[torch.arange(len(g)), labels[real]] -= 1.0
    dw = hidden[real].double().t() @ g / len(g)
    # two roundings to 8 or 11 bits: of the logits' gradient and of the result
    step = torch.finfo(weight.dtype).eps / 2
    bound = (hidden[real].double().abs().t() @ g.abs() / len(g) + dw.abs()) * (step + 2.0 ** -16) + 2.0 ** -24
    assert bool(((dweight.double() - dw).abs()[:, kept] <= bound[:, kept]).all())


@gpu
def test_probabilities_below_the_range_of_float16():
    """Logits of deviation 4 over 60000 classes: most probabilities are below 2^-25.  Columns of dweight that are nobody's label
    are sums of them; two roundings, of the logits' gradient and of the result, leave at most 2^-11 each of a column that one
    term makes up and less of one with more, beside 2^-18 of the logits' and the exponential's."""
    import torch
    from mask_b200 import engine
    hidden, weight, labels = _inputs(256, 64, 60000, "f16", seed=18)
    weight = (2.0 * weight.t().float()).half().t()
    labels %= 1000
    _, dhidden, dweight = engine.linear_cross_entropy(hidden, weight, labels, reduction="sum", grads=True, grad_scale=2.0 ** 12)
    p = torch.softmax(hidden.double() @ weight.double(), 1)
    want = 2.0 ** 12 * (hidden.double().t() @ p)[:, 1000:]
    off = (dweight[:, 1000:].double() - want).norm(dim=0)
    # values of dweight below 2^-14 are rounded to 2^-24
    assert float((off - 2.0 ** -25 * 8.0).div(want.norm(dim=0)).max()) < 2.0 ** -10 + 2.0 ** -17


@gpu
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_sums_over_many_rows_are_not_cut_short(dtype):
    """The tensor core cuts its sum off toward zero after every 16 products; where all terms have one sign that adds up, 16384
    times for 2^18 rows of positive features (1.7e-3).  A quarter of the result's own rounding is granted."""
    import torch
    from mask_b200 import engine
    rows, dim, classes = 1 << 18, 1024, 4096
    hidden, weight, labels = _inputs(rows, dim, classes, dtype, seed=20)
    hidden.abs_()
    labels %= 16
    dweight = engine.linear_cross_entropy(hidden, weight, labels, reduction="sum", grads=True, grad_scale=1.0)[2][:, 16:]
    want = torch.zeros(dim, classes, dtype=torch.float64, device="cuda")
    for part in hidden.split(1 << 15):
        want += part.double().t() @ torch.softmax(part.double() @ weight.double(), 1)
    want = want[:, 16:]
    slope = float((dweight.double() * want).sum() / want.square().sum()) - 1
    assert abs(slope) < torch.finfo(hidden.dtype).eps / 8, slope


@gpu
def test_segments_and_pieces():
    """Contractions over the classes of a piece and over the rows that leave the tensor core more than once, with more than one piece."""
    _both(*_inputs(40000, 64, 60001, "f16", "dim", "some", seed=22), scale=2.0 ** 12)


@gpu
def test_lazily_negated_operands_are_refused():
    """The imaginary part of a conjugate is a view whose sign has yet to be applied."""
    import torch
    from mask_b200 import engine
    hidden, weight, labels = _inputs(20, 8, 5, "f32", "class")
    z = torch.complex(weight, weight).conj().imag
    assert z.is_neg()
    with pytest.raises(RuntimeError, match="weight"):
        engine.linear_cross_entropy(hidden, z, labels)
    assert bool(torch.isfinite(engine.linear_cross_entropy(hidden, z.resolve_neg(), labels)))


@gpu
@pytest.mark.parametrize("classes", [16, 300])
def test_gradient_of_the_weight_over_features_beyond_32_bits(classes):
    """2.2 thousand million features, every other row labelled, half of them behind 2^31 elements.  dweight in 64 bits by pieces: two
    roundings to bfloat16 leave at most 2^-9 each of a sum whose terms are independent; rows taken from another place, most of it."""
    import torch
    from mask_b200 import engine
    rows, dim = (1 << 22) + 5, 520
    g = torch.Generator(device="cuda").manual_seed(38)
    hidden = torch.empty(rows, dim, device="cuda", dtype=torch.bfloat16)
    for part in hidden.split(1 << 20):
        part.copy_(torch.randn(part.shape, generator=g, device="cuda"))
    weight = (torch.randn(classes, dim, generator=g, device="cuda") * (2.0 / dim ** 0.5)).bfloat16().t()
    labels = torch.randint(0, classes, (rows,), generator=g, device="cuda")
    labels[::2] = -1
    loss, dhidden, dweight = engine.linear_cross_entropy(hidden, weight, labels, reduction="sum", grads=True)
    want, total = torch.zeros(dim, classes, dtype=torch.float64, device="cuda"), 0.0
    for part, y in zip(hidden.split(1 << 18), labels.split(1 << 18)):
        keep = y >= 0
        h, y = part[keep].double(), y[keep, None]
        logits = h @ weight.double()
        total += float((torch.logsumexp(logits, 1, keepdim=True) - logits.gather(1, y)).sum())
        want += h.t() @ (torch.softmax(logits, 1).scatter_add_(1, y, -torch.ones_like(y, dtype=torch.float64)))
    assert float((dweight.double() - want).norm() / want.norm()) < 2.0 ** -8
    # half of the rows alone: as far off as if the other half had been taken for it
    assert abs(float(loss) - total) < 2.0 ** -16 * total
    for part in dhidden[::2].split(1 << 19):
        assert bool((part == 0).all())
    assert all(bool(part.any(1).all()) for part in dhidden[1::2].split(1 << 19))


@gpu
def test_same_call_same_bits_whatever_memory_held():
    """Pieces of the classes, pairs of blocks, one pass and tiny heads, in scratch that held NaN."""
    import torch
    from mask_b200 import engine
    for rows, dim, classes, dtype in ((16384, 512, 70001, "bf16"), (5000, 640, 3000, "f16"), (3000, 130, 700, "f32"), (20000, 64, 40, "f32"), (500, 16, 7, "f32")):
        x = _inputs(rows, dim, classes, dtype, labelled="some", seed=19)
        first = [t.clone() for t in engine.linear_cross_entropy(*x, grads=True)]
        for value in (float("nan"), 1.0):
            torch.cuda.empty_cache()
            free = torch.cuda.mem_get_info()[0]
            dirty = [torch.full((min(free // 8, 1 << 30),), value, device="cuda") for _ in range(3)]
            del dirty
            for a, b in zip(engine.linear_cross_entropy(*x, grads=True), first):
                assert torch.equal(a, b)


@gpu
@pytest.mark.parametrize("value", [-3.4028234663852886e38, -1e36])
@pytest.mark.parametrize("rows,dim,classes", MASKED)
def test_float32_classes_masked_by_the_lowest_value(rows, dim, classes, value):
    """A weight that no float32 logit survives counts as infinite: it takes its class out and no bits from the others."""
    import torch
    from mask_b200 import engine
    hidden, weight, labels = _inputs(rows, dim, classes, "f32", "dim", "some", seed=26)
    hidden[:, dim - 1] = 1.0
    masked = torch.arange(classes, device="cuda") % 3 == 1
    labels[(labels >= 0) & (labels < classes) & (labels % 3 == 1)] = 0
    out = weight.clone()
    out[dim - 1, masked] = value
    kept = torch.nonzero(~masked).squeeze(1)
    place = torch.full((classes,), -1, dtype=torch.int64, device="cuda")
    place[kept] = torch.arange(len(kept), device="cuda")
    real = (labels >= 0) & (labels < classes)
    want = _want(hidden, weight[:, kept], torch.where(real, place[labels.clamp(0, classes - 1)], -1), "sum")
    loss, dhidden, dweight = engine.linear_cross_entropy(hidden, out, labels, reduction="sum", grads=True)
    _check(loss, want[0], "loss")
    _check(dweight[:, kept], want[2], "dweight")
    assert bool((dweight[:, masked] == 0).all())
    _check(dhidden[:, :dim - 1], tuple(t[:, :dim - 1] for t in want[1]), "dhidden")


@gpu
@pytest.mark.parametrize("classes", [50, 600])
def test_powers_of_two_beyond_what_a_factor_holds(classes):
    """Operands up to 2^108 and 2^60, whose other values make logits of 2^120 and 0: the label's keeps its size."""
    import torch
    from mask_b200 import engine
    hidden = torch.zeros(70, 64, device="cuda")
    weight = torch.zeros(64, classes, device="cuda")
    hidden[0, 0], hidden[1:, 1] = 2.0 ** 108, -2.0 ** 85
    weight[0, 0], weight[1, 1::2] = 2.0 ** 60, 2.0 ** 35
    labels = torch.arange(70, device="cuda") % classes
    loss = engine.linear_cross_entropy(hidden, weight, labels, reduction="none")
    odd = labels[1:] % 2 == 1
    assert bool(loss[0].isnan())
    assert float((loss[1:][odd] / 2.0 ** 120 - 1).abs().max()) < 2.0 ** -20
    assert float((loss[1:][~odd] - math.log((classes + 1) // 2)).abs().max()) < 2.0 ** -20 * 8
