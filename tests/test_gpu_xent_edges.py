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
