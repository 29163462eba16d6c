"""GPU tests of the class-score losses where weights, scores or derivatives are not
finite, rows are empty, or the number of classes meets a limit of a kernel, in
each of the kernels that take rows: up to 32 classes, rows of up to 8 KB, longer
ones. Helpers, and the tolerances that they hold, are those of
test_gpu_preference.
"""

import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from modern_fm_b200.preference import preference_loss  # noqa: E402

from test_gpu_preference import TYPES, _make, _wide  # noqa: E402


@pytest.mark.parametrize("c", [10, 32, 100, 9001])
@pytest.mark.parametrize("kind", list(TYPES))
def test_masked_rows_under_a_scale_that_is_not_finite(c, kind):
    """A NaN weight, or weights whose sum is too small to divide by: rows that are masked, of
    no sequence or of a pair of weight 0 keep gradient 0; with the NaN the others get NaN."""
    x, y = _make(1, 70, c, kind, pad=0.4)
    y[0] = y[33] = -1
    y[2] = 0
    wide = _wide(kind)
    ip = torch.tensor([1, 20, 40, 50, 68], device="cuda")  # rows 0, 68, 69: of no sequence
    ref = torch.zeros(4, dtype=wide, device="cuda")
    live = (y >= 0) & (y < c)
    row = torch.arange(70, device="cuda")
    inside = (row >= 1) & (row < 68)
    first = (row < 20) | ((row >= 40) & (row < 50))  # the rows of pair 0
    w = torch.tensor([math.nan, 1.0], dtype=wide, device="cuda")
    r = preference_loss(x, y, ip, ref, sample_weight=w)
    assert math.isnan(float(r.loss))
    assert bool((r.grad[~live | ~inside] == 0).all())
    assert torch.isnan(r.grad[live & inside & first].double()).all()
    w = torch.tensor([0.0, math.nan], dtype=wide, device="cuda")
    r = preference_loss(x, y, ip, ref, sample_weight=w)
    assert bool((r.grad[~live | ~inside | first] == 0).all())
    # 1 / the sum of the weights is infinite in float64; in float32 the sum's inverse is
    # finite, but the derivatives are 0
    w = torch.tensor([0.0, 5e-324 if kind == "f64" else 1e-45], dtype=wide, device="cuda")
    r = preference_loss(x, y, ip, ref, sample_weight=w)
    assert bool((r.grad[~live | ~inside | first] == 0).all())
