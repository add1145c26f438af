"""The layer norm's gradients of weight and bias where they come from rows past element 2^31 alone.  The formula and its
tolerances are test_gpu_norm's, where these are derived; the rows whose gradient is zero add nothing to a sum."""
import pytest
import torch

import test_gpu_norm as norm
from test_gpu_far_offsets import big, room  # noqa: F401
from test_gpu_tensor_linear import randn

pytestmark = pytest.mark.gpu
TAIL = 300


def test_sums_over_the_last_rows(gpu, room):  # noqa: F811
    m, d = 530_000, 4096
    x, dy = big(m, d), big(m, d, seed=5)
    assert (m - TAIL) * d > 2 ** 31
    dy[:-TAIL] = 0
    w, b = 1 + randn(d, seed=3, std=0.3), randn(d, seed=4)
    y, gx, gw, gb = norm.run(x, w, b, dy)
    assert not bool(gx[:-TAIL].any())
    (want, _), dx, dw, db = norm.formula(x[-TAIL:], w, b, dy[-TAIL:])
    norm.close(gx[-TAIL:], *dx)
    # (a row of zeros adds no rounding to a column's sum: as many as the formula counts for the last rows alone)
    norm.close(gw, *dw)
    norm.close(gb, *db)
    # a sum that lost the rows would be 0, a thousand tolerances off
    for value, tol in (dw, db):
        assert float((value.abs() / tol).median()) > 1000
