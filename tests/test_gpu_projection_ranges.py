"""Norm and projections at the ends of what their arguments may be, on the GPU against float64."""
from __future__ import annotations

import numpy as np
import pytest

from test_gpu_projection import Case, say

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [4, 40, 90, 300])
def test_scales_at_both_ends_of_fp32(mi355x, stream, rows):
    """Scales whose product leaves the range of fp32 where the result does not.  The sum's conversion and two products
    are a rounding each, the last one of half a subnormal step where the result is subnormal."""
    say(f"scales at the ends, {rows} rows")
    k, n = 2048, 42
    c = Case(7, rows, k, [n], np.float32)
    c.qs = np.resize(np.array([2.0 ** -126, 1.37 * 2.0 ** -110, 0.02, 1.21 * 2.0 ** 115], np.float32), rows)
    c.ws = [np.resize(np.array([2.0 ** -24, 1.5 * 2.0 ** -14, 0.75, 65504.0], np.float16), n)]
    c.w[0][5] = 0
    c.w[0][7] = 0  # under a scale of 65504
    got = c.run(mi355x, stream)[0].astype(np.float64)
    sums = c.q.astype(np.float64) @ c.w[0].astype(np.float64).T
    want = sums * (c.qs[:, None].astype(np.float64) * c.ws[0].astype(np.float64))
    huge = np.abs(want) > 2.0 ** 128
    assert np.array_equal(got[huge], np.sign(want[huge]) * np.inf)
    small = ~huge
    err = np.abs(got[small] - want[small])
    assert np.all(err <= 3.01 * 2.0 ** -24 * np.abs(want[small]) + 2.0 ** -150)
    assert np.all(got[:, [5, 7]] == 0)
