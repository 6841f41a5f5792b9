"""Queries and keys whose squares leave fp32: their direction is what counts, in prompts and row by row."""

import numpy as np
import pytest

from test_gpu_gdn_forgets import Edited

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kh,vh,d,taps", [(2, 4, 64, 4), (2, 2, 128, 4), (3, 3, 64, 3)])
@pytest.mark.parametrize("size,eps", [(1e21, 1e-6), (1e30, 1e-6), (1e37, 1e-6), (1e-23, 1e-30), (1e-18, 1e-30), (1e-23, 1e-6)])
def test_queries_and_keys_of_any_length(ctx, kh, vh, d, taps, size, eps):
    run = Edited(ctx, 81, kh, vh, d, taps, 3, 200, pending=4)
    c = run.layer
    c.eps = float(np.float32(eps))
    real = run.cache.run

    def edit(x, alpha, beta):
        x[:, :2 * c.kh * c.d] *= size

    run.cache.run = lambda *a, **kw: real(*a, **{**kw, "eps": eps})
    # inputs of one magnitude behind the others, so that the convolution cancels no 64-bit numbers
    run.weights_are(conv=np.abs(c.conv) + 0.05)
    run.edited([70, 3, 20], [0, 1, 2], [-1, -1, -1], edit)
    run.edited([5, 4, 66], [0, 1, 2], [0, 2, 0], edit)
    run.close()
