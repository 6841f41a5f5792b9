"""Rows of the delta rule that forget everything, by any margin, among rows that do not."""

import numpy as np
import pytest
import torch

from test_gpu_gdn_rows import Run

pytestmark = pytest.mark.gpu


class Edited(Run):
    """Calls whose inputs, alphas and betas edit(x, alpha, beta) has changed, and weights of the test's own."""

    def __init__(self, ctx, seed, kh, vh, d, taps, slots, max_rows, dtype="f32", pending=0):
        super().__init__(ctx, seed, kh, vh, d, taps, pending, slots, max_rows, dtype)

    def weights_are(self, **what):
        for name, w in zip(("conv", "ssm_a", "ssm_dt"), self.weights):
            if name in what:
                at = getattr(self.layer, name)
                at[...] = np.asarray(what[name], dtype=np.float32)
                w.copy_(torch.from_numpy(at))

    def edited(self, counts, slots, standing, edit):
        c, real, rows = self.layer, self.rng, sum(counts)
        x, alpha, beta = (real.standard_normal((rows, w)) for w in (c.channels, c.vh, c.vh))
        edit(x, alpha, beta)
        drawn = iter((x, alpha, beta))

        class Draw:
            standard_normal = staticmethod(lambda shape: next(drawn))

        self.rng = Draw
        got = self.step(counts, slots, standing)
        self.rng = real
        assert np.isfinite(got).all()
        self.check_storage()
        return got


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("far", [300.0, 1e9, 1e12, 1e15, 1e18, 1e30, 3e38])
def test_rows_that_forget_everything(ctx, far, dtype):
    """What is behind such a row decays as it would by itself, in prompts, drafts and the state they leave."""
    run = Edited(ctx, 61, 2, 4, 64, 4, 2, 300, dtype, pending=4)
    # with 4 the logarithm leaves fp32 at 3e38; alpha + dt does in the last two heads
    run.weights_are(ssm_a=[-1.0, -4.0, -1e-38 if far == 3e38 else -1.0, 0.0], ssm_dt=[0.0, -1.0, far / 2, far])

    def edit(x, alpha, beta):
        alpha[:, 2] = -far / 2 + (np.abs(alpha[:, 2]) if far < 1e6 else 0.0)
        for row in (5, 6, 40, 70, 127, 128):
            if row < len(x):
                alpha[row, :] = far

    run.edited([131, 30], [0, 1], [-1, -1], edit)
    run.edited([131, 4], [0, 1], [0, 0], edit)
    run.edited([4, 9], [0, 1], [0, 3], edit)
    run.edited([3, 20], [0, 1], [2, 0], edit)
    run.close()
