"""Prompts of the delta rule whose numbers are not alike: tokens that are far louder or fainter than those around
them, and states that are."""

import numpy as np
import pytest
import torch

from fortai_amd import backend as B
from gdn_unlike_model import UnlikeLayer
from test_gpu_gdn_forgets import Edited

pytestmark = pytest.mark.gpu


class Unlike(Edited):
    def __init__(self, *shape, **more):
        super().__init__(*shape, **more)
        self.layer.__class__ = UnlikeLayer


HEADS = [(2, 4, 64), (2, 2, 128)]


def loud(c, x, row, factor, dims=None):
    """Values of one row (and the convolution's next ones) times factor; dims: of the value channels, or all."""
    at = 2 * c.kh * c.d
    x[row, at + np.arange(c.vh * c.d) if dims is None else at + np.asarray(dims)] *= factor


@pytest.mark.parametrize("kh,vh,d", HEADS)
@pytest.mark.parametrize("factor", [1e3, 1e5, 1e6, 1e8, 1e12, 1e20, 1e30])
def test_a_loud_token_costs_the_ones_before_it_nothing(ctx, kh, vh, d, factor):
    run = Unlike(ctx, 71, kh, vh, d, 4, 2, 300)
    run.edited([100, 66], [0, 1], [-1, -1], lambda x, alpha, beta: (loud(run.layer, x, 40, factor), loud(run.layer, x, 163, factor)))
    run.edited([70], [1], [0], lambda x, alpha, beta: loud(run.layer, x, 63, factor))
    run.close()


@pytest.mark.parametrize("kh,vh,d", HEADS)
@pytest.mark.parametrize("factor", [1e5, 1e9, 1e15])
def test_one_loud_value(ctx, kh, vh, d, factor):
    """In one value dim of a head, late in its chunk: the dim's rows before it keep their bits."""
    run = Unlike(ctx, 72, kh, vh, d, 4, 1, 300)
    run.edited([64], [0], [-1], lambda x, alpha, beta: loud(run.layer, x, 60, factor, [5, d + 17]))
    run.close()


@pytest.mark.parametrize("kh,vh,d", HEADS)
@pytest.mark.parametrize("factor", [1e4, 1e7, 1e15])
def test_loud_tokens_that_are_forgotten(ctx, kh, vh, d, factor):
    """At once, by degrees, within the chunk and from one to the next, and in the state that a call leaves."""
    run = Unlike(ctx, 73, kh, vh, d, 4, 1, 300)
    run.weights_are(ssm_a=[-1.0, -0.3] * (vh // 2), ssm_dt=0.0)

    def edit(x, alpha, beta):
        for row in (3, 62, 130):
            loud(run.layer, x, row, factor)
        alpha[14] = 600.0
        alpha[64 + 10] = 600.0
        alpha[len(x) - 3] = 5.0

    run.edited([150], [0], [-1], edit)
    run.edited([150], [0], [0], edit)

    def quiet(x, alpha, beta):
        x *= 0.01
        alpha[0], alpha[20] = 12.0, 60.0

    run.edited([90], [0], [0], quiet)
    run.close()


@pytest.mark.parametrize("kh,vh,d", HEADS)
def test_faint_betas_and_silent_rows(ctx, kh, vh, d):
    """Rows that hardly change the state, values that are nothing at all, and a state that fades behind them."""
    run = Unlike(ctx, 74, kh, vh, d, 4, 1, 300)
    at = 2 * run.layer.kh * run.layer.d

    def faint(x, alpha, beta):
        beta[:] = -25.0 + beta
        beta[30] = 1.0

    def silent(x, alpha, beta):
        x[:80, at:] = 0.0

    run.edited([100], [0], [-1], faint)
    run.edited([100], [0], [0], faint)
    run.edited([130], [0], [0], silent)
    run.edited([130], [0], [-1], silent)
    run.close()


def test_many_sequences_of_unlike_tokens(ctx):
    """Enough heads for 32 value dims a workgroup."""
    run = Unlike(ctx, 75, 4, 16, 128, 4, 9, 900)
    counts = [70, 65, 64, 100, 17, 33, 129, 80, 90]

    def edit(x, alpha, beta):
        starts = np.concatenate([[0], np.cumsum(counts)])
        for s in range(9):
            loud(run.layer, x, starts[s] + (7 * s + 11) % counts[s], 10.0 ** (2 * s + 1))
        alpha[starts[4] + 5] = 1e15

    run.edited(counts, list(range(9)), [-1] * 9, edit)
    run.edited(counts, list(range(9)), [0] * 9, edit)
    run.close()


def test_values_near_the_end_of_fp32(ctx):
    """Up to 2^120: their bounds leave fp32 where they themselves do not."""
    run = Unlike(ctx, 76, 2, 2, 64, 4, 1, 200)
    run.edited([100], [0], [-1], lambda x, alpha, beta: loud(run.layer, x, slice(None), 1e35))
    run.edited([100], [0], [0], lambda x, alpha, beta: loud(run.layer, x, slice(None), 1e35))
    run.close()


@pytest.mark.parametrize("count", [40, 100, 192])
def test_numbers_that_are_not_finite(ctx, count):
    """A NaN or an infinity among the values is in its column's outputs from its row on at the latest; the other
    sequence and the chunks before it have nothing of it."""
    for bad in (np.nan, np.inf):
        runs = [Unlike(ctx, 77, 2, 4, 64, 4, 2, 400) for _ in range(2)]
        outs = []
        for run, value in zip(runs, (bad, 1.0)):
            c, row = run.layer, count - 10
            x, alpha, beta = (np.random.default_rng(5).standard_normal((count + 70, w)).astype(np.float32) for w in (c.channels, c.vh, c.vh))
            x[row, 2 * c.kh * c.d + 3] = value
            dev = [torch.from_numpy(a).cuda() for a in (x, alpha, beta)]
            out = torch.zeros(count + 70, c.vh * c.d, device="cuda")
            numbers = [torch.tensor(a, dtype=torch.int32, device="cuda") for a in ([0, count, count + 70], [0, 1], [-1, -1])]
            torch.cuda.synchronize()
            run.cache.run(1, B.GdnBatch(2, count + 70, count + 70, *(a.data_ptr() for a in numbers)), *(a.data_ptr() for a in dev),
                          *(w.data_ptr() for w in run.weights), out.data_ptr())
            ctx.synchronize()
            outs.append(out.cpu().numpy())
            run.close()
        got, want = outs
        assert not np.isfinite(got[row:count, 3]).any()
        assert np.array_equal(got[:row // 64 * 64], want[:row // 64 * 64]) and np.array_equal(got[count:], want[count:])


def test_chunks_that_are_looked_at_twice(ctx):
    """Chunks of every kind one behind the other: ordinary, with rows that go by themselves, all of them, bounds that
    were too far off; with pending rows in front of them, and in 16 bits."""
    for dtype in ("f32", "f16"):
        run = Unlike(ctx, 78, 2, 4, 128, 4, 2, 900, dtype=dtype)
        c = run.layer
        run.weights_are(ssm_a=[-0.01, -0.5, -2.0, -0.1])

        def edit(x, alpha, beta):
            top = 1e4 if dtype == "f16" else 1e9
            loud(c, x, 100, top)
            loud(c, x, 5 * 64 + 63, top)
            alpha[2 * 64:2 * 64 + 30] = 9.0
            x[6 * 64:7 * 64 + 9, 2 * c.kh * c.d:] *= 1e-4
            alpha[7 * 64 + 3] = 300.0

        run.edited([64 * 10 + 13, 200], [0, 1], [-1, -1], edit)
        run.edited([300, 64 * 9], [0, 1], [0, 0], lambda x, alpha, beta: loud(c, x, 310, 1e3))
        run.close()
