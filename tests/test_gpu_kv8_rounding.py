"""What the 8-bit cache's page magnitudes cost tokens that are stored one by one:
each growth rounds the page's codes again, and a dropped token's magnitude stays."""

import numpy as np
import pytest
import torch

from fortai_amd import backend as B
from test_gpu_kv8_cache import batch_of

pytestmark = pytest.mark.gpu

PAGE, KV, HEAD = 16, 2, 64


class Cache:
    def __init__(self, ctx):
        self.ctx, self.cache = ctx, B.Kv8Cache(ctx, 1, 4, PAGE, KV, HEAD)
        self.tables = np.array([[2, 0, 3]], dtype=np.int32)

    def append(self, x, length):
        """x [rows][KV][HEAD] fp32, as keys and as values."""
        d, batch = torch.from_numpy(x).cuda(), batch_of([0, len(x)], [length], self.tables)
        torch.cuda.synchronize()
        self.cache.append(0, batch, d.data_ptr(), d.data_ptr())
        self.ctx.synchronize()

    def read(self, count):
        out, batch = torch.zeros(2, count, KV, HEAD, device="cuda"), batch_of([0, count], [0], self.tables)
        torch.cuda.synchronize()
        self.cache.read(0, batch, out[0].data_ptr(), out[1].data_ptr())
        self.ctx.synchronize()
        return out.double().cpu().numpy()


def allowed(x, magnitudes, t):
    """Token t's error: half a code of its page's magnitude when it was stored, and of each larger one after that; two
    fp32 roundings of the value read."""
    steps, last = np.zeros(KV), np.zeros(KV)
    for a in magnitudes[t:]:
        steps, last = steps + np.where(a > last, a / 254, 0.0), np.maximum(a, last)
    return steps + (np.abs(x[t]).max(axis=-1) + steps) * 3 * 2.0 ** -24


@pytest.mark.parametrize("growth", ["every token", "random"])
def test_every_growth_costs_half_a_code(ctx, growth):
    rng = np.random.default_rng(3)
    x = rng.standard_normal((PAGE, KV, HEAD)).astype(np.float32)
    if growth == "every token":
        x *= (1.1 ** np.arange(PAGE, dtype=np.float32) / np.abs(x).max(axis=(1, 2)))[:, None, None]
        x[:, :, 0] = np.abs(x).max(axis=2) * 1.01
    c = Cache(ctx)
    for t in range(PAGE):
        c.append(x[t:t + 1], t)
    tops = np.maximum.accumulate(np.abs(x.astype(np.float64)).max(axis=2), axis=0)  # [token][head]
    worst = 0.0
    for got in c.read(PAGE):
        for t in range(PAGE):
            off = np.abs(got[t] - x[t]).max(axis=1)
            assert np.all(off <= allowed(x.astype(np.float64), tops, t)), t
            worst = max(worst, float((off / (tops[-1] / 254)).max()))
    if growth == "every token":
        assert worst > 1.0  # it does add up: more than the half code that one rounding may cost
    c.cache.free()


def test_a_dropped_token_leaves_its_magnitude(ctx):
    """A rejected draft that was loud: the tokens before it keep codes of its magnitude, as do those that take its place;
    the next page starts anew."""
    rng = np.random.default_rng(4)
    x = rng.uniform(-1, 1, (PAGE + 4, KV, HEAD)).astype(np.float32)
    loud = rng.uniform(-20, 20, (2, KV, HEAD)).astype(np.float32)
    c = Cache(ctx)
    c.append(x[:5], 0)
    before = c.read(5)
    c.append(loud, 5)           # two drafts
    c.append(x[5:], 5)          # both rejected: other tokens in their place
    top, code = np.abs(x[:PAGE].astype(np.float64)).max(axis=(0, 2)), np.abs(loud.astype(np.float64)).max(axis=(0, 2)) / 127
    for was, got in zip(before, c.read(PAGE + 4)):
        assert np.all(np.abs(was - x[:5]) <= 1.001 * top[:, None] / 254)
        k = got[:PAGE] / code[:, None]
        assert np.all(np.abs(k - np.rint(k)) < 1e-4)                                      # codes of the loud draft's
        assert np.all(np.abs(got[:5] - was) <= 1.001 * code[:, None] / 2)                 # the standing ones, rounded once more
        assert np.all(np.abs(got[5:PAGE] - x[5:PAGE]) <= 1.001 * code[:, None] / 2)
        assert np.all(np.abs(got[PAGE:] - x[PAGE:]) <= 1.001 * np.abs(x[PAGE:]).max(axis=(0, 2))[:, None] / 254)
    c.cache.free()
