"""Attention over shared pages, however the call is cut: for far more tokens than there are, so that what is short here
goes the way of what is long, and for as few as there are, so that what does not gain is the plain call."""

import numpy as np
import pytest
import torch

from test_gpu_kv8_attention_bounds import check
from test_gpu_kv8_shared_attention import Shared

pytestmark = pytest.mark.gpu

LONG = dict(max_length=1 << 16, max_shared=1 << 15)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads,kv,head,counts,lengths,groups", [
    (8, 2, 128, [1, 2, 1, 3, 2], [300, 40, 0, 256, 255], [(0, 5, 256)]),       # shorter than what is shared, or empty
    (16, 4, 256, [1, 1, 1], [150, 140, 131], [(0, 3, 128)]),                   # 12 rows of a group, 4 of a sequence
    (4, 2, 64, [2, 1, 5, 2], [200, 220, 260, 270], [(0, 2, 192), (2, 4, 256)]),
    (12, 1, 64, [1, 40, 2], [130, 150, 140], [(0, 3, 128)])])
def test_cut_for_long_texts(ctx, heads, kv, head, counts, lengths, groups, dtype):
    c = Shared(ctx, heads, kv, head, 32, counts, lengths, groups, dtype, seed=21)
    c.tables[0, 1] = -1 if dtype == "f16" else c.tables[0, 1]  # a page that nobody has
    for first, end, tokens in groups:
        if first == 0 and dtype == "f16":
            c.tables[first:end, 1] = -1
    c.upload()
    check(c, c.run_shared(**LONG))
    check(c, c.run_shared())
    c.cache.free()


def test_groups_with_bad_numbers(ctx):
    c = Shared(ctx, 8, 2, 64, 32, [1, 2, 1, 1], [130, 140, 150, 128], [(0, 4, 128)], "bf16", seed=22)
    c.upload()
    for starts, shared, group_of in (([0, 9], [128], [0] * 4), ([-1, 4], [128], [0] * 4), ([3, 1], [128], [0] * 4),
                                     ([0, 4], [-7], [0] * 4), ([0, 4], [2 ** 31 - 1], [0] * 4), ([0, 4], [128], [7, -9, 0, 0]),
                                     ([1, 4], [128], [0] * 4), ([0, 3], [128], [0] * 4)):
        c.starts_of, c.shared, c.group_of = starts, shared, group_of
        check(c, c.run_shared(**LONG))
    c.cache.free()


@pytest.mark.parametrize("hint", [{}, LONG])
@pytest.mark.parametrize("starts", [[0, 4, 2, 3], [0, 7, 3, 5], [5, 2, 1, 0], [-3, 100, 200, 300], [2, 2, 7, 7], [0, 3, 3, 7], [1, 2, 4, 6]])
def test_row_starts_that_fall_back_or_leave_the_batch(ctx, starts, hint):
    """Rows of one sequence are what the plain call makes of them, rows of none stay as they were."""
    c = Shared(ctx, 8, 2, 64, 32, [4, 2, 1], [130, 140, 150], [(0, 3, 128)], "f32", seed=23)
    c.upload()
    c.dev[0].copy_(torch.tensor(starts, dtype=torch.int32))
    got, want = c.run_shared(**hint), c.run()
    owners = np.zeros(7, dtype=int)
    for b, e in zip(starts, starts[1:]):
        b = min(max(b, 0), 7)
        e = min(max(e, b), 7)
        owners[b:b + min(e - b, 4)] += 1
    got, want = got.reshape(7, -1), want.reshape(7, -1)
    assert (got[owners == 0] == 77.0).all()
    one = owners == 1
    # Either call is off by no more than this: a score's eight roundings of partial sums that `size` bounds and its
    # exponent's distance from its base, at most 2 size; weights 2^-20, each with a value and the result; sums of 160 tokens.
    held = np.unique(c.tables[c.tables >= 0])
    key_top, value_top = (float(x[0, held].max()) for x in (c.key_max, c.value_max))
    size = abs(c.scale) * np.abs(c.q.double().numpy()).sum(axis=-1).max() * key_top
    off = 2 * value_top * ((10 * size + 1) * 2.0 ** -24 + 2.0 ** -20 + (160 / 16 + 16) * 2.0 ** -23)
    assert np.abs(got[one] - want[one]).max(initial=0.0) <= 2 * off and off < 1e-3 * value_top
    c.cache.free()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_what_does_not_gain_is_the_plain_call(ctx, dtype):
    """Bit for bit: few shared tokens, and few rows behind many."""
    for counts, shared in (([1, 1, 1], 192), ([5, 4], 24000)):
        c = Shared(ctx, 16, 4, 64, 64, counts, [shared + 9 + i for i in range(len(counts))], [(0, len(counts), shared)], dtype, seed=24)
        c.upload()
        a, b = c.run_shared(), c.run()
        assert np.array_equal(a, b) or shared > 256
        check(c, a)
        c.cache.free()
