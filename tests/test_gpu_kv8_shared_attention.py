"""Attention of sequences that share their first pages, held row by row and head by head to what fp32 arithmetic rounded
once may be off, as the attention of each by itself is."""

import numpy as np
import pytest
import torch

from fortai_amd import backend as B
from test_gpu_kv8_attention import TYPES, Case
from test_gpu_kv8_attention_bounds import check

pytestmark = pytest.mark.gpu


class Shared(Case):
    """groups: (first sequence, end, shared tokens); what is between them shares nothing."""

    def __init__(self, ctx, heads, kv, head, page, counts, lengths, groups, dtype, **more):
        super().__init__(ctx, heads, kv, head, page, counts, lengths, dtype, **more)
        self.starts_of, self.shared, self.group_of = [], [], [-1] * len(counts)
        at = 0
        for first, end, tokens in groups:
            if first > at:
                self.starts_of.append(at)
                self.shared.append(0)
            for s in range(first, end):
                n = min(tokens // page, -(-max(0, lengths[s] + counts[s]) // page), -(-max(0, lengths[first] + counts[first]) // page))
                self.tables[s, :n] = self.tables[first, :n]
                self.group_of[s] = len(self.starts_of)
            self.starts_of.append(first)
            self.shared.append(tokens)
            at = end
        if at < len(counts):
            self.starts_of.append(at)
            self.shared.append(0)
        self.starts_of.append(len(counts))
        self.group_rows = max(int(self.starts[e] - self.starts[f]) for f, e, _ in groups)

    def run_shared(self, max_length=None, max_shared=None, group_rows=None):
        up = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")
        self.numbers = [up(a) for a in (self.starts_of, self.shared, self.group_of)]
        sharing = B.Kv8Groups(len(self.shared), self.group_rows if group_rows is None else group_rows, *(a.data_ptr() for a in self.numbers))
        parts, at = 2 if self.gate else 1, self.dq.data_ptr()
        self.out.fill_(77.0)
        torch.cuda.synchronize()
        self.cache.shared_attention(0, self.batch, sharing, at, self.heads, self.out.data_ptr(), self.scale,
                                    max(l + c for l, c in zip(self.lengths, self.counts)) if max_length is None else max_length,
                                    max(self.shared) if max_shared is None else max_shared, dtype=self.dtype,
                                    gate=at + self.head * self.dq.element_size() if self.gate else None,
                                    query_head_pitch=parts * self.head, query_pitch=parts * self.heads * self.head)
        self.ctx.synchronize()
        return self.out.double().cpu().numpy()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads,kv,head,page,counts,lengths,groups,gate", [
    # one row each; a sequence that has only the shared tokens before its row
    (8, 2, 256, 64, [1, 1, 1, 1], [128, 130, 200, 333], [(0, 4, 128)], True),
    # two groups, one sequence of no group between them, ragged drafts, one without rows
    (16, 4, 64, 16, [3, 1, 2, 5, 1, 0, 4], [80, 64, 100, 20, 320, 400, 321], [(0, 3, 64), (4, 7, 320)], False),
    # shared tokens that end inside a tile: whole tiles of 64 are shared
    (12, 1, 128, 32, [2, 1, 1], [160, 161, 190], [(0, 3, 160)], True),
    # many rows in the group, few each; more tokens than one split has
    (24, 3, 128, 64, [2] * 20, [1216 + 3 * i for i in range(20)], [(0, 20, 1216)], False),
    # a prompt's chunk behind the shared part, beside a decode step
    (4, 2, 256, 16, [70, 1, 33], [192, 200, 205], [(0, 3, 192)], True),
    # fewer than 64 shared tokens, and a group of one
    (5, 5, 64, 32, [1, 2, 1], [32, 40, 300], [(0, 2, 32), (2, 3, 256)], False)])
def test_groups(ctx, dtype, heads, kv, head, page, counts, lengths, groups, gate):
    c = Shared(ctx, heads, kv, head, page, counts, lengths, groups, dtype, gate=gate, seed=heads + head + len(counts))
    c.upload()
    check(c, c.run_shared())
    # cut as for far more tokens, and for far fewer
    check(c, c.run_shared(max_length=1 << 20, max_shared=1 << 19))
    check(c, c.run_shared(max_length=65, max_shared=64))
    check(c, c.run())
    c.cache.free()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_sequences_that_do_not_see_all_of_it(ctx, dtype):
    """Sequences that are shorter than the shared tokens, or empty, read what they see by themselves."""
    c = Shared(ctx, 8, 2, 128, 16, [1, 2, 1, 3, 2], [300, 40, 0, 256, 255], [(0, 5, 256)], dtype, seed=5)
    c.upload()
    check(c, c.run_shared())
    c.cache.free()


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_missing_pages_and_rows_before_the_first_token(ctx, dtype):
    c = Shared(ctx, 4, 2, 64, 32, [1, 1, 2], [200, 220, 260], [(0, 3, 192)], dtype, seed=6)
    c.tables[:, 2] = -1          # a page that nobody has
    c.tables[1, 4] = c.pages     # the second sequence's own table is not looked at for what is shared
    c.tables[2, 7] = -5
    c.upload()
    got = c.run_shared()
    c.tables[1, 4] = c.tables[0, 4]
    check(c, got)
    c.cache.free()


def test_a_group_of_more_rows_than_the_call_says(ctx):
    """max_rows too small: that group shares nothing, and its rows are right all the same."""
    c = Shared(ctx, 8, 2, 64, 64, [3, 4, 1, 1], [130, 140, 150, 128], [(0, 2, 128), (2, 4, 128)], "f32", seed=7)
    c.upload()
    check(c, c.run_shared(group_rows=2))
    check(c, c.run_shared(group_rows=0))
    c.cache.free()


def test_groups_with_bad_numbers_share_nothing(ctx):
    c = Shared(ctx, 8, 2, 64, 32, [1, 2, 1, 1], [130, 140, 150, 128], [(0, 4, 128)], "bf16", seed=8)
    c.upload()
    good = list(c.starts_of), list(c.shared), list(c.group_of)
    for starts, shared, group_of in (([0, 9], [128], [0] * 4), ([-1, 4], [128], [0] * 4), ([3, 1], [128], [0] * 4),
                                     ([0, 4], [-7], [0] * 4), ([0, 4], [2 ** 31 - 1], [0] * 4), ([0, 4], [128], [7, -9, 0, 0]),
                                     ([1, 4], [128], [0] * 4), ([0, 3], [128], [0] * 4)):
        c.starts_of, c.shared, c.group_of = starts, shared, group_of
        check(c, c.run_shared(max_shared=128))
    c.starts_of, c.shared, c.group_of = good
    check(c, c.run_shared())
    c.cache.free()


def test_row_starts_with_bad_numbers(ctx):
    """Rows that fall back or leave the batch: the group's rows do not hold them, so they share nothing."""
    c = Shared(ctx, 8, 2, 64, 32, [4, 2, 1], [130, 140, 150], [(0, 3, 128)], "f32", seed=9)
    c.upload()
    for starts in ([0, 4, 2, 3], [0, 7, 3, 5], [5, 2, 1, 0], [-3, 100, 200, 300], [2, 2, 7, 7]):
        c.dev[0].copy_(torch.tensor(starts, dtype=torch.int32))
        got = c.run_shared()
        assert np.isfinite(got).all()
    c.dev[0].copy_(torch.from_numpy(c.starts))
    check(c, c.run_shared())
    c.cache.free()


def test_unlike_magnitudes_on_both_sides(ctx):
    """The join holds shared and own results against the larger of their products, whichever side has it."""
    for loud in (1e-20, 1e20):
        c = Shared(ctx, 8, 2, 128, 32, [1, 2], [260, 300], [(0, 2, 256)], "f32", seed=10)
        own = c.tables[1, 8:10]
        c.value_max[0, own] *= np.float32(loud)
        c.key_max[0, own] *= np.float32(3.0)
        c.upload()
        check(c, c.run_shared())
        c.cache.free()


def test_more_rows_than_the_workspace_holds(ctx):
    """Partial results that do not fit: the call is the plain attention's, bit for bit."""
    c = Shared(ctx, 32, 32, 64, 64, [140] * 4, [128] * 4, [(0, 4, 128)], "f16", seed=11)
    c.upload()
    a = c.run_shared()
    assert np.array_equal(a, c.run())
    c.cache.free()


def test_captured_and_replayed():
    ctx = B.Context(0)  # a context holds one graph
    c = Shared(ctx, 8, 2, 128, 32, [2, 1, 3], [200, 260, 300], [(0, 3, 192)], "f32", seed=12)
    c.upload()
    up = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")
    numbers = [up(a) for a in (c.starts_of, c.shared, c.group_of)]
    sharing = B.Kv8Groups(1, 6, *(a.data_ptr() for a in numbers))
    torch.cuda.synchronize()
    ctx.capture_begin()
    c.cache.shared_attention(0, c.batch, sharing, c.dq.data_ptr(), 8, c.out.data_ptr(), c.scale, 303, 192)
    ctx.capture_end()
    for lengths, shared in (([200, 260, 300], 192), ([190, 194, 240], 64), ([128, 100, 301], 128)):
        c.lengths = lengths
        c.dev[1].copy_(torch.tensor(lengths, dtype=torch.int32))
        numbers[1].fill_(shared)
        c.out.fill_(77.0)
        torch.cuda.synchronize()
        ctx.graph_launch()
        ctx.synchronize()
        check(c, c.out.double().cpu().numpy())
    c.cache.free()
    ctx.close()


def test_refusals(ctx):
    c = Shared(ctx, 8, 2, 64, 32, [1, 1], [130, 140], [(0, 2, 128)], "f32", seed=13)
    c.upload()
    at = torch.zeros(8, dtype=torch.int32, device="cuda").data_ptr()
    call = lambda g, shared=128: c.cache.shared_attention(0, c.batch, g, c.dq.data_ptr(), 8, c.out.data_ptr(), c.scale, 141, shared)
    for bad in (B.Kv8Groups(3, 1, at, at, at), B.Kv8Groups(-1, 1, at, at, at), B.Kv8Groups(1, 3, at, at, at), B.Kv8Groups(1, -1, at, at, at),
                B.Kv8Groups(1, 2, None, at, at), B.Kv8Groups(1, 2, at, None, at), B.Kv8Groups(1, 2, at, at, None), B.Kv8Groups(1, 2, at + 2, at, at)):
        with pytest.raises(B.BackendError) as e:
            call(bad)
        assert e.value.code == B.INVALID
    with pytest.raises(B.BackendError):
        call(B.Kv8Groups(1, 2, at, at, at), -1)
    call(B.Kv8Groups(0, 0, None, None, None))  # no groups: the plain attention
    ctx.synchronize()
    check(c, c.out.double().cpu().numpy())
    c.cache.free()
