"""Draft verification where the draw's border falls between two tokens: sums in
another order may tell the two apart, but nothing else may come out."""

import numpy as np
import pytest
import torch

from test_gpu_verify import Step

pytestmark = pytest.mark.gpu

ROWS = 96


def halves(step, first, second, seed):
    """Every row's weight lies in two parts that hold the same logits in another order, with none between them."""
    g = torch.Generator().manual_seed(seed)
    step.target.fill_(-float("inf"))
    for row in range(step.rows):
        logits = 2.0 * torch.randn(len(first), generator=g)
        step.target[row, first] = logits.to(step.target.dtype)
        step.target[row, second] = step.target[row, first][torch.randperm(len(first), generator=g)]


# inside a thread's four tokens and between threads, waves and the chunks of 1024 and (many rows) 4096 tokens
PLACES = [(1024, range(0, 130), range(517, 647)), (1024, range(3, 40), range(40, 77)), (2048, range(100, 1024), range(1024, 1948)),
          (8192, range(0, 4096), range(4096, 8192)), (40000, range(1000, 9000), range(30001, 38001))]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("vocab,first,second", PLACES)
def test_a_draw_at_the_middle(ctx, dtype, vocab, first, second):
    """u = 1/2: half of the weight ends exactly at the first part's last token, so the second part's first is drawn (or,
    where a sum's rounding says that the border is passed, the token before it)."""
    first, second = list(first), list(second)
    s = Step(ctx, [1] * ROWS, vocab, dtype, False, 1)
    halves(s, first, second, vocab)
    s.uniforms[:] = 0.5
    emitted, accepted, _ = s.run()
    assert not accepted.any()
    assert set(emitted.tolist()) <= {first[-1], second[0]}, emitted


@pytest.mark.parametrize("vocab,first,second", PLACES)
def test_a_draw_at_the_middle_of_what_is_left(ctx, vocab, first, second):
    """The same of max(p - q, 0): q covers one token behind both parts, the draft that is turned down."""
    first, second = list(first), list(second)
    s = Step(ctx, [2] * (ROWS // 2), vocab + 4, "f32", True, 2)
    halves(s, first, second, vocab)
    s.target[:, vocab] = 0.0
    s.draft = torch.full((s.rows, vocab + 4), -20.0)
    s.draft[:, vocab] = 5.0
    s.temperatures[:] = 1.0
    s.tokens[:] = vocab
    s.uniforms[0::2], s.uniforms[1::2] = 1.0 - 2.0 ** -24, 0.5
    emitted, accepted, _ = s.run()
    assert not accepted.any()
    assert set(emitted[0::2].tolist()) <= {first[-1], second[0]}, emitted


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("drafts", [False, True])
@pytest.mark.parametrize("vocab", [40, 5000, 150000])
def test_masks_of_the_types_lowest_value(ctx, vocab, drafts, dtype):
    """Tokens masked by the lowest finite number weigh nothing: no u draws them, 0 included, and no draft of them stands."""
    s = Step(ctx, [1, 3, 2], vocab, dtype, drafts, 3)
    allowed = torch.zeros(vocab, dtype=torch.bool)
    allowed[7:vocab - 9:3] = True
    s.target[:, ~allowed] = torch.finfo(s.target.dtype).min
    if drafts:
        s.draft[:, ~allowed] = torch.finfo(s.target.dtype).min
    s.tokens[:] = 2
    for u in (0.0, 1.0 - 2.0 ** -24):
        s.uniforms[:] = u
        got = s.run()
        assert not got[1].any() and np.all(allowed.numpy()[got[0][[0, 1, 4]]])
        if u == 0.0 and not drafts:
            assert np.all(got[0][[0, 1, 4]] == 7)  # the lowest that weighs anything


def test_drafts_that_neither_distribution_gives_any_weight(ctx):
    """At a temperature so low that both probabilities are below what 64 bits hold: not u q < p."""
    s = Step(ctx, [4, 4, 4], 4096, "f32", True, 4)
    s.temperatures[:] = 1e-3
    worst = torch.stack([(t / 1e-3).log_softmax(0) for t in s.target.double()])
    s.tokens[1:] = worst[:-1].argmin(dim=1)
    got = s.run()
    assert not got[1].any()
    s.check(got)
