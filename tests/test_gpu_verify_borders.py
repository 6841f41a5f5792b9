"""Draft verification where the draw's border falls between two tokens: sums in
another order may tell the two apart, but nothing else may come out."""

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
