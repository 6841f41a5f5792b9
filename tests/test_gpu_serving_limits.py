"""The serving operators at the ends of the ranges that the header states."""

import numpy as np
import pytest
import torch

from fortai_amd import backend as B

pytestmark = pytest.mark.gpu

int32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")


def attention64(q, k, v, scale):
    """q [heads][head] over k, v [tokens][head], float64."""
    return torch.softmax((q.double() @ k.t().contiguous()) * scale, -1) @ v


@pytest.mark.parametrize("sequences,heads,kv", [(1, 65535, 1), (16384, 2, 1), (3, 4096, 1024)])
def test_many_heads_and_many_sequences(ctx, sequences, heads, kv):
    """One new token each behind two cached ones, appended and attended to; every sequence on a page of its own."""
    head, page = 64, 16
    g = torch.Generator().manual_seed(heads)
    kvs = torch.randn(2, 3 * sequences, kv, head, generator=g).cuda()
    q = torch.randn(sequences, heads, head, generator=g).cuda()
    out, back = torch.full((sequences + 1, heads, head), 5.0, device="cuda"), torch.zeros_like(kvs)
    starts, lengths, tables = int32(np.arange(sequences + 1)), int32([2] * sequences), int32(np.arange(sequences)[::-1].copy())
    all_starts, none = int32(3 * np.arange(sequences + 1)), int32([0] * sequences)
    cache = B.Kv8Cache(ctx, 1, sequences, page, kv, head)
    step = B.Kv8Batch(sequences, sequences, 1, starts.data_ptr(), lengths.data_ptr(), tables.data_ptr(), 1)
    whole = B.Kv8Batch(sequences, 3 * sequences, 3, all_starts.data_ptr(), none.data_ptr(), tables.data_ptr(), 1)
    torch.cuda.synchronize()
    cache.append(0, whole, kvs[0].data_ptr(), kvs[1].data_ptr())
    cache.read(0, whole, back[0].data_ptr(), back[1].data_ptr())
    cache.attention(0, step, q.data_ptr(), heads, out.data_ptr(), 0.125, 3)
    ctx.synchronize()
    tops = kvs.view(2, sequences, 3, kv, head).abs().amax(dim=(2, 4), keepdim=True).expand(2, sequences, 3, kv, head)
    assert bool(((back - kvs).view(tops.shape).abs() <= tops * (1.001 / 254)).all())
    assert bool((out[sequences] == 5.0).all())
    k, v = (x.view(sequences, 3, kv, head).double() for x in back)
    for s in {0, sequences // 2, sequences - 1}:
        for n in {0, kv // 2, kv - 1}:
            rows = slice(n * (heads // kv), (n + 1) * (heads // kv))
            want = attention64(q[s, rows], k[s, :, n], v[s, :, n], 0.125)
            # what the cache reads back is off by two fp32 roundings, attention's sums of three tokens by some more
            assert float((out[s, rows] - want).abs().max()) <= 2.0 ** -18 * float(v[s, :, n].abs().max())
    cache.free()


def test_a_vocabulary_of_2_to_the_28(ctx):
    """Two rows: a draft that stands, then the draw; all weight on a few tokens at the far ends."""
    vocab = 1 << 28
    target = torch.full((2, vocab), -30.0, dtype=torch.float16, device="cuda")
    target[0, vocab - 5] = 40.0
    target[1, 3], target[1, vocab - 1] = 40.0, 40.0
    tokens = torch.tensor([0, vocab - 5], device="cuda")
    starts, emitted = int32([0, 2]), torch.zeros(2, dtype=torch.int64, device="cuda")
    accepted, logprobs = int32([9]), torch.zeros(2, device="cuda")
    v = B.Verifier(ctx, 2, 1, vocab)
    for u, want in ((0.25, 3), (0.75, vocab - 1)):
        uniforms = torch.full((2,), u, device="cuda")
        torch.cuda.synchronize()
        v.run(target.data_ptr(), tokens.data_ptr(), uniforms.data_ptr(), starts.data_ptr(), 1, 2, emitted.data_ptr(),
              accepted.data_ptr(), dtype="f16", logprobs=logprobs.data_ptr())
        ctx.synchronize()
        assert emitted.tolist() == [vocab - 5, want] and accepted.tolist() == [1]
        assert abs(float(logprobs[1]) + np.log(2.0)) < 1e-6
    v.free()


def test_65535_sequences_of_one_row(ctx):
    n, vocab = 65535, 64
    g = torch.Generator().manual_seed(1)
    target = torch.randn(n, vocab, generator=g).cuda()
    zeros, starts = torch.zeros(n, dtype=torch.int64, device="cuda"), int32(np.arange(n + 1))
    emitted, accepted = torch.full((n,), -9, dtype=torch.int64, device="cuda"), int32([-9] * n)
    uniforms, cold = torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda")
    torch.cuda.synchronize()
    v = B.Verifier(ctx, n, n, vocab)
    v.run(target.data_ptr(), zeros.data_ptr(), uniforms.data_ptr(), starts.data_ptr(), n, n, emitted.data_ptr(), accepted.data_ptr(),
          temperatures=cold.data_ptr())
    ctx.synchronize()
    assert torch.equal(emitted, target.argmax(dim=1)) and not bool(accepted.any())
    v.free()


def test_rotary_positions_of_2_to_the_23_heads(ctx):
    heads = 1 << 23
    x = torch.ones(heads, 4, device="cuda")
    position, rope = int32([2]), B.Rope(ctx, 2)
    torch.cuda.synchronize()
    rope.apply(x.data_ptr(), position.data_ptr(), 1, heads, 4, x.data_ptr())
    ctx.synchronize()
    want = torch.tensor([np.cos(2) - np.sin(2), np.cos(2) + np.sin(2), 1.0, 1.0], dtype=torch.float64, device="cuda")
    assert float((x - want).abs().max()) < 1e-6
    rope.free()
