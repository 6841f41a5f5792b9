"""Attention over the 8-bit cache held, row by row and head by head, to what fp32
arithmetic rounded once may be off: 16-bit types and however many rows a call has, too."""

import numpy as np
import pytest
import torch

from test_gpu_kv8_attention import HALF_STEP, TYPES, Case

LOG2E = 1.4426950408889634


def tight(c, layer=0):
    """The formula in 64 bits, and how far a row and head may be off before its one rounding to the output's type.

    Scores: three digits to the base 256 of the query over a power of two above its row's largest (127 2^16 steps; four
    digits, 127 2^24 steps, for fp32, behind one fp32 rounding), and eight fp32 roundings on the way to the exponent,
    each 2^-24 of partial sums that |scale| sum |q k| bounds; the exponent's distance from its base is rounded once.
    Weights: exp2, its base, the magnitude's mantissa and two fp16 halves: eight times 2^-23.  Sums of n tokens: n / 16
    additions and 16 joins, 2^-23 of the terms' sum.  A lower half below fp16's range is lost: 2^-34 of the largest
    product of weight and magnitude, a token.  An error of the weight of token j moves the result by p_j (v_j - out)."""
    rows, group, page, d = int(c.starts[-1]), c.heads // c.kv, c.page, c.head
    want, bound = np.zeros((rows, c.heads, d)), np.zeros((rows, c.heads, d))
    q64 = c.q.double().numpy()
    for s, (count, length) in enumerate(zip(c.counts, c.lengths)):
        seen_pages = [(j, p) for j, p in enumerate(c.tables[s]) if 0 <= p < c.pages]
        if not seen_pages or length + count <= 0:
            continue
        token = np.concatenate([np.arange(j * page, (j + 1) * page) for j, _ in seen_pages])
        pick = [p for _, p in seen_pages]
        for g in range(c.kv):
            top_k, top_v = (x[layer, pick, g].astype(np.float64) for x in (c.key_max, c.value_max))
            k = (c.keys[layer, pick, g] * (top_k / 127)[:, None, None]).reshape(-1, d)
            v = (c.values[layer, pick, g] * (top_v / 127)[:, None, None]).transpose(0, 2, 1).reshape(-1, d)
            magnitude = np.repeat(top_v, page)
            for h in range(g * group, (g + 1) * group):
                for i in range(count):
                    see = token <= length + i
                    if not see.any():
                        continue
                    row, q = c.starts[s] + i, q64[c.starts[s] + i, h, 0]
                    x = (k[see] @ q) * c.scale
                    p = np.exp(x - x.max())
                    p /= p.sum()
                    out = p @ v[see]
                    size = abs(c.scale) * (np.abs(k[see]) @ np.abs(q))
                    power = 2.0 ** np.frexp(np.abs(q).max())[1]
                    steps = 127 * 2.0 ** (24 if c.dtype == "f32" else 16) / power
                    lost = np.abs(np.rint(q * steps) / steps - q) + (np.abs(q) * 2.0 ** -24 if c.dtype == "f32" else 0.0)
                    delta = abs(c.scale) * (np.abs(k[see]) @ lost) + (8 * size + (x.max() - x) + 1) * 2.0 ** -24
                    gross = p @ np.abs(v[see])
                    off = (p * (delta + 2.0 ** -20)) @ (np.abs(v[see]) + np.abs(out))
                    off += (see.sum() / 16 + 16) * 2.0 ** -23 * (gross + np.abs(out))
                    off += see.sum() * 2.0 ** -34 * np.max(p * magnitude[see])
                    want[row, h], bound[row, h] = out, off
    if c.gate:
        sigmoid = 1 / (1 + np.exp(-q64[:, :, 1]))
        want, bound = want * sigmoid, (bound + np.abs(want) * 2.0 ** -21) * sigmoid
    return want, bound


def allowed(c, layer=0):
    want, bound = tight(c, layer)
    return want, bound + (np.abs(want) + bound) * HALF_STEP[c.dtype] + (2.0 ** -25 if c.dtype == "f16" else 1e-37)


def check(c, got, layer=0):
    want, bound = allowed(c, layer)
    assert np.all(np.abs(got - want) <= bound), float(np.nanmax(np.abs(got - want) / bound))


# calls that take the kernel with 16 rows a workgroup, and (a long max_length) the one with 64
FEW, MANY = None, 1 << 20


@pytest.mark.gpu
@pytest.mark.parametrize("max_length", [FEW, MANY])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads,kv,head,page,counts,lengths", [
    (8, 2, 256, 64, [5, 9, 1], [2, 0, 61]), (16, 4, 128, 16, [9, 40], [3, 1]), (12, 1, 64, 32, [17, 3], [30, 100])])
def test_rows_are_computed_in_fp32(ctx, dtype, heads, kv, head, page, counts, lengths, max_length):
    """Few tokens, so that no error of a weight is lost in the sum; more rows than eight columns hold."""
    c = Case(ctx, heads, kv, head, page, counts, lengths, dtype, gate=False, seed=heads + head)
    c.upload()
    check(c, c.run(max_length=max_length))
    c.cache.free()


@pytest.mark.gpu
@pytest.mark.parametrize("max_length", [FEW, MANY])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_queries_with_one_large_element(ctx, dtype, max_length):
    """An element 2^9 times the others, where the keys are zero: the others decide."""
    c = Case(ctx, 8, 2, 128, 32, [20, 3], [100, 7], dtype, seed=2)
    c.keys[..., 5] = 0
    c.q[:, :, 0, 5] = 2.0 ** 9 * c.q[:, :, 0].float().abs().amax(-1).to(TYPES[dtype])
    c.upload()
    check(c, c.run(max_length=max_length))
    c.cache.free()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_a_row_alone_and_among_others(ctx, dtype):
    """The same token decoded alone, with three drafts of another sequence and beside a prompt's chunk: the same bound."""
    for counts in ([1, 1], [1, 3], [1, 90]):
        for max_length in (FEW, MANY):
            c = Case(ctx, 8, 2, 128, 32, counts, [130, 6], dtype, seed=11)
            c.upload()
            check(c, c.run(max_length=max_length))
            c.cache.free()


def towards(c, s, index, factor):
    """Sequence s's queries lean on its page `index`: every head's kv head's first key there."""
    group = c.heads // c.kv
    for h in range(c.heads):
        code = c.keys[0, c.tables[s, index], h // group, 0].astype(np.float32)
        c.q[c.starts[s]:c.starts[s + 1], h, 0] = torch.from_numpy(code * (factor / 127)).to(TYPES[c.dtype])


# decode (fp32's kernel of 8 rows, four digits), 16 rows a workgroup, 64 (32 with fp32) rows a workgroup
FORMS = [([1, 2], FEW), ([12, 3], FEW), ([12, 3], MANY)]


@pytest.mark.gpu
@pytest.mark.parametrize("counts,max_length", FORMS)
@pytest.mark.parametrize("magnitude", [1e-2, 1e-9, 1e-12, 1e-30])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_pages_of_zeros_beside_quiet_ones(ctx, dtype, magnitude, counts, max_length):
    """Pages of zeros take part in the softmax, and cost the others' values none of their places: with scores like the
    others', and (the second sequence) some 20 to 45 bits ahead of them."""
    c = Case(ctx, 8, 2, 128, 16, counts, [90, 400], dtype, seed=5)
    c.value_max[:] = magnitude
    c.value_max[0, c.tables[0, 1:3]] = c.value_max[0, c.tables[1, 4]] = 0.0
    c.scale *= 0.5
    towards(c, 1, 4, 3.0)
    c.upload()
    check(c, c.run(max_length=max_length))
    c.cache.free()


@pytest.mark.gpu
@pytest.mark.parametrize("counts,max_length", FORMS)
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_magnitudes_up_to_the_largest_number(ctx, dtype, counts, max_length):
    """Pages from 2^90 to 2^127, some beside ordinary ones; quiet pages that are chosen among them."""
    c = Case(ctx, 8, 2, 64, 16, counts, [150, 300], dtype, seed=6)
    c.value_max[:] = 2.0 ** np.random.default_rng(3).uniform(90, 127, c.value_max.shape)
    c.value_max[0, c.tables[0, 3:5]] = 1.5
    c.value_max[0, c.tables[1, 2]] = 3e-30
    towards(c, 1, 2, 60.0)
    c.upload()
    got = c.run(max_length=max_length)
    assert np.all(np.isfinite(got))
    check(c, got)
    c.cache.free()


@pytest.mark.gpu
@pytest.mark.parametrize("counts,max_length", FORMS)
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_scores_beyond_24_bits(ctx, dtype, counts, max_length):
    """Queries so large that the scores' own places are whole numbers and more: one key is half of them ahead and wins
    alone, and its page's magnitude is not mixed up with another's.  Where the weight is one, roundings of the weight are
    those of one product and one quotient: 2^-18 holds all of them."""
    c = Case(ctx, 4, 2, 64, 16, counts, [70, 100], dtype, seed=7)
    c.value_max[0, c.tables[0, :4], 0] = [1e-20, 1e20, 3.0, 1e6]
    for s in range(2):
        towards(c, s, 1, 1e9)
    c.upload()
    want, _ = tight(c)
    assert np.all(np.abs(c.run(max_length=max_length) - want) <= np.abs(want) * (2.0 ** -18 + 1.01 * HALF_STEP[dtype]))
    c.cache.free()


def odd_pages(ctx, head, dtype):
    """Pages that are not there, of zeros, loud and quiet ones, in one sequence; ordinary ones in the other."""
    c = Case(ctx, 8, 2, head, 16, [30, 19], [250, 90], dtype, seed=head)
    c.tables[0, 2:4] = [-1, c.pages + 5]
    c.key_max[:, c.tables[0, 5:8]] = 0.0
    c.value_max[:, c.tables[0, 6:9]] = 0.0
    c.value_max[:, c.tables[0, 10]] = 1e4
    c.value_max[:, c.tables[0, 11]] = 1e-30
    c.key_max[:, c.tables[1, 3]] *= 3.0
    c.scale = -c.scale
    return c


def unlike_magnitudes(ctx, dtype, count):
    """Value pages from 1e-6 to 1e6."""
    c = Case(ctx, 2, 1, 64, 16, [count], [300], dtype, seed=6)
    c.value_max[0, :, 0] = 10.0 ** np.random.default_rng(1).uniform(-6, 6, c.pages)
    return c


@pytest.mark.gpu
@pytest.mark.parametrize("max_length", [FEW, MANY])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("head", [64, 128, 256])
def test_odd_pages(ctx, head, dtype, max_length):
    c = odd_pages(ctx, head, dtype)
    c.upload()
    check(c, c.run(max_length=max_length))
    c.cache.free()


@pytest.mark.gpu
@pytest.mark.parametrize("count,max_length", [(1, FEW), (20, FEW), (40, MANY)])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_unlike_magnitudes(ctx, dtype, count, max_length):
    c = unlike_magnitudes(ctx, dtype, count)
    if dtype == "f16":
        c.value_max /= 100.0  # results within its range
    c.upload()
    check(c, c.run(max_length=max_length))
    c.cache.free()


@pytest.mark.gpu
@pytest.mark.parametrize("counts,max_length", FORMS)
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_a_loud_page_ruled_out_and_a_quiet_one_chosen(ctx, dtype, counts, max_length):
    c = Case(ctx, 8, 2, 128, 64, counts, [100, 200], dtype, seed=8)
    c.value_max[0, c.tables[:, 0]] = 1e-3
    c.value_max[0, c.tables[:, 1]] = 1e3
    for s in range(2):
        towards(c, s, 0, 4.0)
    c.upload()
    check(c, c.run(max_length=max_length))
    c.cache.free()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,counts", [("f32", [1, 1, 1, 1]), ("bf16", [30, 25, 2, 1]), ("bf16", [3, 2, 2, 1])])
def test_row_starts_that_are_out_of_range(ctx, dtype, counts):
    """Clipped to the batch's rows and max_rows: those rows as a batch that says so has them, every other row and what
    lies around the output as they were."""
    c = Case(ctx, 4, 2, 64, 16, counts, [100, 60, 5, 33], dtype, seed=5)
    c.upload()
    rows, most, guard = int(c.starts[-1]), max(counts), 4
    results = []
    for starts in ([0, -5, 2 ** 31 - 1, 1, 0], [0, 0, min(rows, most), rows, rows]):
        around = torch.full((rows + 2 * guard, 4, 64), 77.0, dtype=TYPES[dtype], device="cuda")
        c.dev[0].copy_(torch.tensor(starts, dtype=torch.int32))
        lengths = [9, 60, -rows, 7] if starts[1] == 0 else [9, 60, 5, 7]
        c.dev[1].copy_(torch.tensor(lengths, dtype=torch.int32))
        c.out = around[guard:guard + rows]
        torch.cuda.synchronize()
        c.run()
        results.append(around.clone())
    got, want = (r.double().cpu().numpy() for r in results)
    inside = slice(guard, guard + min(rows, most))
    assert np.array_equal(got[inside], want[inside]) and not np.any(got[inside] == 77.0)
    got[inside] = 77.0
    assert np.all(got == 77.0)


def test_the_bounds_turn_wrong_rows_down():
    """Zeros, the negated result and results without the quieter pages are outside what the checks above allow, in every
    row and head that has a value."""
    cases = [odd_pages(None, head, dtype) for head in (64, 128, 256) for dtype in ("f32", "bf16")]
    cases += [unlike_magnitudes(None, dtype, 20) for dtype in ("f32", "bf16")]
    for c in cases:
        want, bound = allowed(c)
        there = np.abs(want).max(axis=2) > 0
        for wrong in (np.zeros_like(want), -want):
            assert np.all((np.abs(wrong - want) > bound).any(axis=2)[there])
    quiet = unlike_magnitudes(None, "f32", 20)  # half a step of bf16 is more than these pages add
    want, bound = allowed(quiet)
    quiet.value_max = np.where(quiet.value_max < 100.0, 0.0, quiet.value_max).astype(np.float32)
    without, _ = tight(quiet)
    assert np.mean((np.abs(without - want) > bound).any(axis=2)) > 0.9
