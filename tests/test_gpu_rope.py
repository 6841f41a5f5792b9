"""Rotary positions through the C ABI against the formula in 64 bits."""

import math

import numpy as np
import pytest
import torch

from fortai_amd import backend as B

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
HALF_STEP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}


def frequencies(rotary, base, scaling="none", factor=1.0, original=0, fast=32.0, slow=1.0):
    i = np.arange(rotary // 2, dtype=np.float64)
    theta = base ** (-2.0 * i / rotary)
    if scaling == "linear":
        return theta / factor
    if scaling == "yarn":
        at = lambda turns: rotary * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(base))
        low, high = max(math.floor(at(fast)), 0), min(math.ceil(at(slow)), rotary - 1)
        ramp = np.clip((i - low) / max(high - low, 1e-3), 0, 1)
        return theta * (1 - ramp) + theta / factor * ramp
    return theta


def formula(x, positions, theta, interleaved, attention=1.0, weight=None, eps=1e-6):
    """x [rows][heads][head] float64 -> (rotated, the magnitude that its rounding errors scale with)."""
    if weight is not None:
        x = x / np.sqrt((x * x).mean(axis=-1, keepdims=True) + eps) * weight
    r = 2 * len(theta)
    angle = positions.astype(np.float64)[:, None] * theta
    c, s = (attention * np.cos(angle))[:, None], (attention * np.sin(angle))[:, None]
    first, second = (slice(0, r, 2), slice(1, r, 2)) if interleaved else (slice(0, r // 2), slice(r // 2, r))
    out, size = x.copy(), np.abs(x)
    a, b = x[..., first], x[..., second]
    out[..., first], out[..., second] = a * c - b * s, a * s + b * c
    size[..., first] = size[..., second] = attention * (np.abs(a) + np.abs(b))
    return out, size


def check(got, want, size, dtype, normed):
    """fp32: sine and cosine of a fraction of a turn that was rounded to 24 bits (2 pi 2^-25 of the pair's size, 2 ulp of
    the functions), two products and a sum; the norm's sum of up to 256 squares in a tree of 2 + 6 levels, its mean, root,
    quotient and two products.  Then one rounding to the type (fp16 also down to its smallest step)."""
    arithmetic = (2 * math.pi * 2.0 ** -25 + 6 * 2.0 ** -24) + (14 * 2.0 ** -24 if normed else 0.0)
    bound = size * arithmetic + (np.abs(want) + size * arithmetic) * HALF_STEP[dtype] + (2.0 ** -25 if dtype == "f16" else 0)
    assert np.all(np.abs(got - want) <= bound), float(np.max(np.abs(got - want) / np.maximum(bound, 1e-300)))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,heads,head,rotary,interleaved,norm", [
    (1, 1, 256, 64, False, True), (8, 20, 256, 64, False, True), (3, 5, 64, 64, False, False),
    (5, 7, 128, 128, True, True), (2, 33, 128, 32, True, False), (7, 3, 64, 22, False, True),
    (4, 2, 96, 50, True, True), (1, 9, 4, 2, False, False), (9, 1, 256, 256, False, False), (300, 6, 20, 6, False, True)])
def test_rope_matches_the_formula(ctx, dtype, rows, heads, head, rotary, interleaved, norm):
    g = torch.Generator().manual_seed(rows * 1000 + head + rotary)
    x = torch.randn(rows, heads, head, generator=g).to(TYPES[dtype])
    positions = torch.randint(-50, 1_000_000, (rows,), generator=g).to(torch.int32)
    weight = (1 + 0.1 * torch.randn(head, generator=g)) if norm else None
    want, size = formula(x.double().numpy(), positions.numpy(), frequencies(rotary, 1e6), interleaved,
                         weight=None if weight is None else weight.double().numpy())
    dx, dp = x.cuda(), positions.cuda()
    dw = None if weight is None else weight.cuda()
    out = torch.full_like(dx, 7.0)
    torch.cuda.synchronize()
    rope = B.Rope(ctx, rotary, interleaved=interleaved, base=1e6)
    args = dict(dtype=dtype, norm=None if dw is None else dw.data_ptr())
    rope.apply(dx.data_ptr(), dp.data_ptr(), rows, heads, head, out.data_ptr(), **args)
    ctx.synchronize()
    check(out.double().cpu().numpy(), want, size, dtype, norm)
    # in place: the same bits
    rope.apply(dx.data_ptr(), dp.data_ptr(), rows, heads, head, dx.data_ptr(), **args)
    ctx.synchronize()
    assert torch.equal(dx, out)
    rope.free()


@pytest.mark.parametrize("scaling", ["linear", "yarn"])
def test_rope_scaled_contexts(ctx, scaling):
    numbers = dict(factor=8.0, original_context=4096, beta_fast=32.0, beta_slow=1.0)
    theta = frequencies(64, 1e4, scaling, 8.0, 4096)
    x = torch.randn(6, 3, 128, generator=torch.Generator().manual_seed(3))
    positions = torch.tensor([0, 1, 4095, 4096, 32767, 2 ** 31 - 1], dtype=torch.int32)
    want, size = formula(x.double().numpy(), positions.numpy(), theta, False, attention=1.2)
    rope = B.Rope(ctx, 64, base=1e4, scaling=scaling, attention_factor=1.2, **numbers)
    dx, dp = x.cuda(), positions.cuda()
    torch.cuda.synchronize()
    rope.apply(dx.data_ptr(), dp.data_ptr(), 6, 3, 128, dx.data_ptr())
    ctx.synchronize()
    # the last position's turns (up to 3.4e8) keep 2^-24 of a turn in 64 bits
    check(dx.double().cpu().numpy(), want, size, "f32", False)
    rope.free()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("offset", [0, 1])
def test_rope_pitches(ctx, dtype, offset):
    """Query heads out of [row][head][q | gate], keys out of the middle of a fused row, heads outermost, an unaligned base;
    what lies between the vectors stays as it was."""
    rows, heads, head, rotary = 5, 4, 64, 32
    g = torch.Generator().manual_seed(11)
    flat = torch.randn(rows * 1000 + 8, generator=g).to(TYPES[dtype]).cuda()
    positions = torch.arange(rows, dtype=torch.int32).cuda()
    rope = B.Rope(ctx, rotary, base=1e4)
    for row_pitch, head_pitch in ((900, 2 * head), (64, 64 * rows), (777, 65)):
        x = torch.as_strided(flat, (rows, heads, head), (row_pitch, head_pitch, 1), offset)
        want, size = formula(x.double().cpu().numpy(), np.arange(rows), frequencies(rotary, 1e4), False)
        out = torch.full((rows * 1000 + 8,), 5.0, dtype=TYPES[dtype], device="cuda")
        view = torch.as_strided(out, (rows, heads, head), (row_pitch, head_pitch, 1), offset)
        torch.cuda.synchronize()
        rope.apply(x.data_ptr(), positions.data_ptr(), rows, heads, head, view.data_ptr(), dtype=dtype,
                   row_pitch=row_pitch, head_pitch=head_pitch, out_row_pitch=row_pitch, out_head_pitch=head_pitch)
        ctx.synchronize()
        check(view.double().cpu().numpy(), want, size, dtype, False)
        view.fill_(5.0)
        assert bool((out == 5.0).all())
    # one vector broadcast over the heads (input pitch 0)
    out = torch.empty(rows, heads, head, dtype=TYPES[dtype], device="cuda")
    torch.cuda.synchronize()
    rope.apply(flat.data_ptr(), positions.data_ptr(), rows, heads, head, out.data_ptr(), dtype=dtype, row_pitch=head,
               head_pitch=0)
    ctx.synchronize()
    assert all(torch.equal(out[:, 0], out[:, h]) for h in range(heads))
    rope.free()


def test_rope_refusals(ctx):
    for bad in (dict(rope_dim=0), dict(rope_dim=7), dict(rope_dim=258), dict(rope_dim=64, base=0.0),
                dict(rope_dim=64, scaling="linear", factor=0.0), dict(rope_dim=64, scaling="yarn", factor=2.0),
                dict(rope_dim=64, attention_factor=float("nan"))):
        with pytest.raises(B.BackendError) as e:
            B.Rope(ctx, **bad)
        assert e.value.code == B.INVALID
    rope = B.Rope(ctx, 64)
    x = torch.zeros(4096, device="cuda")
    p = torch.zeros(8, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    good = (x.data_ptr(), p.data_ptr(), 2, 2, 64, x.data_ptr())
    rope.apply(*good)
    rope.apply(x.data_ptr(), p.data_ptr(), 0, 2, 64, x.data_ptr())  # no rows: nothing to do
    for args, more in (((x.data_ptr(), p.data_ptr(), -1, 2, 64, x.data_ptr()), {}),
                       ((x.data_ptr(), p.data_ptr(), 2, 2, 32, x.data_ptr()), {}),
                       ((x.data_ptr(), p.data_ptr(), 2, 2, 66, x.data_ptr()), {}),
                       ((None, p.data_ptr(), 2, 2, 64, x.data_ptr()), {}),
                       ((x.data_ptr() + 2, p.data_ptr(), 2, 2, 64, x.data_ptr()), {}),
                       ((x.data_ptr(), p.data_ptr(), 2, 2, 64, x.data_ptr()), dict(out_row_pitch=512)),
                       (good, dict(out_head_pitch=32)), (good, dict(norm=x.data_ptr(), eps=0.0))):
        with pytest.raises(B.BackendError) as e:
            rope.apply(*args, **more)
        assert e.value.code == B.INVALID and "rope" in str(e.value)
    rope.free()


def test_rope_in_a_captured_graph():
    """New positions and inputs in the same arrays, replayed."""
    ctx = B.Context(0)
    rope = B.Rope(ctx, 64, base=1e5)
    x = torch.zeros(4, 6, 128, device="cuda")
    p = torch.zeros(4, dtype=torch.int32, device="cuda")
    out = torch.zeros_like(x)
    torch.cuda.synchronize()
    ctx.capture_begin()
    rope.apply(x.data_ptr(), p.data_ptr(), 4, 6, 128, out.data_ptr())
    ctx.capture_end()
    for k in range(3):
        x.copy_(torch.randn(4, 6, 128, generator=torch.Generator().manual_seed(k)))
        p.copy_(torch.arange(4) + 100 * k)
        torch.cuda.synchronize()
        ctx.graph_launch()
        ctx.synchronize()
        want, size = formula(x.double().cpu().numpy(), p.cpu().numpy(), frequencies(64, 1e5), False)
        check(out.double().cpu().numpy(), want, size, "f32", False)
    rope.free()
    ctx.close()
