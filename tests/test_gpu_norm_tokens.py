"""Residual sum, norm and gate into 8-bit tokens, against the definition in 64 bits: codes and scales exactly,
values to half a step."""

import numpy as np
import pytest
import torch

from fortai_amd import backend as B

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
EPS = 1e-6


def definition(x, residual, norm, group, gate, dtype):
    """Sum (as stored), y in 64 bits, codes and scales [rows][blocks]."""
    h = x if residual is None else (x.double() + residual.double()).to(TYPES[dtype])
    y = h.double()
    if norm is not None:
        parts = y.unflatten(1, (-1, group))
        y = (parts / torch.sqrt(parts.square().mean(dim=2, keepdim=True) + float(np.float32(EPS))) * norm.double()).flatten(1)
    if gate is not None:
        z = gate.double()
        y = y * (z / (1.0 + torch.exp(-z)))
    blocks = y.unflatten(1, (-1, 32))
    top = blocks.abs().amax(dim=2, keepdim=True)
    codes = torch.where(top > 0, torch.round((127.0 * blocks / top).float()), 0.0).flatten(1)
    scales = (top[..., 0] / 127.0).float().half().float()
    return h, y, codes, scales


def planes(tokens, rows, width):
    """Codes [rows][width] and scales [rows][blocks] of a token buffer, and the codes and scales behind the width."""
    ld, blocks = -(-rows // 128) * 128, -(-width // 128) * 4
    codes = tokens[:ld * blocks * 32].view(torch.int8).view(blocks, ld, 32)[:, :rows].transpose(0, 1).flatten(1)
    scales = tokens[ld * blocks * 32:].view(torch.float32).view(blocks, ld)[:, :rows].t()
    return codes[:, :width].float(), scales[:, :width // 32], codes[:, width:], scales[:, width // 32:]


def run(ctx, x, residual, norm, group, gate, dtype, want_sum=True, want_output=True, in_place=False):
    rows, width = x.shape
    ptr = lambda t: None if t is None else t.data_ptr()
    tokens = torch.full((B.load().fortai_hip_q8_tokens_bytes(rows, width),), 0x5A, dtype=torch.uint8, device="cuda")
    total = residual if in_place else torch.empty(rows, width, dtype=TYPES[dtype], device="cuda")
    output = torch.empty(rows, width, dtype=TYPES[dtype], device="cuda")
    values = torch.empty(rows, width, dtype=torch.float32, device="cuda")
    torch.cuda.synchronize()
    pitch = lambda t: None if t is None else t.stride(0)
    ctx.norm_tokens(x.data_ptr(), rows, width, dtype=dtype, residual=ptr(residual), sum=ptr(total) if want_sum else None,
                    norm=ptr(norm), group=group, eps=EPS, gate=ptr(gate), output=ptr(output) if want_output else None,
                    tokens=tokens.data_ptr(), x_pitch=pitch(x), residual_pitch=pitch(residual), sum_pitch=pitch(total),
                    gate_pitch=pitch(gate))
    ctx.tokens_read(tokens.data_ptr(), rows, width, values.data_ptr())
    ctx.synchronize()
    return total, output, tokens, values


def check(got, want, dtype, want_sum=True, want_output=True):
    (total, output, tokens, values), (h, y, codes, scales) = got, want
    rows, width = y.shape
    got_codes, got_scales, pad, pad_scales = planes(tokens, rows, width)
    assert torch.equal(got_codes, codes)
    assert torch.equal(got_scales, scales)
    assert not pad.any() and not pad_scales.any()
    assert torch.equal(values, codes * scales.repeat_interleave(32, dim=1))
    if want_sum:
        assert torch.equal(total, h)
    if want_output:
        # one rounding, of a 64-bit value through 32 bits: half a step (of the smallest normal number, below it), and half one of fp32
        f = torch.finfo(TYPES[dtype])
        assert ((output.double() - y).abs() <= (f.eps / 2 + 2.0 ** -24) * y.abs() + f.eps / 2 * f.tiny).all()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,width", [(1, 32), (3, 1024), (8, 160), (129, 2560), (1030, 96), (1024, 1056), (2, 9216)])
def test_residual(ctx, rows, width, dtype):
    g = torch.Generator().manual_seed(rows + width)
    x, r = ((torch.randn(rows, width, generator=g) * s).to(TYPES[dtype]).cuda() for s in (0.4, 2.0))
    w = (1.0 + 0.2 * torch.randn(width, generator=g)).cuda()
    check(run(ctx, x, r, w, width, None, dtype), definition(x, r, w, width, None, dtype), dtype)
    # into the residual stream itself, and without the sums or the values
    want = definition(x, r, w, width, None, dtype)
    check(run(ctx, x, r.clone(), w, width, None, dtype, in_place=True), want, dtype)
    check(run(ctx, x, r, w, width, None, dtype, want_sum=False, want_output=False), want, dtype, False, False)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,width,group", [(5, 2048, 128), (1, 64, 32), (1100, 320, 64), (9, 4096, 256), (2, 96, 96), (40, 96, 32)])
def test_gated_norm_of_heads(ctx, rows, width, group, dtype):
    g = torch.Generator().manual_seed(rows * width)
    x = torch.randn(rows, width, generator=g).to(TYPES[dtype]).cuda()
    # the gate is one half of a wider projection
    both = torch.randn(rows, 2 * width, generator=g).mul(3).to(TYPES[dtype]).cuda()
    w = (1.0 + 0.2 * torch.randn(group, generator=g)).cuda()
    z = both[:, width:]
    check(run(ctx, x, None, w, group, z, dtype, want_sum=False), definition(x, None, w, group, z, dtype), dtype, False)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,width", [(4, 512), (1025, 352), (33, 9216)])
def test_product_of_gate_and_up(ctx, rows, width, dtype):
    g = torch.Generator().manual_seed(rows)
    x, z = (torch.randn(rows, width, generator=g).to(TYPES[dtype]).cuda() for _ in range(2))
    check(run(ctx, x, None, None, width, z, dtype, want_sum=False), definition(x, None, None, width, z, dtype), dtype, False)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("pitch,offset", [(515, 1), (520, 2), (512, 3)])
def test_odd_addresses_and_pitches(ctx, pitch, offset, dtype):
    g = torch.Generator().manual_seed(pitch)
    rows, width = 6, 480
    store = torch.randn(rows * pitch + 8, generator=g).to(TYPES[dtype]).cuda()
    x = store[offset:offset + rows * pitch].view(rows, pitch)[:, :width]
    r = torch.randn(rows, width, generator=g).to(TYPES[dtype]).cuda()
    w = (1.0 + 0.2 * torch.randn(width, generator=g)).cuda()
    check(run(ctx, x, r, w, width, None, dtype), definition(x.contiguous(), r, w, width, None, dtype), dtype)


def test_quotients_that_are_halves(ctx):
    """Whole numbers up to 127 and halves beside them: every tie goes to the even code."""
    top = torch.tensor([127.0, 254.0, 508.0]).repeat_interleave(32).view(1, 96)
    x = torch.arange(96, dtype=torch.float32).view(1, 96) + 0.5
    x[0, ::32] = top[0, ::32]
    for gate in (None, torch.full((1, 96), 0.7371)):
        got = run(ctx, x.cuda(), None, None, 96, None if gate is None else gate.cuda(), "f32", want_sum=False)
        codes = planes(got[2], 1, 96)[0].cpu()
        assert torch.equal(codes, torch.round(127.0 * x / top))  # round() takes ties to even


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,width,group", [(7, 2048, 128), (1027, 1024, 256), (1500, 4096, 128), (1026, 2560, 2560), (3, 5120, 64)])
def test_codes_of_gated_rows_alone(ctx, rows, width, group, dtype):
    g = torch.Generator().manual_seed(rows + width + group)
    x = torch.randn(rows, width, generator=g).to(TYPES[dtype]).cuda()
    z = torch.randn(rows, width, generator=g).mul(4).to(TYPES[dtype]).cuda()
    w = (1.0 + 0.2 * torch.randn(group, generator=g)).cuda()
    want = definition(x, None, w, group, z, dtype)
    check(run(ctx, x, None, w, group, z, dtype, want_sum=False, want_output=False), want, dtype, False, False)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,width,group", [(6, 1056, 32), (1025, 2560, 128), (3, 5120, 256), (1030, 4096, 4096), (1026, 1792, 1792), (5, 4160, None)])
def test_sums_of_rows_with_any_norm(ctx, rows, width, group, dtype):
    g = torch.Generator().manual_seed(rows + width)
    x, r, z = (torch.randn(rows, width, generator=g).to(TYPES[dtype]).cuda() for _ in range(3))
    w = None if group is None else (1.0 + 0.2 * torch.randn(group, generator=g)).cuda()
    for gate in (None, z):
        want = definition(x, r, w, group or width, gate, dtype)
        check(run(ctx, x, r, w, group or width, gate, dtype), want, dtype)
        check(run(ctx, x, r.clone(), w, group or width, gate, dtype, want_output=False, in_place=True), want, dtype, True, False)


def test_gated_rows_near_the_ends_of_their_type(ctx):
    """Large and small gates, weights and rows, one in each block or all of one: the codes are still the nearest."""
    g = torch.Generator().manual_seed(3)
    width, gates = 256, (-1e4, -103.0, -89.0, -86.0, -79.0, 79.0, 3e5, 1e20)
    x = torch.randn(64, width, generator=g)
    z = torch.randn(64, width, generator=g)
    w = torch.ones(width)
    for k, gate in enumerate(gates):
        z[k, ::32] = gate
        z[8 + k] = gate
        z[16 + k] = gate * (1.0 + 0.1 * torch.rand(width, generator=g))
    x[24:32] *= 1e18
    x[32:40] *= 1e-22
    x[40:48, 32:64] *= 1e-20
    x[48:56] = 0.0
    for scale in (1.0, 1e-12, 1e12):
        want = definition(x.cuda(), None, (w * scale).cuda(), width, z.cuda(), "f32")
        got = run(ctx, x.cuda(), None, (w * scale).cuda(), width, z.cuda(), "f32", want_sum=False, want_output=False)
        fits = want[3] < 65504  # a scale beyond fp16 is infinite, and its block's values are none
        codes, scales = planes(got[2], 64, width)[:2]
        assert torch.equal(codes, want[2]) and torch.equal(scales[fits], want[3][fits]) and not torch.isfinite(scales[~fits]).any()


def test_rows_that_are_not_finite(ctx):
    x = torch.randn(4, 128)
    x[1, 40] = float("nan")
    x[2, 70] = float("inf")
    x[3] = 0.0
    w = torch.ones(128)
    values = run(ctx, x.cuda(), None, w.cuda(), 128, None, "f32", want_sum=False)[3].cpu()
    assert torch.isfinite(values[0]).all() and (values[3] == 0).all()
    assert torch.isnan(values[1]).all()                      # the norm of the row is none
    assert torch.isnan(values[2, 64:96]).all() and (values[2, :64] == 0).all() and (values[2, 96:] == 0).all()
    # without a norm only the block is lost
    values = run(ctx, x.cuda(), None, None, 128, None, "f32", want_sum=False)[3].cpu()
    assert torch.isnan(values[1, 32:64]).all() and torch.isfinite(values[1, :32]).all() and torch.isfinite(values[1, 64:]).all()


def test_tokens_go_into_the_products(ctx):
    """A product over these tokens is the one over the values that they stand for."""
    rng = np.random.default_rng(5)
    rows, width, outs = 37, 288, 64
    quants = rng.integers(-127, 128, (outs, width // 32, 32), dtype=np.int8)
    scales = rng.uniform(1e-3, 1e-1, (outs, width // 32)).astype(np.float16)
    raw = np.concatenate([scales.view(np.uint8).reshape(outs, width // 32, 2), quants.view(np.uint8)], axis=2)
    weights = B.Q8Weights(ctx, raw.reshape(-1), outs, width)
    x = torch.randn(rows, width, generator=torch.Generator().manual_seed(1)).cuda()
    got = run(ctx, x, None, torch.ones(width).cuda(), width, None, "f32", want_sum=False)
    out = torch.zeros(rows, outs, device="cuda")
    torch.cuda.synchronize()
    ctx.call("fortai_hip_q8_mmq_device", ctx.h, weights.h, got[2].data_ptr(), rows, out.data_ptr(), None, None)
    ctx.synchronize()
    w = (quants.astype(np.float64) * scales.astype(np.float64)[:, :, None]).reshape(outs, width)
    want, size = got[3].double().cpu().numpy() @ w.T, np.abs(got[3].double().cpu().numpy()) @ np.abs(w).T
    # the blocks' sums are whole numbers; a product and an addition a block in fp32
    assert (np.abs(out.double().cpu().numpy() - want) <= size * (width // 32 + 2) * 2.0 ** -24).all()
    weights.free()


def test_captured_and_replayed():
    ctx = B.Context(0)  # a context holds one graph
    g = torch.Generator().manual_seed(9)
    rows, width = 5, 256
    x, r = (torch.randn(rows, width, generator=g).cuda() for _ in range(2))
    w = torch.ones(width).cuda()
    total, tokens = torch.empty_like(x), torch.empty(B.load().fortai_hip_q8_tokens_bytes(rows, width), dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    ctx.capture_begin()
    ctx.norm_tokens(x.data_ptr(), rows, width, residual=r.data_ptr(), sum=total.data_ptr(), norm=w.data_ptr(), tokens=tokens.data_ptr())
    ctx.capture_end()
    for _ in range(3):
        x.copy_(torch.randn(rows, width, generator=g))
        torch.cuda.synchronize()
        ctx.graph_launch()
        ctx.synchronize()
        h, _, codes, scales = definition(x, r, w, width, None, "f32")
        got = planes(tokens, rows, width)
        assert torch.equal(total, h) and torch.equal(got[0], codes) and torch.equal(got[1], scales)
    ctx.close()
