"""What the operators around a step's products refuse, and offsets that pass 32 bits."""

import numpy as np
import pytest
import torch

from fortai_amd import backend as B

pytestmark = pytest.mark.gpu


def refused(f):
    with pytest.raises(B.BackendError) as e:
        f()
    assert e.value.code == B.INVALID and str(e.value)


def test_refused_calls_leave_everything_as_it_was(ctx):
    x = torch.randn(4, 64, device="cuda")
    out, ints = torch.full_like(x, 5.0), torch.zeros(8, dtype=torch.int32, device="cuda")
    tokens = torch.full((B.load().fortai_hip_q8_tokens_bytes(4, 64),), 7, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    at, o, i, t = x.data_ptr(), out.data_ptr(), ints.data_ptr(), tokens.data_ptr()
    for kw in (dict(width=48), dict(rows=-1), dict(norm=at, eps=0.0), dict(norm=at, group=48), dict(output=o, output_pitch=63),
               dict(tokens=t + 8), dict(tokens=None), dict(sum=at, sum_pitch=128), dict(residual=at + 2)):
        a = {**dict(rows=4, width=64, tokens=t), **kw}
        refused(lambda: ctx.norm_tokens(at, a.pop("rows"), a.pop("width"), **a))
    for kw in (dict(width=33), dict(rows=-1), dict(out_pitch=63)):
        a = {**dict(rows=4, width=64), **kw}
        refused(lambda: ctx.tokens_read(t, a.pop("rows"), a.pop("width"), o, **a))
    for kw in (dict(pitch=63), dict(out_pitch=63), dict(history=at), dict(masks=at), dict(window=-1), dict(bias=at, bias_pitch=5),
               dict(masks=at, mask_of=i, mask_count=1, mask_pitch=1), dict(rows=65536), dict(sequences=-1), dict(tokens=at + 4)):
        a = {**dict(sequences=1, rows=4), **kw}
        refused(lambda: ctx.adjust_logits(at, 64, o, i, a.pop("sequences"), a.pop("rows"), **a))
    for bad in ((0, 2, 1, 1, 64, 4, 0, 8), (1, 0, 1, 1, 64, 4, 0, 8), (1, 2, 2, 3, 64, 4, 0, 8), (1, 2, 1, 1, 96, 4, 0, 8),
                (1, 2, 1, 1, 64, 1, 0, 8), (1, 2, 1, 1, 64, 9, 0, 8), (1, 2, 1, 1, 64, 4, 17, 8), (1, 2, 1, 1, 64, 4, 0, 0),
                (4096, 2 ** 31 - 1, 1024, 1024, 128, 8, 16, 8)):
        refused(lambda: B.GdnCache(ctx, *bad))
    refused(lambda: B.GdnCache(ctx, 1, 2, 1, 1, 64, 4, 0, 8, storage=at, storage_bytes=64))
    cache = B.GdnCache(ctx, 1, 2, 1, 1, 64, 4, 2, 8)
    good = dict(sequences=1, rows=4, max_rows=4, row_starts=i, slots=i)
    for layer, kw, more in ((1, {}, {}), (-1, {}, {}), (0, dict(rows=9, max_rows=4), {}), (0, dict(max_rows=5), {}), (0, dict(slots=None), {}),
                            (0, dict(standing=i + 2), {}), (0, dict(sequences=-1), {}), (0, {}, dict(eps=0.0)), (0, {}, dict(out_pitch=63)),
                            (0, {}, dict(qkv_pitch=-1))):
        refused(lambda: cache.run(layer, B.GdnBatch(**{**good, **kw}), at, at, at, at, at, at, o, **more))
    refused(lambda: cache.copy_slots([0], [2]))
    refused(lambda: cache.copy_slots([0, 1], [1, 0]))
    ctx.synchronize()
    assert (out == 5.0).all() and (tokens == 7).all()
    # and nothing to do is no error
    ctx.norm_tokens(at, 0, 64, tokens=t)
    ctx.adjust_logits(at, 64, o, i, 0, 4)
    cache.run(0, B.GdnBatch(0, 0, 0, None, None), at, at, at, at, at, at, o)
    cache.copy_slots([], [])
    ctx.synchronize()
    assert (out == 5.0).all() and (tokens == 7).all()
    cache.free()


def test_caches_are_not_made_inside_a_capture():
    ctx = B.Context(0)
    x, out = torch.randn(2, 64, device="cuda"), torch.zeros(2, 64, device="cuda")
    torch.cuda.synchronize()
    ctx.capture_begin()
    refused(lambda: B.GdnCache(ctx, 1, 2, 1, 1, 64, 4, 0, 8))
    ctx.norm_tokens(x.data_ptr(), 2, 64, output=out.data_ptr())
    ctx.capture_end()
    for _ in range(3):
        out.zero_()
        torch.cuda.synchronize()
        ctx.graph_launch()
        ctx.synchronize()
        assert torch.equal(out, x)
    ctx.close()


@pytest.mark.parametrize("rows", [3, 40])
def test_slots_behind_two_to_the_31_floats(ctx, rows):
    """The last of 8300 states of 2^18 floats, and the inputs, keys and updates of slots as far behind."""
    g, shape = torch.Generator().manual_seed(rows), (1, 8300, 16, 16, 128, 4, 4)
    size = B.GdnCache.bytes(*shape)
    assert size > 4 * 2 ** 31
    storage = torch.zeros(size // 4, device="cuda")
    qkv, gates = torch.randn(2 * rows, 48 * 128, generator=g).cuda(), torch.randn(2, 2 * rows, 16, generator=g).cuda()
    conv, a, dt = torch.randn(48 * 128, 4, generator=g).cuda(), -torch.rand(16, generator=g).cuda(), torch.randn(16, generator=g).cuda()
    # the same rows twice
    qkv[rows:], gates[:, rows:] = qkv[:rows], gates[:, :rows]
    out = torch.zeros(2 * rows, 16 * 128, device="cuda")
    starts, slots = (torch.tensor(v, dtype=torch.int32).cuda() for v in ([0, rows, 2 * rows], [1, 8299]))
    torch.cuda.synchronize()
    cache = B.GdnCache(ctx, *shape, 2 * rows, storage=storage.data_ptr(), storage_bytes=size)
    batch = B.GdnBatch(2, 2 * rows, rows, starts.data_ptr(), slots.data_ptr())
    for _ in range(3):
        cache.run(0, batch, qkv.data_ptr(), gates[0].data_ptr(), gates[1].data_ptr(), conv.data_ptr(), a.data_ptr(), dt.data_ptr(),
                  out.data_ptr())
        ctx.synchronize()
        assert torch.isfinite(out).all() and out.abs().max() > 0 and torch.equal(out[:rows], out[rows:])
    state = storage[:8300 * 2 ** 18].view(8300, -1)
    assert torch.equal(state[1], state[8299]) and state[1].abs().max() > 0
    touched = torch.stack([state[i].any() for i in (0, 2, 4096, 8298)])  # 8191 is where 2^31 floats end
    assert not touched.any() and not state[8190:8193].any()
    cache.copy_slots([8299], [8192])
    ctx.synchronize()
    assert torch.equal(state[8192], state[8299])
    cache.free()


def test_rows_behind_two_to_the_31_elements(ctx):
    pitch, width = 3 * 2 ** 29, 96
    x = torch.empty(2 * pitch + 2 * width, dtype=torch.bfloat16, device="cuda")
    rows = torch.randn(3, width, generator=torch.Generator().manual_seed(1)).bfloat16().cuda()
    out = torch.zeros(3, width, dtype=torch.bfloat16, device="cuda")
    for i in range(3):
        x[i * pitch:i * pitch + width] = rows[i] if i < 2 else rows[2]
    torch.cuda.synchronize()
    ctx.norm_tokens(x.data_ptr(), 3, width, dtype="bf16", output=out.data_ptr(), x_pitch=pitch)
    ctx.synchronize()
    assert torch.equal(out, rows)
    ctx.norm_tokens(rows.data_ptr(), 3, width, dtype="bf16", output=x.data_ptr(), sum=out.data_ptr(), output_pitch=pitch)
    starts = torch.tensor([0, 3], dtype=torch.int32).cuda()
    bias = torch.arange(width, dtype=torch.float32, device="cuda")
    torch.cuda.synchronize()
    ctx.adjust_logits(x.data_ptr(), width, x.data_ptr(), starts.data_ptr(), 1, 3, dtype="bf16", pitch=pitch, out_pitch=pitch, bias=bias.data_ptr())
    ctx.synchronize()
    got = torch.stack([x[i * pitch:i * pitch + width] for i in range(3)])
    assert torch.equal(got, (rows.float() + bias).bfloat16())
