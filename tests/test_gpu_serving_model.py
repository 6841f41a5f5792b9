"""A layer's step as the Qwen3.5 models here are laid out: queries and gates of a
head side by side in one projection's output, keys and values in outputs of their
own, query and key norms with weights of their own; drafts, some of them rejected.
Each stage is held to its definition in 64 bits."""

import types

import numpy as np
import pytest
import torch

from fortai_amd import backend as B
from fortai_amd import synth
from test_gpu_kv8_attention_bounds import check as check_attention
from test_gpu_kv8_cache import Store
from test_gpu_rope import check as check_rope
from test_gpu_rope import formula as rotated
from test_gpu_rope import frequencies
from test_gpu_verify import definition

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("model", ["qwen35-tiny", "qwen35-0.8b"])
def test_a_layer_with_two_norms_and_gated_queries(ctx, model, dtype):
    m = synth.CONFIGS[model]
    heads, kv, head, vocab, page, t = m.heads, m.kv_heads, m.head_size, 97, 16, TYPES[dtype]
    g = torch.Generator().manual_seed(heads)
    norms = [1.0 + 0.2 * torch.randn(head, generator=g) for _ in range(2)]
    weights = [n.cuda() for n in norms]
    embed = [torch.randn(vocab, n, head, generator=g) for n in (2 * heads, kv, kv)]
    theta = frequencies(m.rope_dim, m.rope_base)
    rope = B.Rope(ctx, m.rope_dim, base=m.rope_base)
    store = Store(1, 24, page, kv, head, 1)
    storage = torch.from_numpy(store.bytes()).cuda()
    cache = B.Kv8Cache(ctx, 1, 24, page, kv, head, storage=storage.data_ptr(), storage_bytes=storage.numel())
    pool, verifier = B.Kv8Pages(24, page, 2, 9), B.Verifier(ctx, 80, 2, vocab)
    scale, random = head ** -0.5, np.random.default_rng(4)
    texts = [[int(x) for x in random.integers(0, vocab, n)] for n in (37, 6)]
    stood = rejected = 0
    for step in range(7):
        new = texts if step == 0 else [[int(x) for x in random.integers(0, vocab, n)] for n in (1 + step % 4, 5)]
        for s, tokens in enumerate(new):
            for source, target in pool.extend(s, len(tokens)):
                cache.copy_pages([source], [target])
        starts = np.concatenate([[0], np.cumsum([len(x) for x in new])]).astype(np.int32)
        lengths = np.array([pool.length(s) - len(x) for s, x in enumerate(new)], dtype=np.int32)
        tables, rows = pool.tables([0, 1]), int(starts[-1])
        positions = np.concatenate([n + np.arange(len(x)) for n, x in zip(lengths, new)]).astype(np.int32)
        flat = torch.tensor([x for tokens in new for x in tokens])
        q, k, v = (e[flat].to(t).cuda() for e in embed)
        q = q.view(rows, heads, 2, head)  # [query | gate]
        before = [x.double().cpu().numpy() for x in (q, k, v)]
        d_starts, d_lengths, d_tables, d_positions = (torch.from_numpy(x).cuda() for x in (starts, lengths, tables, positions))
        out = torch.full((rows, heads, head), 9.0, dtype=t, device="cuda")
        batch = B.Kv8Batch(2, rows, int(np.diff(starts).max()), d_starts.data_ptr(), d_lengths.data_ptr(), d_tables.data_ptr(), 9)
        torch.cuda.synchronize()
        # the layer: both norms and rotations in place, keys and values stored, gated attention
        at = q.data_ptr()
        rope.apply(at, d_positions.data_ptr(), rows, heads, head, at, dtype=dtype, head_pitch=2 * head, out_head_pitch=2 * head,
                   norm=weights[0].data_ptr())
        rope.apply(k.data_ptr(), d_positions.data_ptr(), rows, kv, head, k.data_ptr(), dtype=dtype, norm=weights[1].data_ptr())
        cache.append(0, batch, k.data_ptr(), v.data_ptr(), dtype=dtype)
        cache.attention(0, batch, at, heads, out.data_ptr(), scale, int((lengths + np.diff(starts)).max()), dtype=dtype,
                        gate=at + head * q.element_size(), query_pitch=2 * heads * head, query_head_pitch=2 * head)
        ctx.synchronize()
        after = [x.double().cpu().numpy() for x in (q, k, v)]
        for x, y, norm in ((before[0][:, :, 0], after[0][:, :, 0], norms[0]), (before[1], after[1], norms[1])):
            want, size = rotated(x, positions, theta, False, weight=norm.double().numpy())
            check_rope(y, want, size, dtype, True)
        assert np.array_equal(before[0][:, :, 1], after[0][:, :, 1]) and np.array_equal(before[2], after[2])
        store.append(0, after[1], after[2], starts, lengths, tables)
        assert np.array_equal(storage.cpu().numpy(), store.bytes())
        check_attention(types.SimpleNamespace(
            starts=starts, heads=heads, kv=kv, page=page, head=head, counts=np.diff(starts), lengths=lengths, tables=tables, pages=24,
            keys=store.keys, values=store.values, key_max=store.key_max, value_max=store.value_max, scale=scale, dtype=dtype,
            gate=True, q=q.cpu()), out.double().cpu().numpy())
        if step == 0:
            continue
        draft = torch.randn(rows, vocab, generator=g)
        draft[torch.arange(rows - 1), flat[1:]] += 2.0
        logits = (draft + 0.5 * torch.randn(rows, vocab, generator=g)).cuda()
        draft, d_tokens, uniforms = draft.cuda(), flat.cuda(), torch.rand(rows, generator=g)
        d_uniforms, temperatures = uniforms.cuda(), torch.tensor([0.8, 0.0], device="cuda")
        emitted, accepted = torch.zeros(rows, dtype=torch.int64, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
        logprobs = torch.zeros(rows, device="cuda")
        torch.cuda.synchronize()
        verifier.run(logits.data_ptr(), d_tokens.data_ptr(), d_uniforms.data_ptr(), d_starts.data_ptr(), 2, rows, emitted.data_ptr(),
                     accepted.data_ptr(), draft_logits=draft.data_ptr(), temperatures=temperatures.data_ptr(),
                     logprobs=logprobs.data_ptr())
        ctx.synchronize()
        host = lambda x: x.cpu().numpy()
        e, a, l = definition(host(logits).astype(np.float64), host(draft).astype(np.float64), flat.numpy(), uniforms.numpy(),
                             host(temperatures), starts)
        assert np.array_equal(host(emitted), e) and np.array_equal(host(accepted), a)
        # computed in 64 bits, rounded once
        assert np.all(np.abs(host(logprobs).astype(np.float64) - l) <= np.abs(l) * 1.01 * 2.0 ** -24 + 1e-12)
        for s in range(2):
            pool.truncate(s, int(lengths[s]) + 1 + int(a[s]))
            stood, rejected = stood + int(a[s]), rejected + len(new[s]) - 1 - int(a[s])
    assert stood > 0 and rejected > 0
    for h in (rope, cache, pool, verifier):
        h.free()
