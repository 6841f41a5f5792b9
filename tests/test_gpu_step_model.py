"""Drafted steps of a small Qwen3.5 model from the operators alone: norms into tokens, the 8-bit products, a layer of
the delta rule, a layer of attention over shared pages, rules on the logits and verification; sequences that fork and
lose drafts.  Each stage is held to its definition in 64 bits on the numbers that the stage before it left."""

import threading
import types

import numpy as np
import pytest
import torch

from fortai_amd import backend as B
from fortai_amd import synth
from gdn_model import Layer, Slot
from test_gpu_kv8_attention_bounds import check as check_attention
from test_gpu_kv8_cache import Store
from test_gpu_logit_rules import Case as Rules
from test_gpu_norm_tokens import definition as norm_definition
from test_gpu_norm_tokens import planes
from test_gpu_rope import check as check_rope
from test_gpu_rope import formula as rotated
from test_gpu_rope import frequencies
from test_gpu_verify import definition as verified

pytestmark = pytest.mark.gpu

M = synth.CONFIGS["qwen35-tiny-q8emb"]
PAGE, PAGES, TABLE, PENDING, ROWS, PROMPT, WINDOW = 16, 40, 12, 4, 100, 84, 50
MATRICES = {0: ["attn_qkv", "attn_gate", "ssm_alpha", "ssm_beta", "ssm_out"], 3: ["attn_q", "attn_k", "attn_v", "attn_output"]}
SCALE = M.head_size ** -0.5


class Model:
    """Layers 0 and 3 of the model for three sequences, and every array of a step, each written by one stage."""

    def __init__(self, ctx, seed=11):
        self.ctx, self.lib = ctx, B.load()
        payload = {n: (shape, synth.tensor_payload(M, seed, n, shape, kind)) for n, shape, kind in synth.tensor_specs(M)
                   if not n.startswith(("blk.1.", "blk.2."))}
        self.w, self.dense = {}, {}
        up = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()
        for n, (shape, data) in payload.items():
            if len(shape) == 2 and "conv1d" not in n:
                self.w[n] = B.Q8Weights(ctx, data, shape[1], shape[0])
                blocks = data.reshape(shape[1], shape[0] // 32, 34)
                self.dense[n] = (blocks[:, :, 2:].view(np.int8).astype(np.float64),
                                 blocks[:, :, :2].copy().view(np.float16)[..., 0].astype(np.float64))
            else:
                self.w[n] = up(data.reshape(shape[::-1]))
        q, s = self.dense["token_embd.weight"]
        self.embed = torch.from_numpy((q * s[:, :, None]).reshape(M.vocab, M.hidden).astype(np.float32))
        self.layer = Layer(M.gdn_key_heads, M.gdn_value_heads, M.gdn_head, M.conv_kernel, PENDING, np.random.default_rng(0), M.eps)
        for name, n in (("conv", "ssm_conv1d.weight"), ("ssm_a", "ssm_a"), ("ssm_dt", "ssm_dt.bias")):
            setattr(self.layer, name, self.w["blk.0." + n].cpu().numpy())
        shape = (1, 4, M.gdn_key_heads, M.gdn_value_heads, M.gdn_head, M.conv_kernel, PENDING)
        self.states = B.GdnCache(ctx, *shape, ROWS)
        self.store = Store(1, PAGES, PAGE, M.kv_heads, M.head_size, 1)
        self.storage = up(self.store.bytes())
        torch.cuda.synchronize()
        self.cache = B.Kv8Cache(ctx, 1, PAGES, PAGE, M.kv_heads, M.head_size, storage=self.storage.data_ptr(),
                                storage_bytes=self.storage.numel())
        self.rope = B.Rope(ctx, M.rope_dim, base=M.rope_base)
        self.verifier = B.Verifier(ctx, ROWS, 3, M.vocab)
        self.pool = B.Kv8Pages(PAGES, PAGE, 3, TABLE)
        f32, wide = (lambda *s: torch.zeros(*s, device="cuda")), M.heads * M.head_size
        self.x, self.qkv, self.z = f32(ROWS, M.hidden), f32(ROWS, M.conv_size), f32(ROWS, M.gdn_inner)
        self.alpha, self.beta, self.inner = f32(ROWS, M.gdn_value_heads), f32(ROWS, M.gdn_value_heads), f32(ROWS, M.gdn_inner)
        self.q, self.k, self.v = f32(ROWS, 2 * wide), f32(ROWS, M.kv_heads * M.head_size), f32(ROWS, M.kv_heads * M.head_size)
        self.attended, self.logits, self.ruled = f32(ROWS, wide), f32(ROWS, M.vocab), f32(ROWS, M.vocab)
        self.sums = [f32(ROWS, M.hidden) for _ in range(5)]
        self.outs = [f32(ROWS, M.hidden) for _ in range(4)]
        self.ffn = [[f32(ROWS, M.ffn) for _ in range(2)] for _ in range(2)]
        self.tokens = [torch.zeros(self.lib.fortai_hip_q8_tokens_bytes(ROWS, w), dtype=torch.uint8, device="cuda")
                       for w in (M.hidden, M.gdn_inner, M.hidden, M.ffn, M.hidden, wide, M.hidden, M.ffn, M.hidden)]
        ints = {"starts": 4, "slots": 3, "standing": 3, "lengths": 3, "positions": ROWS, "mask_of": ROWS, "history_lengths": 3,
                "group_starts": 4, "shared": 3, "group_of": 3, "accepted": 3}
        self.n = {k: torch.zeros(size, dtype=torch.int32, device="cuda") for k, size in ints.items()}
        self.tables = torch.zeros(3, TABLE, dtype=torch.int32, device="cuda")
        self.ids, self.emitted = (torch.zeros(ROWS, dtype=torch.int64, device="cuda") for _ in range(2))
        self.history = torch.zeros(3, 200, dtype=torch.int64, device="cuda")
        self.uniforms, self.logprobs, self.temperatures = f32(ROWS), f32(ROWS), torch.tensor([0.0, 0.7, 0.0]).cuda()
        rng = np.random.default_rng(seed)
        self.penalties = up(np.array([[1.2, 0.1, 0.2], [1.0, 0.0, 0.0], [1.5, 0.3, 0.0]], dtype=np.float32))
        self.bias = up(0.5 * rng.standard_normal((1, M.vocab)).astype(np.float32))
        self.masks = up(rng.integers(0, 2 ** 32, (2, M.vocab // 32), dtype=np.uint32).view(np.int32))

    def product(self, tokens, name, rows, out):
        self.ctx.call("fortai_hip_q8_mmq_exact_device", self.ctx.h, self.w[name].h, tokens.data_ptr(), rows, out.data_ptr(), None, None)

    def norm(self, i, x, rows, weight=None, **more):
        width = x.shape[1]
        at = {k: v.data_ptr() if torch.is_tensor(v) else v for k, v in more.items()}
        self.ctx.norm_tokens(x.data_ptr(), rows, width, norm=None if weight is None else self.w[weight].data_ptr(), eps=M.eps,
                             tokens=self.tokens[i].data_ptr(), **at)

    def feed_forward(self, i, p, rows, tokens):
        gate, up = self.ffn[i]
        self.product(self.tokens[tokens], p + "ffn_gate.weight", rows, gate)
        self.product(self.tokens[tokens], p + "ffn_up.weight", rows, up)
        self.norm(tokens + 1, up, rows, gate=gate)
        self.product(self.tokens[tokens + 1], p + "ffn_down.weight", rows, self.outs[2 * i + 1])

    def enqueue(self, sequences, rows, most, standing, groups, verify):
        """Every launch of a step; what it depends on otherwise is in device memory."""
        n, at = {k: v.data_ptr() for k, v in self.n.items()}, self.x.data_ptr()
        self.norm(0, self.x, rows, "blk.0.attn_norm.weight", sum=self.sums[0])
        for name, out in zip(MATRICES[0], (self.qkv, self.z, self.alpha, self.beta)):
            self.product(self.tokens[0], f"blk.0.{name}.weight", rows, out)
        self.states.run(0, B.GdnBatch(sequences, rows, most, n["starts"], n["slots"], n["standing"] if standing else None),
                        self.qkv.data_ptr(), self.alpha.data_ptr(), self.beta.data_ptr(),
                        *(self.w["blk.0." + w].data_ptr() for w in ("ssm_conv1d.weight", "ssm_a", "ssm_dt.bias")),
                        self.inner.data_ptr(), eps=M.eps)
        self.norm(1, self.inner, rows, "blk.0.ssm_norm.weight", group=M.gdn_head, gate=self.z)
        self.product(self.tokens[1], "blk.0.ssm_out.weight", rows, self.outs[0])
        self.norm(2, self.outs[0], rows, "blk.0.post_attention_norm.weight", residual=self.sums[0], sum=self.sums[1])
        self.feed_forward(0, "blk.0.", rows, 2)
        self.norm(4, self.outs[1], rows, "blk.3.attn_norm.weight", residual=self.sums[1], sum=self.sums[2])
        for name, out in zip(MATRICES[3], (self.q, self.k, self.v)):
            self.product(self.tokens[4], f"blk.3.{name}.weight", rows, out)
        head, at = M.head_size, self.q.data_ptr()
        self.rope.apply(at, n["positions"], rows, M.heads, head, at, head_pitch=2 * head, out_head_pitch=2 * head,
                        norm=self.w["blk.3.attn_q_norm.weight"].data_ptr(), eps=M.eps)
        self.rope.apply(self.k.data_ptr(), n["positions"], rows, M.kv_heads, head, self.k.data_ptr(),
                        norm=self.w["blk.3.attn_k_norm.weight"].data_ptr(), eps=M.eps)
        batch = B.Kv8Batch(sequences, rows, most, n["starts"], n["lengths"], self.tables.data_ptr(), TABLE)
        self.cache.append(0, batch, self.k.data_ptr(), self.v.data_ptr())
        sharing = B.Kv8Groups(groups, rows if groups else 0, n["group_starts"], n["shared"], n["group_of"])
        self.cache.shared_attention(0, batch, sharing, at, M.heads, self.attended.data_ptr(), SCALE, TABLE * PAGE, PROMPT,
                                    gate=at + 4 * head, query_pitch=2 * M.heads * head, query_head_pitch=2 * head)
        self.norm(5, self.attended, rows)
        self.product(self.tokens[5], "blk.3.attn_output.weight", rows, self.outs[2])
        self.norm(6, self.outs[2], rows, "blk.3.post_attention_norm.weight", residual=self.sums[2], sum=self.sums[3])
        self.feed_forward(1, "blk.3.", rows, 6)
        self.norm(8, self.outs[3], rows, "output_norm.weight", residual=self.sums[3], sum=self.sums[4])
        self.product(self.tokens[8], "token_embd.weight", rows, self.logits)
        self.ctx.adjust_logits(self.logits.data_ptr(), M.vocab, self.ruled.data_ptr(), n["starts"], sequences, rows,
                               tokens=self.ids.data_ptr(), history=self.history.data_ptr(), history_pitch=self.history.shape[1],
                               history_lengths=n["history_lengths"], window=WINDOW, penalties=self.penalties.data_ptr(),
                               bias=self.bias.data_ptr(), masks=self.masks.data_ptr(), mask_count=2, mask_of=n["mask_of"])
        if verify:
            self.verifier.run(self.ruled.data_ptr(), self.ids.data_ptr(), self.uniforms.data_ptr(), n["starts"], sequences, rows,
                              self.emitted.data_ptr(), n["accepted"], temperatures=self.temperatures.data_ptr(),
                              logprobs=self.logprobs.data_ptr())

    def close(self):
        for h in [self.states, self.cache, self.rope, self.verifier, self.pool] + [w for w in self.w.values() if not torch.is_tensor(w)]:
            h.free()


class Session:
    """Three sequences that a Model goes on with, one prompt that two fork from, and what a step is told about them."""

    def __init__(self, model):
        self.m, self.texts, self.standing = model, [[], [], []], [-1, -1, -1]
        self.g = torch.Generator().manual_seed(2)

    def prepare(self, who, new, standing):
        """Room in the pages and the numbers of a step: `new` tokens of each of the sequences `who`."""
        m = self.m
        for s, tokens in zip(who, new):
            for source, target in m.pool.extend(s, len(tokens)):
                m.cache.copy_pages([source], [target])
                m.ctx.synchronize()
                for plane in (m.store.keys, m.store.values, m.store.key_max, m.store.value_max):
                    plane[0, target] = plane[0, source]
        counts = [len(t) for t in new]
        self.counts, self.who, self.rows = counts, who, sum(counts)
        self.starts = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
        self.lengths = np.array([m.pool.length(s) - c for s, c in zip(who, counts)], dtype=np.int32)
        self.tables = m.pool.tables(who)
        g_starts, shared, group_of = m.pool.groups(who)
        self.groups, self.stand = len(shared), standing
        positions = np.concatenate([n + np.arange(c) for n, c in zip(self.lengths, counts)])
        mask_of = np.concatenate([np.full(c, 1 if s == 2 else -1) for s, c in zip(who, counts)])
        rows = self.rows
        for name, a in dict(starts=self.starts, slots=who, lengths=self.lengths, positions=positions, mask_of=mask_of,
                            history_lengths=[len(self.texts[s]) for s in who], group_starts=g_starts, shared=shared, group_of=group_of,
                            standing=[] if standing is None else standing).items():
            a = torch.as_tensor(np.asarray(a, dtype=np.int32))
            m.n[name][:len(a)] = a.cuda()
        m.tables[:len(who)] = torch.from_numpy(self.tables).cuda()
        self.flat = torch.tensor([t for tokens in new for t in tokens])
        m.ids[:rows], m.x[:rows] = self.flat.cuda(), m.embed[self.flat].cuda()
        m.uniforms[:rows] = torch.rand(rows, generator=self.g).cuda()
        for i, s in enumerate(who):
            m.history[i, :len(self.texts[s])] = torch.tensor(self.texts[s], dtype=torch.int64).cuda()
        torch.cuda.synchronize()

    def run(self, verify=True):
        self.m.enqueue(len(self.who), self.rows, max(self.counts), self.stand is not None, self.groups, verify)
        self.m.ctx.synchronize()

    def prompt(self):
        text = [int(t) for t in torch.randint(0, M.vocab, (PROMPT,), generator=self.g)]
        self.prepare([0], [text], [-1])
        self.run(verify=False)
        return text

    def fork(self, text):
        m = self.m
        self.texts = [list(text) for _ in range(3)]
        m.states.copy_slots([0, 0], [1, 2])
        m.pool.fork(0, 1, PROMPT)
        m.pool.fork(0, 2, PROMPT)
        self.standing, self.last = [0, 0, 0], m.ruled[PROMPT - 1].argmax().item()
        return [self.last] * 3

    def drop(self, lengths):
        for s, n in zip(self.who, lengths):
            self.m.pool.truncate(s, int(n))


def check_products(m, tokens, name, rows, got):
    q, s = m.dense[name]
    width = q.shape[1] * 32
    codes, scales, _, _ = planes(m.tokens[tokens], rows, width)
    codes, scales = codes.double().cpu().numpy().reshape(rows, -1, 32), scales.double().cpu().numpy()
    want = np.einsum("rbk,obk,rb,ob->ro", codes, q, scales, s, optimize=True)
    size = np.einsum("rbk,obk,rb,ob->ro", np.abs(codes), np.abs(q), np.abs(scales), np.abs(s), optimize=True)
    # each block's sum is an integer below 2^24; its two products with the scales and the additions of the blocks are rounded
    # (in eight lanes, and those joined)
    assert (np.abs(got[:rows].double().cpu().numpy() - want) <= (q.shape[1] + 12) * 2.0 ** -24 * size).all(), name


def check_norm(m, i, x, rows, weight=None, residual=None, total=None, group=None, gate=None):
    w = None if weight is None else m.w[weight]
    cut = lambda a: None if a is None else a[:rows]
    h, y, codes, scales = norm_definition(x[:rows], cut(residual), w, group or x.shape[1], cut(gate), "f32")
    got = planes(m.tokens[i], rows, x.shape[1])
    assert torch.equal(got[0], codes) and torch.equal(got[1], scales), i
    if total is not None:
        assert torch.equal(total[:rows], h)


def check_step(session, slots, verify=True):
    m, rows, c = session.m, session.rows, M
    check_norm(m, 0, m.x, rows, "blk.0.attn_norm.weight", total=m.sums[0])
    for name, out in zip(MATRICES[0], (m.qkv, m.z, m.alpha, m.beta)):
        check_products(m, 0, f"blk.0.{name}.weight", rows, out)
    qkv, alpha, beta = (a[:rows].double().cpu().numpy() for a in (m.qkv, m.alpha, m.beta))
    for i, s in enumerate(session.who):
        part = slice(session.starts[i], session.starts[i + 1])
        want, bound = m.layer.run(slots[s], None if session.stand is None else session.stand[i], qkv[part], alpha[part], beta[part])
        far = np.abs(m.inner[part].double().cpu().numpy().reshape(want.shape) - want)
        assert (far <= bound + 2.0 ** -24 * np.abs(want) + 1e-37).all()
    check_norm(m, 1, m.inner, rows, "blk.0.ssm_norm.weight", group=c.gdn_head, gate=m.z)
    check_products(m, 1, "blk.0.ssm_out.weight", rows, m.outs[0])
    check_norm(m, 2, m.outs[0], rows, "blk.0.post_attention_norm.weight", m.sums[0], m.sums[1])
    for i, (p, at) in enumerate((("blk.0.", 2), ("blk.3.", 6))):
        check_products(m, at, p + "ffn_gate.weight", rows, m.ffn[i][0])
        check_products(m, at, p + "ffn_up.weight", rows, m.ffn[i][1])
        check_norm(m, at + 1, m.ffn[i][1], rows, gate=m.ffn[i][0])
        check_products(m, at + 1, p + "ffn_down.weight", rows, m.outs[2 * i + 1])
    check_norm(m, 4, m.outs[1], rows, "blk.3.attn_norm.weight", m.sums[1], m.sums[2])
    # queries and keys were rotated where they lay: their products again
    before = [torch.zeros_like(a) for a in (m.q, m.k)]
    torch.cuda.synchronize()
    for name, out in zip(MATRICES[3], before):
        m.product(m.tokens[4], f"blk.3.{name}.weight", rows, out)
    m.ctx.synchronize()
    for name, out in zip(MATRICES[3], before + [m.v]):
        check_products(m, 4, f"blk.3.{name}.weight", rows, out)
    positions, theta = m.n["positions"][:rows].cpu().numpy(), frequencies(c.rope_dim, c.rope_base)
    host = lambda a, *shape: a[:rows].double().cpu().numpy().reshape(rows, *shape)
    q, q0 = (host(a, c.heads, 2, c.head_size) for a in (m.q, before[0]))
    k, k0 = (host(a, c.kv_heads, c.head_size) for a in (m.k, before[1]))
    for x, y, norm in ((q0[:, :, 0], q[:, :, 0], "q"), (k0, k, "k")):
        want, size = rotated(x, positions, theta, False, weight=m.w[f"blk.3.attn_{norm}_norm.weight"].double().cpu().numpy())
        check_rope(y, want, size, "f32", True)
    assert np.array_equal(q[:, :, 1], q0[:, :, 1])
    m.store.append(0, k, host(m.v, c.kv_heads, c.head_size), session.starts, session.lengths, session.tables)
    assert np.array_equal(m.storage.cpu().numpy(), m.store.bytes())
    check_attention(types.SimpleNamespace(
        starts=session.starts, heads=c.heads, kv=c.kv_heads, page=PAGE, head=c.head_size, counts=session.counts, lengths=session.lengths,
        tables=session.tables, pages=PAGES, keys=m.store.keys, values=m.store.values, key_max=m.store.key_max,
        value_max=m.store.value_max, scale=SCALE, dtype="f32", gate=True,
        q=m.q[:rows].cpu().view(rows, c.heads, 2, c.head_size)), host(m.attended, c.heads, c.head_size))
    check_norm(m, 5, m.attended, rows)
    check_products(m, 5, "blk.3.attn_output.weight", rows, m.outs[2])
    check_norm(m, 6, m.outs[2], rows, "blk.3.post_attention_norm.weight", m.sums[2], m.sums[3])
    check_norm(m, 8, m.outs[3], rows, "output_norm.weight", m.sums[3], m.sums[4])
    check_products(m, 8, "token_embd.weight", rows, m.logits)
    n = len(session.who)
    rules = types.SimpleNamespace(
        logits=m.logits[:rows].cpu(), vocab=c.vocab, starts=session.starts, penalties=m.penalties.cpu().numpy(), has="pthbm",
        history=m.history.cpu().numpy(), lengths=m.n["history_lengths"][:n].cpu().numpy(), tokens=session.flat.numpy(), window=WINDOW,
        bias=m.bias.cpu().numpy().repeat(n, axis=0), mask_of=m.n["mask_of"][:rows].cpu().numpy(), dtype="f32",
        masks=np.concatenate([m.masks.cpu().numpy().view(np.uint32), np.zeros((1, c.vocab // 32), dtype=np.uint32)]))
    rules.want = lambda: Rules.want(rules)
    ruled = m.ruled[:rows].double().cpu().numpy()
    Rules.check(rules, ruled)
    if not verify:
        return None
    e, a, l = verified(ruled, None, session.flat.numpy(), m.uniforms[:rows].cpu().numpy(), m.temperatures.cpu().numpy(), session.starts)
    assert np.array_equal(m.emitted[:rows].cpu().numpy(), e) and np.array_equal(m.n["accepted"][:n].cpu().numpy(), a)
    assert (np.abs(m.logprobs[:rows].double().cpu().numpy() - l) <= np.abs(l) * 1.01 * 2.0 ** -24 + 1e-12).all()
    return e, a


def test_drafted_steps_of_a_model(ctx):
    m, random = Model(ctx), np.random.default_rng(3)
    session, slots = Session(m), [Slot(m.layer) for _ in range(3)]
    text = session.prompt()
    check_step(session, slots, verify=False)
    last = session.fork(text)
    for s in (1, 2):
        slots[s].S, slots[s].eS, slots[s].inputs = slots[0].S, slots[0].eS, slots[0].inputs
    stood = rejected = shared = 0
    for step in range(5):
        # what would follow: a step of one row each, of which nothing stands
        session.prepare([0, 1, 2], [[t] for t in last], session.standing)
        session.run()
        shared += session.groups
        guess = check_step(session, slots)[0]
        session.drop(session.lengths)
        # the same row again, with drafts behind it: the guess and others
        new = [[t, int(guess[s])] + [int(x) for x in random.integers(0, M.vocab, (step + s) % 3)] for s, t in enumerate(last)]
        if step == 3:
            new[1] = new[1][:1]
        session.prepare([0, 1, 2], new, [0, 0, 0])
        session.run()
        e, a = check_step(session, slots)
        session.drop(session.lengths + 1 + a)
        for s, tokens in enumerate(new):
            session.texts[s] += tokens[:1 + a[s]]
            last[s] = int(e[session.starts[s] + a[s]])
            stood, rejected = stood + int(a[s]), rejected + len(tokens) - 1 - int(a[s])
        session.standing = [int(n) + 1 for n in a]
    assert stood >= 8 and rejected >= 5 and shared == 5  # the greedy sequences' guesses stand, if nothing else does
    m.close()


def drafted(model, captured):
    """Four steps of 3 + 2 + 1 rows; with `captured` the first is captured and the rest replay it."""
    session, results = Session(model), []
    last = session.fork(session.prompt())
    random = np.random.default_rng(5)
    for step in range(4):
        new = [[last[s]] + [int(x) for x in random.integers(0, M.vocab, 2 - s)] for s in range(3)]
        session.prepare([0, 1, 2], new, session.standing)
        if captured and step == 0:
            model.ctx.capture_begin()
            model.enqueue(3, 6, 3, True, session.groups, True)
            model.ctx.capture_end()
        if captured:
            model.ctx.graph_launch()
            model.ctx.synchronize()
        else:
            session.run()
        a = model.n["accepted"].cpu().numpy()
        results.append([t[:6].clone() for t in (model.inner, model.attended, model.ruled, model.emitted, model.logprobs)] + [a])
        session.drop(session.lengths + 1 + a)
        for s in range(3):
            session.texts[s] += new[s][:1 + a[s]]
            last[s] = int(model.emitted[session.starts[s] + a[s]])
        session.standing = [int(n) + 1 for n in a]
    return results


def same(a, b):
    return all(torch.equal(torch.as_tensor(x), torch.as_tensor(y)) for p, q in zip(a, b) for x, y in zip(p, q))


def test_a_captured_step_of_a_model_is_replayed():
    contexts = [B.Context(0) for _ in range(2)]
    models = [Model(c) for c in contexts]
    eager, replayed = (drafted(m, captured) for m, captured in zip(models, (False, True)))
    assert same(eager, replayed)
    for m, c in zip(models, contexts):
        m.close()
        c.close()


def test_two_models_in_two_threads():
    contexts = [B.Context(0) for _ in range(3)]
    models, results = [Model(c) for c in contexts], [None] * 3
    results[2] = drafted(models[2], False)

    def work(i):
        results[i] = drafted(models[i], False)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert results[0] is not None and results[1] is not None and same(results[0], results[2]) and same(results[1], results[2])
    for m, c in zip(models, contexts):
        m.close()
        c.close()
