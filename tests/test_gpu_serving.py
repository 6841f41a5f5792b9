"""The serving operators together, as a step with drafts uses them: rotary
positions, append, attention and verification over sequences that fork, lose their
rejected tokens and are moved by a compaction.  Every stage is held to its definition
in 64 bits on the inputs that the stage before it left; the cache byte for byte."""

import subprocess
import threading

import numpy as np
import pytest
import torch

from fortai_amd import backend as B
from fortai_amd import build
from test_gpu_kv8_cache import Store
from test_gpu_rope import formula as rotated, frequencies
from test_gpu_verify import definition

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
HALF_STEP = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8}
HEADS, KV, HEAD, ROTARY, PAGE, PAGES, VOCAB, LAYERS, LAYER = 8, 2, 64, 32, 16, 24, 96, 2, 1
SCALE = HEAD ** -0.5


def attend(store, q, table, length, single):
    """Rows q [rows][heads][head] (float64) of one sequence: the result, and how far the kernel may be off."""
    rows, group = len(q), HEADS // KV
    want, bound = np.zeros_like(q), np.zeros_like(q)
    pages = table[:-(-(length + rows) // PAGE)]
    for h in range(HEADS):
        top_k, top_v = (x[LAYER, pages, h // group].astype(np.float64)[:, None, None] / 127 for x in (store.key_max, store.value_max))
        k = (store.keys[LAYER, pages, h // group] * top_k).reshape(-1, HEAD)
        v = (store.values[LAYER, pages, h // group] * top_v).transpose(0, 2, 1).reshape(-1, HEAD)
        for i in range(rows):
            n = length + i + 1
            x = k[:n] @ q[i, h] * SCALE
            p = np.exp(x - x.max())
            p /= p.sum()
            want[i, h] = p @ v[:n]
            # the queries keep 2^-23 of their row's largest (two digits: 2^-15), 64 additions, three roundings of the score;
            # exp2, the product with the magnitude and n additions in 16ths; p as one fp16 number: 2^-11, sum p = 1
            size = SCALE * np.abs(k[:n]) @ np.abs(q[i, h])
            delta = np.max(SCALE * np.abs(q[i, h]).max() * np.abs(k[:n]).sum(1) * (2.0 ** -15 if single else 2.0 ** -23)
                           + size * HEAD * 2.0 ** -24 + (np.abs(x) + 150) * 3 * 2.0 ** -24)
            bound[i, h] = (p @ np.abs(v[:n])) * (2 * delta + 8 * 2.0 ** -24 + 2 * (n / 16 + 64) * 2.0 ** -24)
            if single:
                bound[i, h] += 127 * top_v.max() * 2.0 ** -11
    return want, bound


class Serving:
    """Three sequences of one layer over one pool, with buffers for up to `rows` rows."""

    def __init__(self, ctx, dtype, seed, rows=64):
        self.ctx, self.dtype, t = ctx, dtype, TYPES[dtype]
        g = torch.Generator().manual_seed(seed)
        self.g, self.embed = g, torch.randn(VOCAB, (HEADS + 2 * KV) * HEAD, generator=g)
        self.head = torch.randn(HEADS * HEAD, VOCAB, generator=g)
        self.norm = 1.0 + 0.1 * torch.randn(HEAD, generator=g)
        self.rope = B.Rope(ctx, ROTARY, base=1.0e6, scaling="yarn", factor=4.0, original_context=64)
        self.theta = frequencies(ROTARY, 1.0e6, "yarn", 4.0, 64)
        self.store = Store(LAYERS, PAGES, PAGE, KV, HEAD, seed)
        self.storage = torch.from_numpy(self.store.bytes()).cuda()
        self.cache = B.Kv8Cache(ctx, LAYERS, PAGES, PAGE, KV, HEAD, storage=self.storage.data_ptr(), storage_bytes=self.storage.numel())
        self.pool = B.Kv8Pages(PAGES, PAGE, 3, 8)
        self.verifier = B.Verifier(ctx, rows, 3, VOCAB)
        dev = lambda *shape, d=torch.int32: torch.zeros(*shape, dtype=d, device="cuda")
        self.x = dev(rows, HEADS + 2 * KV, HEAD, d=t)  # query heads, key heads, value heads, as a fused projection leaves them
        self.out, self.weights = dev(rows, HEADS * HEAD, d=t), self.norm.cuda()
        self.positions, self.starts, self.lengths, self.tables = dev(rows), dev(4), dev(3), dev(3, 8)
        self.tokens, self.emitted = dev(rows, d=torch.int64), dev(rows, d=torch.int64)
        self.accepted, self.logprobs = dev(3), dev(rows, d=torch.float32)
        self.uniforms, self.temperatures = dev(rows, d=torch.float32), torch.tensor([0.7, 1.0, 0.0], device="cuda")
        self.draft = dev(rows, VOCAB, d=torch.float32)
        self.logits = dev(rows, VOCAB, d=torch.float32)

    def close(self):
        for h in (self.rope, self.cache, self.pool, self.verifier):
            h.free()

    def prepare(self, tokens, copies=True):
        """The step's inputs on the device: tokens[s] are the next tokens of sequence s, with room made for them."""
        pairs = [p for s, new in enumerate(tokens) if new for p in self.pool.extend(s, len(new))]
        if pairs:
            self.move(*zip(*pairs))
        self.host_starts = np.concatenate([[0], np.cumsum([len(x) for x in tokens])]).astype(np.int32)
        self.host_lengths = np.array([self.pool.length(s) - len(x) for s, x in enumerate(tokens)], dtype=np.int32)
        self.host_tables = self.pool.tables([0, 1, 2])
        self.rows = int(self.host_starts[-1])
        flat = torch.tensor([t for x in tokens for t in x])
        self.host_positions = np.concatenate([l + np.arange(len(x)) for l, x in zip(self.host_lengths, tokens)])
        put = lambda to, x: to.view(-1)[:x.numel()].copy_(x.reshape(-1))
        put(self.tokens, flat)
        put(self.positions, torch.from_numpy(self.host_positions.astype(np.int32)))
        for to, x in ((self.starts, self.host_starts), (self.lengths, self.host_lengths), (self.tables, self.host_tables)):
            put(to, torch.from_numpy(x))
        put(self.x, self.embed[flat].to(TYPES[self.dtype]))
        self.before = self.x.double().cpu().numpy()[:self.rows]
        self.batch = B.Kv8Batch(3, self.rows, int(np.diff(self.host_starts).max()), self.starts.data_ptr(), self.lengths.data_ptr(),
                                self.tables.data_ptr(), 8)
        torch.cuda.synchronize()

    def move(self, source, target):
        self.cache.copy_pages(source, target)
        for f, t in zip(source, target):
            for plane in (self.store.keys, self.store.values, self.store.key_max, self.store.value_max):
                plane[:, t] = plane[:, f]

    def layer(self, max_length):
        """Query and key heads rotated in place, keys and values stored, attention."""
        at, e, width = self.x.data_ptr(), self.x.element_size(), (HEADS + 2 * KV) * HEAD
        self.rope.apply(at, self.positions.data_ptr(), self.rows, HEADS + KV, HEAD, at, dtype=self.dtype, row_pitch=width,
                        out_row_pitch=width, norm=self.weights.data_ptr())
        self.cache.append(LAYER, self.batch, at + HEADS * HEAD * e, at + (HEADS + KV) * HEAD * e, dtype=self.dtype, key_pitch=width,
                          value_pitch=width)
        self.cache.attention(LAYER, self.batch, at, HEADS, self.out.data_ptr(), SCALE, max_length, dtype=self.dtype, query_pitch=width)

    def check_layer(self):
        n, rows = HEADS + KV, slice(0, self.rows)
        x = self.x.double().cpu().numpy()[rows]
        want, size = rotated(self.before[:, :n], self.host_positions, self.theta, False, weight=self.norm.double().numpy())
        arithmetic = size * (2 * np.pi * 2.0 ** -25 + 20 * 2.0 ** -24)  # as in the tests of rotary positions
        assert np.all(np.abs(x[:, :n] - want) <= arithmetic + (np.abs(want) + arithmetic) * HALF_STEP[self.dtype])
        assert np.array_equal(x[:, n:], self.before[:, n:])
        self.store.append(LAYER, x[:, HEADS:n], x[:, n:], self.host_starts, self.host_lengths, self.host_tables)
        assert np.array_equal(self.storage.cpu().numpy(), self.store.bytes())
        got = self.out.double().cpu().numpy()[rows].reshape(self.rows, HEADS, HEAD)
        single = self.dtype != "f32" and self.batch.max_rows * HEADS // KV > 8
        for s in range(3):
            a, b = self.host_starts[s:s + 2]
            if a == b:
                continue
            want, bound = attend(self.store, x[a:b, :HEADS], self.host_tables[s], int(self.host_lengths[s]), single)
            bound = bound + (np.abs(want) + bound) * HALF_STEP[self.dtype] + 1e-37
            assert np.all(np.abs(got[a:b] - want) <= bound), float(np.max(np.abs(got[a:b] - want) / bound))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_drafted_steps_over_forks_and_compactions(ctx, dtype):
    m = Serving(ctx, dtype, seed=3)
    random = np.random.default_rng(5)
    texts = [[int(t) for t in torch.randint(0, VOCAB, (37,), generator=m.g)], [], []]
    m.prepare([texts[0], [], []])
    m.layer(37)
    ctx.synchronize()
    m.check_layer()
    for s in (1, 2):
        m.pool.fork(0, s, 37)
        texts[s] = list(texts[0])
    moved, stood = 0, 0
    last = [int(random.integers(VOCAB)) for _ in range(3)]  # drawn, not in the cache yet
    for step in range(12):
        drafts = torch.randn(3, 4, VOCAB, generator=m.g)
        new = [[last[s], *(int(t) for t in torch.multinomial(torch.softmax(drafts[s, :3], 1), 1, generator=m.g)[:, 0])]
               for s in range(3)]
        new[step % 3] = new[step % 3][:1 + step % 4]  # as many drafts as there are
        m.prepare(new)
        m.draft[:m.rows].copy_(torch.cat([drafts[s, :len(x)] for s, x in enumerate(new)]))
        m.uniforms[:m.rows].copy_(torch.rand(m.rows, generator=m.g))
        torch.cuda.synchronize()
        m.layer(int(max(m.host_lengths)) + 4)
        ctx.synchronize()
        m.check_layer()
        # a head that leans towards the drafts' distribution, so that some stand
        m.logits[:m.rows] = m.draft[:m.rows] + 0.03 * m.out[:m.rows].float() @ m.head.cuda()
        torch.cuda.synchronize()
        m.verifier.run(m.logits.data_ptr(), m.tokens.data_ptr(), m.uniforms.data_ptr(), m.starts.data_ptr(), 3, m.rows,
                       m.emitted.data_ptr(), m.accepted.data_ptr(), draft_logits=m.draft.data_ptr(),
                       temperatures=m.temperatures.data_ptr(), logprobs=m.logprobs.data_ptr())
        ctx.synchronize()
        host = lambda x: x[:m.rows].cpu().numpy()
        emitted, accepted, logprobs = definition(host(m.logits).astype(np.float64), host(m.draft).astype(np.float64), host(m.tokens),
                                                 host(m.uniforms), m.temperatures.cpu().numpy(), m.host_starts)
        assert np.array_equal(host(m.emitted), emitted) and np.array_equal(m.accepted.cpu().numpy(), accepted)
        # fp32 of a logarithm that was taken in 64 bits from fp32 exponents: 2^-20 relative, 2^-20 next to 0
        assert np.allclose(host(m.logprobs), logprobs, rtol=2.0 ** -20, atol=2.0 ** -20)
        for s in range(3):
            keep = 1 + int(accepted[s])
            texts[s] += new[s][:keep]
            last[s] = int(emitted[m.host_starts[s] + keep - 1])
            m.pool.truncate(s, len(texts[s]))
            assert m.pool.length(s) == len(texts[s])
        stood += int(accepted.sum())
        if step % 4 == 3:  # one sequence ends, another forks in its place, the pool closes its gaps
            gone, source = step // 4 % 3, (step // 4 + 1) % 3
            m.pool.truncate(gone)
            cut = len(texts[source]) - 3
            m.pool.fork(source, gone, cut)
            texts[gone], last[gone] = texts[source][:cut], texts[source][cut]
            f, t = m.pool.compact()
            moved += len(f)
            if len(f):
                m.move(f, t)
    assert moved > 0 and stood > 0
    m.close()


def test_a_captured_step_is_replayed():
    """A step's four operators in one graph; tokens, lengths and tables change between the replays."""
    ctx = B.Context(0)
    m = Serving(ctx, "bf16", seed=8)

    def inputs(k):
        for s in range(3):
            m.pool.truncate(s)
            m.pool.extend(s, 30 * s + 7 * k)
        m.prepare([[int(t) for t in torch.randint(0, VOCAB, (3,), generator=m.g)] for _ in range(3)])
        m.uniforms.copy_(torch.rand(m.uniforms.shape, generator=m.g))
        m.logits.copy_(torch.randn(m.logits.shape, generator=m.g))
        torch.cuda.synchronize()

    def step():
        m.layer(100)
        m.verifier.run(m.logits.data_ptr(), m.tokens.data_ptr(), m.uniforms.data_ptr(), m.starts.data_ptr(), 3, m.rows,
                       m.emitted.data_ptr(), m.accepted.data_ptr(), temperatures=m.temperatures.data_ptr(),
                       logprobs=m.logprobs.data_ptr())

    results = lambda: [x.clone() for x in (m.x, m.out, m.storage, m.emitted, m.accepted, m.logprobs)]
    inputs(0)
    ctx.capture_begin()
    step()
    ctx.capture_end()
    for k in range(4):
        inputs(k)
        x, storage = m.x.clone(), m.storage.clone()
        torch.cuda.synchronize()
        ctx.graph_launch()
        ctx.synchronize()
        replayed = results()
        m.check_layer()
        m.x.copy_(x)
        m.storage.copy_(storage)
        torch.cuda.synchronize()
        step()
        ctx.synchronize()
        for a, b in zip(replayed, results()):
            assert torch.equal(a, b)
    m.close()
    ctx.close()


def test_handles_are_not_made_inside_a_capture():
    ctx = B.Context(0)
    rope = B.Rope(ctx, 64)
    x, positions = torch.ones(4, 64, device="cuda"), torch.arange(4, dtype=torch.int32, device="cuda")
    out = torch.zeros_like(x)
    torch.cuda.synchronize()
    ctx.capture_begin()
    for make in (lambda: B.Rope(ctx, 64), lambda: B.Kv8Cache(ctx, 1, 2, 16, 1, 64), lambda: B.Verifier(ctx, 4, 1, 100)):
        with pytest.raises(B.BackendError):
            make()
    rope.apply(x.data_ptr(), positions.data_ptr(), 4, 1, 64, out.data_ptr())
    ctx.capture_end()
    for _ in range(3):
        out.zero_()
        torch.cuda.synchronize()
        ctx.graph_launch()
        ctx.synchronize()
        assert torch.equal(out[0], x[0]) and bool((out[1:] != x[1:]).any())
    rope.free()
    ctx.close()


def test_three_caches_and_three_threads(ctx):
    """Two caches of one context and a third of another one, called from three host threads at once."""
    other = B.Context(0)
    g = torch.Generator().manual_seed(0)
    q = torch.randn(4, 8, 64, generator=g).cuda()
    kv = torch.randn(2, 4, 2, 64, generator=g).cuda()
    ints = [torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([0, 3, 4], [0, 0], [[1, 2], [0, 3]])]
    batch = B.Kv8Batch(2, 4, 3, *(i.data_ptr() for i in ints), 2)
    torch.cuda.synchronize()
    made = [(c, B.Kv8Cache(c, 1, 4, 16, 2, 64), torch.zeros(4, 8, 64, device="cuda")) for c in (ctx, ctx, other)]
    torch.cuda.synchronize()

    def work(c, cache, out):
        for _ in range(20):
            cache.append(0, batch, kv[0].data_ptr(), kv[1].data_ptr())
            cache.attention(0, batch, q.data_ptr(), 8, out.data_ptr(), 0.125, 1 << 16)

    threads = [threading.Thread(target=work, args=m) for m in made]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for c, _, _ in made:
        c.synchronize()
    assert torch.equal(made[0][2], made[1][2]) and torch.equal(made[0][2], made[2][2])
    assert bool((made[0][2].abs().amax(-1) > 0).all())  # single elements may be codes of zero
    for _, cache, _ in made:
        cache.free()
    other.close()


def test_fortran_callers():
    r = subprocess.run([build.SERVING_SMOKE, "gpu"], capture_output=True, text=True, timeout=120)
    print(r.stdout, r.stderr, flush=True)
    assert r.returncode == 0 and "fortran serving smoke ok" in r.stdout
