"""Draft verification through the C ABI against its definition in 64 bits: the same
tokens, the same counts."""

import numpy as np
import pytest
import torch

from fortai_amd import backend as B

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def softmax(x, t):
    x = np.minimum(np.where(np.isnan(x), -np.inf, x), np.float64(np.finfo(np.float32).max))
    if not np.any(x > -np.inf):
        return np.zeros_like(x), np.full_like(x, -np.inf)
    with np.errstate(invalid="ignore"):
        z = np.where(x > -np.inf, (x - x.max()) / (t if t > 0 else 1.0), -np.inf)
    log_sum = np.log(np.exp(z).sum())
    return np.exp(z - log_sum), z - log_sum


def definition(target, draft, tokens, uniforms, temperatures, starts):
    """emitted, accepted, logprobs; None where a float64 sum in another order could decide otherwise."""
    emitted, accepted, logprobs = np.full(len(tokens), -2), [], np.full(len(tokens), 7.0)
    for s in range(len(starts) - 1):
        a, b = starts[s], starts[s + 1]
        count, t = 0, float(temperatures[s])
        for r in range(a, b):
            p, logp = softmax(target[r], t)
            best = int(np.argmax(p)) if p.any() else -1
            x, left = (int(tokens[r + 1]), None) if r + 1 < b else (-1, p)
            if left is None:
                if draft is None:
                    q = np.zeros_like(p)
                    if 0 <= x < len(p):
                        q[x] = 1.0
                else:
                    q = softmax(draft[r], t)[0]
                if 0 <= x < len(p):
                    stands = x == best if t <= 0 else float(uniforms[r]) * q[x] < p[x]
                    if t > 0 and p[x] > 0:
                        assert abs(float(uniforms[r]) * q[x] / p[x] - 1) > 1e-11
                else:
                    stands = False
                if stands:
                    emitted[r], logprobs[r] = x, logp[x]
                    count += 1
                    continue
                left = np.maximum(p - q, 0.0)
                left = left if left.sum() > 0 else p
            if t <= 0:
                y = best
            else:
                c = np.cumsum(left)
                border = float(uniforms[b - 1]) * c[-1]
                over = np.nonzero((c > border) & (left > 0))[0]
                y = int(over[0]) if len(over) else int(np.nonzero(left)[0][-1]) if left.any() else -1
                if border > 0:
                    assert np.min(np.abs(c / border - 1)) > 1e-12
            emitted[r], logprobs[r] = y, logp[y] if y >= 0 else -np.inf
            emitted[r + 1:b], logprobs[r + 1:b] = -1, 0.0
            break
        accepted.append(count)
    return emitted, np.array(accepted), logprobs


class Step:
    def __init__(self, ctx, counts, vocab, dtype, drafts, seed, masked=False, near=0.3):
        g = torch.Generator().manual_seed(seed)
        self.ctx, self.vocab, self.dtype = ctx, vocab, dtype
        self.starts = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
        rows = int(self.starts[-1])
        self.rows = rows
        target = 3.0 * torch.randn(rows, vocab, generator=g)
        if masked:
            target[:, torch.rand(vocab, generator=g) < 0.3] = -float("inf")
        self.target = target.to(TYPES[dtype])
        self.draft = (target + near * torch.randn(rows, vocab, generator=g)).to(TYPES[dtype]) if drafts else None
        source = self.draft if drafts else self.target
        chosen = torch.multinomial(torch.softmax(source.float(), 1), 1, generator=g)[:, 0]
        self.tokens = torch.cat([torch.zeros(1, dtype=torch.int64), chosen[:-1]])
        self.uniforms = torch.rand(rows, generator=g)
        self.temperatures = 0.5 + torch.rand(len(counts), generator=g)

    def run(self, verifier=None, use_temperatures=True, target_pitch=None, draft_pitch=None):
        dev = lambda x: None if x is None else x.cuda()
        def pitched(x, pitch):
            if x is None or pitch is None:
                return dev(x)
            flat = torch.full((x.shape[0] * pitch + 1,), 1e4, dtype=x.dtype, device="cuda")
            view = torch.as_strided(flat, x.shape, (pitch, 1), 1)
            view.copy_(x)
            return view
        t, d = pitched(self.target, target_pitch), pitched(self.draft, draft_pitch)
        tokens, uniforms, temperatures, starts = dev(self.tokens), dev(self.uniforms), dev(self.temperatures), torch.from_numpy(self.starts).cuda()
        n = len(self.starts) - 1
        emitted = torch.full((self.rows + 1,), -2, dtype=torch.int64, device="cuda")
        accepted = torch.full((n + 1,), -2, dtype=torch.int32, device="cuda")
        logprobs = torch.full((self.rows + 1,), 7.0, device="cuda")
        torch.cuda.synchronize()
        v = verifier or B.Verifier(self.ctx, self.rows, n, self.vocab)
        v.run(t.data_ptr(), tokens.data_ptr(), uniforms.data_ptr(), starts.data_ptr(), n, self.rows, emitted.data_ptr(), accepted.data_ptr(),
              dtype=self.dtype, draft_logits=None if d is None else d.data_ptr(), temperatures=temperatures.data_ptr() if use_temperatures else None,
              logprobs=logprobs.data_ptr(), target_pitch=target_pitch, draft_pitch=draft_pitch)
        self.ctx.synchronize()
        if verifier is None:
            v.free()
        assert int(emitted[-1]) == -2 and int(accepted[-1]) == -2 and float(logprobs[-1]) == 7.0
        return emitted[:-1].cpu().numpy(), accepted[:-1].cpu().numpy(), logprobs[:-1].double().cpu().numpy()

    def check(self, got, use_temperatures=True):
        e, a, l = definition(self.target.double().numpy(), None if self.draft is None else self.draft.double().numpy(), self.tokens.numpy(),
                             self.uniforms.numpy(), self.temperatures.numpy() if use_temperatures else np.ones(len(self.starts)), self.starts)
        assert np.array_equal(got[0], e) and np.array_equal(got[1], a)
        # computed in 64 bits, rounded once
        same = np.isinf(l)
        assert np.array_equal(same, np.isinf(got[2])) and np.all(np.abs(got[2] - l)[~same] <= np.abs(l[~same]) * 1.01 * 2.0 ** -24 + 1e-12)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("counts,vocab,drafts,masked", [
    ([1], 1, False, False), ([5], 1000, True, False), ([5, 1, 3, 0, 9], 4096, True, True), ([2, 2, 2], 4099, False, True),
    ([4, 5, 1], 50001, True, False), ([3] * 20, 777, True, True), ([40], 129, True, False), ([5, 4], 150000, False, False)])
def test_verify_matches_the_definition(ctx, dtype, counts, vocab, drafts, masked):
    for seed in range(3):
        s = Step(ctx, counts, vocab, dtype, drafts, 100 * seed + vocab, masked)
        s.check(s.run())
    s.check(s.run(use_temperatures=False), use_temperatures=False)
    s.temperatures[::2] = 0.0
    s.temperatures[1::3] = -1.0
    s.check(s.run())


def test_verify_large_chunks_and_pitches(ctx):
    """Enough rows for the wide chunks; odd pitches and an unaligned base take the scalar loads."""
    s = Step(ctx, [5, 5, 4, 5, 2, 1, 5, 5], 70000, "f32", True, 3)
    s.check(s.run())
    s.check(s.run(target_pitch=70001, draft_pitch=70013))
    s = Step(ctx, [5] * 8, 70000, "bf16", False, 4)
    s.check(s.run(target_pitch=70002))


def test_verify_edges(ctx):
    """Uniforms of zero and next to one, certain acceptance, ties of the argmax, drafts outside the vocabulary, rows
    whose logits leave nothing, infinities and NaN."""
    vocab = 300
    s = Step(ctx, [4, 4, 4, 4, 4, 4, 4], vocab, "f32", True, 9)
    s.uniforms[:4] = 0.0                                   # all stand that have any probability
    s.uniforms[4:8] = 1.0 - 2.0 ** -24
    s.tokens[9], s.tokens[13] = vocab, -5                  # outside: do not stand
    s.target[16:20, :] = 0.0                               # all equal
    s.temperatures[4] = 0.0
    s.tokens[17:20] = torch.tensor([0, 0, 7])
    s.target[20] = -float("inf")                           # nothing left in the deciding row
    s.target[24, 3], s.target[24, 5], s.target[24, 7] = float("inf"), float("inf"), float("nan")
    s.tokens[25] = 3
    s.draft[25] = -float("inf")                            # q of a row without any weight is zero
    got = s.run()
    s.check(got)
    assert got[0][16:20].tolist() == [0, 0, 0, -1] and got[1][4] == 2
    assert got[0][20] == -1 and np.isneginf(got[2][20]) and got[1][5] == 0
    # the draft's own distribution: every draft stands, whatever the uniforms
    s = Step(ctx, [6, 6], vocab, "f32", True, 10)
    s.draft = s.target.clone()
    assert s.run()[1].tolist() == [5, 5]
    # a draft without probability under both: turned down, and what is drawn comes from p
    s = Step(ctx, [2], 8, "f32", True, 11)
    s.target[0, 2] = -float("inf")
    s.draft = s.target.clone()
    s.tokens[1] = 2
    s.check(s.run())


def test_verify_draws_the_targets_distribution(ctx):
    """20,000 sequences over 5 tokens: what comes out first is distributed as p, not as q (5 sigma)."""
    n, vocab = 20000, 5
    p, q = torch.tensor([0.5, 0.1, 0.05, 0.3, 0.05]), torch.tensor([0.1, 0.3, 0.2, 0.2, 0.2])
    g = torch.Generator().manual_seed(2)
    s = Step(ctx, [2] * n, vocab, "f32", True, 1)
    s.target = torch.log(p).repeat(2 * n, 1)
    s.draft = torch.log(q).repeat(2 * n, 1)
    s.tokens[1::2] = torch.multinomial(q, n, replacement=True, generator=g)
    s.temperatures[:] = 1.0
    emitted, accepted, _ = s.run()
    first = emitted[::2]
    for k in range(vocab):
        share = np.mean(first == k)
        assert abs(share - float(p[k])) < 5 * np.sqrt(float(p[k]) * (1 - float(p[k])) / n)
    assert abs(accepted.mean() - float(torch.minimum(p, q).sum())) < 5 * 0.5 / np.sqrt(n)


def test_verify_bad_row_starts(ctx):
    """Out of order or out of range: nothing outside the arrays moves, other sequences are right."""
    s = Step(ctx, [3, 3, 3], 100, "f32", True, 5)
    right = s.run()
    s.starts = np.array([0, 3, 1, 2 ** 31 - 1], dtype=np.int32)
    got = s.run()
    assert got[1][0] == right[1][0] and np.array_equal(got[0][:1], right[0][:1])
    s.starts = np.array([-4, 3, 6, 7], dtype=np.int32)
    got = s.run()
    assert np.array_equal(got[0][:6], right[0][:6]) and np.all(got[0][7:] == -2) and np.all(got[2][7:] == 7.0)


def test_verify_refusals(ctx):
    for bad in ((0, 1, 10), (1, 0, 10), (1, 1, 0), (65536, 1, 10), (1, 65536, 10), (1, 1, (1 << 28) + 1)):
        with pytest.raises(B.BackendError) as e:
            B.Verifier(ctx, *bad)
        assert e.value.code == B.INVALID
    v = B.Verifier(ctx, 4, 2, 64)
    x = torch.zeros(4, 64, device="cuda")
    t = torch.zeros(4, dtype=torch.int64, device="cuda")
    i = torch.zeros(3, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    good = dict(target_logits=x.data_ptr(), tokens=t.data_ptr(), uniforms=x.data_ptr(), row_starts=i.data_ptr(), sequences=2, rows=4,
                emitted=t.data_ptr(), accepted=i.data_ptr())
    for bad in (dict(sequences=3), dict(rows=5), dict(rows=-1), dict(target_logits=None), dict(tokens=None), dict(uniforms=None),
                dict(row_starts=None), dict(emitted=None), dict(accepted=None), dict(target_pitch=63), dict(draft_logits=x.data_ptr(), draft_pitch=10),
                dict(tokens=t.data_ptr() + 4), dict(target_logits=x.data_ptr() + 1), dict(logprobs=x.data_ptr() + 2)):
        with pytest.raises(B.BackendError) as e:
            v.run(**{**good, **bad})
        assert e.value.code == B.INVALID
    v.run(**{**good, "sequences": 0})
    accepted = torch.full((2,), 9, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    v.run(**{**good, "rows": 0, "target_logits": None, "accepted": accepted.data_ptr()})  # sequences without rows
    ctx.synchronize()
    assert accepted.tolist() == [0, 0]
    v.free()


def test_verify_in_a_captured_graph():
    ctx = B.Context(0)
    s = Step(ctx, [5, 3], 5000, "f32", True, 20)
    dev = [x.cuda() for x in (s.target, s.draft, s.tokens, s.uniforms, s.temperatures, torch.from_numpy(s.starts))]
    emitted, accepted = torch.empty(8, dtype=torch.int64, device="cuda"), torch.empty(2, dtype=torch.int32, device="cuda")
    logprobs = torch.empty(8, device="cuda")
    v = B.Verifier(ctx, 8, 2, 5000)
    torch.cuda.synchronize()
    ctx.capture_begin()
    v.run(dev[0].data_ptr(), dev[2].data_ptr(), dev[3].data_ptr(), dev[5].data_ptr(), 2, 8, emitted.data_ptr(), accepted.data_ptr(),
          draft_logits=dev[1].data_ptr(), temperatures=dev[4].data_ptr(), logprobs=logprobs.data_ptr())
    ctx.capture_end()
    for k in range(4):
        n = Step(ctx, [5, 3] if k % 2 else [2, 6], 5000, "f32", True, 21 + k)
        for to, x in zip(dev, (n.target, n.draft, n.tokens, n.uniforms, n.temperatures, torch.from_numpy(n.starts))):
            to.copy_(x)
        torch.cuda.synchronize()
        ctx.graph_launch()
        ctx.synchronize()
        n.check((emitted.cpu().numpy(), accepted.cpu().numpy(), logprobs.double().cpu().numpy()))
    v.free()
    ctx.close()
