"""The gated delta rule over a batch's rows, against the definition in 64 bits row by row: decode steps, drafts
that stand or do not, prompts, and all of them in one call."""

import numpy as np
import pytest
import torch

from fortai_amd import backend as B
from gdn_model import Layer, Slot

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


class Run:
    """A cache of two layers over storage of its own, beside the model's slots of the second."""

    def __init__(self, ctx, seed, kh, vh, d, taps, pending, slots, max_rows, dtype="f32"):
        self.ctx, self.rng, self.dtype, self.slots = ctx, np.random.default_rng(seed), dtype, slots
        self.layer = Layer(kh, vh, d, taps, pending, self.rng)
        c = self.layer
        shape = (2, slots, kh, vh, d, taps, pending)
        self.storage = torch.zeros(B.GdnCache.bytes(*shape) // 4, device="cuda")
        torch.cuda.synchronize()
        self.cache = B.GdnCache(ctx, *shape, max_rows, storage=self.storage.data_ptr(), storage_bytes=4 * self.storage.numel())
        self.model = [Slot(c) for _ in range(slots)]
        self.weights = [torch.from_numpy(a).cuda() for a in (c.conv, c.ssm_a, c.ssm_dt)]

    def planes(self):
        c, n = self.layer, self.slots
        shapes = [(n, c.vh, c.d, c.d), (n, c.taps - 1 + c.pending, c.channels), (n, c.pending, c.kh, c.d),
                  (n, c.pending, c.vh, c.d), (n, c.pending, c.vh), (n,)]
        out, at = [], 0
        for shape in shapes:
            size = int(np.prod(shape))
            out.append(self.storage[at + size:at + 2 * size].cpu().numpy().reshape(shape))  # the second layer
            assert not self.storage[at:at + size].any()  # the first is left alone
            at += 2 * size
        out[5] = out[5].view(np.int32)
        return out

    def step(self, counts, slots, standing, pad=0, extra=0):
        """One call; counts[s] rows of the sequence in slots[s]; the arrays have `extra` rows of nobody and pitches
        that are `pad` larger than dense."""
        c, t, rows = self.layer, TYPES[self.dtype], sum(counts)
        draw = lambda width: torch.from_numpy(self.rng.standard_normal((rows + extra, width + pad)).astype(np.float32)).to(t)
        x, alpha, beta = draw(c.channels), draw(c.vh), draw(c.vh)
        out = torch.full((rows + extra, c.vh * c.d + pad), 9.0, dtype=t)
        dev = [a.cuda() for a in (x, alpha, beta, out)]
        starts = torch.tensor(np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)).cuda()
        slot = torch.tensor(slots, dtype=torch.int32).cuda()
        stand = None if standing is None else torch.tensor(standing, dtype=torch.int32).cuda()
        batch = B.GdnBatch(len(counts), rows + extra, max(counts), starts.data_ptr(), slot.data_ptr(), None if stand is None else stand.data_ptr())
        torch.cuda.synchronize()
        self.cache.run(1, batch, *(a.data_ptr() for a in dev[:3]), *(w.data_ptr() for w in self.weights), dev[3].data_ptr(),
                       dtype=self.dtype, qkv_pitch=c.channels + pad, alpha_pitch=c.vh + pad, beta_pitch=c.vh + pad,
                       out_pitch=c.vh * c.d + pad)
        self.ctx.synchronize()
        got = dev[3].double().cpu().numpy()
        assert (got[rows:] == 9.0).all() and (got[:, c.vh * c.d:] == 9.0).all()
        half, at = torch.finfo(t).eps / 2, 0
        x, alpha, beta = (a.double().numpy()[:, :w] for a, w in ((x, c.channels), (alpha, c.vh), (beta, c.vh)))
        worst = 0.0
        for s, n in enumerate(counts):
            if n == 0:
                continue
            want, bound = c.run(self.model[slots[s]], None if standing is None else standing[s], x[at:at + n], alpha[at:at + n], beta[at:at + n])
            far = np.abs(got[at:at + n, :c.vh * c.d].reshape(want.shape) - want)
            bound = bound + half * np.abs(want) + torch.finfo(t).tiny * half
            assert (far <= bound).all(), (s, n, (far / bound).max())
            at += n
        return got

    def check_storage(self):
        c = self.layer
        S, inputs, keys, updates, decays, counts = (a.astype(np.float64) for a in self.planes())
        for i, m in enumerate(self.model):
            assert (np.linalg.norm(S[i] - m.S, axis=2) <= m.eS + 1e-30).all(), (i, np.linalg.norm(S[i] - m.S, axis=2).max(), m.eS.max())
            assert counts[i] == len(m.waiting)
            seen = np.concatenate([m.inputs] + [w[6][None] for w in m.waiting])
            assert np.array_equal(inputs[i, :len(seen)], seen)
            for j, (k, ek, dv, ed, a, ea, _) in enumerate(m.waiting):
                k, ek = k[::c.vh // c.kh], ek[::c.vh // c.kh]
                assert (np.linalg.norm(keys[i, j] - k, axis=1) <= ek).all()
                assert (np.abs(updates[i, j] - dv) <= ed + 1e-30).all()
                assert (np.abs(decays[i, j] - a) <= ea).all()

    def close(self):
        self.cache.free()


SHAPES = [(2, 4, 64, 4), (1, 1, 128, 4), (3, 9, 64, 2), (2, 2, 128, 8), (4, 8, 128, 3)]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("kh,vh,d,taps", SHAPES)
def test_decode_steps_and_drafts(ctx, kh, vh, d, taps, dtype):
    """Steps of up to six rows; every number of them may stand, and sequences begin and go on in any slot."""
    run = Run(ctx, vh * d + taps, kh, vh, d, taps, 6, 5, 24, dtype)
    run.step([1, 6, 3], [4, 0, 2], [-1, -1, -1])
    run.check_storage()
    run.step([4, 1, 0, 5], [2, 4, 1, 0], [0, 1, 0, 6])
    run.check_storage()
    run.step([2, 2, 1, 6], [0, 4, 3, 2], [2, 99, -1, 1], pad=4)
    run.check_storage()
    run.step([1, 1], [2, 0], None, pad=3, extra=2)
    run.check_storage()
    run.step([1, 1, 1], [2, 0, 3], [1, 0, 1])
    run.check_storage()
    run.close()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("kh,vh,d,taps", SHAPES)
def test_prompts(ctx, kh, vh, d, taps, dtype):
    """Prompts of any length beside decode steps, after pending rows and before drafts."""
    run = Run(ctx, 31 + vh * d + taps, kh, vh, d, taps, 4, 4, 420, dtype)
    run.step([64, 17, 4, 130], [0, 1, 2, 3], [-1, -1, -1, -1])
    run.check_storage()
    run.step([3, 16, 65, 1], [1, 0, 2, 3], [0, 0, 2, 0])
    run.check_storage()
    run.step([18, 128, 20], [3, 1, 2], [1, 3, 0], pad=4)
    run.check_storage()
    run.step([200, 5], [0, 1], None, pad=1, extra=3)
    run.check_storage()
    run.close()


@pytest.mark.parametrize("pending", [0, 16])
def test_no_and_most_pending_rows(ctx, pending):
    run = Run(ctx, 7 + pending, 2, 4, 64, 4, pending, 3, 60)
    run.step([1, 16, 2], [0, 1, 2], [-1, -1, -1])
    run.check_storage()
    run.step([16, 15, 17], [2, 1, 0], [1, 9, 1])
    run.check_storage()
    run.step([1, 1, 1], [2, 1, 0], None)
    run.check_storage()
    run.close()


def test_workgroups_of_more_rows(ctx):
    """Enough heads for the kernel with 32 rows of S a workgroup."""
    run = Run(ctx, 3, 8, 32, 128, 4, 3, 5, 20)
    run.step([1, 3, 2, 1, 1], [0, 1, 2, 3, 4], [-1] * 5)
    run.check_storage()
    run.step([1, 3, 2, 4, 1], [4, 1, 2, 3, 0], [1, 2, 0, 0, 1])
    run.check_storage()
    run.close()


@pytest.mark.parametrize("lengths", [[70], [17, 300], [1, 64, 129]])
def test_chunks_equal_rows_one_by_one(ctx, lengths):
    """The same rows at once and one a call: the states that are left agree as closely as either does with 64 bits."""
    a, b = (Run(ctx, 11, 2, 4, 128, 4, 0, len(lengths), 512) for _ in range(2))
    slots = list(range(len(lengths)))
    a.step(lengths, slots, [-1] * len(lengths))
    a.check_storage()
    rng_state = np.random.default_rng(11)
    Layer(2, 4, 128, 4, 0, rng_state)
    # the same inputs, row by row
    c, rows = a.layer, sum(lengths)
    x, alpha, beta = (rng_state.standard_normal((rows, w)).astype(np.float32) for w in (c.channels, c.vh, c.vh))
    starts = np.concatenate([[0], np.cumsum(lengths)])
    up = lambda t: torch.from_numpy(np.ascontiguousarray(t)).cuda()
    one, out = up(np.array([0, 1], dtype=np.int32)), torch.empty(1, c.vh * c.d, device="cuda")
    for s, n in enumerate(lengths):
        slot = up(np.array([s], dtype=np.int32))
        for i in range(n):
            dev = [up(t[starts[s] + i]) for t in (x, alpha, beta)]
            batch = B.GdnBatch(1, 1, 1, one.data_ptr(), slot.data_ptr(), None)
            torch.cuda.synchronize()
            b.cache.run(1, batch, *(t.data_ptr() for t in dev), *(w.data_ptr() for w in b.weights), out.data_ptr())
            b.ctx.synchronize()
    b.model = a.model
    b.check_storage()
    a.close(), b.close()


def test_far_and_equal_keys(ctx):
    """Keys that are all the same (the triangle's worst), decays down to nothing, and none at all."""
    run = Run(ctx, 13, 1, 3, 64, 4, 0, 1, 200)
    c = run.layer
    c.ssm_a[:] = [-60.0, -1e-6, -1e30]
    run.weights[1].copy_(torch.from_numpy(c.ssm_a))
    rng = np.random.default_rng(1)
    real = run.rng.standard_normal
    same = rng.standard_normal(c.channels)
    # inputs of the keys' channels that repeat from row to row
    def draw(shape):
        x = real(shape)
        if shape[1] == c.channels:
            x[:, :2 * c.d] = same[:2 * c.d]
        return x
    class Draw:
        standard_normal = staticmethod(draw)
    run.rng = Draw
    run.step([150], [0], [-1])
    run.check_storage()
    run.step([16], [0], [0])
    run.check_storage()
    run.close()


@pytest.mark.parametrize("d", [64, 128])
def test_queries_that_are_the_keys(ctx, d):
    """A chunk's rows ask for what they have just stored: an error of any operand's lower half shows in the outputs."""
    for seed in range(4):
        run = Run(ctx, 40 + seed, 2, 4, d, 4, 0, 2, 400)
        c = run.layer
        n = c.kh * d
        c.conv[n:2 * n] = c.conv[:n]
        run.weights[0].copy_(torch.from_numpy(c.conv))
        real = run.rng.standard_normal

        class Draw:
            @staticmethod
            def standard_normal(shape):
                x = real(shape)
                if shape[1] == c.channels:
                    x[:, n:2 * n] = x[:, :n]
                return x

        run.rng = Draw
        run.step([200, 70], [0, 1], [-1, -1])
        run.step([65, 130], [0, 1], [0, 0])
        run.check_storage()
        run.close()


def test_one_sequence_that_may_have_many_rows(ctx):
    """Alone and without pending rows a sequence goes through chunks however few its rows are."""
    run = Run(ctx, 53, 2, 4, 64, 4, 0, 2, 100)
    c = run.layer
    for count, standing in ((1, -1), (2, 0), (40, 0), (5, 0), (1, 0), (16, -1)):
        x, alpha, beta = (run.rng.standard_normal((40, w)).astype(np.float32) for w in (c.channels, c.vh, c.vh))
        dev = [torch.from_numpy(a).cuda() for a in (x, alpha, beta)]
        out = torch.full((40, c.vh * c.d), 9.0, device="cuda")
        numbers = [torch.tensor(a, dtype=torch.int32, device="cuda") for a in ([0, count], [1], [standing])]
        torch.cuda.synchronize()
        run.cache.run(1, B.GdnBatch(1, 40, 40, *(a.data_ptr() for a in numbers)), *(a.data_ptr() for a in dev), *(w.data_ptr() for w in run.weights), out.data_ptr())
        ctx.synchronize()
        want, bound = c.run(run.model[1], standing, *(a[:count].astype(np.float64) for a in (x, alpha, beta)), chunked=True)
        got = out.double().cpu().numpy()
        assert (np.abs(got[:count].reshape(want.shape) - want) <= bound + 2.0 ** -24 * np.abs(want)).all() and (got[count:] == 9.0).all()
        run.check_storage()
    run.close()


def test_slots_that_are_not_there(ctx):
    """Rows of a slot outside the cache, and row starts outside the arrays, reach nothing else."""
    run = Run(ctx, 17, 2, 4, 64, 4, 3, 2, 40)
    run.step([2, 20], [0, 1], [-1, -1])
    before = run.storage.clone()
    c = run.layer
    x, alpha, beta = (torch.randn(8, w, device="cuda") for w in (c.channels, c.vh, c.vh))
    out = torch.full((8, c.vh * c.d), 9.0, device="cuda")
    for starts, slots in (([0, 3, 8], [-1, 2]), ([0, -5, -9], [0, 1]), ([100, 200, 300], [0, 1]), ([4, 2, 0], [0, 1])):
        dev = [torch.tensor(t, dtype=torch.int32, device="cuda") for t in (starts, slots)]
        batch = B.GdnBatch(2, 8, 8, dev[0].data_ptr(), dev[1].data_ptr(), None)
        torch.cuda.synchronize()
        run.cache.run(1, batch, x.data_ptr(), alpha.data_ptr(), beta.data_ptr(), *(w.data_ptr() for w in run.weights), out.data_ptr())
        run.ctx.synchronize()
        assert (out == 9.0).all() and torch.equal(run.storage, before)
    run.check_storage()
    run.close()


def test_copies_of_slots(ctx):
    run = Run(ctx, 19, 2, 4, 64, 4, 3, 4, 40)
    run.step([3, 20], [0, 1], [-1, -1])
    run.cache.copy_slots([0, 1], [3, 2])
    ctx.synchronize()
    planes = run.planes()
    for plane in planes:
        assert np.array_equal(plane[0], plane[3]) and np.array_equal(plane[1], plane[2])
    import copy
    run.model[3], run.model[2] = copy.deepcopy(run.model[0]), copy.deepcopy(run.model[1])
    # a fork and its origin go on with different verdicts
    run.step([1, 2, 1], [0, 3, 2], [1, 3, 0])
    run.check_storage()
    for bad in (([0], [0]), ([0], [4]), ([-1], [0]), ([0, 1], [2, 2]), ([0, 1], [1, 2])):
        with pytest.raises(B.BackendError) as e:
            run.cache.copy_slots(*bad)
        assert e.value.code == B.INVALID
    run.close()


@pytest.mark.parametrize("most", [4, 40])
def test_captured_and_replayed(most):
    """One graph serves steps whose rows, slots and verdicts differ: few rows only, and the launches for many."""
    ctx = B.Context(0)  # a context holds one graph
    run = Run(ctx, 23, 2, 4, 128, 4, 4, 3, 80)
    c = run.layer
    dev = {k: torch.zeros(s, dtype=t, device="cuda") for k, s, t in
           (("x", (80, c.channels), torch.float32), ("alpha", (80, c.vh), torch.float32), ("beta", (80, c.vh), torch.float32),
            ("out", (80, c.vh * c.d), torch.float32), ("starts", (4,), torch.int32), ("slots", (3,), torch.int32), ("standing", (3,), torch.int32))}
    batch = B.GdnBatch(3, 80, most, dev["starts"].data_ptr(), dev["slots"].data_ptr(), dev["standing"].data_ptr())
    torch.cuda.synchronize()
    ctx.capture_begin()
    run.cache.run(1, batch, dev["x"].data_ptr(), dev["alpha"].data_ptr(), dev["beta"].data_ptr(), *(w.data_ptr() for w in run.weights), dev["out"].data_ptr())
    ctx.capture_end()
    for counts, slots, standing in (([most, 2, 1], [0, 1, 2], [-1, -1, -1]), ([1, 4, most], [2, 0, 1], [1, 2, 0]), ([2, most, 3], [1, 2, 0], [1, 9, 4])):
        rows = sum(counts)
        new = {k: run.rng.standard_normal(dev[k].shape).astype(np.float32) for k in ("x", "alpha", "beta")}
        new["starts"], new["slots"], new["standing"] = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32), np.array(slots, np.int32), np.array(standing, np.int32)
        for k, v in new.items():
            dev[k].copy_(torch.from_numpy(v))
        torch.cuda.synchronize()
        ctx.graph_launch()
        ctx.synchronize()
        got, at = dev["out"].double().cpu().numpy(), 0
        for s, n in enumerate(counts):
            part = [new[k][at:at + n].astype(np.float64) for k in ("x", "alpha", "beta")]
            want, bound = c.run(run.model[slots[s]], standing[s], *part)
            assert (np.abs(got[at:at + n].reshape(want.shape) - want) <= bound + 2.0 ** -24 * np.abs(want) + 1e-37).all()
            at += n
        run.check_storage()
    run.close()
    ctx.close()


def test_created_cleared(ctx):
    """A cache with storage of its own begins with empty states."""
    rng = np.random.default_rng(29)
    layer, slot = Layer(2, 2, 64, 4, 2, rng), None
    cache = B.GdnCache(ctx, 1, 2, 2, 2, 64, 4, 2, 8)
    x, alpha, beta = (rng.standard_normal((2, w)).astype(np.float32) for w in (layer.channels, 2, 2))
    up = lambda t: torch.from_numpy(np.ascontiguousarray(t)).cuda()
    dev, weights = [up(t) for t in (x, alpha, beta)], [up(t) for t in (layer.conv, layer.ssm_a, layer.ssm_dt)]
    out, starts, slots = torch.empty(2, 128, device="cuda"), up(np.array([0, 2], np.int32)), up(np.array([1], np.int32))
    torch.cuda.synchronize()
    cache.run(0, B.GdnBatch(1, 2, 2, starts.data_ptr(), slots.data_ptr()), *(t.data_ptr() for t in dev), *(t.data_ptr() for t in weights), out.data_ptr())
    ctx.synchronize()
    slot = Slot(layer)
    want, bound = layer.run(slot, None, *(t.astype(np.float64) for t in (x, alpha, beta)))
    assert (np.abs(out.double().cpu().numpy().reshape(want.shape) - want) <= bound + 2.0 ** -24 * np.abs(want)).all()
    cache.free()
