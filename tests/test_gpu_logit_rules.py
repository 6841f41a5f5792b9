"""Rules on logits against the definition in 64 bits."""

import numpy as np
import pytest
import torch

from fortai_amd import backend as B

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


class Case:
    """A ragged batch with everything that rules can have; `has` names what is given to the call."""

    def __init__(self, seed, counts, vocab, lengths, window, dtype, has="pthbm", pitch=None):
        rng = np.random.default_rng(seed)
        self.vocab, self.window, self.dtype, self.has = vocab, window, dtype, has
        n, self.rows = len(counts), sum(counts)
        self.starts = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
        self.lengths, self.pitch = np.array(lengths, dtype=np.int32), max(lengths) + 2
        # few different tokens, so that many repeat; some are no tokens at all
        draw = lambda *shape: rng.choice(np.concatenate([rng.integers(0, vocab, 40), [0, vocab - 1, -1, vocab, 2 ** 40]]), shape)
        self.history, self.tokens = draw(n, self.pitch).astype(np.int64), draw(self.rows).astype(np.int64)
        self.penalties = np.stack([rng.uniform(1, 1.5, n), rng.uniform(0, 0.5, n), rng.uniform(0, 0.5, n)], axis=1).astype(np.float32)
        self.bias = rng.standard_normal((n, vocab)).astype(np.float32)
        self.words = -(-vocab // 32)
        self.masks = rng.integers(0, 2 ** 32, (3, self.words), dtype=np.uint32)
        self.mask_of = rng.integers(-1, 4, self.rows).astype(np.int32)  # 3: there is no such mask
        self.row_pitch = vocab if pitch is None else pitch
        self.logits = torch.from_numpy(4 * rng.standard_normal((self.rows, self.row_pitch)).astype(np.float32)).to(TYPES[dtype])

    def want(self):
        """Results, and what the fp32 operations may be off."""
        x = self.logits[:, :self.vocab].double().numpy().copy()
        size = np.abs(x)
        for s, (begin, end) in enumerate(zip(self.starts, self.starts[1:])):
            rep, freq, pres = self.penalties[s].astype(np.float64)
            for row in range(begin, end):
                text = list(self.history[s, :self.lengths[s]]) if "h" in self.has else []
                text += list(self.tokens[begin:row + 1]) if "t" in self.has else []
                text = np.array(text[-self.window:] if self.window else text, dtype=np.int64)
                text = text[(text >= 0) & (text < self.vocab)]
                n = np.bincount(text, minlength=self.vocab).astype(np.float64)
                if "p" in self.has:
                    y = np.where(x[row] > 0, x[row] / rep, x[row] * rep)
                    size[row] = np.where(n > 0, np.abs(y) + n * freq + pres, size[row])
                    x[row] = np.where(n > 0, y - n * freq - pres, x[row])
                if "b" in self.has:
                    x[row] += self.bias[s]
                    size[row] += np.abs(self.bias[s])
                if "m" in self.has and 0 <= self.mask_of[row] < 3:
                    bits = np.unpackbits(self.masks[self.mask_of[row]].view(np.uint8), bitorder="little")[:self.vocab]
                    x[row][bits == 0] = -np.inf
        return x, size

    def run(self, ctx, in_place=False):
        up = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()
        d = {k: up(getattr(self, k) if k != "masks" else self.masks.view(np.int32)) for k in
             ("starts", "lengths", "history", "tokens", "penalties", "bias", "masks", "mask_of")}
        logits = self.logits.cuda()
        out = logits if in_place else torch.full_like(logits, 7.0)
        ptr = lambda key, name: d[name].data_ptr() if key in self.has else None
        torch.cuda.synchronize()
        ctx.adjust_logits(logits.data_ptr(), self.vocab, out.data_ptr(), d["starts"].data_ptr(), len(self.lengths), self.rows,
                          dtype=self.dtype, tokens=ptr("t", "tokens"), history=ptr("h", "history"), history_pitch=self.pitch,
                          history_lengths=ptr("h", "lengths"), window=self.window, penalties=ptr("p", "penalties"),
                          bias=ptr("b", "bias"), bias_pitch=self.vocab, masks=ptr("m", "masks"), mask_count=3,
                          mask_pitch=self.words, mask_of=ptr("m", "mask_of"), pitch=self.row_pitch, out_pitch=self.row_pitch)
        ctx.synchronize()
        got = out.cpu()
        if not in_place:
            assert (got[:, self.vocab:] == 7.0).all()
        return got[:, :self.vocab].double().numpy()

    def check(self, got):
        want, size = self.want()
        masked = np.isinf(want)
        assert np.array_equal(masked, np.isinf(got)) and (got[masked] < 0).all()
        # five roundings to fp32 of parts no larger than `size`, then one to the type
        bound = 5 * 2.0 ** -24 * size + torch.finfo(TYPES[self.dtype]).eps / 2 * np.abs(want) + 2.0 ** -25
        assert (np.abs(got[~masked] - want[~masked]) <= bound[~masked]).all()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("window", [0, 1, 3, 70])
@pytest.mark.parametrize("vocab,pitch", [(1000, None), (97, None), (1028, 1028), (5001, 5003), (1, 4), (20480, None)])
def test_rules(ctx, vocab, pitch, window, dtype):
    case = Case(vocab + window, [1, 5, 0, 3], vocab, [0, 40, 7, 300], window, dtype, pitch=pitch)
    case.check(case.run(ctx))


@pytest.mark.parametrize("has", ["p", "pt", "ph", "b", "m", "bm", "", "pthb", "pthm"])
@pytest.mark.parametrize("vocab", [256, 333])
def test_parts_of_the_rules(ctx, has, vocab):
    case = Case(len(has), [4, 2], vocab, [20, 3], 10, "f32", has=has)
    got = case.run(ctx)
    case.check(got)
    if has == "":
        assert np.array_equal(got, case.logits.double().numpy())


def test_many_rows_of_a_sequence(ctx):
    """More rows than one workgroup takes: each starts with the text up to its own first row."""
    for window in (0, 9):
        case = Case(3, [41, 1, 30], 515, [11, 0, 64], window, "f32")
        case.check(case.run(ctx))


@pytest.mark.parametrize("window", [0, 5, 400])
def test_all_rows_in_one_of_many_sequences(ctx, window):
    """One workgroup then has them all, and looks up their tokens in several turns."""
    case = Case(4, [0] * 120 + [600] + [0] * 179, 300, [0] * 120 + [30] + [2] * 179, window, "f32")
    case.check(case.run(ctx))


def test_in_place_and_large(ctx):
    case = Case(4, [5] * 8, 70000, [500] * 8, 0, "f32")
    case.check(case.run(ctx, in_place=True))


def test_infinities_and_rows_of_nobody(ctx):
    case = Case(5, [2, 1], 64, [3, 3], 0, "f32", has="pth")
    case.logits[0, :4] = torch.tensor([float("inf"), -float("inf"), float("nan"), 0.0])
    case.history[0, :3] = [0, 1, 2]
    case.rows += 2  # behind the last sequence
    case.logits = torch.cat([case.logits, torch.ones(2, 64)])
    case.tokens = np.concatenate([case.tokens, [0, 0]])
    got = case.run(ctx)
    assert got[0, 0] == np.inf and got[0, 1] == -np.inf and np.isnan(got[0, 2])
    assert (got[3:] == 7.0).all()


def test_bad_numbers_reach_nothing_else(ctx):
    """Row starts and lengths outside their arrays are brought into range."""
    case = Case(6, [2, 2], 300, [5, 5], 0, "f32")
    case.starts = np.array([-4, 2, 900], dtype=np.int32)
    case.lengths = np.array([-3, 10 ** 9], dtype=np.int32)
    got = case.run(ctx)
    case.starts, case.lengths = np.array([0, 2, 4], dtype=np.int32), np.array([0, case.pitch], dtype=np.int32)
    case.check(got)


def test_captured_and_replayed():
    ctx = B.Context(0)  # a context holds one graph
    case = Case(7, [3, 2], 600, [9, 30], 0, "f32")
    up = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()
    d = {k: up(getattr(case, k) if k != "masks" else case.masks.view(np.int32)) for k in
         ("starts", "lengths", "history", "tokens", "penalties", "bias", "masks", "mask_of")}
    logits, out = case.logits.cuda(), torch.empty(case.rows, 600, device="cuda")
    torch.cuda.synchronize()
    ctx.capture_begin()
    ctx.adjust_logits(logits.data_ptr(), 600, out.data_ptr(), d["starts"].data_ptr(), 2, case.rows, tokens=d["tokens"].data_ptr(),
                      history=d["history"].data_ptr(), history_pitch=case.pitch, history_lengths=d["lengths"].data_ptr(),
                      penalties=d["penalties"].data_ptr(), bias=d["bias"].data_ptr(), bias_pitch=600, masks=d["masks"].data_ptr(),
                      mask_count=3, mask_of=d["mask_of"].data_ptr())
    ctx.capture_end()
    for step in range(3):
        case.lengths = np.array([9 + step, 30 - step], dtype=np.int32)
        case.logits = torch.randn(case.rows, 600)
        d["lengths"].copy_(torch.from_numpy(case.lengths))
        logits.copy_(case.logits)
        torch.cuda.synchronize()
        ctx.graph_launch()
        ctx.synchronize()
        case.check(out.double().cpu().numpy())
    ctx.close()
