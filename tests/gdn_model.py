"""The gated delta rule over rows in 64 bits, row by row, with what fp32 arithmetic may be off."""

import numpy as np

U = 2.0 ** -24


def sigmoid(x):
    return 1.0 / (1.0 + np.exp(-x))


class Slot:
    """One sequence's state; errors are bounds of what a kernel in fp32 may have differently."""

    def __init__(self, layer):
        c = layer
        self.layer = c
        self.S, self.eS = np.zeros((c.vh, c.d, c.d)), np.zeros((c.vh, c.d))  # a row's error as a length
        self.inputs, self.waiting = np.zeros((c.taps - 1, c.channels)), []


class Layer:
    """Shape and weights of one layer; run() takes one sequence's rows."""

    def __init__(self, kh, vh, d, taps, pending, rng, eps=1e-6):
        self.kh, self.vh, self.d, self.taps, self.pending, self.eps = kh, vh, d, taps, pending, float(np.float32(eps))
        self.channels = (2 * kh + vh) * d
        f = lambda a: a.astype(np.float32)
        self.conv = f(0.3 * rng.standard_normal((self.channels, taps)))
        self.ssm_a, self.ssm_dt = f(-np.exp(rng.standard_normal(vh) - 1.0)), f(rng.standard_normal(vh))

    def row(self, seen, alpha, beta):
        """q, k, v, a, b of one row from the inputs seen [taps][channels], and their errors (of q, k: lengths)."""
        kh, vh, d = self.kh, self.vh, self.d
        w = self.conv.astype(np.float64)
        u, size = (w * seen.T).sum(axis=1), (np.abs(w) * np.abs(seen.T)).sum(axis=1)
        # a sum of `taps` fused products; silu: exp (2 steps), an addition, a division, slope at most 1.1
        y, e = u * sigmoid(u), 1.1 * self.taps * U * size
        e = e + 6 * U * np.abs(y) + 1e-37
        out = []
        for part, n in ((slice(0, kh * d), kh), (slice(kh * d, 2 * kh * d), kh)):
            t, et = y[part].reshape(n, d), np.linalg.norm(e[part].reshape(n, d), axis=1)
            length = np.maximum(np.linalg.norm(t, axis=1), self.eps)
            # the length is as far off as the vector; d squares, a root, a division, a product
            out.append((t / length[:, None], 2 * et / length + (d / 64 + 14) * U))
        (q, eq), (k, ek) = out
        q, eq = q / np.sqrt(d), (eq + 2 * U) / np.sqrt(d)
        x = alpha + self.ssm_dt.astype(np.float64)
        soft = np.maximum(x, 0) + np.log1p(np.exp(-np.abs(x)))
        g = self.ssm_a.astype(np.float64) * soft
        # the sum alpha + dt (slope at most 1), log1p, exp: a few steps of g's parts; then exp
        eg = np.abs(self.ssm_a) * U * (np.abs(x) + 10 * soft + 4)
        a = np.exp(g)
        rep = self.vh // self.kh
        spread = lambda t: np.repeat(t, rep, axis=0)
        v, ev = y[2 * kh * d:].reshape(vh, d), e[2 * kh * d:].reshape(vh, d)
        return spread(q), spread(eq), spread(k), spread(ek), v, ev, a, a * (eg + 4 * U), sigmoid(beta), 6 * U * sigmoid(beta), k

    def run(self, slot, standing, x, alpha, beta, chunked=None):
        """Outputs [rows][vh][d] and their bounds.  standing: None: all, -1: anew."""
        d = self.d
        if standing is not None and standing < 0:
            slot.__init__(self)
        stands = len(slot.waiting) if standing is None else min(max(standing, 0), len(slot.waiting))
        for k, ek, dv, ed, a, ea, seen in slot.waiting[:stands]:
            size = np.linalg.norm(slot.S, axis=2)
            slot.eS = a[:, None] * slot.eS + ea[:, None] * size + np.abs(dv) * ek[:, None] + ed + 3 * U * (size + np.abs(dv))
            slot.S = a[:, None, None] * slot.S + dv[:, :, None] * k[:, None, :]
            slot.inputs = np.concatenate([slot.inputs[1:], seen[None]])
        slot.waiting = []
        waits = len(x) <= self.pending
        chunked = len(x) > 16 if chunked is None else chunked
        S, eS, inputs = slot.S, slot.eS, slot.inputs
        out, bound, waiting, recent = [], [], [], np.zeros((self.vh, d))
        rows, least = [], np.zeros((len(x), self.vh, d))
        for i in range(len(x)):
            seen = np.concatenate([inputs, x[i][None]])
            rows.append(self.row(seen, alpha[i], beta[i]))
            inputs = seen[1:]
        if chunked and len(x):
            # a chunk's values and updates are pairs of fp16 of at most 2^10, their columns' largest: the lower half's
            # smallest step is 2^-24, so that each is off by 2^-25 of 2^10 at least, 2^-35 of the largest
            T, values, updates = S, [], []
            for q, eq, k, ek, v, ev, a, ea, b, eb, key in rows:
                dv = b[:, None] * (v - a[:, None] * np.einsum("hrc,hc->hr", T, k))
                T = a[:, None, None] * T + dv[:, :, None] * k[:, None, :]
                values.append(np.abs(v))
                updates.append(np.abs(dv))
            for i in range(0, len(x), 64):
                least[i:i + 64] = 2.0 ** -35 * (np.max(values[i:i + 64], axis=0) + np.max(updates[i:i + 64], axis=0))
        inputs = slot.inputs
        for i in range(len(x)):
            seen = np.concatenate([inputs, x[i][None]])
            q, eq, k, ek, v, ev, a, ea, b, eb, key = rows[i]
            size = np.linalg.norm(S, axis=2)
            asked = a[:, None] * np.einsum("hrc,hc->hr", S, k)
            dv = b[:, None] * (v - asked)
            # sums of a row of S with k or q: d / 8 products a lane and three additions; in chunks all d of them, 64
            # rows' updates (each at most its own size) beside them, through the triangle (64 more) and back
            n = d / 8 + 8 if not chunked else d + 16
            among = np.zeros((self.vh, d)) if not chunked else 4 * 64 * U * recent
            ed = b[:, None] * (ev + a[:, None] * size * (ek[:, None] + n * U) + ea[:, None] * size + among) + least[i] + \
                np.abs(dv) * (4 * U) + np.abs(v - asked) * eb[:, None]
            # an error of S goes through a (1 - b k k^T), which makes nothing larger
            S = a[:, None, None] * S + dv[:, :, None] * k[:, None, :]
            local = ed + ea[:, None] * size + np.abs(dv) * ek[:, None] + 3 * U * (np.linalg.norm(S, axis=2) + np.abs(dv)) + among
            eS = a[:, None] * eS + local
            recent = a[:, None] * recent + np.abs(dv)
            size = np.linalg.norm(S, axis=2)
            length = np.linalg.norm(q, axis=1)[:, None]
            out.append(np.einsum("hrc,hc->hr", S, q))
            bound.append(eS * length + size * (eq[:, None] + (n + 4) * U * length) + among * length)
            inputs = seen[1:]
            # what is kept of an update is as far off as the state that it asks, and its own arithmetic
            waiting.append((k, ek, dv, ed + b[:, None] * (eS + 0), a, ea, x[i]))
        if waits:
            slot.waiting = waiting
        else:
            slot.S, slot.eS, slot.inputs = S, eS, inputs
        return np.array(out), np.array(bound)
