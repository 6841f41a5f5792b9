"""The gated delta rule over rows in 64 bits, for numbers of unlike magnitude: what a row's result may be off is held
against what its text has in it so far, with the decays since, not against what comes after it or is forgotten."""

import numpy as np

from gdn_model import U, Layer

# Chunks hold values (times beta), updates and states as pairs of fp16 against the largest R of a value dim in the chunk,
# its state before the chunk included, and the triangle's numbers, keys and weights against 1 (2^15, the weights 2^18).
# What is left of a number in the lower half is off by 2^-25 of 2^14 of its largest, 2^-39, or 2^-40 of 1.  An update is
# a sum of up to 64 values with numbers of the triangle, each at most 1, and of 128 of the state's:
#   64 (2^-39 + 2^-40) + 128 2^-40 < 2^-32.4 ... of R, and of the update's own half 2^-39 sqrt(head) of R: 2^-31 in all;
# an output adds 64 updates (of at most 13 R) with weights of at most 1 / 8: 64 13 2^-39 / 8 + 64 2 2^-43 < 2^-32.
UPDATE, OUTPUT = 2.0 ** -31, 2.0 ** -32
# A row below this of R goes by itself, in fp32: then nothing of R is in its error.  (The border is at 2^-20, with what
# the logarithms of decays and powers of two round.)
ALONE = 2.0 ** -21.5


class UnlikeLayer(Layer):
    def run(self, slot, standing, x, alpha, beta, chunked=None):
        d = self.d
        if standing is not None and standing < 0:
            slot.__init__(self)
        assert not slot.waiting and len(x) > self.pending  # of rows that stand at once
        chunked = len(x) > 16 if chunked is None else chunked
        S, eS, inputs = slot.S, slot.eS, slot.inputs
        rows = []
        for i in range(len(x)):
            seen = np.concatenate([inputs, x[i][None]])
            rows.append(self.row(seen, alpha[i], beta[i]))
            inputs = seen[1:]
        out, bound, recent = [], [], np.zeros((self.vh, d))
        for i, (q, eq, k, ek, v, ev, a, ea, b, eb, key) in enumerate(rows):
            if chunked and i % 64 == 0:
                so_far, held = np.abs(S).max(axis=2), 0.0
                most = np.max([so_far] + [r[8][:, None] * np.abs(r[4]) for r in rows[i:i + 64]], axis=0)
            size = np.linalg.norm(S, axis=2)
            dv = b[:, None] * (v - a[:, None] * np.einsum("hrc,hc->hr", S, k))
            n = d / 8 + 8 if not chunked else d + 16
            among = np.zeros((self.vh, d)) if not chunked else 4 * 64 * U * recent
            left = 0.0  # what the chunk's halves leave in S so far
            if chunked:
                so_far = np.maximum(a[:, None] * so_far, b[:, None] * np.abs(v))
                held, alone = a[:, None] * held + UPDATE * most, so_far < ALONE * most
                left = np.where(alone, 0.0, held)
            ed = b[:, None] * (ev + a[:, None] * size * (ek[:, None] + n * U) + ea[:, None] * size + among) + \
                np.abs(dv) * (4 * U) + (np.abs(v) + size) * eb[:, None]
            S = a[:, None, None] * S + dv[:, :, None] * k[:, None, :]
            local = ed + ea[:, None] * size + np.abs(dv) * ek[:, None] + 3 * U * (np.linalg.norm(S, axis=2) + np.abs(dv)) + among
            eS = a[:, None] * eS + local
            recent = a[:, None] * recent + np.abs(dv)
            size, length = np.linalg.norm(S, axis=2), np.linalg.norm(q, axis=1)[:, None]
            out.append(np.einsum("hrc,hc->hr", S, q))
            own = (eS + left) * length + size * (eq[:, None] + (n + 4) * U * length) + among * length
            bound.append(own + np.where(alone, 0.0, OUTPUT * most) if chunked else own)
            if chunked and (i % 64 == 63 or i + 1 == len(x)):
                eS = eS + left
        slot.S, slot.eS, slot.inputs = S, eS, inputs
        return np.array(out), np.array(bound)
