"""One long row of the paged attention whose pieces, and whose batches of 256 of them, all differ: inputs, the sum in 64
bits, the bound of an f32 kernel's error, and what merges that go wrong would give."""
import numpy as np

import pages_ref as R
import steps_ref as S

SLOTS, PAGE = 262144 + 5, 1024
BATCH = 256  # pieces that the merge takes at once


class LongRow:
    """A row of SLOTS slots of one kv head, two q heads. Head h's q is element h alone, so its scores are element h of
    K: a wave of 0 to 1 along the row, and two peaks, 5 and 8 high (one in the first batch of pieces, one in the last; the
    heads have them the other way round). V is the same for 128 slots each, and differs from block to block."""

    def __init__(self, rng, t, hd):
        self.t, self.hd, n = t, hd, SLOTS
        j = np.arange(n)
        score = 0.5 + 0.5 * np.sin(j[None] / 8000.0 + np.array([[0.0], [2.0]]))
        score[0, [20000, n - 150]] = 5.0, 8.0
        score[1, [20000, n - 150]] = 8.0, 5.0
        v = rng.standard_normal((n // 128 + 1, hd))[j // 128]
        self.pages = -(-n // PAGE)
        units = self.pages * PAGE // 32
        nb = R.nb(hd)
        slot, d = np.arange(32)[:, None], np.arange(hd)[None]
        wide = {w: np.zeros((units * 32, x), np.float64) for w, x in (("k", 2), ("v", hd))}
        wide["k"][:n], wide["v"][:n] = score.T, v
        self.bytes, self.held = {}, {}
        for w, x in wide.items():
            at = R.place(t, w, hd, slot, d[:, :x.shape[1]])
            x = x.reshape(units, 32, -1)
            if t == R.F16:
                unit = np.zeros((units, nb * 1024), np.float16)
                unit[:, at] = x
                self.held[w] = unit[:, at].astype(np.float64)
            else:
                step = np.float16(8 / 127 if w == "k" else 0.04)
                values = np.zeros((units, nb * 1024), np.int8)
                values[:, at] = np.clip(np.rint(x / np.float64(step)), -127, 127)
                self.held[w] = values[:, at] * np.float64(step)
                scales = np.full((units, nb * 32), step).view(np.uint8).reshape(units, -1)
                unit = np.concatenate([values.view(np.uint8), scales], 1)
            self.held[w] = self.held[w].reshape(units * 32, -1)[:n]
            self.bytes[w] = unit.view(np.uint8).reshape(self.pages, -1)
        self.q = np.zeros((2, hd), np.float32)
        self.q[0, 0] = self.q[1, 1] = 1.0

    def share(self):
        """Units of a piece: the line's units over the workgroups that run at once (8193 or more of them: all; a unit of
        one block of 32 elements leaves a CU room for four workgroups, up to six blocks for two), in whole rounds of four
        waves."""
        units, workgroups = -(-SLOTS // 32), 256 * (4 if R.nb(self.hd) == 1 else 2)
        return -(-units // workgroups // 4) * 4

    def parts(self):
        """The pieces' greatest scores, and sums and outputs relative to them: (pieces, heads), the same, (pieces, heads, hd)."""
        step, m, l, o = self.share() * 32, [], [], []
        for j in range(0, SLOTS, step):
            s, v = self.held["k"][j:j + step], self.held["v"][j:j + step]
            top = s.max(0)
            e = np.exp(s - top)
            m.append(top)
            l.append(e.sum(0))
            o.append(e.T @ v)
        return np.array(m), np.array(l), np.array(o)

    def want(self, m, l, o):
        """out (heads, hd), and the bound of the error of an f32 kernel, in units of F32 times the weighted mean of |v|.
        Of each weight: the score (three roundings of |s| <= 8, in nats 24), and then at most ten scalings (the running
        maximum of a wave's at most five units, the waves', the pieces' and the batches' joins), each the rounding of an
        argument of at most 12 (12 ln 2 < 9), of the exponential (2) and of the product (1): 24 + 120 = 144, as much
        again for the sum it is divided by. The outputs' sums: 32 products in each of five units, the weights' two parts
        (4), four waves, a rounding for each piece; the weights' sums: eight and three a unit and lane, 2 + 4 + 6 + 4 + 3
        joins, under 80; the quotient."""
        f = np.exp(m - m.max(0))
        total = (f * l).sum(0)
        out = (f[..., None] * o).sum(0) / total[:, None]
        s = self.held["k"]
        w = np.exp(s - s.max(0))
        size = (w / w.sum(0)).T @ np.abs(self.held["v"])
        return out, (2 * 144 + 160 + 8 + len(m) + 80 + 1) * S.F32 * size

    @staticmethod
    def wrong(m, l, o):
        """What merges give that lose a piece, take another's values, or do not scale from batch to batch."""
        def join(m, l, o, keep=True, ml=None):
            f = np.exp(m - m.max(0))
            if not keep:  # each batch relative to its own maximum
                f = np.concatenate([np.exp(m[k:k + BATCH] - m[k:k + BATCH].max(0)) for k in range(0, len(m), BATCH)])
            return (f[..., None] * o).sum(0) / (f * (l if ml is None else ml)).sum(0)[:, None]
        again = np.arange(len(m)) % BATCH
        yield "the first batch alone", join(m[:BATCH], l[:BATCH], o[:BATCH])
        yield "the last batch alone", join(m[len(m) // BATCH * BATCH:], l[len(m) // BATCH * BATCH:], o[len(m) // BATCH * BATCH:])
        yield "the first batch's values", join(m, l, o[again])
        yield "the first batch's maxima and sums", join(m[again], l[again], o)
        yield "the first batch's sums", join(m, l, o, ml=l[again])
        yield "values of the next piece", join(m, l, np.roll(o, -1, 0))
        yield "maxima and sums of the next piece", join(np.roll(m, -1, 0), np.roll(l, -1, 0), o)
        yield "no scaling between batches", join(m, l, o, keep=False)
        yield "the greatest score of the first batch for all", join(np.maximum(m, m[:BATCH].max(0)), l, o)
        for k in (0, 1, BATCH - 1, BATCH, BATCH + 1, len(m) // 2, len(m) - 2):
            keep = np.arange(len(m)) != k
            yield f"piece {k} lost", join(m[keep], l[keep], o[keep])
            yield f"piece {k} twice", join(*(np.concatenate([x, x[k:k + 1]]) for x in (m, l, o)))
        at = np.arange(len(m))
        at[[10, 300]] = 300, 10
        yield "values of two pieces exchanged", join(m, l, o[at])
