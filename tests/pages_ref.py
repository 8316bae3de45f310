"""The paged cache and the verification of drafts, from their definitions (numpy, 64 bits)."""
import numpy as np

import steps_ref as S

F16, Q8_0 = 1, 8


def nb(hd):
    return (hd + 31) // 32


def unit_bytes(t, hd):
    return nb(hd) * (2048 if t == F16 else 1088)


def page_bytes(t, page, nkh, hd):
    return nkh * (page // 32) * unit_bytes(t, hd)


def place(t, which, hd, slot, d):
    """The index of (slot, element) among a unit's values."""
    b, g, e = d // 32, d % 32 // 8, d % 8
    if which == "k":
        h, tt, j = slot // 8, slot % 8 // 4, slot % 4
        if t == F16:
            return ((((tt * nb(hd) + b) * 4 + g) * 4 + h) * 4 + j) * 8 + e
        return ((((b * 4 + g) * 4 + h) * 4 + j) * 2 + tt) * 8 + e
    tt, r, g, e = d % 32 // 16, d % 16, slot // 8, slot % 8
    if t == F16:
        return (((b * 2 + tt) * 4 + g) * 16 + r) * 8 + e
    return (((b * 4 + g) * 16 + r) * 2 + tt) * 8 + e


def half_store(x):
    """f32 to f16 bits as the cache stores them: to nearest even; below the least normal half up, under 2^-25 to 0, NaN
    0x7C01 (include/vbs_half.h)."""
    x = np.asarray(x, np.float32)
    with np.errstate(all="ignore"):
        out = x.astype(np.float16).view(np.uint16).copy()
    mag = np.abs(x.astype(np.float64))
    sign = np.signbit(x).astype(np.uint16) << 15
    small = mag < 2.0 ** -14
    up = np.floor(np.where(small, mag, 0) * 2.0 ** 24 + 0.5).astype(np.uint16)
    up = np.where(mag < 2.0 ** -25, 0, up)
    out = np.where(small, sign | up.astype(np.uint16), out)
    return np.where(np.isnan(x), sign | np.uint16(0x7C01), out).astype(np.uint16)


def quantise(x):
    """x (..., hd) f32: int8 (..., nb * 32) and f16 scales (..., nb) of Q8_0."""
    hd = x.shape[-1]
    full = np.zeros(x.shape[:-1] + (nb(hd) * 32,))
    full[..., :hd] = x
    blocks = full.reshape(x.shape[:-1] + (nb(hd), 32))
    with np.errstate(all="ignore"):
        top = np.abs(blocks).max(-1)  # (NaN stays NaN)
        d = (top / 127).astype(np.float16)  # one rounding: top has 24 bits, 127 times a border 19
        d = np.where(np.isfinite(d), d, np.float16(np.nan))
        dd = d.astype(np.float64)[..., None]
        q = np.where(dd > 0, np.rint(blocks / np.where(dd > 0, dd, 1.0)), 0.0)
        q = np.clip(np.nan_to_num(q), -127, 127)
    return q.reshape(full.shape).astype(np.int8), d


def held(t, x):
    """The values that pages hold of rows x (..., hd), in f64."""
    if t == F16:
        return half_store(x).view(np.float16).astype(np.float64)
    q, d = quantise(x)
    v = q.reshape(d.shape + (32,)).astype(np.float64) * d.astype(np.float64)[..., None]
    v = np.where(np.isnan(d)[..., None], np.nan, v)
    return v.reshape(x.shape[:-1] + (-1,))[..., :x.shape[-1]]


class Pool:
    """A pool of one layer on the host, filled and read by the layout's definition."""

    def __init__(self, t, page, n_pages, nkh, hd, fill):
        self.t, self.page, self.nkh, self.hd = t, page, nkh, hd
        self.bytes = {w: fill(w).reshape(n_pages, nkh, page // 32, unit_bytes(t, hd)) for w in "kv"}

    def _values(self, w):
        n = nb(self.hd) * 1024
        part = self.bytes[w][..., :n * (2 if self.t == F16 else 1)]
        return part.view(np.uint16 if self.t == F16 else np.int8)

    def scales(self, w):
        return self.bytes[w][..., nb(self.hd) * 1024:].view(np.uint16)

    def put(self, w, page, slot, row):
        """row (nkh, hd) f32 into a slot of a page."""
        wide = np.zeros((self.nkh, nb(self.hd) * 32), np.float32)
        wide[:, :self.hd] = row
        at = place(self.t, w, self.hd, slot % 32, np.arange(nb(self.hd) * 32))
        if self.t == F16:
            self._values(w)[page, :, slot // 32, at] = half_store(wide).T
            return
        q, d = quantise(row)
        self._values(w)[page, :, slot // 32, at] = q.T
        for b in range(nb(self.hd)):
            self.scales(w)[page, :, slot // 32, b * 32 + slot % 32] = d[:, b].view(np.uint16)

    def get(self, w, page, slot):
        """The values of a slot, (nkh, hd) f64."""
        d = np.arange(self.hd)
        at = place(self.t, w, self.hd, slot % 32, d)
        x = self._values(w)[page, :, slot // 32][:, at]
        if self.t == F16:
            return x.view(np.float16).astype(np.float64)
        s = self.scales(w)[page, :, slot // 32][:, d // 32 * 32 + slot % 32].view(np.float16)
        return x.astype(np.float64) * s.astype(np.float64)

    def rows(self, w, pages, n):
        """Slots 0 .. n - 1 of a sequence of pages, (n, nkh, hd) f64."""
        return np.array([self.get(w, pages[j // self.page], j % self.page) for j in range(n)]).reshape(n, self.nkh, self.hd)


# The weights stand in two f16 parts, 2^14 high at the greatest: the lower part's last step is 2^-24, half of it 2^-39
# of the greatest weight, times a value of V at most (Q8_0: times 127 of the greatest scale).
FLOOR = 2.0 ** -39


def attend(q, k, v, scale, vmax=None):
    """q (heads, hd), k and v (slots, kv heads, hd), all f64: out (heads, hd) and the bound of an f32 kernel's error
    (steps_ref.attend's, with the weights' floor)."""
    n = k.shape[0]
    if n == 0:
        return np.zeros(q.shape), np.zeros(q.shape)
    with np.errstate(all="ignore"):
        out, w, tol, _ = S.attend(q[None], k, v, np.ones((1, n), bool), scale, n - 1)
        # (weights are at most 1; an infinity or a NaN of V stays with its own element, whose bound it makes infinite or NaN)
        size = np.where(np.isfinite(v), np.abs(v), 0.0).sum(0).max() if vmax is None else n * vmax
        tol = tol + FLOOR * size
    return out[0], tol[0]


def softmax(x, temp):
    x = np.asarray(x, np.float32).astype(np.float64)
    with np.errstate(all="ignore"):
        if temp == 0:
            key = np.where(np.isnan(x), -np.inf, x)
            p = np.zeros_like(x)
            if not np.isnan(x).all():
                seen = np.flatnonzero((key == key.max()) & ~np.isnan(x))
                p[seen[0]] = 1.0
            else:
                p[:] = np.nan
            return p
        e = np.exp((x - x.max()) / np.float64(np.float32(temp)))
        return e / e.sum()


def verify(logits, draft, drafted, u, temp):
    """One sequence: logits (n + 1, vocab), draft (n, vocab) or None, drafted (n,), u (n + 1,). Returns (accepted,
    tokens, margin): how far, relative to what is compared, every decision lay from its border."""
    n, vocab = len(drafted), logits.shape[1]
    tokens, margin, less = [-1] * (n + 1), 1.0, None
    k = 0
    with np.errstate(all="ignore"):
        while k < n and 0 <= drafted[k] < vocab:
            p, x = softmax(logits[k], temp), drafted[k]
            if draft is None or temp == 0:
                q = np.zeros(vocab)
                q[x] = 1.0
            else:
                q = softmax(draft[k], temp)
            a, b = float(u[k]) * q[x], p[x]
            if a != b and not np.isnan(a) and not np.isnan(b):
                margin = min(margin, abs(a - b) / max(a, b))
            if not a < b:
                less = np.where(p - q > 0, p - q, 0.0)
                break
            tokens[k] = int(x)
            k += 1
        r = less if less is not None and less.sum() > 0 else softmax(logits[k], temp)
        c = np.cumsum(r)
        if c[-1] > 0:
            want = max(float(u[n]), 0.0) * c[-1]
            over = np.flatnonzero(c > want)
            tokens[k] = int(over[0]) if len(over) else int(np.flatnonzero(r > 0)[-1])
            margin = min(margin, np.abs(c - want).min() / c[-1] if 0 < u[n] else 1.0)
    return k, tokens, margin
