"""The operators for steps of several tokens, from their formulas in 64 bits
(numpy), and how far an f32 kernel may be from them."""
import math

import numpy as np

# Products with f32 operands held as two f16 parts: each part rounds by half a step of 11
# bits, the low part being at most 2^-11 of the whole, so 2^-22 of an operand is lost.
SPLIT = 2.0 ** -22
F32 = 2.0 ** -24


def half(bits):
    return np.asarray(bits, np.uint16).view(np.float16).astype(np.float64)


def sees_chunk(n, past, prefix=0, docs=None):
    j, i = np.arange(past + n)[None], past + np.arange(n)[:, None]
    see = (j <= i) | (j < prefix)
    return see if docs is None else see & (docs[None] == docs[past:, None])


def sees_tree(n, past, mask):
    """mask: (n, ceil(n / 64)) uint64."""
    t = np.arange(n)
    bits = (mask[:, t // 64] >> (t % 64).astype(np.uint64)) & np.uint64(1)
    return np.concatenate([np.ones((n, past), bool), bits.astype(bool)], 1)


def attend(q, k, v, see, scale, past, cap=0.0, slopes=None):
    """q (n, heads, hd), k and v (slots, kv heads, hd) in float64, see (n, slots). Returns out (n, heads, hd), the
    weights (n, heads, slots), and bounds for the error of an f32 kernel on both.

    The bound: a score's dot of hd products, each of two operands (q off by SPLIT), loses at most (SPLIT +
    (2 hd + 4) F32) scale sum |q k| (hd products and sums, and twice that for the two parts; scale; bias), the
    cap's tanh 8 F32 of what it gives. e^s then is off by that much of itself plus 4 F32 for the exponential
    and what forms its argument loses, |s - m| F32 each; the maximum cancels. The weights e / sum e are off by
    twice the largest such error plus the rounding of as many sums as there are slots, and the outputs by the
    same with SPLIT for the weights' two parts and one more sum over the slots."""
    n, heads, hd = q.shape
    slots, kvh, _ = k.shape
    group = heads // kvh
    out, w = np.zeros((n, heads, hd)), np.zeros((n, heads, slots))
    tol, wtol = np.zeros((n, heads, hd)), np.zeros((n, heads, slots))
    at, j = past + np.arange(n)[:, None], np.arange(slots)[None]
    with np.errstate(all="ignore"):
        for h in range(heads):
            kk, vv = k[:, h // group], v[:, h // group]
            dot = np.stack([(q[i, h] * np.where(see[i][:, None], kk, 0.0)).sum(1) for i in range(n)])
            size = np.stack([np.abs(q[i, h] * np.where(see[i][:, None], kk, 0.0)).sum(1) for i in range(n)])
            s = dot * scale
            off = (SPLIT + (2 * hd + 4) * F32) * abs(scale) * size
            if cap:
                s = cap * np.tanh(s / cap)
                off = off + 8 * F32 * np.abs(s)
            if slopes is not None:
                far = slopes[h] * np.abs(at - j)
                s = s - far
                off = off + 2 * F32 * (np.abs(far) + np.abs(s))
            s = np.where(see, s, -np.inf)
            m = s.max(1, keepdims=True)
            top = np.where(m == -np.inf, 0.0, m)
            e = np.where(see, np.exp(s - top), 0.0)
            total = e.sum(1, keepdims=True)
            p = np.where(total == 0.0, 0.0, e / np.where(total == 0.0, 1.0, total))
            off = np.where(see & (s > -np.inf), off + (4 + 3 * np.minimum(np.abs(s - top), 110.0)) * F32, 0.0)
            worst = off.max(1, keepdims=True)
            for i in range(n):
                vi = np.where(see[i][:, None], vv, 0.0)
                if total[i] == 0.0:  # nothing seen, or scores of -inf alone: 0 by definition
                    continue
                out[i, h] = p[i] @ vi
                tol[i, h] = (p[i] @ np.abs(vi)) * (2 * worst[i] + SPLIT + (2 * slots + 8) * F32)
            w[:, h], wtol[:, h] = p, p * (2 * worst + (slots + 8) * F32) + 2.0 ** -100
    return out, w, tol + 2.0 ** -100, wtol


def mass(w, wtol, kvh):
    """Weights (n, heads, slots) summed per kv head, and the bound of the sums."""
    n, heads, slots = w.shape
    g = w.reshape(n, kvh, heads // kvh, slots)
    t = wtol.reshape(n, kvh, heads // kvh, slots).sum((0, 2)) + g.sum((0, 2)) * (n * heads // kvh + 2) * F32
    return g.sum((0, 2)), t


def rope_axes(x, pos, sections, theta):
    """x (n, heads, hd) float64 rotated at pos (axes, n)."""
    n, heads, hd = x.shape
    axis = np.repeat(np.arange(len(sections)), sections)
    freq = np.exp(-2.0 * np.arange(hd // 2) / hd * math.log(theta))
    angle = pos[axis].T.astype(np.float64) * freq  # (n, pairs)
    z = (x[..., 0::2] + 1j * x[..., 1::2]) * np.exp(1j * angle)[:, None]
    out = np.empty_like(x)
    out[..., 0::2], out[..., 1::2] = z.real, z.imag
    return out


def evict(weights, length, budget, first, last):
    """The slots kept of one head's weights, ascending."""
    key = [(-math.inf if math.isnan(x) else float(x)) for x in weights[:length]]
    open_ = list(range(first, length - last))
    # NaN is the least of all, below -inf
    best = sorted(open_, key=lambda j: (math.isnan(weights[j]), -key[j], j))[:budget - first - last]
    return np.array(sorted(list(range(first)) + best + list(range(length - last, length))), np.int64)
