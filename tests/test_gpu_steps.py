"""Steps of several tokens over the f16 KV cache (vbs_gfx950_rope_axes, _attention_tree, _attention_chunk and
_cache_evict) against their formulas in 64 bits (steps_ref.py), at the sizes, masks, strides and values where
they can go wrong. No counterpart in the reference (its loop takes one token at a time,
src/vbs_specializer.c:353-357): parity unpinned; the formulas are the ops' own (src/vbs_host_math.h:38-51, 150-209)
with the terms of include/vbs_gfx950.h."""
import ctypes as C
import math
import threading

import numpy as np
import pytest

import steps_ref as R
import vbs_gfx950 as V
from test_gpu_kernels import Mem, mem  # noqa: F401 (mem: fixture)

pytestmark = pytest.mark.gpu

NAN16, INF16 = 0x7E00, 0x7C00


def f16_bits(rng, *shape):
    return rng.standard_normal(shape).astype(np.float16).view(np.uint16)


def random_tree(rng, n):
    rows = []
    for i in range(n):
        parent = int(rng.integers(max(-1, i - 8), i)) if i else -1
        rows.append((rows[parent] if parent >= 0 else 0) | 1 << i)
    return pack(rows, n)


def pack(rows, n):
    words = (n + 63) // 64
    return np.array([[r >> 64 * w & (1 << 64) - 1 for w in range(words)] for r in rows], np.uint64).reshape(n, words)


class Step:
    """One attention call's inputs on the device: caches of `layers` layers with NaN rows behind the last slot in
    use, q and out with rows of their own stride, the pointers `shift` elements off their allocations."""

    def __init__(self, rng, mem, dev, n, past, nqh, nkh, hd, layer=1, spare=5, q_pad=0, out_pad=0, shift=0, size=2.0):
        self.__dict__.update(dev=dev, n=n, past=past, nqh=nqh, nkh=nkh, hd=hd, layer=layer, shift=shift)
        self.max_ctx, self.layers = past + n + spare, layer + 1
        self.kc = f16_bits(rng, self.layers, self.max_ctx, nkh, hd)
        self.vc = f16_bits(rng, self.layers, self.max_ctx, nkh, hd)
        self.kc[:, past + n:] = self.vc[:, past + n:] = NAN16
        self.qs, self.os = nqh * hd + q_pad, nqh * hd + out_pad
        self.q = (size * rng.standard_normal((n, self.qs))).astype(np.float32)
        self.scale = float(np.float32(1.0 / math.sqrt(hd)))
        self.mem = mem

    def up(self, a):
        flat = np.ascontiguousarray(a).reshape(-1)
        return self.mem.up(np.concatenate([np.zeros(self.shift, flat.dtype), flat])) + self.shift * flat.itemsize

    def load(self):
        self.pq, self.pk, self.pv = self.up(self.q), self.up(self.kc), self.up(self.vc)
        self.out0 = np.full((self.n + 1, self.os), 7.5, np.float32)  # a row behind the last
        self.po = self.up(self.out0)
        return self

    def tree(self, mask):
        self.load()
        self.dev.attention_tree(self.pq, self.qs, self.pk, self.pv, self.po, self.os, self.n, self.past,
                                self.mem.up(mask), self.layer, self.max_ctx, self.nqh, self.nkh, self.hd, self.scale)
        return self.got()

    def chunk(self, **terms):
        self.load()
        keep = {k: self.mem.up(v) if isinstance(v, np.ndarray) else v for k, v in terms.items()}
        self.pm = keep.get("mass")
        self.dev.attention_chunk(self.pq, self.qs, self.pk, self.pv, self.po, self.os, self.n, self.past, self.layer,
                                 self.max_ctx, self.nqh, self.nkh, self.hd, self.scale, **keep)
        return self.got()

    def got(self):
        o = self.dev.download(self.po, (self.n + 1, self.os), np.float32)
        w = self.nqh * self.hd
        # rows behind the last and the gaps between rows stay as they were
        assert np.array_equal(o[self.n], self.out0[self.n]) and np.array_equal(o[:, w:], self.out0[:, w:])
        return o[:self.n, :w].reshape(self.n, self.nqh, self.hd).astype(np.float64)

    def want(self, see, **terms):
        t = self.past + self.n
        q = self.q[:, :self.nqh * self.hd].reshape(self.n, self.nqh, self.hd).astype(np.float64)
        return R.attend(q, R.half(self.kc[self.layer, :t]), R.half(self.vc[self.layer, :t]), see, self.scale, self.past,
                        **terms)


def close(got, want, tol):
    bad = ~(np.abs(got - want) <= tol) & ~(np.isnan(want) & np.isnan(got)) & ~(np.isinf(want) & (got == want))
    assert not bad.any(), (int(bad.sum()), got[bad][:4], want[bad][:4], np.argwhere(bad)[:4])


# ---- the rotation --------------------------------------------------------------------------------

@pytest.mark.parametrize("n,nqh,nkh,hd,sections,far", [
    (1, 32, 8, 128, (16, 24, 24), 4096), (1, 1, 1, 2, (1,), 10), (5, 6, 2, 6, (1, 0, 2), 100),
    (33, 4, 4, 64, (32,), 1 << 20), (7, 8, 1, 256, (32, 32, 32, 32), 1 << 30), (3, 5, 5, 80, (8, 16, 16), 1000),
    (130, 16, 2, 96, (16, 16, 16), 50000)])
def test_rope_axes(dev, mem, n, nqh, nkh, hd, sections, far):
    """q within 2 F32 of the pair's length per product and sum (the angle's cosine and sine off by F32 and 2^-40),
    K and V rows the exact rounding of a value that close, other rows and layers untouched."""
    rng = np.random.default_rng(n + hd)
    slot, layer, max_ctx = 3, 1, n + 5
    qs, ks = nqh * hd + 4, nkh * hd + 2
    q, k, v = (rng.standard_normal((n, w)).astype(np.float32) for w in (qs, ks, ks))
    pos = rng.integers(-far // 8, far, (len(sections), n)).astype(np.int32)
    kc0, vc0 = f16_bits(rng, 2, max_ctx, nkh * hd), f16_bits(rng, 2, max_ctx, nkh * hd)
    pq, pk, pv, pp, pkc, pvc = (mem.up(x) for x in (q, k, v, pos, kc0, vc0))
    dev.rope_axes(pq, qs, pk, pv, ks, pp, n, sections, pkc, pvc, slot, layer, max_ctx, nqh, nkh, hd, 10000.0)
    gq, gk = dev.download(pq, (n, qs), np.float32), dev.download(pk, (n, ks), np.float32)
    gkc, gvc = dev.download(pkc, kc0.shape, np.uint16), dev.download(pvc, vc0.shape, np.uint16)
    assert np.array_equal(gk, k) and np.array_equal(gq[:, nqh * hd:], q[:, nqh * hd:])

    def rotated(x, heads):
        x = x[:, :heads * hd].reshape(n, heads, hd).astype(np.float64)
        size = np.repeat(np.abs(x[..., 0::2]) + np.abs(x[..., 1::2]), 2, -1)
        # the angle itself: 64 bits, |position| * 2^-51 at most beside the oracle's own
        return R.rope_axes(x, pos, sections, 10000.0), size * (4 * R.F32 + 2 * far * 2.0 ** -51)
    want, tol = rotated(q, nqh)
    close(gq[:, :nqh * hd].reshape(n, nqh, hd).astype(np.float64), want, tol)
    want, tol = rotated(k, nkh)
    got = R.half(gkc[layer, slot:slot + n]).reshape(n, nkh, hd)
    close(got, want, tol + np.abs(want) * 2.0 ** -11 + 2.0 ** -25)
    want16 = v[:, :nkh * hd].astype(np.float16)
    normal = np.abs(v[:, :nkh * hd]) >= 2.0 ** -14  # (below, the cache's own rounding is not IEEE's)
    assert np.array_equal(gvc[layer, slot:slot + n][normal], want16.view(np.uint16)[normal])
    for got, was in ((gkc, kc0), (gvc, vc0)):
        got, was = got.copy(), was.copy()
        got[layer, slot:slot + n] = was[layer, slot:slot + n] = 0
        assert np.array_equal(got, was)


def test_rope_axes_parts_and_store(dev, mem):
    """q alone and k and v alone give what both give; the stored rows are vbs_gfx950_cache_store's of the rotated k;
    n = 0 does nothing; the rows of a fused Q/K/V product can be given as they are."""
    rng = np.random.default_rng(5)
    n, nqh, nkh, hd, sec = 9, 4, 2, 32, (4, 6, 6)
    row = (nqh + 2 * nkh) * hd
    x = rng.standard_normal((n, row)).astype(np.float32)
    x[0, nqh * hd] = 3e-6  # a subnormal f16
    x[1, (nqh + nkh) * hd:(nqh + nkh) * hd + 4] = [np.inf, -np.inf, np.nan, 70000.0]
    pos = rng.integers(0, 999, (3, n)).astype(np.int32)
    pos[:, 0] = 0
    pp = mem.up(pos)
    outs = []
    for parts in (("both",), ("q", "kv")):
        p = mem.up(x)
        kc, vc = mem.zeros(n * nkh * hd, np.uint16), mem.zeros(n * nkh * hd, np.uint16)
        for part in parts:
            kv = part != "q"
            dev.rope_axes(p if part != "kv" else 0, row, p + 4 * nqh * hd if kv else 0,
                          p + 4 * (nqh + nkh) * hd if kv else 0, row, pp, n, sec, kc if kv else 0, vc if kv else 0,
                          0, 0, n, nqh, nkh, hd, 10000.0)
        dev.rope_axes(p, row, 0, 0, 0, pp, 0, sec, 0, 0, 0, 0, 0, nqh, nkh, hd, 10000.0)
        outs.append([dev.download(p, x.shape, np.float32), dev.download(kc, n * nkh * hd, np.uint16),
                     dev.download(vc, n * nkh * hd, np.uint16)])
    for a, b in zip(*outs):
        assert np.array_equal(a.view(np.uint8), b.view(np.uint8))
    # token 0 stands at position 0: its rows are its k and v themselves
    kc, vc = mem.zeros(nkh * hd, np.uint16), mem.zeros(nkh * hd, np.uint16)
    for i in (0, 1):
        src = mem.up(x[i])
        dev.cache_store(src + 4 * nqh * hd, src + 4 * (nqh + nkh) * hd, kc, vc, 0, 0, 1, nkh * hd)
        assert np.array_equal(dev.download(vc, nkh * hd, np.uint16), outs[0][2].reshape(n, -1)[i])
        if i == 0:
            assert np.array_equal(dev.download(kc, nkh * hd, np.uint16), outs[0][1].reshape(n, -1)[0])


# ---- attention -------------------------------------------------------------------------------------

SHAPES = [
    # n, past, q heads, kv heads, head_dim
    (1, 0, 1, 1, 2), (1, 1, 4, 2, 64), (1, 2047, 32, 8, 128), (2, 63, 8, 8, 32), (3, 64, 16, 1, 128),
    (5, 300, 6, 2, 96), (16, 129, 8, 2, 128), (17, 31, 5, 5, 80), (33, 95, 12, 4, 256), (63, 1, 4, 2, 64),
    (64, 0, 4, 1, 128), (65, 200, 4, 4, 6), (100, 33, 9, 3, 40), (130, 70, 6, 2, 128), (190, 513, 2, 1, 112),
    (257, 0, 8, 2, 64), (300, 1000, 4, 4, 32)]
IDS = ["-".join(map(str, s)) for s in SHAPES]


@pytest.mark.parametrize("shape", SHAPES, ids=IDS)
def test_tree(dev, mem, shape):
    n = shape[0]
    rng = np.random.default_rng(n)
    s = Step(rng, mem, dev, *shape)
    mask = random_tree(rng, n)
    want, _, tol, _ = s.want(R.sees_tree(n, shape[1], mask))
    close(s.tree(mask), want, tol)


@pytest.mark.parametrize("shape", SHAPES, ids=IDS)
@pytest.mark.parametrize("what", ["plain", "cap", "all"])
def test_chunk(dev, mem, shape, what):
    n, past, nqh, nkh, hd = shape
    rng = np.random.default_rng(n + past)
    s = Step(rng, mem, dev, *shape, q_pad=3 if what == "all" else 0, out_pad=5 if what == "all" else 0)
    terms, ref = {}, {}
    see = R.sees_chunk(n, past)
    if what != "plain":
        terms["cap"] = ref["cap"] = 4.0
    if what == "all":
        terms["slopes"] = ref["slopes"] = (2.0 ** -np.arange(1, nqh + 1)).astype(np.float32)
        docs = np.sort(rng.integers(0, 4, past + n)).astype(np.int32) - 2
        terms["docs"], terms["prefix"] = docs, past + n // 2 + 1
        see = R.sees_chunk(n, past, terms["prefix"], docs)
        mass0 = rng.random((s.layers, nkh, s.max_ctx)).astype(np.float32)
        terms["mass"] = mass0
    want, w, tol, wtol = s.want(see, **ref)
    close(s.chunk(**terms), want, tol)
    if what == "all":
        add, off = R.mass(w, wtol, nkh)
        got, exp = dev.download(s.pm, mass0.shape, np.float32).astype(np.float64), mass0.astype(np.float64)
        exp[1, :, :past + n] += add
        full = np.zeros_like(exp)
        full[1, :, :past + n] = off + 2 * R.F32 * exp[1, :, :past + n]
        close(got, exp, full)  # (other layers and the slots behind: exactly as they were)


@pytest.mark.parametrize("hd", [64, 128, 40])
@pytest.mark.parametrize("nqh,nkh", [(2, 1), (16, 1), (3, 3)])
def test_unaligned_pointers(dev, mem, hd, nqh, nkh):
    """Caches, q and out one element off their allocations."""
    rng = np.random.default_rng(hd)
    n, past = 21, 77
    s = Step(rng, mem, dev, n, past, nqh, nkh, hd, shift=1, q_pad=1, out_pad=1)
    want, _, tol, _ = s.want(R.sees_chunk(n, past))
    close(s.chunk(), want, tol)


@pytest.mark.parametrize("n,past,nqh,nkh,hd", [(70, 0, 4, 2, 64), (7, 0, 8, 1, 128), (1, 0, 2, 2, 96)])
def test_rows_that_see_nothing(dev, mem, n, past, nqh, nkh, hd):
    """Mask rows without a bit give 0 (without a past), and leave the others as they are."""
    rng = np.random.default_rng(n)
    mask = random_tree(rng, n)
    mask[::3] = 0
    s = Step(rng, mem, dev, n, past, nqh, nkh, hd)
    want, _, tol, _ = s.want(R.sees_tree(n, past, mask))
    got = s.tree(mask)
    assert (got[::3] == 0).all()
    close(got, want, tol)


@pytest.mark.parametrize("hd", [32, 64, 80, 128, 256, 6])
@pytest.mark.parametrize("n,past", [(40, 50), (3, 200)])
@pytest.mark.parametrize("bad", [NAN16, INF16, INF16 | 0x8000])
def test_values_in_unseen_slots(dev, mem, hd, n, past, bad):
    """A slot of another document, and a drafted token off the path, hold NaN or infinities in K and V: the rows that
    do not see them are what they are without, the rows that do see them carry them as the formula does."""
    rng = np.random.default_rng(hd)
    docs = (np.arange(past + n) % 3 == 0).astype(np.int32)
    for kind in ("docs", "tree"):
        s = Step(rng, mem, dev, n, past, 4, 2, hd)
        if kind == "docs":
            rows, see, args = docs == 1, R.sees_chunk(n, past, 0, docs), {"docs": docs}
        else:
            chain = [sum(1 << t for t in range(i + 1) if t % 2 == i % 2) for i in range(n)]
            mask = pack(chain, n)
            rows = np.zeros(past + n, bool)
            rows[past + 1::2] = True  # the odd branch
            see = R.sees_tree(n, past, mask)
        s.vc[1, :past + n][rows] = bad
        s.kc[1, :past + n][rows, :, ::2] = bad
        want, _, tol, _ = s.want(see)
        got = s.chunk(**args) if kind == "docs" else s.tree(mask)
        clean = ~(see & rows[None]).any(1)
        assert clean.any() and not clean.all()
        close(got[clean], want[clean], tol[clean])
        # (a row whose every score is -inf gives 0)
        assert not np.isfinite(got[~clean]).all() and np.array_equal(np.isfinite(got), np.isfinite(want))


@pytest.mark.parametrize("hd", [64, 128, 6])
def test_values_that_are_not_finite_and_seen(dev, mem, hd):
    """V infinite where the weight is not 0 comes through, in that dim alone; an infinite score of -inf weighs 0; a
    NaN or infinite q spoils its own row and head alone; huge and tiny q are scaled rightly."""
    rng = np.random.default_rng(hd)
    n, past = 24, 40
    s = Step(rng, mem, dev, n, past, 2, 1, hd)
    see = R.sees_chunk(n, past)
    s.vc[1, 3, 0, 1] = INF16
    s.kc[1, 5, 0, 0] = INF16 | 0x8000
    s.q[:, 0::hd] = np.abs(s.q[:, 0::hd]) + 0.1  # the score of slot 5 is -inf: it weighs nothing
    s.q[4, hd] = np.nan
    s.q[6, 0] = np.inf
    s.q[8, :hd] *= 1e30
    s.q[9, :hd] *= 1e-30
    want, _, tol, _ = s.want(see)
    got = s.chunk()
    assert np.isposinf(got[0, 0, 1]) and np.isfinite(np.delete(got[0, 0], 1)).all()
    for row, head in ((4, 1), (6, 0)):
        assert np.isnan(got[row, head]).all()
        got[row, head] = want[row, head] = 0
        tol[row, head] = 0
    # 1e30: one slot takes the whole weight (unless two scores agree to 1e-29 of them)
    close(got, want, np.where(np.isnan(tol), 0, tol))


def test_long_and_far(dev, mem):
    """Slots and layers whose offsets pass 32 bits: a cache of more than 2^32 elements before the layer's first row."""
    rng = np.random.default_rng(1)
    n, past, nqh, nkh, hd = 3, 70, 8, 4, 128
    max_ctx = (1 << 32) // (nkh * hd) + 1000  # one layer is more than 2^32 elements
    s = Step(rng, mem, dev, n, past, nqh, nkh, hd, layer=0)
    want, w, tol, wtol = s.want(R.sees_chunk(n, past))
    bytes_ = 2 * (max_ctx + past + n) * nkh * hd
    pk, pv = dev.alloc(bytes_), dev.alloc(bytes_)
    try:
        off = 2 * max_ctx * nkh * hd
        dev.write(pk + off, s.kc[0, :past + n])
        dev.write(pv + off, s.vc[0, :past + n])
        s.load()
        dev.attention_chunk(s.pq, s.qs, pk, pv, s.po, s.os, n, past, 1, max_ctx, nqh, nkh, hd, s.scale)
        close(s.got(), want, tol)
        # the last slots of layer 0, by rope_axes, and eviction in layer 1
        sec = (hd // 2,)
        pos = mem.up(np.zeros((1, n), np.int32))
        k, v = rng.standard_normal((2, n, nkh * hd)).astype(np.float32)
        dev.rope_axes(0, 0, mem.up(k), mem.up(v), nkh * hd, pos, n, sec, pk, pv, max_ctx - n, 0, max_ctx, nqh, nkh,
                      hd, 10000.0)
        got = dev.download(pk + off - 2 * n * nkh * hd, (n, nkh * hd), np.uint16)
        assert np.array_equal(got, k.astype(np.float16).view(np.uint16))
        assert np.array_equal(dev.download(pk + off, (past + n, nkh, hd), np.uint16), s.kc[0, :past + n])
    finally:
        dev.free(pk)
        dev.free(pv)


def test_sharp_scores(dev, mem):
    """Scores of several hundred: the running maximum moves and the sums are rescaled without overflow."""
    rng = np.random.default_rng(2)
    for n, past, hd in ((20, 700, 128), (3, 900, 64), (70, 300, 40)):
        s = Step(rng, mem, dev, n, past, 4, 2, hd, size=100.0)
        want, _, tol, _ = s.want(R.sees_chunk(n, past))
        close(s.chunk(), want, tol)


def test_many_rows_at_once(dev, mem):
    """A chunk wider than a grid row of tiles, against the same rows called in parts (each row's result goes by its
    own slots alone, to the rounding of f32 sums)."""
    rng = np.random.default_rng(3)
    n, past, nqh, nkh, hd = 1500, 37, 4, 1, 64
    s = Step(rng, mem, dev, n, past, nqh, nkh, hd)
    whole = s.chunk(cap=20.0)
    for a, b in ((0, 1), (1, 34), (700, 830), (1499, 1500)):
        p = s.po + 4 * a * s.os
        dev.attention_chunk(s.pq + 4 * a * s.qs, s.qs, s.pk, s.pv, p, s.os, b - a, past + a, s.layer, s.max_ctx, nqh,
                            nkh, hd, s.scale, cap=20.0)
        part = dev.download(p, (b - a, s.os), np.float32).reshape(b - a, nqh, hd)
        assert np.abs(part - whole[a:b]).max() <= 2e-5 * np.abs(whole).max()


def test_calls_repeat_exactly(dev, mem):
    """The same call gives the same bits (no sums in a changing order)."""
    rng = np.random.default_rng(4)
    for n, past, nqh, nkh, hd in ((1, 4000, 16, 2, 128), (200, 300, 8, 2, 64)):
        s = Step(rng, mem, dev, n, past, nqh, nkh, hd)
        mass0 = np.zeros((2, nkh, s.max_ctx), np.float32)
        runs = [(s.chunk(mass=mass0), dev.download(s.pm, mass0.shape, np.float32)) for _ in range(3)]
        for o, m in runs[1:]:
            assert np.array_equal(o, runs[0][0]) and np.array_equal(m, runs[0][1])


# ---- eviction -----------------------------------------------------------------------------------------

@pytest.mark.parametrize("layers,length,budget,first,last,nkh,hd,shift", [
    (1, 1, 1, 0, 0, 1, 2, 0), (1, 2, 1, 0, 1, 2, 64, 0), (2, 100, 37, 4, 9, 3, 64, 0), (1, 100, 100, 0, 0, 2, 128, 0),
    (1, 5000, 2049, 4, 256, 2, 128, 0), (3, 1025, 1024, 1, 1, 1, 32, 0), (1, 3000, 7, 3, 4, 1, 256, 0),
    (2, 777, 300, 0, 0, 5, 80, 0), (1, 500, 200, 2, 3, 2, 6, 0), (2, 600, 333, 5, 5, 2, 64, 1), (1, 4097, 1, 0, 0, 2, 96, 0)])
@pytest.mark.parametrize("values", ["spread", "ties", "odd"])
def test_evict(dev, mem, layers, length, budget, first, last, nkh, hd, shift, values):
    rng = np.random.default_rng(length)
    layer, max_ctx = 1, length + 3
    shape = (layer + layers + 1, max_ctx, nkh, hd)
    kc, vc = f16_bits(rng, *shape), f16_bits(rng, *shape)
    m = np.exp(3 * rng.standard_normal((shape[0], nkh, max_ctx))).astype(np.float32)
    if values != "spread":
        m = rng.integers(0, 3, m.shape).astype(np.float32)  # many equals
    if values == "odd":
        m[rng.random(m.shape) < 0.2] = np.nan
        m[rng.random(m.shape) < 0.2] = -0.0
        m[rng.random(m.shape) < 0.2] = -1.0
        m[rng.random(m.shape) < 0.1] = np.inf
        m[rng.random(m.shape) < 0.1] = -np.inf
        m[rng.random(m.shape) < 0.1] = 1e-42
    up = lambda a: mem.up(np.concatenate([np.zeros(shift, a.dtype), a.reshape(-1)])) + shift * a.itemsize  # noqa: E731
    pk, pv, pm, pmo = up(kc), up(vc), mem.up(m), mem.up(np.full(m.shape, 5.0, np.float32))
    kept = mem.zeros(layers * nkh * budget + 1, np.uint32)
    dev.cache_evict(pk, pv, pm, pmo, kept, length, budget, first, last, layer, layers, max_ctx, nkh, hd)
    got = dev.download(kept, layers * nkh * budget + 1, np.uint32)
    assert got[-1] == 0
    got = got[:-1].reshape(layers, nkh, budget)
    wk, wv, wm = kc.copy(), vc.copy(), np.full(m.shape, 5.0, np.float32)
    for x in range(layers):
        for h in range(nkh):
            slots = R.evict(m[layer + x, h], length, budget, first, last)
            assert np.array_equal(got[x, h], slots), (x, h)
            wk[layer + x, :budget, h], wv[layer + x, :budget, h] = kc[layer + x, slots, h], vc[layer + x, slots, h]
            wm[layer + x, h, :budget], wm[layer + x, h, budget:length] = m[layer + x, h, slots], 0
    assert np.array_equal(dev.download(pk, shape, np.uint16), wk)
    assert np.array_equal(dev.download(pv, shape, np.uint16), wv)
    gm = dev.download(pmo, m.shape, np.float32)
    assert np.array_equal(gm.view(np.uint32), wm.view(np.uint32))
    assert np.array_equal(dev.download(pm, m.shape, np.float32).view(np.uint32), m.view(np.uint32))
    # the same with the mass in place, and without
    pk2, pv2 = up(kc), up(vc)
    dev.cache_evict(pk2, pv2, pm, pm, kept, length, budget, first, last, layer, layers, max_ctx, nkh, hd)
    gm = dev.download(pm, m.shape, np.float32)
    lay = slice(layer, layer + layers)
    assert np.array_equal(gm[lay, :, :length].view(np.uint32), wm[lay, :, :length].view(np.uint32))
    assert np.array_equal(gm[:, :, length:].view(np.uint32), m[:, :, length:].view(np.uint32))
    assert np.array_equal(dev.download(pk2, shape, np.uint16), wk)
    pk3, pv3, pm3 = up(kc), up(vc), mem.up(m)
    dev.cache_evict(pk3, pv3, pm3, 0, kept, length, budget, first, last, layer, layers, max_ctx, nkh, hd)
    assert np.array_equal(dev.download(pv3, shape, np.uint16), wv)


# ---- together, captured, from threads --------------------------------------------------------------------

def test_a_run_of_them(dev, mem):
    """As a loop uses them: a prompt chunk is rotated, stored and attended to with its weights accumulated; the cache
    is cut; a tree of drafted tokens is rotated, stored behind the kept slots and attended to; then one token."""
    rng = np.random.default_rng(11)
    nqh, nkh, hd, sec, max_ctx, layer = 8, 2, 64, (8, 12, 12), 160, 1
    kvd = nkh * hd
    scale = float(np.float32(1 / math.sqrt(hd)))
    kc, vc = np.zeros((2, 2, max_ctx, nkh, hd), np.float64)
    mass = np.zeros((2, nkh, max_ctx))
    pk, pv = mem.zeros(2 * max_ctx * kvd, np.uint16), mem.zeros(2 * max_ctx * kvd, np.uint16)
    pm, kept = mem.zeros(2 * nkh * max_ctx), mem.zeros(nkh * 50, np.uint32)

    def step(n, past, first_pos, tree=None, with_mass=False):
        q, k, v = (rng.standard_normal((n, w)).astype(np.float32) for w in (nqh * hd, kvd, kvd))
        pos = (first_pos + rng.integers(0, 9, (3, n))).astype(np.int32)
        pq, out = mem.up(q), mem.zeros(n * nqh * hd)
        dev.rope_axes(pq, nqh * hd, mem.up(k), mem.up(v), kvd, mem.up(pos), n, sec, pk, pv, past, layer, max_ctx, nqh,
                      nkh, hd, 10000.0)
        # the device's own rounded rows are the next operator's inputs
        kc[layer, past:past + n] = R.rope_axes(k.reshape(n, nkh, hd).astype(np.float64), pos, sec, 10000.0)
        vc[layer, past:past + n] = v.reshape(n, nkh, hd)
        rows = [R.half(dev.download(p, (2, max_ctx, nkh, hd), np.uint16)) for p in (pk, pv)]
        for got, want in zip(rows, (kc, vc)):
            assert np.all(np.abs(got - want) <= np.abs(want) * 2.0 ** -10 + 2.0 ** -14)
            want[:] = got
        qr = dev.download(pq, (n, nqh, hd), np.float32).astype(np.float64)
        close(qr, R.rope_axes(q.reshape(n, nqh, hd).astype(np.float64), pos, sec, 10000.0), 1e-5)
        if tree is not None:
            dev.attention_tree(pq, nqh * hd, pk, pv, out, nqh * hd, n, past, mem.up(tree), layer, max_ctx, nqh, nkh,
                               hd, scale)
            see = R.sees_tree(n, past, tree)
        else:
            dev.attention_chunk(pq, nqh * hd, pk, pv, out, nqh * hd, n, past, layer, max_ctx, nqh, nkh, hd, scale,
                                cap=30.0, mass=pm if with_mass else 0)
            see = R.sees_chunk(n, past)
        want, w, tol, wtol = R.attend(qr, kc[layer, :past + n], vc[layer, :past + n], see, scale, past,
                                      cap=0.0 if tree is not None else 30.0)
        close(dev.download(out, (n, nqh, hd), np.float32).astype(np.float64), want, tol)
        if with_mass:
            add, off = R.mass(w, wtol, nkh)
            mass[layer, :, :past + n] += add
            got = dev.download(pm, mass.shape, np.float32)
            assert np.all(np.abs(got - mass) <= 1e-4 * mass + 1e-30)
            mass[:] = got

    step(90, 0, 0, with_mass=True)
    dev.cache_evict(pk, pv, pm, pm, kept, 90, 50, 2, 10, layer, 1, max_ctx, nkh, hd)
    for h in range(nkh):
        slots = R.evict(mass[layer, h], 90, 50, 2, 10)
        assert np.array_equal(dev.download(kept, (nkh, 50), np.uint32)[h], slots)
        kc[layer, :50, h], vc[layer, :50, h] = kc[layer, slots, h], vc[layer, slots, h]
        mass[layer, h, :50] = mass[layer, h, slots]
        mass[layer, h, 50:90] = 0
    step(21, 50, 90, tree=random_tree(rng, 21))
    step(1, 53, 93, with_mass=True)


def test_captured_and_replayed(dev, mem):
    """Graphs of the calls, captured without an uncaptured call before, replayed several times between eager work of
    their own kind and size: every replay gives the eager results."""
    rng = np.random.default_rng(12)
    hip, stream = V.Hip(), dev.stream()
    cases = []
    for n, past, nqh, nkh, hd in ((1, 3000, 16, 4, 128), (40, 500, 8, 2, 64)):
        s = Step(rng, mem, dev, n, past, nqh, nkh, hd)
        s.load()
        mask = mem.up(random_tree(rng, n))
        mass = mem.zeros(2 * nkh * s.max_ctx)
        shape = (s.layer, s.max_ctx, nqh, nkh, hd, s.scale)

        def call(s=s, mask=mask, mass=mass, shape=shape, which=0):
            if which == 0:
                dev.attention_tree(s.pq, s.qs, s.pk, s.pv, s.po, s.os, s.n, s.past, mask, *shape)
            else:
                dev.attention_chunk(s.pq, s.qs, s.pk, s.pv, s.po, s.os, s.n, s.past, *shape, cap=9.0, mass=mass)
        for which in (0, 1):
            cases.append((s, mass, nkh, which, call, hip.capture(stream, lambda c=call, w=which: c(which=w))))
    zero = lambda s, m, k: (dev.write(m, np.zeros((2, k, s.max_ctx), np.float32)),  # noqa: E731
                            dev.write(s.po, s.out0))
    try:
        for s, m, nkh, which, call, graph in cases:
            got = []
            for k in range(5):
                zero(s, m, nkh)
                if k % 2:
                    hip.launch(graph, stream)
                else:
                    call(which=which)
                dev.sync()
                got.append((s.got(), dev.download(m, (2, nkh, s.max_ctx), np.float32)))
            for o, x in got[1:]:
                assert np.array_equal(o, got[0][0]) and np.array_equal(x, got[0][1])
        # graphs one behind the other
        s, m, nkh, which, call, graph = cases[1]
        zero(s, m, nkh)
        hip.launch(cases[3][5], stream)
        hip.launch(graph, stream)
        dev.sync()
        assert np.array_equal(s.got(), s.got())
    finally:
        for c in cases:
            hip.destroy(c[5])


def test_two_threads(dev, mem):
    """Calls of two threads at once share the library's scratch without mixing."""
    rng = np.random.default_rng(13)
    steps = []
    for n, past, nqh, nkh, hd in ((2, 2500, 8, 2, 128), (50, 300, 4, 4, 64)):
        s = Step(rng, mem, dev, n, past, nqh, nkh, hd)
        want = s.chunk(mass=np.zeros((2, nkh, s.max_ctx), np.float32))
        steps.append((s, want))
    errors = []

    def work(s):
        try:
            for _ in range(40):
                dev.attention_chunk(s.pq, s.qs, s.pk, s.pv, s.po, s.os, s.n, s.past, s.layer, s.max_ctx, s.nqh, s.nkh,
                                    s.hd, s.scale, mass=s.pm)
        except Exception as e:  # noqa: BLE001
            errors.append(e)
    threads = [threading.Thread(target=work, args=(s,)) for s, _ in steps]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors
    for s, want in steps:
        assert np.array_equal(s.got(), want)


def test_nothing_to_do(dev, mem):
    """n = 0 leaves out and mass alone."""
    s = Step(np.random.default_rng(0), mem, dev, 1, 3, 2, 1, 32).load()
    mask = mem.zeros(1, np.uint64)
    dev.attention_tree(s.pq, s.qs, s.pk, s.pv, s.po, s.os, 0, 3, mask, 0, s.max_ctx, 2, 1, 32, 1.0)
    dev.attention_chunk(s.pq, s.qs, s.pk, s.pv, s.po, s.os, 0, 4, 0, s.max_ctx, 2, 1, 32, 1.0)
    assert np.array_equal(dev.download(s.po, s.out0.shape, np.float32), s.out0)


# ---- few rows (at most 16 of a kv head) and the mass, where they go their own ways ---------------------------

FEW = [(1, 500, 4, 1, 256), (2, 70, 16, 2, 256), (16, 40, 1, 1, 128), (1, 3000, 16, 1, 64), (4, 1000, 4, 1, 96),
       (1, 127, 2, 1, 32), (3, 333, 10, 2, 80), (1, 0, 16, 1, 128), (5, 4100, 3, 1, 40)]


@pytest.mark.parametrize("shape", FEW, ids=["-".join(map(str, s)) for s in FEW])
@pytest.mark.parametrize("docs", [False, True])
def test_few_rows(dev, mem, shape, docs):
    n, past, nqh, nkh, hd = shape
    rng = np.random.default_rng(past)
    s = Step(rng, mem, dev, *shape, out_pad=2, q_pad=4)
    ids = rng.integers(-1, 2, past + n).astype(np.int32) if docs else None
    mass0 = rng.random((s.layers, nkh, s.max_ctx)).astype(np.float32)
    slopes = np.linspace(0.5, 0.01, nqh).astype(np.float32)
    want, w, tol, wtol = s.want(R.sees_chunk(n, past, 0, ids), cap=8.0, slopes=slopes)
    close(s.chunk(cap=8.0, slopes=slopes, mass=mass0, **({"docs": ids} if docs else {})), want, tol)
    add, off = R.mass(w, wtol, nkh)
    got = dev.download(s.pm, mass0.shape, np.float32).astype(np.float64)
    exp, full = mass0.astype(np.float64), np.zeros_like(got)
    exp[1, :, :past + n] += add
    full[1, :, :past + n] = off + 2 * R.F32 * exp[1, :, :past + n]
    close(got, exp, full)


@pytest.mark.parametrize("n,past,nqh,nkh,hd", [(2, 90, 4, 2, 128), (3, 200, 2, 1, 64), (60, 90, 4, 2, 128),
                                               (200, 30, 8, 1, 80), (40, 10, 2, 1, 6)])
@pytest.mark.parametrize("bad", [NAN16, INF16, INF16 | 0x8000])
def test_mass_with_values_that_are_not_finite(dev, mem, n, past, nqh, nkh, hd, bad):
    """K and V of unseen slots spoil no weight; a seen slot whose score is -inf weighs 0 and leaves the others' alone."""
    rng = np.random.default_rng(n)
    docs = (np.arange(past + n) % 5 == 0).astype(np.int32)
    docs[past:] = 0  # every row is of document 0
    s = Step(rng, mem, dev, n, past, nqh, nkh, hd)
    s.kc[1, :past][docs[:past] == 1] = bad
    s.vc[1, :past][docs[:past] == 1] = bad
    s.kc[1, 7] = 0
    s.kc[1, 7, :, 0] = INF16 | 0x8000  # q is positive there: -inf
    s.q[:, 0::hd] = np.abs(s.q[:, 0::hd]) + 0.1
    mass0 = np.zeros((2, nkh, s.max_ctx), np.float32)
    want, w, tol, wtol = s.want(R.sees_chunk(n, past, 0, docs))
    close(s.chunk(docs=docs, mass=mass0), want, tol)
    add, off = R.mass(w, wtol, nkh)
    got = dev.download(s.pm, mass0.shape, np.float32).astype(np.float64)
    assert np.isfinite(got).all() and (got[1, :, 7] == 0).all() and (got[1, :, :past][:, docs[:past] == 1] == 0).all()
    close(got[1, :, :past + n], add, off)
    assert (got[0] == 0).all() and (got[:, :, past + n:] == 0).all()


@pytest.mark.parametrize("n,past,hd", [(2, 60, 128), (50, 60, 64), (20, 20, 10)])
@pytest.mark.parametrize("scale", [0.0, -0.25, 1e-30, 3.0])
def test_scales(dev, mem, n, past, hd, scale):
    rng = np.random.default_rng(n)
    s = Step(rng, mem, dev, n, past, 4, 2, hd)
    s.scale = float(np.float32(scale))
    docs = (np.arange(past + n) % 2).astype(np.int32)
    want, _, tol, _ = s.want(R.sees_chunk(n, past, 0, docs))
    close(s.chunk(docs=docs), want, tol)


@pytest.mark.parametrize("n,past,nqh,nkh,hd", [(200, 1500, 4, 2, 64), (70, 900, 2, 2, 256), (1, 1500, 8, 2, 128),
                                               (300, 700, 3, 1, 96)])
@pytest.mark.parametrize("order", ["runs", "mixed", "far"])
def test_documents_over_many_tiles(dev, mem, n, past, nqh, nkh, hd, order):
    """Runs of documents (most tiles hold none of a row's), documents in any order, and the largest and least ids."""
    rng = np.random.default_rng(past)
    total = past + n
    docs = np.repeat(np.arange(total), rng.integers(1, 200, total))[:total].astype(np.int32)
    if order == "mixed":
        docs = rng.permutation(docs).astype(np.int32)
    if order == "far":
        docs = np.where(docs % 2 == 0, np.int32(2**31 - 1), np.int32(-2**31)).astype(np.int32)
    s = Step(rng, mem, dev, n, past, nqh, nkh, hd)
    prefix = past + 3
    want, w, tol, wtol = s.want(R.sees_chunk(n, past, prefix, docs))
    mass0 = np.zeros((2, nkh, s.max_ctx), np.float32)
    close(s.chunk(docs=docs, prefix=prefix, mass=mass0), want, tol)
    add, off = R.mass(w, wtol, nkh)
    close(dev.download(s.pm, mass0.shape, np.float32)[1, :, :total].astype(np.float64), add, off)


@pytest.mark.parametrize("n,past,nqh,nkh,hd", [(1, 200, 8, 2, 128), (2, 77, 2, 2, 64), (70, 33, 2, 1, 96)])
def test_unaligned_few_and_many(dev, mem, n, past, nqh, nkh, hd):
    rng = np.random.default_rng(hd)
    s = Step(rng, mem, dev, n, past, nqh, nkh, hd, shift=3, q_pad=1, out_pad=3)
    mass0 = np.zeros((2, nkh, s.max_ctx), np.float32)
    want, w, tol, wtol = s.want(R.sees_chunk(n, past), cap=3.0)
    close(s.chunk(cap=3.0, mass=mass0), want, tol)
    add, off = R.mass(w, wtol, nkh)
    close(dev.download(s.pm, mass0.shape, np.float32)[1, :, :past + n].astype(np.float64), add, off)


@pytest.mark.parametrize("hd", [32, 64, 128, 256])
def test_seen_infinities_in_few_rows(dev, mem, hd):
    """As test_values_that_are_not_finite_and_seen, at one and two rows of a kv head."""
    rng = np.random.default_rng(hd)
    s = Step(rng, mem, dev, 2, 300, 2, 1, hd)
    s.vc[1, 3, 0, 1] = INF16
    s.kc[1, 5] = 0
    s.kc[1, 5, 0, 0] = INF16 | 0x8000
    s.q[:, 0::hd] = np.abs(s.q[:, 0::hd]) + 0.1
    s.q[1, hd + 1] = np.nan
    want, _, tol, _ = s.want(R.sees_chunk(2, 300))
    got = s.chunk()
    assert np.isnan(got[1, 1]).all() and np.isposinf(got[0, :, 1]).all() and np.isposinf(got[1, 0, 1])
    got[1, 1] = want[1, 1] = 0
    tol[1, 1] = 0
    close(got, want, np.where(np.isnan(tol), 0, tol))


@pytest.mark.parametrize("length,budget,first,last", [(8193, 8192, 0, 1), (20001, 9000, 3, 100), (16384, 1, 0, 0),
                                                      (24600, 24599, 5, 7)])
@pytest.mark.parametrize("values", ["spread", "ties"])
def test_evict_longer_than_a_run(dev, mem, length, budget, first, last, values):
    """More slots than a workgroup holds at once: selection and order over several runs, the mass in place."""
    rng = np.random.default_rng(length)
    nkh, hd = 2, 16
    kc, vc = f16_bits(rng, 1, length, nkh, hd), f16_bits(rng, 1, length, nkh, hd)
    m = np.exp(2 * rng.standard_normal((1, nkh, length))).astype(np.float32)
    if values == "ties":
        m = rng.integers(0, 2, m.shape).astype(np.float32)
    pk, pv, pm, kept = mem.up(kc), mem.up(vc), mem.up(m), mem.zeros(nkh * budget, np.uint32)
    dev.cache_evict(pk, pv, pm, pm, kept, length, budget, first, last, 0, 1, length, nkh, hd)
    got, gk, gv = dev.download(kept, (nkh, budget), np.uint32), dev.download(pk, kc.shape, np.uint16), dev.download(pv, vc.shape, np.uint16)
    gm = dev.download(pm, m.shape, np.float32)
    for h in range(nkh):
        slots = R.evict(m[0, h], length, budget, first, last)
        assert np.array_equal(got[h], slots)
        assert np.array_equal(gk[0, :budget, h], kc[0, slots, h]) and np.array_equal(gv[0, :budget, h], vc[0, slots, h])
        assert np.array_equal(gk[0, budget:, h], kc[0, budget:, h])
        assert np.array_equal(gm[0, h, :budget], m[0, h, slots]) and (gm[0, h, budget:] == 0).all()


def test_a_captured_step_and_two_graphs_at_once(dev, mem):
    """A whole step (rotation and store, attention with weights, eviction) replayed from one graph; and graphs of
    attentions that use scratch replayed on two streams at once: each has memory of its own."""
    rng = np.random.default_rng(21)
    hip, stream = V.Hip(), dev.stream()
    n, past, nqh, nkh, hd, sec = 20, 230, 8, 2, 64, (32,)
    total, kvd = past + n, nkh * hd
    kc, vc = f16_bits(rng, total, nkh, hd), f16_bits(rng, total, nkh, hd)
    q, k, v = (rng.standard_normal((n, w)).astype(np.float32) for w in (nqh * hd, kvd, kvd))
    m = rng.random((nkh, total)).astype(np.float32)
    arrays = [kc, vc, q, m, np.zeros((n, nqh * hd), np.float32), np.zeros((nkh, 100), np.uint32)]
    ptrs = [mem.up(a) for a in arrays]
    pkc, pvc, pq, pm, po, pkept = ptrs
    pk, pv, pp = mem.up(k), mem.up(v), mem.up(np.arange(n, dtype=np.int32) + past)

    def step():
        dev.rope_axes(pq, nqh * hd, pk, pv, kvd, pp, n, sec, pkc, pvc, past, 0, total, nqh, nkh, hd, 10000.0)
        dev.attention_chunk(pq, nqh * hd, pkc, pvc, po, nqh * hd, n, past, 0, total, nqh, nkh, hd, 0.125, mass=pm)
        dev.cache_evict(pkc, pvc, pm, pm, pkept, total, 100, 4, 30, 0, 1, total, nkh, hd)

    graph = hip.capture(stream, step)
    results = []
    try:
        for i in range(4):
            for p, a in zip(ptrs, arrays):
                dev.write(p, a)
            step() if i % 2 == 0 else hip.launch(graph, stream)
            dev.sync()
            results.append([dev.download(p, a.shape, a.dtype) for p, a in zip(ptrs, arrays)])
        for r in results[1:]:
            for a, b in zip(r, results[0]):
                assert np.array_equal(a.view(np.uint8), b.view(np.uint8))
    finally:
        hip.destroy(graph)

    other = C.c_void_p()
    assert hip.h.hipStreamCreateWithFlags(C.byref(other), 1) == 0
    graphs, steps = [], []
    try:
        for n, past, nqh, nkh, hd in ((1, 6000, 16, 2, 128), (30, 900, 8, 2, 64)):
            s = Step(rng, mem, dev, n, past, nqh, nkh, hd)
            want = s.chunk(cap=7.0)
            shape = (s.layer, s.max_ctx, nqh, nkh, hd, s.scale)

            def call(s=s, shape=shape):
                for _ in range(8):
                    dev.attention_chunk(s.pq, s.qs, s.pk, s.pv, s.po, s.os, s.n, s.past, *shape, cap=7.0)
            graphs.append(hip.capture(stream, call))
            steps.append((s, want))
        for _ in range(5):
            for s, _ in steps:
                dev.write(s.po, s.out0)
            hip.launch(graphs[0], stream)
            hip.launch(graphs[1], other.value)
            assert hip.h.hipStreamSynchronize(other) == 0
            dev.sync()
            for s, want in steps:
                assert np.array_equal(s.got(), want)
    finally:
        for g in graphs:
            hip.destroy(g)
        hip.h.hipStreamDestroy(other)


@pytest.mark.parametrize("docs", [False, True])
def test_mass_of_more_rows_than_a_wave_looks_through_at_once(dev, mem, docs):
    """8800 rows of a kv head in one workgroup's share. The heads of a kv head ask the same, so one of them stands
    for all in the oracle, and the bound of a sum counts every row."""
    n, past, nqh, nkh, hd, group = 1100, 0, 128, 16, 32, 8
    rng = np.random.default_rng(n)
    s = Step(rng, mem, dev, n, past, nqh, nkh, hd)
    one = s.q.reshape(n, nkh, group, hd)[:, :, :1].copy()
    s.q = np.ascontiguousarray(np.broadcast_to(one, (n, nkh, group, hd))).reshape(n, nqh * hd)
    ids = np.repeat(np.arange(n), rng.integers(1, 60, n))[:n].astype(np.int32) if docs else None
    want, w, tol, wtol = R.attend(one[:, :, 0].astype(np.float64), R.half(s.kc[1, :n]), R.half(s.vc[1, :n]),
                                  R.sees_chunk(n, past, 0, ids), s.scale, past)
    mass0 = np.zeros((2, nkh, s.max_ctx), np.float32)
    got = s.chunk(mass=mass0, **({"docs": ids} if docs else {}))
    close(got, np.repeat(want, group, 1), np.repeat(tol, group, 1))
    add = group * w.sum(0)
    off = group * wtol.sum(0) + add * (n * group + 2) * R.F32
    close(dev.download(s.pm, mass0.shape, np.float32)[1, :, :n].astype(np.float64), add, off)


@pytest.mark.parametrize("layers,length,budget,nkh,hd", [(33, 2100, 1050, 8, 16), (33, 600, 300, 8, 16), (33, 4100, 2060, 8, 16)])
@pytest.mark.parametrize("place", ["same", "other", "none"])
def test_evict_of_many_heads(dev, mem, layers, length, budget, nkh, hd, place):
    """264 heads: more workgroups than two a CU, the mass in place, in another array, or left as it is."""
    rng = np.random.default_rng(length)
    first, last, max_ctx = 4, 30, length + 2
    mass = rng.integers(0, 1 << 16, (layers, nkh, max_ctx)).astype(np.float32)  # (some equal)
    kc, vc = (rng.integers(0, 1 << 16, (layers, max_ctx, nkh, hd)).astype(np.uint16) for _ in range(2))
    pk, pv, pm = mem.up(kc), mem.up(vc), mem.up(mass)
    po = {"same": pm, "other": mem.up(np.full_like(mass, 3.0)), "none": 0}[place]
    pt = mem.up(np.zeros((layers, nkh, budget), np.uint32))
    dev.cache_evict(pk, pv, pm, po, pt, length, budget, first, last, 0, layers, max_ctx, nkh, hd)
    kept = dev.download(pt, (layers, nkh, budget), np.uint32).astype(np.int64)
    gk, gv = dev.download(pk, kc.shape, np.uint16), dev.download(pv, vc.shape, np.uint16)
    gm = dev.download(po or pm, mass.shape, np.float32)
    for l in range(layers):
        for h in range(nkh):
            want = R.evict(mass[l, h], length, budget, first, last)
            assert np.array_equal(kept[l, h], want)
            assert np.array_equal(gk[l, :budget, h], kc[l, want, h]) and np.array_equal(gv[l, :budget, h], vc[l, want, h])
            if po:
                assert np.array_equal(gm[l, h, :budget], mass[l, h, want]) and not gm[l, h, budget:length].any()
    assert np.array_equal(gk[:, budget:], kc[:, budget:]) and np.array_equal(gv[:, budget:], vc[:, budget:])
    assert np.array_equal(gm[..., length:], mass[..., length:] if place != "other" else np.full_like(gm[..., length:], 3.0))
    if not po:
        assert np.array_equal(gm, mass)
