"""The paged cache (vbs_gfx950_page_store, _page_load, _attention_paged) and vbs_gfx950_verify_draft against their
definitions in 64 bits (pages_ref.py), at the sizes, places, strides and values where they can go wrong. No counterpart
in the reference (one cache, one token at a time: src/vbs_host_math.h:150-209, src/vbs_specializer.c:353-357): parity
unpinned."""
import ctypes as C
import math
import threading

import numpy as np
import pytest

import pages_ref as R
import steps_ref as S
import vbs_gfx950 as V
from test_gpu_kernels import Mem, mem  # noqa: F401 (mem: fixture)
from test_gpu_steps import close

pytestmark = pytest.mark.gpu

TYPES = pytest.mark.parametrize("t", [V.F16, V.Q8_0], ids=["f16", "q8"])


def filler(rng, t, page, n_pages, nkh, hd, size=1.0):
    """Pages of earlier tokens: values about N(0, size), scales of blocks that differ."""
    def fill(_):
        n = n_pages * nkh * (page // 32)
        if t == V.F16:
            return (size * rng.standard_normal((n, R.nb(hd) * 1024))).astype(np.float16).view(np.uint8)
        q = np.clip(np.rint(45 * rng.standard_normal((n, R.nb(hd) * 1024))), -127, 127).astype(np.int8).view(np.uint8)
        d = (size * 0.02 * np.exp(0.4 * rng.standard_normal((n, R.nb(hd) * 32)))).astype(np.float16).view(np.uint8)
        return np.ascontiguousarray(np.concatenate([q, d], 1))
    return fill


class Cache:
    """A pool of `layers` layers on the device (only `layer` is the pool on the host, the others guard it) and a table."""

    def __init__(self, rng, mem, dev, t, page, nkh, hd, seqs, per_seq, spare=2, layer=1, size=1.0):
        self.n_pages, self.layer, self.mem, self.dev = seqs * per_seq + spare, layer, mem, dev
        self.pool = R.Pool(t, page, self.n_pages, nkh, hd, filler(rng, t, page, self.n_pages, nkh, hd, size))
        self.table = rng.permutation(self.n_pages)[:seqs * per_seq].reshape(seqs, per_seq).astype(np.int32)
        self.t, self.page, self.nkh, self.hd, self.seqs, self.per_seq = t, page, nkh, hd, seqs, per_seq
        self.guard = rng.integers(0, 256, self.pool.bytes["k"].nbytes).astype(np.uint8)

    def load(self):
        """Everything on the device, as it now is on the host."""
        self.ptr = {w: self.mem.up(np.concatenate([self.guard] * self.layer + [self.pool.bytes[w].reshape(-1), self.guard]))
                    for w in "kv"}
        self.ptable = self.mem.up(self.table)
        self.pages = V.Pages(self.ptr["k"], self.ptr["v"], self.t, self.page, self.n_pages, self.nkh, self.hd, self.ptable,
                             self.seqs, self.per_seq)
        return self

    def check(self):
        """The device's pools are the host's, and the layers around them are as they were."""
        for w in "kv":
            n = self.guard.nbytes
            got = self.dev.download(self.ptr[w], n * (self.layer + 2), np.uint8)
            for i in range(self.layer + 2):
                want = self.pool.bytes[w].reshape(-1) if i == self.layer else self.guard
                part = got[i * n:(i + 1) * n]
                assert np.array_equal(part, want), (w, i, np.flatnonzero(part != want)[:8], int((part != want).sum()))

    def place(self, seq, at):
        """(page, slot) of a token, or None."""
        if at < 0 or not 0 <= seq < self.seqs or at // self.page >= self.per_seq:
            return None
        p = int(self.table[seq, at // self.page])
        return (p, at % self.page) if 0 <= p < self.n_pages else None


def places(rng, kind, cache, n):
    """n tokens' (seq, at), no place twice."""
    per = cache.per_seq * cache.page
    if kind == "prompt":  # consecutive slots of one sequence, beginning anywhere
        first = int(rng.integers(0, per - n + 1))
        return np.full(n, cache.seqs - 1, np.int32), first + np.arange(n, dtype=np.int32)
    every = rng.permutation(cache.seqs * per)[:n]
    if kind == "several":  # runs of several sequences, one after the other
        every = np.sort(every)
    return (every // per).astype(np.int32), (every % per).astype(np.int32)


# ---- rows into pages ----------------------------------------------------------------------------

STORES = [("prompt", 32, 1, 2, 1, 5), ("prompt", 64, 2, 128, 2, 100), ("prompt", 32, 3, 80, 3, 70), ("several", 32, 1, 256, 2, 33),
          ("any", 64, 2, 96, 4, 50), ("any", 256, 1, 6, 2, 200), ("prompt", 128, 8, 128, 1, 1), ("prompt", 32, 1, 32, 4, 128),
          ("several", 1024, 2, 64, 2, 300), ("prompt", 64, 1, 160, 2, 97), ("prompt", 32, 2, 30, 5, 160)]


@TYPES
@pytest.mark.parametrize("kind,page,nkh,hd,seqs,n", STORES)
@pytest.mark.parametrize("pad", [0, 3])
def test_store(dev, mem, t, kind, page, nkh, hd, seqs, n, pad):
    """Every byte of the pools: the stored slots as the definition has them, everything else as it was."""
    rng = np.random.default_rng(n + hd)
    c = Cache(rng, mem, dev, t, page, nkh, hd, seqs, (n + page - 1) // page + 1).load()
    seq, at = places(rng, kind, c, n)
    stride = nkh * hd + pad
    x = {w: (rng.standard_normal((n, stride)) * np.exp(rng.standard_normal(stride))).astype(np.float32) for w in "kv"}
    dev.page_store(c.pages, 1, mem.up(x["k"]), mem.up(x["v"]), stride, mem.up(seq), mem.up(at), n)
    for i in range(n):
        page_, slot = c.place(seq[i], at[i])
        for w in "kv":
            c.pool.put(w, page_, slot, x[w][i, :nkh * hd].reshape(nkh, hd))
    c.check()


@TYPES
def test_store_skips_what_has_no_place(dev, mem, t):
    """Negative slots, sequences and slots outside the table, and table entries that are no page store nothing; seq NULL."""
    rng = np.random.default_rng(7)
    c = Cache(rng, mem, dev, t, 32, 2, 64, 9, 3)
    c.table[0, 0], c.table[1, 1], c.table[2, 2], c.table[3, 0] = -1, c.n_pages, -2**31, 2**31 - 1
    c.load()
    at = np.array([3, 40, 70, 31, 96, -1, -2**31, 2**31 - 1, 5], np.int32)
    x = {w: rng.standard_normal((9, 128)).astype(np.float32) for w in "kv"}
    px = {w: mem.up(x[w]) for w in "kv"}
    dev.page_store(c.pages, 1, px["k"], px["v"], 128, 0, mem.up(at), 9)
    seq = np.array([9, -1, 2**31 - 1, -2**31, 4, 5, 6, 7, 8], np.int32)
    late = np.array([0, 0, 0, 0, 17, 18, 95, 1, -7], np.int32)
    dev.page_store(c.pages, 1, px["k"], px["v"], 128, mem.up(seq), mem.up(late), 9)
    dev.page_store(c.pages, 1, px["k"], px["v"], 128, 0, mem.up(at), 0)  # none
    for s, a in ((np.arange(9), at), (seq, late)):
        for i in range(9):
            p = c.place(int(s[i]), int(a[i]))
            for w in "kv" if p else "":
                c.pool.put(w, *p, x[w][i].reshape(2, 64))
    c.check()


def test_quantisation_borders(dev, mem):
    """Quotients on, next to and between borders; scales that are subnormal, zero, on a border of f16, or pass its range."""
    rng = np.random.default_rng(11)
    rows = []
    for d in (1.0, 0.013977, 2.0 ** -14, 2.0 ** -24, 5 * 2.0 ** -24, 600.0, 65504.0):
        d = float(np.float16(d))
        k = rng.integers(-126, 127, (40, 32)) + rng.choice([0.0, 0.5, 0.25], (40, 32))
        b = np.float32(k * d)
        b[:, 0] = np.float32(127 * d)
        near = rng.integers(-1, 2, b.shape)
        b = np.where(near > 0, np.nextafter(b, np.float32(np.inf)), np.where(near < 0, np.nextafter(b, -np.float32(np.inf)), b))
        b[::2, 0] = np.float32(127 * d)
        rows.append(b)
    # maxima on and next to the border between two scales: 127 times a midpoint
    mid = np.float16(rng.random(200) + 0.5)
    top = 127 * (mid.astype(np.float64) + np.nextafter(mid, np.float16(9)).astype(np.float64)) / 2
    b = (rng.standard_normal((200, 32)) * 20).astype(np.float32)
    b[:, 5] = np.float32(top)
    b[::3, 5] = np.nextafter(b[::3, 5], np.float32(np.inf))
    b[1::3, 5] = np.nextafter(b[1::3, 5], np.float32(0))
    rows.append(b)
    odd = np.float32([[0.0] * 32, [1e-45] * 32, [127 * 2.0 ** -25] * 32, [127 * 2.0 ** -25 * 1.0001] * 32, [-3e38] * 32,
                      [127 * 65519.9] * 32, [127 * 65520.0] * 32, [1.0] * 31 + [np.nan], [np.inf] + [0] * 31,
                      [-np.inf] * 32, [-0.0] * 32, [3e-39, -3e-39] * 16])
    x = np.concatenate(rows + [odd]).astype(np.float32)
    n = len(x)
    c = Cache(rng, mem, dev, V.Q8_0, 64, 1, 32, 1, (n + 63) // 64).load()
    px, at = mem.up(x), mem.up(np.arange(n, dtype=np.int32))
    seq = mem.up(np.zeros(n, np.int32))
    dev.page_store(c.pages, 1, px, px, 32, seq, at, n)
    for i in range(n):
        for w in "kv":
            c.pool.put(w, *c.place(0, i), x[i].reshape(1, 32))
    c.check()


def test_f16_rounding(dev, mem):
    """F16 pages hold what vbs_gfx950_cache_store holds, at every kind of value, and give it back."""
    rng = np.random.default_rng(12)
    x = rng.integers(0, 1 << 32, 64 * 256, dtype=np.uint64).astype(np.uint32).view(np.float32).reshape(64, 256)
    x[0, :8] = [np.inf, -np.inf, np.nan, 65519, 65520, 2.0 ** -25, 2.0 ** -24 * 1.5, 0]
    c = Cache(rng, mem, dev, V.F16, 32, 1, 256, 1, 2).load()
    px, at, seq = mem.up(x), mem.up(np.arange(64, dtype=np.int32)), mem.up(np.zeros(64, np.int32))
    dev.page_store(c.pages, 1, px, px, 256, seq, at, 64)
    flat = [mem.zeros(64 * 256, np.uint16) for _ in range(4)]
    for i in range(64):
        dev.cache_store(px + 4 * 256 * i, px + 4 * 256 * i, flat[0], flat[1], i, 0, 64, 256)
    dev.page_load(c.pages, 1, V.F16, flat[2], flat[3], 256, seq, at, 64)
    k, v, gk, gv = (dev.download(p, 64 * 256, np.uint16) for p in flat)
    assert np.array_equal(k, gk) and np.array_equal(v, gv)


# ---- rows out of pages --------------------------------------------------------------------------

@TYPES
@pytest.mark.parametrize("out", [V.F16, V.F32], ids=["to_f16", "to_f32"])
@pytest.mark.parametrize("kind,page,nkh,hd,seqs,n", STORES)
def test_load(dev, mem, t, out, kind, page, nkh, hd, seqs, n):
    """Each row's values exactly (q d: one product in f32, exact; f16: the cache's rounding); gaps and rows behind
    the last are left, rows of negative slots too, and a place without a page gives NaN."""
    rng = np.random.default_rng(n + hd)
    c = Cache(rng, mem, dev, t, page, nkh, hd, seqs, (n + page - 1) // page + 1)
    if t == V.Q8_0:  # some scales of every kind
        s = c.pool.scales("v").reshape(-1)
        s[::37] = np.float16([0.0, np.nan, 6e-8, -0.5, 65504, np.inf])[np.arange(len(s[::37])) % 6].view(np.uint16)
    seq, at = places(rng, kind, c, n)
    gone = rng.random(n) < 0.05
    at[gone] = -1 - at[gone]
    if kind == "any":
        c.table[-1, -1] = -5
    c.load()
    dt, stride = (np.uint16, nkh * hd + 1) if out == V.F16 else (np.uint32, nkh * hd + 2)
    was = rng.integers(0, 1 << 15, (n + 1, stride)).astype(dt)
    po = {w: mem.up(was) for w in "kv"}
    dev.page_load(c.pages, 1, out, po["k"], po["v"], stride, mem.up(seq), mem.up(at), n)
    for w in "kv":
        want = was.copy()
        lost = np.zeros((n + 1, stride), bool)
        for i in range(n):
            p = c.place(seq[i], at[i])
            if at[i] < 0:
                continue
            if p is None:
                lost[i, :nkh * hd] = True
                continue
            with np.errstate(all="ignore"):
                x = c.pool.get(w, *p).reshape(-1).astype(np.float32)
            lost[i, :nkh * hd] = np.isnan(x)
            if out == V.F32:
                want[i, :nkh * hd] = x.view(np.uint32)
            elif t == V.F16:
                want[i, :nkh * hd] = x.astype(np.float16).view(np.uint16)
            else:
                want[i, :nkh * hd] = R.half_store(x)
        got = dev.download(po[w], was.shape, dt)
        assert np.isnan(got.view(np.float16 if out == V.F16 else np.float32)[lost]).all()
        assert np.array_equal(got[~lost], want[~lost])


# ---- attention ----------------------------------------------------------------------------------

class Rows:
    """One attention call: rows of the sequences `seq` with the lengths `lens` over a cache whose slots behind the
    longest row of a sequence, and pages of no sequence, hold NaN."""

    def __init__(self, rng, mem, dev, t, lens, nqh, nkh, hd, page=32, seq=None, pad=0, q_size=3.0, size=1.0, max_len=None,
                 layer=1, junk=True):
        self.lens = np.asarray(lens, np.int32)
        self.seq = np.arange(len(lens), dtype=np.int32) if seq is None else np.asarray(seq, np.int32)
        self.null_seq = seq is None
        longest = int(max(self.lens.max(), 1))
        self.max_len = longest if max_len is None else max_len
        self.c = Cache(rng, mem, dev, t, page, nkh, hd, int(self.seq.max()) + 1, -(-max(self.max_len, 1) // page), layer=layer, size=size)
        self.nqh, self.nkh, self.hd, self.mem, self.dev, self.layer = nqh, nkh, hd, mem, dev, layer
        self.stride = nqh * hd + pad
        self.q = (q_size * rng.standard_normal((len(lens), self.stride))).astype(np.float32)
        self.scale = float(np.float32(1 / math.sqrt(hd)))
        if junk:
            self.junk()

    def junk(self):
        c = self.c
        used = np.zeros((c.n_pages, c.page), bool)
        for s, n in zip(self.seq, self.lens):
            for j in range(max(0, n)):
                used[c.table[s, j // c.page], j % c.page] = True
        page, slot = np.nonzero(~used)
        for w in "kv":
            if c.t == V.Q8_0:
                for b in range(R.nb(c.hd)):
                    c.pool.scales(w)[page, :, slot // 32, b * 32 + slot % 32] = 0x7E00
                continue
            d = np.arange(R.nb(c.hd) * 32)
            at = R.place(c.t, w, c.hd, (slot % 32)[:, None], d[None])
            c.pool._values(w)[page[:, None], :, (slot // 32)[:, None], at] = 0xFE00

    def run(self):
        self.c.load()
        n = len(self.lens)
        self.pq, self.pl = self.mem.up(self.q), self.mem.up(self.lens)
        self.out0 = np.full((n + 1, self.stride), 7.5, np.float32)
        self.po = self.mem.up(self.out0)
        self.ps = 0 if self.null_seq else self.mem.up(self.seq)
        self.call()
        return self.got()

    def call(self):
        self.dev.attention_paged(self.c.pages, self.layer, self.pq, self.stride, self.po, self.stride, self.ps, self.pl,
                                 len(self.lens), self.max_len, self.nqh, self.scale)

    def got(self):
        n, w = len(self.lens), self.nqh * self.hd
        o = self.dev.download(self.po, (n + 1, self.stride), np.float32)
        assert np.array_equal(o[n], self.out0[n]) and np.array_equal(o[:, w:], self.out0[:, w:])
        return o[:n, :w].reshape(n, self.nqh, self.hd).astype(np.float64)

    def want(self):
        out, tol = [], []
        for s, n, q in zip(self.seq, self.lens, self.q):
            k, v = (self.c.pool.rows(w, self.c.table[s], n) for w in "kv")
            vmax = None
            if self.c.t == V.Q8_0 and n:
                d = [self.c.pool.scales("v")[self.c.table[s, j // self.c.page], :, j % self.c.page // 32].reshape(self.nkh, -1, 32)[..., j % 32]
                     for j in range(n)]
                vmax = 127.0 * float(np.max(np.abs(np.array(d).view(np.float16).astype(np.float64))))
            o, e = R.attend(q[:self.nqh * self.hd].reshape(self.nqh, self.hd).astype(np.float64), k, v, self.scale, vmax)
            out.append(o)
            tol.append(e)
        return np.array(out), np.array(tol)


ATT = [([1], 1, 1, 32, 32), ([1], 8, 1, 128, 64), ([31, 32, 33], 4, 2, 64, 32), ([0, 5, 64], 6, 2, 80, 64), ([127, 128, 129, 130], 8, 8, 96, 32),
       ([300], 16, 1, 128, 128), ([1000, 3], 24, 2, 64, 32), ([513], 9, 1, 2, 32), ([700, 0, 1], 5, 1, 256, 256),
       ([257, 90], 32, 8, 128, 64), ([200], 10, 2, 160, 32), ([77], 12, 4, 192, 1024), ([160, 161], 4, 1, 224, 32),
       ([2100], 2, 2, 32, 64), ([40] * 70, 4, 4, 30, 32)]


@TYPES
@pytest.mark.parametrize("lens,nqh,nkh,hd,page", ATT, ids=["-".join(map(str, (len(a[0]), max(a[0])) + a[1:])) for a in ATT])
def test_attention(dev, mem, t, lens, nqh, nkh, hd, page):
    rng = np.random.default_rng(sum(lens) + hd)
    r = Rows(rng, mem, dev, t, lens, nqh, nkh, hd, page)
    got = r.run()
    want, tol = r.want()
    close(got, want, tol)
    assert (got[np.asarray(lens) == 0] == 0).all()


@TYPES
@pytest.mark.parametrize("rows,longest,nqh,nkh,hd", [(70, 900, 8, 2, 64), (300, 600, 2, 1, 30), (64, 2000, 8, 8, 34), (70, 640, 16, 8, 64),
                                                     (3, 3000, 2, 1, 128), (17, 1100, 12, 1, 256)])
def test_attention_of_many_rows(dev, mem, t, rows, longest, nqh, nkh, hd):
    """Shares that hold several rows and heads, begin and end anywhere in them, more rows than a wave has lanes, empty
    rows and rows out of range among them."""
    rng = np.random.default_rng(rows)
    lens = rng.integers(1, longest + 1, rows)
    lens[0] = longest
    lens[1::7] = 0
    r = Rows(rng, mem, dev, t, lens, nqh, nkh, hd, max_len=longest)
    want, tol = r.want()
    r.lens[2::9] = -5
    r.lens[3::31] = longest + 1
    got = r.run()
    bad = (r.lens < 0) | (r.lens > longest)
    assert np.isnan(got[bad]).all() and (got[r.lens == 0] == 0).all()
    close(got[~bad], want[~bad], tol[~bad])


@TYPES
def test_a_row_in_many_pieces(dev, mem, t):
    """One row and head over more shares than a merging workgroup has threads; every slot the same but for the last, so
    the oracle is a formula."""
    rng = np.random.default_rng(40)
    n, hd = 262144 + 5, 32
    r = Rows(rng, mem, dev, t, [64], 1, 1, hd, page=1024, junk=False)
    r.c.table = np.full((1, n // 1024 + 1), int(r.c.table[0, 0]), np.int32)  # one page again and again
    page = r.c.table[0, 0]
    for j in range(1024):
        r.c.pool.put("k", page, j, np.zeros((1, hd), np.float32))
        r.c.pool.put("v", page, j, np.full((1, hd), 2.0 if j == (n - 1) % 1024 else 1.0, np.float32))
    r.c.per_seq, r.lens, r.max_len = n // 1024 + 1, np.array([n], np.int32), n
    k, v = (r.c.pool.get(w, page, (n - 1) % 1024) for w in "kv")
    assert (k == 0).all()
    got = r.run()
    one = r.c.pool.get("v", page, 0)
    hits = (n - 1) // 1024 + 1  # the slot comes once in every round of the page
    want = (one * (n - hits) + v * hits) / n
    # weights are equal and exact (2^0); n additions of a sum that ends at n, in f32, however they are grouped
    close(got[0], want, 2 * n * S.F32 * np.abs(want) / 64)


@TYPES
def test_many_short_rows(dev, mem, t):
    """Thousands of rows of few sequences, with empty ones and rows out of range, in one call."""
    rng = np.random.default_rng(41)
    rows, seqs, nkh, hd = 3000, 4, 2, 32
    seq = rng.integers(0, seqs, rows)
    lens = rng.integers(0, 3, rows)
    lens[7], seq[7] = 700, 2
    r = Rows(rng, mem, dev, t, lens, 2, nkh, hd, seq=seq, max_len=704, junk=False)
    r.lens[11::50] = -1
    r.lens[7] = 700
    r.seq[13::50] = seqs
    got = r.run()
    bad = (r.lens < 0) | (r.seq >= seqs)
    assert np.isnan(got[bad]).all() and (got[~bad & (r.lens == 0)] == 0).all()
    kv = [[r.c.pool.rows(w, r.c.table[i], 700 if i == 2 else 2) for w in "kv"] for i in range(seqs)]
    for i in np.flatnonzero(~bad & (r.lens > 0)):
        k, v = kv[r.seq[i]]
        n = r.lens[i]
        close(got[i], *R.attend(r.q[i].reshape(2, hd).astype(np.float64), k[:n], v[:n], r.scale, 127 * 0.2 if t == V.Q8_0 else None))


def test_many_pieces_that_are_not_finite(dev, mem):
    """Shares of more than 64 rows and heads, infinities in many of them: each is taken again by itself. A row of one slot
    is that slot's V, exactly."""
    rng = np.random.default_rng(33)
    rows, nkh, hd, seqs = 1200, 64, 2, 6
    lens = np.ones(rows, np.int64)
    lens[5] = 600
    r = Rows(rng, mem, dev, V.F16, lens, nkh, nkh, hd, q_size=0.1, seq=np.arange(rows) % seqs, junk=False)
    for i in (0, 2, 4):
        p, slot = r.c.place(i, 0)
        for h in range(i, nkh, 5):
            r.c.pool._values("v")[p, h, 0, R.place(V.F16, "v", hd, slot, 1)] = 0x7C00
    want = np.array([r.c.pool.get("v", *r.c.place(i, 0)) for i in range(seqs)])[np.arange(rows) % seqs]
    got = r.run()
    k, v = (r.c.pool.rows(w, r.c.table[5], 600) for w in "kv")
    close(got[5], *R.attend(r.q[5].reshape(nkh, hd).astype(np.float64), k, v, r.scale))
    got[5] = want[5]
    assert np.array_equal(got, want) and np.isposinf(got[0, 0, 1])


@TYPES
def test_attention_rows_of_a_sequence(dev, mem, t):
    """Drafted tokens: several rows of a sequence, each a slot longer, sequences in any order; a max_len far above."""
    rng = np.random.default_rng(5)
    r = Rows(rng, mem, dev, t, [50, 51, 52, 53, 7, 8, 0, 64], 8, 2, 64, seq=[2, 2, 2, 2, 0, 0, 1, 1], pad=5, max_len=4096)
    got = r.run()
    close(got, *r.want())


@TYPES
def test_shared_pages(dev, mem, t):
    """Two sequences with the same first pages."""
    rng = np.random.default_rng(6)
    r = Rows(rng, mem, dev, t, [90, 75], 4, 2, 64, junk=False)
    r.c.table[1, :2] = r.c.table[0, :2]
    close(r.run(), *r.want())


@TYPES
def test_rows_out_of_range_are_nan(dev, mem, t):
    """A length that is negative or passes max_len, a sequence that is none, a page that is none: that row is NaN, the
    others are right, and a page that a row does not reach does not matter."""
    rng = np.random.default_rng(8)
    r = Rows(rng, mem, dev, t, [70, 64, 70, 70, 70, 40, 70, 70], 4, 2, 64, seq=[0, 1, 2, 3, 4, 5, 6, 7], max_len=70)
    want, tol = r.want()
    r.c.table[1, 2] = -1            # behind its 64 slots
    r.c.table[2, 1] = r.c.n_pages
    r.c.table[3, 0] = -2**31
    r.lens[0], r.lens[4] = 71, -1
    r.seq[6], r.seq[7] = 8, -1
    got = r.run()
    bad = [0, 2, 3, 4, 6, 7]
    assert np.isnan(got[bad]).all()
    close(got[[1, 5]], want[[1, 5]], tol[[1, 5]])


@TYPES
@pytest.mark.parametrize("lens,nqh,nkh,hd", [([3000, 100], 8, 1, 64), ([5000], 2, 1, 128)])
def test_scores_of_all_sizes(dev, mem, t, lens, nqh, nkh, hd):
    """Scores in the hundreds (one slot takes all), and q of far sizes: 1e-30 and 1e30 with a scale to match."""
    rng = np.random.default_rng(hd)
    r = Rows(rng, mem, dev, t, lens, nqh, nkh, hd, q_size=100.0)
    close(r.run(), *r.want())
    q = r.q.copy()
    for f in (2.0 ** -90, 2.0 ** 90):
        r.q, r.scale = q * np.float32(f), float(np.float32(0.02 / f))
        close(r.run(), *r.want())
    for scale in (0.0, -0.03, 1e-30):
        r.q, r.scale = q, float(np.float32(scale))
        close(r.run(), *r.want())


@TYPES
def test_small_weights_beside_a_great_one(dev, mem, t):
    """Weights down to 2^-25 of the greatest with values of V 2^14 times as large as its own."""
    rng = np.random.default_rng(9)
    hd = 64
    r = Rows(rng, mem, dev, t, [400], 2, 1, hd, junk=False)
    x = np.zeros((1, hd), np.float32)
    for j in range(400):
        x[0, 0] = 8.0 if j == 123 else 8.0 - 17.5 / 2 * (1 + j % 2)
        r.c.pool.put("k", *r.c.place(0, j), x)
        r.c.pool.put("v", *r.c.place(0, j), (rng.standard_normal((1, hd)) * (1e-3 if j == 123 else 16.0)).astype(np.float32))
    r.q[:] = 0
    r.q[:, ::hd] = 1.0
    r.scale = 1.0
    close(r.run(), *r.want())


@TYPES
def test_subnormal_values(dev, mem, t):
    """K and V whose f16 (or whose scales) are subnormal, beside a q that makes scores of ordinary size of them."""
    rng = np.random.default_rng(16)
    hd = 64
    r = Rows(rng, mem, dev, t, [300], 4, 1, hd, junk=False)
    for j in range(300):
        for w in "kv":
            r.c.pool.put(w, *r.c.place(0, j), (rng.standard_normal((1, hd)) * 2e-5).astype(np.float32))
    r.q = (rng.standard_normal(r.q.shape) * 1e4).astype(np.float32)
    got = r.run()
    want, tol = r.want()
    assert np.abs(want).max() > 1e-7 and (tol < np.abs(want).max() / 100).all()
    close(got, want, tol)


def test_scales_of_both_signs(dev, mem):
    """Pages that callers build themselves may hold negative scales."""
    rng = np.random.default_rng(17)
    r = Rows(rng, mem, dev, V.Q8_0, [200, 33], 8, 2, 64, junk=False)
    for w in "kv":
        d = r.c.pool.scales(w)
        d ^= (rng.integers(0, 2, d.shape) << 15).astype(np.uint16)
    close(r.run(), *r.want())


def test_values_that_are_not_finite(dev, mem):
    """Seen infinities and NaN of an F16 cache, and NaN blocks of a Q8_0 one, give what the formula gives."""
    rng = np.random.default_rng(10)
    for hd, nqh in ((64, 4), (128, 8), (30, 9)):
        r = Rows(rng, mem, dev, V.F16, [300, 300, 300, 300, 300], nqh, 1, hd, q_size=0.5)
        r.q = np.abs(r.q) + np.float32(0.01)

        def value(w, seq, j, d, bits):
            p, slot = r.c.place(seq, j)
            r.c.pool._values(w)[p, 0, slot // 32, R.place(V.F16, w, hd, slot % 32, d)] = bits
        value("v", 0, 3, 1, 0x7C00)      # an infinite value: its element alone
        value("v", 0, 200, 2, 0xFC00)
        value("k", 1, 5, 0, 0xFC00)      # a score of -inf: weight 0
        value("k", 2, 299, 0, 0x7C00)    # +inf: the row is NaN
        value("v", 3, 100, 4, 0x7E00)
        r.q[4, 0] = np.nan               # one head
        got = r.run()
        want, tol = r.want()
        assert np.isposinf(got[0, :, 1]).all() and np.isneginf(got[0, :, 2]).all() and np.isnan(got[2]).all()
        assert np.isnan(got[4, 0]).all() and np.isfinite(got[4, 1:]).all()
        want[2], want[4, 0] = np.nan, np.nan
        close(got, want, np.where(np.isfinite(tol), tol, 0))
    r = Rows(rng, mem, dev, V.Q8_0, [300, 300], 8, 2, 64, q_size=0.5)
    p, slot = r.c.place(0, 150)
    r.c.pool.scales("v")[p, 1, slot // 32, 32 + slot % 32] = 0x7E00
    p, slot = r.c.place(1, 7)
    r.c.pool.scales("k")[p, 0, slot // 32, slot % 32] = 0x7E00
    got = r.run()
    want, tol = r.want()
    assert np.isnan(got[0, 4:, 32:]).all() and np.isfinite(got[0, :4]).all() and np.isfinite(got[0, 4:, :32]).all()
    assert np.isnan(got[1, :4]).all()
    want[1, :4] = np.nan
    close(got, want, np.where(np.isfinite(tol), tol, 1e-5))


def test_scores_of_minus_infinity_alone(dev, mem):
    rng = np.random.default_rng(13)
    r = Rows(rng, mem, dev, V.F16, [40], 2, 2, 32)
    r.q = np.abs(r.q) + np.float32(0.1)
    for j in range(40):
        p, slot = r.c.place(0, j)
        r.c.pool._values("k")[p, 0, slot // 32, R.place(V.F16, "k", 32, slot % 32, 3)] = 0xFC00
    got = r.run()
    want, tol = r.want()
    assert (got[0, 0] == 0).all()
    close(got[0, 1], want[0, 1], tol[0, 1])


def test_scales_of_far_sizes(dev, mem):
    """Q8_0 scales from the least subnormal to 60000, the great ones late, early and in turn."""
    rng = np.random.default_rng(14)
    for kind in ("up", "down", "turn"):
        r = Rows(rng, mem, dev, V.Q8_0, [600], 4, 1, 64, q_size=0.0)
        r.q[:] = (0.05 * rng.standard_normal(r.q.shape)).astype(np.float32)
        for j in range(600):
            p, slot = r.c.place(0, j)
            e = {"up": j / 600, "down": 1 - j / 600, "turn": (j % 7) / 7}[kind]
            for b in range(2):
                r.c.pool.scales("v")[p, 0, slot // 32, b * 32 + slot % 32] = np.float16(6e-8 * 1e12 ** e).view(np.uint16)
        close(r.run(), *r.want())


def test_offsets_past_32_bits(dev, mem):
    """A pool of more than 4 GiB a layer: pages at its end, and a second layer."""
    nkh, hd, page = 8, 256, 1024
    rng = np.random.default_rng(15)
    size = dev.page_bytes(V.F16, page, nkh, hd)
    n_pages = (1 << 32) // size + 3
    k, v = dev.alloc(2 * n_pages * size), dev.alloc(2 * n_pages * size)
    try:
        table = mem.up(np.array([[n_pages - 1], [n_pages - 2]], np.int32))
        pages = V.Pages(k, v, V.F16, page, n_pages, nkh, hd, table, 2, 1)
        n = 40
        x = {w: rng.standard_normal((2 * n, nkh * hd)).astype(np.float32) for w in "kv"}
        seq, at = np.repeat(np.arange(2), n).astype(np.int32), np.tile(np.arange(n), 2).astype(np.int32)
        ps, pa, px = mem.up(seq), mem.up(at), {w: mem.up(x[w]) for w in "kv"}
        q = rng.standard_normal((2, nkh * hd)).astype(np.float32)
        pq, po, pl = mem.up(q), mem.zeros(2 * nkh * hd), mem.up(np.full(2, n, np.int32))
        back = [mem.zeros(2 * n * nkh * hd) for _ in range(2)]
        for layer in (0, 1):
            dev.page_store(pages, layer, px["k"], px["v"], nkh * hd, ps, pa, 2 * n)
            dev.page_load(pages, layer, V.F32, *back, nkh * hd, ps, pa, 2 * n)
            held = {}
            for w, p in zip("kv", back):
                held[w] = R.held(V.F16, x[w]).reshape(2, n, nkh, hd)
                assert np.array_equal(dev.download(p, (2, n, nkh, hd), np.float32).astype(np.float64), held[w])
            dev.attention_paged(pages, layer, pq, nkh * hd, po, nkh * hd, 0, pl, 2, n, nkh, 1 / 16)
            got = dev.download(po, (2, nkh, hd), np.float32).astype(np.float64)
            for s in range(2):
                close(got[s], *R.attend(q[s].reshape(nkh, hd).astype(np.float64), held["k"][s], held["v"][s], 1 / 16))
    finally:
        dev.free(k)
        dev.free(v)


# ---- verification -------------------------------------------------------------------------------

class Draft:
    """One call; sequences whose decisions all lie further from a border than 1e-9 of what is compared (the 64-bit sums'
    order moves a border by less than vocab * 2^-52) have one right answer."""

    def __init__(self, rng, mem, dev, batch, n, vocab, temp, draft=True, pad=0, spread=2.0):
        self.__dict__.update(mem=mem, dev=dev, batch=batch, n=n, vocab=vocab, temp=temp, stride=vocab + pad)
        self.logits = (spread * rng.standard_normal((batch, n + 1, self.stride))).astype(np.float32)
        self.draft = (self.logits[:, :n] + rng.standard_normal((batch, n, self.stride)).astype(np.float32) * 0.7) if draft else None
        near = self.logits[:, :n, :vocab] + rng.gumbel(size=(batch, n, vocab)) * max(temp, 0.3)
        self.drafted = near.argmax(-1).astype(np.int32).reshape(batch, n)
        self.u = rng.random((batch, n + 1)).astype(np.float32)

    def run(self):
        up = self.mem.up
        self.po, self.pt = self.mem.zeros(self.batch + 1, np.int32), up(np.full(self.batch * (self.n + 1) + 1, 77, np.int32))
        self.args = (up(self.logits), self.stride, 0 if self.draft is None else up(self.draft), self.stride, up(self.drafted),
                     up(self.u), self.batch, self.n, self.vocab, self.temp, self.po, self.pt)
        self.dev.verify_draft(*self.args)
        return self.got()

    def got(self):
        a = self.dev.download(self.po, self.batch + 1, np.int32)
        t = self.dev.download(self.pt, self.batch * (self.n + 1) + 1, np.int32)
        assert a[-1] == 0 and t[-1] == 77
        return a[:-1], t[:-1].reshape(self.batch, self.n + 1)

    def check(self):
        accepted, tokens = self.run()
        for b in range(self.batch):
            d = None if self.draft is None else self.draft[b, :, :self.vocab]
            k, want, margin = R.verify(self.logits[b, :, :self.vocab], d, self.drafted[b], self.u[b], self.temp)
            if margin > 1e-9:
                assert (accepted[b], list(tokens[b])) == (k, want), (b, accepted[b], tokens[b], k, want, margin)
        return accepted, tokens


@pytest.mark.parametrize("batch,n,vocab,pad", [(1, 1, 2, 0), (3, 4, 1000, 3), (2, 7, 32000, 0), (5, 0, 4096, 0), (4, 64, 257, 1),
                                               (2, 3, 4097, 0), (1, 2, 131072, 0), (9, 5, 1, 0), (200, 3, 64, 2), (2, 2, 600001, 3)])
@pytest.mark.parametrize("temp", [0.0, 0.7, 1.5])
@pytest.mark.parametrize("draft", [True, False])
def test_verify(dev, mem, batch, n, vocab, pad, temp, draft):
    rng = np.random.default_rng(vocab + n)
    d = Draft(rng, mem, dev, batch, n, vocab, temp, draft, pad)
    accepted, _ = d.check()
    assert batch < 100 or len(set(accepted)) > 1  # both kinds of decision


def test_verify_short_drafts_and_random_numbers_at_the_ends(dev, mem):
    rng = np.random.default_rng(21)
    d = Draft(rng, mem, dev, 40, 4, 300, 0.9)
    d.drafted[0, 0], d.drafted[1, 2], d.drafted[2, 3], d.drafted[3, 1] = -1, 300, -2**31, 2**31 - 1
    d.u[4:8] = 0.0
    d.u[8:12] = np.float32(1 - 2.0 ** -24)
    d.check()


def test_verify_masked_logits(dev, mem):
    """Logits of -inf and of the type's lowest value; rows without a distribution; equal rows (nothing is left)."""
    rng = np.random.default_rng(22)
    low = np.finfo(np.float32).min
    for temp in (0.0, 1.0):
        for draft in (True, False):
            d = Draft(rng, mem, dev, 12, 3, 500, temp, draft)
            d.logits[0, :, 100:] = -np.inf
            d.logits[1, :, 100:] = low
            d.logits[2] = low                    # an even distribution
            d.logits[3, 1] = -np.inf             # none
            d.logits[4, 0, 7] = np.nan
            d.logits[5, 0, 7] = np.inf
            d.logits[6, 3, 499] = -np.inf
            d.logits[7, 2] = np.nan
            if draft:
                d.draft[8, 1, 3] = np.nan
                d.draft[9, 0] = -np.inf
                d.draft[10] = d.logits[10, :3]
                d.u[10, :3] = 1.0                # refused although equal: drawn from the target
            if temp:
                d.check()
                continue
            accepted, tokens = d.run()
            for b in range(12):
                if b == 5:
                    continue  # +inf is the greatest at temperature 0
                k, want, _ = R.verify(d.logits[b], None, d.drafted[b], d.u[b], 0.0)
                assert (accepted[b], list(tokens[b])) == (k, want), b


def test_verify_far_logits(dev, mem):
    """Logits of up to 1e4 and tiny temperatures: probabilities far below f32's range still add up in order."""
    rng = np.random.default_rng(23)
    Draft(rng, mem, dev, 8, 5, 2000, 1.0, spread=2000.0).check()
    Draft(rng, mem, dev, 8, 5, 2000, 1e-6).check()
    Draft(rng, mem, dev, 8, 5, 2000, 1e6).check()


# ---- together, and beside each other --------------------------------------------------------------

@TYPES
def test_a_serving_step(dev, mem, t):
    """q and k rotated, a prompt into pages, read back for the attention of several tokens, drafted tokens stored and
    attended as rows of their sequence, verified, the next step written over what was refused."""
    rng = np.random.default_rng(30)
    nqh, nkh, hd, page, past, n, vocab = 8, 2, 64, 32, 75, 4, 512
    kvd, qd = nkh * hd, nqh * hd
    c = Cache(rng, mem, dev, t, page, nkh, hd, 2, 4, layer=0).load()
    total = past + n
    x = {w: rng.standard_normal((total, kvd)).astype(np.float32) for w in "kv"}
    px = {w: mem.up(x[w]) for w in "kv"}
    seq, at = mem.up(np.ones(total, np.int32)), mem.up(np.arange(total, dtype=np.int32))
    dev.rope_axes(px["k"], kvd, 0, 0, 0, at, total, (hd // 2,), 0, 0, 0, 0, 0, nkh, nkh, hd, 10000.0)
    x["k"] = dev.download(px["k"], (total, kvd), np.float32)
    dev.page_store(c.pages, 0, px["k"], px["v"], kvd, seq, at, past)                                     # the prompt
    off = 4 * past
    dev.page_store(c.pages, 0, px["k"] + off * kvd, px["v"] + off * kvd, kvd, seq + off, at + off, n)    # the draft
    q = (2 * rng.standard_normal((n, qd))).astype(np.float32)
    pq, out = mem.up(q), mem.zeros(n * qd)
    dev.rope_axes(pq, qd, 0, 0, 0, at + off, n, (hd // 2,), 0, 0, 0, 0, 0, nqh, nkh, hd, 10000.0)
    q = dev.download(pq, (n, qd), np.float32)
    lens = mem.up(np.arange(past + 1, total + 1, dtype=np.int32))
    dev.attention_paged(c.pages, 0, pq, qd, out, qd, seq, lens, n, 128, nqh, 0.125)
    got = dev.download(out, (n, nqh, hd), np.float32).astype(np.float64)
    held = {w: R.held(t, x[w].reshape(total, nkh, hd)) for w in "kv"}
    for i in range(n):
        close(got[i], *R.attend(q[i].reshape(nqh, hd).astype(np.float64), held["k"][:past + 1 + i], held["v"][:past + 1 + i], 0.125))
    # the same from the contiguous cache of several tokens
    flat = {w: mem.zeros(total * kvd, np.uint16) for w in "kv"}
    dev.page_load(c.pages, 0, V.F16, flat["k"], flat["v"], kvd, seq, at, total)
    dev.attention_chunk(pq, qd, flat["k"], flat["v"], out, qd, n, past, 0, total, nqh, nkh, hd, 0.125)
    chunk = dev.download(out, (n, nqh, hd), np.float32).astype(np.float64)
    f16 = {w: S.half(dev.download(flat[w], (total, nkh, hd), np.uint16)) for w in "kv"}
    want, _, tol, _ = S.attend(q.reshape(n, nqh, hd).astype(np.float64), f16["k"], f16["v"], S.sees_chunk(n, past), 0.125, past)
    close(chunk, want, tol)
    d = Draft(rng, mem, dev, 1, n, vocab, 0.8)
    accepted, tokens = d.check()
    keep = past + int(accepted[0]) + 1
    again = rng.standard_normal((1, 2 * kvd)).astype(np.float32)
    pn = mem.up(again)
    dev.page_store(c.pages, 0, pn, pn + 4 * kvd, 2 * kvd, seq, mem.up(np.array([keep - 1], np.int32)), 1)
    held = {w: np.concatenate([held[w][:keep - 1], R.held(t, again.reshape(2, 1, nkh, hd)[i])]) for i, w in enumerate("kv")}
    dev.attention_paged(c.pages, 0, pq, qd, out, qd, seq, mem.up(np.array([keep], np.int32)), 1, 128, nqh, 0.125)
    close(dev.download(out, (nqh, hd), np.float32).astype(np.float64),
          *R.attend(q[0].reshape(nqh, hd).astype(np.float64), held["k"][:keep], held["v"][:keep], 0.125))


def test_captured_steps_and_two_graphs_at_once(dev, mem):
    """A step (store, attention over several splits, verification) replayed with new lengths and tokens, equal to the
    eager one; then graphs that use scratch replayed on two streams at once."""
    rng = np.random.default_rng(31)
    hip, stream = V.Hip(), dev.stream()
    r = Rows(rng, mem, dev, V.Q8_0, [900, 2000, 1], 8, 2, 64, junk=False, max_len=2048)
    first = r.run()
    d = Draft(rng, mem, dev, 3, 4, 9000, 0.8)
    d.run()
    new = mem.up(rng.standard_normal((3, 2 * 128)).astype(np.float32))
    at = mem.up(np.zeros(3, np.int32))

    def step():
        dev.page_store(r.c.pages, 1, new, new + 512, 256, 0, at, 3)
        r.call()
        dev.verify_draft(*d.args)

    graph = hip.capture(stream, step)
    try:
        for i in range(3):
            dev.write(r.pl, np.array([901 + i, 2001 + i, 2 + 40 * i], np.int32))
            dev.write(at, np.array([900 + i, 2000 + i, 1 + 40 * i], np.int32))
            dev.write(d.args[5], rng.random((3, 5)).astype(np.float32))
            for w in "kv":
                dev.write(r.c.ptr[w] + r.c.guard.nbytes, r.c.pool.bytes[w])
            hip.launch(graph, stream)
            dev.sync()
            a = (r.got(), *d.got())
            dev.write(r.po, r.out0)
            dev.write(d.pt, np.full(16, 77, np.int32))
            step()
            b = (r.got(), *d.got())
            assert all(np.array_equal(x, y) for x, y in zip(a, b))
    finally:
        hip.destroy(graph)
    dev.write(r.pl, r.lens)
    for w in "kv":
        dev.write(r.c.ptr[w] + r.c.guard.nbytes, r.c.pool.bytes[w])
    want = d.run()
    other = C.c_void_p()
    assert hip.h.hipStreamCreateWithFlags(C.byref(other), 1) == 0
    graphs = []
    try:
        graphs.append(hip.capture(stream, lambda: [r.call() for _ in range(8)]))
        graphs.append(hip.capture(stream, lambda: [dev.verify_draft(*d.args) for _ in range(8)]))
        for _ in range(5):
            dev.write(r.po, r.out0)
            dev.write(d.pt, np.full(16, 77, np.int32))
            hip.launch(graphs[0], stream)
            hip.launch(graphs[1], other.value)
            assert hip.h.hipStreamSynchronize(other) == 0
            dev.sync()
            assert np.array_equal(r.got(), first) and all(np.array_equal(x, y) for x, y in zip(d.got(), want))
    finally:
        for g in graphs:
            hip.destroy(g)
        hip.h.hipStreamDestroy(other)


def test_calls_of_several_threads(dev, mem):
    """Calls that share the library's scratch, from three threads: each gets its own result, the same every time."""
    rng = np.random.default_rng(32)
    rows = [Rows(rng, mem, dev, t, lens, 8, 2, 64, max_len=3000) for t, lens in ((V.Q8_0, [3000, 10]), (V.F16, [1500]))]
    want = [r.run() for r in rows]
    d = Draft(rng, mem, dev, 2, 3, 20000, 1.0)
    verified = d.run()
    failed = []

    def work(fn):
        try:
            for _ in range(30):
                fn()
        except Exception as e:  # noqa: BLE001
            failed.append(e)
    threads = [threading.Thread(target=work, args=(fn,)) for fn in (rows[0].call, rows[1].call, lambda: dev.verify_draft(*d.args))]
    for x in threads:
        x.start()
    for x in threads:
        x.join()
    dev.sync()
    assert not failed
    assert all(np.array_equal(r.got(), w) for r, w in zip(rows, want))
    assert all(np.array_equal(x, y) for x, y in zip(d.got(), verified))
