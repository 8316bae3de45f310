"""vbs_gfx950_attention_paged where the units of the rows are shared out over workgroups (more than 512 slots by max_len)
against its definition in 64 bits: no row with a slot, rows in many pieces, pieces that are not finite, every head size.
No counterpart in the reference (src/vbs_host_math.h:150-209 has one cache and one token): parity unpinned."""
import numpy as np
import pytest

import pages_long as L
import pages_ref as R
import vbs_gfx950 as V
from test_gpu_kernels import mem  # noqa: F401 (fixture)
from test_gpu_pages import TYPES, Rows
from test_gpu_steps import close

pytestmark = pytest.mark.gpu


# ---- no row with a slot -------------------------------------------------------------------------

# one row, rows that a wave looks up, more of them; the last with more rows x kv heads than workgroups
EMPTY = [(1, 1, 32), (1, 8, 128), (3, 2, 64), (64, 2, 32), (100, 1, 32), (300, 8, 32)]


@TYPES
@pytest.mark.parametrize("rows,nkh,hd", EMPTY)
def test_no_row_has_a_slot(dev, mem, t, rows, nkh, hd):
    """Every row empty (zeros), every row out of range (NaN), and both in one call: a step whose sequences are all
    padding. Pages hold NaN."""
    rng = np.random.default_rng(rows + nkh)
    r = Rows(rng, mem, dev, t, [0] * rows, nkh, nkh, hd, seq=np.arange(rows) % 4, max_len=2048)
    assert (r.run() == 0).all()
    for lens, seq in ((-1, 0), (2049, 0), (2**31 - 1, 3), (0, 4), (64, -1)):
        dev.write(r.pl, np.full(rows, lens, np.int32))
        dev.write(r.ps, np.full(rows, seq, np.int32))
        dev.write(r.po, r.out0)
        r.call()
        assert np.isnan(r.got()).all(), (lens, seq)
    lens = np.where(np.arange(rows) % 3 == 1, -7, 0).astype(np.int32)
    dev.write(r.pl, lens)
    dev.write(r.ps, r.seq)
    r.call()
    got = r.got()
    assert np.isnan(got[lens < 0]).all() and (got[lens == 0] == 0).all()


@TYPES
def test_a_captured_step_whose_rows_become_empty(dev, mem, t):
    """A graph replayed with lengths, without any, and with the lengths again: as the eager calls."""
    rng = np.random.default_rng(3)
    r = Rows(rng, mem, dev, t, [700, 33, 1025], 8, 2, 64, max_len=2048, junk=False)
    first = r.run()
    graph = V.Hip().capture(dev.stream(), r.call)
    try:
        for lens in ([0, 0, 0], r.lens, [0, -1, 5000], [0, 0, 0], r.lens):
            lens = np.asarray(lens, np.int32)
            dev.write(r.pl, lens)
            dev.write(r.po, r.out0)
            V.Hip().launch(graph, dev.stream())
            dev.sync()
            got = r.got()
            bad = (lens < 0) | (lens > 2048)
            assert np.isnan(got[bad]).all() and (got[lens == 0] == 0).all()
            if lens[2] == r.lens[2]:
                assert np.array_equal(got, first)
    finally:
        V.Hip().destroy(graph)


# ---- rows in many pieces ------------------------------------------------------------------------

@TYPES
@pytest.mark.parametrize("hd", [32, 160])
def test_batches_of_pieces_that_differ(dev, mem, t, hd):
    """One row in 683 (heads of 32) or 410 pieces, more than the merge takes at once: every piece's values and every
    batch's maximum differ, and a lost, repeated, moved or unscaled piece is seen (test_pages_long.py)."""
    row = L.LongRow(np.random.default_rng(hd), t, hd)
    order = np.random.default_rng(1).permutation(row.pages)
    pool = {}
    for w in "kv":
        x = np.empty_like(row.bytes[w])
        x[order] = row.bytes[w]
        pool[w] = mem.up(x)
    pages = V.Pages(pool["k"], pool["v"], t, L.PAGE, row.pages, 1, hd, mem.up(order.astype(np.int32)), 1, row.pages)
    out = mem.up(np.full(3 * hd, 7.5, np.float32))
    dev.attention_paged(pages, 0, mem.up(row.q), 2 * hd, out, 2 * hd, 0, mem.up(np.int32([L.SLOTS])), 1, L.SLOTS, 2, 1.0)
    got = dev.download(out, (3, hd), np.float32)
    assert (got[2] == 7.5).all()
    close(got[:2].astype(np.float64), *row.want(*row.parts()))


# ---- every head size and group ------------------------------------------------------------------

class Want:
    """The rows of a call by the formula, a sequence's slots read once."""

    def __init__(self, r):
        self.r, c = r, r.c
        long = {int(s): int(max(r.lens[r.seq == s].max(), 0)) for s in np.unique(r.seq)}
        self.kv = {s: [c.pool.rows(w, c.table[s], n) for w in "kv"] for s, n in long.items()}
        self.vmax = {}
        for s, n in long.items():
            self.vmax[s] = None
            if c.t == V.Q8_0 and n:
                d = c.pool.scales("v")[c.table[s, :-(-n // c.page)]].view(np.float16).astype(np.float64)
                self.vmax[s] = 127.0 * float(np.abs(d[np.isfinite(d)]).max())

    def __call__(self):
        out, tol = zip(*(self.row(i) for i in range(len(self.r.lens))))
        return np.array(out), np.array(tol)

    def row(self, i):
        r, s, n = self.r, int(self.r.seq[i]), int(self.r.lens[i])
        q = r.q[i, :r.nqh * r.hd].reshape(r.nqh, r.hd).astype(np.float64)
        return R.attend(q, self.kv[s][0][:n], self.kv[s][1][:n], r.scale, self.vmax[s])


SIZES = [(8, 2, 80, 0), (6, 2, 96, 0), (12, 4, 96, 2), (9, 1, 96, 0), (24, 2, 96, 0), (16, 1, 80, 0), (9, 1, 128, 0), (24, 2, 128, 0),
         (32, 2, 128, 6), (4, 1, 160, 0), (10, 1, 160, 0), (3, 3, 192, 0), (16, 1, 192, 2), (4, 2, 224, 0), (12, 1, 256, 0)]


@TYPES
@pytest.mark.parametrize("nqh,nkh,hd,pad", SIZES)
def test_long_rows_of_every_head_size(dev, mem, t, nqh, nkh, hd, pad):
    """Ragged rows in several pieces each, empty and short ones among them, shares that end with their head."""
    rng = np.random.default_rng(nqh + hd)
    r = Rows(rng, mem, dev, t, [1500, 0, 700, 33, 1101], nqh, nkh, hd, pad=pad, max_len=1536)
    got = r.run()
    close(got, *Want(r)())
    assert (got[1] == 0).all()


@TYPES
@pytest.mark.parametrize("rows,nqh,nkh,hd", [(130, 48, 4, 96), (70, 8, 8, 192), (40, 16, 16, 80), (100, 9, 3, 224), (130, 36, 4, 128)])
def test_shares_across_rows_of_every_head_size(dev, mem, t, rows, nqh, nkh, hd):
    """More rows x kv heads than workgroups: shares go on from head to head and row to row."""
    rng = np.random.default_rng(rows + hd)
    lens = rng.integers(0, 601, rows)
    lens[::17] = 600
    r = Rows(rng, mem, dev, t, lens, nqh, nkh, hd, seq=np.arange(rows) % 5, max_len=608)
    close(r.run(), *Want(r)())


# ---- pieces that are not finite -----------------------------------------------------------------

# A score of -inf or +inf for a q that is positive throughout, in kv head h: an element of K, or (Q8_0) the 32 of a block
# at 1 or -1 and their scale.
def infinite_k(c, seq, slots, h, sign):
    for j in slots:
        page, slot = c.place(seq, j)
        if c.t == V.F16:
            c.pool._values("k")[page, h, slot // 32, R.place(V.F16, "k", c.hd, slot % 32, 1)] = 0x7C00 if sign > 0 else 0xFC00
            continue
        c.pool._values("k")[page, h, slot // 32, R.place(V.Q8_0, "k", c.hd, slot % 32, np.arange(32))] = sign
        c.pool.scales("k")[page, h, slot // 32, slot % 32] = 0x7C00


# V's element 2 of kv head h; Q8_0: its block of 32, all of one sign.
def odd_v(c, seq, j, h, bits):
    page, slot = c.place(seq, j)
    if c.t == V.F16:
        c.pool._values("v")[page, h, slot // 32, R.place(V.F16, "v", c.hd, slot % 32, 2)] = bits
        return
    c.pool._values("v")[page, h, slot // 32, R.place(V.Q8_0, "v", c.hd, slot % 32, np.arange(32))] = 5
    c.pool.scales("v")[page, h, slot // 32, slot % 32] = bits


# rows, nqh, nkh, hd: six long rows alone (shares of four units, which end with their head), with one q head per kv head
# and with nine; and among 64 short rows of their sequences, in shares of 20 units that go on across rows
ODD = [(6, 4, 2, 64), (6, 18, 2, 64), (70, 8, 8, 64), (6, 10, 1, 160)]


@TYPES
@pytest.mark.parametrize("rows,nqh,nkh,hd", ODD)
def test_pieces_that_are_not_finite(dev, mem, t, rows, nqh, nkh, hd):
    """Infinities and NaN in the first, a middle and the last piece of long rows, joined with pieces that are finite."""
    rng = np.random.default_rng(rows + hd)
    lens = np.full(rows, 300)
    lens[::12 if rows > 6 else 1] = [2100, 2300, 2000, 2047, 2200, 1999]
    r = Rows(rng, mem, dev, t, lens, nqh, nkh, hd, seq=np.arange(rows) % 6 if rows == 6 else (np.arange(rows) + np.arange(rows) // 12) % 6,
             q_size=0.5, max_len=2304)
    long = {int(s): int(n) for s, n in zip(r.seq, r.lens) if n > 300}
    assert len(long) == 6
    r.q = np.abs(r.q) + np.float32(0.01)
    c, last = r.c, nkh - 1
    odd_v(c, 0, 3, 0, 0x7C00)                               # +inf in the first piece and in the last, -inf in the middle
    odd_v(c, 0, long[0] - 1, last, 0x7C00)
    odd_v(c, 1, 1100, 0, 0xFC00)
    infinite_k(c, 1, (0, 64, 1000, long[1] - 1), last, -1)  # weights 0
    infinite_k(c, 2, range(380, 1800), 0, -1)               # whole pieces of them, at either share
    odd_v(c, 3, long[3] - 1, 0, 0x7E00)                     # NaN
    infinite_k(c, 4, (1024,), 0, 1)                         # a score of +inf: the kv head's rows are NaN
    infinite_k(c, 5, range(long[5]), last, -1)              # nothing but -inf: 0
    nan_row = int(np.flatnonzero(r.seq == 3)[0])
    r.q[nan_row, hd - 1] = np.nan                           # one head
    got = r.run()
    want, tol = Want(r)()
    group = nqh // nkh
    reached = (r.seq == 4) & (r.lens > 1024)
    want[reached, :group] = np.nan
    want[nan_row, 0] = np.nan
    for i in np.flatnonzero(r.lens > 300):  # the inputs are what they are meant to be
        s = r.seq[i]
        assert np.isposinf(want[i, :group, 2]).all() if s == 0 else True
        assert np.isneginf(want[i, :group, 2]).all() if s == 1 else True
        assert np.isnan(want[i, (0 if i != nan_row else 1):group, 2]).all() if s == 3 else True
        assert (want[i, -group:] == 0).all() if s == 5 else True
        assert np.isfinite(want[i]).all() if s in (2, 5) else True
    # (where the bound itself is none, the value is an infinity or NaN, which `close` wants to be the same)
    close(got, want, np.where(np.isfinite(tol), tol, 0.0))


@TYPES
@pytest.mark.parametrize("rows,nqh,nkh,hd", ODD)
def test_pages_that_are_none_in_long_rows(dev, mem, t, rows, nqh, nkh, hd):
    """A table entry that is no page makes the rows that reach it NaN, in whichever piece it lies, and no others."""
    rng = np.random.default_rng(rows + hd + 1)
    lens = np.full(rows, 300)
    lens[::12 if rows > 6 else 1] = [2100, 2300, 2000, 2048, 2200, 1999]
    r = Rows(rng, mem, dev, t, lens, nqh, nkh, hd, seq=np.arange(rows) % 6 if rows == 6 else (np.arange(rows) + np.arange(rows) // 12) % 6,
             max_len=2304)
    want, tol = Want(r)()
    c = r.c
    lost = np.full(6, 1 << 30)  # the first slot without a page
    for s, entry, page in ((0, 0, -1), (1, 35, c.n_pages), (2, 2000 // 32, -2**31), (3, 2048 // 32, -1), (4, 70, 2**31 - 1)):
        c.table[s, entry] = page
        lost[s] = entry * 32
    got = r.run()
    bad = r.lens > lost[r.seq]
    assert bad.any() and not bad.all() and not bad[(r.seq == 3) | (r.seq == 4)].any()
    assert np.isnan(got[bad]).all()
    close(got[~bad], want[~bad], tol[~bad])


# ---- q of far sizes within a head ---------------------------------------------------------------

@TYPES
@pytest.mark.parametrize("lens", [[300], [1500, 64]], ids=["whole", "split"])
def test_small_elements_of_q_beside_great_ones(dev, mem, t, lens):
    """Elements 2^-24 of their head's greatest, that meet all of K (the great ones meet zeros), make scores of ordinary
    size. As two f16 parts with the greatest between 2^13 and 2^14 an element is off by half of the last step, 2^-25, so by
    2^-38 of the greatest: a score by that times scale sum |k|, a weight by twice the largest of these."""
    rng = np.random.default_rng(18)
    hd, nqh = 64, 4
    r = Rows(rng, mem, dev, t, lens, nqh, 1, hd, junk=False)
    for s, n in enumerate(lens):
        for j in range(n):
            x = rng.standard_normal((1, hd)).astype(np.float32)
            x[:, :32] = 0
            r.c.pool.put("k", *r.c.place(s, j), x)
    r.q = rng.standard_normal(r.q.shape).astype(np.float32).reshape(-1, nqh, hd)
    r.q[..., :32] *= 2.0 ** 10
    r.q[..., 32:] *= 2.0 ** -14
    r.q, r.scale = r.q.reshape(len(lens), -1), 2.0 ** 12
    got, want = r.run(), Want(r)
    got, want = r.run(), Want(r)
    plain, tol = want()
    for i, n in enumerate(lens):
        k, v = (x[:n, 0] for x in want.kv[i])
        for h in range(nqh):
            q = r.q[i].reshape(nqh, hd)[h].astype(np.float64)
            s = r.scale * (k @ q)
            assert s.std() > 0.5
            w = np.exp(s - s.max())
            off = 2.0 ** -38 * np.abs(q).max() * r.scale * np.abs(k).sum(1).max()
            tol[i, h] += 2 * off * ((w / w.sum()) @ np.abs(v))
            assert (tol[i, h] < 0.05 * np.abs(plain[i, h]).max()).all()
    close(got, plain, tol)
