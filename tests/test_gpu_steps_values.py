"""Attention of several tokens (vbs_gfx950_attention_chunk, _attention_tree) where scores, caps or weights are far from
the usual: finite caches, so that the matrix-core path itself is seen. Against the formulas in 64 bits (steps_ref.py),
with bounds of their own that do not grow with the size of a score."""
import numpy as np
import pytest

import steps_ref as R
from test_gpu_kernels import mem  # noqa: F401 (fixture)
from test_gpu_steps import Step, close, random_tree

pytestmark = pytest.mark.gpu


def exact_scores(s, slots):
    """(n, heads, slots) of scale q.k in 64 bits, and sum |q k| scale."""
    q = s.q[:, :s.nqh * s.hd].reshape(s.n, s.nqh, s.hd).astype(np.float64)
    k = np.repeat(R.half(s.kc[s.layer, :slots]), s.nqh // s.nkh, 1)
    return np.einsum("nhd,jhd->nhj", q, k) * s.scale, np.einsum("nhd,jhd->nhj", np.abs(q), np.abs(k)) * abs(s.scale)


# ---- scores whose differences, but not whose sizes, an f32 exponent holds ------------------------------------------

FAR_SHAPES = [(1, 300, 4, 2, 128), (2, 1500, 4, 1, 64), (3, 90, 6, 2, 80), (16, 700, 2, 2, 128), (70, 40, 2, 2, 64),
              (40, 500, 4, 1, 128), (33, 200, 4, 2, 256), (20, 900, 3, 1, 40), (130, 5, 2, 1, 6)]


@pytest.mark.parametrize("shape", FAR_SHAPES, ids=["-".join(map(str, s)) for s in FAR_SHAPES])
@pytest.mark.parametrize("size", [1e3, 3e5, 1.1e7, 3e8, 1e9, 1e12, 1e30])
@pytest.mark.parametrize("sign", ["both", "below"])
def test_one_slot_takes_the_whole_weight(dev, mem, shape, size, sign):
    """Scores of `size`: where the greatest lies further above the second than f32 can be off, its V is the output, and 1
    is its weight. A score is off by at most SPLIT + (2 hd + 8) F32 of sum |q k| scale (steps_ref.attend); 40 beyond
    twice that the second's weight is below e^-40. The output is then V (f16) times a weight in two f16 parts over the same
    weight in f32: 2^-22, and a division and a product. Every third row keeps scores of the usual size."""
    n, past, nqh, nkh, hd = shape
    rng = np.random.default_rng([n, int(np.log10(size)), sign == "below"])
    s = Step(rng, mem, dev, *shape)
    slots = past + n
    if sign == "below":  # every score is negative
        s.q, k = np.abs(s.q) + 0.1, s.kc.view(np.float16)
        s.kc = (-np.abs(k) - np.float16(0.1)).astype(np.float16).view(np.uint16)
        s.kc[:, slots:] = 0x7E00
    usual = np.arange(n) % 3 == 2
    s.q[~usual] *= np.float32(size)
    score, total = exact_scores(s, slots)
    see = R.sees_chunk(n, past)
    score = np.where(see[:, None], score, -np.inf)
    order = np.sort(score, -1)
    off = (R.SPLIT + (2 * hd + 8) * R.F32) * np.where(see[:, None], total, 0).max(-1)
    clear = (order[..., -1] - order[..., -2] > 2 * off + 40) & ~usual[:, None]
    if n > 2:
        assert clear[~usual].mean() > 0.5  # (most rows say something)
    best = score.argmax(-1)
    group = nqh // nkh
    v = R.half(s.vc[s.layer, :slots])
    mass0 = np.zeros((2, nkh, s.max_ctx), np.float32)
    # a slot's weight of the rows that are not clear is anything from 0 to 1
    want_out, w, tol, wtol = s.want(see)
    want = np.stack([[v[best[i, h], h // group] for h in range(nqh)] for i in range(n)])
    low, high = np.zeros((nkh, slots)), np.zeros((nkh, slots))
    for i in range(n):
        for h in range(nqh):
            if usual[i]:
                low[h // group] += w[i, h] - wtol[i, h]
                high[h // group] += w[i, h] + wtol[i, h]
            elif clear[i, h]:
                low[h // group, best[i, h]] += 1 - 2.0 ** -20
                high[h // group, best[i, h]] += 1 + 2.0 ** -20
            else:
                high[h // group] += np.where(see[i], 1 + 2.0 ** -20, 0)
    for with_mass in (False, True):
        got = s.chunk(**({"mass": mass0} if with_mass else {}))
        assert np.isfinite(got).all()
        close(got[clear], want[clear], np.abs(want[clear]) * 2.0 ** -20)
        close(got[usual], want_out[usual], tol[usual])
        if with_mass:
            m = s.dev.download(s.pm, mass0.shape, np.float32)[1, :, :slots].astype(np.float64)
            slack = (n * group + 2) * R.F32 * high + 2.0 ** -60
            assert ((m >= low - slack) & (m <= high + slack)).all(), np.argwhere((m < low - slack) | (m > high + slack))[:4]
            # each row hands out a weight of 1 in all
            assert np.abs(m.sum(-1) - n * group).max() <= n * group * (2.0 ** -20 + slots * R.F32)
    mask = random_tree(rng, n)
    see = R.sees_tree(n, past, mask)
    seen = np.where(see[:, None], score, -np.inf)
    same = clear & (seen.argmax(-1) == best) & np.isfinite(seen.max(-1))
    if past:
        close(s.tree(mask)[same], want[same], np.abs(want[same]) * 2.0 ** -20)


@pytest.mark.parametrize("shape", [(1, 2100, 4, 2, 64), (5, 300, 6, 3, 128), (150, 400, 4, 2, 80), (90, 30, 2, 1, 256)])
@pytest.mark.parametrize("size", [1e5, 1e9])
def test_far_scores_in_documents_with_a_bias(dev, mem, shape, size):
    """As above with the slots of other documents unseen, a prefix, and a bias by distance, which adds 2 F32 of its size
    and of the score's to the bound."""
    n, past, nqh, nkh, hd = shape
    rng = np.random.default_rng([n, int(size)])
    s = Step(rng, mem, dev, *shape, size=2 * size)
    slots, group = past + n, nqh // nkh
    docs = rng.integers(0, 3, slots).astype(np.int32)
    slopes = np.linspace(0.5, 20.0, nqh).astype(np.float32)
    see = R.sees_chunk(n, past, past // 2, docs)
    score, total = exact_scores(s, slots)
    far = slopes[None, :, None] * np.abs(past + np.arange(n)[:, None] - np.arange(slots)[None])[:, None]
    off = np.where(see[:, None], (R.SPLIT + (2 * hd + 10) * R.F32) * total + 4 * R.F32 * far, 0).max(-1)
    score = np.where(see[:, None], score - far, -np.inf)
    order = np.sort(score, -1)
    clear = order[..., -1] - order[..., -2] > 2 * off + 40
    assert clear.mean() > 0.5
    best, v = score.argmax(-1), R.half(s.vc[s.layer, :slots])
    mass0 = np.zeros((2, nkh, s.max_ctx), np.float32)
    got = s.chunk(docs=docs, slopes=slopes, prefix=past // 2, mass=mass0)
    want = np.stack([[v[best[i, h], h // group] for h in range(nqh)] for i in range(n)])
    close(got[clear], want[clear], np.abs(want[clear]) * 2.0 ** -20)
    m = s.dev.download(s.pm, mass0.shape, np.float32)[1, :, :slots].astype(np.float64)
    low, high = np.zeros((nkh, slots)), np.zeros((nkh, slots))
    for i, h in np.ndindex(n, nqh):
        if clear[i, h]:
            low[h // group, best[i, h]] += 1 - 2.0 ** -20
            high[h // group, best[i, h]] += 1 + 2.0 ** -20
        else:
            high[h // group] += np.where(see[i], 1 + 2.0 ** -20, 0)
    slack = (n * group + 2) * R.F32 * high + 2.0 ** -60
    assert ((m >= low - slack) & (m <= high + slack)).all()


# ---- caps far above the scores ---------------------------------------------------------------------------------------

@pytest.mark.parametrize("shape", [(1, 300, 4, 2, 128), (3, 700, 2, 2, 80), (40, 200, 4, 1, 64), (90, 100, 4, 2, 128),
                                   (33, 70, 2, 1, 256)])
@pytest.mark.parametrize("cap", [2e12, 1e20, 1e30, 3e36, 3e37, 1.7e38, 3e38, 3.4028234e38])
@pytest.mark.parametrize("bias", [False, True])
def test_a_cap_far_above_every_score_changes_nothing(dev, mem, shape, cap, bias):
    """cap tanh(s / cap) is s to (s / cap)^2 / 3 of it, below F32 here. What may differ is a rounding of the score in
    either call (F32 of its size, which is below 100) and, with it, each weight by 4 F32 times that size at most."""
    n, past, nqh, nkh, hd = shape
    rng = np.random.default_rng(n)
    s = Step(rng, mem, dev, *shape, size=4.0)
    score, _ = exact_scores(s, past + n)
    assert np.abs(score).max() < 100
    terms = {"mass": np.zeros((2, nkh, s.max_ctx), np.float32)}
    if bias:
        terms["slopes"] = np.linspace(0.02, 0.01, nqh).astype(np.float32)
    plain, plain_mass = s.chunk(**terms), s.dev.download(s.pm, terms["mass"].shape, np.float32).astype(np.float64)
    got = s.chunk(cap=float(np.float32(cap)), **terms)
    rel = 4 * R.F32 * 100
    v = np.abs(R.half(s.vc[1, :past + n])).max((0, 2)).repeat(nqh // nkh)[None, :, None]
    assert (np.abs(got - plain) <= rel * v).all()
    m = s.dev.download(s.pm, terms["mass"].shape, np.float32).astype(np.float64)
    assert (np.abs(m - plain_mass) <= rel * plain_mass + 2.0 ** -80).all()


@pytest.mark.parametrize("shape", [(2, 300, 4, 2, 128), (70, 60, 2, 1, 64)])
@pytest.mark.parametrize("size,cap", [(1e12, 1e25), (1e12, 1e34), (1e25, 3.4e38)])
def test_far_scores_below_a_farther_cap(dev, mem, shape, size, cap):
    """Both calls take such rows in the same f32 products, and the cap leaves their scores as they are."""
    s = Step(np.random.default_rng(3), mem, dev, *shape, size=size)
    plain = s.chunk()
    assert np.isfinite(plain).all() and np.array_equal(s.chunk(cap=cap), plain)


@pytest.mark.parametrize("shape", [(2, 300, 4, 2, 128), (70, 60, 2, 1, 64)])
@pytest.mark.parametrize("cap", [1e-30, 1e-20, 1e-6])
@pytest.mark.parametrize("size", [1.0, 1e15, 1e30])
def test_caps_far_below_the_scores(dev, mem, shape, cap, size):
    """Every score lies within cap of 0: the weights are even, to e^(2 cap) and the rounding of the sums."""
    n, past, nqh, nkh, hd = shape
    s = Step(np.random.default_rng(4), mem, dev, *shape, size=size)
    got, slots = s.chunk(cap=cap), past + n
    v = R.half(s.vc[1, :slots])
    even = R.sees_chunk(n, past) / (past + 1.0 + np.arange(n))[:, None]
    want = np.einsum("nj,jhd->nhd", even, v).repeat(nqh // nkh, 1)
    size_v = np.einsum("nj,jhd->nhd", even, np.abs(v)).repeat(nqh // nkh, 1)
    close(got, want, size_v * (2 * cap + R.SPLIT + (2 * slots + 8) * R.F32))


# ---- many small weights beside a great one --------------------------------------------------------------------------

@pytest.mark.parametrize("n,past,nqh,nkh", [(132, 65536, 128, 8), (1, 16384, 300, 300)])
def test_many_small_weights(dev, mem, n, past, nqh, nkh):
    """One slot of V = 0 and past - 1 of e^-22.875 = 2^-33 of its weight with V = 1, in one range of slots (more row tiles
    than half the workgroups that share the work). A weight's low part is off by half of f16's least step, 2^-25,
    where the greatest weighs 2^11: 2^-36 for each slot; the sums lose a rounding a slot at most."""
    hd = 8
    s = Step(np.random.default_rng(1), mem, dev, n, past, nqh, nkh, hd, layer=0)
    s.q[:] = 0
    s.q.reshape(n, nqh, hd)[..., 0] = 1
    s.scale = 1.0
    k, v = np.zeros(s.kc.shape, np.float16), np.ones(s.vc.shape, np.float16)
    k[0, 0, :, 0], v[0, 0] = 22.875, 0
    k[0, past:, :, 0] = -60000  # the tokens themselves weigh nothing
    s.kc, s.vc = k.view(np.uint16), v.view(np.uint16)
    rest = (past - 1) * np.exp(-22.875)
    want = rest / (1 + rest)
    tol = past * 2.0 ** -36 + want * (past + 200) * R.F32
    assert want > 6 * tol
    assert np.abs(s.chunk() - want).max() <= tol


# ---- a scale that is no number --------------------------------------------------------------------------------------

@pytest.mark.parametrize("shape", [(1, 200, 4, 2, 128), (3, 60, 2, 2, 80), (70, 30, 4, 1, 64), (5, 0, 2, 1, 256)])
@pytest.mark.parametrize("scale", [float("nan"), float("inf"), float("-inf")])
def test_scales_that_are_no_numbers(dev, mem, shape, scale):
    """A NaN scale makes every seen score, row and weight NaN; an infinite one every row that has a score of +inf (all
    but by chance), and its weights. Rows that see nothing stay 0."""
    n, past, nqh, nkh, hd = shape
    rng = np.random.default_rng(n)
    s = Step(rng, mem, dev, *shape)
    s.scale = scale
    s.q[:, :nqh * hd] = np.abs(s.q[:, :nqh * hd]) + 0.1
    slots = past + n
    s.kc[1, slots - 1 if n == 1 else past, :, :] = np.array([2.0 if scale > 0 else -2.0], np.float16).view(np.uint16)[0]
    mass0 = np.zeros((2, nkh, s.max_ctx), np.float32)
    got = s.chunk(mass=mass0)
    assert np.isnan(got).all()
    m = s.dev.download(s.pm, mass0.shape, np.float32)
    assert (m[0] == 0).all() and (m[1, :, slots:] == 0).all()
    if np.isnan(scale):
        assert np.isnan(m[1, :, :slots]).all()
    else:
        assert np.isnan(m[1, :, past]).all()
    mask = np.zeros((n, (n + 63) // 64), np.uint64)
    got = s.tree(mask)
    assert (got == 0).all() if past == 0 else np.isnan(got).all() or not np.isnan(scale)


# ---- thetas below 1: the later pairs turn faster -------------------------------------------------------------------

@pytest.mark.parametrize("theta,far", [(0.5, 1 << 20), (2.0 ** -21, 300), (1.0, 1 << 30), (2.0 ** -21, 1 << 31), (3e38, 1000)])
def test_thetas_far_from_the_usual(dev, mem, theta, far):
    """The rotated pairs' elements within 3 F32 of their length (cosine and sine, products, sum; 3 sqrt 2 for the length
    itself) and the angle's own error: a position times a frequency that the
    oracle and the library each have to 2^-49, so |angle| 2^-48; where that is more than a turn, only the length holds
    (and the angle is that of the product in 64 bits, whatever its last bits)."""
    rng = np.random.default_rng(5)
    n, heads, hd, sec = 17, 4, 64, (8, 24)
    q = rng.standard_normal((n, heads * hd)).astype(np.float32)
    pos = rng.integers(-far // 2, far - 1, (2, n)).astype(np.int32)
    p = mem.up(q)
    dev.rope_axes(p, heads * hd, 0, 0, 0, mem.up(pos), n, sec, 0, 0, 0, 0, 0, heads, 1, hd, theta)
    got = dev.download(p, (n, heads, hd), np.float32).astype(np.float64)
    x = q.reshape(n, heads, hd).astype(np.float64)
    length = np.hypot(x[..., 0::2], x[..., 1::2])
    assert np.all(np.abs(np.hypot(got[..., 0::2], got[..., 1::2]) - length) <= 5 * R.F32 * length)
    t = float(np.float32(theta))
    freq = np.exp(-2.0 * np.arange(hd // 2) / hd * np.log(t))
    angle = np.abs(pos[np.repeat([0, 1], sec)].T * freq)[:, None]  # (n, 1, pairs)
    size = np.repeat(np.abs(x[..., 0::2]) + np.abs(x[..., 1::2]), 2, -1)
    close(got, R.rope_axes(x, pos, sec, t), size * (4 * R.F32 + np.repeat(np.minimum(angle * 2.0 ** -48, 2.0), 2, -1)))
