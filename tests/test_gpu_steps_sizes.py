"""Steps of several tokens over the f16 KV cache at sizes, head sizes and launches of their own: more ranges of slots than
a wave has lanes, offsets past 32 bits inside a layer, head sizes between the templates', graphs back to back. Against
the formulas in 64 bits (steps_ref.py)."""
import numpy as np
import pytest

import steps_ref as R
import vbs_gfx950 as V
from test_gpu_kernels import mem  # noqa: F401 (fixture)
from test_gpu_steps import Step, close, f16_bits, random_tree

pytestmark = pytest.mark.gpu


def check_chunk(s, see, **terms):
    """One call with a mass against the oracle: out, the mass of the slots in use, everything else as it was."""
    ref = {k: terms[k] for k in ("cap", "slopes") if k in terms}
    want, w, tol, wtol = s.want(see, **ref)
    total = s.past + s.n
    mass0 = np.random.default_rng(9).random((s.layers, s.nkh, s.max_ctx)).astype(np.float32)
    close(s.chunk(mass=mass0, **terms), want, tol)
    add, off = R.mass(w, wtol, s.nkh)
    exp = mass0.astype(np.float64)
    exp[s.layer, :, :total] += add
    full = np.zeros_like(exp)
    full[s.layer, :, :total] = off + 2 * R.F32 * exp[s.layer, :, :total]
    close(s.dev.download(s.pm, mass0.shape, np.float32).astype(np.float64), exp, full)


@pytest.mark.parametrize("n,past,nqh,nkh,hd", [
    (1, 10000, 4, 1, 64), (1, 16383, 16, 1, 128), (2, 16382, 6, 2, 40), (1, 20500, 2, 2, 96), (1, 40000, 3, 1, 32),
    (3, 16381, 16, 2, 64), (20, 9000, 2, 1, 128), (1, 9000, 2, 1, 250), (5, 10000, 4, 1, 256)])
def test_more_ranges_than_lanes(dev, mem, n, past, nqh, nkh, hd):
    """65 to 128 ranges of slots a row, and contexts whose ranges are longer for the limit of 128."""
    s = Step(np.random.default_rng(past), mem, dev, n, past, nqh, nkh, hd, layer=0, out_pad=3)
    check_chunk(s, R.sees_chunk(n, past), cap=12.0)


@pytest.mark.parametrize("hd", [130, 136, 160, 192, 200, 248, 254])
@pytest.mark.parametrize("n,past,nqh,nkh", [(1, 300, 4, 2), (9, 200, 3, 1), (40, 130, 4, 2), (100, 0, 2, 2)])
def test_head_sizes_between_128_and_256(dev, mem, hd, n, past, nqh, nkh):
    rng = np.random.default_rng(hd + n)
    s = Step(rng, mem, dev, n, past, nqh, nkh, hd, q_pad=4, out_pad=1)
    docs = np.sort(rng.integers(0, 3, past + n)).astype(np.int32)
    check_chunk(s, R.sees_chunk(n, past, 5, docs), docs=docs, prefix=5, slopes=np.linspace(0.3, 0.1, nqh).astype(np.float32))
    mask = random_tree(rng, n)
    want, _, tol, _ = s.want(R.sees_tree(n, past, mask))
    close(s.tree(mask), want, tol)


@pytest.mark.parametrize("n,past,nqh,nkh,hd", [(1, 25, 2, 1, 64), (7, 20, 4, 2, 128), (12, 18, 2, 2, 32), (30, 3, 4, 1, 96),
                                               (24, 10, 2, 1, 256), (20, 9, 3, 1, 40)])
def test_both_parts_of_q_and_of_the_weights(dev, mem, n, past, nqh, nkh, hd):
    """Few slots and small scores of eight dims (the others of q are 0 and add nothing), so that the bound of an f32 kernel
    is far below what a lost low part of q or of the weights would show: both are planted in the oracle, and seen."""
    rng = np.random.default_rng(n)
    s = Step(rng, mem, dev, n, past, nqh, nkh, hd, size=1.0)
    s.q.reshape(n, nqh, hd)[..., 8:] = 0
    s.scale = 0.25
    slots, group = past + n, nqh // nkh
    see = R.sees_chunk(n, past)
    k = np.repeat(R.half(s.kc[1, :slots]), group, 1)[..., :8]
    v = np.repeat(R.half(s.vc[1, :slots]), group, 1)
    q = s.q.reshape(n, nqh, hd)[..., :8].astype(np.float64)

    def attend(q, half_weights=False, v=v):
        sc = np.where(see[:, None], np.einsum("nhd,jhd->nhj", q, k) * s.scale, -np.inf)
        e = np.exp(sc - sc.max(-1, keepdims=True))
        total = e.sum(-1, keepdims=True)
        if half_weights:
            e = (e * 2048).astype(np.float16).astype(np.float64) / 2048
        return np.einsum("nhj,jhd->nhd", e / total, v)
    want = attend(q)
    # as steps_ref.attend, with 8 products a score
    score = np.where(see[:, None], np.einsum("nhd,jhd->nhj", q, k) * s.scale, np.nan)
    spread = np.nanmax(score, -1) - np.nanmin(score, -1)
    off = (R.SPLIT + 20 * R.F32) * s.scale * np.einsum("nhd,jhd->nhj", np.abs(q), np.abs(k)).max(-1) + (4 + 3 * spread) * R.F32
    size = attend(q, v=np.abs(v))
    tol = size * (2 * off[..., None] + R.SPLIT + (2 * slots + 8) * R.F32)
    close(s.chunk(), want, tol)
    wrong_q = q.astype(np.float16).astype(np.float64)
    assert (np.abs(attend(wrong_q) - want) > tol).any() and (np.abs(attend(q, True) - want) > tol).any()


def test_offsets_past_32_bits_inside_a_layer(dev, mem):
    """Slots whose elements lie past 2^32 of their layer, and a second layer behind them: stored by rope_axes, attended to
    (few rows and many, with the weights of slots), and cut by cache_evict in both layers."""
    rng = np.random.default_rng(6)
    nqh, nkh, hd = 16, 8, 256
    row = nkh * hd
    past = (1 << 32) // row + 500
    max_ctx, near = past + 100, 90  # the tokens' document holds `near` slots before them
    pk, pv = (dev.alloc(2 * row * 2 * max_ctx) for _ in range(2))
    try:
        for n in (1, 40):
            slots = past + n
            s = Step(rng, mem, dev, n, near, nqh, nkh, hd, layer=0)
            for x in (s.kc, s.vc):  # (below 2^-14 the cache's own rounding is not IEEE's)
                x[np.abs(R.half(x)) < 2.0 ** -14] = 0x3C00
            for p, rows in ((pk, s.kc), (pv, s.vc)):
                dev.write(p + 2 * row * (past - near), rows[0, :near])
            # the tokens' own rows, by rope_axes at position 0: k and v as they are
            k, v = (R.half(x[0, near:near + n]).reshape(n, row).astype(np.float32) for x in (s.kc, s.vc))
            dev.rope_axes(0, 0, mem.up(k), mem.up(v), row, mem.up(np.zeros((1, n), np.int32)), n, (hd // 2,), pk, pv, past, 0,
                          max_ctx, nqh, nkh, hd, 10000.0)
            for p, rows in ((pk, k), (pv, v)):
                assert np.array_equal(dev.download(p + 2 * row * past, (n, row), np.uint16), rows.astype(np.float16).view(np.uint16))
            docs = np.zeros(slots, np.int32)
            docs[past - near:] = 1
            pd, pm = mem.up(docs), mem.up(np.zeros((nkh, max_ctx), np.float32))
            want, w, tol, wtol = s.want(R.sees_chunk(n, near))
            s.load()
            dev.attention_chunk(s.pq, s.qs, pk, pv, s.po, s.os, n, past, 0, max_ctx, nqh, nkh, hd, s.scale, docs=pd, mass=pm)
            close(s.got(), want, tol)
            add, off = R.mass(w, wtol, nkh)
            m = dev.download(pm, (nkh, max_ctx), np.float32).astype(np.float64)
            close(m[:, past - near:slots], add, off + 2.0 ** -60)
            assert not m[:, :past - near].any() and not m[:, slots:].any()
        # layer 0 of 40 tokens more cut to 64 slots: the greatest weights, most of them past 2^32 elements, and the last 10
        slots, budget, last = past + 40, 64, 10
        at = np.sort(np.concatenate([rng.choice(past - near, 20, replace=False), past - near + rng.choice(near, 34, replace=False)]))
        weights = np.zeros((nkh, max_ctx), np.float32)
        weights[:, at] = 1 + rng.random((nkh, 54)).astype(np.float32)
        kept = np.concatenate([at, np.arange(slots - last, slots)])
        rows = f16_bits(rng, 2, budget, row)
        for j, i in enumerate(kept):
            dev.write(pk + 2 * row * int(i), rows[0, j])
            dev.write(pv + 2 * row * int(i), rows[1, j])
        pt = mem.zeros(nkh * budget, np.uint32)
        pw = mem.up(weights)
        dev.cache_evict(pk, pv, pw, pw, pt, slots, budget, 0, last, 0, 1, max_ctx, nkh, hd)
        assert (dev.download(pt, (nkh, budget), np.uint32) == kept).all()
        for p, r in ((pk, rows[0]), (pv, rows[1])):
            assert np.array_equal(dev.download(p, (budget, row), np.uint16), r)
        m = dev.download(pw, (nkh, max_ctx), np.float32)
        assert np.array_equal(m[:, :54], weights[:, at]) and not m[:, 54:].any()
        # layer 1: 300 slots to 100
        rows = f16_bits(rng, 2, 300, row)
        for p, r in ((pk, rows[0]), (pv, rows[1])):
            dev.write(p + 2 * row * max_ctx, r)
        weights = np.zeros((2, nkh, max_ctx), np.float32)
        weights[1, :, :300] = rng.random((nkh, 300)).astype(np.float32)
        pw, pt = mem.up(weights), mem.zeros(nkh * 100, np.uint32)
        dev.cache_evict(pk, pv, pw, 0, pt, 300, 100, 4, 20, 1, 1, max_ctx, nkh, hd)
        kept = dev.download(pt, (nkh, 100), np.uint32)
        gk, gv = (dev.download(p + 2 * row * max_ctx, (100, nkh, hd), np.uint16) for p in (pk, pv))
        for h in range(nkh):
            slots_h = R.evict(weights[1, h], 300, 100, 4, 20)
            assert np.array_equal(kept[h], slots_h)
            assert np.array_equal(gk[:, h], rows[0].reshape(300, nkh, hd)[slots_h, h])
            assert np.array_equal(gv[:, h], rows[1].reshape(300, nkh, hd)[slots_h, h])
    finally:
        dev.free(pk)
        dev.free(pv)


def test_graphs_back_to_back(dev, mem):
    """Graphs of attentions whose scratch differs, launched one behind the other in every order without a wait: each
    gives its eager out and mass."""
    rng = np.random.default_rng(31)
    hip, stream = V.Hip(), dev.stream()
    cases = []
    for n, past, nqh, nkh, hd, terms in ((1, 3000, 16, 4, 128, {"cap": 9.0}), (40, 500, 8, 2, 64, {}), (200, 700, 8, 4, 32, {"cap": 5.0}),
                                         (1, 16383, 4, 1, 64, {})):
        s = Step(rng, mem, dev, n, past, nqh, nkh, hd, layer=0)
        mass0 = np.zeros((1, nkh, s.max_ctx), np.float32)
        out = s.chunk(mass=mass0, **terms)
        mass = dev.download(s.pm, mass0.shape, np.float32)
        want, _, tol, _ = s.want(R.sees_chunk(n, past), **terms)
        close(out, want, tol)

        def call(s=s, terms=terms):
            dev.attention_chunk(s.pq, s.qs, s.pk, s.pv, s.po, s.os, s.n, s.past, 0, s.max_ctx, s.nqh, s.nkh, s.hd, s.scale,
                                mass=s.pm, **terms)
        cases.append((s, mass0, out, mass, hip.capture(stream, call)))
    try:
        for k in range(6):
            order = rng.permutation(len(cases))
            for s, mass0, _, _, _ in cases:
                dev.write(s.po, s.out0)
                dev.write(s.pm, mass0)
            for i in order:
                hip.launch(cases[i][4], stream)
            dev.sync()
            for s, mass0, out, mass, _ in cases:
                assert np.array_equal(s.got(), out), k
                assert np.array_equal(dev.download(s.pm, mass0.shape, np.float32), mass), k
    finally:
        for c in cases:
            hip.destroy(c[4])
