"""vbs_gfx950_verify_draft where many logits are equal, against its definition in 64 bits (pages_ref.py). No counterpart in
the reference: parity unpinned."""
import numpy as np
import pytest

from test_gpu_kernels import mem  # noqa: F401 (fixture)
from test_gpu_pages import Draft

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("vocab,pad", [(300, 0), (9001, 0), (9000, 1), (40961, 3)])
def test_greatest_logits_that_are_equal(dev, mem, vocab, pad):
    """Temperature 0: the lowest place among equals, wherever they lie: in a lane, over lanes, waves and chunks; NaN among
    them is never the greatest."""
    rng = np.random.default_rng(vocab)
    d = Draft(rng, mem, dev, 24, 4, vocab, 0.0, draft=False, pad=pad)
    d.logits = rng.integers(-1, 2, d.logits.shape).astype(np.float32)
    d.logits[3:6] = 0.0                     # all equal, signs of zero as they come
    d.logits[4] *= rng.choice([-1.0, 1.0], d.logits[4].shape).astype(np.float32)
    for b in range(6, 20):                  # two or three equal places above all others
        for i in range(5):
            d.logits[b, i, np.sort(rng.choice(vocab, 3, replace=False))[b % 2:]] = 5.0
    d.logits[20:22, :, ::2] = np.nan
    d.logits[22, :, :vocab - 1] = -np.inf
    d.logits[23, :, :vocab - 1] = np.nan
    best = np.array([[np.flatnonzero(x == np.nanmax(x))[0] for x in rows] for rows in d.logits[:, :4, :vocab]])
    d.drafted = np.where(rng.random(best.shape) < 0.8, best, rng.integers(0, vocab, best.shape)).astype(np.int32)
    accepted, _ = d.check()
    assert len(set(accepted)) > 2


@pytest.mark.parametrize("vocab,pad", [(4096, 0), (9001, 0)])
@pytest.mark.parametrize("draft", [True, False])
def test_even_distributions(dev, mem, vocab, pad, draft):
    """Every token as probable as any other, of all or of a part of the vocabulary: the token drawn is where u says, to the
    place."""
    rng = np.random.default_rng(vocab + 1)
    d = Draft(rng, mem, dev, 40, 2, vocab, 0.7, draft=draft, pad=pad)
    d.logits[:] = 3.0
    d.logits[::2, :, 1::3] = -np.inf
    if draft:
        d.draft[:] = 1.0
        d.draft[::3, :, :vocab // 2] = -np.inf
    d.drafted = rng.integers(0, vocab, d.drafted.shape).astype(np.int32)
    d.check()
