"""What the operators for steps of several tokens refuse, and why: checked on the host before a device is looked
at, so also without one (every call here is refused; nothing is launched)."""
import ctypes as C

import numpy as np
import pytest

import vbs_gfx950 as V

P, P2 = 0x10000000, 0x20000000  # stand-ins for device memory: no refused call touches it
BIG = 0xFFFFFFFF


@pytest.fixture(scope="module")
def lib():
    return V.DeviceLib()


def refused(lib, fn, args, why):
    with pytest.raises(V.GpuError, match=why):
        fn(**args)


ROPE = dict(q=P, q_stride=256, k=P2, v=P2, kv_stride=128, pos=P, n=4, sections=(8, 8, 16), kc=P, vc=P2, slot=0,
            layer=0, max_ctx=16, nqh=4, nkh=2, hd=64, theta=10000.0)


@pytest.mark.parametrize("change,why", [
    (dict(pos=0), "null"), (dict(q=0, k=0, v=0, kc=0, vc=0), "null"), (dict(k=0), "null"), (dict(vc=0), "null"),
    (dict(nqh=0), "empty"), (dict(nkh=0), "empty"), (dict(hd=0), "empty"), (dict(n=65536, max_ctx=BIG), "65535"),
    (dict(slot=13), "max_ctx"), (dict(slot=BIG), "max_ctx"), (dict(nqh=5), "multiple"), (dict(hd=63), "even"),
    (dict(hd=258), "256"), (dict(sections=()), "axes"), (dict(sections=(8,) * 5), "axes"),
    (dict(sections=(8, 8, 8)), "sections"), (dict(sections=(8, 8, 17)), "sections"),
    (dict(sections=(BIG, 33)), "sections"), (dict(theta=0.0), "theta"), (dict(theta=float("nan")), "theta"),
    (dict(q_stride=255), "stride"), (dict(kv_stride=127), "stride"), (dict(nqh=34), "group")])
def test_rope_axes_refuses(lib, change, why):
    refused(lib, lib.rope_axes, {**ROPE, **change}, why)


ATT = dict(q=P, q_stride=256, kc=P, vc=P, out=P2, out_stride=256, n=4, past=10, layer=0, max_ctx=16, nqh=4, nkh=2, hd=64,
           scale=0.1)
ATT_BAD = [
    (dict(q=0), "null"), (dict(kc=0), "null"), (dict(vc=0), "null"), (dict(out=0), "null"), (dict(nqh=0), "empty"),
    (dict(nkh=0), "empty"), (dict(hd=0), "empty"), (dict(n=65536, max_ctx=BIG), "65535"), (dict(past=13), "max_ctx"),
    (dict(past=BIG), "max_ctx"), (dict(past=1 << 31, max_ctx=BIG), "2.31"), (dict(nqh=3), "multiple"), (dict(nqh=34), "group"), (dict(hd=65), "even"),
    (dict(hd=258), "256"), (dict(q_stride=255), "stride"), (dict(out_stride=255), "stride"), (dict(out=P), "overlaps"),
    (dict(out=P + 4 * 1023), "overlaps"), (dict(out=P - 4), "overlaps")]


@pytest.mark.parametrize("change,why", ATT_BAD)
def test_attention_refuses(lib, change, why):
    refused(lib, lib.attention_chunk, {**ATT, **change}, why)
    refused(lib, lib.attention_tree, {**ATT, "mask": P2, **change}, why)


def test_terms_and_mask(lib):
    refused(lib, lib.attention_tree, {**ATT, "mask": 0}, "null")
    for cap in (-1.0, float("nan"), float("inf"), 1e-31):
        refused(lib, lib.attention_chunk, {**ATT, "cap": cap}, "cap")


EV = dict(kc=P, vc=P2, mass=P, mass_out=P2, kept=P, n_len=100, budget=50, first=4, last=8, layer=0, n_layers=2,
          max_ctx=128, nkh=2, hd=64)


@pytest.mark.parametrize("change,why", [
    (dict(kc=0), "null"), (dict(vc=0), "null"), (dict(mass=0), "null"), (dict(kept=0), "null"), (dict(n_len=0), "empty"),
    (dict(budget=0), "empty"), (dict(n_layers=0), "empty"), (dict(nkh=0), "empty"), (dict(hd=0), "empty"),
    (dict(n_len=129), "max_ctx"), (dict(n_len=(1 << 31) + 1, max_ctx=BIG), "2.31"), (dict(budget=101), "budget"), (dict(first=43), "budget"), (dict(last=BIG), "budget"),
    (dict(n_layers=65536), "65535"), (dict(hd=7), "even"), (dict(hd=512), "256"), (dict(vc=P), "overlap"),
    (dict(vc=P + 2 * 2 * 128 * 2 * 64 - 2), "overlap"), (dict(mass_out=P + 4), "overlaps")])
def test_evict_refuses(lib, change, why):
    refused(lib, lib.cache_evict, {**EV, **change}, why)


def test_struct_layout():
    """AttnTerms is vbs_gfx950_attn_terms_t as the C compiler lays it out."""
    T = V.AttnTerms
    assert [getattr(T, f).offset for f in ("cap", "slopes", "docs", "prefix", "mass")] == [0, 8, 16, 24, 32]
    assert C.sizeof(T) == 40


def test_reference_helpers():
    """The 64-bit oracle itself: rows that see nothing, an even mix, the order of eviction."""
    import steps_ref as R
    q, k = np.ones((2, 1, 2)), np.zeros((3, 1, 2))
    v = np.array([[1.0, 2], [3, 4], [5, 6]])[:, None]
    see = np.array([[True, True, False], [False, False, False]])
    out, w, _, _ = R.attend(q, k, v, see, 1.0, 1)
    assert np.allclose(out[0, 0], [2, 3]) and (out[1] == 0).all() and np.allclose(w[0, 0], [0.5, 0.5, 0])
    nan = float("nan")
    assert list(R.evict(np.array([9.0, 1, nan, 1, -np.inf, 2, 0]), 7, 5, 1, 1)) == [0, 1, 3, 5, 6]
    assert list(R.evict(np.array([nan, -np.inf, nan]), 3, 2, 0, 0)) == [0, 1]


def test_sizes_beyond_a_launch(lib):
    """Shapes whose launches would pass 2^32 threads of a dimension."""
    wide = dict(n=65535, nqh=4112, nkh=257, hd=2, q_stride=8224, out_stride=8224, past=0, max_ctx=65535, out=1 << 50)
    refused(lib, lib.attention_chunk, {**ATT, **wide}, "2.28")
    refused(lib, lib.attention_tree, {**ATT, "mask": P2, **wide}, "2.28")
    refused(lib, lib.attention_chunk, {**ATT, "past": 1 << 26, "max_ctx": BIG, "mass": P}, "2.27")
    refused(lib, lib.cache_evict, {**EV, "n_layers": 4097, "nkh": 256}, "2.20")
