"""What the operators over the paged cache refuse, and why: checked on the host before a device is looked at, so also
without one (every call here is refused; nothing is launched), and the 64-bit oracle itself."""
import ctypes as C

import numpy as np
import pytest

import pages_ref as R
import vbs_gfx950 as V

P, P2, P3 = 0x10000000, 0x40000000, 0x70000000  # stand-ins for device memory: no refused call touches it
BIG = 0xFFFFFFFF
PAGES = dict(k=P, v=P2, type=V.Q8_0, page_slots=64, n_pages=10, n_kv_heads=2, head_dim=64, table=P, n_seqs=3,
             table_stride=4)
# changes of the pages that every operator refuses
BAD = [
    (dict(k=0), "null"), (dict(v=0), "null"), (dict(table=0), "null"), (dict(type=V.F32), "F16 or Q8_0"),
    (dict(type=V.Q4_0), "F16 or Q8_0"), (dict(page_slots=16), "power of two"), (dict(page_slots=96), "power of two"),
    (dict(page_slots=2048), "power of two"), (dict(page_slots=0), "power of two"), (dict(n_pages=0), "empty"),
    (dict(n_seqs=0), "empty"), (dict(table_stride=0), "empty"), (dict(n_kv_heads=0), "empty"),
    (dict(head_dim=0), "empty"), (dict(n_pages=1 << 31), "2.31"), (dict(n_seqs=BIG), "2.31"),
    (dict(n_kv_heads=65536), "65535"), (dict(head_dim=65), "even"), (dict(head_dim=258), "256"), (dict(k=P + 8), "aligned"),
    (dict(v=P2 + 2), "aligned"), (dict(v=P), "overlap"), (dict(v=P + 16), "overlap"),
    (dict(v=P + 10 * 2 * 2 * 2176 - 16), "overlap"), (dict(n_pages=(1 << 31) - 1, n_kv_heads=65535, page_slots=1024), "2.48")]


@pytest.fixture(scope="module")
def lib():
    return V.DeviceLib()


def pages(**change):
    return V.Pages(**{**PAGES, **change})


def refused(fn, args, why):
    with pytest.raises(V.GpuError, match=why):
        fn(**args)


STORE = dict(layer=0, k=P3, v=P3, kv_stride=128, seq=P3, at=P3, n=4)
LOAD = dict(STORE, out_type=V.F32)
ATT = dict(layer=0, q=P3, q_stride=256, out=P2, out_stride=256, seq=0, lens=P3, rows=3, max_len=256, nqh=4, scale=0.1)


@pytest.mark.parametrize("change,why", BAD)
def test_pages_refused(lib, change, why):
    for fn, args in ((lib.page_store, STORE), (lib.page_load, LOAD), (lib.attention_paged, ATT)):
        refused(fn, {**args, "pages": pages(**change)}, why)


def test_layers_beyond_an_address(lib):
    for fn, args in ((lib.page_store, STORE), (lib.page_load, LOAD), (lib.attention_paged, ATT)):
        refused(fn, {**args, "pages": pages(n_pages=1 << 20), "layer": BIG}, "2.48")


@pytest.mark.parametrize("change,why", [
    (dict(k=0), "null"), (dict(v=0), "null"), (dict(at=0), "null"), (dict(n=65536), "65535"), (dict(kv_stride=127), "stride")])
def test_rows_refused(lib, change, why):
    refused(lib.page_store, {**STORE, "pages": pages(), **change}, why)
    refused(lib.page_load, {**LOAD, "pages": pages(), **change}, why)


def test_load_type_refused(lib):
    for t in (V.Q8_0, -1, 7):
        refused(lib.page_load, {**LOAD, "pages": pages(), "out_type": t}, "F32 or F16")


@pytest.mark.parametrize("change,why", [
    (dict(q=0), "null"), (dict(out=0), "null"), (dict(lens=0), "null"), (dict(nqh=0), "empty"), (dict(nqh=3), "multiple"),
    (dict(nqh=34, q_stride=9999, out_stride=9999), "group"), (dict(rows=65536), "65535"), (dict(max_len=257), "max_len"),
    (dict(max_len=BIG), "max_len"), (dict(q_stride=255), "stride"), (dict(out_stride=255), "stride"), (dict(out=P3), "overlaps"),
    (dict(out=P3 + 4 * (2 * 256 + 255)), "overlaps"), (dict(out=P3 - 4), "overlaps")])
def test_attention_refused(lib, change, why):
    refused(lib.attention_paged, {**ATT, "pages": pages(), **change}, why)


def test_attention_sizes_refused(lib):
    wide = pages(n_kv_heads=1024, head_dim=2, table_stride=1 << 26)
    refused(lib.attention_paged, {**ATT, "pages": wide, "rows": 65535, "nqh": 8192, "q_stride": 16384, "out_stride": 16384},
            "2.28")
    refused(lib.attention_paged, {**ATT, "pages": pages(table_stride=1 << 26), "max_len": (1 << 31) + 1}, "2.31")


VERIFY = dict(logits=P, stride=100, draft=P2, draft_stride=100, drafted=P, u=P, batch=2, n=3, vocab=100, temperature=1.0,
              accepted=P3, tokens=P3)


@pytest.mark.parametrize("change,why", [
    (dict(logits=0), "null"), (dict(u=0), "null"), (dict(drafted=0), "null"), (dict(accepted=0), "null"),
    (dict(tokens=0), "null"), (dict(vocab=0), "empty"), (dict(vocab=(1 << 24) + 1), "2.24"), (dict(n=65), "64"),
    (dict(batch=65536), "65535"), (dict(stride=99), "stride"), (dict(draft_stride=99), "stride"),
    (dict(temperature=-0.5), "temperature"), (dict(temperature=float("nan")), "temperature"),
    (dict(temperature=float("inf")), "temperature")])
def test_verify_refused(lib, change, why):
    refused(lib.verify_draft, {**VERIFY, **change}, why)


def test_page_bytes(lib):
    for t in (V.F16, V.Q8_0):
        for page, nkh, hd in ((32, 1, 2), (64, 8, 128), (1024, 3, 80), (256, 65535, 256)):
            assert lib.page_bytes(t, page, nkh, hd) == R.page_bytes(t, page, nkh, hd)
    for args in ((V.F32, 64, 1, 64), (V.F16, 48, 1, 64), (V.F16, 16, 1, 64), (V.F16, 64, 0, 64), (V.F16, 64, 1, 63),
                 (V.F16, 64, 1, 258), (V.Q8_0, 64, 65536, 64)):
        assert lib.page_bytes(*args) == 0


def test_struct_layout():
    """Pages is vbs_gfx950_pages_t as the C compiler lays it out."""
    names = ("k", "v", "type", "page_slots", "n_pages", "n_kv_heads", "head_dim", "table", "n_seqs", "table_stride")
    assert [getattr(V.Pages, f).offset for f in names] == [0, 8, 16, 20, 24, 28, 32, 40, 48, 52]
    assert C.sizeof(V.Pages) == 56


# ---- the oracle ----------------------------------------------------------------------------------

@pytest.mark.parametrize("t", (R.F16, R.Q8_0))
@pytest.mark.parametrize("hd", (2, 32, 80, 256))
def test_layout_holds_every_place_once(t, hd):
    slot, d = np.meshgrid(np.arange(32), np.arange(R.nb(hd) * 32), indexing="ij")
    for w in "kv":
        assert sorted(R.place(t, w, hd, slot, d).reshape(-1)) == list(range(1024 * R.nb(hd)))


def test_quantise():
    q, d = R.quantise(np.array([[127.0, -63.5, 0.5, -0.5, 1.5] + [0.0] * 27], np.float32))
    assert d[0, 0] == 1 and list(q[0, :5]) == [127, -64, 0, 0, 2]  # ties to even
    for bad in (np.nan, np.inf, -np.inf, 127 * 65520.0):
        q, d = R.quantise(np.array([[1.0, bad]], np.float32))
        assert np.isnan(d).all()
    q, d = R.quantise(np.array([[1e-30, -1e-30]], np.float32))
    assert d[0, 0] == 0 and not q.any()
    assert np.isfinite(R.quantise(np.array([[127 * 65519.0]], np.float32))[1]).all()


def test_verify_gives_the_targets_distribution():
    """Over evenly spread random numbers, what stays and is drawn at the first place is distributed as the target."""
    rng = np.random.default_rng(3)
    logits, draft = rng.standard_normal((2, 5)).astype(np.float32), rng.standard_normal((1, 5)).astype(np.float32)
    p, q = R.softmax(logits[0], 0.7), R.softmax(draft[0], 0.7)
    m, got = 60, np.zeros(5)
    grid = (np.arange(m) + 0.5) / m
    for x in range(5):
        for a in grid:
            for b in grid:
                k, tok, _ = R.verify(logits, draft, [x], np.array([a, b]), 0.7)
                got[tok[0]] += q[x] / m ** 2
    assert np.abs(got - p).max() < 2 / m  # each of the two borders is met within a step of the grid


def test_verify_edges():
    lo = np.float32([[0, 1, 1, -np.inf], [0, 0, 0, 0]])
    assert R.verify(lo, None, [-1], np.float32([0, 0.0]), 1.0)[:2] == (0, [0, -1])
    assert R.verify(lo, None, [1], np.float32([0, 0.99]), 0.0)[:2] == (1, [1, 0])
    assert R.verify(lo, None, [2], np.float32([0, 0.5]), 0.0)[:2] == (0, [1, -1])  # ties: the lowest is the greatest
    assert R.verify(lo, None, [3], np.float32([0, 0.999]), 1.0)[:2] == (0, [2, -1])  # p = 0 never stays
    nan = np.float32([[np.nan, 1], [0, 0]])
    assert R.verify(nan, None, [1], np.float32([0, 0.5]), 1.0)[:2] == (0, [-1, -1])
