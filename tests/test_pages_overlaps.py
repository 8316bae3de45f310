"""Results of the operators over the paged cache that would lie in what they read, or in each other: refused on the host
before a device is looked at (nothing is launched); and rows that lie beside each other, which are not."""
import numpy as np
import pytest

import pages_ref as R
import vbs_gfx950 as V
from test_gpu_kernels import mem  # noqa: F401 (fixture)
from test_pages_refusals import ATT, LOAD, P, P2, P3, PAGES, STORE, pages, refused

LAYER = 10 * 2 * 2 * 2176  # bytes of a layer's K, or V: pages, kv heads, units, bytes of a unit


@pytest.fixture(scope="module")
def lib():
    return V.DeviceLib()


def test_sizes():
    p = pages()
    assert LAYER == PAGES["n_pages"] * V.DeviceLib().page_bytes(p.type, p.page_slots, p.n_kv_heads, p.head_dim)


@pytest.mark.parametrize("name", ["k", "v"])
@pytest.mark.parametrize("at", [P, P + LAYER - 4, P2, P2 + LAYER - 4, P - 4 * (3 * 128 + 127), P2 - 4 * (3 * 128 + 127)])
def test_rows_in_the_pages(lib, name, at):
    other = {"k": P3, "v": P3 + (1 << 20)}
    refused(lib.page_store, {**STORE, **other, "pages": pages(), name: at}, "rows overlap the pages")
    refused(lib.page_load, {**LOAD, **other, "pages": pages(), name: at}, "rows overlap the pages")


def test_rows_in_another_layers_pages(lib):
    """It is the layer that the call works on that counts."""
    refused(lib.page_store, {**STORE, "pages": pages(), "layer": 3, "k": P + 3 * LAYER}, "rows overlap the pages")


@pytest.mark.parametrize("stride,apart", [(128, 0), (128, 4), (128, 127), (128, 128), (128, 3 * 128), (128, 3 * 128 + 127), (256, 0),
                                          (256, 64), (256, 192), (256, 3 * 256), (256, 2 * 256 + 129), (1000, 3 * 1000 - 127)])
@pytest.mark.parametrize("t", [V.F32, V.F16])
def test_loaded_rows_in_each_other(lib, stride, apart, t):
    size = 4 if t == V.F32 else 2
    for k, v in ((P3, P3 + size * apart), (P3 + size * apart, P3)):
        refused(lib.page_load, {**LOAD, "pages": pages(), "kv_stride": stride, "out_type": t, "k": k, "v": v}, "k and v overlap")


def test_out_in_the_pages(lib):
    for at in (P, P + LAYER - 4, P2 + LAYER - 4, P2 - 4 * (2 * 256 + 255)):
        refused(lib.attention_paged, {**ATT, "pages": pages(), "out": at}, "out overlaps the pages")
    refused(lib.attention_paged, {**ATT, "pages": pages(), "layer": 2, "out": P2 + 2 * LAYER}, "out overlaps the pages")


# batch 2, n 3, vocab 100, strides of 104: logits 8 rows, draft 6, drafted 6, u 8, accepted 2, tokens 8 words
L, D, X, U, A, T = (P3 + i * 0x10000 for i in range(6))
CALL = dict(logits=L, stride=104, draft=D, draft_stride=104, drafted=X, u=U, batch=2, n=3, vocab=100, temperature=1.0, accepted=A,
            tokens=T)


@pytest.mark.parametrize("change", [
    dict(tokens=X), dict(tokens=X + 20), dict(tokens=X - 28), dict(tokens=U), dict(tokens=U + 28), dict(tokens=L), dict(tokens=D),
    dict(tokens=L + 4 * (7 * 104 + 99)), dict(tokens=D + 4 * (5 * 104 + 99)), dict(tokens=A), dict(tokens=A + 4), dict(tokens=A - 28),
    dict(accepted=X), dict(accepted=X + 20), dict(accepted=U + 28), dict(accepted=L), dict(accepted=D - 4), dict(accepted=T + 28),
    dict(tokens=X, draft=0), dict(tokens=X, temperature=0.0), dict(tokens=U, n=0, drafted=0), dict(accepted=U + 4, n=0, drafted=0)])
def test_verified_in_the_arguments(lib, change):
    refused(lib.verify_draft, {**CALL, **change}, "results overlap")


@pytest.mark.gpu
@pytest.mark.parametrize("t", [V.F16, V.Q8_0], ids=["f16", "q8"])
@pytest.mark.parametrize("out", [V.F16, V.F32], ids=["to_f16", "to_f32"])
def test_rows_between_each_other(dev, mem, t, out):
    """k and v stored from and loaded into one array of fused rows, a layer's pages next to those of the other layer."""
    rng = np.random.default_rng(2)
    n, nkh, hd, page = 70, 2, 48, 32
    kvd, pool = nkh * hd, 3 * dev.page_bytes(t, page, nkh, hd)
    both = mem.zeros(4 * pool, np.uint8)  # K of two layers, then V of two
    p = V.Pages(both, both + 2 * pool, t, page, 3, nkh, hd, mem.up(np.int32([[2, 0, 1]])), 1, 3)
    x = rng.standard_normal((n, 2, nkh, hd)).astype(np.float32)
    px, at, seq = mem.up(x), mem.up(np.arange(n, dtype=np.int32)), mem.zeros(n, np.int32)
    dt = np.uint16 if out == V.F16 else np.float32
    rows = mem.up(np.full((n + 1, 2 * kvd), 5, dt))
    for layer in (0, 1):
        dev.page_store(p, layer, px, px + 4 * kvd, 2 * kvd, seq, at, n)
        dev.page_load(p, layer, out, rows, rows + np.dtype(dt).itemsize * kvd, 2 * kvd, seq, at, n)
        got = dev.download(rows, (n + 1, 2, nkh, hd), dt)
        want = R.held(t, x).astype(np.float32)
        assert np.array_equal(got[:n], R.half_store(want) if out == V.F16 else want) and (got[n] == 5).all()
