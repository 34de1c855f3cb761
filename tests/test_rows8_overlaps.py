"""Rows in 8 bits, their products and drawn tokens without a GPU: outputs that overlap
an input or one another are refused, neighbours and columns of one array are not."""
import pytest

from nativebit_amd import _lib
from tests.conftest import gpu_available

P = 0x100000   # aligned, never dereferenced
MB = 1 << 20
F32, BF16 = _lib.NB_F32, _lib.NB_BF16
pytestmark = pytest.mark.skipif(gpu_available(), reason="made-up addresses could reach a kernel")


def call(fn, base, kw):
    assert set(kw) <= set(base)
    return getattr(_lib.load(), fn)(*{**base, **kw}.values())


# 4 rows of 300: 4800 bytes of x, 1200 of codes, 16 of scales
QUANTIZE = dict(x=P, dtype=F32, ld=300, rows=4, width=300, codes=P + MB, scale=P + 2 * MB, stream=None)
QUANTIZE_BAD = [dict(codes=P), dict(codes=P + 4799), dict(codes=P - 1199), dict(scale=P), dict(scale=P + 4796),
                dict(scale=P - 12), dict(scale=P + MB), dict(scale=P + MB + 1196), dict(scale=P + MB - 12),
                dict(ld=400, codes=P + 1600), dict(ld=400, codes=P + 1200), dict(ld=400, scale=P + 1588),
                dict(dtype=BF16, codes=P + 2399)]
QUANTIZE_OK = [{}, dict(codes=P + 4800), dict(codes=P - 1200), dict(scale=P + 4800), dict(scale=P - 16),
               dict(scale=P + MB + 1200), dict(ld=400, scale=P + 1200), dict(ld=400, scale=P + 1584),
               dict(dtype=BF16, codes=P + 2400), dict(rows=1, codes=P + 1200)]
VALUES = dict(codes=P, scale=P + MB, rows=4, width=300, out=P + 2 * MB, dtype=F32, ld=300, stream=None)
VALUES_BAD = [dict(out=P), dict(out=P + 1196), dict(out=P - 4796), dict(out=P + MB), dict(out=P + MB - 4796),
              dict(out=P + MB - 1196, ld=400)]
VALUES_OK = [{}, dict(out=P + 1200), dict(out=P - 4800), dict(out=P + MB + 16), dict(out=P + MB - 1200, ld=400)]
# 3 rows of 256 codes, 40 outputs: 3 x 2 tiles of 896 bytes
LINEAR = dict(x=P, ld_x=256, x_scale=P + MB, tiles=P + 2 * MB, scale=P + 3 * MB, bias=P + 4 * MB, activation=0,
              residual=None, ld_residual=0, y=P + 5 * MB, y_dtype=F32, ld_y=40, M=3, N=40, K=256, stream=None)
LINEAR_BAD = [dict(y=P), dict(y=P + 764), dict(y=P - 476), dict(y=P + MB), dict(y=P + MB - 476), dict(y=P + MB + 8),
              dict(y=P + 2 * MB + 5372), dict(y=P + 2 * MB - 476), dict(y=P + 3 * MB + 156), dict(y=P + 4 * MB + 156),
              dict(y=P + 4 * MB - 476), dict(x=P, ld_x=512, y=P + 252, ld_y=128),
              dict(y=P + 4 * MB + 156, y_dtype=BF16)]
LINEAR_OK = [{}, dict(y=P + 768), dict(y=P - 480), dict(y=P + MB + 12), dict(y=P + 2 * MB + 5376),
             dict(y=P + 3 * MB + 160), dict(y=P + 4 * MB + 160), dict(bias=None, y=P + 4 * MB),
             dict(x=P, ld_x=512, y=P + 256, ld_y=128), dict(residual=P + 5 * MB, ld_residual=40)]
LAYOUT = dict(packed=P, codebook=P + MB, N=40, K=256, tiles=P + 2 * MB, scale=P + 3 * MB, stream=None)
LAYOUT_BAD = [dict(tiles=P), dict(tiles=P + 3824), dict(tiles=P + MB + 2544), dict(scale=P + 3836),
              dict(scale=P + MB + 2556), dict(scale=P + 2 * MB), dict(scale=P + 2 * MB + 5372)]
LAYOUT_OK = [{}, dict(tiles=P + 3840), dict(tiles=P + MB + 2560), dict(scale=P + 3840), dict(scale=P + 2 * MB + 5376)]
SAMPLE = dict(logits=P, dtype=F32, ld=100, rows=3, V=100, u=P + MB, temperature=P + MB, top_k=P + MB, top_p=P + MB,
              min_p=P + MB, tokens=P + 2 * MB, logprobs=P + 3 * MB, ws=P + 4 * MB, ws_bytes=1 << 40, stream=None)
SAMPLE_BAD = [dict(tokens=P), dict(tokens=P + 1196), dict(logprobs=P + 4), dict(ws=P), dict(ws=P + 1184),
              dict(tokens=P + 3 * MB), dict(tokens=P + 3 * MB + 8), dict(logprobs=P + 4 * MB), dict(tokens=P + MB),
              dict(tokens=P + MB + 8), dict(ld=200, tokens=P + 396)] + [
    {name: P + at, other: P + at} for name, at in (("tokens", 5 * MB), ("logprobs", 5 * MB), ("ws", 5 * MB))
    for other in ("u", "temperature", "top_k", "top_p", "min_p")]
SAMPLE_OK = [{}, dict(tokens=P + 1200), dict(tokens=P + MB + 12), dict(ld=200, tokens=P + 400),
             dict(tokens=P + 3 * MB + 12), dict(logprobs=None), dict(top_k=None, tokens=P + 4 * MB - 12)]
ALL = [("nb_quantize8", QUANTIZE, QUANTIZE_BAD, QUANTIZE_OK), ("nb_rows8_values", VALUES, VALUES_BAD, VALUES_OK),
       ("nb_linear8", LINEAR, LINEAR_BAD, LINEAR_OK), ("nb_linear8_layout", LAYOUT, LAYOUT_BAD, LAYOUT_OK),
       ("nb_sample", SAMPLE, SAMPLE_BAD, SAMPLE_OK)]


@pytest.mark.parametrize("fn,base,kw", [(fn, base, kw) for fn, base, bad, _ in ALL for kw in bad])
def test_overlaps_are_refused(fn, base, kw):
    assert call(fn, base, kw) == _lib.NB_EINVAL and "overlap" in _lib.last_error()


@pytest.mark.parametrize("fn,base,kw", [(fn, base, kw) for fn, base, _, ok in ALL for kw in ok])
def test_neighbours_are_taken(fn, base, kw):
    assert call(fn, base, kw) == _lib.NB_ENODEV
