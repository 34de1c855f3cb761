"""Rows in 8 bits, their products and drawn tokens without a GPU: bad arguments
are refused on the host before anything is launched, host tensors by the
wrappers."""
import pytest
import torch

from nativebit_amd import _lib, ops
from tests.conftest import gpu_available

P = 0x100000   # aligned, never dereferenced
F32, BF16 = _lib.NB_F32, _lib.NB_BF16
EINVAL, EUNSUP, EALIGN = _lib.NB_EINVAL, _lib.NB_EUNSUPPORTED, _lib.NB_EALIGN


def call(fn, base, kw):
    assert set(kw) <= set(base)
    return getattr(_lib.load(), fn)(*{**base, **kw}.values())


# Arguments that are taken end at the missing device; with one they would be launched.
no_gpu = pytest.mark.skipif(gpu_available(), reason="made-up addresses would reach a kernel")


QUANTIZE = dict(x=P, dtype=F32, ld=300, rows=4, width=300, codes=P, scale=P, stream=None)


@pytest.mark.parametrize("kw,status", [
    (dict(rows=-1), EINVAL), (dict(width=0), EINVAL), (dict(width=(1 << 24) + 1, ld=1 << 25), EUNSUP),
    (dict(rows=1 << 22), EUNSUP), (dict(x=None), EINVAL), (dict(dtype=_lib.NB_U8), EINVAL),
    (dict(ld=299), EINVAL), (dict(x=P + 2), EALIGN), (dict(codes=None), EINVAL),
    (dict(scale=None), EINVAL), (dict(scale=P + 2), EALIGN), (dict(dtype=BF16, x=P + 1), EALIGN),
])
def test_quantize_refuses(kw, status):
    assert call("nb_quantize8", QUANTIZE, kw) == status and _lib.last_error()


def test_nothing_to_do():
    assert call("nb_quantize8", QUANTIZE, dict(rows=0)) == 0
    assert call("nb_rmsnorm8", NORM, dict(rows=0)) == 0
    assert call("nb_linear8", LINEAR, dict(M=0)) == 0 and call("nb_linear8", LINEAR, dict(N=0)) == 0
    assert call("nb_linear8_layout", LAYOUT, dict(N=0)) == 0
    assert call("nb_sample", SAMPLE, dict(rows=0)) == 0


VALUES = dict(codes=P, scale=P, rows=4, width=300, out=P, dtype=F32, ld=300, stream=None)


@pytest.mark.parametrize("kw,status", [
    (dict(rows=-1), EINVAL), (dict(width=0), EINVAL), (dict(out=None), EINVAL), (dict(codes=None), EINVAL),
    (dict(scale=None), EINVAL), (dict(ld=299), EINVAL), (dict(dtype=2), EINVAL), (dict(out=P + 2), EALIGN),
    (dict(scale=P + 1), EALIGN), (dict(rows=1 << 22), EUNSUP),
])
def test_values_refuse(kw, status):
    assert call("nb_rows8_values", VALUES, kw) == status and _lib.last_error()


NORM = dict(x=P, dtype=F32, ld_x=300, residual=P + (1 << 20), ld_residual=300, sum=P + (2 << 20),
            ld_sum=300, weight=P, eps=1e-6, rows=4, width=300, codes=P, scale=P, stream=None)


@pytest.mark.parametrize("kw,status", [
    (dict(eps=-1.0), EINVAL), (dict(eps=float("nan")), EINVAL), (dict(eps=float("inf")), EINVAL),
    (dict(weight=None), EINVAL), (dict(weight=P + 2), EALIGN), (dict(residual=None), EINVAL),
    (dict(ld_residual=299), EINVAL), (dict(ld_sum=20), EINVAL), (dict(sum=P + 4), EINVAL),
    (dict(sum=P, ld_sum=400), EINVAL), (dict(sum=P + (1 << 20) + 400), EINVAL),
    (dict(residual=P + 2), EALIGN), (dict(sum=P + 2), EALIGN), (dict(rows=-1), EINVAL),
    (dict(dtype=7), EINVAL), (dict(codes=None), EINVAL), (dict(x=None), EINVAL),
])
def test_norm_refuses(kw, status):
    assert call("nb_rmsnorm8", NORM, kw) == status and _lib.last_error()


@no_gpu
def test_norm_in_place_is_taken():
    for kw in (dict(sum=P), dict(sum=P + (1 << 20)), dict(sum=None), dict(residual=None, sum=None)):
        assert call("nb_rmsnorm8", NORM, kw) == _lib.NB_ENODEV


LAYOUT = dict(packed=P, codebook=P, N=40, K=256, tiles=P, scale=P, stream=None)


@pytest.mark.parametrize("kw,status", [
    (dict(N=-1), EINVAL), (dict(K=0), EINVAL), (dict(K=200), EINVAL), (dict(K=(1 << 17) + 128), EUNSUP),
    (dict(N=1 << 20, K=1 << 16), EUNSUP), (dict(N=(1 << 24) + 1, K=128), EUNSUP), (dict(packed=None), EINVAL), (dict(codebook=None), EINVAL),
    (dict(tiles=None), EINVAL), (dict(scale=None), EINVAL), (dict(tiles=P + 8), EALIGN),
    (dict(packed=P + 2), EALIGN), (dict(scale=P + 1), EALIGN), (dict(codebook=P + 2), EALIGN),
])
def test_layout_refuses(kw, status):
    assert call("nb_linear8_layout", LAYOUT, kw) == status and _lib.last_error()


def test_sizes():
    lib = _lib.load()
    assert lib.nb_linear8_tiles_bytes(17, 256) == 2 * 2 * 896
    assert lib.nb_linear8_tiles_bytes(16, 128) == 896 and lib.nb_linear8_tiles_bytes(16, 100) == 0
    assert lib.nb_sample_ws_bytes(0, 100) == 0


LINEAR = dict(x=P, ld_x=256, x_scale=P, tiles=P, scale=P, bias=P, activation=0,
              residual=P + (1 << 20), ld_residual=40, y=P + (2 << 20), y_dtype=F32, ld_y=40, M=3, N=40,
              K=256, stream=None)


@pytest.mark.parametrize("kw,status", [
    (dict(M=-1), EINVAL), (dict(N=-1), EINVAL), (dict(K=100), EINVAL), (dict(K=0), EINVAL),
    (dict(M=(1 << 20) + 1), EUNSUP), (dict(K=1 << 18, ld_x=1 << 18), EUNSUP),
    (dict(activation=4), EINVAL), (dict(activation=-1), EINVAL), (dict(activation=3, N=41), EINVAL),
    (dict(x=None), EINVAL), (dict(x_scale=None), EINVAL), (dict(tiles=None), EINVAL),
    (dict(scale=None), EINVAL), (dict(y=None), EINVAL), (dict(ld_x=255), EINVAL), (dict(ld_x=264), EINVAL),
    (dict(ld_x=128), EINVAL), (dict(x=P + 8), EALIGN), (dict(tiles=P + 8), EALIGN),
    (dict(bias=P + 2), EALIGN), (dict(x_scale=P + 2), EALIGN), (dict(ld_y=39), EINVAL),
    (dict(y_dtype=_lib.NB_U8), EINVAL), (dict(ld_residual=39), EINVAL), (dict(y=P + (1 << 20) + 4), EINVAL),
    (dict(y=P + (1 << 20), ld_y=48), EINVAL), (dict(y=P + 2), EALIGN), (dict(ld_x=(1 << 22) + 16), EUNSUP),
    (dict(M=1 << 20, N=1 << 17), EUNSUP), (dict(N=(1 << 24) + 1), EUNSUP),
])
def test_linear_refuses(kw, status):
    assert call("nb_linear8", LINEAR, kw) == status and _lib.last_error()


@no_gpu
def test_linear_takes():
    for kw in (dict(y=P + (1 << 20)), dict(bias=None, residual=None), dict(activation=3, ld_y=20),
               dict(activation=3, N=40, ld_y=20, ld_residual=20)):
        assert call("nb_linear8", LINEAR, kw) == _lib.NB_ENODEV


SAMPLE = dict(logits=P, dtype=F32, ld=100, rows=3, V=100, u=P, temperature=P, top_k=P, top_p=P, min_p=P,
              tokens=P, logprobs=P, ws=P, ws_bytes=1 << 40, stream=None)


@pytest.mark.parametrize("kw,status", [
    (dict(rows=-1), EINVAL), (dict(V=0), EINVAL), (dict(V=(1 << 24) + 1, ld=1 << 25), EUNSUP),
    (dict(rows=65536), EUNSUP), (dict(logits=None), EINVAL), (dict(u=None), EINVAL),
    (dict(tokens=None), EINVAL), (dict(ld=99), EINVAL), (dict(dtype=2), EINVAL), (dict(u=P + 2), EALIGN),
    (dict(temperature=P + 1), EALIGN), (dict(top_k=P + 2), EALIGN), (dict(top_p=P + 2), EALIGN),
    (dict(min_p=P + 2), EALIGN), (dict(tokens=P + 2), EALIGN), (dict(logprobs=P + 2), EALIGN),
    (dict(logits=P + 2), EALIGN), (dict(ws=P + 8), EALIGN),
])
def test_sample_refuses(kw, status):
    assert call("nb_sample", SAMPLE, kw) == status and _lib.last_error()


def test_wrappers_refuse_host_tensors():
    x = torch.zeros(2, 128)
    w = ops.Weights8(torch.zeros(896, dtype=torch.uint8), torch.zeros(16), 16, 128)
    for f in (lambda: ops.quantize8(x), lambda: ops.Rows8(x.to(torch.int8), torch.ones(2)).values(),
              lambda: ops.rmsnorm8(x, torch.ones(128)),
              lambda: ops.linear8(ops.Rows8(x.to(torch.int8), torch.ones(2)), w),
              lambda: ops.linear8_layout(torch.zeros(768, dtype=torch.uint8), torch.zeros(16, 8), 16, 128),
              lambda: ops.sample(x, torch.zeros(2))):
        with pytest.raises(ValueError, match="GPU"):
            f()
