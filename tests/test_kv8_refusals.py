"""Calls of the serving operators that no correct result exists for, refused on
the host before anything is launched."""
import pytest

from nativebit_amd import _lib
from tests.conftest import gpu_available
from tests.test_serving_refusals import P, attention


@pytest.mark.parametrize("cap", [1.0001e20, 1e30, 3e38])
def test_attention_refuses_caps_without_range(cap):
    assert attention(softcap=cap) == _lib.NB_EINVAL and "softcap" in _lib.last_error()


def plan(**kw):
    a = dict(table=P, stride=4, lens=P + 256, new=P + 512, free=P + 768, state=P + 1024, R=3, width=4,
             n_blocks=20, n_tokens=5, max_len=100, slots=P + 1280, positions=P + 1536, chunks=P + 1792,
             lens_out=P + 2048, state_out=P + 2304, stream=None)
    return _lib.load().nb_kv_plan_max_len(*{**a, **kw}.values())


@pytest.mark.parametrize("kw,status", [
    (dict(max_len=-1), _lib.NB_EINVAL), (dict(R=0), _lib.NB_EINVAL), (dict(n_tokens=-1), _lib.NB_EINVAL),
    (dict(lens_out=P + 256), _lib.NB_EINVAL), (dict(slots=P + 1), _lib.NB_EALIGN),
])
def test_plan_max_len_refuses(kw, status):
    assert plan(**kw) == status and "nb_kv_plan_max_len" in _lib.last_error()
    if not gpu_available():
        assert plan() == _lib.NB_ENODEV
