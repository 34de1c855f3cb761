"""Calls of the serving operators that no correct result exists for, refused on
the host before anything is launched."""
import pytest

from nativebit_amd import _lib
from tests.test_serving_refusals import attention


@pytest.mark.parametrize("cap", [1.0001e20, 1e30, 3e38])
def test_attention_refuses_caps_without_range(cap):
    assert attention(softcap=cap) == _lib.NB_EINVAL and "softcap" in _lib.last_error()
