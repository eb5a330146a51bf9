"""Refusals of the sequence operators at the ends of what they take, at the C ABI (nothing is launched)."""
import ctypes

import pytest

from after_amd import _lib
from test_attention_cpu import E_INVALID, P, cache, error, packed


@pytest.mark.parametrize("scale", [2.4e38, -2.4e38, 3.4e38, float("inf"), float("-inf"), float("nan")])
def test_a_scale_whose_kernels_factor_is_not_finite_is_refused(scale):
    """The kernels multiply by scale x log2 e, in 32 bits."""
    assert packed(scale=scale) == E_INVALID and "scale" in error()
    L, c = _lib.lib(), ctypes.byref(cache(capacity=64))
    assert L.after_kv4_attend(c, bytes(_lib.KV4Query(P, P, P, 1 << 40, 256, 256, 64, 1, 4, 1, scale, 0, 1.0)), None) == E_INVALID and "scale" in error()
