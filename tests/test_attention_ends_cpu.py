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


@pytest.mark.parametrize("q_rows, heads, kv", [(1 << 62, 8, 2), ((1 << 63) - 1, 2, 2), (1 << 31, 4, 4), ((1 << 61) + 4, 16, 2)])
def test_more_queries_than_64_bits_multiply_are_refused(q_rows, heads, kv):
    """Their product with the heads of a group wraps around to an allowed one."""
    n = ctypes.c_longlong()
    assert packed(q_rows=q_rows, heads=heads, kv=kv) == E_INVALID and "attend_packed" in error()
    assert _lib.lib().after_attend_packed_workspace(1, q_rows, 8, 1, heads, kv, 64, 0, ctypes.byref(n)) == E_INVALID
