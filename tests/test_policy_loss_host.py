"""Refusals of the policy loss's C entries around kept logits.  No GPU needed."""
import ctypes

import pytest


@pytest.fixture(scope="module")
def lib():
    from airgym_amd import _native
    return _native.load()


def test_kept_rows_are_for_float16_with_a_place_for_the_logits(lib):
    from airgym_amd import _native as N
    p = ctypes.cast((ctypes.c_float * 64)(), ctypes.c_void_p).value
    for dtype, dlogits in ((0, p), (1, p), (2, None)):
        a = N.AgTokenLossArgs(ctypes.sizeof(N.AgTokenLossArgs), dtype, 9, 1, 3, 27, 9, p, p, p, p, None, None, 0.2, 0.0, 0.0, p, p, dlogits, p,
                              1 << 20, p)
        assert lib.ag_token_policy_loss(ctypes.byref(a), None) == -1


def test_gradient_of_kept_logits_refuses(lib):
    p = ctypes.cast((ctypes.c_float * 64)(), ctypes.c_void_p).value
    good = [p, p, 3, 9, 2, p, None]
    for at, value, rc in ((0, None, -1), (1, None, -1), (5, None, -1), (2, 0, -1), (3, 0, -1), (4, 0, -6), (4, 1, -6), (4, 3, -6), (2, 1 << 31, -6),
                          (3, (1 << 30) + 1, -6)):
        args = list(good)
        args[at] = value
        assert lib.ag_token_policy_grad(*args) == rc, (at, value)
