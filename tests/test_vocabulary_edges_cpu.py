"""Refusals of the vocabulary entry points that need no GPU."""
import ctypes

import pytest

from memoryefficientclip_b200 import _lib, build


@pytest.fixture(scope="module")
def lib():
    build.build_library()
    return _lib.load()


def test_temperatures_without_a_finite_inverse_are_refused(lib):
    p, big = ctypes.c_void_p(0x1000), 1 << 30
    for t in (1e-39, 1e-45, 0.0, float("nan")):
        assert lib.meclip_token_log_probs(p, p, _lib.BF16, 4, 9, 8, 8, 8, t, p, 1, p, p, 0, None, None, p, p, p, big, None,
                                          None) == _lib.EINVAL
        assert lib.meclip_token_log_probs_grad(p, p, _lib.BF16, 4, 9, 8, 8, 8, t, p, 1, p, p, p, p, p, p, _lib.STORE_BF16, 8, p,
                                               _lib.STORE_BF16, 8, p, big, None, None) == _lib.EINVAL
        for student, teacher in ((t, 1.0), (1.0, t)):
            assert lib.meclip_distill(p, p, _lib.BF16, 4, 9, 8, 8, 8, student, p, p, _lib.F32, 2, teacher, 1, p, p, p, p, p, p,
                                      p, p, big, None, None) == _lib.EINVAL
