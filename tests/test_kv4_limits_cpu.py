"""The paged cache's refusals at the ends of its arguments' ranges."""
import ctypes

import pytest
import torch

from oumu_b200 import _lib, build, ops


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _lib.load()


P = ctypes.c_void_p(1 << 20)  # never dereferenced


@pytest.mark.parametrize("scale", [float("inf"), 3e38, -1.0, 0.0, float("nan")])
def test_scales_that_leave_no_logits_are_refused(lib, scale):
    assert lib.oumu_attn_decode_kv4(P, P, P, P, 1 << 24, P, None, P, 4, 16, 2, 128, 8, 8, scale, None) == _lib.ERR_INVALID
    assert lib.oumu_attn_decode_kv4_step(P, P, P, None, P, 1 << 24, None, None, 0, P, None, P, 4, 16, 2, 128, 8, 8, scale,
                                         None) == _lib.ERR_INVALID


@pytest.mark.parametrize("extra", [-1, 1 << 31, 1 << 32, (1 << 32) + 1])
def test_extends_by_more_than_an_int_are_refused(extra):
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    with pytest.raises(ValueError, match="extra"):
        ops.pages_extend(i32(2, 4), i32(8), i32(2), extra, i32(1))
