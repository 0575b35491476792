"""Scales that a relative bias over the 4-bit cache cannot be divided by (CPU: the
refusal comes before any launch)."""
import ctypes

import pytest

NULL, P = ctypes.c_void_p(0), ctypes.c_void_p(16)


@pytest.mark.parametrize("scale", [2.0 ** -61, 1e-30, 1e-38])
def test_bias_at_tiny_scales(tm, scale):
    lib, e = tm._lib.load(), tm._lib
    assert lib.tmopt_attn_decode_mx4(
        P, P, P, 8, 0, P, 4, 32, 4, 128, 16, 9, 0, scale, 0.0, NULL, P, 8, 4, 0,
        P, NULL, P, 1 << 40, NULL) == e.TMOPT_EINVAL
    for extra in ((), (0,)):
        fn = getattr(lib, "tmopt_attn_prefill_mx4" + "_strided" * len(extra))
        assert fn(P, 4096, 128, P, NULL, 2, 64, 0, P, P, 8, 16, 9, 32, 4, 128, 0,
                  scale, 0.0, NULL, P, 32 * 64, 64, 64, P, 4096, 128, NULL,
                  *extra, NULL, NULL, 0, NULL) == e.TMOPT_EINVAL
