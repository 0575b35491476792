"""LSE row strides of the prefills' entry points (CPU: refused before a launch)."""
import ctypes

NULL, P = ctypes.c_void_p(0), ctypes.c_void_p(16)


def test_lse_strides(tm):
    """A negative LSE stride is refused by every entry point that takes one."""
    lib, e = tm._lib.load(), tm._lib
    assert lib.tmopt_attn_prefill_mx4_strided(
        P, 4096, 128, P, NULL, 2, 64, 0, P, P, 8, 16, 9, 32, 4, 128, 0, 0.1, 0.0,
        NULL, NULL, 0, 0, 0, P, 4096, 128, P, -1, NULL, NULL, 0,
        NULL) == e.TMOPT_EINVAL
    assert lib.tmopt_attn_prefill_scored_strided(
        P, 4096, 128, P, 512, 128, P, 512, 128, P, NULL, 2, 64, 0, NULL, NULL,
        NULL, 8, 16, 9, 32, 4, 128, 0, 0.1, 0.0, NULL, NULL, NULL, P, 4096, 128, P,
        -1, NULL, NULL, 0, NULL) == e.TMOPT_EINVAL
    assert lib.tmopt_attn_prefill_varlen_strided_split(
        P, 4096, 128, P, 0, 512, 128, 1, P, 0, 512, 128, 1, P, NULL, 2, 64, NULL,
        NULL, NULL, 0, 0, 16, 0, 32, 4, 128, 0, 0.1, NULL, 0, 0, 0, P, 4096, 128,
        P, -1, NULL, NULL, 0, NULL) == e.TMOPT_EINVAL
