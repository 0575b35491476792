"""Caps far above the scores, and scores above them (scored and 4-bit
attention): a score far below the cap stays what it is."""
import pytest
import torch

from oracle import scored_ref as ref
from test_gpu_scored import D, _gen, _rand
from test_gpu_scored_caps import _pages, _pages4, _prefill_of

pytestmark = pytest.mark.gpu

BIG = [256.0, 257.0, 1e3, 2048.0, 2049.0, 4000.0, 1e4, 1e6, 1e9, 1e20, 1e30]


def _one_far_key(g, dev, n, hq, hkv, z):
    """Keys of ordinary scores and one of score z."""
    q = _rand((n, hq, D), g, dev, 3.0)
    k = _rand((n, hkv, D), g, dev)
    q[:, :, 0] = 64.0
    k[:, :, 0] = 0.0
    k[5] = 0.0
    k[5, :, 0] = z / (64 * D ** -0.5)
    return q, k, _rand((n, hkv, D), g, dev)


@pytest.mark.parametrize("source", ["packed", "paged", "four"])
@pytest.mark.parametrize("cap", BIG)
@pytest.mark.parametrize("slopes", [0, 1])
def test_prefill_large_caps(tm, dev, source, cap, slopes):
    """Scores far below the cap stay what they are, also beside one that is not."""
    g = _gen(71)
    kw = dict(softcap=cap)
    if slopes:
        kw["slopes"] = (torch.rand(8, generator=g) * 0.1).to(dev)
    for z in (0.0, -0.8 * cap, 0.3 * cap, -0.01 * cap):
        q, k, v = _one_far_key(g, dev, 200, 8, 2, z)
        _prefill_of(tm, source, q, k, v, D ** -0.5, g, dev, **kw)


@pytest.mark.parametrize("four", [0, 1])
@pytest.mark.parametrize("cap", BIG)
def test_decode_large_caps(tm, dev, four, cap):
    g = _gen(72)
    for z in (0.0, -0.8 * cap, 0.3 * cap, -0.01 * cap):
        q, k, v = _one_far_key(g, dev, 500, 8, 2, z)
        q = q[:1]
        c = _pages4(tm, k, v, g, dev) if four else _pages(k, v, g, dev)
        if four:
            out, lse = tm.decode_mx4_paged(q, c.pool, c.table, c.ctx,
                                           D ** -0.5, softcap=cap)
        else:
            out, lse = tm.decode_scored_paged(q, c.kp, c.vp, c.table, c.ctx,
                                              D ** -0.5, softcap=cap)
        ref.check(out, lse, ref.decode(q, c.kp, c.vp, c.table, c.ctx,
                                       D ** -0.5, softcap=cap), f"{cap} {z}")
