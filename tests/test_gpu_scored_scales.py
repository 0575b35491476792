"""Softmax scales far from one (scored and 4-bit attention)."""
import pytest
import torch

from oracle import scored_ref as ref
from test_gpu_mx4 import Cache4
from test_gpu_scored import Cache, _gen, _i32, _packed, _rand

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("scale,cap", [(1e-38, 0.0), (1e-37, 0.0), (1e-20, 0.0),
                                       (1e-9, 0.0), (1e9, 0.0), (1e-20, 3.0),
                                       (1e-9, 3.0), (1e9, 3.0)])
@pytest.mark.parametrize("bias", [1, 0])
def test_scales(tm, dev, scale, cap, bias):
    g = _gen(97)
    kw = dict(softcap=cap)
    if bias:
        kw["slopes"] = (torch.rand(8, generator=g) * 0.3 - 0.05).to(dev)
    lens, prior = [150, 20], [60, 0]
    q, k, v, cu = _packed(lens, 8, 2, g, dev)
    got = tm.prefill_scored_varlen(q, k, v, cu, scale, **kw)
    ref.check(*got, ref.prefill(q, k, v, cu, scale, **kw), "packed")
    p, ends = _i32(prior, dev), [a + b for a, b in zip(lens, prior)]
    c = Cache4(tm, ends, 2, g, dev)
    pools = dict(k_pool=c.kp, v_pool=c.vp, table=c.table)
    got = tm.prefill_mx4_varlen(q, c.pool, c.table, cu, p, scale, **kw)
    ref.check(*got, ref.prefill(q, None, None, cu, scale, prior=p, **pools,
                                **kw), "4 bits")
    q = q[:2].contiguous()
    want = ref.decode(q, c.kp, c.vp, c.table, c.ctx, scale, **kw)
    ref.check(*tm.decode_mx4_paged(q, c.pool, c.table, c.ctx, scale, **kw),
              want, "decode, 4 bits")
    ref.check(*tm.decode_scored_paged(q, c.kp, c.vp, c.table, c.ctx, scale,
                                      **kw), want, "decode")
