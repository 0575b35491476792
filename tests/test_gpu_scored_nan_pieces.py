"""A key that is no number in one piece of a prefill whose keys are split over
work-groups: the queries that see it get NaN as outputs and LSE, the others their
results."""
import math

import pytest
import torch

from oracle import scored_ref as ref
from test_gpu_mx4 import Cache4
from test_gpu_scored import Cache, PAGE, _function, _gen, _i32, _packed

pytestmark = pytest.mark.gpu


NAMES = ["plain", "soft", "slopes", "cap slopes"]


@pytest.mark.parametrize("name,four", [(x, 0) for x in NAMES] +
                         [(x, 1) for x in NAMES + ["rel"]])
@pytest.mark.parametrize("at", [4000, 8999])
def test_no_number_in_one_piece(tm, dev, name, four, at):
    g = _gen(95)
    n, prior, window = 64, 9000, 9000 + 32 - at   # queries below 32 see it
    c = (Cache4(tm, [n + prior], 2, g, dev) if four else
         Cache([n + prior], 2, g, dev))
    q, _, _, cu = _packed([n], 16, 1, g, dev)
    p = _i32([prior], dev)
    kw = dict(_function(name, 16, g, dev), window=window)
    if name == "rel":
        kw["rel"] = torch.randn((n, 16, 700), generator=g).to(q)
    size = tm._lib.load().tmopt_attn_prefill_mx4_workspace_size
    if at == 4000:
        assert size(1, n, 0, 16, 2, c.table.shape[1], window) > 0
    want = ref.prefill(q, None, None, cu, 0.1, prior=p, k_pool=c.kp,
                       v_pool=c.vp, table=c.table, **kw)
    page, row = int(c.table[0, at // PAGE]), at % PAGE
    if four:
        c.pool[page, 0, 2048 + 16 * 2 + row] = 255      # block 2 of the key
        out, lse = tm.prefill_mx4_varlen(q, c.pool, c.table, cu, p, 0.1, **kw)
    else:
        c.kp[page, row, 0, 70] = math.nan
        out, lse = tm.prefill_scored_varlen(
            q, None, None, cu, 0.1, prior_lens=p, k_pool=c.kp, v_pool=c.vp,
            block_table=c.table, **kw)
    sees = torch.zeros((n, 16), dtype=torch.bool, device=dev)
    sees[:32, :8] = True
    assert torch.isnan(out[sees]).all() and torch.isnan(lse.T[sees]).all()
    # the others, within their bounds
    out, lse = out.clone(), lse.clone()
    out[sees], lse.T[sees] = want[0][sees].to(out), want[1].T[sees].to(lse)
    ref.check(out, lse, want, name)
