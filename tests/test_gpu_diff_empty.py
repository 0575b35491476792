"""Steps without a token under a bound that is not zero (a loop that passes the
longest chunk it takes)."""
import pytest
import torch

pytestmark = pytest.mark.gpu
D, BF = 128, torch.bfloat16


@pytest.mark.parametrize("paged", [False, True])
def test_prefill_without_tokens_under_a_bound(tm, dev, paged):
    e = torch.empty((0, 4, D), dtype=BF, device=dev)
    lam = torch.ones(2, device=dev)
    cu = torch.zeros(3, dtype=torch.int32, device=dev)
    kw = dict(max_seqlen=512)
    if paged:
        pool = torch.zeros((4, 16, 2, D), dtype=BF, device=dev)
        kw.update(k_pool=pool, v_pool=pool, prior_lens=cu[:2],
                  block_table=torch.zeros((2, 400), dtype=torch.int32,
                                          device=dev))
    k = None if paged else e[:, :2]
    out, lse = tm.prefill_diff_varlen(e, k, k, cu, lam, 0.1, **kw)
    assert out.shape == (0, 2, 256) and lse.shape == (4, 0)
