"""What an entry that names no page means, by the entry point: the decode's keys
are absent, the prefill's are zero rows (as in the plain pair). The same table,
the same token through both."""
import pytest
import torch

from oracle import diff_ref

pytestmark = pytest.mark.gpu
D, PAGE, BF = 128, 16, torch.bfloat16


@pytest.mark.parametrize("n", [100, 3000])
@pytest.mark.parametrize("window", [0, 40])
def test_missing_page_in_both(tm, dev, n, window):
    g = torch.Generator().manual_seed(n)
    hq, hkv, pages = 16, 4, -(-n // PAGE)
    rand = lambda *s: torch.randn(s, generator=g).to(BF).to(dev)   # noqa: E731
    kp, vp = rand(pages + 1, PAGE, hkv, D), rand(pages + 1, PAGE, hkv, D)
    kp[pages] = vp[pages] = 0
    table = torch.randperm(pages, generator=g).int()[None].to(dev)
    q = rand(1, hq, D)
    lam = torch.full((hq // 2,), 0.4, device=dev)
    ctx = torch.tensor([n], dtype=torch.int32, device=dev)
    cu = torch.tensor([0, 1], dtype=torch.int32, device=dev)

    def both(t):
        o, l = tm.decode_diff_paged(q, kp[:pages], vp[:pages], t, ctx, lam,
                                    0.1, window=window)
        o2, l2 = tm.prefill_diff_varlen(
            q, None, None, cu, lam, 0.1, window=window, max_seqlen=1,
            prior_lens=ctx - 1, k_pool=kp[:pages], v_pool=vp[:pages],
            block_table=t)
        return (o, l.T), (o2, l2)
    at, pos = torch.tensor([n - 1], device=dev), torch.arange(n, device=dev)
    gone = pages - 2                      # (inside the window)

    def want(t, keys):
        return diff_ref.attend(q, diff_ref.rows_of(kp, t[0], keys),
                               diff_ref.rows_of(vp, t[0], keys), at, keys, lam,
                               0.1, window=window)
    for out, lse in both(table):
        diff_ref.check(out, lse, want(table, pos), "all there")
    hole, zero = table.clone(), table.clone()
    hole[0, gone], zero[0, gone] = -1, pages
    decode, prefill = both(hole)
    diff_ref.check(*decode, want(zero, pos[pos // PAGE != gone]), "absent")
    diff_ref.check(*prefill, want(zero, pos), "zeros")
    # a page wholly before the window is neither
    if window:
        hole = table.clone()
        hole[0, 0] = -1
        for out, lse in both(hole):
            diff_ref.check(out, lse, want(table, pos), "before the window")
