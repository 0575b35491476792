"""Bytes that no key of a request owns never show in its results (4-bit cache)."""
import pytest
import torch

from test_gpu_mx4 import Cache4, _gen, _rand

pytestmark = pytest.mark.gpu
D, PAGE = 128, 16


@pytest.mark.parametrize("window", [0, 37])
@pytest.mark.parametrize("kw", [dict(softcap=5.0), dict(softcap=50.0), {}],
                         ids=["cap5", "cap50", "plain"])
@pytest.mark.parametrize("slopes", [0, 1])
def test_decode_bytes_past_the_end(tm, dev, window, kw, slopes):
    """Rows past a request's last key, and before its window, hold zeros, large
    keys or no number: the same bits of results."""
    g = _gen(90)
    ends = [1, 15, 17, 40, 70, 200, 333]
    c = Cache4(tm, ends, 2, g, dev)
    q = _rand((len(ends), 8, D), g, 0.5).to(dev)
    kw = dict(kw, window=window)
    if slopes:
        kw["slopes"] = (torch.rand(8, generator=g) * 0.1).to(dev)
    rows = []
    for i, n in enumerate(ends):
        pages = -(-n // PAGE)
        pos = list(range(n, pages * PAGE))
        if window:
            pos += range(0, max(0, n - window))
        pos = torch.tensor(pos, dtype=torch.long)
        rows.append(c.table.cpu()[i][pos // PAGE].long() * PAGE + pos % PAGE)
    rows = torch.cat(rows).to(dev)
    res = []
    for std in (0.0, 1e-3, 40.0, 1e6, float("nan")):
        x = (torch.randn((len(rows), 2, D), generator=g) * std).to(dev)
        tm.kv_write_mx4(x.bfloat16(), x.bfloat16(), rows, c.pool)
        for split in (dict(), dict(min_pages=1, num_workgroups=9)):
            res.append(tm.decode_mx4_paged(q, c.pool, c.table, c.ctx, 0.1,
                                           **kw, **split))
    for i, (out, lse) in enumerate(res):
        assert torch.isfinite(out).all() and torch.isfinite(lse).all()
        assert torch.equal(out, res[i % 2][0])
        assert torch.equal(lse, res[i % 2][1])
