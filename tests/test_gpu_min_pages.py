"""Decodes with the largest bounds of pages per work-group: every request in one
piece, whatever the grid."""
import pytest
import torch

from test_gpu_mx4 import Cache4
from test_gpu_scored import Cache, _gen, _rand

pytestmark = pytest.mark.gpu


def _same(call):
    want = call(min_pages=10000, return_lse=True)
    for n in (32768, 2 ** 30, 2 ** 31 - 1):
        for wgs in (0, 7, 3000):
            got = call(min_pages=n, num_workgroups=wgs, return_lse=True)
            for x, y in zip(got, want):
                assert torch.equal(x, y)


def test_largest_min_pages(tm, dev):
    g = _gen(99)
    ends = [300, 0, 17, 1000, 64]
    c, c4 = Cache(ends, 4, g, dev), Cache4(tm, ends, 4, g, dev)
    q = _rand((len(ends), 16, 128), g, dev)
    lam = torch.full((8,), 0.3, device=dev)
    a = (c.kp, c.vp, c.table, c.ctx, 0.1)
    _same(lambda **kw: tm.decode_paged(q, *a, **kw))
    _same(lambda **kw: tm.decode_scored_paged(q, *a, softcap=5.0, **kw))
    _same(lambda **kw: tm.decode_mx4_paged(q, c4.pool, c4.table, c4.ctx, 0.1,
                                           **kw))
    _same(lambda **kw: tm.decode_diff_paged(q, c.kp, c.vp, c.table, c.ctx, lam,
                                            0.1, **kw))
    pos = torch.tensor([300 - 1, 17 - 1], device=dev)
    flat = torch.zeros((2, 320), dtype=torch.int64, device=dev)
    at = torch.arange(320, device=dev)
    for i, b in enumerate((0, 2)):
        page = at // 16 % c.table.shape[1]
        flat[i] = c.table[b][page].long() * 16 + at % 16
    qf = q[[0, 2]].contiguous()
    _same(lambda **kw: tm.decode_flat(qf, c.kp, c.vp, flat, pos, 0.1, **kw))
