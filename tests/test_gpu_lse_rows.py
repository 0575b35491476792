"""Prefills whose runs end before the rows do (a step planned for a fixed number
of tokens): LSE rows are as long as q's, their columns behind the last run stay
as they were."""
from importlib import import_module

import pytest
import torch

from oracle import attn_ref
from oracle import scored_ref as ref
from helpers import assert_lse_close, assert_out_close
from test_gpu_mx4 import Cache4
from test_gpu_scored import Cache, D, _function, _gen, _i32, _packed

pytestmark = pytest.mark.gpu


def _rows_behind(call, n, total, hq, dev):
    """call(rows, **kw) at n rows and at total ones, the same runs: outputs and
    LSE [hq, total] of the longer call, checked to hold what the shorter gives."""
    want = call(n)
    for reject in (None, _i32([0], dev)):
        lse = torch.full((hq, total), 7.0, device=dev)
        out, got = call(total, lse=lse, reject=reject)
        assert got is lse
        assert torch.equal(out[:n], want[0][:n])
        assert torch.equal(lse[:, :n], want[1][:, :n])
        assert (lse[:, n:] == 7).all()
    got = call(total)
    assert got[1].shape == (hq, total)
    assert torch.equal(got[1][:, :n], want[1][:, :n])
    out, lse = call(total, reject=_i32([1], dev))
    assert torch.isnan(out).all() and torch.isnan(lse).all()
    return got


@pytest.mark.parametrize("source", ["packed", "paged", "four"])
@pytest.mark.parametrize("split", [0, 1])
@pytest.mark.parametrize("name", ["plain", "soft", "slopes", "cap slopes"])
def test_scored_and_mx4(tm, dev, source, split, name):
    g = _gen(60 + split)
    if split:
        lens, prior, hq, hkv = (([3300], [0], 4, 1) if source == "packed" else
                                ([64], [9000], 16, 2))
    else:
        lens, prior, hq, hkv = [50, 0, 70], [0, 3, 30], 8, 2
    if source == "packed":
        prior = [0] * len(lens)
    n = sum(lens)
    total = n + 57
    x, k, v, _ = _packed([total], hq, hkv, g, dev)
    cu = _i32([sum(lens[:i]) for i in range(len(lens) + 1)], dev)
    ends = [a + b for a, b in zip(lens, prior)]
    kw = _function(name, hq, g, dev)
    p = _i32(prior, dev)
    if source == "packed":
        args = dict(k=k[:n], v=v[:n])

        def call(rows, **more):
            return tm.prefill_scored_varlen(x[:rows], k[:rows], v[:rows], cu,
                                            0.1, **kw, **more)
    elif source == "paged":
        c = Cache(ends, hkv, g, dev)
        args = dict(k=None, v=None, prior=p, k_pool=c.kp, v_pool=c.vp,
                    table=c.table)

        def call(rows, **more):
            return tm.prefill_scored_varlen(
                x[:rows], None, None, cu, 0.1, prior_lens=p, k_pool=c.kp,
                v_pool=c.vp, block_table=c.table, **kw, **more)
    else:
        c = Cache4(tm, ends, hkv, g, dev)
        args = dict(k=None, v=None, prior=p, k_pool=c.kp, v_pool=c.vp,
                    table=c.table)

        def call(rows, **more):
            return tm.prefill_mx4_varlen(x[:rows], c.pool, c.table, cu, p, 0.1,
                                         **kw, **more)
    size = tm._lib.load().tmopt_attn_prefill_scored_workspace_size
    assert (size(len(lens), max(lens), 0, hq, hkv,
                 0 if source == "packed" else c.table.shape[1], 0) > 0) == split
    out, lse = _rows_behind(call, n, total, hq, dev)
    ref.check(out[:n], lse[:, :n], ref.prefill(x[:n], cu=cu, scale=0.1, **args,
                                               **kw), name)


@pytest.mark.parametrize("source", ["packed", "padded", "paged", "mixed"])
@pytest.mark.parametrize("split", [0, 1])
@pytest.mark.parametrize("E", [0, 200])
def test_prefill_varlen(tm, dev, source, split, E):
    g = torch.Generator().manual_seed(61 + split)
    r = lambda *s: torch.randn(s, generator=g).to(torch.bfloat16)  # noqa: E731
    own_only = source in ("packed", "padded")
    if split:
        lens, prior, hq, hkv = (([3300], [0], 4, 1) if own_only else
                                ([64], [3000], 16, 2))
    else:
        lens, prior, hq, hkv = [50, 0, 70], [0, 3, 30], 8, 2
    n, S = sum(lens), len(lens)
    total = n + 57
    cu = torch.tensor([0] + lens).cumsum(0).to(torch.int32)
    q, rel = r(total, hq, D), r(total, hq, E) if E else None
    a = dict(cu_seqlens=cu, scale=D ** -0.5, k=None, v=None)
    if source == "padded":
        a.update(k=r(S, max(lens), hkv, D), v=r(S, max(lens), hkv, D))
    elif source != "paged":
        a.update(k=r(total, hkv, D), v=r(total, hkv, D))
    if not own_only:
        wl = import_module("tm-opt_amd.workloads")
        table, P = wl.paged_layout(lens, g, prior=prior)
        a.update(prior_lens=torch.tensor(prior, dtype=torch.int32),
                 k_pool=r(P, 16, hkv, D), v_pool=r(P, 16, hkv, D),
                 block_table=table)
    size = tm._lib.load().tmopt_attn_prefill_workspace_size
    assert (size(S, max(lens), hq, hkv, 0 if own_only else table.shape[1], 0,
                 0) > 0) == split

    def rows(x, m):
        return x[:m] if source in ("packed", "mixed") else x

    def call(m, **more):
        d = {k: x.to(dev) if torch.is_tensor(x) else x for k, x in a.items()}
        if d["k"] is not None:
            d.update(k=rows(d["k"], m), v=rows(d["v"], m))
        return tm.prefill_varlen(q[:m].to(dev), **d, **more,
                                 rel=rel[:m].to(dev) if E else None)
    out, lse = _rows_behind(call, n, total, hq, dev)
    if source == "padded":
        a.update({x: torch.cat([a[x][i, :m] for i, m in enumerate(lens)])
                  for x in ("k", "v")})
    elif source != "paged":
        a.update(k=a["k"][:n], v=a["v"][:n])
    ref_o, ref_l = attn_ref.prefill_varlen(q[:n], rel=rel[:n] if E else None,
                                           **a)
    assert_out_close(out[:n], ref_o, source)
    assert_lse_close(lse[:, :n], ref_l, source)
