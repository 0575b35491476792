"""Refusals of the differential attention and page plan entry points (CPU:
they come before any launch), and the float64 oracle against torch's softmax
two maps at a time: the definition written a second way."""
import ctypes
import math

import pytest
import torch

from oracle import diff_ref

NULL, P, ODD = (ctypes.c_void_p(x) for x in (0, 16, 18))


def test_decode_refusals(tm):
    lib, e = tm._lib.load(), tm._lib
    size = lib.tmopt_attn_decode_diff_workspace_size
    assert size(0, 32, 4, 128, 0) == 0 and size(4, 32, 0, 128, 0) == 0
    need = size(4, 32, 4, 128, 0)
    assert 0 < need < 1 << 30

    def call(q=P, kp=P, vp=P, bt=P, bts=8, wrap=0, ctx=P, B=4, HQ=32, HKV=4,
             D=128, ps=16, pages=9, window=0, scale=0.1, lam=P, lst=1, w=P,
             eps=1e-5, mp=8, wgs=0, out=P, ws=P, nbytes=1 << 40):
        return lib.tmopt_attn_decode_diff(
            q, kp, vp, bt, bts, wrap, ctx, B, HQ, HKV, D, ps, pages, window,
            scale, lam, lst, w, eps, 1.0, mp, wgs, out, NULL, ws, nbytes, NULL)
    assert call(B=0, q=NULL) == 0
    for kw in (dict(B=-1), dict(q=NULL), dict(q=ODD), dict(kp=ODD),
               dict(vp=NULL), dict(bt=NULL), dict(ctx=NULL), dict(out=NULL),
               dict(HQ=33), dict(HKV=3, HQ=33), dict(HKV=0), dict(HQ=0),
               dict(bts=0), dict(pages=0), dict(window=-1), dict(scale=0.0),
               dict(scale=-1.0), dict(scale=math.nan), dict(lam=NULL),
               dict(lst=2), dict(eps=0.0), dict(eps=math.nan), dict(w=ODD),
               dict(mp=0), dict(wgs=-1), dict(wgs=65536), dict(wrap=-1),
               dict(wrap=9), dict(wrap=4), dict(wrap=4, window=65)):
        assert call(**kw) == e.TMOPT_EINVAL, kw
    for kw in (dict(B=8193), dict(D=64), dict(ps=32),
               dict(HKV=1 << 18, HQ=1 << 18)):
        assert call(**kw) == e.TMOPT_EUNSUPPORTED, kw
    for kw in (dict(ws=NULL), dict(ws=ctypes.c_void_p(8)),
               dict(nbytes=need - 1)):
        assert call(**kw) == e.TMOPT_EWORKSPACE, kw


def test_prefill_refusals(tm):
    lib, e = tm._lib.load(), tm._lib
    size = lib.tmopt_attn_prefill_diff_workspace_size
    for bad in ((0, 64, 0, 32, 4), (1, 0, 0, 32, 4), (1, 64, 0, 0, 4),
                (1, 64, 0, 32, 0), (-1, 64, 0, 32, 4), (1, 64, 0, 33, 4)):
        assert size(*bad, 500, 0) == 0

    def call(q=P, qt=4096, k=P, kt=512, kh=128, v=P, cu=P, prior=NULL, S=2,
             n=64, most=0, kp=NULL, vp=NULL, bt=NULL, bts=8, ps=16, pages=9, HQ=32,
             HKV=4, D=128, window=0, scale=0.1, lam=P, out=P, ot=4096, lse=P,
             ws=NULL, nbytes=0):
        return lib.tmopt_attn_prefill_diff(
            q, qt, 128, k, kt, kh, v, kt, kh, cu, prior, S, n, most, kp, vp, bt,
            bts, ps, pages, HQ, HKV, D, window, scale, lam, 1, NULL, 0.0, 1.0,
            out, ot, 256, lse, 128, NULL, ws, nbytes, NULL)
    pool = dict(k=NULL, v=NULL, kp=P, vp=P, bt=P)
    assert call(S=0, q=NULL) == call(n=0, q=NULL) == 0
    for kw in (dict(S=-1), dict(S=65536), dict(n=-1), dict(q=NULL),
               dict(cu=NULL), dict(out=NULL), dict(q=ODD), dict(out=ODD),
               dict(qt=4092), dict(ot=4100), dict(k=NULL), dict(v=NULL),
               dict(k=ODD), dict(kt=500), dict(kt=-512), dict(kh=100),
               dict(prior=P), dict(HQ=33), dict(HQ=3, HKV=3),
               dict(window=-1), dict(scale=0.0), dict(scale=math.nan),
               dict(most=-1), dict(lam=NULL), dict(bt=P, kp=P, vp=P),
               dict(pool, kp=NULL), dict(pool, vp=ODD), dict(pool, bts=0),
               dict(pool, pages=0)):
        assert call(**kw) == e.TMOPT_EINVAL, kw
    for kw in (dict(D=64), dict(pool, ps=32), dict(n=1 << 18),
               dict(n=1 << 17, qt=128, kt=1 << 14)):
        assert call(**kw) == e.TMOPT_EUNSUPPORTED, kw
    need = size(2, 64, 0, 32, 4, 500, 0)
    assert 0 < need <= 256 * 3 * 258 * 1024
    for kw in (dict(ws=ctypes.c_void_p(8), nbytes=need),
               dict(ws=P, nbytes=need - 1)):
        assert call(**dict(pool, bts=500, **kw)) == e.TMOPT_EWORKSPACE, kw
    # without a block table only the run's own length counts
    assert size(1, 200, 0, 32, 4, 0, 0) == 0 < size(1, 4000, 0, 4, 2, 0, 0)
    assert size(1, 4000, 0, 4, 2, 0, 100) == 0
    # a bound of the contexts counts where it is below the table's width
    assert size(2, 64, 900, 32, 4, 500, 0) == 0
    assert size(2, 64, 1 << 40, 32, 4, 500, 0) == need


def test_plan_refusals(tm):
    lib, e = tm._lib.load(), tm._lib

    def plan(pt=P, S=9, W=8, slots=P, ctx=P, new=P, B=4, free=P, F=40,
             count=P, T=64, width=8, bt=P, seq=P, cu=P, sm=P, pos=P, n=P,
             rej=P):
        return lib.tmopt_plan_pages(pt, S, W, slots, ctx, new, B, free, F,
                                    count, T, width, bt, seq, cu, sm, pos, n,
                                    rej, NULL)
    for x in ("pt", "slots", "ctx", "new", "free", "count", "bt", "seq", "cu",
              "sm", "pos", "n", "rej"):
        assert plan(**{x: NULL}) == e.TMOPT_EINVAL, x
    for kw in (dict(B=-1), dict(B=8193), dict(S=0), dict(S=(1 << 18) + 1),
               dict(W=0), dict(W=(1 << 24) + 1), dict(F=0),
               dict(F=1 << 31), dict(T=-1), dict(T=(1 << 24) + 1),
               dict(width=0), dict(width=(1 << 24) + 1)):
        assert plan(**kw) == e.TMOPT_EUNSUPPORTED, kw
    size = lib.tmopt_release_pages_workspace_size
    assert size(0) == 0 and size(-1) == 0 and size(3) == 16

    def release(pt=P, S=9, W=8, slots=P, lens=P, B=5, free=P, F=40, count=P,
                n=P, rej=P, ws=P, nbytes=32):
        return lib.tmopt_release_pages(pt, S, W, slots, lens, B, free, F,
                                       count, n, rej, ws, nbytes, NULL)
    for x in ("pt", "slots", "lens", "free", "count", "n", "rej"):
        assert release(**{x: NULL}) == e.TMOPT_EINVAL, x
    for kw in (dict(B=-1), dict(B=8193), dict(S=0), dict(W=0), dict(F=0)):
        assert release(**kw) == e.TMOPT_EUNSUPPORTED, kw
    for kw in (dict(ws=NULL), dict(nbytes=16), dict(ws=ctypes.c_void_p(8))):
        assert release(**kw) == e.TMOPT_EWORKSPACE, kw


def test_wrappers_assert_before_launch(tm):
    bf, i32, i64 = torch.bfloat16, torch.int32, torch.int64
    q = torch.zeros((2, 8, 128), dtype=bf)
    pool = torch.zeros((4, 16, 4, 128), dtype=bf)
    table, ctx = torch.zeros((2, 4), dtype=i32), torch.ones(2, dtype=i32)
    lam = torch.zeros(4)

    def decode(q=q, kp=pool, vp=pool, table=table, ctx=ctx, lam=lam, **kw):
        with pytest.raises(AssertionError):
            tm.decode_diff_paged(q, kp, vp, table, ctx, lam, 0.1, **kw)
    decode(q=q.float())
    decode(q=q.transpose(0, 1))
    decode(kp=pool.float())
    decode(kp=pool[:, :, :3])
    decode(kp=pool[..., :64])
    decode(table=table.long())
    decode(table=torch.zeros((2, 8), dtype=i32)[:, :4])
    decode(table=table[:1])
    decode(ctx=ctx.long())
    decode(ctx=ctx[:1])
    decode(lam=lam.double())
    decode(lam=lam[:3])
    decode(lam=torch.zeros(8)[::2])
    decode(norm_weight=torch.ones(128))
    decode(norm_weight=torch.ones(256, dtype=bf))
    decode(out=torch.zeros((2, 8, 128), dtype=bf))
    decode(lse=torch.zeros((2, 4)))
    decode(table_wrap=2)
    decode(table_wrap=2, window=33)

    k = torch.zeros((2, 4, 128), dtype=bf)
    cu = torch.tensor([0, 2], dtype=i32)

    def prefill(q=q, k=k, v=k, cu=cu, lam=lam, **kw):
        with pytest.raises(AssertionError):
            tm.prefill_diff_varlen(q, k, v, cu, lam, 0.1, max_seqlen=2, **kw)
    prefill(q=q.float())
    prefill(cu=cu.long())
    prefill(k=k[:1])
    prefill(k=k[:, :3], v=k[:, :3])
    prefill(k=k.float())
    prefill(prior_lens=ctx[:1])
    prefill(k_pool=pool, v_pool=pool)
    prefill(k_pool=pool, v_pool=pool, block_table=table)
    prefill(k=None, v=None, k_pool=pool, v_pool=pool,
            block_table=table.long())
    prefill(k=None, v=None, k_pool=pool, v_pool=pool, block_table=table,
            prior_lens=ctx)
    prefill(lam=lam[:2])
    prefill(out=torch.zeros((2, 4, 256)))
    prefill(lse=torch.zeros((2, 8)))

    pt, free = torch.zeros((3, 4), dtype=i32), torch.zeros(9, dtype=i32)
    slots, one = torch.zeros(2, dtype=i64), torch.ones(1, dtype=i32)

    def plan(pt=pt, slots=slots, ctx=ctx, new=ctx, free=free, count=one, **kw):
        with pytest.raises(AssertionError):
            tm.plan_pages(pt, slots, ctx, new, free, count, 8, **kw)
    plan(pt=pt.long())
    plan(pt=pt[:, :2])
    plan(slots=slots.int())
    plan(ctx=ctx[:1])
    plan(new=ctx.long())
    plan(free=free.long())
    plan(count=ctx)
    o = tm.PagePlan(pt[:2], ctx, torch.zeros(3, dtype=i32),
                    torch.zeros(8, dtype=i64), torch.zeros(8, dtype=i64), one,
                    one)
    plan(out=o._replace(cu_seqlens=ctx))
    plan(out=o._replace(slot_mapping=slots))
    plan(out=o._replace(block_table=pt))
    plan(out=o, width=3)
    with pytest.raises(AssertionError):
        tm.release_pages(pt, slots.int(), ctx, free, one)
    with pytest.raises(AssertionError):
        tm.release_pages(pt, slots, ctx, free, one, out=(one, ctx))


def test_oracle_restates_the_definition():
    """attend() against two softmaxes and a difference written out for one
    head pair and one query at a time."""
    g = torch.Generator().manual_seed(1)
    T, N, hq, hkv = 3, 9, 4, 2
    q = torch.randn((T, hq, 128), generator=g, dtype=torch.float64)
    k = torch.randn((N, hkv, 128), generator=g, dtype=torch.float64)
    v = torch.randn((N, hkv, 128), generator=g, dtype=torch.float64)
    lam, w = torch.tensor([0.3, -0.7]), torch.rand(256, generator=g)
    qpos = torch.tensor([0, 4, 8])
    out, lse, err, _ = diff_ref.attend(q, k, v, qpos, torch.arange(N), lam,
                                       0.2, w, 1e-3, 0.5, window=5)
    for t in range(T):
        p = int(qpos[t])
        lo = max(0, p - 4)
        V = v[lo:p + 1].reshape(-1, 256)
        for h in range(2):
            maps = [torch.softmax(0.2 * k[lo:p + 1, m] @ q[t, 2 * h + m], 0)
                    for m in range(2)]
            o = (maps[0] - lam[h].double() * maps[1]) @ V
            o = o / (o.pow(2).mean() + 1e-3).sqrt() * w.double() * 0.5
            assert (out[t, h] - o).abs().max() < 1e-12
            assert abs(lse[2 * h, t] - torch.logsumexp(
                0.2 * k[lo:p + 1, 0] @ q[t, 2 * h], 0)) < 1e-12
    assert (err > 0).all() and err.max() < 0.1


def test_oracle_of_the_plan():
    """A step small enough to write down."""
    got = diff_ref.plan([[5, -1, -1], [8, 9, -1]], [1, 0], [17, 15], [1, 3],
                        [40, 41, 42], 3, 6)
    assert got == ([[5, 42, -1], [8, 9, -1]], [[8, 9, -1], [5, 42, -1]],
                   [18, 18], [0, 1, 4], [145, 95, 672, 673, -1, -1],
                   [17, 15, 16, 17, 0, 0], 2, 0)
    assert diff_ref.release(got[0], [0, 1], [18, 16], [40, 41, -1, -1, -1],
                            2) == ([40, 41, 5, 42, 8], 5, 0)
