"""Refusals of the scored attention and of the 4-bit cache's entry points (CPU:
they come before any launch), and their oracle against the definition written a
second way."""
import ctypes
import importlib
import math

import pytest
import torch

from oracle import scored_ref as ref

NULL, P, ODD = (ctypes.c_void_p(x) for x in (0, 16, 18))
EIGHT = ctypes.c_void_p(8)


def test_rows_refusals(tm):
    lib, e = tm._lib.load(), tm._lib

    def write(k=P, v=P, kt=512, kh=128, vt=512, vh=128, slots=P, T=5, H=4,
              D=128, ps=16, pool=P, pages=9):
        return lib.tmopt_kv_write_mx4(k, v, kt, kh, vt, vh, slots, T, H, D, ps,
                                      pool, pages, NULL)

    def read(pool=P, pages=9, slots=P, T=5, H=4, D=128, ps=16, k=P, v=P):
        return lib.tmopt_kv_read_mx4(pool, pages, slots, T, H, D, ps, k, v,
                                     NULL)
    assert write(T=0, k=NULL) == read(T=0, pool=NULL) == 0
    for fn in (write, read):
        for kw in (dict(k=NULL), dict(v=NULL), dict(k=ODD), dict(v=EIGHT),
                   dict(slots=NULL), dict(pool=NULL), dict(pool=EIGHT),
                   dict(T=-1), dict(H=0), dict(H=-4), dict(pages=0),
                   dict(pages=1 << 31)):
            assert fn(**kw) == e.TMOPT_EINVAL, (fn, kw)
        for kw in (dict(D=64), dict(ps=32), dict(H=65536),
                   dict(T=1 << 34, H=8)):
            assert fn(**kw) == e.TMOPT_EUNSUPPORTED, (fn, kw)
    for kw in (dict(kt=516), dict(kh=100), dict(vt=4), dict(vh=1)):
        assert write(**kw) == e.TMOPT_EINVAL, kw


def _decode_calls(tm):
    lib = tm._lib.load()

    def scored(q=P, kp=P, vp=P, bt=P, bts=8, wrap=0, ctx=P, B=4, HQ=32, HKV=4,
               D=128, ps=16, pages=9, window=0, scale=0.1, cap=0.0, mp=8,
               wgs=0, out=P, ws=P, nbytes=1 << 40):
        return lib.tmopt_attn_decode_scored(
            q, kp, vp, bt, bts, wrap, ctx, B, HQ, HKV, D, ps, pages, window,
            scale, cap, NULL, NULL, mp, wgs, out, NULL, ws, nbytes, NULL)

    def mx4(q=P, kp=P, vp=P, bt=P, bts=8, wrap=0, ctx=P, B=4, HQ=32, HKV=4,
            D=128, ps=16, pages=9, window=0, scale=0.1, cap=0.0, mp=8, wgs=0,
            out=P, ws=P, nbytes=1 << 40, slopes=NULL, rel=NULL, E=0):
        pool = vp if kp is P else kp
        return lib.tmopt_attn_decode_mx4(
            q, pool, bt, bts, wrap, ctx, B, HQ, HKV, D, ps, pages, window,
            scale, cap, slopes, rel, E, mp, wgs, out, NULL, ws, nbytes, NULL)
    return (scored, lib.tmopt_attn_decode_workspace_size), (
        mx4, lib.tmopt_attn_decode_mx4_workspace_size)


def test_decode_refusals(tm):
    e = tm._lib
    for call, size in _decode_calls(tm):
        need = size(4, 32, 4, 128, 0)
        assert 0 < need < 1 << 30
        assert call(B=0, q=NULL) == 0
        for kw in (dict(B=-1), dict(q=NULL), dict(q=ODD), dict(kp=ODD),
                   dict(vp=NULL), dict(bt=NULL), dict(ctx=NULL),
                   dict(out=NULL), dict(out=EIGHT), dict(HQ=33), dict(HKV=0),
                   dict(HQ=0), dict(bts=0), dict(pages=0), dict(window=-1),
                   dict(scale=0.0), dict(scale=-1.0), dict(scale=math.nan),
                   dict(scale=math.inf), dict(cap=-1.0), dict(cap=math.nan),
                   dict(cap=math.inf), dict(cap=1e-39), dict(cap=3e38), dict(mp=0), dict(wgs=-1),
                   dict(wgs=65536), dict(wrap=-1), dict(wrap=9), dict(wrap=4),
                   dict(wrap=4, window=65)):
            assert call(**kw) == e.TMOPT_EINVAL, kw
        for kw in (dict(B=8193), dict(D=64), dict(ps=32),
                   dict(HKV=1 << 18, HQ=1 << 18)):
            assert call(**kw) == e.TMOPT_EUNSUPPORTED, kw
        for kw in (dict(ws=NULL), dict(ws=EIGHT), dict(nbytes=need - 1)):
            assert call(**kw) == e.TMOPT_EWORKSPACE, kw
    for kw in (dict(rel=P, E=0), dict(rel=ctypes.c_void_p(17), E=8),
               dict(rel=P, E=1 << 24)):
        assert call(**kw) == e.TMOPT_EINVAL, kw
    for kw in (dict(rel=P, E=8, cap=1.0), dict(rel=P, E=8, slopes=P)):
        assert call(**kw) == e.TMOPT_EUNSUPPORTED, kw
    assert size(0, 32, 4, 128, 0) == size(4, 33, 4, 128, 0) == 0


def test_prefill_refusals(tm):
    lib, e = tm._lib.load(), tm._lib

    def scored(q=P, qt=4096, k=P, kt=512, kh=128, v=P, cu=P, prior=NULL, S=2,
               n=64, most=0, kp=NULL, vp=NULL, bt=NULL, bts=8, ps=16, pages=9,
               HQ=32, HKV=4, D=128, window=0, scale=0.1, cap=0.0, out=P,
               ot=4096, ws=NULL, nbytes=0):
        return lib.tmopt_attn_prefill_scored(
            q, qt, 128, k, kt, kh, v, kt, kh, cu, prior, S, n, most, kp, vp,
            bt, bts, ps, pages, HQ, HKV, D, window, scale, cap, NULL, NULL,
            NULL, out, ot, 128, NULL, NULL, ws, nbytes, NULL)

    def mx4(q=P, qt=4096, cu=P, S=2, n=64, most=0, kp=P, bt=P, bts=8, ps=16,
            pages=9, HQ=32, HKV=4, D=128, window=0, scale=0.1, cap=0.0, out=P,
            ot=4096, ws=NULL, nbytes=0, slopes=NULL, rel=NULL, rt=32 * 64,
            rh=64, E=64, k=NULL, v=NULL, vp=NULL):
        return lib.tmopt_attn_prefill_mx4(
            q, qt, 128, cu, NULL, S, n, most, kp, bt, bts, ps, pages, HQ, HKV,
            D, window, scale, cap, slopes, rel, rt, rh, E, out, ot, 128, NULL,
            NULL, ws, nbytes, NULL)
    pool = dict(k=NULL, v=NULL, kp=P, vp=P, bt=P)
    for call in (scored, mx4):
        assert call(S=0, q=NULL) == call(n=0, q=NULL) == 0
        for kw in (dict(S=-1), dict(S=65536), dict(n=-1), dict(q=NULL),
                   dict(cu=NULL), dict(out=NULL), dict(q=ODD),
                   dict(out=ctypes.c_void_p(20)), dict(qt=4092),
                   dict(qt=-4096), dict(ot=4098), dict(HQ=33),
                   dict(HQ=4, HKV=0), dict(window=-1), dict(scale=0.0),
                   dict(scale=math.nan), dict(cap=-2.0), dict(cap=math.inf), dict(cap=1e-39),
                   dict(most=-1), dict(pool, kp=NULL), dict(pool, kp=ODD),
                   dict(pool, bts=0), dict(pool, pages=0)):
            assert call(**kw) == e.TMOPT_EINVAL, (call, kw)
        for kw in (dict(D=64), dict(pool, ps=32), dict(n=1 << 18),
                   dict(pool, HQ=3 * 65535, HKV=65535)):
            assert call(**kw) == e.TMOPT_EUNSUPPORTED, (call, kw)
    for kw in (dict(k=NULL), dict(v=NULL), dict(k=ODD), dict(kt=500),
               dict(kt=-512), dict(kh=100), dict(prior=P),
               dict(bt=P, kp=P, vp=P), dict(pool, vp=NULL)):
        assert scored(**kw) == e.TMOPT_EINVAL, kw
    assert scored(n=1 << 17, qt=128, kt=1 << 14) == e.TMOPT_EUNSUPPORTED
    for kw in (dict(rel=P, E=0), dict(rel=ctypes.c_void_p(17)),
               dict(bt=NULL)):
        assert mx4(**kw) == e.TMOPT_EINVAL, kw
    for kw in (dict(rel=P, cap=1.0), dict(rel=P, slopes=P),
               dict(rel=P, rt=63), dict(rel=P, rh=-1),
               dict(rel=P, rt=1 << 26)):
        assert mx4(**kw) == e.TMOPT_EUNSUPPORTED, kw
    for name, call in (("scored", scored), ("mx4", mx4)):
        size = getattr(lib, f"tmopt_attn_prefill_{name}_workspace_size")
        for bad in ((0, 64, 0, 32, 4), (1, 0, 0, 32, 4), (1, 64, 0, 0, 4),
                    (1, 64, 0, 32, 0), (-1, 64, 0, 32, 4), (1, 64, 0, 33, 4)):
            assert size(*bad, 500, 0) == 0
        need = size(2, 64, 0, 32, 4, 500, 0)
        assert 0 < need <= 256 * 2 * 130 * 1024
        for kw in (dict(ws=EIGHT, nbytes=need), dict(ws=P, nbytes=need - 1)):
            assert call(**dict(pool, bts=500, **kw)) == e.TMOPT_EWORKSPACE, kw
        # a bound of the contexts counts where it is below the table's width
        assert size(2, 64, 512, 32, 4, 500, 0) == 0
        assert size(2, 64, 1 << 40, 32, 4, 500, 0) == need
    size = lib.tmopt_attn_prefill_scored_workspace_size
    assert size(1, 200, 0, 32, 4, 0, 0) == 0 < size(1, 4000, 0, 4, 1, 0, 0)
    assert lib.tmopt_attn_prefill_mx4_workspace_size(1, 4000, 0, 4, 1, 0,
                                                     0) == 0


def test_python_checks(tm):
    """The Python entry points refuse what the kernels do not take."""
    BF, I32 = torch.bfloat16, torch.int32
    q = torch.zeros((2, 8, 128), dtype=BF)
    pool = tm.mx4_pool(3, 2, "cpu")
    assert pool.shape == (3, 2, 2176) and pool.dtype == torch.uint8
    table = torch.zeros((2, 4), dtype=I32)
    ctx = torch.zeros(2, dtype=I32)
    kp = torch.zeros((3, 16, 2, 128), dtype=BF)
    cu = torch.tensor([0, 1, 2], dtype=I32)
    one = torch.zeros((2, 2, 128), dtype=BF)
    rows = torch.zeros(2, dtype=torch.int64)
    f32 = torch.zeros(8)
    calls = [
        lambda: tm.kv_write_mx4(one.float(), one.float(), rows, pool),
        lambda: tm.kv_write_mx4(one, one[:1], rows, pool),
        lambda: tm.kv_write_mx4(one, one, rows.int(), pool),
        lambda: tm.kv_write_mx4(one, one, rows[:1], pool),
        lambda: tm.kv_write_mx4(one[:, :1], one[:, :1], rows, pool),
        lambda: tm.kv_write_mx4(one, one, rows, pool[..., :2100]),
        lambda: tm.kv_write_mx4(one, one, rows, pool.to(torch.int8)),
        lambda: tm.kv_read_mx4(pool, rows.int()),
        lambda: tm.kv_read_mx4(pool, rows, k=one[:1]),
        lambda: tm.decode_mx4_paged(q.float(), pool, table, ctx, 0.1),
        lambda: tm.decode_mx4_paged(q, pool, table.long(), ctx, 0.1),
        lambda: tm.decode_mx4_paged(q, pool, table[:, :2], ctx, 0.1),
        lambda: tm.decode_mx4_paged(q, pool, table, ctx[:1], 0.1),
        lambda: tm.decode_mx4_paged(q, pool, table, ctx, 0.1, table_wrap=2),
        lambda: tm.decode_mx4_paged(q, pool, table, ctx, 0.1, slopes=f32[:4]),
        lambda: tm.decode_mx4_paged(q, pool, table, ctx, 0.1,
                                    rel=torch.zeros((2, 4, 9), dtype=BF)),
        lambda: tm.decode_mx4_paged(q, pool, table, ctx, 0.1, out=q.float()),
        lambda: tm.prefill_mx4_varlen(q, pool, table, cu.long(), ctx, 0.1),
        lambda: tm.prefill_mx4_varlen(q, pool, table, cu, ctx[:1], 0.1),
        lambda: tm.prefill_mx4_varlen(q, pool, table[:1], cu, ctx, 0.1),
        lambda: tm.decode_scored_paged(q, kp, kp[:2], table, ctx, 0.1),
        lambda: tm.decode_scored_paged(q, kp, kp, table, ctx, 0.1,
                                       first_keys=ctx.long()),
        lambda: tm.decode_scored_paged(q, kp, kp, table, ctx, 0.1,
                                       slopes=f32.double()),
        lambda: tm.prefill_scored_varlen(q, one, one, cu, 0.1,
                                         prior_lens=ctx),
        lambda: tm.prefill_scored_varlen(q, one, one, cu, 0.1,
                                         first_keys=ctx[:1]),
        lambda: tm.prefill_scored_varlen(q, one, one, cu, 0.1,
                                         prefix_lens=ctx.long()),
        lambda: tm.prefill_scored_varlen(q, one, one, cu, 0.1,
                                         block_table=table, k_pool=kp,
                                         v_pool=kp),
        lambda: tm.prefill_scored_varlen(q, one, one[:1], cu, 0.1),
    ]
    # numbers whose low 32 bits alone would be another call
    for kw in (dict(window=(1 << 32) + 5), dict(window=1 << 31)):
        calls += [
            lambda kw=kw: tm.decode_mx4_paged(q, pool, table, ctx, 0.1, **kw),
            lambda kw=kw: tm.decode_scored_paged(q, kp, kp, table, ctx, 0.1,
                                                 **kw),
            lambda kw=kw: tm.prefill_mx4_varlen(q, pool, table, cu, ctx, 0.1,
                                                max_seqlen=1, **kw),
            lambda kw=kw: tm.prefill_scored_varlen(q, one, one, cu, 0.1,
                                                   max_seqlen=1, **kw)]
    for kw in (dict(min_pages=(1 << 32) + 1),
               dict(num_workgroups=(1 << 32) + 1),
               dict(window=16, table_wrap=(1 << 32) + 1)):
        calls += [
            lambda kw=kw: tm.decode_mx4_paged(q, pool, table, ctx, 0.1, **kw),
            lambda kw=kw: tm.decode_scored_paged(q, kp, kp, table, ctx, 0.1,
                                                 **kw)]
    calls += [
        lambda: tm.prefill_mx4_varlen(q, pool, table, cu, ctx, 0.1,
                                      max_seqlen=(1 << 32) + 1),
        lambda: tm.prefill_scored_varlen(q, one, one, cu, 0.1,
                                         max_seqlen=(1 << 32) + 1)]
    for i, call in enumerate(calls):
        with pytest.raises(AssertionError):
            call()
            print("call", i)


def test_oracle_quantise():
    """By trying every scale and element: the smallest scale whose elements
    stay within a step of half the largest, then the nearest element."""
    g = torch.Generator().manual_seed(0)
    x = (torch.randn((40, 128), generator=g) * torch.exp(
        4 * torch.randn((40, 1), generator=g))).bfloat16()
    x[0] = 0
    x[1, :32] = torch.tensor([7.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0] * 4)
    x[2, :32] = 7.03125
    code, sc = ref.quantise(x)
    held = ref.dequantise(code, sc)
    mags = ref.E2M1[:8]
    for r in range(40):
        for b in range(4):
            v = x[r, 32 * b:32 * b + 32].double()
            amax = float(v.abs().max())
            fits = [e for e in range(-125, 126) if amax <= 7 * 2.0 ** e]
            assert int(sc[r, b]) - 127 == fits[0]
            for i in range(32):
                y = abs(float(v[i])) / 2.0 ** fits[0]
                best = min(abs(y - m) for m in mags)
                near = [c for c in range(8) if abs(y - mags[c]) == best]
                want = near[0] if len(near) == 1 else [
                    c for c in near if c % 2 == 0][0]
                c = int(code[r, 32 * b + i])
                assert c % 8 == want and (c >= 8) == bool(
                    math.copysign(1.0, float(v[i])) < 0)
                assert abs(float(held[r, 32 * b + i]) - float(v[i])) <= (
                    2.0 ** fits[0])
    assert ref.block_scale(math.nan) == ref.block_scale(math.inf) == 255
    assert ref.block_scale(7 * 2.0 ** 125) == 252
    assert ref.block_scale(0.0) == 2


def test_oracle_attend():
    """Against scores made pair by pair in Python."""
    g = torch.Generator().manual_seed(1)
    T, N, hq, hkv = 3, 9, 2, 1
    q = torch.randn((T, hq, 128), generator=g)
    k, v = (torch.randn((N, hkv, 128), generator=g) for _ in range(2))
    slopes = torch.tensor([0.3, 0.1])
    rel = torch.randn((T, hq, 4), generator=g)
    first, prefix, window, cap, scale = [0, 2, 8], 7, 6, 3.0, 0.2
    out, lse, _, _ = ref.attend(
        q, k, v, torch.tensor([4, 5, 6]), torch.arange(N), scale, cap, slopes,
        rel, window, torch.tensor(first), prefix)
    for t, p in enumerate((4, 5, 6)):
        for h in range(hq):
            w, acc = 0.0, torch.zeros(128, dtype=torch.float64)
            for j in range(N):
                if j < first[t] or j > max(p, prefix - 1) or p - j >= window:
                    continue
                z = scale * sum(float(a) * float(b)
                                for a, b in zip(q[t, h], k[j, 0]))
                x = cap * math.tanh(z / cap) - float(slopes[h]) * abs(p - j)
                if 0 <= p - j < 4:
                    x += float(rel[t, h, p - j])
                w += math.exp(x)
                acc += math.exp(x) * v[j, 0].double()
            if w == 0.0:
                assert float(lse[h, t]) == -math.inf
                assert (out[t, h] == 0).all()
            else:
                assert abs(float(lse[h, t]) - math.log(w)) < 1e-5
                assert (out[t, h] - acc / w).abs().max() < 1e-5


def test_plain_forms_of_the_timed_cases():
    """perf/more_operators.py: its plain forms against its definition in 64
    bits, on the CPU, at small sizes: bf16 outputs, rounded once (2^-8 of the
    value; sums of up to 230 probabilities and 128 products in fp32 beside it,
    below 2^-14 of values up to 8), LSE in fp32."""
    m = importlib.import_module("perf.more_operators")
    keep, m.DEV = m.DEV, "cpu"
    try:
        base = dict(name="x", hq=8, hkv=2, lens=5, b=3, s=2, lo=20, hi=90,
                    prior_lo=30, prior_hi=100, t=33, cap=0.0, slopes=0, docs=0,
                    prefix=0, rel=0, window=0)
        for kind, kw in (
                ("decode", dict(cap=30.0, slopes=1, docs=1)),
                ("prefill", dict(cap=50.0, docs=1, prefix=1)),
                ("chunk", dict(slopes=1, docs=1, window=40)),
                ("decode4", dict(rel=1, window=33)),
                ("chunk4", dict(cap=30.0, slopes=1))):
            case = dict(base, kind=kind, **kw)
            for got, want in zip(m.run(m.prepare(case, 7)), m.exact(case, 7)):
                tol = 2.0 ** -8 if got.dtype == torch.bfloat16 else 2.0 ** -18
                assert ((got.double() - want).abs() <=
                        tol * want.abs() + 2.0 ** -14).all(), kind
            assert m.work(case)["flops"] > 0
        case = dict(base, kind="write4")
        for got, want in zip(m.run(m.prepare(case, 7)), m.exact(case, 7)):
            assert torch.equal(got.double(), want)
        import random
        assert len({repr(m.draw(random.Random(i))) for i in range(6)}) == 6
    finally:
        m.DEV = keep
