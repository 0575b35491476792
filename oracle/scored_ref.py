"""Attention with score functions, and the 4-bit cache, from their definitions
(TEST INFRASTRUCTURE ONLY): float64, no tiling, no split.

With each output comes how far a right kernel may be from it. A score of a key
is off by dx, the sum of
  * (128 + 4) x 2^-24 of sum |q_i k_i| scale: 128 exact products added in fp32,
    and the scale;
  * the cap: 2^-19 of it. softcap tanh(z / softcap) moves by at most what z
    moves; the tanh itself may be off by 2^-20 (in fp32 a t = exp(2 y) off by
    2 x 2^-23 of itself, 1 + t rounded, its reciprocal off by 2^-23 and a last
    rounding add up to 5.5 x 2^-23 < 2^-20), and so may its argument: 4 x 2^-24
    of y sech^2(y) is less than 2^-22. Of a cap above 256 that would be more than
    2^-11, so there it is 2^-18 of z at most: up to |z| = cap / 2 a polynomial in y
    takes the tanh's place, off by 2^-18.7 of y (y -> 0, where its error is the
    largest share of it) and by some roundings of 2^-24, and beyond 2^-20 of the
    cap is 2^-19 of z;
  * a bias of size w: 4 x 2^-24 (w + |x|) for its product and the sum, and
    bf16 biases are exact. Slopes may also join q.k as the first term of its
    sum: then each of the eight sums of 16 products rounds at their size, by
    2^-23 w at most, 16 x 2^-24 w in all.
Then p changes by p dx relative to the rest, so LSE = log sum exp is off by at
most sum p dx (and n x 2^-24 for a sum of n terms, 16 x 2^-24 for exp2, log2 and
the last products, and 8 x 2^-24 of |LSE| and of the maximum). Outputs: p is
rounded to bf16 for its product with the values, half a step is 2^-8 of it, so O
is off by sum p (2^-8 + dx + dLSE + (2 n + 64) 2^-24) |v|, and rounded once more
(2^-8 of it). A probability below 2^-126 of its reference point is no normal fp32
number and may count as zero, once in its key's walk, where the reference may be
2^40 above the largest, and once when pieces join: 2^-85 of sum |v|. A tenth is
added for products of errors.
"""
import math

import torch

PAGE, D = 16, 128
HALF_BF16 = 2.0 ** -8
HALF_F32 = 2.0 ** -24
RECORD = 2176

# code -> value of an element
E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
E2M1 += [-x for x in E2M1]


# --------------------------------------------------------------------------
# the 4-bit cache
# --------------------------------------------------------------------------

def block_scale(amax):
    """Scale byte of a block by its largest magnitude (a Python float)."""
    if not amax <= 7 * 2.0 ** 125:
        return 255
    e = -125
    while amax > 7 * 2.0 ** e:
        e += 1
    return e + 127


def quantise(x):
    """x [..., 128] (CPU): (codes [..., 128], scale bytes [..., 4]) int64."""
    shape = x.shape[:-1]
    x = x.double().reshape(-1, 32)
    sc = torch.tensor([block_scale(float(a)) for a in x.abs().amax(-1)])
    bad = sc == 255
    step = torch.tensor([2.0 ** (int(s) - 127) for s in sc.clamp(max=254)],
                        dtype=torch.float64)
    y = torch.where(bad[:, None], 0.0, x / step[:, None])
    grid = torch.tensor(E2M1[:8], dtype=torch.float64)
    d = (y.abs()[..., None] - grid).abs()
    # nearest; of two as near the even code
    d = d + torch.tensor([0.0, 1.0] * 4, dtype=torch.float64) * 1e-12
    code = d.argmin(-1) + 8 * torch.signbit(y)
    return code.view(*shape, 128), sc.view(*shape, 4)


def dequantise(code, sc):
    """float64 [..., 128] of codes and scale bytes (255: NaN)."""
    power = torch.tensor([2.0 ** (i - 127) for i in range(255)] + [math.nan],
                         dtype=torch.float64)
    val = torch.tensor(E2M1, dtype=torch.float64)[code]
    return val * power[sc].repeat_interleave(32, -1)


def held(x):
    """What the cache holds of rows x [..., 128], float64 (CPU)."""
    return dequantise(*quantise(x))


def put(pool, row, k, v):
    """Write token rows k, v [HKV, 128] at pool row `row`: pool [P, HKV, 2176]
    uint8 (CPU), byte by byte."""
    page, t = row // PAGE, row % PAGE
    for x, is_v in ((k, 0), (v, 1)):
        code, sc = quantise(x)
        pair = (code[:, 0::2] | code[:, 1::2] << 4).to(torch.uint8)
        for i in range(64):
            at = 1024 + i // 4 * 64 + t * 4 + i % 4 if is_v else t * 64 + i
            pool[page, :, at] = pair[:, i]
        for b in range(4):
            pool[page, :, 2048 + 64 * is_v + b * 16 + t] = sc[:, b].to(
                torch.uint8)


# --------------------------------------------------------------------------
# attention
# --------------------------------------------------------------------------

def attend(q, K, V, qpos, kpos, scale, softcap=0.0, slopes=None, rel=None,
           window=0, first=None, prefix=0):
    """q [T, HQ, 128] at qpos [T], K and V [N, HKV, 128] at kpos [N]; rel
    [T, HQ, E]; first [T]. Returns float64 (out [T, HQ, 128], lse [HQ, T], and
    the bounds of both)."""
    T, HQ, _ = q.shape
    N, HKV = K.shape[0], K.shape[1]
    q, K, V = q.double(), K.double(), V.double()
    dist = qpos[:, None] - kpos[None, :]
    seen = kpos[None, :] <= torch.clamp(qpos, min=prefix - 1)[:, None]
    if window:
        seen &= dist < window
    if first is not None:
        seen &= kpos[None, :] >= first[:, None]
    # (rows that no query sees may hold anything)
    V = torch.where(seen.any(0)[:, None, None], V, 0.0)
    out = q.new_zeros((T, HQ, D))
    err = torch.zeros_like(out)
    lse = q.new_full((HQ, T), -math.inf)
    lerr = torch.zeros_like(lse)
    if N == 0:
        return out, lse, err + 1e-30, lerr
    for h in range(HQ):
        g = h // (HQ // HKV)
        x = q[:, h] @ K[:, g].T * scale
        dx = (128 + 4) * HALF_F32 * (q[:, h].abs() @ K[:, g].abs().T * scale)
        if softcap:
            share = softcap * 2.0 ** -19
            if softcap > 256:
                share = torch.clamp(2.0 ** -18 * x.abs(), max=share)
            x = softcap * torch.tanh(x / softcap)
            dx = dx + share
        if slopes is not None:
            w = slopes[h].double() * dist.abs()
            x = x - w
            dx = dx + HALF_F32 * (20 * w.abs() + 4 * x.abs())
        if rel is not None:
            E = rel.shape[2]
            b = rel[:, h].double().gather(1, dist.clamp(0, E - 1))
            b = torch.where((dist >= 0) & (dist < E), b, 0.0)
            x = x + b
            dx = dx + 4 * HALF_F32 * (b.abs() + x.abs())
        x = x.masked_fill(~seen, -math.inf)
        l = torch.logsumexp(x, 1)
        some = seen.any(1)
        p = torch.exp(x - torch.where(some, l, 0.0)[:, None])
        p = torch.where(seen, p, 0.0)
        n = seen.sum(1)
        big = torch.where(some, x.masked_fill(~seen, -1e300).amax(1).abs(),
                          0.0)
        dl = (p * torch.where(seen, dx, 0.0)).sum(1) + (
            n + 16 + 8 * (l.abs().nan_to_num(0.0, 0.0) + big)) * HALF_F32
        each = HALF_BF16 + dx + dl[:, None] + (2 * n[:, None] + 64) * HALF_F32
        out[:, h] = p @ V[:, g]
        err[:, h] = (p * torch.where(seen, each, 0.0)) @ V[:, g].abs()
        err[:, h] += 2.0 ** -85 * (seen.double() @ V[:, g].abs())
        lse[h], lerr[h] = l, torch.where(some, dl, 0.0)
    return out, lse, 1.1 * (err + HALF_BF16 * out.abs()) + 1e-30, 1.1 * lerr


def rows_of(pool, table_row, pos, table_wrap=0):
    """Pool rows at positions pos of one request."""
    lp = pos // PAGE
    if table_wrap:
        lp = lp % table_wrap
    return pool[table_row[lp].long(), pos % PAGE]


def decode(q, k_pool, v_pool, table, ctx, scale, window=0, table_wrap=0,
           first=None, rel=None, **kw):
    """Request by request (table entries must be pages); pools [P, 16, HKV,
    128] of the values held."""
    parts = []
    for b in range(q.shape[0]):
        n = int(ctx[b])
        lo = max(0, n - window) if window else 0
        pos = torch.arange(lo, max(n, 0), device=q.device)
        o, l, e, le = attend(
            q[b:b + 1], rows_of(k_pool, table[b], pos, table_wrap),
            rows_of(v_pool, table[b], pos, table_wrap),
            torch.tensor([n - 1], device=q.device), pos, scale, window=window,
            first=None if first is None else first[b:b + 1],
            rel=None if rel is None else rel[b:b + 1], **kw)
        parts.append((o, l.T, e, le.T))
    return tuple(torch.cat(x) for x in zip(*parts))


def prefill(q, k, v, cu, scale, prior=None, k_pool=None, v_pool=None,
            table=None, window=0, first=None, prefix=None, rel=None, **kw):
    """Run by run; keys from k, v [total, HKV, 128] or through the table."""
    T, HQ, _ = q.shape
    out = torch.zeros((T, HQ, D), dtype=torch.float64, device=q.device)
    err = torch.zeros_like(out)
    lse = torch.full((HQ, T), -math.inf, dtype=torch.float64, device=q.device)
    lerr = torch.zeros_like(lse)
    cu = [int(x) for x in cu]
    for i in range(len(cu) - 1):
        a, b = cu[i], cu[i + 1]
        if a == b:
            continue
        p = 0 if prior is None else int(prior[i])
        kpos = torch.arange(0, p + b - a, device=q.device)
        if table is None:
            K, V = k[a:b], v[a:b]
        else:
            kpos = kpos[max(0, p - window + 1) if window else 0:]
            K = rows_of(k_pool, table[i], kpos)
            V = rows_of(v_pool, table[i], kpos)
        out[a:b], lse[:, a:b], err[a:b], lerr[:, a:b] = attend(
            q[a:b], K, V, torch.arange(p, p + b - a, device=q.device), kpos,
            scale, window=window,
            first=None if first is None else first[a:b],
            prefix=0 if prefix is None else int(prefix[i]),
            rel=None if rel is None else rel[a:b], **kw)
    return out, lse, err, lerr


def check(got, lse, ref, what=""):
    """Assert that a kernel's (out, lse) are within the bounds of ref."""
    out, ref_lse, err, lerr = ref
    got = got.double()
    assert torch.isfinite(got).all(), f"{what}: non-finite output"
    far = (got - out).abs() / err
    assert far.amax() <= 1, (
        f"{what}: {int((far > 1).sum())} of {far.numel()} outputs outside "
        f"their bound, worst {float(far.amax()):.3g} of it")
    if lse is not None:
        fin = torch.isfinite(ref_lse)
        assert torch.equal(fin, torch.isfinite(lse)), f"{what}: LSE finiteness"
        assert (lse[~fin] == -math.inf).all(), f"{what}: LSE of empty rows"
        d = (lse.double() - ref_lse).abs()[fin]
        assert (d <= lerr[fin]).all(), (
            f"{what}: LSE {float((d / lerr[fin]).amax()):.3g} of its bound")
