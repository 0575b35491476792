"""Differential attention and the page plan from their definitions (TEST
INFRASTRUCTURE ONLY): float64 and Python integers, no tiling, no split.

With each output comes how far a right kernel may be from it. Probabilities are
rounded to bf16 before their product with the values: half a step is 2^-8 of
the value, so O_m is off by at most 2^-8 A_m, A_m = sum_j p_j |v_j|, and the
difference by 2^-8 (A_1 + |lam| A_2). The norm multiplies by r = (mean O^2 +
eps)^-1/2, whose relative change is at most r^2 mean(|O| |dO|). The output is
rounded once more (2^-8 of it). What fp32 adds (a score of 128 products, each
exact, is off by at most 128 x 2^-24 of the sum of their sizes; sums of n
probabilities by n x 2^-24) is counted too, and a tenth of everything for
products of errors.

Over long contexts these bounds, which add every rounding with one sign, pass
the outputs themselves. power_inputs() makes inputs for which they need not be
added: scores that are whole numbers of powers of two (scale ln 2, whose
product with log2 e is 1 in fp32, queries of two entries of 1 or -1, keys of
-1, 0 and 1) and values of -2 to 2. Probabilities are then 2^-4 to 2^4, bf16
holds them as they are, and all sums within a piece are multiples of 2^-4 below
2^20: fp32 holds them too. What is left is each piece's LSE (below 22: log2 by
2^-19, its sum with the maximum by 2^-20, the product with ln 2 by 2^-20 and
ln 2 itself by 2^-20.5: 3.6e-6) that weighs it, and up to 64 roundings of
2^-24 in a join, both above and below the line: 1.5e-5, below 2^-16
(exact=True)."""
import math

import torch

PAGE = 16
HALF_BF16 = 2.0 ** -8
HALF_F32 = 2.0 ** -24


def power_inputs(T, N, hq, hkv, g):
    """q [T, hq, 128], k and v [N, hkv, 128] (bf16) for exact=True, scale
    ln 2."""
    q = torch.zeros((T, hq, 128))
    at = torch.rand((T, hq, 128), generator=g).topk(2, -1).indices
    q.scatter_(-1, at, torch.randint(0, 2, at.shape, generator=g) * 2.0 - 1)
    k = torch.randint(-1, 2, (N, hkv, 128), generator=g, dtype=torch.int8)
    v = torch.randint(-2, 3, (N, hkv, 128), generator=g, dtype=torch.int8)
    return q.bfloat16(), k.bfloat16(), v.bfloat16()


def attend(q, K, V, qpos, kpos, lam, scale, weight=None, eps=1e-5,
           out_scale=1.0, window=0, exact=False):
    """q [T, HQ, 128] at qpos [T], K and V [N, HKV, 128] at kpos [N]; exact:
    inputs of power_inputs(). Returns float64 (out [T, HQ/2, 256], lse [HQ, T],
    and the bounds of both)."""
    T, HQ, D = q.shape
    N, HKV = K.shape[0], K.shape[1]
    rep = HQ // HKV
    q, K, V = q.double(), K.double(), V.double()
    dist = qpos[:, None] - kpos[None, :]
    seen = dist >= 0
    if window:
        seen &= dist < window
    out = q.new_zeros((T, HQ // 2, 2 * D))
    err = torch.zeros_like(out)
    lse = q.new_full((HQ, T), -math.inf)
    lerr = torch.zeros_like(lse)
    for h in range(HQ // 2):
        g = h // rep
        v = torch.cat([V[:, 2 * g], V[:, 2 * g + 1]], 1)
        for m in range(2):
            x, k = q[:, 2 * h + m], K[:, 2 * g + m]
            s = (x @ k.T * scale).masked_fill(~seen, -math.inf)
            size = (x.abs() @ k.abs().T * scale).masked_fill(~seen, 0.0)
            ds = ((128 + 4) * HALF_F32 * size).amax(1) if N else lerr[0]
            lse[2 * h + m] = torch.logsumexp(s, 1)
            big = s.clamp(min=-1e30).amax(1).abs() if N else lerr[0]
            lerr[2 * h + m] = ds + (N + 16) * HALF_F32 + 8 * HALF_F32 * (
                big + 10)
            p = torch.exp(s - lse[2 * h + m][:, None]).nan_to_num(0.0)
            f = lam[h if lam.numel() > 1 else 0].double()
            f = 1.0 if m == 0 else -float(f)
            out[:, h] += f * (p @ v)
            rel = HALF_BF16 + 2 * ds + (2 * N + 64) * HALF_F32
            if exact:
                rel = torch.full_like(rel, 2.0 ** -16)
                lerr[2 * h + m] = 2.0 ** -16
            err[:, h] += abs(f) * rel[:, None] * (p @ v.abs())
    if weight is not None:
        r = 1.0 / torch.sqrt(out.square().mean(-1, keepdim=True) + eps)
        y = out * r * weight.double()
        turn = r * r * (out.abs() * err).mean(-1, keepdim=True)
        err = err * r * weight.double().abs() + y.abs() * turn
        out = y
    out, err = out * out_scale, err * abs(out_scale)
    return out, lse, 1.1 * err + 1.1 * HALF_BF16 * out.abs() + 1e-30, lerr


def rows_of(pool, table_row, pos, table_wrap=0):
    """Pool rows at positions pos of one request."""
    lp = pos // PAGE
    if table_wrap:
        lp = lp % table_wrap
    return pool[table_row[lp].long(), pos % PAGE]


def decode(q, k_pool, v_pool, table, ctx, lam, scale, window=0, table_wrap=0,
           **kw):
    """decode_diff_paged, request by request (table entries must be pages)."""
    parts = []
    for b in range(q.shape[0]):
        n = int(ctx[b])
        lo = max(0, n - window) if window else 0
        pos = torch.arange(lo, max(n, 0), device=q.device)
        o, l, e, le = attend(
            q[b:b + 1], rows_of(k_pool, table[b], pos, table_wrap),
            rows_of(v_pool, table[b], pos, table_wrap),
            torch.tensor([n - 1], device=q.device), pos, lam, scale,
            window=window, **kw)
        parts.append((o, l.T, e, le.T))
    return tuple(torch.cat(x) for x in zip(*parts))


def prefill(q, k, v, cu, lam, scale, prior=None, k_pool=None, v_pool=None,
            table=None, window=0, **kw):
    """prefill_diff_varlen, run by run."""
    T, HQ, D = q.shape
    out = torch.zeros((T, HQ // 2, 2 * D), dtype=torch.float64,
                      device=q.device)
    err = torch.zeros_like(out)
    lse = torch.full((HQ, T), -math.inf, dtype=torch.float64, device=q.device)
    lerr = torch.zeros_like(lse)
    cu = [int(x) for x in cu]
    for i in range(len(cu) - 1):
        a, b = cu[i], cu[i + 1]
        p = 0 if prior is None else int(prior[i])
        kpos = torch.arange(0, p + b - a, device=q.device)
        if table is None:
            K, V = k[a:b], v[a:b]
        else:
            lo = max(0, p - window + 1) if window else 0
            kpos = kpos[lo:]
            K = rows_of(k_pool, table[i], kpos)
            V = rows_of(v_pool, table[i], kpos)
        out[a:b], lse[:, a:b], err[a:b], lerr[:, a:b] = attend(
            q[a:b], K, V, torch.arange(p, p + b - a, device=q.device), kpos,
            lam, scale, window=window, **kw)
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
        d = (lse.double() - ref_lse).abs()[fin]
        assert (d <= lerr[fin]).all(), (
            f"{what}: LSE {float((d / lerr[fin]).amax()):.3g} of its bound")


def plan(page_table, slots, ctx, new, free, count, max_tokens, width=None):
    """plan_pages over Python lists; page_table and free are not changed.
    Returns (page_table, block, seq, cu, slot_mapping, positions, count,
    reject)."""
    table = [list(r) for r in page_table]
    S, W, B = len(table), len(table[0]), len(slots)
    width = W if width is None else width
    pages = lambda n: (n + PAGE - 1) // PAGE               # noqa: E731
    live = [i for i in range(B) if slots[i] >= 0]
    bad = not 0 <= count <= len(free)
    bad |= len({slots[i] for i in live}) < len(live)
    need = tokens = 0
    for i in live:
        bad |= slots[i] >= S or ctx[i] < 0 or new[i] < 0
        bad |= ctx[i] + new[i] > PAGE * min(W, width)
        need += pages(ctx[i] + new[i]) - pages(ctx[i])
        tokens += new[i]
    bad |= tokens > max_tokens or need > count
    block = [[-1] * width for _ in range(B)]
    seq = [ctx[i] if slots[i] >= 0 else 0 for i in range(B)]
    cu, where, at = [0], [-1] * max_tokens, [0] * max_tokens
    for i in range(B):
        add = 0 if bad or slots[i] < 0 else new[i]
        if not bad and slots[i] >= 0:
            row = table[slots[i]]
            for j in range(pages(ctx[i]), pages(ctx[i] + add)):
                count -= 1
                row[j] = free[count]
            n = pages(ctx[i] + add)
            block[i][:n] = row[:n]
        for t in range(add):
            p = seq[i] + t
            pg = block[i][p // PAGE]
            where[cu[-1] + t] = -1 if pg < 0 else pg * PAGE + p % PAGE
            at[cu[-1] + t] = p
        seq[i] += add
        cu.append(cu[-1] + add)
    return table, block, seq, cu, where, at, count, int(bad)


def release(page_table, slots, lens, free, count):
    """release_pages over Python lists. Returns (free, count, reject)."""
    S, W = len(page_table), len(page_table[0])
    live = [i for i in range(len(slots)) if slots[i] >= 0]
    bad = not 0 <= count <= len(free)
    bad |= len({slots[i] for i in live}) < len(live)
    back = []
    for i in live:
        if slots[i] >= S or not 0 <= lens[i] <= PAGE * W:
            bad = True
            continue
        row = page_table[slots[i]][:(lens[i] + PAGE - 1) // PAGE]
        back += [p for p in row if p >= 0]         # (the others name no page)
    if bad or count + len(back) > len(free):
        return list(free), count, 1
    free = list(free)
    free[count:count + len(back)] = back
    return free, count + len(back), 0
