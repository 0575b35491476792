"""Timed cases of differential attention over the paged cache, and of the page
plan that a serving step builds on the GPU.

listed() holds the cases, draw() one more of the same ranges. A case is a dict
of plain values; "lens" seeds the lengths of its requests, so that the work of
a case does not depend on the seed of its data.

  kind     entry point          stands for
  decode   decode_diff_paged    one new token per request, over block tables
  prefill  prefill_diff_varlen  whole prompts, packed
  chunk    prefill_diff_varlen  a chunk of prompt after cached context, paged
  plan     plan_pages           a step's block table, slot map, positions and
                                run bounds from the requests' lengths, with
                                the pages its new tokens need
  release  release_pages        the pages of finished requests handed back

Differential attention (heads 2h and 2h + 1 are the two maps of pair h; stored
heads 2g and 2g + 1 hold their keys, and side by side pair g's 256-wide
values):

  O_h = softmax(q_2h K_2g^T s) V_g - lam_h softmax(q_2h+1 K_2g+1^T s) V_g
  out_h = O_h / sqrt(mean(O_h^2) + eps) * weight * out_scale

With `own` false, run() computes it in elementary torch operations; with it
true, by the package's operators.
"""
import importlib
import math
import random

import torch

own = False

PAGE, D = 16, 128
DEV = "cuda"
BF = torch.bfloat16
EPS = 1e-5
LAM_INIT = 0.784        # 0.8 - 0.6 exp(-0.3 l) at layer l = 12


# --------------------------------------------------------------------------
# the cases
# --------------------------------------------------------------------------

def listed():
    return [
        # a few short chats at once: the smallest attention call, where
        # launches and the host's work count
        dict(name="decode_b4", kind="decode", b=4, lo=128, hi=1024, window=0,
             hq=32, hkv=4, norm=1, lens=1),
        # a busy server's decode step, 1K-8K contexts
        dict(name="decode_b64", kind="decode", b=64, lo=1024, hi=8192,
             window=0, hq=32, hkv=4, norm=1, lens=2),
        # one user with one long document
        dict(name="decode_b1_long", kind="decode", b=1, lo=50001, hi=50001,
             window=0, hq=32, hkv=4, norm=1, lens=3),
        # a sliding-window layer's decode step, the model's window heads,
        # the plain difference
        dict(name="decode_window_b96", kind="decode", b=96, lo=200, hi=30000,
             window=512, hq=64, hkv=16, norm=0, lens=5),
        # packed prompts of 2K-8K tokens, the largest call
        dict(name="prefill_4_prompts", kind="prefill", s=4, lo=2048, hi=8192,
             window=0, hq=32, hkv=4, norm=1, lens=7),
        # one ordinary prompt of an odd length, the plain difference
        dict(name="prefill_b1_777", kind="prefill", s=1, lo=777, hi=777,
             window=0, hq=64, hkv=8, norm=0, lens=8),
        # one chunk of a long prompt after what is cached
        dict(name="chunk_500_after_15000", kind="chunk", s=1, lo=500, hi=500,
             prior_lo=15000, prior_hi=15000, window=0, hq=64, hkv=8, norm=1,
             lens=9),
        # the smallest plan: a decode step of four short chats
        dict(name="plan_b4", kind="plan", n_decode=4, lo=128, hi=1024,
             chunks=0, chunk=0, width=64, lens=11),
        # a busy server's decode step
        dict(name="plan_b64", kind="plan", n_decode=64, lo=1024, hi=8192,
             chunks=0, chunk=0, width=512, lens=12),
        # a continuous-batching step: two 2048-token chunks and 96 decode
        # rows of up to 64K tokens
        dict(name="plan_mixed", kind="plan", n_decode=96, lo=1024, hi=65536,
             chunks=2, chunk=2048, width=4224, lens=13),
        # one long request has finished
        dict(name="release_1", kind="release", n=1, lo=8000, hi=8000,
             width=512, lens=14),
        # a whole batch of long requests is dropped
        dict(name="release_64", kind="release", n=64, lo=1024, hi=65536,
             width=4096, lens=15),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["decode", "decode", "prefill", "chunk", "plan",
                       "release"])
    lens = rng.randrange(1, 1 << 20)
    # the configurations' heads, the model's two layer kinds, and shards of
    # them over 2 or 4 GPUs
    hq, hkv = rng.choice([(32, 4), (32, 4), (64, 8), (64, 16), (32, 8),
                          (16, 2)])
    norm = rng.choice([1, 1, 0])
    if kind == "decode":
        window = rng.choice([0, 0, 512, 4096])
        hi = _log(rng, 64, 65536)
        lo = max(1, int(hi * rng.choice([1.0, 0.5, 0.125])))
        vis = min(hi, window) if window else hi
        most = min(128, max(1, 500000 * 4 // (vis * hkv)))
        return dict(kind=kind, b=_log(rng, 1, most), lo=lo, hi=hi,
                    window=window, hq=hq, hkv=hkv, norm=norm, lens=lens)
    if kind == "prefill":
        hi = _log(rng, 16, 8192)
        most = min(8, max(1, int(4 * 8192 * 8192 * 32 / (hi * hi * hq))))
        return dict(kind=kind, s=_log(rng, 1, most), lo=max(1, hi // 8),
                    hi=hi, window=rng.choice([0, 0, 512, 4096]), hq=hq,
                    hkv=hkv, norm=norm, lens=lens)
    if kind == "chunk":
        hi = _log(rng, 1, 2048)
        s = rng.choice([1, 1, 2, 3])
        p = _log(rng, 16, min(32768, int(4e9 / (s * hi * hq))))
        return dict(kind=kind, s=s, lo=max(1, hi // 2), hi=hi,
                    prior_lo=p // 2, prior_hi=p,
                    window=rng.choice([0, 0, 4096]), hq=hq, hkv=hkv,
                    norm=norm, lens=lens)
    hi = _log(rng, 64, 65536)
    if kind == "plan":
        chunks = rng.choice([0, 0, 1, 2, 4])
        return dict(kind=kind, n_decode=_log(rng, 1, 256),
                    lo=max(1, hi // 8), hi=hi, chunks=chunks,
                    chunk=_log(rng, 16, 4096) if chunks else 0,
                    width=-(-(hi + 4096) // PAGE) + rng.randrange(8),
                    lens=lens)
    return dict(kind=kind, n=_log(rng, 1, 64), lo=max(1, hi // 8), hi=hi,
                width=-(-hi // PAGE) + rng.randrange(8), lens=lens)


# --------------------------------------------------------------------------
# lengths (from the case alone) and inputs (from the seed)
# --------------------------------------------------------------------------

def _lens(case):
    """[(new tokens, tokens before them)] of the requests."""
    r = random.Random(case["lens"])
    k = case["kind"]
    one = lambda: r.randint(case["lo"], case["hi"])        # noqa: E731
    if k == "decode":
        return [(1, one() - 1) for _ in range(case["b"])]
    if k == "prefill":
        return [(one(), 0) for _ in range(case["s"])]
    if k == "chunk":
        return [(one(), r.randint(case["prior_lo"], case["prior_hi"]))
                for _ in range(case["s"])]
    if k == "plan":
        return ([(case["chunk"], one() - 1) for _ in range(case["chunks"])] +
                [(1, one() - 1) for _ in range(case["n_decode"])])
    return [(0, one()) for _ in range(case["n"])]          # release


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _cu(lens):
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    return _i32(cu)


def _pages(n):
    return -(-n // PAGE)


def _gens(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    c = torch.Generator()
    c.manual_seed(seed)
    return g, c


def _rows(shape, g):
    return torch.randn(shape, generator=g, device=DEV, dtype=BF)


def _queries(shape, g):
    """Query rows whose heads are flat to peaked: scores of spread 0.5-3."""
    gain = torch.rand(shape[-2:-1], generator=g, device=DEV) * 2.5 + 0.5
    return (torch.randn(shape, generator=g, device=DEV) *
            gain[:, None]).to(BF)


def _values(shape, g):
    """Values around a mean of their own per head and dimension."""
    mean = torch.randn(shape[-2:], generator=g, device=DEV) * 0.25
    return (torch.randn(shape, generator=g, device=DEV) + mean).to(BF)


def _shuffled_table(pages, width, c):
    """Block table [len(pages), width] int32 of shuffled pages, out of a pool
    of twice as many (unused entries: -1). Returns (table, pool pages)."""
    total = 2 * sum(pages) + 1
    perm = torch.randperm(total, generator=c).to(torch.int32)
    t = torch.full((len(pages), width), -1, dtype=torch.int32)
    off = 0
    for r, n in enumerate(pages):
        t[r, :n] = perm[off:off + n]
        off += n
    return t, total


def _prepare_attention(case, seed):
    g, c = _gens(seed)
    lens = _lens(case)
    new, prior = [a for a, _ in lens], [b for _, b in lens]
    T, hq, hkv = sum(new), case["hq"], case["hkv"]
    ends = [a + b for a, b in lens]
    lam = LAM_INIT + 0.1 * torch.randn(hq // 2, generator=g, device=DEV)
    weight = 1 + 0.1 * torch.randn(2 * D, generator=g, device=DEV)
    st = dict(case=case, q=_queries((T, hq, D), g), lam=lam,
              weight=weight if case["norm"] else None,
              out_scale=1 - LAM_INIT if case["norm"] else 1.0,
              scale=D ** -0.5, window=case["window"], cu=_cu(new),
              prior=_i32(prior), longest=max(new), most=max(ends))
    if case["kind"] == "prefill":
        st.update(k=_rows((T, hkv, D), g), v=_values((T, hkv, D), g))
    else:
        t, P = _shuffled_table([_pages(n) for n in ends],
                               _pages(max(ends)), c)
        st.update(ctx=_i32(ends), table=t.to(DEV),
                  kp=_rows((P, PAGE, hkv, D), g),
                  vp=_values((P, PAGE, hkv, D), g))
    return st


def _prepare_pages(case, seed):
    """A cache's page table with rows for twice the step's requests, and the
    stack of its free pages."""
    g, c = _gens(seed)
    lens = _lens(case)
    B, W = len(lens), case["width"]
    S = 2 * B + 1
    slots = torch.randperm(S, generator=c)[:B]
    held = [_pages(b) for _, b in lens]
    need = sum(_pages(a + b) for a, b in lens) - sum(held)
    t, P = _shuffled_table(held, W, c)
    used = torch.zeros(P, dtype=torch.bool)
    used[t[t >= 0].long()] = True
    free = torch.nonzero(~used)[:, 0].to(torch.int32)
    free = free[torch.randperm(free.numel(), generator=c)]
    extra = torch.arange(P, P + need, dtype=torch.int32)   # enough for all
    free = torch.cat([extra, free])
    stack = torch.full((P + need,), -1, dtype=torch.int32)
    stack[:free.numel()] = free
    table = torch.full((S, W), -1, dtype=torch.int32)
    table[slots] = t
    return dict(case=case, table=table.to(DEV), slots=slots.to(DEV),
                ctx=_i32([b for _, b in lens]), new=_i32([a for a, _ in lens]),
                free=stack.to(DEV), count=_i32([free.numel()]),
                tokens=sum(a for a, _ in lens))


def prepare(case, seed):
    if case["kind"] in ("plan", "release"):
        return _prepare_pages(case, seed)
    return _prepare_attention(case, seed)


# --------------------------------------------------------------------------
# one pass
# --------------------------------------------------------------------------

def _difference(st, q, K, V, kpos, qpos):
    """q [S, T, HQ, D] at positions qpos [S, T], keys and values [S, N, HKV,
    D] at positions kpos [S, N] (negative: none), all fp32. Returns
    (out [S, T, HQ / 2, 2 D], lse [S, T, HQ]), fp32."""
    S, T, hq, _ = q.shape
    N, hkv = K.shape[1], K.shape[2]
    G, rep = hkv // 2, hq // hkv
    # [S, HKV, rep * T, D]: the queries of stored head 2g + m
    x = q.view(S, T, G, rep, 2, D).permute(0, 2, 4, 3, 1, 5)
    x = x.reshape(S, hkv, rep * T, D)
    s = torch.matmul(x, K.permute(0, 2, 3, 1)).mul_(st["scale"])
    dist = qpos[:, :, None] - kpos[:, None, :]
    dead = (dist < 0) | (kpos < 0)[:, None, :]
    if st["window"]:
        dead |= dist >= st["window"]
    s = s.view(S, hkv, rep, T, N)
    s.masked_fill_(dead[:, None, None], -math.inf)
    m = s.amax(-1, keepdim=True).clamp_(min=-3e38)
    s.sub_(m).exp_()
    l = s.sum(-1, keepdim=True)
    lse = (m + torch.log(l))[..., 0]
    s.div_(torch.where(l > 0, l, 1.0))
    V = V.reshape(S, N, G, 2 * D).transpose(1, 2)
    o = torch.matmul(s.view(S, G, 2 * rep * T, N), V)
    o = o.view(S, G, 2, rep, T, 2 * D)
    lam = st["lam"].view(G, rep)[None, :, :, None, None]
    o = (o[:, :, 0] - lam * o[:, :, 1]).permute(0, 3, 1, 2, 4)
    o = o.reshape(S, T, hq // 2, 2 * D)
    if st["weight"] is not None:
        o = o * torch.rsqrt(o.square().mean(-1, keepdim=True) + EPS)
        o = o * st["weight"]
    lse = lse.view(S, G, 2, rep, T).permute(0, 4, 1, 3, 2)
    return o * st["out_scale"], lse.reshape(S, T, hq)


def _cached(st, pool, kpos):
    """Pool rows at positions kpos [S, N] of the requests, fp32."""
    p = kpos.clamp(min=0)
    pages = torch.gather(st["table"].long(), 1, p // PAGE)
    return pool[pages, p % PAGE].float()


def _decode(st):
    ctx = st["ctx"].long()
    n = min(st["most"], st["window"]) if st["window"] else st["most"]
    kpos = ctx[:, None] - n + torch.arange(n, device=DEV)
    o, lse = _difference(st, st["q"].float()[:, None],
                         _cached(st, st["kp"], kpos),
                         _cached(st, st["vp"], kpos), kpos, ctx[:, None] - 1)
    return o[:, 0].to(BF), lse[:, 0]


def _prefill(st):
    cu, prior = st["cu"].long(), st["prior"].long()
    T = st["q"].shape[0]
    t = torch.arange(T, device=DEV)
    run = torch.searchsorted(cu[1:], t, right=True)
    j = t - cu[run]
    pad = torch.arange(st["longest"], device=DEV)
    new = (cu[1:] - cu[:-1])[:, None]
    row = (cu[:-1, None] + pad).clamp(max=T - 1)
    qpos = torch.where(pad < new, prior[:, None] + pad, -1)
    if "k" in st:
        kpos, K, V = qpos, st["k"].float()[row], st["v"].float()[row]
    else:
        n = torch.arange(st["most"], device=DEV)
        kpos = torch.where(n < prior[:, None] + new, n, -1)
        K, V = _cached(st, st["kp"], kpos), _cached(st, st["vp"], kpos)
    o, lse = _difference(st, st["q"].float()[row], K, V, kpos, qpos)
    return o[run, j].to(BF), lse[run, j].t().contiguous()


def _plan(st):
    table, slots, free = st["table"], st["slots"], st["free"]
    ctx, new = st["ctx"].long(), st["new"].long()
    S, W = table.shape
    end = ctx + new
    old, have = (ctx + 15) // PAGE, (end + 15) // PAGE
    need = (have - old).cumsum(0)
    first = need - (have - old)
    cu = torch.cat([new.new_zeros(1), new.cumsum(0)])
    uses = torch.zeros(S, dtype=torch.int32, device=DEV)
    uses.index_add_(0, slots, torch.ones_like(slots, dtype=torch.int32))
    bad = ((need[-1] > st["count"][0]) | (cu[-1] > st["tokens"]) |
           (have.amax() > W) | (uses.amax() > 1))
    j = torch.arange(W, device=DEV)
    fresh = (j >= old[:, None]) & (j < have[:, None])
    top = st["count"].long() - 1 - first[:, None] - (j - old[:, None])
    rows = torch.where(fresh, free[top.clamp(0, free.numel() - 1)],
                       table[slots])
    table[slots] = torch.where(bad, table[slots], rows)
    block = torch.where((j < have[:, None]) & ~bad, rows, -1)
    t = torch.arange(st["tokens"], device=DEV)
    run = torch.searchsorted(cu[1:], t, right=True).clamp_(max=len(slots) - 1)
    pos = ctx[run] + t - cu[run]
    page = block[run, (pos // PAGE).clamp(max=W - 1)].long()
    live = (t < cu[-1]) & ~bad
    return (table, block, torch.where(bad, ctx, end).int(),
            torch.where(bad, 0, cu).int(),
            torch.where(live & (page >= 0), page * PAGE + pos % PAGE, -1),
            torch.where(live, pos, 0),
            st["count"] - torch.where(bad, 0, need[-1:]).int(),
            bad.int().view(1))


def _release(st):
    free, count = st["free"], st["count"].long()
    n = (st["ctx"].long() + 15) // PAGE
    end = n.cumsum(0)
    bad = count + end[-1] > free.numel()
    k = torch.arange(free.numel(), device=DEV) - count
    r = torch.searchsorted(end, k, right=True).clamp_(max=n.numel() - 1)
    j = (k - (end - n)[r]).clamp_(0, st["table"].shape[1] - 1)
    put = (k >= 0) & (k < end[-1]) & ~bad
    free.copy_(torch.where(put, st["table"][st["slots"][r], j], free))
    return free, (count + torch.where(bad, 0, end[-1])).int(), bad.int()


def run(st):
    k = st["case"]["kind"]
    if not own:
        return {"decode": _decode, "prefill": _prefill, "chunk": _prefill,
                "plan": _plan, "release": _release}[k](st)
    tm = importlib.import_module("tm-opt_amd")
    if k == "decode":
        return tm.decode_diff_paged(
            st["q"], st["kp"], st["vp"], st["table"], st["ctx"], st["lam"],
            st["scale"], norm_weight=st["weight"], norm_eps=EPS,
            out_scale=st["out_scale"], window=st["window"])
    if k == "prefill":
        return tm.prefill_diff_varlen(
            st["q"], st["k"], st["v"], st["cu"], st["lam"], st["scale"],
            norm_weight=st["weight"], norm_eps=EPS,
            out_scale=st["out_scale"], window=st["window"],
            max_seqlen=st["longest"])
    if k == "chunk":
        return tm.prefill_diff_varlen(
            st["q"], None, None, st["cu"], st["lam"], st["scale"],
            norm_weight=st["weight"], norm_eps=EPS,
            out_scale=st["out_scale"], window=st["window"],
            max_seqlen=st["longest"], prior_lens=st["prior"],
            k_pool=st["kp"], v_pool=st["vp"], block_table=st["table"])
    if k == "plan":
        p = tm.plan_pages(st["table"], st["slots"], st["ctx"], st["new"],
                          st["free"], st["count"], st["tokens"])
        return (st["table"], p.block_table, p.seq_lens, p.cu_seqlens,
                p.slot_mapping, p.positions, p.free_count, p.reject)
    count, reject = tm.release_pages(st["table"], st["slots"], st["ctx"],
                                     st["free"], st["count"])
    return st["free"], count, reject


# --------------------------------------------------------------------------
# what a pass cannot do without
# --------------------------------------------------------------------------

def _pairs(new, prior, window):
    """Visible (query, key) pairs of a run."""
    if not window:
        return new * prior + new * (new + 1) // 2
    full = min(max(window - prior, 0), new)     # queries seeing all keys
    return (full * prior + full * (full + 1) // 2 + (new - full) * window)


def work(case):
    k = case["kind"]
    lens = _lens(case)
    if k == "plan":
        old = sum(_pages(b) for _, b in lens)
        need = sum(_pages(a + b) for a, b in lens) - old
        T, B = sum(a for a, _ in lens), len(lens)
        return {"bytes": 16 * B + 4 * old + 8 * need +
                4 * B * case["width"] + 8 * B + 16 * T + 16, "flops": 0}
    if k == "release":
        return {"bytes": 12 * len(lens) + 12 +
                8 * sum(_pages(b) for _, b in lens), "flops": 0}
    hq, hkv, w = case["hq"], case["hkv"], case["window"]
    T = sum(a for a, _ in lens)
    keys = sum(a + (min(b, w - 1) if w else b) for a, b in lens)
    table = 0 if k == "prefill" else 4 * sum(
        _pages(a + (min(b, w - 1) if w else b)) for a, b in lens)
    # scores over 128 dims for each of the HQ maps, each times 256-wide values
    return {"bytes": 4 * T * hq * D + 4 * T * hq + 4 * keys * hkv * D + table,
            "flops": 2 * 3 * D * hq * sum(_pairs(a, b, w) for a, b in lens)}


# --------------------------------------------------------------------------
# the same in 64 bits, request by request and pair by pair
# --------------------------------------------------------------------------

def _exact_run(st, q, K, V, first, kfirst):
    """One request: q [T, HQ, D] at positions first.., K, V [N, HKV, D] at
    positions kfirst..; float64 (out [T, HQ / 2, 2 D], lse [HQ, T])."""
    T, hq, _ = q.shape
    N, hkv = K.shape[0], K.shape[1]
    rep = hq // hkv
    out = torch.empty((T, hq // 2, 2 * D), dtype=torch.float64, device=DEV)
    lse = torch.empty((hq, T), dtype=torch.float64, device=DEV)
    key = torch.arange(kfirst, kfirst + N, device=DEV)
    for a in range(0, T, 2048):
        rows = slice(a, min(a + 2048, T))
        at = torch.arange(first + rows.start, first + rows.stop, device=DEV)
        seen = key[None, :] <= at[:, None]
        if st["window"]:
            seen &= key[None, :] > at[:, None] - st["window"]
        for h in range(hq // 2):
            g = h // rep
            v = torch.cat([V[:, 2 * g], V[:, 2 * g + 1]], 1).double()
            o = []
            for m in (0, 1):
                z = q[rows, 2 * h + m].double() @ K[:, 2 * g + m].double().t()
                z = torch.where(seen, z * st["scale"], -math.inf)
                lse[2 * h + m, rows] = torch.logsumexp(z, 1)
                o.append(torch.softmax(z, 1) @ v)
            out[rows, h] = o[0] - st["lam"][h].double() * o[1]
    if st["weight"] is not None:
        ms = (out * out).sum(2, keepdim=True) / (2 * D)
        out = out / torch.sqrt(ms + EPS) * st["weight"].double()
    return out * st["out_scale"], lse


def exact(case, seed):
    """None for whole-number outputs."""
    if case["kind"] in ("plan", "release"):
        return None
    st = prepare(case, seed)
    outs, lses, t = [], [], 0
    for r, (a, b) in enumerate(_lens(case)):
        if "k" in st:
            lo, K, V = 0, st["k"][t:t + a], st["v"][t:t + a]
        else:
            lo = max(0, b - case["window"] + 1) if case["window"] else 0
            p = torch.arange(lo, a + b, device=DEV)
            pg = st["table"][r, p // PAGE].long()
            K, V = st["kp"][pg, p % PAGE], st["vp"][pg, p % PAGE]
        o, l = _exact_run(st, st["q"][t:t + a], K, V, b, lo)
        outs.append(o)
        lses.append(l)
        t += a
    lse = torch.cat(lses, 1)
    return torch.cat(outs), lse.t() if case["kind"] == "decode" else lse
