"""Timed cases of attention with score functions (a tanh cap, a bias by
distance, document and prefix masks) and of attention over a cache held in 4
bits, with the write that quantises its rows.

listed() holds the cases, draw() one more of the same ranges. A case is a dict
of plain values; "lens" seeds the lengths of its requests, so that the work of
a case does not depend on the seed of its data.

  kind      entry point            stands for
  decode    decode_scored_paged    one new token per request, bf16 pages
  prefill   prefill_scored_varlen  whole prompts, packed
  chunk     prefill_scored_varlen  chunks of prompts after cached context
  write4    kv_write_mx4,          a step's new rows into the 4-bit pages, and
            kv_read_mx4            the same rows back as the values they hold
  decode4   decode_mx4_paged       one new token per request, 4-bit pages
  chunk4    prefill_mx4_varlen     chunks of prompts over 4-bit pages

Scores of query q (position p) and key k (position j) of a head:

  z = scale q.k;  x = cap tanh(z / cap)  (cap 0: x = z)
  x -= slope |p - j|  (slopes);  x += rel[p - j] for 0 <= p - j < E  (rel)

and the query sees the keys with max(first, p - window + 1) <= j <=
max(p, prefix - 1) that its request has.

4 bits: the 128 values of a token's head are four blocks of 32. A block has
one scale 2^e, e the smallest (from -125) with amax <= 7 * 2^e, and its values
are the nearest of 0, .5, 1, 1.5, 2, 3, 4, 6 times it (ties to the even code,
signed). e above 125, or a value that is no number: the block is NaN.
A page's record for one head, 2176 bytes:
  [16 tokens][64]           keys, dims 2i and 2i + 1 in byte i (low, high)
  [16 groups][16 tokens][4] values, group c holding dims 8c .. 8c + 7
  [4 blocks][16 tokens]     scales of the keys, e + 127 (255: NaN)
  [4 blocks][16 tokens]     scales of the values

With `own` false, run() computes it in elementary torch operations; with it
true, by the package's operators.
"""
import importlib
import math
import random

import torch

own = False

PAGE, D = 16, 128
REC = 2176
EXTENT = 1024           # the relative bias's band
DEV = "cuda"
BF = torch.bfloat16


# --------------------------------------------------------------------------
# the cases
# --------------------------------------------------------------------------

def listed():
    return [
        # a few short chats of a model with capped scores: the smallest
        # attention call, where launches and the host's work count
        dict(name="decode_cap_b4", kind="decode", b=4, lo=128, hi=1024,
             window=0, hq=32, hkv=4, cap=50.0, slopes=0, docs=0, lens=1),
        # a busy server's decode step of the same model, 1K-8K contexts
        dict(name="decode_cap_b64", kind="decode", b=64, lo=1024, hi=8192,
             window=0, hq=32, hkv=4, cap=50.0, slopes=0, docs=0, lens=2),
        # distance bias over requests that hold several documents each
        dict(name="decode_slopes_docs_b24", kind="decode", b=24, lo=1000,
             hi=20000, window=0, hq=64, hkv=8, cap=0.0, slopes=1, docs=1,
             lens=3),
        # packed prompts of 2K-8K tokens with capped scores, the largest call
        dict(name="prefill_cap_4_prompts", kind="prefill", s=4, lo=2048,
             hi=8192, window=0, hq=32, hkv=4, cap=50.0, slopes=0, docs=0,
             prefix=0, lens=7),
        # one ordinary prompt of an odd length whose first part is read in
        # both directions
        dict(name="prefill_prefix_b1_777", kind="prefill", s=1, lo=777,
             hi=777, window=0, hq=64, hkv=8, cap=0.0, slopes=0, docs=0,
             prefix=1, lens=8),
        # one chunk of a long request of several documents, distance bias
        dict(name="chunk_docs_slopes_1500", kind="chunk", s=1, lo=1500,
             hi=1500, prior_lo=15000, prior_hi=15000, window=0, hq=64, hkv=8,
             cap=0.0, slopes=1, docs=1, prefix=0, lens=9),
        # the new rows of a decode step
        dict(name="write4_b64", kind="write4", t=64, hkv=4, hq=32, lens=11),
        # the rows of a step's prompts
        dict(name="write4_12001", kind="write4", t=12001, hkv=8, hq=64,
             lens=12),
        # a busy server's decode step over 4-bit pages
        dict(name="decode4_b64", kind="decode4", b=64, lo=1024, hi=8192,
             window=0, hq=32, hkv=4, cap=0.0, slopes=0, rel=0, lens=2),
        # one user with one long document over 4-bit pages
        dict(name="decode4_b1_long", kind="decode4", b=1, lo=50001, hi=50001,
             window=0, hq=32, hkv=4, cap=0.0, slopes=0, rel=0, lens=13),
        # a sliding-window layer's decode step with the relative bias, the
        # model's window heads
        dict(name="decode4_window_rel_b96", kind="decode4", b=96, lo=200,
             hi=30000, window=512, hq=64, hkv=16, cap=0.0, slopes=0, rel=1,
             lens=14),
        # one chunk of a long prompt after what is cached in 4 bits
        dict(name="chunk4_500_after_15000", kind="chunk4", s=1, lo=500,
             hi=500, prior_lo=15000, prior_hi=15000, window=0, hq=64, hkv=8,
             cap=0.0, slopes=0, rel=0, lens=15),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["decode", "prefill", "chunk", "write4", "decode4",
                       "decode4", "chunk4"])
    lens = rng.randrange(1, 1 << 20)
    # the configurations' heads, the model's two layer kinds, and shards of
    # them over 2 or 4 GPUs
    hq, hkv = rng.choice([(32, 4), (32, 4), (64, 8), (64, 16), (32, 8),
                          (16, 2)])
    c = dict(kind=kind, hq=hq, hkv=hkv, lens=lens)
    if kind == "write4":
        return dict(c, t=_log(rng, 1, 12001))
    # score functions: at least one of them for the bf16 kinds
    cap = rng.choice([0.0, 30.0, 50.0])
    slopes = rng.choice([0, 0, 1])
    docs = rng.choice([0, 0, 1])
    if kind in ("decode", "prefill", "chunk"):
        prefix = 0 if kind == "decode" else rng.choice([0, 0, 1])
        if not (cap or slopes or docs or prefix):
            cap = 50.0
        c.update(cap=cap, slopes=slopes, docs=docs)
        if kind != "decode":
            c.update(prefix=prefix)
    else:
        rel = rng.choice([0, 0, 1])
        c.update(cap=0.0 if rel else cap, slopes=0 if rel else slopes,
                 rel=rel)
    if kind in ("decode", "decode4"):
        window = rng.choice([0, 0, 512, 4096])
        hi = _log(rng, 64, 65536)
        lo = max(1, int(hi * rng.choice([1.0, 0.5, 0.125])))
        vis = min(hi, window) if window else hi
        most = min(128, max(1, 500000 * 4 // (vis * hkv)))
        return dict(c, b=_log(rng, 1, most), lo=lo, hi=hi, window=window)
    if kind == "prefill":
        hi = _log(rng, 16, 8192)
        most = min(8, max(1, int(1.7 * 8192 * 8192 * 32 / (hi * hi * hq))))
        return dict(c, s=_log(rng, 1, most), lo=max(1, hi // 8), hi=hi,
                    window=rng.choice([0, 0, 512, 4096]))
    hi = _log(rng, 1, 2048)
    s = rng.choice([1, 1, 2, 3])
    p = _log(rng, 16, min(32768, int(1.5e9 / (s * hi * hq))))
    return dict(c, s=s, lo=max(1, hi // 2), hi=hi, prior_lo=p // 2,
                prior_hi=p, window=rng.choice([0, 0, 4096]))


# --------------------------------------------------------------------------
# lengths and masks (from the case alone) and inputs (from the seed)
# --------------------------------------------------------------------------

def _lens(case):
    """[(new tokens, tokens before them)] of the requests."""
    r = random.Random(case["lens"])
    k = case["kind"]
    one = lambda: r.randint(case["lo"], case["hi"])        # noqa: E731
    if k == "write4":
        return [(case["t"], 0)]
    if k in ("decode", "decode4"):
        return [(1, one() - 1) for _ in range(case["b"])]
    if k == "prefill":
        return [(one(), 0) for _ in range(case["s"])]
    return [(one(), r.randint(case["prior_lo"], case["prior_hi"]))
            for _ in range(case["s"])]                     # chunk, chunk4


def _firsts(case):
    """For each request the first position of the document that each of its
    new tokens belongs to (documents of an eighth to a half of the request)."""
    r = random.Random(case["lens"] + 1)
    res = []
    for new, prior in _lens(case):
        n = new + prior
        at, start = [], 0
        while len(at) < n:
            size = min(r.randint(max(1, n // 8), max(1, n // 2)),
                       n - len(at))
            at += [start] * size
            start += size
        res.append(at[prior:])
    return res


def _prefixes(case):
    """Of each request, how many of its first tokens all of it may see."""
    r = random.Random(case["lens"] + 2)
    return [b + r.randint(a // 4, a) for a, b in _lens(case)]


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


def _queries(shape, g, capped):
    """Query rows whose heads are flat to peaked: scores of spread 0.5-3, and
    under a cap every fourth head eight times that."""
    gain = torch.rand(shape[-2:-1], generator=g, device=DEV) * 2.5 + 0.5
    if capped:
        gain[3::4] *= 8
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


def _power(e):
    """2^e in fp32 of whole e from -126 to 127, by its bits."""
    return ((e.int() + 127) << 23).view(torch.float32)


def _quantise(x):
    """x [..., 128]: codes [..., 128] and scale bytes [..., 4] (uint8)."""
    x = x.float().unflatten(-1, (4, 32))
    amax = x.abs().amax(-1)
    f, e = torch.frexp(amax)             # amax = f 2^e, f in [0.5, 1)
    e = (e - 3 + (f > 0.875)).clamp(min=-125)
    e = torch.where(amax > 0, e, -125)
    bad = ~torch.isfinite(x).all(-1) | (e > 125)
    y = x.abs() * _power(-e.clamp(max=125))[..., None]
    code = ((y > 0.25).int() + (y >= 0.75) + (y > 1.25) + (y >= 1.75) +
            (y > 2.5) + (y >= 3.5) + (y > 5)) + 8 * torch.signbit(x).int()
    code = torch.where(bad[..., None], 0, code).to(torch.uint8)
    return code.flatten(-2), torch.where(bad, 255, e + 127).to(torch.uint8)


def _pack(k, v):
    """Pages of k and v [P, 16, HKV, 128] as the records [P, HKV, 2176]."""
    P, _, H, _ = k.shape
    rec = torch.empty((P, H, REC), dtype=torch.uint8, device=DEV)
    code, scale = _quantise(k.transpose(1, 2))          # [P, H, 16, ...]
    rec[..., :1024] = (code[..., ::2] | code[..., 1::2] << 4).flatten(2)
    rec[..., 2048:2112] = scale.transpose(2, 3).flatten(2)
    code, scale = _quantise(v.transpose(1, 2))
    pair = (code[..., ::2] | code[..., 1::2] << 4).unflatten(-1, (16, 4))
    rec[..., 1024:2048] = pair.transpose(2, 3).flatten(2)
    rec[..., 2112:] = scale.transpose(2, 3).flatten(2)
    return rec


def _pack_pool(P, hkv, g):
    """A pool of P pages, some thousands of them at a time."""
    pool = torch.empty((P, hkv, REC), dtype=torch.uint8, device=DEV)
    mean = torch.randn((hkv, D), generator=g, device=DEV) * 0.25
    for a in range(0, P, 8192):
        n = min(8192, P - a)
        x = torch.randn((2, n, PAGE, hkv, D), generator=g, device=DEV)
        pool[a:a + n] = _pack(x[0].to(BF), (x[1] + mean).to(BF))
    return pool


def prepare(case, seed):
    g, c = _gens(seed)
    kind, hq, hkv = case["kind"], case["hq"], case["hkv"]
    lens = _lens(case)
    new, prior = [a for a, _ in lens], [b for _, b in lens]
    T = sum(new)
    if kind == "write4":
        # K and V as parts of the fused projection's rows; the pool's other
        # pages are another request's
        P = 2 * _pages(T) + 1
        qkv = torch.empty((T, hq + 2 * hkv, D), dtype=BF, device=DEV)
        qkv[:, hq:hq + hkv] = _rows((T, hkv, D), g)
        qkv[:, hq + hkv:] = _values((T, hkv, D), g)
        slots = torch.randperm(P, generator=c)[:_pages(T)]
        slots = (slots[:, None] * PAGE + torch.arange(PAGE)).flatten()[:T]
        return dict(case=case, k=qkv[:, hq:hq + hkv], v=qkv[:, hq + hkv:],
                    slots=slots.to(DEV),
                    pool=torch.zeros((P, hkv, REC), dtype=torch.uint8,
                                     device=DEV))
    ends = [a + b for a, b in lens]
    st = dict(case=case, q=_queries((T, hq, D), g, case["cap"] > 0),
              cap=case["cap"], slopes=None, first=None, prefix=None, rel=None,
              scale=D ** -0.5, window=case["window"], cu=_cu(new),
              prior=_i32(prior), longest=max(new), most=max(ends))
    if case["slopes"]:
        st["slopes"] = torch.exp2(-8 * torch.arange(1, hq + 1, device=DEV) /
                                  hq).float()
    if case.get("docs"):
        st["first"] = _i32(sum(_firsts(case), []))
    if case.get("prefix"):
        st["prefix"] = _i32(_prefixes(case))
    if case.get("rel"):
        st["rel"] = _rows((T, hq, EXTENT), g)
    if kind == "prefill":
        st.update(k=_rows((T, hkv, D), g), v=_values((T, hkv, D), g))
        return st
    t, P = _shuffled_table([_pages(n) for n in ends], _pages(max(ends)), c)
    st.update(ctx=_i32(ends), table=t.to(DEV))
    if kind in ("decode4", "chunk4"):
        st.update(pool=_pack_pool(P, hkv, g))
    else:
        st.update(kp=_rows((P, PAGE, hkv, D), g),
                  vp=_values((P, PAGE, hkv, D), g))
    return st


# --------------------------------------------------------------------------
# one pass
# --------------------------------------------------------------------------

def _attention(st, q, K, V, kpos, qpos, first, prefix, rel):
    """q [S, T, HQ, D] at positions qpos [S, T] (negative: none), keys and
    values [S, N, HKV, D] at positions kpos [S, N] (negative: none), all fp32;
    first [S, T], prefix [S] or None. Returns (out [S, T, HQ, D], lse
    [S, T, HQ]), fp32."""
    S, T, hq, _ = q.shape
    N, hkv = K.shape[1], K.shape[2]
    rep = hq // hkv
    x = q.view(S, T, hkv, rep, D).permute(0, 2, 3, 1, 4)
    x = x.reshape(S, hkv, rep * T, D)
    s = torch.matmul(x, K.permute(0, 2, 3, 1)).mul_(st["scale"])
    if st["cap"]:
        s.div_(st["cap"]).tanh_().mul_(st["cap"])
    s = s.view(S, hkv, rep, T, N)
    dist = qpos[:, :, None] - kpos[:, None, :]
    if st["slopes"] is not None:
        far = dist.abs().float()
        for h in range(hq):
            s[:, h // rep, h % rep] -= st["slopes"][h] * far
    if rel is not None:                       # [S, T, HQ, E]
        E = rel.shape[3]
        inside = (dist >= 0) & (dist < E)
        at = dist.clamp(0, E - 1)
        for h in range(hq):
            b = torch.gather(rel[:, :, h], 2, at)
            s[:, h // rep, h % rep] += torch.where(inside, b, 0.0)
    top = qpos if prefix is None else torch.maximum(qpos, prefix[:, None] - 1)
    dead = (kpos[:, None, :] > top[:, :, None]) | (kpos < 0)[:, None, :]
    dead |= (qpos < 0)[:, :, None]
    if st["window"]:
        dead |= dist >= st["window"]
    if first is not None:
        dead |= kpos[:, None, :] < first[:, :, None]
    s.masked_fill_(dead[:, None, None], -math.inf)
    m = s.amax(-1, keepdim=True).clamp_(min=-3e38)
    s.sub_(m).exp_()
    l = s.sum(-1, keepdim=True)
    lse = (m + torch.log(l))[..., 0]
    s.div_(torch.where(l > 0, l, 1.0))
    o = torch.matmul(s.view(S, hkv, rep * T, N), V.transpose(1, 2))
    o = o.view(S, hkv, rep, T, D).permute(0, 3, 1, 2, 4)
    return (o.reshape(S, T, hq, D),
            lse.permute(0, 3, 1, 2).reshape(S, T, hq))


def _dequantise(code, scale):
    """Packed bytes [..., 64] and scale bytes [..., 4] -> fp32 [..., 128]."""
    code = torch.stack([code & 15, code >> 4], -1).flatten(-2).int()
    e, m = code >> 1 & 3, (code & 1).float()
    y = torch.where(e > 0, (1 + 0.5 * m) * _power(e - 1), 0.5 * m)
    y = torch.where(code > 7, -y, y).unflatten(-1, (4, 32))
    y = y * _power(scale.int().clamp(1, 254) - 127)[..., None]
    return torch.where(scale[..., None] == 255, math.nan, y).flatten(-2)


def _rows4(rec):
    """Records [..., HKV, 2176] -> K and V fp32 [..., 16, HKV, 128]."""
    k = _dequantise(rec[..., :1024].unflatten(-1, (16, 64)),
                    rec[..., 2048:2112].unflatten(-1, (4, 16)).transpose(
                        -1, -2))
    v = rec[..., 1024:2048].unflatten(-1, (16, 16, 4)).transpose(-2, -3)
    v = _dequantise(v.flatten(-2), rec[..., 2112:].unflatten(
        -1, (4, 16)).transpose(-1, -2))
    return k.transpose(-2, -3), v.transpose(-2, -3)


def _cached(st, kpos):
    """K and V rows at positions kpos [S, N] of the requests, fp32."""
    p = kpos.clamp(min=0)
    pages = torch.gather(st["table"].long(), 1, p // PAGE)
    if "pool" not in st:
        return (st["kp"][pages, p % PAGE].float(),
                st["vp"][pages, p % PAGE].float())
    # whole pages of each request, then the rows
    first = (p[:, 0] // PAGE)[:, None]
    n = kpos.shape[1] // PAGE + 2
    j = (first + torch.arange(n, device=DEV)).clamp(
        max=st["table"].shape[1] - 1)
    ids = torch.gather(st["table"].long(), 1, j).clamp(min=0)
    at = (p - first * PAGE)[:, :, None, None]
    K, V = _rows4(st["pool"][ids])
    row = at.expand(-1, -1, K.shape[3], D)
    return (torch.gather(K.flatten(1, 2), 1, row),
            torch.gather(V.flatten(1, 2), 1, row))


def _decode(st):
    ctx = st["ctx"].long()
    n = min(st["most"], st["window"]) if st["window"] else st["most"]
    # (a request shorter than that starts at its position 0)
    kpos = (ctx[:, None] - n).clamp(min=0) + torch.arange(n, device=DEV)
    kpos = torch.where(kpos < ctx[:, None], kpos, -1)
    K, V = _cached(st, kpos)
    first = None if st["first"] is None else st["first"].long()[:, None]
    rel = None if st["rel"] is None else st["rel"].float()[:, None]
    o, lse = _attention(st, st["q"].float()[:, None], K, V, kpos,
                        ctx[:, None] - 1, first, None, rel)
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
        K, V = _cached(st, kpos)
    first = None if st["first"] is None else st["first"].long()[row]
    prefix = None if st["prefix"] is None else st["prefix"].long()
    rel = None if st["rel"] is None else st["rel"][row].float()
    o, lse = _attention(st, st["q"].float()[row], K, V, kpos, qpos, first,
                        prefix, rel)
    return o[run, j].to(BF), lse[run, j].t().contiguous()


def _write4(st):
    pool, page, off = st["pool"], st["slots"] // PAGE, st["slots"] % PAGE
    heads = torch.arange(pool.shape[1], device=DEV)[:, None]
    at, i = off[:, None, None], torch.arange(64, device=DEV)
    b = torch.arange(4, device=DEV) * PAGE
    res = []
    for x, code_at, scale_at in (
            (st["k"], at * 64 + i, 2048 + b + at),
            (st["v"], 1024 + i // 4 * 64 + at * 4 + i % 4, 2112 + b + at)):
        code_at = (page[:, None, None], heads, code_at)
        scale_at = (page[:, None, None], heads, scale_at)
        code, scale = _quantise(x)
        pool[code_at] = code[..., ::2] | code[..., 1::2] << 4
        pool[scale_at] = scale
        res.append(_dequantise(pool[code_at], pool[scale_at]).to(BF))
    return tuple(res)


def run(st):
    k = st["case"]["kind"]
    if not own:
        return {"decode": _decode, "decode4": _decode, "write4": _write4}.get(
            k, _prefill)(st)
    tm = importlib.import_module("tm-opt_amd")
    if k == "decode":
        return tm.decode_scored_paged(
            st["q"], st["kp"], st["vp"], st["table"], st["ctx"], st["scale"],
            softcap=st["cap"], slopes=st["slopes"], first_keys=st["first"],
            window=st["window"])
    if k == "prefill":
        return tm.prefill_scored_varlen(
            st["q"], st["k"], st["v"], st["cu"], st["scale"],
            softcap=st["cap"], slopes=st["slopes"], first_keys=st["first"],
            prefix_lens=st["prefix"], window=st["window"],
            max_seqlen=st["longest"])
    if k == "chunk":
        return tm.prefill_scored_varlen(
            st["q"], None, None, st["cu"], st["scale"], softcap=st["cap"],
            slopes=st["slopes"], first_keys=st["first"],
            prefix_lens=st["prefix"], window=st["window"],
            max_seqlen=st["longest"], prior_lens=st["prior"],
            k_pool=st["kp"], v_pool=st["vp"], block_table=st["table"],
            max_context=st["most"])
    if k == "write4":
        tm.kv_write_mx4(st["k"], st["v"], st["slots"], st["pool"])
        return tm.kv_read_mx4(st["pool"], st["slots"])
    if k == "decode4":
        return tm.decode_mx4_paged(
            st["q"], st["pool"], st["table"], st["ctx"], st["scale"],
            softcap=st["cap"], slopes=st["slopes"], rel=st["rel"],
            window=st["window"])
    return tm.prefill_mx4_varlen(
        st["q"], st["pool"], st["table"], st["cu"], st["prior"], st["scale"],
        softcap=st["cap"], slopes=st["slopes"], rel=st["rel"],
        window=st["window"], max_seqlen=st["longest"],
        max_context=st["most"])


# --------------------------------------------------------------------------
# what a pass cannot do without
# --------------------------------------------------------------------------

def _visible(case):
    """(query-key pairs, keys that some query sees) of each request."""
    w = case["window"]
    firsts = _firsts(case) if case.get("docs") else None
    prefixes = _prefixes(case) if case.get("prefix") else None
    res = []
    for r, (new, prior) in enumerate(_lens(case)):
        pairs, low = 0, prior + new
        for i in range(new):
            p = prior + i
            lo = max(0, p - w + 1) if w else 0
            if firsts:
                lo = max(lo, firsts[r][i])
            hi = p
            if prefixes:
                hi = min(max(p, prefixes[r] - 1), prior + new - 1)
            pairs += hi - lo + 1
            low = min(low, lo)
        res.append((pairs, prior + new - low))
    return res


def work(case):
    hq, hkv = case["hq"], case["hkv"]
    if case["kind"] == "write4":
        # rows in, their part of the records and the values held out
        return {"bytes": case["t"] * (hkv * (4 * D + 136 + 4 * D) + 8),
                "flops": 0}
    T = sum(a for a, _ in _lens(case))
    seen = _visible(case)
    keys = sum(n for _, n in seen)
    row = hkv * (136 if case["kind"] in ("decode4", "chunk4") else 4 * D)
    table = 0 if case["kind"] == "prefill" else 4 * sum(
        _pages(n) for _, n in seen)
    # of a relative bias, the part of the band that a query's keys fall in
    rel = 2 * hq * sum(min(EXTENT, b + i + 1, case["window"] or EXTENT)
                       for a, b in _lens(case)
                       for i in range(a)) if case.get("rel") else 0
    return {"bytes": 4 * T * hq * D + 4 * T * hq + keys * row + table + rel,
            "flops": 4 * D * hq * sum(p for p, _ in seen)}


# --------------------------------------------------------------------------
# the same in 64 bits, request by request and head by head
# --------------------------------------------------------------------------

_E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def _exact_rows4(rec, h):
    """K and V of head h of the records [N, HKV, 2176]: float64 [16 N, 128]."""
    lut = torch.tensor(_E2M1 + [-x for x in _E2M1], dtype=torch.float64,
                       device=DEV)
    power = torch.tensor([2.0 ** (i - 127) for i in range(255)] + [math.nan],
                         dtype=torch.float64, device=DEV)
    r = rec[:, h].long()
    out = []
    for el, sc in ((r[:, :1024].view(-1, 16, 64), r[:, 2048:2112]),
                   (r[:, 1024:2048].view(-1, 16, 16, 4).transpose(
                       1, 2).reshape(-1, 16, 64), r[:, 2112:])):
        x = torch.empty(el.shape[:2] + (D,), dtype=torch.float64, device=DEV)
        x[..., 0::2] = lut[el % 16]
        x[..., 1::2] = lut[el // 16]
        s = power[sc.view(-1, 4, 16)].transpose(1, 2)
        out.append((x * s.repeat_interleave(32, 2)).view(-1, D))
    return out


def _exact_run(st, r, t, new, prior):
    """Request r, whose first query is row t; float64 (out [new, HQ, D], lse
    [HQ, new])."""
    q = st["q"][t:t + new]
    hq, hkv = q.shape[1], st["case"]["hkv"]
    N = prior + new
    out = torch.empty((new, hq, D), dtype=torch.float64, device=DEV)
    lse = torch.empty((hq, new), dtype=torch.float64, device=DEV)
    # (positions before every query's window are left out)
    base = max(0, prior - st["window"] + 1) if st["window"] else 0
    base -= base % PAGE
    key = torch.arange(base, N, device=DEV)
    if "table" in st:
        ids = st["table"][r, base // PAGE:_pages(N)].long()
    for h in range(hq):
        g = h // (hq // hkv)
        if "k" in st:
            K, V = (st[x][t + base:t + N, g].double() for x in ("k", "v"))
        elif "pool" in st:
            K, V = (x[:N - base] for x in _exact_rows4(st["pool"][ids], g))
        else:
            K, V = (st[x][ids, :, g].double().reshape(-1, D)[:N - base]
                    for x in ("kp", "vp"))
        for a in range(0, new, 4096):
            rows = slice(a, min(a + 4096, new))
            at = torch.arange(prior + rows.start, prior + rows.stop,
                              device=DEV)[:, None]
            z = q[rows, h].double() @ K.t() * st["scale"]
            if st["cap"]:
                z = st["cap"] * torch.tanh(z / st["cap"])
            if st["slopes"] is not None:
                z -= st["slopes"][h].double() * (at - key).abs()
            if st["rel"] is not None:
                E = st["rel"].shape[2]
                b = torch.cat([st["rel"][t + rows.start:t + rows.stop, h],
                               torch.zeros((z.shape[0], 1), device=DEV,
                                           dtype=BF)], 1).double()
                far = at - key
                z += b.gather(1, torch.where((far < 0) | (far >= E), E, far))
            top = at
            if st["prefix"] is not None:
                top = torch.maximum(at, st["prefix"][r].long() - 1)
            seen = key <= top
            if st["window"]:
                seen &= key > at - st["window"]
            if st["first"] is not None:
                seen &= key >= st["first"][t + rows.start:t + rows.stop,
                                           None]
            z = torch.where(seen, z, -math.inf)
            lse[h, rows] = torch.logsumexp(z, 1)
            out[rows, h] = torch.softmax(z, 1) @ V
    return out, lse


def _exact_values4(x):
    """What is held of the rows x [T, HKV, 128], by the nearest value."""
    x = x.double().reshape(*x.shape[:2], 4, 32)
    amax = x.abs().amax(-1, keepdim=True)
    power = torch.full_like(amax, 2.0 ** -125)
    for e in range(-124, 127):
        power = torch.where(amax > 7 * 2.0 ** (e - 1), 2.0 ** e, power)
    y = x.abs() / power
    grid = torch.tensor(_E2M1, dtype=torch.float64, device=DEV)
    low = (grid <= y[..., None]).sum(-1).clamp(min=1) - 1
    up = (low + 1).clamp(max=7)
    dl, du = y - grid[low], grid[up] - y
    code = torch.where((du < dl) | ((du == dl) & (low % 2 == 1)), up, low)
    y = torch.copysign(grid[code] * power, x)
    bad = (power > 2.0 ** 125) | ~torch.isfinite(amax)
    return torch.where(bad, math.nan, y).flatten(-2)


def exact(case, seed):
    st = prepare(case, seed)
    if case["kind"] == "write4":
        return _exact_values4(st["k"]), _exact_values4(st["v"])
    outs, lses, t = [], [], 0
    for r, (a, b) in enumerate(_lens(case)):
        o, l = _exact_run(st, r, t, a, b)
        outs.append(o)
        lses.append(l)
        t += a
    lse = torch.cat(lses, 1)
    one = case["kind"] in ("decode", "decode4")
    return torch.cat(outs), lse.t() if one else lse
