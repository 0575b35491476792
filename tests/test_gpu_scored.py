"""Attention with score functions and masks (decode_scored_paged,
prefill_scored_varlen) and the prefill over the 4-bit cache
(prefill_mx4_varlen) against their definition in float64, within the bounds that
oracle/scored_ref.py derives. Pools hold NaN wherever no request owns a row."""
import math

import pytest
import torch

from oracle import scored_ref as ref
from test_gpu_mx4 import Cache4

pytestmark = pytest.mark.gpu
D, PAGE = 128, 16
BF = torch.bfloat16
NAN = float("nan")


def _gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def _rand(shape, g, dev, std=1.0):
    return (torch.randn(shape, generator=g) * std).to(BF).to(dev)


def _i32(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


class Cache:
    """bf16 pools in which request i's positions [first_i, n_i) hold values and
    everything else is NaN, behind shuffled pages."""

    def __init__(self, ends, hkv, g, dev, first=None, wrap=0, width=None):
        pages = [wrap or -(-n // PAGE) for n in ends]
        P = sum(pages) + 3
        perm = torch.randperm(P - 1, generator=g).to(torch.int32)
        w = width or max(pages + [1])
        self.table = torch.full((len(ends), w), P - 1, dtype=torch.int32)
        off = 0
        for i, n in enumerate(pages):
            self.table[i, :n] = perm[off:off + n]
            off += n
        self.table = self.table.to(dev)
        self.kp = torch.full((P, PAGE, hkv, D), NAN, dtype=BF, device=dev)
        self.vp = torch.full_like(self.kp, NAN)
        for i, n in enumerate(ends):
            pos = torch.arange(0 if first is None else first[i], n, device=dev)
            lp = pos // PAGE % wrap if wrap else pos // PAGE
            rows = self.table[i][lp].long(), pos % PAGE
            self.kp[rows] = _rand((len(pos), hkv, D), g, dev)
            self.vp[rows] = _rand((len(pos), hkv, D), g, dev)
        self.ctx = _i32(ends, dev)


def _function(name, hq, g, dev):
    """Score functions by name: cap (strong), soft (hardly bent), slopes."""
    kw = {}
    if "cap" in name:
        kw["softcap"] = 2.0
    if "soft" in name:
        kw["softcap"] = 50.0
    if "slopes" in name:
        kw["slopes"] = (torch.rand(hq, generator=g) * 0.3 - 0.05).to(dev)
    return kw


# --------------------------------------------------------------------------
# decode
# --------------------------------------------------------------------------

def _decode(tm, c, q, scale, what="", window=0, wrap=0, first=None, split=(),
            **kw):
    out, lse = tm.decode_scored_paged(q, c.kp, c.vp, c.table, c.ctx, scale,
                                      window=window, table_wrap=wrap,
                                      first_keys=first, **dict(split), **kw)
    ref.check(out, lse, ref.decode(q, c.kp, c.vp, c.table, c.ctx, scale,
                                   window=window, table_wrap=wrap, first=first,
                                   **kw), what)
    return out, lse


EDGES = [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 300, 700]


@pytest.mark.parametrize("hq,hkv", [(1, 1), (8, 1), (32, 4), (64, 16), (64, 8),
                                    (12, 4), (3, 3), (10, 2), (16, 1), (34, 2),
                                    (20, 5), (40, 2)])
def test_decode_heads(tm, dev, hq, hkv):
    g = _gen(hq * 100 + hkv)
    c = Cache(EDGES, hkv, g, dev)
    q = _rand((len(EDGES), hq, D), g, dev, 2.0)
    _decode(tm, c, q, D ** -0.5, f"{hq}/{hkv}",
            **_function("cap slopes", hq, g, dev))
    _decode(tm, c, q, D ** -0.5, f"{hq}/{hkv} split", split=[("min_pages", 1)],
            **_function("soft", hq, g, dev))


@pytest.mark.parametrize("name", ["plain", "cap", "soft", "slopes",
                                  "cap slopes"])
@pytest.mark.parametrize("window", [0, 1, 16, 100, 512])
@pytest.mark.parametrize("docs", [0, 1])
@pytest.mark.parametrize("min_pages,wgs", [(8, 0), (1, 7), (3, 64)])
def test_decode_masks_and_splits(tm, dev, name, window, docs, min_pages, wgs):
    g = _gen(window * 10 + min_pages)
    ends = [0, 1, 16, 99, 100, 101, 511, 512, 513, 800, 1500, 640, 77]
    starts = [0, 0, 15, 99, 0, 37, 64, 512, 600, 16, -5, 333, 2 ** 31 - 1]
    lo = [max(0, n - window) if window else 0 for n in ends]
    if docs:
        lo = [min(max(a, b), n) for a, b, n in zip(lo, starts, ends)]
    c = Cache(ends, 4, g, dev, first=lo)
    q = _rand((len(ends), 16, D), g, dev, 1.5)
    _decode(tm, c, q, 0.1, name, window=window,
            first=_i32(starts, dev) if docs else None,
            split=[("min_pages", min_pages), ("num_workgroups", wgs)],
            **_function(name, 16, g, dev))


@pytest.mark.parametrize("window,wrap", [(40, 4), (64, 4), (1, 1)])
def test_decode_ring_at_the_last_positions(tm, dev, window, wrap):
    g = _gen(21)
    ends = [2 ** 31 - 1, 2 ** 31 - 16, 2 ** 31 - 17, 5, 100]
    starts = [0, 2 ** 31 - 20, 0, 0, 90]
    c = Cache(ends, 4, g, dev, first=[max(0, n - window) for n in ends],
              wrap=wrap)
    q = _rand((5, 16, D), g, dev)
    for first in (None, _i32(starts, dev)):
        _decode(tm, c, q, 0.1, window=window, wrap=wrap, first=first,
                **_function("soft slopes", 16, g, dev))


def test_decode_absent_pages(tm, dev):
    g = _gen(4)
    c = Cache([200, 208, 40], 4, g, dev)
    q = _rand((3, 16, D), g, dev)
    c.table[0, 3] = -1
    c.table[0, 7] = 10 ** 6
    c.table[2] = -7
    c.ctx[1] = 5000                       # the row holds 13 pages
    out, lse = tm.decode_scored_paged(q, c.kp, c.vp, c.table, c.ctx, 0.1,
                                      softcap=3.0, min_pages=1)
    for b, gone, n in ((0, (3, 7), 200), (1, (), 208)):
        pos = torch.tensor([p for p in range(n) if p // PAGE not in gone],
                           device=dev)
        table = c.table[b].clamp(0, c.kp.shape[0] - 1)
        r = ref.attend(q[b:b + 1], ref.rows_of(c.kp, table, pos),
                       ref.rows_of(c.vp, table, pos),
                       torch.tensor([4999], device=dev), pos, 0.1, softcap=3.0)
        ref.check(out[b:b + 1], lse[b:b + 1], (r[0], r[1].T, r[2], r[3].T))
    assert (out[2] == 0).all() and (lse[2] == -math.inf).all()


def test_decode_no_number(tm, dev):
    """A visible key of score NaN gives NaN; an infinite score is capped."""
    g = _gen(7)
    c = Cache([50, 400, 30], 2, g, dev)
    q = _rand((3, 8, D), g, dev)
    c.kp[c.table[1, 12], 3, 1, 5] = NAN
    for kw in (dict(min_pages=1), dict(min_pages=100)):
        out, lse = tm.decode_scored_paged(q, c.kp, c.vp, c.table, c.ctx, 0.1,
                                          softcap=9.0, **kw)
        assert torch.isnan(out[1, 4:]).all() and torch.isnan(lse[1, 4:]).all()
        assert torch.isfinite(out[1, :4]).all() and torch.isfinite(lse[0]).all()
        assert torch.isfinite(out[[0, 2]]).all()
    q[0, :4, 0] = 1.0
    c.kp[c.table[0, 0], 2, 0] = 0.0
    c.kp[c.table[0, 0], 2, 0, 0] = math.inf
    # (scores of +infinity: the cap itself)
    out, lse = tm.decode_scored_paged(q, c.kp, c.vp, c.table, c.ctx, 0.1,
                                      softcap=9.0)
    c.kp[c.table[0, 0], 2, 0, 0] = 1e30
    want = tm.decode_scored_paged(q, c.kp, c.vp, c.table, c.ctx, 0.1,
                                  softcap=9.0)
    assert torch.equal(out[0], want[0][0]) and torch.equal(lse[0], want[1][0])


def test_decode_graph_and_streams(tm, dev):
    g = _gen(8)
    c = Cache([90, 1000, 3, 555], 4, g, dev)
    q = _rand((4, 32, D), g, dev)
    first = _i32([10, 0, 2, 300], dev)
    kw = _function("soft slopes", 32, g, dev)
    ws = tm.decode_workspace(4, 32, 4, dev)
    out = torch.empty_like(q)
    lse = torch.empty((4, 32), device=dev)
    ctx = c.ctx.clone()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        tm.decode_scored_paged(q, c.kp, c.vp, c.table, ctx, 0.1,
                               first_keys=first, out=out, lse=lse,
                               workspace=ws, **kw)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        tm.decode_scored_paged(q, c.kp, c.vp, c.table, ctx, 0.1,
                               first_keys=first, out=out, lse=lse,
                               workspace=ws, **kw)
    for lens, starts in (([90, 1000, 3, 555], [10, 0, 2, 300]),
                         ([11, 64, 0, 300], [10, 63, 0, 300]),
                         ([90, 999, 2, 16], [0, 500, 1, 0])):
        ctx.copy_(_i32(lens, dev))
        first.copy_(_i32(starts, dev))
        graph.replay()
        torch.cuda.synchronize()
        eager = tm.decode_scored_paged(q, c.kp, c.vp, c.table, ctx, 0.1,
                                       first_keys=first, **kw)
        assert torch.equal(out, eager[0]) and torch.equal(lse, eager[1])


def test_decode_without_functions_is_decode_paged(tm, dev):
    """No cap, slope or first key: the attention of decode_paged."""
    g = _gen(9)
    c = Cache(EDGES, 4, g, dev)
    q = _rand((len(EDGES), 32, D), g, dev)
    a = tm.decode_scored_paged(q, c.kp, c.vp, c.table, c.ctx, 0.1, min_pages=8)
    b = tm.decode_paged(q, c.kp, c.vp, c.table, c.ctx, 0.1, min_pages=8)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_decode_largest_batch(tm, dev):
    """8192 requests of 0 to 40 tokens; and work-split knobs at their ends."""
    g = _gen(10)
    ends = [int(x) for x in torch.randint(0, 41, (8192,), generator=g)]
    rows = torch.cumsum(torch.tensor([0] + [-(-n // PAGE) for n in ends]), 0)
    table = torch.full((8192, 3), -1, dtype=torch.int32)
    for i, n in enumerate(ends):
        k = -(-n // PAGE)
        table[i, :k] = torch.arange(int(rows[i]), int(rows[i]) + k)
    table = table.to(dev)
    kp, vp = (_rand((int(rows[-1]), PAGE, 1, D), g, dev) for _ in range(2))
    ctx = _i32(ends, dev)
    first = torch.randint(-3, 20, (8192,), generator=g).int().to(dev)
    q = _rand((8192, 2, D), g, dev)
    pick = [0, 1, 4095, 4096, 8190, 8191] + list(range(100, 8000, 97))
    r = ref.decode(q[pick], kp, vp, table[pick], ctx[pick], 0.1,
                   first=first[pick], softcap=3.0)
    for kw in (dict(), dict(min_pages=2 ** 31 - 1),
               dict(num_workgroups=65535), dict(num_workgroups=1)):
        o, l = tm.decode_scored_paged(q, kp, vp, table, ctx, 0.1, softcap=3.0,
                                      first_keys=first, **kw)
        ref.check(o[pick], l[pick], r, str(kw))


def test_decode_lengths_past_the_table(tm, dev):
    g = _gen(11)
    c = Cache([64] * 100, 1, g, dev)
    q = _rand((100, 4, D), g, dev)
    c.ctx.fill_(2 ** 31 - 1)
    out, lse = tm.decode_scored_paged(q, c.kp, c.vp, c.table, c.ctx, 0.1)
    pos = torch.arange(64, device=dev)
    for b in (0, 1, 57, 99):
        r = ref.attend(q[b:b + 1], ref.rows_of(c.kp, c.table[b], pos),
                       ref.rows_of(c.vp, c.table[b], pos),
                       torch.tensor([2 ** 31 - 2], device=dev), pos, 0.1)
        ref.check(out[b:b + 1], lse[b:b + 1], (r[0], r[1].T, r[2], r[3].T))
    out, lse = tm.decode_scored_paged(q, c.kp, c.vp, c.table, c.ctx, 0.1,
                                      window=500)
    assert (out == 0).all() and (lse == -math.inf).all()


@pytest.mark.parametrize("cap", [0.01, 1.0, 53.0, 54.0, 62.0, 63.0, 4000.0])
def test_caps(tm, dev, cap):
    """Caps from far below the scores to far above them, scores that the
    polynomial takes and that it does not."""
    g = _gen(12)
    c = Cache([33, 500], 1, g, dev)
    q = _rand((2, 8, D), g, dev, 4.0)
    _decode(tm, c, q, 0.1, softcap=cap)
    _decode(tm, c, q * 0.01, 0.1, softcap=cap)
    q, k, v, cu = _packed([300, 70], 8, 1, g, dev)
    for gain in (8.0, 1.0, 0.02):
        _prefill(tm, q * gain, k, v, cu, 0.1, f"gain {gain}", softcap=cap)


# --------------------------------------------------------------------------
# prefill: packed prompts
# --------------------------------------------------------------------------

def _packed(lens, hq, hkv, g, dev):
    """q, k, v as parts of one wider row (as a fused projection gives them),
    and the runs' bounds."""
    T = sum(lens)
    x = _rand((T, hq + 2 * hkv, D), g, dev)
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    return x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:], _i32(cu, dev)


def _firsts(lens, prior, g, dev, empty=True):
    """First keys of every kind: the start, the query's own position, random
    ones, and (empty) positions past the query's."""
    rows = []
    for n, p in zip(lens, prior):
        pos = torch.arange(p, p + n)
        f = (torch.rand(n, generator=g) * (pos + 1)).long()
        f = torch.where(pos % 7 == 3, pos, f)
        f = torch.where(pos % 5 == 0, torch.zeros_like(f), f)
        if empty:
            f = torch.where(pos % 11 == 6, pos + 1 + pos % 3, f)
        rows.append(f)
    return torch.cat(rows).to(torch.int32).to(dev)


def _documents(lens, prior, g, dev):
    rows = []
    for n, p in zip(lens, prior):
        at, start = [], 0
        while len(at) < n + p:
            size = int(torch.randint(1, max(2, (n + p) // 3), (1,),
                                     generator=g))
            at += [start] * size
            start += size
        rows += at[p:p + n]
    return _i32(rows, dev)


def _prefill(tm, q, k, v, cu, scale, what="", prefix=None, first=None, **kw):
    out, lse = tm.prefill_scored_varlen(q, k, v, cu, scale, first_keys=first,
                                        prefix_lens=prefix, **kw)
    ref.check(out, lse, ref.prefill(q, k, v, cu, scale, first=first,
                                    prefix=prefix, **kw), what)
    return out, lse


@pytest.mark.parametrize("cap", [30.0, 53.0])
def test_prefill_cap_one_key(tm, dev, cap):
    """Queries that see themselves only: their value as it is (its probability is
    1, which bf16 holds); the others' keys hold no number."""
    g = _gen(31)
    lens = [1, 70, 200]
    q, k, v, cu = _packed(lens, 8, 2, g, dev)
    own = torch.cat([torch.arange(n) for n in lens]).to(torch.int32).to(dev)
    out, lse = tm.prefill_scored_varlen(q, k, v, cu, 0.1, softcap=cap,
                                        first_keys=own)
    assert torch.equal(out, v.repeat_interleave(4, 1))
    z = 0.1 * (q.double() * k.repeat_interleave(4, 1).double()).sum(2)
    x = cap * torch.tanh(z / cap)
    # the cap 2^-19 of itself; the score's products and sums, the LSE's own
    far = cap * 2.0 ** -19 + 132 * 2.0 ** -24 * 0.1 * (
        q.double() * k.repeat_interleave(4, 1).double()).abs().sum(2) + \
        24 * 2.0 ** -24 * (1 + x.abs())
    assert ((lse.T.double() - x).abs() <= far).all()


@pytest.mark.parametrize("cap", [30.0, 53.0])
@pytest.mark.parametrize("order", ["up", "down", "low"])
def test_prefill_cap_far_first_tile(tm, dev, cap, order):
    """A first tile at one end of the cap and the rest at the other: what is
    taken as the reference of a query is far from what its keys come to."""
    g = _gen(32)
    n = 400
    base = _rand((1, 1, D), g, dev, 2.0)
    q = base.expand(n, 8, D).contiguous()
    sign = torch.ones(n, 1, 1, dtype=BF, device=dev)
    sign[:70] = {"up": -1.0, "down": 1.0, "low": -1.0}[order]
    if order != "up":
        sign[70:] = -1.0
    k = (base * sign * 3.0).expand(n, 2, D).contiguous()
    v = _rand((n, 2, D), g, dev, 100.0)
    _prefill(tm, q, k, v, _i32([0, n], dev), 0.1, order, softcap=cap)
    first = torch.arange(n, dtype=torch.int32, device=dev) // 3 * 2
    _prefill(tm, q, k, v, _i32([0, n], dev), 0.1, order, softcap=cap,
             first=first)


RUNS = [1, 0, 33, 64, 65, 200, 31, 7]


@pytest.mark.parametrize("hq,hkv", [(1, 1), (8, 1), (32, 4), (64, 16), (12, 4),
                                    (3, 1), (10, 2), (16, 1), (6, 3)])
def test_prefill_heads(tm, dev, hq, hkv):
    g = _gen(hq * 100 + hkv)
    q, k, v, cu = _packed(RUNS, hq, hkv, g, dev)
    _prefill(tm, q, k, v, cu, 0.1, f"{hq}/{hkv}",
             **_function("cap slopes", hq, g, dev))
    _prefill(tm, q, k, v, cu, 0.1, f"{hq}/{hkv} masks",
             prefix=_i32([5, 3, 20, 64, 1, 150, 0, 7], dev),
             first=_firsts(RUNS, [0] * 8, g, dev))


@pytest.mark.parametrize("name", ["plain", "cap", "soft", "slopes",
                                  "cap slopes"])
@pytest.mark.parametrize("window", [0, 1, 50, 130])
@pytest.mark.parametrize("masks", ["", "prefix", "docs", "any", "both"])
def test_prefill_masks(tm, dev, name, window, masks):
    g = _gen(window + len(name) * 7 + len(masks))
    lens = [70, 300, 5, 129]
    q, k, v, cu = _packed(lens, 8, 2, g, dev)
    kw = _function(name, 8, g, dev)
    if masks in ("prefix", "both"):
        kw["prefix"] = _i32([70, 100, 9, 0], dev)     # whole, part, past, none
    if masks in ("docs", "both"):
        kw["first"] = _documents(lens, [0] * 4, g, dev)
    if masks == "any":
        kw["first"] = _firsts(lens, [0] * 4, g, dev)
    _prefill(tm, q, k, v, cu, 0.09, f"{name} {masks}", window=window, **kw)


@pytest.mark.parametrize("name", ["soft", "cap slopes", "plain"])
def test_prefill_long(tm, dev, name):
    """Many tiles a query, runs of every kind beside each other."""
    g = _gen(31)
    lens = [2100, 1, 777, 1500]
    q, k, v, cu = _packed(lens, 8, 1, g, dev)
    kw = _function(name, 8, g, dev)
    _prefill(tm, q, k, v, cu, D ** -0.5, name,
             prefix=_i32([1000, 1, 0, 1500], dev),
             first=_documents(lens, [0] * 4, g, dev), **kw)
    _prefill(tm, q, k, v, cu, D ** -0.5, name, **kw)


def test_prefill_split_prompt(tm, dev):
    """One prompt of few heads: its keys are split over work-groups."""
    g = _gen(33)
    q, k, v, cu = _packed([3300], 4, 1, g, dev)
    lib = tm._lib.load()
    assert lib.tmopt_attn_prefill_scored_workspace_size(
        1, 3300, 0, 4, 1, 0, 0) > 0
    for name in ("soft", "slopes"):
        _prefill(tm, q, k, v, cu, 0.1, name, **_function(name, 4, g, dev))
    _prefill(tm, q, k, v, cu, 0.1, "masks", prefix=_i32([2000], dev),
             first=_firsts([3300], [0], g, dev))


def test_prefill_empty_rows(tm, dev):
    """Rows whose mask leaves nothing: zeros, LSE -inf, whole blocks and whole
    runs among them."""
    g = _gen(34)
    lens = [100, 300, 40]
    q, k, v, cu = _packed(lens, 8, 2, g, dev)
    first = torch.full((440,), 2 ** 31 - 1, dtype=torch.int32, device=dev)
    first[120:130] = 0
    first[400:] = 39
    out, lse = _prefill(tm, q, k, v, cu, 0.1, first=first, softcap=5.0)
    assert (out[:100] == 0).all() and (out[130:400] == 0).all()
    assert (lse[:, :100] == -math.inf).all()
    assert (lse[:, 439:] != -math.inf).all()
    _prefill(tm, q, k, v, cu, 0.1, first=first, prefix=_i32([50, 0, 40], dev),
             slopes=torch.full((8,), 0.1, device=dev))


def test_prefill_given_outputs_and_refusal(tm, dev):
    g = _gen(35)
    lens = [50, 130]
    q, k, v, cu = _packed(lens, 8, 2, g, dev)
    want = tm.prefill_scored_varlen(q, k, v, cu, 0.1, softcap=5.0)
    big = torch.full((200, 10, D), 7.0, dtype=BF, device=dev)
    lse = torch.full((8, 180), 7.0, device=dev)
    reject = _i32([0], dev)
    tm.prefill_scored_varlen(q, k, v, cu, 0.1, softcap=5.0,
                             out=big[:180, 1:9], lse=lse, max_seqlen=130,
                             reject=reject)
    assert torch.equal(big[:180, 1:9], want[0]) and torch.equal(lse, want[1])
    assert (big[180:] == 7).all() and (big[:, 0] == 7).all()
    reject.fill_(1)
    tm.prefill_scored_varlen(q, k, v, cu, 0.1, softcap=5.0,
                             out=big[:180, 1:9], lse=lse, reject=reject)
    assert torch.isnan(big[:180, 1:9]).all() and torch.isnan(lse).all()
    assert (big[180:] == 7).all() and (big[:, 9] == 7).all()
    # rows behind the last run stay; no run and no token at all
    out = torch.full((180, 8, D), 7.0, dtype=BF, device=dev)
    tm.prefill_scored_varlen(q, k, v, cu[:2], 0.1, softcap=5.0, out=out)
    assert torch.equal(out[:50], want[0][:50]) and (out[50:] == 7).all()
    o, l = tm.prefill_scored_varlen(q[:0], k[:0], v[:0], cu[:1], 0.1,
                                    softcap=5.0)
    assert o.shape == (0, 8, D) and l.shape == (8, 0)


def test_prefill_no_number(tm, dev):
    g = _gen(36)
    q, k, v, cu = _packed([100, 90], 4, 1, g, dev)
    k[60, 0, 3] = NAN
    out, lse = tm.prefill_scored_varlen(q, k, v, cu, 0.1, softcap=5.0)
    assert torch.isnan(out[60:100]).all() and torch.isnan(lse[:, 60:100]).all()
    assert torch.isfinite(out[:60]).all() and torch.isfinite(out[100:]).all()
    assert torch.isfinite(lse[:, :60]).all()


# --------------------------------------------------------------------------
# prefill: chunks over the pages, bf16 and 4 bits
# --------------------------------------------------------------------------

def _chunk(tm, c, q, cu, prior, scale, what="", four=False, first=None,
           prefix=None, most=None, **kw):
    if four:
        out, lse = tm.prefill_mx4_varlen(q, c.pool, c.table, cu, prior, scale,
                                         max_context=most, **kw)
    else:
        out, lse = tm.prefill_scored_varlen(
            q, None, None, cu, scale, prior_lens=prior, k_pool=c.kp,
            v_pool=c.vp, block_table=c.table, first_keys=first,
            prefix_lens=prefix, max_context=most, **kw)
    ref.check(out, lse, ref.prefill(q, None, None, cu, scale, prior=prior,
                                    k_pool=c.kp, v_pool=c.vp, table=c.table,
                                    first=first, prefix=prefix, **kw), what)
    return out, lse


CHUNKS = [(1, 0), (17, 100), (64, 64), (0, 50), (130, 0), (5, 1000), (40, 17),
          (1, 333)]


@pytest.mark.parametrize("hq,hkv", [(8, 1), (32, 4), (64, 16), (6, 2), (5, 5)])
@pytest.mark.parametrize("four", [0, 1])
def test_chunk_heads(tm, dev, hq, hkv, four):
    g = _gen(hq * 100 + hkv)
    ends = [a + b for a, b in CHUNKS]
    c = Cache4(tm, ends, hkv, g, dev) if four else Cache(ends, hkv, g, dev)
    lens, prior = [a for a, _ in CHUNKS], [b for _, b in CHUNKS]
    q, _, _, cu = _packed(lens, hq, 1, g, dev)
    for name in ("soft slopes", "plain"):
        _chunk(tm, c, q, cu, _i32(prior, dev), 0.1, name, four,
               **_function(name, hq, g, dev))
    if four:
        _chunk(tm, c, q, cu, _i32(prior, dev), 0.1, "rel", four,
               rel=_rand((sum(lens), hq, 77), g, dev))


@pytest.mark.parametrize("window", [0, 1, 30, 128, 500])
@pytest.mark.parametrize("name", ["plain", "cap", "slopes", "cap slopes",
                                  "rel", "wide rel"])
def test_chunk4_windows(tm, dev, window, name):
    g = _gen(window)
    ends = [a + b for a, b in CHUNKS]
    prior = [b for _, b in CHUNKS]
    c = Cache4(tm, ends, 2, g, dev, first=[max(0, p - window + 1)
                                           if window else 0 for p in prior])
    q, _, _, cu = _packed([a for a, _ in CHUNKS], 8, 1, g, dev)
    kw = _function(name, 8, g, dev)
    if "rel" in name:
        kw["rel"] = _rand((q.shape[0], 8, 600 if "wide" in name else 33), g,
                          dev)
    _chunk(tm, c, q, cu, _i32(prior, dev), 0.1, name, 1, window=window, **kw)


@pytest.mark.parametrize("window", [0, 40, 300])
@pytest.mark.parametrize("masks", ["prefix", "docs", "any", "both"])
def test_chunk_masks(tm, dev, window, masks):
    g = _gen(window + len(masks))
    lens, prior = [a for a, _ in CHUNKS], [b for _, b in CHUNKS]
    ends = [a + b for a, b in CHUNKS]
    c = Cache(ends, 2, g, dev, first=[max(0, p - window + 1) if window else 0
                                      for p in prior])
    q, _, _, cu = _packed(lens, 8, 1, g, dev)
    kw = _function("soft slopes", 8, g, dev)
    if masks in ("prefix", "both"):
        kw["prefix"] = _i32([1, 110, 128, 40, 64, 1002, 0, 5000], dev)
    if masks in ("docs", "both"):
        kw["first"] = _documents(lens, prior, g, dev)
    if masks == "any":
        kw["first"] = _firsts(lens, prior, g, dev)
    _chunk(tm, c, q, cu, _i32(prior, dev), 0.1, masks, window=window, **kw)


@pytest.mark.parametrize("four", [0, 1])
@pytest.mark.parametrize("lens,prior", [([64], [9000]), ([1, 3], [5000, 7001]),
                                        ([200], [3000])])
def test_chunk_split_keys(tm, dev, four, lens, prior):
    """Few queries after much context: the keys are split over work-groups."""
    g = _gen(len(lens) + prior[0])
    ends = [a + b for a, b in zip(lens, prior)]
    c = Cache4(tm, ends, 2, g, dev) if four else Cache(ends, 2, g, dev)
    q, _, _, cu = _packed(lens, 16, 1, g, dev)
    p = _i32(prior, dev)
    size = tm._lib.load().tmopt_attn_prefill_mx4_workspace_size
    assert size(len(lens), max(lens), max(ends), 16, 2, c.table.shape[1],
                0) > 0
    for name in ("soft", "slopes", "plain"):
        _chunk(tm, c, q, cu, p, 0.1, name, four, most=max(ends),
               **_function(name, 16, g, dev))
    # in one launch, where the bound says that contexts are short: same rows
    if four:
        _chunk(tm, c, q, cu, p, 0.1, "rel", 1, most=max(ends),
               rel=_rand((sum(lens), 16, 1024), g, dev))
        _chunk(tm, c, q, cu, p, 0.1, "one launch", 1, most=1)
    else:
        _chunk(tm, c, q, cu, p, 0.1, "masks", prefix=_i32(
            [x - 20 for x in prior], dev), first=_firsts(lens, prior, g, dev))
        _chunk(tm, c, q, cu, p, 0.1, "one launch", most=1, softcap=9.0)


@pytest.mark.parametrize("four", [0, 1])
def test_pages_far_into_the_pool(tm, dev, four):
    """Rows past 2^32 bytes of the pools, by decode and prefill."""
    g = _gen(33)
    hkv = 16
    P = 2 ** 32 // (hkv * (ref.RECORD if four else PAGE * D * 2)) + 40
    ids = [P - 1, 3, P - 7, P - 2]
    c = Cache([60], hkv, g, dev)
    far = _i32([ids], dev)
    pos = torch.arange(60, device=dev)
    near = c.table[0][pos // PAGE].long(), pos % PAGE
    q = _rand((9, 32, D), g, dev)
    cu, prior = _i32([0, 9], dev), _i32([51], dev)
    kw = dict(softcap=3.0)
    if four:
        pool = torch.empty((P, hkv, ref.RECORD), dtype=torch.uint8, device=dev)
        rows = far[0][pos // PAGE].long() * PAGE + pos % PAGE
        tm.kv_write_mx4(c.kp[near], c.vp[near], rows, pool)
        c.kp[near], c.vp[near] = tm.kv_read_mx4(pool, rows)
        got = tm.decode_mx4_paged(q[8:], pool, far, c.ctx, 0.1, **kw)
        chunk = tm.prefill_mx4_varlen(q, pool, far, cu, prior, 0.1, **kw)
    else:
        kp, vp = (torch.empty((P, PAGE, hkv, D), dtype=BF, device=dev)
                  for _ in range(2))
        for i, page in enumerate(ids):
            kp[page], vp[page] = c.kp[c.table[0, i]], c.vp[c.table[0, i]]
        got = tm.decode_scored_paged(q[8:], kp, vp, far, c.ctx, 0.1, **kw)
        chunk = tm.prefill_scored_varlen(
            q, None, None, cu, 0.1, prior_lens=prior, k_pool=kp, v_pool=vp,
            block_table=far, **kw)
    ref.check(*got, ref.decode(q[8:], c.kp, c.vp, c.table, c.ctx, 0.1, **kw))
    ref.check(*chunk, ref.prefill(q, None, None, cu, 0.1, prior=prior,
                                  k_pool=c.kp, v_pool=c.vp, table=c.table,
                                  **kw))


@pytest.mark.parametrize("four", [0, 1])
def test_chunk_missing_pages(tm, dev, four):
    """Entries before the window may name no page; ones that a query sees read
    as zeros."""
    g = _gen(41)
    ends = [330, 64]
    c = Cache4(tm, ends, 2, g, dev) if four else Cache(ends, 2, g, dev)
    q, _, _, cu = _packed([30, 4], 8, 1, g, dev)
    p = _i32([300, 60], dev)
    want = _chunk(tm, c, q, cu, p, 0.1, "all", four, window=100, softcap=4.0)
    c.table[0, :12] = torch.tensor([-1, 10 ** 6] * 6, dtype=torch.int32)
    kw = dict(window=100, softcap=4.0)
    if four:
        got = tm.prefill_mx4_varlen(q, c.pool, c.table, cu, p, 0.1, **kw)
    else:
        got = tm.prefill_scored_varlen(q, None, None, cu, 0.1, prior_lens=p,
                                       k_pool=c.kp, v_pool=c.vp,
                                       block_table=c.table, **kw)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    c.table[1, 2] = -1
    if four:
        got = tm.prefill_mx4_varlen(q, c.pool, c.table, cu, p, 0.1)
    else:
        got = tm.prefill_scored_varlen(q, None, None, cu, 0.1, prior_lens=p,
                                       k_pool=c.kp, v_pool=c.vp,
                                       block_table=c.table)
    pos = torch.arange(64, device=dev)
    K, V = (ref.rows_of(x, c.table[1].clamp(min=0), pos).clone()
            for x in (c.kp, c.vp))
    K[32:48], V[32:48] = 0, 0
    r = ref.attend(q[30:], K, V, pos[60:], pos, 0.1)
    ref.check(got[0][30:], got[1][:, 30:], r)


def test_chunk4_refused_and_replayed(tm, dev):
    g = _gen(42)
    c = Cache4(tm, [400, 64], 2, g, dev)
    q, _, _, cu = _packed([30, 4], 8, 1, g, dev)
    p, reject = _i32([370, 60], dev), _i32([0], dev)
    want = tm.prefill_mx4_varlen(q, c.pool, c.table, cu, p, 0.1, softcap=3.0,
                                 max_seqlen=30)
    out, lse = torch.empty_like(want[0]), torch.empty_like(want[1])
    graph = torch.cuda.CUDAGraph()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        tm.prefill_mx4_varlen(q, c.pool, c.table, cu, p, 0.1, softcap=3.0,
                              max_seqlen=30, out=out, lse=lse, reject=reject)
    torch.cuda.current_stream().wait_stream(s)
    with torch.cuda.graph(graph):
        tm.prefill_mx4_varlen(q, c.pool, c.table, cu, p, 0.1, softcap=3.0,
                              max_seqlen=30, out=out, lse=lse, reject=reject)
    for bad in (0, 1, 0, 0, 1):
        reject.fill_(bad)
        graph.replay()
        torch.cuda.synchronize()
        if bad:
            assert torch.isnan(out).all() and torch.isnan(lse).all()
        else:
            assert torch.equal(out, want[0]) and torch.equal(lse, want[1])


def test_chunk4_no_number(tm, dev):
    g = _gen(43)
    c = Cache4(tm, [400], 1, g, dev)
    q, _, _, cu = _packed([100], 4, 1, g, dev)
    p = _i32([300], dev)
    c.pool[int(c.table[0, 350 // 16]), 0, 2048 + 350 % 16] = 255   # K, block 0
    for kw in (dict(), dict(softcap=4.0), dict(most=0)):
        kw.pop("most", None)
        out, lse = tm.prefill_mx4_varlen(q, c.pool, c.table, cu, p, 0.1, **kw)
        assert torch.isnan(out[50:]).all() and torch.isnan(lse[:, 50:]).all()
        assert torch.isfinite(out[:50]).all()
        assert torch.isfinite(lse[:, :50]).all()


# --------------------------------------------------------------------------
# the operators together, as a step uses them
# --------------------------------------------------------------------------

def test_serving_steps_over_the_4_bit_cache(tm, dev):
    """plan_pages, kv_write_mx4, prefill_mx4_varlen and decode_mx4_paged over
    three steps of two requests: rows as the definition has them of what the
    cache holds."""
    g = _gen(51)
    hq, hkv, P = 8, 2, 40
    pool = tm.mx4_pool(P, hkv, dev)
    pages = torch.full((4, 16), -1, dtype=torch.int32, device=dev)
    free = torch.randperm(P, generator=g).to(torch.int32).to(dev)
    count = _i32([P], dev)
    slots = torch.tensor([2, 0], device=dev)
    ctx = _i32([0, 0], dev)
    kept = [[], []]
    for new in ([70, 33], [21, 60], [1, 1]):
        T = sum(new)
        plan = tm.plan_pages(pages, slots, ctx, _i32(new, dev), free, count, T)
        assert int(plan.reject) == 0
        q, k, v, _ = _packed(new, hq, hkv, g, dev)
        tm.kv_write_mx4(k, v, plan.slot_mapping, pool)
        for i in range(2):
            a, b = int(plan.cu_seqlens[i]), int(plan.cu_seqlens[i + 1])
            kept[i].append((ref.held(k[a:b].cpu()), ref.held(v[a:b].cpu())))
        if T > 2:
            out, lse = tm.prefill_mx4_varlen(
                q, pool, plan.block_table, plan.cu_seqlens, ctx, 0.1,
                softcap=6.0, max_seqlen=max(new), reject=plan.reject)
        else:
            out, lse = tm.decode_mx4_paged(
                q.contiguous(), pool, plan.block_table, plan.seq_lens, 0.1,
                softcap=6.0)
            lse = lse.T
        for i in range(2):
            a, b = int(plan.cu_seqlens[i]), int(plan.cu_seqlens[i + 1])
            K, V = (torch.cat([x[j] for x in kept[i]]).to(dev) for j in (0, 1))
            n = K.shape[0]
            r = ref.attend(q[a:b], K, V, torch.arange(n - (b - a), n,
                                                      device=dev),
                           torch.arange(n, device=dev), 0.1, softcap=6.0)
            ref.check(out[a:b], lse[:, a:b], r, f"request {i}")
        ctx, count = plan.seq_lens, plan.free_count


def test_scored_prefill_then_decode(tm, dev):
    """A prompt with a prefix, written to the pages, then decoded token by
    token: the decode's rows are the prefill's of the longer prompt."""
    g = _gen(52)
    hq, hkv, n = 8, 2, 75
    q, k, v, _ = _packed([n + 3], hq, hkv, g, dev)
    kp = torch.full((9, PAGE, hkv, D), NAN, dtype=BF, device=dev)
    vp = torch.full_like(kp, NAN)
    table = torch.randperm(9, generator=g).to(torch.int32).to(dev)[None]
    kw = _function("soft slopes", hq, g, dev)
    prefix = _i32([40], dev)
    tm.kv_write_paged(k[:n], v[:n], table, _i32([0], dev), kp, vp,
                      cu_seqlens=_i32([0, n], dev))
    _prefill(tm, q[:n], k[:n], v[:n], _i32([0, n], dev), 0.1, prefix=prefix,
             **kw)
    for i in range(n, n + 3):
        tm.kv_write_paged(k[i:i + 1], v[i:i + 1], table, _i32([i], dev), kp,
                          vp)
        out, lse = tm.decode_scored_paged(q[i:i + 1].contiguous(), kp, vp,
                                          table, _i32([i + 1], dev), 0.1, **kw)
        r = ref.attend(q[i:i + 1], k[:i + 1], v[:i + 1],
                       torch.tensor([i], device=dev),
                       torch.arange(i + 1, device=dev), 0.1, prefix=40, **kw)
        ref.check(out, lse.T, r)


def test_captured_step_over_the_4_bit_cache(tm, dev):
    """Plan, write and decode of a step in one graph, replayed while the requests
    grow over page borders, with eager work between the replays."""
    g = _gen(53)
    B, hq, hkv, P = 3, 16, 2, 12
    pool = tm.mx4_pool(P, hkv, dev)
    pages = torch.full((B, 5), -1, dtype=torch.int32, device=dev)
    free = torch.randperm(P, generator=g).to(torch.int32).to(dev)
    slots = torch.arange(B, device=dev)
    q, k, v = (torch.empty((B, h, D), dtype=BF, device=dev)
               for h in (hq, hkv, hkv))
    ctx, count, new = _i32([0, 0, 0], dev), _i32([P], dev), _i32([1] * B, dev)
    plan = tm.plan_pages(pages, slots, ctx, new, free, count, B)
    plan = plan._replace(seq_lens=ctx, free_count=count)
    ws = tm.decode_mx4_workspace(B, hq, hkv, dev)
    out = torch.empty_like(q)
    lse = torch.empty((B, hq), device=dev)

    def step():
        tm.plan_pages(pages, slots, ctx, new, free, count, B, out=plan)
        tm.kv_write_mx4(k, v, plan.slot_mapping, pool)
        tm.decode_mx4_paged(q, pool, plan.block_table, plan.seq_lens, 0.1,
                            softcap=9.0, out=out, lse=lse, workspace=ws)

    for x in (q, k, v):
        x.copy_(_rand(x.shape, g, dev))
    step()
    pages.fill_(-1)
    count.fill_(P)
    ctx.zero_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    held = []
    for i in range(40):
        for x in (q, k, v):
            x.copy_(_rand(x.shape, g, dev))
        graph.replay()
        torch.cuda.synchronize()
        assert int(plan.reject) == 0 and ctx.tolist() == [i + 1] * B
        held.append((ref.held(k.cpu()), ref.held(v.cpu())))
        if i % 8 and i not in (15, 17):
            continue
        for b in range(B):
            K, V = (torch.stack([x[j][b] for x in held]).to(dev)
                    for j in (0, 1))
            r = ref.attend(q[b:b + 1], K, V, torch.tensor([i], device=dev),
                           torch.arange(i + 1, device=dev), 0.1, softcap=9.0)
            ref.check(out[b:b + 1], lse[b:b + 1].T, r, f"step {i}")


# --------------------------------------------------------------------------
# what else the documentation allows
# --------------------------------------------------------------------------

def test_calls_of_nothing(tm, dev):
    g = _gen(54)
    c, c4 = Cache([20], 2, g, dev), Cache4(tm, [20], 2, g, dev)
    q = _rand((4, 8, D), g, dev)
    none, cu0 = q[:0], _i32([0], dev)
    t0, n0 = c.table[:0], c.ctx[:0]
    for out, lse in (
            tm.decode_scored_paged(none, c.kp, c.vp, t0, n0, 0.1),
            tm.decode_mx4_paged(none, c4.pool, t0, n0, 0.1)):
        assert out.shape == (0, 8, D) and lse.shape == (0, 8)
    kept = torch.full_like(q, 3.0)
    paged = dict(k_pool=c.kp, v_pool=c.vp, block_table=t0)
    for run in (
            lambda **kw: tm.prefill_scored_varlen(q, None, None, cu0, 0.1,
                                                  **paged, **kw),
            lambda **kw: tm.prefill_mx4_varlen(q, c4.pool, t0, cu0, None, 0.1,
                                               **kw)):
        run(out=kept)                    # no run: every row as it was
        assert (kept == 3.0).all()
    for cu in ([0, 0], [0, 0, 0]):       # runs without a query
        tm.prefill_scored_varlen(q, q[:, :2], q[:, :2], _i32(cu, dev), 0.1,
                                 out=kept)
        assert (kept == 3.0).all()
    out, lse = tm.prefill_scored_varlen(none, none[:, :2], none[:, :2],
                                        _i32([0, 0], dev), 0.1, max_seqlen=64)
    assert out.shape == (0, 8, D) and lse.shape == (8, 0)


@pytest.mark.parametrize("extent", [1, 2, 5, 16, 63, 900])
def test_bias_views(tm, dev, extent):
    """A bias whose rows begin at any two bytes."""
    g = _gen(55 + extent)
    ends = [1, 5, 17, 64, 100, 700]
    c = Cache4(tm, ends, 2, g, dev)
    B, hq = len(ends), 8
    q = _rand((B, hq, D), g, dev)
    store = _rand((B * hq * extent + 3,), g, dev)
    for off in (0, 1, 3):
        rel = store[off:off + B * hq * extent].view(B, hq, extent)
        out, lse = tm.decode_mx4_paged(q, c.pool, c.table, c.ctx, 0.1, rel=rel)
        ref.check(out, lse, ref.decode(q, c.kp, c.vp, c.table, c.ctx, 0.1,
                                       rel=rel), f"offset {off}")
    lens = [1, 4, 16, 30, 77, 600]
    q, _, _, cu = _packed(lens, hq, 1, g, dev)
    wide = _rand((q.shape[0], hq, extent + 5), g, dev)
    for off in (0, 1, 4):
        _chunk(tm, c, q, cu, _i32([n - m for n, m in zip(ends, lens)], dev),
               0.1, f"offset {off}", 1, rel=wide[..., off:off + extent])


@pytest.mark.parametrize("four", [0, 1])
def test_many_short_runs(tm, dev, four):
    g = _gen(56)
    n = 3000
    lens = torch.randint(0, 4, (n,), generator=g).tolist()
    prior = torch.randint(0, 20, (n,), generator=g).tolist()
    ends = [a + b for a, b in zip(lens, prior)]
    c = Cache4(tm, ends, 1, g, dev) if four else Cache(ends, 1, g, dev)
    q, _, _, cu = _packed(lens, 4, 1, g, dev)
    kw = dict(softcap=9.0)
    if four:
        got = tm.prefill_mx4_varlen(q, c.pool, c.table, cu, _i32(prior, dev),
                                    0.1, **kw)
    else:
        got = tm.prefill_scored_varlen(
            q, None, None, cu, 0.1, prior_lens=_i32(prior, dev), k_pool=c.kp,
            v_pool=c.vp, block_table=c.table, **kw)
    assert torch.isfinite(got[0]).all()
    for i in list(range(0, n, 61)) + [n - 1]:
        a, b = int(cu[i]), int(cu[i + 1])
        if a == b:
            continue
        pos = torch.arange(ends[i], device=dev)
        rows = c.table[i][pos // PAGE].long(), pos % PAGE
        r = ref.attend(q[a:b], c.kp[rows], c.vp[rows],
                       torch.arange(prior[i], ends[i], device=dev), pos, 0.1,
                       **kw)
        ref.check(got[0][a:b], got[1][:, a:b], r, f"run {i}")


def test_prefills_at_once_on_two_streams(tm, dev):
    """Calls that split their keys, each with scratch of its own."""
    g = _gen(57)
    c = Cache([5200], 2, g, dev)
    c4 = Cache4(tm, [5200], 2, g, dev)
    q, _, _, cu = _packed([200], 16, 1, g, dev)
    p = _i32([5000], dev)

    def calls():
        return (tm.prefill_scored_varlen(
                    q, None, None, cu, 0.1, softcap=30.0, prior_lens=p,
                    k_pool=c.kp, v_pool=c.vp, block_table=c.table,
                    max_seqlen=200),
                tm.prefill_mx4_varlen(q, c4.pool, c4.table, cu, p, 0.1,
                                      max_seqlen=200))
    want = calls()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(5):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(calls())
    torch.cuda.synchronize()
    for a in got:
        for x, y in zip(a, want):
            assert torch.equal(x[0], y[0]) and torch.equal(x[1], y[1])
