"""The 4-bit cache (kv_write_mx4, kv_read_mx4, decode_mx4_paged) against its
definition: rows byte by byte, attention in float64 within the bounds that
oracle/scored_ref.py derives. Bytes that no request owns are 0xff: elements of
-6 under a scale that is no number."""
import math

import pytest
import torch

from oracle import scored_ref as ref

pytestmark = pytest.mark.gpu
D, PAGE = 128, 16
BF = torch.bfloat16


def _gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def _rand(shape, g, std=1.0):
    return (torch.randn(shape, generator=g) * std).to(BF)


def _junk_pool(P, hkv, dev):
    return torch.full((P, hkv, ref.RECORD), 255, dtype=torch.uint8, device=dev)


class Cache4:
    """A 4-bit cache in which request i's positions [first_i, n_i) hold values
    (written by the package) behind shuffled pages; kp, vp: what it holds."""

    def __init__(self, tm, ends, hkv, g, dev, first=None, wrap=0, width=None,
                 spare=3):
        pages = [wrap or -(-n // PAGE) for n in ends]
        P = sum(pages) + spare
        perm = torch.randperm(P - 1, generator=g).to(torch.int32)
        w = width or max(pages + [1])
        self.table = torch.full((len(ends), w), P - 1, dtype=torch.int32)
        off = 0
        for i, n in enumerate(pages):
            self.table[i, :n] = perm[off:off + n]
            off += n
        self.pool = _junk_pool(P, hkv, dev)
        rows = []
        for i, n in enumerate(ends):
            pos = torch.arange(0 if first is None else first[i], n)
            lp = pos // PAGE % wrap if wrap else pos // PAGE
            rows.append(self.table[i][lp].long() * PAGE + pos % PAGE)
        rows = torch.cat(rows).to(dev)
        T = rows.numel()
        if T:
            tm.kv_write_mx4(_rand((T, hkv, D), g).to(dev),
                            _rand((T, hkv, D), g).to(dev), rows, self.pool)
        every = torch.arange(P * PAGE, device=dev)
        self.kp, self.vp = (x.view(P, PAGE, hkv, D)
                            for x in tm.kv_read_mx4(self.pool, every))
        self.table = self.table.to(dev)
        self.ctx = torch.tensor(ends, dtype=torch.int32, device=dev)


def _decode(tm, c, q, scale, what="", wrap=0, window=0, **kw):
    split = {k: kw.pop(k) for k in ("min_pages", "num_workgroups")
             if k in kw}
    out, lse = tm.decode_mx4_paged(q, c.pool, c.table, c.ctx, scale,
                                   window=window, table_wrap=wrap, **kw,
                                   **split)
    ref.check(out, lse, ref.decode(q, c.kp, c.vp, c.table, c.ctx, scale,
                                   window=window, table_wrap=wrap, **kw),
              what)
    return out, lse


# --------------------------------------------------------------------------
# rows in and out
# --------------------------------------------------------------------------

SPECIAL = [0.0, -0.0, 1.0, -7.0, 7.0, 7.03125, 6.0, 5.0, 3.5, 2.5, 1.75, 1.25,
           0.75, 0.25, 0.2490234375, 0.251953125, -5.0, -3.5, 448.0, 2e-38,
           9.1835e-41, 7 * 2.0 ** 125, 3e38, math.inf, -math.inf, math.nan,
           1e30, 2.0 ** -125, 2.0 ** -126, 3 * 2.0 ** -125]


@pytest.mark.parametrize("hkv,T", [(1, 1), (4, 15), (2, 16), (3, 17),
                                   (8, 70), (16, 33)])
def test_write_bytes(tm, dev, hkv, T):
    g = _gen(hkv * 100 + T)
    k, v = _rand((T, hkv, D), g, 3.0), _rand((T, hkv, D), g, 0.01)
    # blocks of every kind: one special value among small ones, or alone
    for i, x in enumerate(SPECIAL):
        t, h, b = i % T, i % hkv, i % 4
        k[t, h, 32 * b:32 * b + 32] *= 0.1 if i % 2 else 0.0
        k[t, h, 32 * b + (7 * i) % 32] = x
        v[t, h, 32 * b + (5 * i) % 32] = x
    P = T // PAGE + 3
    rows = torch.randperm(P * PAGE, generator=g)[:T]
    want = _junk_pool(P, hkv, "cpu")
    for t in range(T):
        ref.put(want, int(rows[t]), k[t], v[t])
    pool = _junk_pool(P, hkv, dev)
    # rows as parts of wider ones
    wide = torch.zeros((T, hkv + 2, 2 * D), dtype=BF)
    wide[:, 1:-1, :D], wide[:, 2:, D:] = k, v
    wide = wide.to(dev)
    tm.kv_write_mx4(wide[:, 1:-1, :D], wide[:, 2:, D:], rows.to(dev), pool)
    assert torch.equal(pool.cpu(), want)
    K, V = tm.kv_read_mx4(pool, rows.to(dev))
    for got, x in ((K, k), (V, v)):
        assert torch.equal(torch.nan_to_num(got.cpu().double(), 77.0),
                           torch.nan_to_num(ref.held(x), 77.0))


def test_every_value(tm, dev):
    """Each finite bf16 as the largest of its block, beside each of a few."""
    x = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(BF)
    x = x[torch.isfinite(x)]
    rows = torch.zeros((x.numel(), 4, 32), dtype=BF)
    part = torch.tensor([1.0, 0.5, -0.27, 0.1])
    rows[:, 0, 0] = x
    rows[:, 1, :4] = (x.double()[:, None] * part.double()).to(BF)
    rows[:, 2, 31] = x
    rows[:, 2, 30] = 1.0
    rows[:, 3] = 3.0
    rows = rows.view(-1, 1, D)
    n = rows.shape[0]
    pool = tm.mx4_pool(-(-n // PAGE), 1, dev)
    at = torch.arange(n, device=dev)
    tm.kv_write_mx4(rows.to(dev), rows.flip(0).to(dev), at, pool)
    K, V = tm.kv_read_mx4(pool, at)
    want = ref.held(rows)
    # (bf16 flushes nothing here: a value of 2^-126 is the smallest held)
    assert torch.equal(torch.nan_to_num(K.cpu().double(), 77.0),
                       torch.nan_to_num(want, 77.0))
    assert torch.equal(torch.nan_to_num(V.cpu().double(), 77.0),
                       torch.nan_to_num(want.flip(0), 77.0))


def test_rows_outside_the_pool(tm, dev):
    g = _gen(5)
    k, v = _rand((5, 2, D), g).to(dev), _rand((5, 2, D), g).to(dev)
    pool = _junk_pool(3, 2, dev)
    rows = torch.tensor([-1, 3 * PAGE, 7, 2 ** 40, -2 ** 40], device=dev)
    tm.kv_write_mx4(k, v, rows, pool)
    want = _junk_pool(3, 2, "cpu")
    ref.put(want, 7, k[2].cpu(), v[2].cpu())
    assert torch.equal(pool.cpu(), want)
    K, V = tm.kv_read_mx4(pool, rows)
    assert (K[[0, 1, 3, 4]] == 0).all() and (V[[0, 1, 3, 4]] == 0).all()
    assert torch.equal(K[2].cpu().double(), ref.held(k[2].cpu()))
    tm.kv_write_mx4(k[:0], v[:0], rows[:0], pool)
    assert tm.kv_read_mx4(pool, rows[:0])[0].shape == (0, 2, D)


# --------------------------------------------------------------------------
# decode
# --------------------------------------------------------------------------

EDGES = [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 129, 300, 700]


@pytest.mark.parametrize("hq,hkv", [(1, 1), (8, 1), (32, 4), (64, 16), (64, 8),
                                    (12, 4), (3, 3), (10, 2), (16, 1), (34, 2),
                                    (20, 5), (24, 2), (18, 2)])
def test_decode_heads(tm, dev, hq, hkv):
    g = _gen(hq * 100 + hkv)
    c = Cache4(tm, EDGES, hkv, g, dev)
    q = _rand((len(EDGES), hq, D), g, 2.0).to(dev)
    _decode(tm, c, q, D ** -0.5, f"{hq}/{hkv}")
    _decode(tm, c, q, D ** -0.5, f"{hq}/{hkv} split", min_pages=1)


FUNCTIONS = ["plain", "cap", "slopes", "both", "rel", "odd rel"]


def _function(name, hq, B, g, dev):
    kw = {}
    if name in ("cap", "both"):
        kw["softcap"] = 5.0
    if name in ("slopes", "both"):
        kw["slopes"] = (torch.rand(hq, generator=g) * 0.3 - 0.05).to(dev)
    if "rel" in name:
        kw["rel"] = _rand((B, hq, 33 if "odd" in name else 100), g).to(dev)
    return kw


@pytest.mark.parametrize("name", FUNCTIONS)
@pytest.mark.parametrize("window", [0, 1, 16, 100, 512])
@pytest.mark.parametrize("min_pages,wgs", [(8, 0), (1, 0), (1, 7), (3, 64),
                                           (200, 0)])
def test_decode_windows_and_splits(tm, dev, name, window, min_pages, wgs):
    g = _gen(window * 10 + min_pages)
    ends = [0, 1, 16, 99, 100, 101, 511, 512, 513, 800, 1500]
    first = [max(0, n - window) if window else 0 for n in ends]
    c = Cache4(tm, ends, 4, g, dev, first=first)
    q = _rand((len(ends), 16, D), g, 1.5).to(dev)
    _decode(tm, c, q, 0.1, name, window=window, min_pages=min_pages,
            num_workgroups=wgs, **_function(name, 16, len(ends), g, dev))


@pytest.mark.parametrize("name", FUNCTIONS)
@pytest.mark.parametrize("window", [100, 128])
def test_decode_ring(tm, dev, name, window):
    """Rows that are rings of 8 pages: positions wrap around."""
    g = _gen(3)
    ends = [1, 100, 128, 129, 500, 1000]
    c = Cache4(tm, ends, 2, g, dev, first=[max(0, n - 128) for n in ends],
               wrap=8)
    q = _rand((len(ends), 8, D), g).to(dev)
    _decode(tm, c, q, 0.1, name, window=window, wrap=8, min_pages=2,
            **_function(name, 8, len(ends), g, dev))


@pytest.mark.parametrize("window,wrap", [(40, 4), (64, 4), (1, 1)])
@pytest.mark.parametrize("name", ["plain", "slopes", "rel"])
def test_decode_ring_at_the_last_positions(tm, dev, name, window, wrap):
    """A ring's positions may come up to what int32 holds."""
    g = _gen(21)
    ends = [2 ** 31 - 1, 2 ** 31 - 16, 2 ** 31 - 17, 5]
    c = Cache4(tm, ends, 4, g, dev, first=[max(0, n - window) for n in ends],
               wrap=wrap)
    _decode(tm, c, _rand((4, 16, D), g).to(dev), 0.1, name, window=window,
            wrap=wrap, **_function(name, 16, 4, g, dev))


def test_decode_absent_pages(tm, dev):
    """Entries outside the pool and positions past the row's width count as
    absent; a request that has no other page gives zeros."""
    g = _gen(4)
    c = Cache4(tm, [200, 208, 40], 4, g, dev)
    q = _rand((3, 16, D), g).to(dev)
    c.table[0, 3] = -1
    c.table[0, 7] = 10 ** 6
    c.table[2] = -7
    c.ctx[1] = 5000                       # the row holds 13 pages
    for kw in (dict(min_pages=1), dict(min_pages=8)):
        out, lse = tm.decode_mx4_paged(q, c.pool, c.table, c.ctx, 0.1, **kw)
        for b, gone, n in ((0, (3, 7), 200), (1, (), 208)):
            pos = torch.tensor([p for p in range(n) if p // PAGE not in gone],
                               device=dev)
            table = c.table[b].clamp(0, c.pool.shape[0] - 1)
            r = ref.attend(q[b:b + 1], ref.rows_of(c.kp, table, pos),
                           ref.rows_of(c.vp, table, pos),
                           torch.tensor([4999], device=dev), pos, 0.1)
            ref.check(out[b:b + 1], lse[b:b + 1], (r[0], r[1].T, r[2], r[3].T),
                      f"request {b}")
        assert (out[2] == 0).all() and (lse[2] == -math.inf).all()


def test_decode_many_short_and_one_long(tm, dev):
    g = _gen(6)
    ends = [int(x) for x in torch.randint(0, 40, (700,), generator=g)]
    ends[333] = 30001
    c = Cache4(tm, ends, 2, g, dev)
    q = _rand((700, 8, D), g).to(dev)
    _decode(tm, c, q, 0.1, "mixed")
    _decode(tm, c, q, 0.1, "few ranges", num_workgroups=1)


def test_decode_no_number(tm, dev):
    """A key block that is no number makes its requests' outputs and LSE so, a
    value block its 32 dims."""
    g = _gen(7)
    c = Cache4(tm, [50, 400, 400, 30], 2, g, dev)
    q = _rand((4, 8, D), g).to(dev)
    row = lambda b, p: int(c.table[b, p // PAGE])           # noqa: E731
    c.pool[row(1, 200), 1, 2048 + 16 * 2 + 200 % 16] = 255      # K of head 1
    c.pool[row(2, 7), 0, 2112 + 16 * 3 + 7] = 255               # V of head 0
    for kw in (dict(min_pages=1), dict(min_pages=100)):
        out, lse = tm.decode_mx4_paged(q, c.pool, c.table, c.ctx, 0.1, **kw)
        assert torch.isnan(out[1, 4:]).all() and torch.isnan(lse[1, 4:]).all()
        assert torch.isfinite(out[1, :4]).all()
        assert torch.isnan(out[2, :4, 96:]).all()
        assert torch.isfinite(out[2, :4, :96]).all()
        assert torch.isfinite(out[2, 4:]).all() and torch.isfinite(lse[2]).all()
        for b in (0, 3):
            assert torch.isfinite(out[b]).all()


def test_decode_given_outputs_and_streams(tm, dev):
    """Given outputs and workspace, a second stream, and a graph that is
    replayed with other lengths: the same bits."""
    g = _gen(8)
    c = Cache4(tm, [90, 1000, 3, 555], 4, g, dev)
    q = _rand((4, 32, D), g).to(dev)
    want = tm.decode_mx4_paged(q, c.pool, c.table, c.ctx, 0.1)
    ws = tm.decode_mx4_workspace(4, 32, 4, dev)
    out, lse = torch.full_like(want[0], 7), torch.full_like(want[1], 7)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        tm.decode_mx4_paged(q, c.pool, c.table, c.ctx, 0.1, out=out, lse=lse,
                            workspace=ws)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(out, want[0]) and torch.equal(lse, want[1])
    ctx = c.ctx.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        tm.decode_mx4_paged(q, c.pool, c.table, ctx, 0.1, out=out, lse=lse,
                            workspace=ws)
    for lens in ([90, 1000, 3, 555], [1, 64, 0, 300], [90, 999, 2, 16]):
        ctx.copy_(torch.tensor(lens, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        eager = tm.decode_mx4_paged(q, c.pool, c.table, ctx, 0.1)
        assert torch.equal(out, eager[0]) and torch.equal(lse, eager[1])
    o, l = tm.decode_mx4_paged(q, c.pool, c.table, ctx, 0.1, return_lse=False)
    assert l is None and torch.equal(o, out)


def test_decode_large_pool(tm, dev):
    """Records past 2^32 bytes of the pool."""
    g = _gen(9)
    hkv = 16
    P = 2 ** 32 // (hkv * ref.RECORD) + 40
    pool = torch.empty((P, hkv, ref.RECORD), dtype=torch.uint8, device=dev)
    table = torch.tensor([[P - 1, 3, P - 7, P - 2]], dtype=torch.int32,
                         device=dev)
    pos = torch.arange(60, device=dev)
    rows = table[0][pos // PAGE].long() * PAGE + pos % PAGE
    k, v = (_rand((60, hkv, D), g).to(dev) for _ in range(2))
    tm.kv_write_mx4(k, v, rows, pool)
    K, V = tm.kv_read_mx4(pool, rows)
    assert torch.equal(K.cpu().double(), ref.held(k.cpu()))
    q = _rand((1, 64, D), g).to(dev)
    out, lse = tm.decode_mx4_paged(
        q, pool, table, torch.tensor([60], dtype=torch.int32, device=dev), 0.1)
    r = ref.attend(q, K, V, torch.tensor([59], device=dev), pos, 0.1)
    ref.check(out, lse, (r[0], r[1].T, r[2], r[3].T))


def test_decode_largest_batch(tm, dev):
    """8192 requests of 0 to 40 tokens; and work-split knobs at their ends."""
    g = _gen(10)
    ends = [int(x) for x in torch.randint(0, 41, (8192,), generator=g)]
    c = Cache4(tm, ends, 1, g, dev)
    q = _rand((8192, 2, D), g).to(dev)
    out, lse = tm.decode_mx4_paged(q, c.pool, c.table, c.ctx, 0.1)
    pick = [0, 1, 4095, 4096, 8190, 8191] + list(range(100, 8000, 97))
    r = ref.decode(q[pick], c.kp, c.vp, c.table[pick], c.ctx[pick], 0.1)
    ref.check(out[pick], lse[pick], r)
    for kw in (dict(min_pages=2 ** 31 - 1), dict(num_workgroups=65535),
               dict(num_workgroups=1, min_pages=1)):
        o, l = tm.decode_mx4_paged(q, c.pool, c.table, c.ctx, 0.1, **kw)
        ref.check(o[pick], l[pick], r, str(kw))


def test_decode_lengths_past_the_table(tm, dev):
    """Lengths far past what the table's rows hold: those keys are absent."""
    g = _gen(11)
    c = Cache4(tm, [64] * 100, 1, g, dev)
    q = _rand((100, 4, D), g).to(dev)
    c.ctx.fill_(2 ** 31 - 1)
    out, lse = tm.decode_mx4_paged(q, c.pool, c.table, c.ctx, 0.1)
    pos = torch.arange(64, device=dev)
    for b in (0, 1, 57, 99):
        r = ref.attend(q[b:b + 1], ref.rows_of(c.kp, c.table[b], pos),
                       ref.rows_of(c.vp, c.table[b], pos),
                       torch.tensor([2 ** 31 - 2], device=dev), pos, 0.1)
        ref.check(out[b:b + 1], lse[b:b + 1], (r[0], r[1].T, r[2], r[3].T))
    # a window that begins past the table: no key at all
    out, lse = tm.decode_mx4_paged(q, c.pool, c.table, c.ctx, 0.1, window=500)
    assert (out == 0).all() and (lse == -math.inf).all()


@pytest.mark.parametrize("cap", [0.01, 1.0, 62.0, 63.0, 4000.0])
def test_decode_caps(tm, dev, cap):
    """Caps from far below the scores to far above them."""
    g = _gen(12)
    c = Cache4(tm, [33, 500], 1, g, dev)
    q = _rand((2, 8, D), g, 4.0).to(dev)
    _decode(tm, c, q, 0.1, softcap=cap)
    _decode(tm, c, q * 0.01, 0.1, softcap=cap)
