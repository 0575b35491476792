"""Differential attention (decode_diff_paged, prefill_diff_varlen) against its
definition in float64, within the bounds that oracle/diff_ref.py derives.
Pools hold NaN wherever no request owns a row."""
import pytest
import torch

from oracle import diff_ref

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


def _weights(hq, g, dev, norm=True, one=False):
    kw = dict(lam=(torch.rand(1 if one else hq // 2, generator=g) * 1.2 -
                   0.2).to(dev))
    if norm:
        kw.update(weight=(1 + 0.3 * torch.randn(256, generator=g)).to(dev),
                  eps=1e-5, out_scale=0.4)
    return kw


def _user(kw):
    """The oracle's names as the entry points have them."""
    kw = dict(kw)
    if "weight" in kw:
        kw["norm_weight"], kw["norm_eps"] = kw.pop("weight"), kw.pop("eps")
    return kw


class Cache:
    """Pools in which request i's positions [first_i, n_i) hold values and
    everything else is NaN, behind shuffled pages; table entries of pages it
    does not hold name a poisoned page."""

    def __init__(self, ends, hkv, g, dev, first=None, spare=3, width=None,
                 wrap=0):
        pages = [wrap or -(-n // PAGE) for n in ends]
        P = sum(pages) + spare
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
            lo = 0 if first is None else first[i]
            pos = torch.arange(lo, n, device=dev)
            lp = pos // PAGE % wrap if wrap else pos // PAGE
            rows = self.table[i][lp].long(), pos % PAGE
            self.kp[rows] = _rand((n - lo, hkv, D), g, dev)
            self.vp[rows] = _rand((n - lo, hkv, D), g, dev)
        self.ctx = torch.tensor(ends, dtype=torch.int32, device=dev)


def _decode(tm, c, q, scale, w, window=0, wrap=0, what="", **split):
    out, lse = tm.decode_diff_paged(q, c.kp, c.vp, c.table, c.ctx, w["lam"],
                                    scale, window=window, table_wrap=wrap,
                                    **{k: v for k, v in _user(w).items()
                                       if k != "lam"}, **split)
    ref = diff_ref.decode(q, c.kp, c.vp, c.table, c.ctx, w["lam"], scale,
                          window=window, table_wrap=wrap,
                          **{k: v for k, v in w.items() if k != "lam"})
    diff_ref.check(out, lse, ref, what)
    return out, lse


EDGES = [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 300, 700]


@pytest.mark.parametrize("hq,hkv", [(2, 2), (32, 4), (64, 16), (64, 8),
                                    (12, 4), (6, 2), (10, 2), (24, 2),
                                    (34, 2), (20, 10), (24, 12), (16, 2)])
def test_decode_heads(tm, dev, hq, hkv):
    g = _gen(hq * 100 + hkv)
    c = Cache(EDGES, hkv, g, dev)
    q = _rand((len(EDGES), hq, D), g, dev, 2.0)
    _decode(tm, c, q, D ** -0.5, _weights(hq, g, dev),
            what=f"{hq}/{hkv}")
    _decode(tm, c, q, D ** -0.5, _weights(hq, g, dev, norm=False, one=True),
            what=f"{hq}/{hkv} plain", min_pages=1)


@pytest.mark.parametrize("window", [0, 1, 16, 100, 512])
@pytest.mark.parametrize("min_pages,wgs", [(1, 0), (1, 7), (3, 64), (2, 1),
                                           (128, 0)])
def test_decode_windows_and_splits(tm, dev, window, min_pages, wgs):
    g = _gen(window * 10 + min_pages)
    ends = [0, 1, 16, 99, 100, 101, 511, 512, 513, 800, 1500]
    first = [max(0, n - window) if window else 0 for n in ends]
    c = Cache(ends, 4, g, dev, first=first)
    q = _rand((len(ends), 16, D), g, dev, 1.5)
    _decode(tm, c, q, 0.1, _weights(16, g, dev), window=window,
            min_pages=min_pages, num_workgroups=wgs)


@pytest.mark.parametrize("window", [100, 128])
def test_decode_ring(tm, dev, window):
    """Rows that are rings of 8 pages: positions wrap around."""
    g = _gen(3)
    ends = [1, 100, 128, 129, 500, 1000]
    c = Cache(ends, 2, g, dev, first=[max(0, n - 128) for n in ends], wrap=8)
    q = _rand((len(ends), 8, D), g, dev)
    _decode(tm, c, q, 0.1, _weights(8, g, dev), window=window, wrap=8,
            min_pages=2)


@pytest.mark.parametrize("window,wrap", [(40, 4), (64, 4), (1, 1)])
def test_decode_ring_at_the_last_positions(tm, dev, window, wrap):
    """A ring's positions may come up to what int32 holds."""
    g = _gen(21)
    ends = [2 ** 31 - 1, 2 ** 31 - 16, 2 ** 31 - 17, 5]
    c = Cache(ends, 4, g, dev, first=[max(0, n - window) for n in ends],
              wrap=wrap)
    _decode(tm, c, _rand((4, 16, D), g, dev), 0.1, _weights(16, g, dev),
            window=window, wrap=wrap)


def test_decode_absent_pages(tm, dev):
    """Entries outside the pool and positions past the row's width count as
    absent; a request that has no other page gives zeros."""
    g = _gen(4)
    c = Cache([200, 208, 40], 4, g, dev)
    q = _rand((3, 16, D), g, dev)
    w = _weights(16, g, dev)
    c.table[0, 3] = -1
    c.table[0, 7] = 10 ** 6
    c.table[2] = -7
    c.ctx[1] = 5000                       # the row holds 13 pages
    kw = {k: v for k, v in w.items() if k != "lam"}
    out, lse = tm.decode_diff_paged(q, c.kp, c.vp, c.table, c.ctx, w["lam"],
                                    0.1, min_pages=1,
                                    **{k: v for k, v in _user(w).items()
                                       if k != "lam"})
    for b, gone, n in ((0, (3, 7), 200), (1, (), 208)):
        pos = torch.tensor([p for p in range(n) if p // PAGE not in gone],
                           device=dev)
        ref = diff_ref.attend(
            q[b:b + 1], diff_ref.rows_of(c.kp, c.table[b], pos),
            diff_ref.rows_of(c.vp, c.table[b], pos),
            torch.tensor([4999], device=dev), pos, w["lam"], 0.1, **kw)
        diff_ref.check(out[b:b + 1], lse[b:b + 1].T, ref, f"row {b}")
    assert (out[2] == 0).all() and (lse[2] == -torch.inf).all()


@pytest.mark.parametrize("window", [0, 50])
def test_decode_lengths_past_the_table(tm, dev, window):
    """Lengths far past the row's width, up to the largest int32, and negative
    ones: the walk is bounded by the table, what it cannot name is absent."""
    g = _gen(20)
    c = Cache([96, 96, 96, 60, 60], 2, g, dev)
    q = _rand((5, 4, D), g, dev)
    w = _weights(4, g, dev)
    for b, n in ((1, 2 ** 31 - 1), (2, 100), (3, -5)):
        c.ctx[b] = n
    out, lse = tm.decode_diff_paged(q, c.kp, c.vp, c.table, c.ctx, w["lam"],
                                    0.1, window=window)
    for b, n in ((0, 96), (1, 2 ** 31 - 1), (2, 100), (3, 0), (4, 60)):
        lo = max(0, n - window) if window else 0
        pos = torch.arange(min(lo, 96), min(n, 96), device=dev)
        ref = diff_ref.attend(
            q[b:b + 1], diff_ref.rows_of(c.kp, c.table[b], pos),
            diff_ref.rows_of(c.vp, c.table[b], pos),
            torch.tensor([n - 1], device=dev), pos, w["lam"], 0.1,
            window=window)
        diff_ref.check(out[b:b + 1], lse[b:b + 1].T, ref, f"row {b}")


def test_decode_no_requests(tm, dev):
    c = Cache([5], 2, _gen(21), dev)
    out, lse = tm.decode_diff_paged(
        torch.empty((0, 4, D), dtype=BF, device=dev), c.kp, c.vp, c.table,
        c.ctx[:0], torch.ones(2, device=dev), 0.1)
    assert out.shape == (0, 2, 256) and lse.shape == (0, 4)


@pytest.mark.parametrize("std", [0.0, 30.0])
def test_decode_flat_and_peaked(tm, dev, std):
    """Equal scores everywhere, and scores so far apart that each softmax is
    one key."""
    g = _gen(5)
    c = Cache([1, 17, 900], 4, g, dev)
    q = _rand((3, 32, D), g, dev, std)
    _decode(tm, c, q, D ** -0.5, _weights(32, g, dev), min_pages=4)


def test_decode_long(tm, dev):
    """A context that the whole grid shares, beside short ones."""
    g = _gen(6)
    c = Cache([200001, 5, 0, 3000], 2, g, dev)
    q = _rand((4, 16, D), g, dev)
    a, la = _decode(tm, c, q, 0.1, _weights(16, _gen(7), dev))
    b, lb = _decode(tm, c, q, 0.1, _weights(16, _gen(7), dev))
    assert torch.equal(a, b) and torch.equal(la, lb)


def test_decode_many_requests(tm, dev):
    g = _gen(8)
    ends = torch.randint(0, 60, (1500,), generator=g).tolist()
    c = Cache(ends, 2, g, dev)
    q = _rand((1500, 4, D), g, dev)
    _decode(tm, c, q, 0.1, _weights(4, g, dev))


def test_decode_far_pages(tm, dev):
    """Pages past 4 GiB of the pools."""
    g = _gen(9)
    P, hkv, n = 300000, 4, 100
    kp = torch.zeros((P, PAGE, hkv, D), dtype=BF, device=dev)
    vp = torch.zeros_like(kp)
    c = Cache([n, n], hkv, g, dev)
    far = torch.tensor([[P - 1 - i for i in range(7)],
                        [P // 2 + i for i in range(7)]], device=dev)
    kp[far] = c.kp[c.table.long()]
    vp[far] = c.vp[c.table.long()]
    c.kp, c.vp, c.table = kp, vp, far.int()
    _decode(tm, c, _rand((2, 16, D), g, dev), 0.1, _weights(16, g, dev))


def test_decode_buffers_streams_and_graph(tm, dev):
    """Given outputs and workspaces, another stream, and a captured call that
    follows the lengths; a second graph keeps its own workspace."""
    g = _gen(10)
    c = Cache([900, 33, 2000], 4, g, dev)
    q = _rand((3, 32, D), g, dev)
    w = _weights(32, g, dev)
    kw = {k: v for k, v in _user(w).items() if k != "lam"}
    ref, rl = _decode(tm, c, q, 0.1, w)
    out = torch.full((3, 16, 256), NAN, dtype=BF, device=dev)
    lse = torch.full((3, 32), NAN, device=dev)
    ws = tm.decode_diff_workspace(3, 32, 4, dev)
    ws.fill_(255)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        o, l = tm.decode_diff_paged(q, c.kp, c.vp, c.table, c.ctx, w["lam"],
                                    0.1, out=out, lse=lse, workspace=ws, **kw)
    st.synchronize()
    assert o is out and l is lse
    assert torch.equal(out, ref) and torch.equal(lse, rl)
    graphs = []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            res = tm.decode_diff_paged(q, c.kp, c.vp, c.table, c.ctx,
                                       w["lam"], 0.1, **kw)
        graphs.append((gr, res))
    for ends in ([900, 33, 2000], [1, 0, 1999], [800, 16, 3], [900, 33, 2000]):
        c.ctx.copy_(torch.tensor(ends, dtype=torch.int32))
        want = tm.decode_diff_paged(q, c.kp, c.vp, c.table, c.ctx, w["lam"],
                                    0.1, **kw)
        for gr, res in graphs:
            gr.replay()
        torch.cuda.synchronize()
        for gr, res in graphs:
            assert torch.equal(res[0], want[0])
            assert torch.equal(res[1], want[1])


def _cu(lens, dev):
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    return torch.tensor(cu, dtype=torch.int32, device=dev)


def _prefill(tm, q, k, v, cu, w, scale=0.1, what="", call=None, **kw):
    call = dict(call or {})
    call.update({x: y for x, y in _user(w).items() if x != "lam"})
    out, lse = tm.prefill_diff_varlen(
        q, k, v, cu, w["lam"], scale, prior_lens=kw.get("prior"),
        k_pool=kw.get("k_pool"), v_pool=kw.get("v_pool"),
        block_table=kw.get("table"), window=kw.get("window", 0), **call)
    ref = diff_ref.prefill(q, k, v, cu.tolist(), w["lam"], scale,
                           **{x: y for x, y in w.items() if x != "lam"}, **kw)
    n = int(cu[-1])
    diff_ref.check(out[:n], None if lse is None else lse[:, :n],
                   (ref[0][:n], ref[1][:, :n], ref[2][:n], ref[3][:, :n]),
                   what)
    return out, lse


RUNS = [0, 1, 2, 31, 32, 33, 63, 64, 65, 0, 127, 128, 129, 200, 513]


@pytest.mark.parametrize("hq,hkv", [(2, 2), (32, 4), (64, 16), (12, 4),
                                    (24, 2), (10, 2), (16, 2), (20, 10)])
@pytest.mark.parametrize("window", [0, 100])
def test_prefill_heads(tm, dev, hq, hkv, window):
    g = _gen(hq + hkv)
    T = sum(RUNS)
    q = _rand((T, hq, D), g, dev, 2.0)
    k, v = _rand((T, hkv, D), g, dev), _rand((T, hkv, D), g, dev)
    _prefill(tm, q, k, v, _cu(RUNS, dev), _weights(hq, g, dev), D ** -0.5,
             window=window)
    _prefill(tm, q, k, v, _cu(RUNS, dev),
             _weights(hq, g, dev, norm=False, one=True), D ** -0.5,
             window=window, call=dict(max_seqlen=700))


@pytest.mark.parametrize("window", [1, 31, 64, 65, 300])
def test_prefill_windows(tm, dev, window):
    g = _gen(window)
    lens = [1, 64, 65, 700, 1000]
    T = sum(lens)
    _prefill(tm, _rand((T, 8, D), g, dev), _rand((T, 2, D), g, dev),
             _rand((T, 2, D), g, dev), _cu(lens, dev), _weights(8, g, dev),
             window=window)


@pytest.mark.parametrize("hq,hkv,window", [(16, 4, 0), (16, 4, 100),
                                           (64, 8, 0), (4, 2, 1000)])
def test_prefill_paged(tm, dev, hq, hkv, window):
    """Keys from the pools: no context, contexts that end inside a page and
    on its edge, runs of one token; poison outside what a run may see."""
    g = _gen(hq + window)
    lens = [1, 40, 0, 33, 130, 1, 64]
    prior = [0, 16, 50, 100, 15, 700, 1001]
    ends = [a + b for a, b in zip(lens, prior)]
    first = [max(0, p - window + 1) if window else 0 for p in prior]
    c = Cache(ends, hkv, g, dev, first=first)
    q = _rand((sum(lens), hq, D), g, dev)
    _prefill(tm, q, None, None, _cu(lens, dev), _weights(hq, g, dev),
             prior=torch.tensor(prior, dtype=torch.int32, device=dev),
             k_pool=c.kp, v_pool=c.vp, table=c.table, window=window)


@pytest.mark.parametrize("n,prior", [(1, 20000), (64, 9000), (500, 6000),
                                     (200, 0)])
def test_prefill_chunk_after_long_context(tm, dev, n, prior):
    """Few queries, many keys: split over work-groups and joined."""
    g = _gen(n)
    c = Cache([n + prior, 50], 4, g, dev)
    q = _rand((n + 20, 16, D), g, dev)
    cu, w = _cu([n, 20], dev), _weights(16, g, dev)
    args = dict(prior=torch.tensor([prior, 30], dtype=torch.int32,
                                   device=dev),
                k_pool=c.kp, v_pool=c.vp, table=c.table)
    a, la = _prefill(tm, q, None, None, cu, w, **args)
    b, lb = _prefill(tm, q, None, None, cu, w, **args)
    assert torch.equal(a, b) and torch.equal(la, lb)
    for most in (n + prior, 1):           # (a bound that is too low: one launch)
        _prefill(tm, q, None, None, cu, w, call=dict(max_context=most), **args)


def test_prefill_strides_and_outputs(tm, dev):
    """Tensors inside wider ones, outputs given, rows past the last run left
    as they were, no LSE."""
    g = _gen(12)
    lens = [70, 1, 130]
    T, n = 230, 201
    q = _rand((T, 3, 16, 136), g, dev)[:, 1, :, 8:]
    kv = _rand((T, 2, 6, D), g, dev)
    k, v = kv[:, 0, 1:5], kv[:, 1, 2:]
    cu, w = _cu(lens, dev), _weights(16, g, dev)
    ref, rl = _prefill(tm, q, k, v, cu, w)
    big = torch.full((T, 9, 264), 7.0, dtype=BF, device=dev)
    out, lse = big[:, :8, :256], torch.full((16, T), 7.0, device=dev)
    _prefill(tm, q, k, v, cu, w, call=dict(out=out, lse=lse))
    assert torch.equal(out[:n], ref[:n]) and torch.equal(lse[:, :n],
                                                         rl[:, :n])
    assert (big[n:] == 7).all() and (big[:, 8] == 7).all()
    assert (big[..., 256:] == 7).all() and (lse[:, n:] == 7).all()
    o, none = _prefill(tm, q, k, v, cu, w, call=dict(return_lse=False))
    assert none is None and torch.equal(o[:n], ref[:n])


def test_prefill_reject(tm, dev):
    g = _gen(13)
    q = _rand((40, 8, D), g, dev)
    k = _rand((40, 2, D), g, dev)
    w = _weights(8, g, dev)
    for flag in (0, 1, 0):
        r = torch.tensor([flag], dtype=torch.int32, device=dev)
        out, lse = tm.prefill_diff_varlen(q, k, k, _cu([8, 32], dev),
                                          w["lam"], 0.1, reject=r)
        assert torch.isnan(out).all() == bool(flag)
        assert torch.isnan(lse).all() == bool(flag)
        assert torch.isfinite(out).all() != bool(flag)


@pytest.mark.parametrize("std", [0.0, 30.0])
def test_prefill_flat_and_peaked(tm, dev, std):
    g = _gen(14)
    T = 700
    _prefill(tm, _rand((T, 8, D), g, dev, std), _rand((T, 2, D), g, dev),
             _rand((T, 2, D), g, dev), _cu([T], dev), _weights(8, g, dev),
             D ** -0.5)


def test_prefill_far_pages(tm, dev):
    """Pages past 4 GiB of the pools."""
    g = _gen(22)
    P, hkv, n = 300000, 4, 100
    kp = torch.zeros((P, PAGE, hkv, D), dtype=BF, device=dev)
    vp = torch.zeros_like(kp)
    c = Cache([n, n], hkv, g, dev)
    far = torch.tensor([[P - 1 - i for i in range(7)],
                        [P // 2 + i for i in range(7)]], device=dev)
    kp[far], vp[far] = c.kp[c.table.long()], c.vp[c.table.long()]
    _prefill(tm, _rand((130, 16, D), g, dev), None, None, _cu([90, 40], dev),
             _weights(16, g, dev), k_pool=kp, v_pool=vp, table=far.int(),
             prior=torch.tensor([10, 60], dtype=torch.int32, device=dev))


@pytest.mark.parametrize("split", [0, 1])
def test_prefill_pages_without_an_entry(tm, dev, split):
    """Entries outside the pool, and positions past the row's width, read as
    zero rows (of runs long enough to be split, and of short ones)."""
    g = _gen(23)
    n, prior = (40, 3000) if split else (40, 70)
    c = Cache([n + prior], 2, g, dev)
    w = _weights(4, g, dev)
    kp = torch.cat([c.kp, torch.zeros_like(c.kp[:1])])
    vp = torch.cat([c.vp, torch.zeros_like(c.vp[:1])])
    P = c.kp.shape[0]
    gone = [1, 4, (n + prior - 1) // PAGE]
    zero = c.table.clone()
    zero[0, gone] = P
    c.table[0, gone[0]], c.table[0, gone[1]] = -1, P
    q = _rand((n, 4, D), g, dev)
    cu = _cu([n], dev)
    pr = torch.tensor([prior], dtype=torch.int32, device=dev)
    ref = diff_ref.prefill(q, None, None, cu.tolist(), w["lam"], 0.1,
                           prior=pr, k_pool=kp, v_pool=vp, table=zero,
                           **{x: y for x, y in w.items() if x != "lam"})
    out, lse = tm.prefill_diff_varlen(
        q, None, None, cu, w["lam"], 0.1, max_seqlen=n, prior_lens=pr,
        k_pool=c.kp, v_pool=c.vp,
        block_table=c.table[:, :gone[2]].contiguous(),
        **{x: y for x, y in _user(w).items() if x != "lam"})
    diff_ref.check(out, lse, ref)


def test_prefill_without_tokens(tm, dev):
    e = torch.empty((0, 4, D), dtype=BF, device=dev)
    lam = torch.ones(2, device=dev)
    for cu in ([0], [0, 0, 0]):
        out, lse = tm.prefill_diff_varlen(
            e, e[:, :2], e[:, :2],
            torch.tensor(cu, dtype=torch.int32, device=dev), lam, 0.1)
        assert out.shape == (0, 2, 256) and lse.shape == (4, 0)


def test_prefill_many_runs(tm, dev):
    g = _gen(15)
    lens = torch.randint(0, 70, (150,), generator=g).tolist()
    T = sum(lens)
    _prefill(tm, _rand((T, 4, D), g, dev), _rand((T, 2, D), g, dev),
             _rand((T, 2, D), g, dev), _cu(lens, dev), _weights(4, g, dev))


def test_prefill_graph(tm, dev):
    """Replays follow the lengths and contexts; two graphs at once keep
    their own scratch."""
    g = _gen(16)
    c = Cache([5000, 700], 4, g, dev)
    q = _rand((300, 16, D), g, dev)
    w = _weights(16, g, dev)
    kw = {k: v for k, v in _user(w).items() if k != "lam"}
    cu = _cu([100, 200], dev)
    prior = torch.tensor([4900, 500], dtype=torch.int32, device=dev)

    def call():
        return tm.prefill_diff_varlen(
            q, None, None, cu, w["lam"], 0.1, max_seqlen=300,
            prior_lens=prior, k_pool=c.kp, v_pool=c.vp, block_table=c.table,
            **kw)
    call()
    graphs = []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            graphs.append((gr, call()))
    for lens, pr in (([100, 200], [4900, 500]), ([300, 0], [0, 0]),
                     ([1, 299], [4999, 401]), ([100, 200], [4900, 500])):
        cu.copy_(_cu(lens, dev))
        prior.copy_(torch.tensor(pr, dtype=torch.int32))
        want = call()
        for gr, _ in graphs:
            gr.replay()
        torch.cuda.synchronize()
        for _, res in graphs:
            assert torch.equal(res[0], want[0])
            assert torch.equal(res[1], want[1])


@pytest.mark.parametrize("window", [0, 40])
def test_serving_steps_together(tm, dev, window):
    """Two requests are prefilled in chunks and decoded, a third joins, one
    finishes and its pages serve another: plan, KV write, attention, release,
    each step against whole-prompt attention in float64."""
    g = _gen(17)
    hq, hkv, S, W = 16, 4, 4, 12
    w = _weights(hq, g, dev)
    kw = {k: v for k, v in _user(w).items() if k != "lam"}
    kp = torch.full((40, PAGE, hkv, D), NAN, dtype=BF, device=dev)
    vp = torch.full_like(kp, NAN)
    pt = torch.full((S, W), -1, dtype=torch.int32, device=dev)
    free = torch.randperm(30, generator=g).int().to(dev)
    count = torch.tensor([30], dtype=torch.int32, device=dev)
    seen = {}

    def step(slots, new):
        nonlocal count
        B, T = len(slots), sum(new)
        ctx = torch.tensor([len(seen.get(s, ([],))[0]) for s in slots],
                           dtype=torch.int32, device=dev)
        p = tm.plan_pages(pt, torch.tensor(slots, device=dev), ctx,
                          torch.tensor(new, dtype=torch.int32, device=dev),
                          free, count, T)
        count = p.free_count
        q = _rand((T, hq, D), g, dev)
        k, v = _rand((T, hkv, D), g, dev), _rand((T, hkv, D), g, dev)
        tm.kv_write_slots(k, v, p.slot_mapping, kp, vp)
        if T == B:
            out, lse = tm.decode_diff_paged(q, kp, vp, p.block_table,
                                            p.seq_lens, w["lam"], 0.1,
                                            window=window, **kw)
            lse = lse.T
        else:
            out, lse = tm.prefill_diff_varlen(
                q, None, None, p.cu_seqlens, w["lam"], 0.1, window=window,
                max_seqlen=max(new), prior_lens=ctx, k_pool=kp, v_pool=vp,
                block_table=p.block_table, reject=p.reject, **kw)
        assert p.reject.item() == 0
        t = 0
        for s, n in zip(slots, new):
            old = seen.get(s, (k[:0], v[:0]))
            K = torch.cat([old[0], k[t:t + n]])
            V = torch.cat([old[1], v[t:t + n]])
            pos = torch.arange(K.shape[0], device=dev)
            ref = diff_ref.attend(
                q[t:t + n], K, V, pos[K.shape[0] - n:], pos, w["lam"], 0.1,
                window=window,
                **{x: y for x, y in w.items() if x != "lam"})
            diff_ref.check(out[t:t + n], lse[:, t:t + n], ref, f"{s}")
            assert p.positions[t:t + n].tolist() == \
                pos[K.shape[0] - n:].tolist()
            seen[s] = (K, V)
            t += n
    step([2, 0], [50, 17])
    step([2, 0], [33, 1])
    for _ in range(3):
        step([0, 2], [1, 1])
    step([0, 1, 2], [1, 90, 1])
    n = len(seen.pop(2)[0])
    count, bad = tm.release_pages(
        pt, torch.tensor([2], device=dev),
        torch.tensor([n], dtype=torch.int32, device=dev), free, count)
    assert bad.item() == 0
    step([3, 1], [150, 1])
    step([3, 0, 1], [1, 1, 1])


@pytest.mark.parametrize("bad", [NAN, float("inf"), -float("inf")])
@pytest.mark.parametrize("hq,hkv", [(16, 4), (4, 4)])
def test_prefill_keys_that_are_no_numbers(tm, dev, hq, hkv, bad):
    """A key that a query does not see, by causality or by the window, may
    hold anything."""
    g = _gen(19)
    n, at, window = 150, 40, 32
    w = _weights(hq, g, dev)
    kw = {k: v for k, v in w.items() if k != "lam"}
    q = _rand((n, hq, D), g, dev)
    k, v = _rand((n, hkv, D), g, dev), _rand((n, hkv, D), g, dev)
    k[at] = bad
    cu = torch.tensor([0, n], dtype=torch.int32, device=dev)
    pos = torch.arange(n, device=dev)
    good = k.clone()
    good[at] = 0
    for win in (0, window):
        out, lse = tm.prefill_diff_varlen(
            q, k, v, cu, w["lam"], 0.1, window=win, max_seqlen=n,
            **{x: y for x, y in _user(w).items() if x != "lam"})
        for rows in [slice(0, at)] + ([slice(at + win, n)] if win else []):
            ref = diff_ref.attend(q[rows], good, v, pos[rows], pos, w["lam"],
                                  0.1, window=win, **kw)
            diff_ref.check(out[rows], lse[:, rows], ref, f"{win} {rows}")


def test_decode_step_in_a_graph(tm, dev):
    """Plan, KV write and attention of a decode step as one graph: each replay
    goes on from where the last one was, takes pages as the requests reach
    them, and from the first step without a page on changes nothing."""
    g = _gen(20)
    hq, hkv, S, W, lens = 16, 4, 5, 8, [14, 16, 45]
    B = len(lens) + 1                       # the last row is padding
    w = _weights(hq, g, dev)
    kw = {k: v for k, v in _user(w).items() if k != "lam"}
    kp = torch.full((24, PAGE, hkv, D), NAN, dtype=BF, device=dev)
    vp = torch.full_like(kp, NAN)
    pt = torch.full((S, W), -1, dtype=torch.int32, device=dev)
    free = torch.randperm(11, generator=g).int().to(dev)
    count = torch.tensor([11], dtype=torch.int32, device=dev)
    slots = torch.tensor([4, 0, 2, -1], device=dev)
    T = sum(lens)
    K, V = _rand((T, hkv, D), g, dev), _rand((T, hkv, D), g, dev)
    p = tm.plan_pages(pt, slots, torch.zeros(B, dtype=torch.int32, device=dev),
                      torch.tensor(lens + [0], dtype=torch.int32, device=dev),
                      free, count, T)
    tm.kv_write_slots(K, V, p.slot_mapping, kp, vp)
    seen = [(a, b) for a, b in zip(K.split(lens), V.split(lens))]
    count.copy_(p.free_count)
    ctx, one = p.seq_lens.clone(), torch.ones(B, dtype=torch.int32, device=dev)
    q = torch.zeros((B, hq, D), dtype=BF, device=dev)
    k = torch.zeros((B, hkv, D), dtype=BF, device=dev)
    v = torch.zeros_like(k)
    plan = tm.plan_pages(pt, slots, ctx, torch.zeros_like(one), free, count, B)
    plan = plan._replace(seq_lens=ctx, free_count=count)

    def step():
        tm.plan_pages(pt, slots, ctx, one, free, count, B, out=plan)
        tm.kv_write_slots(k, v, plan.slot_mapping, kp, vp)
        return tm.decode_diff_paged(q, kp, vp, plan.block_table,
                                    plan.seq_lens, w["lam"], 0.1, **kw)

    def refill():
        for x in (q, k, v):
            x.copy_(_rand(x.shape, g, dev))

    def check(res, what):
        assert plan.reject.item() == 0 and count.item() >= 0
        for i in range(B - 1):
            seen[i] = tuple(torch.cat([o, x[i:i + 1]])
                            for o, x in zip(seen[i], (k, v)))
            n = seen[i][0].shape[0]
            assert ctx[i].item() == n
            pos = torch.arange(n, device=dev)
            ref = diff_ref.attend(
                q[i:i + 1], *seen[i], pos[n - 1:], pos, w["lam"], 0.1,
                **{x: y for x, y in w.items() if x != "lam"})
            diff_ref.check(res[0][i:i + 1], res[1][i:i + 1].T, ref,
                           f"{what} {i}")
        assert (res[0][B - 1] == 0).all()
        assert (res[1][B - 1] == -float("inf")).all()

    refill()
    check(step(), "eager")                  # (and the warm-up)
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        res = step()
    # five of the eleven pages are taken at first, the last one at step 20; the
    # second request's 49th token, at step 33, finds none
    while True:
        need = sum(s[0].shape[0] % PAGE == 0 for s in seen)
        refill()
        before = count.item(), ctx.tolist(), pt.tolist()
        have = kp.clone()
        gr.replay()
        torch.cuda.synchronize()
        if need > before[0]:
            break
        check(res, f"replay at {ctx.tolist()}")
    assert before[0] == 0 and len(seen[1][0]) == 48
    for _ in range(2):                      # refused: nothing has changed
        assert plan.reject.item() == 1
        assert (count.item(), ctx.tolist(), pt.tolist()) == before
        assert torch.equal(kp.isnan(), have.isnan())
        assert torch.equal(kp.nan_to_num(), have.nan_to_num())
        assert (plan.block_table == -1).all() and (res[0] == 0).all()
        gr.replay()
        torch.cuda.synchronize()


@pytest.mark.parametrize("B,hq,hkv,wgs,norm", [
    (128, 32, 4, 0, True), (192, 8, 4, 0, True), (193, 8, 2, 0, False),
    (700, 8, 4, 0, True), (64, 64, 16, 0, True), (63, 64, 16, 0, True),
    (97, 64, 16, 0, False), (50, 16, 4, 7, True), (50, 16, 4, 50, True),
    (33, 16, 8, 11, True)])
def test_decode_short_requests(tm, dev, B, hq, hkv, wgs, norm):
    """Batches of short requests: whole ones per range, several per range, and
    what a range's neighbours share."""
    g = _gen(22)
    ends = torch.randint(0, 200, (B,), generator=g).tolist()
    ends[B // 2] = 0
    ends[-1] = 1
    c = Cache(ends, hkv, g, dev)
    _decode(tm, c, _rand((B, hq, D), g, dev), 0.1,
            _weights(hq, g, dev, norm=norm), num_workgroups=wgs)
    even = [199] * B                        # no request longer than another
    c = Cache(even, hkv, g, dev)
    _decode(tm, c, _rand((B, hq, D), g, dev), 0.1,
            _weights(hq, g, dev, norm=norm), num_workgroups=wgs, window=150)


@pytest.mark.parametrize("hq,hkv,window", [
    (32, 4, 0), (32, 4, 40), (16, 8, 0), (12, 4, 70), (6, 2, 0), (24, 8, 33)])
@pytest.mark.parametrize("paged", [False, True])
def test_prefill_large_launches(tm, dev, hq, hkv, window, paged):
    """More work-groups than the chip holds at once: the same edges as the
    smaller launches."""
    g = _gen(23)
    lens = (RUNS[:-2] + [1, 95, 96, 97, 0, 17]) * 4 + [160]
    S = len(lens)
    q = _rand((sum(lens), hq, D), g, dev)
    w = _weights(hq, g, dev, norm=window != 40)
    call = dict(max_seqlen=300)
    if not paged:
        k, v = (_rand((sum(lens), hkv, D), g, dev) for _ in "kv")
        _prefill(tm, q, k, v, _cu(lens, dev), w, window=window, call=call)
        return
    prior = torch.randint(0, 60, (S,), generator=g).tolist()
    first = [max(0, p - window + 1) if window else 0 for p in prior]
    c = Cache([a + b for a, b in zip(lens, prior)], hkv, g, dev, first=first)
    _prefill(tm, q, None, None, _cu(lens, dev), w,
             prior=torch.tensor(prior, dtype=torch.int32, device=dev),
             k_pool=c.kp, v_pool=c.vp, table=c.table, window=window,
             call=call)


@pytest.mark.parametrize("n,prior,hq,hkv,window", [
    (16, 1000, 16, 4, 0), (16, 1000, 12, 4, 900), (40, 1500, 24, 8, 0),
    (1, 3000, 8, 2, 0), (70, 1100, 4, 4, 0), (300, 1000, 32, 4, 0),
    (500, 6000, 32, 8, 0)])
def test_prefill_pieces_of_either_size(tm, dev, n, prior, hq, hkv, window):
    """Split launches with work-groups of four and of eight waves, beside runs
    that are not worth a split or have no tokens."""
    g = _gen(n + hq)
    lens, before = [n, 0, n // 3, 1], [prior, 9, 33, prior // 2]
    first = [max(0, p - window + 1) if window else 0 for p in before]
    c = Cache([a + b for a, b in zip(lens, before)], hkv, g, dev, first=first)
    q = _rand((sum(lens), hq, D), g, dev)
    pr = torch.tensor(before, dtype=torch.int32, device=dev)
    for norm in (True, False):
        _prefill(tm, q, None, None, _cu(lens, dev),
                 _weights(hq, g, dev, norm=norm), prior=pr, k_pool=c.kp,
                 v_pool=c.vp, table=c.table, window=window)


@pytest.mark.parametrize("n,hq,hkv", [(1100, 4, 2), (1500, 8, 2), (2050, 4, 4)])
def test_prefill_packed_pieces(tm, dev, n, hq, hkv):
    g = _gen(n)
    lens = [n, 3]
    T = sum(lens)
    _prefill(tm, _rand((T, hq, D), g, dev), _rand((T, hkv, D), g, dev),
             _rand((T, hkv, D), g, dev), _cu(lens, dev), _weights(hq, g, dev))


@pytest.mark.parametrize("hq,hkv,window", [(32, 4, 0), (12, 4, 50), (8, 8, 0)])
def test_prefill_many_short_runs(tm, dev, hq, hkv, window):
    """More work-groups than the chip holds, of few keys each."""
    g = _gen(24)
    lens = torch.randint(0, 230, (90,), generator=g).tolist() + [230, 0]
    T = sum(lens)
    _prefill(tm, _rand((T, hq, D), g, dev), _rand((T, hkv, D), g, dev),
             _rand((T, hkv, D), g, dev), _cu(lens, dev), _weights(hq, g, dev),
             window=window)


@pytest.mark.parametrize("bound", [400, 200])
def test_prefill_large_strides_outputs_and_reject(tm, dev, bound):
    """As the smaller launches: tensors inside wider ones, outputs given, rows
    past the last run left as they were, a refused step."""
    g = _gen(25)
    lens = [70, 1, 130, 0, 33] * 16
    n = sum(lens)
    T = n + 29
    q = _rand((T, 3, 16, 136), g, dev)[:, 1, :, 8:]
    kv = _rand((T, 2, 6, D), g, dev)
    k, v = kv[:, 0, 1:5], kv[:, 1, 2:]
    cu, w = _cu(lens, dev), _weights(16, g, dev)
    big = torch.full((T, 9, 264), 7.0, dtype=BF, device=dev)
    out, lse = big[:, :8, :256], torch.full((16, T), 7.0, device=dev)
    _prefill(tm, q, k, v, cu, w, call=dict(out=out, lse=lse,
                                           max_seqlen=bound))
    assert (big[n:] == 7).all() and (big[:, 8] == 7).all()
    assert (big[..., 256:] == 7).all() and (lse[:, n:] == 7).all()
    for flag in (0, 1, 0):
        r = torch.tensor([flag], dtype=torch.int32, device=dev)
        o, l = tm.prefill_diff_varlen(
            q[:n], k[:n], v[:n], cu, w["lam"], 0.1, max_seqlen=bound,
            reject=r, **{x: y for x, y in _user(w).items() if x != "lam"})
        assert torch.isnan(o).all() == bool(flag)
        assert torch.isnan(l).all() == bool(flag)
        assert flag or (torch.equal(o, out[:n]) and torch.equal(l, lse[:, :n]))
