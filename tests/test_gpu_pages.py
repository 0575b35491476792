"""plan_pages and release_pages against the same in Python integers."""
import random

import pytest
import torch

from oracle import diff_ref

pytestmark = pytest.mark.gpu


def _state(S, W, F, rng):
    table = [[rng.randrange(10 ** 6) for _ in range(W)] for _ in range(S)]
    return table, [10 ** 6 + i for i in range(F)]


def _dev(x, dev, dtype=torch.int32):
    return torch.tensor(x, dtype=dtype, device=dev)


def _plan(tm, dev, table, slots, ctx, new, free, count, T, width=None):
    """One call, checked whole; returns (page table, plan)."""
    t = _dev(table, dev)
    p = tm.plan_pages(t, _dev(slots, dev, torch.int64), _dev(ctx, dev),
                      _dev(new, dev), _dev(free, dev), _dev([count], dev), T,
                      width=width)
    want = diff_ref.plan(table, slots, ctx, new, free, count, T, width)
    got = (t, p.block_table, p.seq_lens, p.cu_seqlens, p.slot_mapping,
           p.positions, p.free_count, p.reject)
    names = ("page table", "block table", "seq_lens", "cu_seqlens",
             "slot_mapping", "positions", "free_count", "reject")
    for n, g, w in zip(names, got, want):
        w = [w] if isinstance(w, int) else w
        assert g.tolist() == w, (n, slots, ctx, new, T, width)
    return t, p


# sizes on both sides of each launch shape: requests over 64 (a wave), 1024 (a
# pass of the sums), table widths that 4 divides or not
SIZES = [
    (1, 1, 1), (1, 3, 7), (3, 8, 12), (4, 64, 64), (64, 33, 33), (65, 16, 20),
    (130, 130, 130), (40, 512, 512), (1025, 5, 5), (1030, 40, 40),
]


@pytest.mark.parametrize("B,width,W", SIZES)
@pytest.mark.parametrize("kind", ["decode", "prompt", "mixed"])
def test_plan(tm, dev, B, width, W, kind):
    rng = random.Random(B * 1000 + width)
    table, free = _state(B + 3, W, B * W + 5, rng)
    slots = rng.sample(range(B + 3), B)
    most = 16 * min(width, W)
    ctx, new = [], []
    for i in range(B):
        n = {"decode": 1, "prompt": rng.randint(1, min(most, 700)),
             "mixed": rng.choice([0, 1, 1, min(most, 33)])}[kind]
        c = 0 if kind == "prompt" else rng.randint(0, most - n)
        if rng.random() < 0.2:
            c = c // 16 * 16               # a page just filled
        if rng.random() < 0.1:
            slots[i] = -1 - rng.randrange(3)
        ctx.append(c)
        new.append(n)
    T = sum(n for n, s in zip(new, slots) if s >= 0)
    count = len(free) - rng.randrange(3)
    _plan(tm, dev, table, slots, ctx, new, free, count, T, width)
    _plan(tm, dev, table, slots, ctx, new, free, count, T + 131, width)


def test_plan_long_requests(tm, dev):
    """A step whose tokens and table fill many work-groups."""
    rng = random.Random(5)
    table, free = _state(9, 4100, 9000, rng)
    slots = [7, 2, 5, 0]
    ctx = [65000, 17, 16, 0]
    new = [600, 30001, 1, 20000]
    _plan(tm, dev, table, slots, ctx, new, free, 8000, sum(new) + 7)
    _plan(tm, dev, table, slots, ctx, new, free, 100, sum(new))   # too few


def test_plan_without_requests_or_tokens(tm, dev):
    rng = random.Random(6)
    table, free = _state(3, 4, 8, rng)
    _plan(tm, dev, table, [], [], [], free, 8, 0)
    _plan(tm, dev, table, [], [], [], free, 8, 5)
    _plan(tm, dev, table, [1, -1], [33, 7], [0, 3], free, 8, 0)
    _plan(tm, dev, table, [1, 0], [33, 0], [0, 0], free, 0, 4)


@pytest.mark.parametrize("B,T", [(6, 40), (6, 6000)])
def test_plan_rejects_whole_steps(tm, dev, B, T):
    """One bad request refuses the step: nothing is taken, every output is
    the empty step's."""
    rng = random.Random(7)
    table, free = _state(8, 6, 40, rng)
    slots, ctx, new = [3, 1, 7, 0, -1, 5], [5, 0, 16, 90, 4, 31], [1] * 6
    _plan(tm, dev, table, slots, ctx, new, free, 40, T)
    for i, (s, c, n) in enumerate([(8, 5, 1), (1 << 40, 5, 1), (1, 5, 1),
                                   (2, -1, 1), (2, 5, -1), (2, 96, 1),
                                   (2, 2 ** 31 - 1, 2 ** 31 - 1),
                                   (2, 0, T + 1)]):
        bad = (slots[:2] + [s] + slots[3:], ctx[:2] + [c] + ctx[3:],
               new[:2] + [n] + new[3:])
        _, p = _plan(tm, dev, table, *bad, free, 40, T)
        assert p.reject.item() == 1, i
    _, p = _plan(tm, dev, table, slots, ctx, new, free, 1, T)
    assert p.reject.item() == 1          # two pages are needed
    for count in (-1, 41):
        _, p = _plan(tm, dev, table, slots, ctx, new, free, count, T)
        assert p.reject.item() == 1
    _, p = _plan(tm, dev, table, slots, ctx, new, free, 40, T, width=5)
    assert p.reject.item() == 1          # 91 tokens do not fit 5 pages


def test_plan_missing_pages(tm, dev):
    """Rows that name no page give no slot (and are not dereferenced)."""
    table = [[-1, 4, -1], [2, -5, 9]]
    _plan(tm, dev, table, [1, 0], [14, 30], [6, 2], [7, 8], 2, 10)


@pytest.mark.parametrize("B,W", [(1, 1), (3, 10), (64, 33), (70, 300),
                                 (1100, 20)])
def test_release(tm, dev, B, W):
    rng = random.Random(B)
    table, free = _state(B + 2, W, (B + 2) * W, rng)
    slots = rng.sample(range(B + 2), B)
    lens = [rng.choice([0, 1, 16 * W, rng.randint(0, 16 * W)])
            for _ in range(B)]
    for i in range(0, B, 7):
        slots[i] = -1
    for count in (0, 5, len(free), -2):
        f = _dev(free, dev)
        got = tm.release_pages(_dev(table, dev), _dev(slots, dev, torch.int64),
                               _dev(lens, dev), f, _dev([count], dev))
        want = diff_ref.release(table, slots, lens, free, count)
        assert f.tolist() == want[0]
        assert [x.item() for x in got] == list(want[1:])
        f, n = _dev(free, dev), _dev([count], dev)         # and in place
        got = tm.release_pages(_dev(table, dev), _dev(slots, dev, torch.int64),
                               _dev(lens, dev), f, n,
                               out=(n, torch.empty_like(n)))
        assert f.tolist() == want[0]
        assert [x.item() for x in got] == list(want[1:])
    for i, (s, n) in ((1, (B + 2, 3)), (1, (slots[2 % B], 3)),
                      (1, (slots[1 % B], -1)),
                      (1, (slots[1 % B], 16 * W + 1))):
        if B < 3:
            continue
        s2, l2 = list(slots), list(lens)
        s2[i], l2[i] = s, n
        f = _dev(free, dev)
        got = tm.release_pages(_dev(table, dev), _dev(s2, dev, torch.int64),
                               _dev(l2, dev), f, _dev([0], dev))
        assert got[1].item() == 1 and got[0].item() == 0
        assert f.tolist() == free


def test_plan_grows_in_a_graph(tm, dev):
    """A captured decode step that plans in place (heights and lengths step on
    from replay to replay), with eager work between the replays."""
    rng = random.Random(9)
    B, W, T = 5, 8, 5
    table, free = _state(6, W, 60, rng)
    slots, ctx = [4, 0, 5, -1, 2], [15, 0, 30, 0, 47]
    new = [1, 1, 1, 1, 1]
    dt, ds = _dev(table, dev), _dev(slots, dev, torch.int64)
    dc, dn, df = _dev(ctx, dev), _dev(new, dev), _dev(free, dev)
    count = _dev([60], dev)
    tok = torch.empty((2, T), dtype=torch.int64, device=dev)
    out = tm.PagePlan(torch.empty((B, W), dtype=torch.int32, device=dev), dc,
                      torch.empty(B + 1, dtype=torch.int32, device=dev),
                      tok[0], tok[1], count,
                      torch.empty(1, dtype=torch.int32, device=dev))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        tm.plan_pages(dt, ds, dc, dn, df, count, T, out=out)
    height = 60
    for step in range(40):
        g.replay()
        torch.zeros(100, device=dev).sum().item()
        want = diff_ref.plan(table, slots, ctx, new, free, height, T)
        table, ctx, height = want[0], want[2], want[6]
        got = (dt, out.block_table, dc, out.cu_seqlens, out.slot_mapping,
               out.positions)
        assert [x.tolist() for x in got] == list(want[:6]), step
        assert count.item() == height and out.reject.item() == want[7]


@pytest.mark.parametrize("B,W,T", [(3, 8, 40), (70, 300, 5000),
                                   (1100, 4, 1200)])
def test_plan_in_place(tm, dev, B, W, T):
    """Heights and lengths that the plan writes over, both and each alone:
    the same as into buffers of their own."""
    rng = random.Random(B)
    table, free = _state(B, W, B * W, rng)
    slots = rng.sample(range(B), B)
    new = [rng.choice([0, 1, 1, 7]) for _ in range(B)]
    new[0] = T - sum(new[1:]) if sum(new[1:]) < T < 16 * W else 1
    ctx = [rng.randint(0, 16 * W - n) for n in new]
    for count in (B * W, 0):
        want = diff_ref.plan(table, slots, ctx, new, free, count, T)
        for over in ((1, 1), (0, 1), (1, 0)):
            dt, dc = _dev(table, dev), _dev(ctx, dev)
            n = _dev([count], dev)
            tok = torch.empty((2, T), dtype=torch.int64, device=dev)
            out = tm.PagePlan(
                torch.empty((B, W), dtype=torch.int32, device=dev),
                dc if over[0] else torch.empty_like(dc),
                torch.empty(B + 1, dtype=torch.int32, device=dev), tok[0],
                tok[1], n if over[1] else torch.empty_like(n),
                torch.empty(1, dtype=torch.int32, device=dev))
            got = tm.plan_pages(dt, _dev(slots, dev, torch.int64), dc,
                                _dev(new, dev), _dev(free, dev), n, T,
                                out=out)
            assert got is out
            got = [dt] + list(out)
            for g, w in zip(got, want):
                assert g.tolist() == ([w] if isinstance(w, int) else w)


def test_plan_then_release_comes_back(tm, dev):
    """Requests grow on one stream, finish, and their pages serve others."""
    S, W, F = 6, 8, 30
    dt = torch.full((S, W), -1, dtype=torch.int32, device=dev)
    free = torch.arange(F, dtype=torch.int32, device=dev)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        count = _dev([F], dev)
        s1 = _dev([0, 3, 5], dev, torch.int64)
        lens = _dev([0, 0, 0], dev)
        for new in ([100, 16, 1], [1, 1, 1], [20, 0, 15]):
            p = tm.plan_pages(dt, s1, lens, _dev(new, dev), free, count, 120)
            count, lens = p.free_count, p.seq_lens
        assert lens.tolist() == [121, 17, 17] and p.reject.item() == 0
        assert count.item() == F - 8 - 2 - 2
        n, bad = tm.release_pages(dt, s1[:2], lens[:2], free, count)
        assert (n.item(), bad.item()) == (F - 2, 0)
        p = tm.plan_pages(dt, _dev([1], dev, torch.int64), _dev([0], dev),
                          _dev([128], dev), free, n, 128)
        held = p.block_table[0].tolist() + dt[5, :2].tolist()
        left = free[:p.free_count.item()].tolist()
    assert sorted(held + left) == list(range(F))
