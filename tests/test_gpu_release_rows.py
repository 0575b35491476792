"""Releases of rows that do not name a page everywhere (a window's pages that
were handed back before): what is pushed is pages, in order, and nothing
else."""
import random

import pytest
import torch

from oracle import diff_ref

pytestmark = pytest.mark.gpu


def _dev(x, dev, dtype=torch.int32):
    return torch.tensor(x, dtype=dtype, device=dev)


def _release(tm, dev, table, slots, lens, free, count):
    """One release, with a height of its own and in place, checked whole."""
    want = diff_ref.release(table, slots, lens, free, count)
    for over in (False, True):
        f, n = _dev(free, dev), _dev([count], dev)
        t = _dev(table, dev)
        got = tm.release_pages(
            t, _dev(slots, dev, torch.int64), _dev(lens, dev), f, n,
            out=(n, torch.empty_like(n)) if over else None)
        assert f.tolist() == want[0]
        assert [x.item() for x in got] == list(want[1:])
        assert t.tolist() == table
    return want


@pytest.mark.parametrize("B,W", [(1, 1), (1, 40), (3, 10), (40, 200),
                                 (64, 33), (70, 300), (2, 5000), (1, 9001),
                                 (1024, 8), (1024, 9), (1100, 20)])
def test_release_rows_with_gaps(tm, dev, B, W):
    rng = random.Random(B * 7 + W)
    S = B + 2
    table = [[rng.randrange(10 ** 6) for _ in range(W)] for _ in range(S)]
    lens = [rng.choice([0, 1, 16 * W, rng.randint(0, 16 * W)])
            for _ in range(B)]
    slots = rng.sample(range(S), B)
    for i in range(3, B, 11):
        slots[i] = -1
    for i, s in enumerate(slots):
        if s < 0:
            continue
        row, kind = table[s], rng.randrange(5)
        if kind == 0:                       # a window's: the first are gone
            for j in range(rng.randint(0, W)):
                row[j] = -1
        elif kind == 1:                     # here and there
            for j in range(W):
                if rng.random() < 0.3:
                    row[j] = -1 - rng.randrange(9)
        elif kind == 2:                     # every one
            table[s] = [-1] * W
        elif kind == 3:                     # one
            row[rng.randrange(W)] = -1
    free = [10 ** 6 + i for i in range(B * W + 9)]
    for count in (0, 9):
        got = _release(tm, dev, table, slots, lens, free, count)
        assert got[2] == 0 and all(x >= 0 for x in got[0][:got[1]])
    pushed = got[1] - 9
    # a stack that holds the pages, though not the entries; one too small
    if pushed:
        short = free[:pushed + 4]
        assert _release(tm, dev, table, slots, lens, short, 4)[2] == 0
        assert _release(tm, dev, table, slots, lens, short, 5)[2] == 1


def test_windowed_request_comes_back(tm, dev):
    """A request that gave its early pages back goes whole, and the next plan
    hands out pages only."""
    table = torch.full((2, 8), -1, dtype=torch.int32, device=dev)
    free = torch.arange(8, dtype=torch.int32, device=dev)
    slot = torch.tensor([1], device=dev)
    p = tm.plan_pages(table, slot, _dev([0], dev), _dev([100], dev), free,
                      _dev([8], dev), 100)
    assert p.free_count.item() == 1
    # the first three pages leave the window
    n, bad = tm.release_pages(table, slot, _dev([48], dev), free, p.free_count)
    table[1, :3] = -1
    assert (n.item(), bad.item()) == (4, 0)
    n, bad = tm.release_pages(table, slot, _dev([100], dev), free, n)
    assert (n.item(), bad.item()) == (8, 0)
    assert sorted(free.tolist()) == list(range(8))
    p = tm.plan_pages(table, _dev([0], dev, torch.int64), _dev([0], dev),
                      _dev([128], dev), free, n, 128)
    assert p.reject.item() == 0
    assert sorted(p.block_table[0].tolist()) == list(range(8))
    assert (p.slot_mapping >= 0).all()


def test_release_in_a_graph(tm, dev):
    """In place, replayed with eager work in between: heights go on."""
    rng = random.Random(3)
    B, W, F = 9, 700, 15000
    table = [[rng.choice([-1, rng.randrange(10 ** 6)]) for _ in range(W)]
             for _ in range(B)]
    slots = rng.sample(range(B), B)
    lens = [rng.randint(0, 16 * W) for _ in range(B)]
    free, height = [0] * F, 5
    t, s = _dev(table, dev), _dev(slots, dev, torch.int64)
    l, f, n = _dev(lens, dev), _dev(free, dev), _dev([5], dev)
    bad = torch.empty_like(n)
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        tm.release_pages(t, s, l, f, n, out=(n, bad))
    refused = 0
    for _ in range(14):
        gr.replay()
        torch.zeros(100, device=dev).sum().item()
        free, height, r = diff_ref.release(table, slots, lens, free, height)
        assert (n.item(), bad.item()) == (height, r)
        assert f.tolist() == free
        refused += r
    assert 0 < refused < 14
