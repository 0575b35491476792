"""plan_pages and release_pages at the batch sizes between which their sums
change shape. A plan of up to 1024 requests with outputs of its own is one
launch whose work-groups of 256 threads each sum all requests, 256 a pass; a
larger one sums 1024 a pass."""
import random

import pytest
import torch

from oracle import diff_ref

pytestmark = pytest.mark.gpu
BATCHES = [255, 256, 257, 512, 600, 1023, 1024, 1025, 2049]


def _dev(x, dev, dtype=torch.int32):
    return torch.tensor(x, dtype=dtype, device=dev)


def _step(B, W, rng):
    """(page table, slots, contexts, new tokens, free pages), padding among
    them."""
    S = B + 3
    table = [[rng.randrange(10 ** 6) for _ in range(W)] for _ in range(S)]
    slots = rng.sample(range(S), B)
    ctx = [rng.randint(0, 16 * W - 20) for _ in range(B)]
    new = [rng.choice([0, 1, 1, 20]) for _ in range(B)]
    for i in range(0, B, 29):
        slots[i] = -1 - i
    return table, slots, ctx, new, [10 ** 6 + i for i in range(2 * B + 5)]


def _plan(tm, dev, table, slots, ctx, new, free, count, T):
    t = _dev(table, dev)
    p = tm.plan_pages(t, _dev(slots, dev, torch.int64), _dev(ctx, dev),
                      _dev(new, dev), _dev(free, dev), _dev([count], dev), T)
    want = diff_ref.plan(table, slots, ctx, new, free, count, T)
    for got, w in zip((t,) + tuple(p), want):
        assert got.tolist() == ([w] if isinstance(w, int) else w)
    return p.reject.item()


@pytest.mark.parametrize("B", BATCHES)
def test_plan_batches(tm, dev, B):
    rng = random.Random(B)
    table, slots, ctx, new, free = _step(B, 6, rng)
    T = sum(n for n, s in zip(new, slots) if s >= 0)
    assert _plan(tm, dev, table, slots, ctx, new, free, len(free), T) == 0
    assert _plan(tm, dev, table, slots, ctx, new, free, len(free), T + 99) == 0
    # one token, one page too many, each only in the sum of all passes
    assert _plan(tm, dev, table, slots, ctx, new, free, len(free), T - 1) == 1
    need = sum((c + n + 15) // 16 - (c + 15) // 16
               for c, n, s in zip(ctx, new, slots) if s >= 0)
    assert _plan(tm, dev, table, slots, ctx, new, free, need, T) == 0
    assert _plan(tm, dev, table, slots, ctx, new, free, need - 1, T) == 1
    # the same row in the first and in the last pass, a bad one in the last
    for i, s in ((B - 1, slots[1]), (B - 1, len(table)), (B // 2, slots[2])):
        twice = list(slots)
        twice[i] = s
        assert _plan(tm, dev, table, twice, ctx, new, free, len(free),
                     T + 99) == 1


def _release(tm, dev, table, slots, lens, free, count):
    want = diff_ref.release(table, slots, lens, free, count)
    for over in (False, True):
        f, n = _dev(free, dev), _dev([count], dev)
        got = tm.release_pages(
            _dev(table, dev), _dev(slots, dev, torch.int64), _dev(lens, dev),
            f, n, out=(n, torch.empty_like(n)) if over else None)
        assert f.tolist() == want[0]
        assert [x.item() for x in got] == list(want[1:])
    return want[2]


@pytest.mark.parametrize("B,W", [(b, 6) for b in BATCHES] +
                         [(300, 40), (1024, 9), (1500, 16)])
def test_release_batches(tm, dev, B, W):
    rng = random.Random(B + W)
    table, slots, lens, _, _ = _step(B, W, rng)
    total = sum((n + 15) // 16 for n, s in zip(lens, slots) if s >= 0)
    free = [10 ** 6 + i for i in range(total + 40)]
    for count, bad in ((0, 0), (40, 0), (41, 1), (7, 0)):
        assert _release(tm, dev, table, slots, lens, free, count) == bad
    for i, s in ((B - 1, slots[1]), (B - 1, len(table)), (B // 2, slots[2])):
        twice = list(slots)
        twice[i] = s
        assert _release(tm, dev, table, twice, lens, free, 0) == 1


@pytest.mark.parametrize("B", [8192, 3])
def test_largest_table(tm, dev, B):
    """As many requests and table rows as one call takes, and a small step in
    a table of as many rows."""
    rng = random.Random(B)
    S, W = 262144, 2
    table = [[7 * i, 7 * i + 1] for i in range(S)]
    slots = rng.sample(range(S), B)
    slots[-1] = S - 1 if S - 1 not in slots else slots[-1]
    ctx = [rng.randint(0, 31) for _ in range(B)]
    new = [rng.randint(0, 32 - c) for c in ctx]
    free = [10 ** 7 + i for i in range(2 * B + 9)]
    assert _plan(tm, dev, table, slots, ctx, new, free, len(free) - 5,
                 sum(new)) == 0
    total = sum((c + 15) // 16 for c in ctx)
    assert _release(tm, dev, table, slots, ctx, free, len(free) - total) == 0
    assert _release(tm, dev, table, slots, ctx, free,
                    len(free) - total + 1) == 1
    slots[0] = slots[-1]
    assert _plan(tm, dev, table, slots, ctx, new, free, len(free),
                 sum(new)) == 1
