"""First keys, prefixes and windows at the ends of int32 (scored attention): the
same results, bit by bit, as without them."""
import pytest
import torch

from test_gpu_scored import Cache, _function, _gen, _i32, _packed, _rand

pytestmark = pytest.mark.gpu
LAST = 2 ** 31 - 1


def _same(a, b):
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("name", ["plain", "soft", "slopes", "cap slopes"])
@pytest.mark.parametrize("paged", [0, 1])
def test_masks_at_the_ends_of_int32(tm, dev, name, paged):
    g = _gen(80)
    lens, prior = [300, 1, 70, 5], [333, 0, 64, 700]
    ends = [a + b for a, b in zip(lens, prior)]
    q, k, v, cu = _packed(lens, 8, 2, g, dev)
    kw = dict(_function(name, 8, g, dev))
    if paged:
        c = Cache(ends, 2, g, dev)
        k = v = None
        kw.update(prior_lens=_i32(prior, dev), k_pool=c.kp, v_pool=c.vp,
                  block_table=c.table)

    def call(**more):
        return tm.prefill_scored_varlen(q, k, v, cu, 0.1, **kw, **more)
    T, S = sum(lens), len(lens)
    want = call()
    for x in (0, -1, -1000, -2 ** 31 + 1, -2 ** 31):
        _same(call(first_keys=_i32([x] * T, dev)), want)
        _same(call(prefix_lens=_i32([x] * S, dev)), want)
    _same(call(window=LAST), want)
    _same(call(window=LAST - 3, first_keys=_i32([-2 ** 31] * T, dev),
               prefix_lens=_i32([-2 ** 31] * S, dev)), want)
    # a prefix of whole runs: every key ahead of its query
    want = call(prefix_lens=_i32(ends, dev))
    _same(call(prefix_lens=_i32([LAST] * S, dev)), want)
    for w in (LAST, LAST - 1, LAST - 70):
        _same(call(prefix_lens=_i32([LAST] * S, dev), window=w), want)
    # nothing visible, whatever else is
    for more in (dict(), dict(window=LAST), dict(window=1)):
        out, lse = call(first_keys=_i32([LAST] * T, dev), **more)
        assert (out == 0).all() and (lse == -float("inf")).all()


@pytest.mark.parametrize("name", ["plain", "soft", "cap slopes"])
def test_decode_masks_at_the_ends_of_int32(tm, dev, name):
    g = _gen(81)
    c = Cache([1, 16, 333, 700], 2, g, dev)
    q = _rand((4, 8, 128), g, dev)

    def call(**more):
        return tm.decode_scored_paged(q, c.kp, c.vp, c.table, c.ctx, 0.1,
                                      **_kw, **more)
    _kw = _function(name, 8, g, dev)
    want = call()
    for x in (0, -1, -2 ** 31):
        _same(call(first_keys=_i32([x] * 4, dev)), want)
    _same(call(window=LAST), want)
    out, lse = call(first_keys=_i32([LAST] * 4, dev))
    assert (out == 0).all() and (lse == -float("inf")).all()
