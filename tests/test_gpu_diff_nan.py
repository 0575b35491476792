"""Keys that are no numbers where a query sees them: the outputs of their map
and the LSE are NaN, in whole results and in joined ones, and nothing else
changes."""
import pytest
import torch

pytestmark = pytest.mark.gpu
D, PAGE = 128, 16
BF = torch.bfloat16
NAN = float("nan")


def _rand(shape, seed, dev):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(shape, generator=g).to(BF).to(dev)


def _cache(ends, hkv, dev):
    """Pools, a table of shuffled pages and the lengths."""
    pages = [-(-n // PAGE) for n in ends]
    g = torch.Generator().manual_seed(len(ends))
    perm = torch.randperm(sum(pages), generator=g).int()
    table = torch.zeros((len(ends), max(pages)), dtype=torch.int32)
    at = 0
    for i, n in enumerate(pages):
        table[i, :n] = perm[at:at + n]
        at += n
    shape = (sum(pages), PAGE, hkv, D)
    return (_rand(shape, 1, dev), _rand(shape, 2, dev), table.to(dev),
            torch.tensor(ends, dtype=torch.int32, device=dev))


@pytest.mark.parametrize("ends,hq,hkv,call", [
    ([40], 8, 4, {}),                              # whole, two waves
    ([40, 7, 60, 33] * 300, 8, 2, {}),             # whole, several per range
    ([900, 41, 2500], 16, 4, {}),                  # joined, both waves' halves
    ([5000], 32, 4, {}), ([700] * 9, 16, 2, {}),   # eight and two groups
    ([300, 200], 8, 2, dict(min_pages=1)),
    ([300, 200], 64, 16, dict(num_workgroups=3)),
])
@pytest.mark.parametrize("norm", [False, True])
def test_decode_key_that_is_no_number(tm, dev, ends, hq, hkv, call, norm):
    kp, vp, table, ctx = _cache(ends, hkv, dev)
    q = _rand((len(ends), hq, D), 3, dev)
    lam = torch.full((hq // 2,), 0.7, device=dev)
    kw = dict(call, norm_weight=torch.ones(256, device=dev) if norm else None)
    out, lse = tm.decode_diff_paged(q, kp, vp, table, ctx, lam, 0.1, **kw)
    assert torch.isfinite(out).all() and torch.isfinite(lse).all()
    rep = hq // hkv
    for b, at, head in ((0, 0, 0), (0, ends[0] - 1, 1),
                        (len(ends) - 1, ends[-1] // 2, hkv - 1)):
        bad = kp.clone()
        bad[table[b, at // PAGE].long(), at % PAGE, head] = NAN
        o, l = tm.decode_diff_paged(q, bad, vp, table, ctx, lam, 0.1, **kw)
        pairs = slice(head // 2 * rep, (head // 2 + 1) * rep)
        maps = torch.arange(hq // 2, device=dev)[pairs] * 2 + head % 2
        hit_o = torch.zeros_like(out, dtype=torch.bool)
        hit_l = torch.zeros_like(lse, dtype=torch.bool)
        hit_o[b, pairs] = True
        hit_l[b, maps] = True
        assert torch.equal(torch.isnan(o), hit_o), (b, at, head)
        assert torch.equal(torch.isnan(l), hit_l), (b, at, head)
        assert torch.equal(o[~hit_o], out[~hit_o])
        assert torch.equal(l[~hit_l], lse[~hit_l])


@pytest.mark.parametrize("lens,prior,hq,hkv", [
    ([40], None, 8, 4), ([150, 70], None, 64, 8),          # four waves, whole
    ([600] * 12, None, 32, 4),                             # eight waves, whole
    ([16], [1000], 16, 4), ([300, 5], [1000, 3], 32, 4),   # pieces of four
    ([64], [9000], 16, 4), ([500], [6000], 32, 8),         # pieces of eight
])
@pytest.mark.parametrize("norm", [False, True])
def test_prefill_key_that_is_no_number(tm, dev, lens, prior, hq, hkv, norm):
    T, S = sum(lens), len(lens)
    q = _rand((T, hq, D), 3, dev)
    cu = torch.tensor([sum(lens[:i]) for i in range(S + 1)],
                      dtype=torch.int32, device=dev)
    lam = torch.full((hq // 2,), 0.7, device=dev)
    kw = dict(norm_weight=torch.ones(256, device=dev) if norm else None,
              max_seqlen=max(lens))
    before = prior or [0] * S
    if prior is None:
        k, v = _rand((T, hkv, D), 1, dev), _rand((T, hkv, D), 2, dev)

        def run(keys):
            return tm.prefill_diff_varlen(q, keys, v, cu, lam, 0.1, **kw)
    else:
        k, vp, table, _ = _cache([a + b for a, b in zip(lens, prior)], hkv,
                                 dev)
        pr = torch.tensor(prior, dtype=torch.int32, device=dev)

        def run(keys):
            return tm.prefill_diff_varlen(
                q, None, None, cu, lam, 0.1, prior_lens=pr, k_pool=keys,
                v_pool=vp, block_table=table, **kw)
    out, lse = run(k)
    assert torch.isfinite(out).all() and torch.isfinite(lse).all()
    rep = hq // hkv
    i = S - 1
    t0 = int(cu[i])
    for at, head in ((0, 0), (before[i] + lens[i] // 2, 1),
                     (max(before[i] // 2, 1), hkv - 1)):
        bad = k.clone()
        if prior is None:
            bad[t0 + at, head] = NAN
        else:
            bad[table[i, at // PAGE].long(), at % PAGE, head] = NAN
        o, l = run(bad)
        first = t0 + max(0, at - before[i])        # the first row that sees it
        pairs = slice(head // 2 * rep, (head // 2 + 1) * rep)
        maps = torch.arange(hq // 2, device=dev)[pairs] * 2 + head % 2
        hit_o = torch.zeros_like(out, dtype=torch.bool)
        hit_l = torch.zeros_like(lse, dtype=torch.bool)
        hit_o[first:, pairs] = True
        hit_l[maps, first:] = True
        assert torch.equal(torch.isnan(o), hit_o), (at, head)
        assert torch.equal(torch.isnan(l), hit_l), (at, head)
        assert torch.equal(o[~hit_o], out[~hit_o])
        assert torch.equal(l[~hit_l], lse[~hit_l])


def test_all_keys_that_are_no_numbers(tm, dev):
    """Not a key left that is one: NaN, not the zeros of a query without
    keys."""
    kp, vp, table, ctx = _cache([50, 3000], 2, dev)
    kp.fill_(NAN)
    q, lam = _rand((2, 4, D), 3, dev), torch.ones(2, device=dev)
    out, lse = tm.decode_diff_paged(q, kp, vp, table, ctx, lam, 0.1)
    assert torch.isnan(out).all() and torch.isnan(lse).all()
    out, lse = tm.prefill_diff_varlen(
        q, None, None, torch.tensor([0, 1, 2], dtype=torch.int32, device=dev),
        lam, 0.1, max_seqlen=1, prior_lens=ctx - 1, k_pool=kp, v_pool=vp,
        block_table=table)
    assert torch.isnan(out).all() and torch.isnan(lse).all()


@pytest.mark.parametrize("n", [40, 3000])
def test_infinite_scores(tm, dev, n):
    """One dimension of one key is infinite: by the sign of the query's, the
    score is the largest (NaN) or the smallest (weight 0)."""
    kp, vp, table, ctx = _cache([n], 2, dev)
    q, lam = _rand((1, 16, D), 3, dev), torch.ones(8, device=dev)
    kp[table[0, 1].long(), 3, :, 5] = float("inf")
    up = q[0, :, 5] > 0
    both = up[0::2] | up[1::2]
    assert up.any() and not both.all()
    o, l = tm.decode_diff_paged(q, kp, vp, table, ctx, lam, 0.1)
    o2, l2 = tm.prefill_diff_varlen(
        q, None, None, torch.tensor([0, 1], dtype=torch.int32, device=dev),
        lam, 0.1, max_seqlen=1, prior_lens=ctx - 1, k_pool=kp, v_pool=vp,
        block_table=table)
    for out, lse in ((o, l[0]), (o2, l2[:, 0])):
        assert torch.equal(torch.isnan(lse), up)
        assert torch.equal(torch.isnan(out[0]),
                           both[:, None].expand(8, 256))
        assert torch.isfinite(lse[~up]).all()
        assert torch.isfinite(out[0][~both]).all()
