"""Differential attention over long contexts, where a bound that adds every
rounding of a probability is wider than the outputs: inputs whose
probabilities are powers of two (diff_ref.power_inputs), so that a page, a
piece or a row in the wrong place shows. The first tests plant such mistakes
in the oracle's own results and see them found."""
import math

import pytest
import torch

from oracle import diff_ref

D, PAGE, LN2 = 128, 16, math.log(2.0)
BF = torch.bfloat16


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _weights(hq, g, dev, norm):
    kw = dict(lam=(torch.rand(hq // 2, generator=g) * 1.2 - 0.2).to(dev))
    if norm:
        kw.update(weight=(1 + 0.3 * torch.randn(256, generator=g)).to(dev),
                  eps=1e-5, out_scale=0.4)
    return kw


def _user(w):
    kw = {x: y for x, y in w.items() if x != "lam"}
    if "weight" in kw:
        kw["norm_weight"], kw["norm_eps"] = kw.pop("weight"), kw.pop("eps")
    return kw


@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("N", [6500, 9064, 20001, 200001])
def test_check_finds_planted_mistakes(N, norm):
    g = _gen(N)
    q, k, v = diff_ref.power_inputs(1, N, 4, 2, g)
    w = _weights(4, g, "cpu", norm)
    at, pos = torch.tensor([N - 1]), torch.arange(N)

    def attend(k, v, pos):
        return diff_ref.attend(q, k, v, at, pos, scale=LN2, exact=True, **w)
    ref = attend(k, v, pos)

    def passes(k, v, pos=pos, lse=None):
        got = attend(k, v, pos)
        try:
            diff_ref.check(got[0].to(BF), lse if lse is not None else
                           got[1].float(), ref)
        except AssertionError:
            return False
        return True
    right = ref[1].float()
    assert passes(k, v) and passes(k, v, lse=right)
    page = torch.ones(N, dtype=torch.bool)
    page[PAGE * (N // 40):PAGE * (N // 40) + PAGE] = False
    piece = torch.ones(N, dtype=torch.bool)
    piece[N // 3 // PAGE * PAGE:N // 3 // PAGE * PAGE + 68 * PAGE] = False
    for keep in (page, piece):            # lost, also where the LSE is right
        assert not passes(k[keep], v[keep], pos[keep])
        assert not passes(k[keep], v[keep], pos[keep], lse=right)
    rows = torch.arange(N)
    rows[:PAGE], rows[64 * PAGE:65 * PAGE] = (
        torch.arange(64 * PAGE, 65 * PAGE), torch.arange(PAGE))
    assert not passes(k, v[rows])         # the values of two pages swapped
    assert not passes(k, v[torch.randperm(N, generator=g)])
    gone = v.clone()
    gone[~page] = 0
    assert not passes(k, gone)            # a page of values read as zeros
    twice = torch.cat([pos, pos[~page]])
    assert not passes(k[twice], v[twice], twice)
    with pytest.raises(AssertionError):
        diff_ref.check(torch.zeros((1, 2, 256), dtype=BF), right, ref)


def test_powers_are_exact_in_bf16():
    """What the bound rests on: the scaled score in fp32 is a whole number."""
    g = _gen(1)
    q, k, _ = diff_ref.power_inputs(3, 50, 4, 2, g)
    scale = torch.tensor(LN2, dtype=torch.float32) * torch.tensor(
        1.4426950408889634, dtype=torch.float32)
    assert scale.item() == 1.0
    s = torch.einsum("thd,nd->thn", q.float(), k[:, 0].float()) * scale
    assert torch.equal(s, s.round()) and s.abs().max() == 2
    p = torch.exp2(s - s.amax(-1, keepdim=True))
    assert torch.equal(p.to(BF).float(), p)


class _Cache:
    """Requests of the given lengths behind shuffled pages; NaN elsewhere."""

    def __init__(self, ends, hkv, g, dev):
        pages = [-(-n // PAGE) for n in ends]
        P = sum(pages) + 2
        perm = torch.randperm(P - 1, generator=g).int()
        self.table = torch.full((len(ends), max(pages)), P - 1,
                                dtype=torch.int32)
        self.kp = torch.full((P, PAGE, hkv, D), math.nan, dtype=BF, device=dev)
        self.vp = torch.full_like(self.kp, math.nan)
        at = 0
        for i, n in enumerate(ends):
            self.table[i, :pages[i]] = perm[at:at + pages[i]]
            at += pages[i]
            _, k, v = diff_ref.power_inputs(1, n, 2, hkv, g)
            pos = torch.arange(n)
            rows = self.table[i][pos // PAGE].long().to(dev), \
                (pos % PAGE).to(dev)
            self.kp[rows], self.vp[rows] = k.to(dev), v.to(dev)
        self.table = self.table.to(dev)
        self.ctx = torch.tensor(ends, dtype=torch.int32, device=dev)


@pytest.mark.gpu
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("ends,hq,hkv,call", [
    ([200001, 5, 0, 3000], 16, 2, {}),    # 184 pieces, later rounds of a join
    ([200001], 16, 2, dict(num_workgroups=128, min_pages=1)),
    ([50001], 32, 4, {}), ([20000, 20001, 33], 64, 8, {}),
    ([20001] * 20, 32, 4, {}), ([9064], 64, 16, {}),
    ([6500], 24, 12, dict(num_workgroups=5))])
def test_decode_long_contexts(tm, dev, ends, hq, hkv, call, norm):
    g = _gen(len(ends) + hq)
    c = _Cache(ends, hkv, g, dev)
    q = diff_ref.power_inputs(len(ends), 0, hq, hkv, g)[0].to(dev)
    w = _weights(hq, g, dev, norm)
    out, lse = tm.decode_diff_paged(q, c.kp, c.vp, c.table, c.ctx, w["lam"],
                                    LN2, **call, **_user(w))
    diff_ref.check(out, lse, diff_ref.decode(
        q, c.kp, c.vp, c.table, c.ctx, scale=LN2, exact=True, **w))


@pytest.mark.gpu
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("n,prior,hq,hkv", [
    (1, 20000, 16, 4), (64, 9000, 16, 4), (500, 6000, 16, 4),
    (3, 20000, 64, 8), (16, 1000, 64, 8), (300, 1000, 32, 4),
    (70, 6000, 24, 12)])
def test_prefill_long_contexts(tm, dev, n, prior, hq, hkv, norm):
    """Chunks after long contexts, cut into pieces and joined."""
    g = _gen(n + prior)
    c = _Cache([n + prior, 50], hkv, g, dev)
    q = diff_ref.power_inputs(n + 20, 0, hq, hkv, g)[0].to(dev)
    w = _weights(hq, g, dev, norm)
    cu = torch.tensor([0, n, n + 20], dtype=torch.int32, device=dev)
    pr = torch.tensor([prior, 30], dtype=torch.int32, device=dev)
    for most in (None, 1):                # (a bound that is too low: one launch)
        out, lse = tm.prefill_diff_varlen(
            q, None, None, cu, w["lam"], LN2, max_seqlen=max(n, 20),
            prior_lens=pr, k_pool=c.kp, v_pool=c.vp, block_table=c.table,
            max_context=most, **_user(w))
        diff_ref.check(out, lse, diff_ref.prefill(
            q, None, None, cu.tolist(), scale=LN2, exact=True, prior=pr,
            k_pool=c.kp, v_pool=c.vp, table=c.table, **w))


@pytest.mark.gpu
@pytest.mark.parametrize("n,hq,hkv", [(2050, 4, 4), (6500, 16, 2),
                                      (4000, 8, 2)])
def test_prefill_long_packed(tm, dev, n, hq, hkv):
    """One prompt, whole or in pieces; rows far down see thousands of keys."""
    g = _gen(n)
    q, k, v = (x.to(dev) for x in diff_ref.power_inputs(n, n, hq, hkv, g))
    w = _weights(hq, g, dev, True)
    cu = torch.tensor([0, n], dtype=torch.int32, device=dev)
    out, lse = tm.prefill_diff_varlen(q, k, v, cu, w["lam"], LN2,
                                      max_seqlen=n, **_user(w))
    diff_ref.check(out, lse, diff_ref.prefill(
        q, k, v, cu.tolist(), scale=LN2, exact=True, **w))
