"""A step that plan_pages refuses, followed by the prefill that takes its
tensors: the plan has no tokens then, and every output row is NaN all the same
(never what the buffer held before)."""
import pytest
import torch

pytestmark = pytest.mark.gpu
D, PAGE, HQ, HKV = 128, 16, 8, 2
BF = torch.bfloat16


class Serving:
    """Two requests in a cache of a few pages, a chunk of prompt each."""

    def __init__(self, dev, new=(40, 21), spare=0):
        g = torch.Generator().manual_seed(sum(new))
        self.T = sum(new) + spare
        rand = lambda *s: torch.randn(s, generator=g).to(BF).to(dev)  # noqa: E731
        i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
        self.q = rand(self.T, HQ, D)
        self.kp, self.vp = rand(30, PAGE, HKV, D), rand(30, PAGE, HKV, D)
        self.lam = torch.full((HQ // 2,), 0.5, device=dev)
        self.table = torch.full((3, 8), -1, dtype=torch.int32, device=dev)
        self.slots = torch.tensor([2, 0], device=dev)
        self.ctx, self.new, self.most = i32([0, 0]), i32(list(new)), max(new)
        self.free = torch.arange(30, dtype=torch.int32, device=dev)
        self.count = i32([30])

    def plan(self, tm, out=None):
        return tm.plan_pages(self.table, self.slots, self.ctx, self.new,
                             self.free, self.count, self.T, out=out)

    def prefill(self, tm, diff, p, max_seqlen, **kw):
        kw.update(max_seqlen=max_seqlen, prior_lens=self.ctx, k_pool=self.kp,
                  v_pool=self.vp, block_table=p.block_table, reject=p.reject)
        if diff:
            return tm.prefill_diff_varlen(self.q, None, None, p.cu_seqlens,
                                          self.lam, 0.1, **kw)
        return tm.prefill_varlen(self.q, None, None, p.cu_seqlens, 0.1, **kw)


def _shape(diff):
    return (HQ // 2, 2 * D) if diff else (HQ, D)


@pytest.mark.parametrize("diff", [True, False])
@pytest.mark.parametrize("known", [True, False])
def test_refused_plan_gives_nan(tm, dev, diff, known):
    """With max_seqlen from the host, or read from the (empty) bounds."""
    s = Serving(dev)
    s.count.fill_(4)                               # five pages are needed
    p = s.plan(tm)
    out = torch.full((s.T,) + _shape(diff), 7.0, dtype=BF, device=dev)
    lse = torch.full((HQ, s.T), 7.0, device=dev)
    s.prefill(tm, diff, p, s.most if known else None, out=out, lse=lse)
    assert p.reject.item() == 1 and p.cu_seqlens.tolist() == [0, 0, 0]
    assert torch.isnan(out).all() and torch.isnan(lse).all()
    o, l = s.prefill(tm, diff, p, s.most if known else None,
                     return_lse=False)
    assert torch.isnan(o).all() and l is None


@pytest.mark.parametrize("diff", [True, False])
def test_refused_plan_in_a_graph(tm, dev, diff):
    """Replays of one captured step: taken, refused, taken again."""
    s = Serving(dev)

    def step():
        p = s.plan(tm)
        return (p,) + s.prefill(tm, diff, p, s.most)
    want = [x.clone() for x in step()[1:]]
    assert all(torch.isfinite(x).all() for x in want)
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        p, out, lse = step()
    for count in (30, 4, 30, 0, 4, 30):
        s.count.fill_(count)
        gr.replay()
        torch.zeros(100, device=dev).sum().item()
        assert p.reject.item() == (count < 5)
        if count < 5:
            assert torch.isnan(out).all() and torch.isnan(lse).all()
        else:
            assert torch.equal(out, want[0]) and torch.equal(lse, want[1])


@pytest.mark.parametrize("diff", [True, False])
def test_refused_rows_of_a_wider_tensor(tm, dev, diff):
    """Many rows, outputs inside a wider tensor: nothing beside them is
    written; a step that is taken leaves the rows past its tokens."""
    s = Serving(dev, new=(100, 28), spare=5000)
    heads, dim = _shape(diff)
    for count in (30, 3):
        s.count.fill_(count)
        big = torch.full((s.T + 1, heads + 1, dim + 8), 7.0, dtype=BF,
                         device=dev)
        out = big[:s.T, :heads, :dim]
        p = s.plan(tm)
        s.prefill(tm, diff, p, s.most, out=out, return_lse=False)
        rows = 128 if count == 30 else s.T
        assert (big[s.T] == 7).all() and (big[:, heads] == 7).all()
        assert (big[..., dim:] == 7).all() and (out[rows:] == 7).all()
        assert torch.isnan(out[:rows]).all() == (count == 3)


def test_refused_rows_are_those_of_q(tm, dev):
    """prefill_varlen takes outputs longer than its queries: the rows behind
    these stay as they are, in a refused step too."""
    s = Serving(dev)
    s.count.fill_(4)
    p = s.plan(tm)
    out = torch.full((s.T + 9, HQ, D), 7.0, dtype=BF, device=dev)
    s.prefill(tm, False, p, s.most, out=out, return_lse=False)
    assert torch.isnan(out[:s.T]).all() and (out[s.T:] == 7).all()


def test_refused_lse_as_one_row(tm, dev):
    """prefill_varlen asks of an LSE buffer that it holds HQ x total values:
    one row of them, at the end of an allocation, is filled and no more."""
    s = Serving(dev)
    s.count.fill_(4)
    p = s.plan(tm)
    buf = torch.full((HQ * s.T + 4096,), 7.0, device=dev)
    s.prefill(tm, False, p, s.most, lse=buf[:HQ * s.T])
    assert torch.isnan(buf[:HQ * s.T]).all() and (buf[HQ * s.T:] == 7).all()
