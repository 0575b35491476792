"""Capped prefills whose first tile has scores far below the others', with values
as large as fp32 sums of them allow."""
import pytest
import torch

from oracle import scored_ref as ref
from test_gpu_mx4 import Cache4
from test_gpu_scored import BF, Cache, D, PAGE, _gen, _i32, _rand

pytestmark = pytest.mark.gpu


def _pages(k, v, g, dev):
    """Rows k, v [n, HKV, 128] in bf16 pages: pools and a table of one row."""
    n, hkv = k.shape[:2]
    c = Cache([n], hkv, g, dev)
    at = torch.arange(n, device=dev)
    rows = c.table[0][at // PAGE].long(), at % PAGE
    c.kp[rows], c.vp[rows] = k, v
    return c


def _pages4(tm, k, v, g, dev):
    """The same in 4 bits, with what they hold."""
    n, hkv = k.shape[:2]
    c = Cache4(tm, [n], hkv, g, dev)
    at = torch.arange(n, device=dev)
    rows = c.table[0][at // PAGE].long() * PAGE + at % PAGE
    tm.kv_write_mx4(k, v, rows, c.pool)
    P = c.pool.shape[0]
    c.kp, c.vp = (x.view(P, PAGE, hkv, D) for x in tm.kv_read_mx4(
        c.pool, torch.arange(P * PAGE, device=dev)))
    return c


def _prefill_of(tm, source, q, k, v, scale, g, dev, **kw):
    """One run from packed rows, bf16 pages or 4-bit pages, checked."""
    cu = _i32([0, q.shape[0]], dev)
    if source == "packed":
        out, lse = tm.prefill_scored_varlen(q, k, v, cu, scale, **kw)
        want = ref.prefill(q, k, v, cu, scale, **kw)
    else:
        zero = _i32([k.shape[0] - q.shape[0]], dev)
        if source == "paged":
            c = _pages(k, v, g, dev)
            out, lse = tm.prefill_scored_varlen(
                q, None, None, cu, scale, prior_lens=zero, k_pool=c.kp,
                v_pool=c.vp, block_table=c.table, **kw)
        else:
            c = _pages4(tm, k, v, g, dev)
            out, lse = tm.prefill_mx4_varlen(q, c.pool, c.table, cu, zero,
                                             scale, **kw)
        want = ref.prefill(q, None, None, cu, scale, prior=zero, k_pool=c.kp,
                           v_pool=c.vp, table=c.table, **kw)
    ref.check(out, lse, want, f"{source} {kw}")


@pytest.mark.parametrize("source", ["packed", "paged", "four"])
@pytest.mark.parametrize("cap", [30.0, 50.0, 53.0, 60.0])
@pytest.mark.parametrize("size", [1e-20, 1.0, 1e10, 1e20, 1e28])
def test_large_values_behind_low_scores(tm, dev, source, cap, size):
    """A first tile at the cap's low end and the others at its top; scores that
    rise from one key to the next."""
    g = _gen(70)
    n = 700
    base = _rand((1, 1, D), g, dev, 2.0)
    q = base.expand(n, 8, D).contiguous()
    square = float((base.float() ** 2).sum())
    v = (_rand((n, 2, D), g, dev).float() * size).to(BF)
    step = torch.ones(n, device=dev)
    step[:70] = -1.0
    ramp = torch.linspace(-0.45, 0.45, n, device=dev)
    for z in (3 * cap * step, cap * ramp, 4 * cap * ramp, -cap * ramp):
        k = base.float() * (z / (0.1 * square))[:, None, None]
        _prefill_of(tm, source, q, k.expand(n, 2, D).to(BF).contiguous(), v,
                    0.1, g, dev, softcap=cap)
