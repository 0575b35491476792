"""Differential attention over the paged cache: decode_diff_paged (one new
token per request) and prefill_diff_varlen (packed runs of queries).

Query heads 2h and 2h + 1 are the two maps of head pair h; stored heads 2g and
2g + 1, g = h // (HQ / HKV), hold their keys, and side by side the pair's
256-wide values:

  O_h = softmax(scale q_2h K_2g^T) V_g
        - lam_h softmax(scale q_2h+1 K_2g+1^T) V_g
  out_h = O_h / sqrt(mean(O_h^2) + norm_eps) * norm_weight * out_scale

(norm_weight None: out_h = O_h * out_scale; a query that sees no key gives
zeros). K and V rows, pools and block tables are laid out as for the other
entry points, so kv_write_slots, kv_write_paged and plan_pages serve them as
they are; HKV is even. lam: fp32 [HQ / 2], or [1] for all pairs; norm_weight:
fp32 [256].
"""
import functools

import torch

from . import _lib
from .attn import (HEAD_DIM, PAGE_SIZE, _check_rows, _ptr, _refused_rows,
                   _stream)

_BF16, _F32, _I32 = torch.bfloat16, torch.float32, torch.int32
_DECODE_SIZE = "tmopt_attn_decode_diff_workspace_size"
_PREFILL_SIZE = "tmopt_attn_prefill_diff_workspace_size"


def _call(dev, name, *args):
    """A launch on the current stream of dev, with dev the current device (the
    library sizes its grids by that device's compute units)."""
    if dev.type == "cuda" and dev.index != torch._C._cuda_getDevice():
        with torch.cuda.device(dev):
            return _lib.call(name, *args, _stream(dev))
    return _lib.call(name, *args, _stream(dev))


def _weights(lam, norm_weight, norm_eps, out_scale, HQ, dev):
    """The C arguments of the learned weights, checked."""
    n = lam.numel()
    assert lam.dtype == _F32 and lam.dim() == 1 and lam.device == dev
    assert n == HQ // 2 or n == 1, (tuple(lam.shape), HQ)
    assert lam.is_contiguous()
    if norm_weight is None:
        return lam.data_ptr(), n > 1, None, 0.0, float(out_scale)
    assert norm_weight.dtype == _F32 and norm_weight.shape == (2 * HEAD_DIM,)
    assert norm_weight.is_contiguous() and norm_weight.device == dev
    return (lam.data_ptr(), n > 1, norm_weight.data_ptr(), float(norm_eps),
            float(out_scale))


def _pools(k_pool, v_pool, HQ, D, dev):
    shape = k_pool.shape
    P, page_size, HKV, Dk = shape
    assert k_pool.is_contiguous() and v_pool.is_contiguous()
    assert k_pool.dtype == _BF16 and v_pool.dtype == _BF16
    assert v_pool.shape == shape and Dk == D, (shape, D)
    assert k_pool.device == dev and v_pool.device == dev
    assert HKV % 2 == 0 and HQ % HKV == 0, (shape, HQ)
    return P, page_size, HKV


def _table(block_table, rows, dev):
    """The row width of a block table, which is the stride that the kernels
    bound every row read by (so rows must be whole; one row may be part of a
    wider one)."""
    have, width = block_table.shape
    stride = block_table.stride()
    assert block_table.dtype == _I32 and block_table.device == dev
    assert have >= rows and stride[1] == 1
    assert stride[0] == width or rows <= 1, \
        "block-table rows must be whole (the row width is the stride)"
    return width


@functools.lru_cache(maxsize=1024)
def _workspace_size(dev, name, *shape):
    """The library's answer for a launch shape on a device, asked once."""
    fn = getattr(_lib.load(), name)
    if dev.type != "cuda":
        return int(fn(*shape))
    with torch.cuda.device(dev):
        return int(fn(*shape))


def decode_diff_workspace(B, HQ, HKV, device, num_workgroups=0):
    """Scratch for decode_diff_paged: the partial results of split requests,
    two rows of 1 KB per query head and range of pages (12.6 MB for 32Q/4KV,
    12.6 or 25.2 for 64Q/8KV on 256 compute units), and 4 bytes a request."""
    device = torch.device(device)
    if device.type == "cuda" and device.index is None:
        device = torch.device("cuda", torch.cuda.current_device())
    n = _workspace_size(device, _DECODE_SIZE, B, HQ, HKV, HEAD_DIM,
                        int(num_workgroups))
    return torch.empty(n, dtype=torch.uint8, device=device)


def decode_diff_paged(q, k_pool, v_pool, block_table, ctx_lens, lam, scale,
                      norm_weight=None, norm_eps=1e-5, out_scale=1.0,
                      window=0, table_wrap=0, min_pages=2, num_workgroups=0,
                      out=None, lse=None, workspace=None, return_lse=True):
    """Differential attention of one new token per request, paged.

    q [B, HQ, 128] bf16 contiguous (request b's query at position
    ctx_lens[b] - 1); k_pool/v_pool [num_pages, 16, HKV, 128] bf16;
    block_table [B, bt_stride] int32 (keys of entries that name no page are
    absent); ctx_lens [B] int32; lam fp32 [HQ / 2] or [1]; window 0 = global;
    table_wrap > 0 = each table row is a ring of that many pages; min_pages /
    num_workgroups: work-split knobs (see the C header; shares of 8 / 4 / 2
    pages at least, us per call, 32Q/4KV: one request of 1000 tokens 15.6 /
    13.8 / 13.2, 4 up to 1K 16.7 / 15.0 / 14.4, 16 up to 2K 18.9 each). workspace: from decode_diff_workspace() (allocated
    if None; it needs no initialisation; calls that overlap need one each).
    Returns (out [B, HQ / 2, 256] bf16, lse [B, HQ] fp32 or None)."""
    B, HQ, D = q.shape
    dev, num_workgroups = q.device, int(num_workgroups)
    assert q.dtype == _BF16 and q.is_contiguous()
    P, page_size, HKV = _pools(k_pool, v_pool, HQ, D, dev)
    bts = _table(block_table, B, dev)
    assert ctx_lens.dtype == _I32 and ctx_lens.shape == (B,)
    assert ctx_lens.is_contiguous() and ctx_lens.device == dev
    if table_wrap:
        assert 0 < window <= table_wrap * page_size, \
            "a ring table needs a window no wider than the ring"
    w = _weights(lam, norm_weight, norm_eps, out_scale, HQ, dev)
    if out is None:
        out = torch.empty((B, HQ // 2, 2 * D), dtype=_BF16, device=dev)
    else:
        assert out.shape == (B, HQ // 2, 2 * D) and out.device == dev
        assert out.dtype == _BF16 and out.is_contiguous()
    if lse is not None:
        assert lse.shape == (B, HQ) and lse.dtype == _F32
        assert lse.is_contiguous() and lse.device == dev
    elif return_lse:
        lse = torch.empty((B, HQ), dtype=_F32, device=dev)
    if workspace is None:
        n = _workspace_size(dev, _DECODE_SIZE, B, HQ, HKV, D, num_workgroups)
        workspace = torch.empty(n, dtype=torch.uint8, device=dev)
    else:
        assert workspace.device == dev and workspace.is_contiguous()
        n = workspace.numel() * workspace.element_size()
    _call(dev, "tmopt_attn_decode_diff", q.data_ptr(), k_pool.data_ptr(),
          v_pool.data_ptr(), block_table.data_ptr(), bts, int(table_wrap),
          ctx_lens.data_ptr(), B, HQ, HKV, D, page_size, P, int(window),
          float(scale), *w, int(min_pages), num_workgroups, out.data_ptr(),
          _ptr(lse), workspace.data_ptr(), n)
    return out, lse


def prefill_diff_varlen(q, k, v, cu_seqlens, lam, scale, norm_weight=None,
                        norm_eps=1e-5, out_scale=1.0, window=0,
                        max_seqlen=None, prior_lens=None, k_pool=None,
                        v_pool=None, block_table=None, out=None, lse=None,
                        return_lse=True, reject=None, max_context=None):
    """Varlen causal (optionally windowed) differential attention.

    q [total, HQ, 128] bf16 (head_dim contiguous, any token / head strides);
    cu_seqlens [S + 1] int32; query j of run i at position prior_lens[i] + j.
    Keys:
      * block_table None: k/v [total, HKV, 128] hold each run's own keys,
        packed like q, and there is no prior context;
      * block_table [S, bt_stride] int32 given, k/v None: every key, prior
        context included, from k_pool/v_pool [num_pages, 16, HKV, 128]; the
        run's own keys must already be there. Pages without an entry read as
        zeros, keys of score 0 (to decode_diff_paged they are absent): a table
        may lack pages before the window, not ones that a query sees.
    lam fp32 [HQ / 2] or [1]. reject: optional int32 device scalar; nonzero
    gives NaN in every row of out and lse, those that cu_seqlens gives no run
    included. max_seqlen bounds the run lengths (read from the device, with a
    synchronisation, if None).
    A launch of few query blocks that may see many keys splits these over
    work-groups and joins the pieces: a second launch, up to 3 x 257 KB of
    scratch per compute unit, and last bits that depend on the launch's other
    runs and the table's width. (So may those of a window's rows on how many
    runs share a launch: small ones take blocks of other sizes.) max_context: an
    upper bound of prior + run length, where the host has one; without it the
    row width of the block table bounds the keys, and short contexts under a
    wide table (plan_pages' is as wide as the cache's rows) pay for the second
    launch (64Q/8KV, 4,134 pages: 64 tokens without context 16.8 us against
    9.0, 30 after 2,000 31.2 against 24.6). It decides about the launch's
    layout alone.
    Returns (out [total, HQ / 2, 256] bf16, lse [HQ, total] fp32 or None)."""
    total, HQ, D = q.shape
    dev = q.device
    _check_rows(q, "q")
    assert cu_seqlens.dtype == torch.int32 and cu_seqlens.dim() == 1
    assert cu_seqlens.is_contiguous() and cu_seqlens.device == dev
    S = cu_seqlens.shape[0] - 1
    if total == 0:
        max_seqlen = 0                   # no run, whatever the bound
    if max_seqlen is None:
        max_seqlen = int((cu_seqlens[1:] - cu_seqlens[:-1]).max()) if S else 0
    if block_table is not None:
        assert k is None and v is None, "keys come from k/v or from the pools"
        P, page_size, HKV = _pools(k_pool, v_pool, HQ, D, dev)
        bts = _table(block_table, S, dev)
        if prior_lens is not None:
            assert prior_lens.dtype == torch.int32 and prior_lens.shape == (S,)
            assert prior_lens.is_contiguous() and prior_lens.device == dev
        strides = (0, 0, 0, 0)
    else:
        assert prior_lens is None, "prior context needs the paged source"
        assert k_pool is None and v_pool is None, "pools need a block table"
        assert k.shape == v.shape and k.dim() == 3 and k.shape[0] == total
        assert k.shape[2] == D and k.device == dev and v.device == dev
        _check_rows(k, "k")
        _check_rows(v, "v")
        P, page_size, HKV, bts = 0, PAGE_SIZE, k.shape[1], 0
        assert HKV % 2 == 0 and HQ % HKV == 0, (k.shape, HQ)
        strides = (k.stride(0), k.stride(1), v.stride(0), v.stride(1))
    w = _weights(lam, norm_weight, norm_eps, out_scale, HQ, dev)
    if reject is not None:
        assert reject.dtype == torch.int32 and reject.numel() >= 1
        assert reject.device == dev
    if out is None:
        out = torch.empty((total, HQ // 2, 2 * D), dtype=torch.bfloat16,
                          device=dev)
    else:
        assert out.shape == (total, HQ // 2, 2 * D) and out.device == dev
        _check_rows(out, "out")
    if lse is not None:
        assert lse.shape == (HQ, total) and lse.dtype == torch.float32
        assert lse.is_contiguous() and lse.device == dev
    elif return_lse:
        lse = torch.empty((HQ, total), dtype=torch.float32, device=dev)
    most = 0 if max_context is None else max(1, int(max_context))
    max_seqlen, window = int(max_seqlen), int(window)
    n = _workspace_size(dev, _PREFILL_SIZE, S, max_seqlen, most, HQ, HKV, bts,
                        window)
    ws = torch.empty(n, dtype=torch.uint8, device=dev) if n else None
    _call(dev, "tmopt_attn_prefill_diff", q.data_ptr(), q.stride(0),
          q.stride(1), _ptr(k), strides[0], strides[1], _ptr(v), strides[2],
          strides[3], cu_seqlens.data_ptr(), _ptr(prior_lens), S, max_seqlen,
          most, _ptr(k_pool), _ptr(v_pool), _ptr(block_table), bts, page_size, P,
          HQ, HKV, D, window, float(scale), *w, out.data_ptr(), out.stride(0),
          out.stride(1), _ptr(lse), total, _ptr(reject), _ptr(ws), n)
    if reject is not None:
        _call(dev, "tmopt_refused_rows",
              *_refused_rows(reject, out, lse, *out.shape, HQ))
    return out, lse
