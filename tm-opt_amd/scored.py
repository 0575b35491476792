"""Attention with score functions and masks over the paged cache and packed
prompts: decode_scored_paged (one new token per request) and
prefill_scored_varlen (packed runs of queries).

The score of query q (position p) and key k (position j) of head h is

  z = scale q.k
  x = softcap * tanh(z / softcap)       (softcap 0: x = z)
  x - slopes[h] * |p - j|               (slopes: fp32 [HQ], a bias by distance)

and the query sees the keys j of its request with

  j >= first_keys                       (int32, one per query: the start of its
                                         document in a request of several)
  j > p - window                        (window > 0)
  j <= max(p, prefix_lens - 1)          (int32, one per run: its first tokens,
                                         read in both directions)

A query that sees no key gives zeros, LSE -inf. A capped score is off by 2^-19 of
the cap at most, with caps above 256 by 2^-18 of z at most. K and V rows, pools and block tables are those of the other
entry points.
"""
import torch

from .attn import (HEAD_DIM, PAGE_SIZE, _check_rows, _ptr, _refused_rows)
from .diff import _call, _table, _workspace_size

_BF16, _F32, _I32 = torch.bfloat16, torch.float32, torch.int32
_DECODE_SIZE = "tmopt_attn_decode_workspace_size"
_PREFILL_SIZE = "tmopt_attn_prefill_scored_workspace_size"


def _slopes(slopes, HQ, dev):
    if slopes is not None:
        assert slopes.dtype == _F32 and slopes.shape == (HQ,)
        assert slopes.is_contiguous() and slopes.device == dev
    return _ptr(slopes)


def _int32(x):
    """x as the C entry points take it: ctypes would drop what is above."""
    x = int(x)
    assert -1 << 31 <= x < 1 << 31, x
    return x


def _index(t, n, dev):
    """The pointer of an optional int32 tensor [n], checked."""
    if t is not None:
        assert t.dtype == _I32 and t.shape == (n,), (t.dtype, t.shape, n)
        assert t.is_contiguous() and t.device == dev
    return _ptr(t)


def _pools(k_pool, v_pool, HQ, D, dev):
    shape = k_pool.shape
    P, page_size, HKV, Dk = shape
    assert k_pool.is_contiguous() and v_pool.is_contiguous()
    assert k_pool.dtype == _BF16 and v_pool.dtype == _BF16
    assert v_pool.shape == shape and Dk == D, (shape, D)
    assert k_pool.device == dev and v_pool.device == dev
    assert HQ % HKV == 0, (shape, HQ)
    return P, page_size, HKV


def _runs(cu_seqlens, total, max_seqlen, dev):
    """(runs, bound of their lengths) of cu_seqlens, checked."""
    assert cu_seqlens.dtype == _I32 and cu_seqlens.dim() == 1
    assert cu_seqlens.is_contiguous() and cu_seqlens.device == dev
    S = cu_seqlens.shape[0] - 1
    if total == 0:
        max_seqlen = 0                   # no run, whatever the bound
    if max_seqlen is None:
        max_seqlen = int((cu_seqlens[1:] - cu_seqlens[:-1]).max()) if S else 0
    return S, _int32(max_seqlen)


def _prefill_outputs(q, out, lse, return_lse, reject):
    """out like q and lse [HQ, total], given ones checked."""
    total, HQ, D = q.shape
    dev = q.device
    if reject is not None:
        assert reject.dtype == _I32 and reject.numel() >= 1
        assert reject.device == dev
    if out is None:
        out = torch.empty((total, HQ, D), dtype=_BF16, device=dev)
    else:
        assert out.shape == q.shape and out.device == dev
        _check_rows(out, "out")
    if lse is not None:
        assert lse.shape == (HQ, total) and lse.dtype == _F32
        assert lse.is_contiguous() and lse.device == dev
    elif return_lse:
        lse = torch.empty((HQ, total), dtype=_F32, device=dev)
    return out, lse


def decode_scored_paged(q, k_pool, v_pool, block_table, ctx_lens, scale,
                        softcap=0.0, slopes=None, first_keys=None, window=0,
                        table_wrap=0, min_pages=1, num_workgroups=0, out=None,
                        lse=None, workspace=None, return_lse=True):
    """Attention of one new token per request, paged, with score functions.

    q [B, HQ, 128] bf16 contiguous (request b's query at position
    ctx_lens[b] - 1); k_pool/v_pool [num_pages, 16, HKV, 128] bf16; block_table
    [B, bt_stride] int32 (keys of entries that name no page are absent);
    ctx_lens [B] int32; softcap, slopes, first_keys [B] as above; window 0 =
    global; table_wrap > 0 = each table row is a ring of that many pages;
    min_pages / num_workgroups: work-split knobs (see the C header; shares of 1
    / 2 / 8 pages at least, us per call, 32Q/4KV: 64 requests of 16 tokens 8.5 /
    10.4 / 22.3, 4 of 1,000 11.5 / 11.5 / 14.3, 64 of 4,096 73.8 each).
    workspace: from decode_workspace() (allocated if None; it needs no
    initialisation; calls that overlap need one each).
    Returns (out [B, HQ, 128] bf16, lse [B, HQ] fp32 or None)."""
    B, HQ, D = q.shape
    dev, num_workgroups = q.device, _int32(num_workgroups)
    assert q.dtype == _BF16 and q.is_contiguous()
    P, page_size, HKV = _pools(k_pool, v_pool, HQ, D, dev)
    bts = _table(block_table, B, dev)
    assert ctx_lens.dtype == _I32 and ctx_lens.shape == (B,)
    assert ctx_lens.is_contiguous() and ctx_lens.device == dev
    if table_wrap:
        assert 0 < window <= table_wrap * page_size, \
            "a ring table needs a window no wider than the ring"
    if out is None:
        out = torch.empty_like(q)
    else:
        assert out.shape == q.shape and out.device == dev
        assert out.dtype == _BF16 and out.is_contiguous()
    if lse is not None:
        assert lse.shape == (B, HQ) and lse.dtype == _F32
        assert lse.is_contiguous() and lse.device == dev
    elif return_lse:
        lse = torch.empty((B, HQ), dtype=_F32, device=dev)
    if workspace is None:
        n = _workspace_size(dev, _DECODE_SIZE, B, HQ, HKV, D, num_workgroups)
        workspace = torch.empty(max(n, 16), dtype=torch.uint8, device=dev)
    else:
        assert workspace.device == dev and workspace.is_contiguous()
        n = workspace.numel() * workspace.element_size()
    _call(dev, "tmopt_attn_decode_scored", q.data_ptr(), k_pool.data_ptr(),
          v_pool.data_ptr(), block_table.data_ptr(), bts, _int32(table_wrap),
          ctx_lens.data_ptr(), B, HQ, HKV, D, page_size, P, _int32(window),
          float(scale), float(softcap), _slopes(slopes, HQ, dev),
          _index(first_keys, B, dev), _int32(min_pages), num_workgroups,
          out.data_ptr(), _ptr(lse), workspace.data_ptr(), n)
    return out, lse


def prefill_scored_varlen(q, k, v, cu_seqlens, scale, softcap=0.0, slopes=None,
                          first_keys=None, prefix_lens=None, window=0,
                          max_seqlen=None, prior_lens=None, k_pool=None,
                          v_pool=None, block_table=None, out=None, lse=None,
                          return_lse=True, reject=None, max_context=None):
    """Varlen attention with score functions and masks.

    q [total, HQ, 128] bf16 (head_dim contiguous, any token / head strides);
    cu_seqlens [S + 1] int32; query j of run i at position prior_lens[i] + j.
    Keys:
      * block_table None: k/v [total, HKV, 128] hold each run's own keys,
        packed like q, and there is no prior context;
      * block_table [S, bt_stride] int32 given, k/v None: every key, prior
        context included, from k_pool/v_pool [num_pages, 16, HKV, 128]; the
        run's own keys must already be there. Pages without an entry read as
        zeros.
    softcap, slopes, first_keys [total], prefix_lens [S] as above (a prefix ends
    where the run does). reject: optional int32 device scalar; nonzero gives NaN
    in every row of out and lse, those that cu_seqlens gives no run included.
    max_seqlen bounds the run lengths (read from the device, with a
    synchronisation, if None); max_context: an upper bound of prior + run
    length, where the host has one (the row width of the block table bounds it
    otherwise): whether keys are split over work-groups goes by it.
    Returns (out [total, HQ, 128] bf16, lse [HQ, total] fp32 or None); rows behind
    the last run keep what they held."""
    total, HQ, D = q.shape
    dev = q.device
    _check_rows(q, "q")
    S, max_seqlen = _runs(cu_seqlens, total, max_seqlen, dev)
    if block_table is not None:
        assert k is None and v is None, "keys come from k/v or from the pools"
        P, page_size, HKV = _pools(k_pool, v_pool, HQ, D, dev)
        bts = _table(block_table, S, dev)
        strides = (0, 0, 0, 0)
    else:
        assert prior_lens is None, "prior context needs the paged source"
        assert k_pool is None and v_pool is None, "pools need a block table"
        assert k.shape == v.shape and k.dim() == 3 and k.shape[0] == total
        assert k.shape[2] == D and k.device == dev and v.device == dev
        _check_rows(k, "k")
        _check_rows(v, "v")
        P, page_size, HKV, bts = 0, PAGE_SIZE, k.shape[1], 0
        assert HQ % HKV == 0, (k.shape, HQ)
        strides = (k.stride(0), k.stride(1), v.stride(0), v.stride(1))
    out, lse = _prefill_outputs(q, out, lse, return_lse, reject)
    most = 0 if max_context is None else max(1, int(max_context))
    n = _workspace_size(dev, _PREFILL_SIZE, S, max_seqlen, most, HQ, HKV, bts,
                        _int32(window))
    ws = torch.empty(n, dtype=torch.uint8, device=dev) if n else None
    _call(dev, "tmopt_attn_prefill_scored_strided", q.data_ptr(), q.stride(0),
          q.stride(1), _ptr(k), strides[0], strides[1], _ptr(v), strides[2],
          strides[3], cu_seqlens.data_ptr(), _index(prior_lens, S, dev), S,
          max_seqlen, most, _ptr(k_pool), _ptr(v_pool), _ptr(block_table), bts,
          page_size, P, HQ, HKV, D, _int32(window), float(scale), float(softcap),
          _slopes(slopes, HQ, dev), _index(first_keys, total, dev),
          _index(prefix_lens, S, dev), out.data_ptr(), out.stride(0),
          out.stride(1), _ptr(lse), total, _ptr(reject), _ptr(ws), n)
    if reject is not None:
        _call(dev, "tmopt_refused_rows",
              *_refused_rows(reject, out, lse, *out.shape, HQ))
    return out, lse
