"""Attention over a cache held in 4 bits: kv_write_mx4 and kv_read_mx4 (rows
into the pages and back), decode_mx4_paged (one new token per request) and
prefill_mx4_varlen (packed runs of queries).

A token's head is four blocks of 32 dims; a block keeps a scale 2^e in one byte
and 32 elements of 4 bits (0, .5, 1, 1.5, 2, 3, 4, 6 and their negatives): a
quarter of the bf16 pools' bytes, 136 a head for K and V. e is the smallest
exponent (from -125) with amax <= 7 * 2^e, and a value becomes the nearest
element times 2^e, ties to the even code: off by 2^e at most. A block that holds
a value which is no number, infinite or above 7 * 2^125 reads as NaN.

The cache is one tensor [num_pages, HKV, RECORD] uint8, from mx4_pool() (the C
header has the layout of a record). Pages, block tables and slot mappings are
those of the other entry points, so plan_pages serves it as it is.

Scores are scale q.k, and with
  softcap  x = softcap * tanh(scale q.k / softcap)
  slopes   x - slopes[h] * (pos_q - pos_k), fp32 [HQ]
  rel      x + rel[.., h, pos_q - pos_k] inside the band, without the other two
"""
import torch

from .attn import HEAD_DIM, PAGE_SIZE, _check_rows, _ptr, _refused_rows
from .diff import _call, _table, _workspace_size
from .scored import _index, _int32, _prefill_outputs, _runs, _slopes

_BF16, _F32, _I32 = torch.bfloat16, torch.float32, torch.int32
_DECODE_SIZE = "tmopt_attn_decode_mx4_workspace_size"
_PREFILL_SIZE = "tmopt_attn_prefill_mx4_workspace_size"

RECORD = 2176      # bytes of a page's part for one KV head


def mx4_pool(num_pages, HKV, device):
    """A cache of num_pages pages of 16 tokens, 2176 * HKV bytes each."""
    return torch.zeros((num_pages, HKV, RECORD), dtype=torch.uint8,
                       device=device)


def _pool(pool, dev):
    """(pages, HKV) of a 4-bit cache, checked."""
    assert pool.dtype == torch.uint8 and pool.dim() == 3, "not an mx4_pool"
    assert pool.shape[2] == RECORD and pool.is_contiguous(), pool.shape
    assert pool.device == dev
    return pool.shape[0], pool.shape[1]


def kv_write_mx4(k, v, slot_mapping, pool):
    """Rows k, v [T, HKV, 128] bf16 (head_dim contiguous, strides multiples of
    8, 16-byte aligned) into rows slot_mapping [T] int64 (page * 16 + offset)
    of the 4-bit cache. Rows outside the pool, negative ones among them, are
    skipped; a row that is named twice holds unspecified values."""
    T, HKV, D = k.shape
    dev = k.device
    assert v.shape == k.shape and v.device == dev
    _check_rows(k, "k")
    _check_rows(v, "v")
    P, H = _pool(pool, dev)
    assert H == HKV, (pool.shape, k.shape)
    assert slot_mapping.dtype == torch.int64 and slot_mapping.shape == (T,)
    assert slot_mapping.is_contiguous() and slot_mapping.device == dev
    _call(dev, "tmopt_kv_write_mx4", k.data_ptr(), v.data_ptr(), k.stride(0),
          k.stride(1), v.stride(0), v.stride(1), slot_mapping.data_ptr(), T,
          HKV, D, PAGE_SIZE, pool.data_ptr(), P)


def kv_read_mx4(pool, slot_mapping, k=None, v=None):
    """The values that rows slot_mapping [T] int64 of the 4-bit cache hold:
    (k, v) [T, HKV, 128] bf16, exact; zeros for a row outside the pool. k, v:
    contiguous outputs (allocated if None)."""
    dev = pool.device
    P, HKV = _pool(pool, dev)
    assert slot_mapping.dtype == torch.int64 and slot_mapping.dim() == 1
    assert slot_mapping.is_contiguous() and slot_mapping.device == dev
    T = slot_mapping.shape[0]
    shape = (T, HKV, HEAD_DIM)
    if k is None:
        k = torch.empty(shape, dtype=_BF16, device=dev)
    if v is None:
        v = torch.empty(shape, dtype=_BF16, device=dev)
    for x in (k, v):
        assert x.shape == shape and x.dtype == _BF16 and x.device == dev
        assert x.is_contiguous()
    _call(dev, "tmopt_kv_read_mx4", pool.data_ptr(), P,
          slot_mapping.data_ptr(), T, HKV, HEAD_DIM, PAGE_SIZE, k.data_ptr(),
          v.data_ptr())
    return k, v


def decode_mx4_workspace(B, HQ, HKV, device, num_workgroups=0):
    """Scratch for decode_mx4_paged: the partial results of split requests,
    516 bytes per query head and range of pages."""
    device = torch.device(device)
    if device.type == "cuda" and device.index is None:
        device = torch.device("cuda", torch.cuda.current_device())
    n = _workspace_size(device, _DECODE_SIZE, B, HQ, HKV, HEAD_DIM,
                        _int32(num_workgroups))
    return torch.empty(max(n, 16), dtype=torch.uint8, device=device)


def decode_mx4_paged(q, pool, block_table, ctx_lens, scale, softcap=0.0,
                     slopes=None, rel=None, window=0, table_wrap=0,
                     min_pages=4, num_workgroups=0, out=None, lse=None,
                     workspace=None, return_lse=True):
    """Attention of one new token per request over the 4-bit cache.

    q [B, HQ, 128] bf16 contiguous (request b's query at position
    ctx_lens[b] - 1); pool from mx4_pool(); block_table [B, bt_stride] int32
    (keys of entries that name no page are absent); ctx_lens [B] int32;
    softcap, slopes, rel (bf16 [B, HQ, E] contiguous) as above; window 0 =
    global; table_wrap > 0 = each table row is a ring of that many pages;
    min_pages / num_workgroups: work-split knobs (see the C header; shares of 4
    / 8 / 16 pages at least, us per call, 32Q/4KV: 64 requests of 16 tokens 8.2
    / 10.3 / 14.8, 4 of 1,000 10.5 / 10.6 / 12.6, 64 of 4,096 28.8 each).
    workspace: from decode_mx4_workspace() (allocated if None; it needs no
    initialisation; calls that overlap need one each).
    Returns (out [B, HQ, 128] bf16, lse [B, HQ] fp32 or None)."""
    B, HQ, D = q.shape
    dev, num_workgroups = q.device, _int32(num_workgroups)
    assert q.dtype == _BF16 and q.is_contiguous()
    P, HKV = _pool(pool, dev)
    assert HQ % HKV == 0, (pool.shape, HQ)
    bts = _table(block_table, B, dev)
    assert ctx_lens.dtype == _I32 and ctx_lens.shape == (B,)
    assert ctx_lens.is_contiguous() and ctx_lens.device == dev
    extent = 0
    if rel is not None:
        assert rel.dtype == _BF16 and rel.is_contiguous()
        assert rel.shape[:2] == (B, HQ) and rel.device == dev, rel.shape
        extent = rel.shape[2]
    if table_wrap:
        assert 0 < window <= table_wrap * PAGE_SIZE, \
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
    _call(dev, "tmopt_attn_decode_mx4", q.data_ptr(), pool.data_ptr(),
          block_table.data_ptr(), bts, _int32(table_wrap),
          ctx_lens.data_ptr(), B, HQ, HKV, D, PAGE_SIZE, P, _int32(window),
          float(scale), float(softcap), _slopes(slopes, HQ, dev), _ptr(rel),
          extent, _int32(min_pages), num_workgroups, out.data_ptr(), _ptr(lse),
          workspace.data_ptr(), n)
    return out, lse


def prefill_mx4_varlen(q, pool, block_table, cu_seqlens, prior_lens, scale,
                       softcap=0.0, slopes=None, rel=None, window=0,
                       max_seqlen=None, out=None, lse=None, return_lse=True,
                       reject=None, max_context=None):
    """Varlen causal (optionally windowed) attention over the 4-bit cache.

    q [total, HQ, 128] bf16 (head_dim contiguous, any token / head strides);
    block_table [S, bt_stride] int32; cu_seqlens [S + 1] int32; prior_lens [S]
    int32 or None (no prior context): query j of run i sits at position
    prior_lens[i] + j, and all its keys, the run's own among them, are in the
    pages already. Pages without an entry read as zeros. softcap, slopes, rel
    (bf16 [total, HQ, E], E contiguous) as above. reject: optional int32 device
    scalar; nonzero gives NaN in every row of out and lse, those that cu_seqlens
    gives no run included. max_seqlen bounds the run lengths (read from the
    device, with a synchronisation, if None); max_context: an upper bound of
    prior + run length, where the host has one (the row width of the block table
    bounds it otherwise): whether keys are split over work-groups goes by it.
    Returns (out [total, HQ, 128] bf16, lse [HQ, total] fp32 or None); rows behind
    the last run keep what they held."""
    total, HQ, D = q.shape
    dev = q.device
    _check_rows(q, "q")
    P, HKV = _pool(pool, dev)
    assert HQ % HKV == 0, (pool.shape, HQ)
    S, max_seqlen = _runs(cu_seqlens, total, max_seqlen, dev)
    bts = _table(block_table, S, dev)
    r_st = r_sh = extent = 0
    if rel is not None:
        assert rel.dtype == _BF16 and rel.stride(2) == 1
        assert rel.shape[:2] == (total, HQ) and rel.device == dev, rel.shape
        r_st, r_sh, extent = rel.stride(0), rel.stride(1), rel.shape[2]
    out, lse = _prefill_outputs(q, out, lse, return_lse, reject)
    most = 0 if max_context is None else max(1, int(max_context))
    n = _workspace_size(dev, _PREFILL_SIZE, S, max_seqlen, most, HQ, HKV, bts,
                        _int32(window))
    ws = torch.empty(n, dtype=torch.uint8, device=dev) if n else None
    _call(dev, "tmopt_attn_prefill_mx4_strided", q.data_ptr(), q.stride(0),
          q.stride(1), cu_seqlens.data_ptr(), _index(prior_lens, S, dev), S,
          max_seqlen, most, pool.data_ptr(), block_table.data_ptr(), bts,
          PAGE_SIZE, P, HQ, HKV, D, _int32(window), float(scale), float(softcap),
          _slopes(slopes, HQ, dev), _ptr(rel), r_st, r_sh, extent,
          out.data_ptr(), out.stride(0), out.stride(1), _ptr(lse), total,
          _ptr(reject), _ptr(ws), n)
    if reject is not None:
        _call(dev, "tmopt_refused_rows",
              *_refused_rows(reject, out, lse, *out.shape, HQ))
    return out, lse
