"""The page plan of a serving step, made on the GPU from its requests' lengths
(plan_pages), and the way back of finished requests' pages (release_pages).

A cache keeps, on the device, a page table [S, W] int32 with one row per
request it can hold, and a stack of free pages: free_pages [F] int32 with the
height free_count [1] int32. plan_pages takes the pages a step's new tokens
need off the stack into the requests' rows, and gives the index tensors that
decode_paged, decode_diff_paged, prefill_varlen, prefill_diff_varlen,
kv_write_slots and kv_write_paged take. Nothing is read back to the host, so a
whole step can be captured and replayed while the requests grow.
"""
from typing import NamedTuple

import torch

from . import _lib
from .attn import _ptr
from .diff import _call


class PagePlan(NamedTuple):
    """The index tensors of a step of B requests (on the device)."""
    block_table: torch.Tensor    # [B, width] int32, -1 past a request's pages
    seq_lens: torch.Tensor       # [B] int32: tokens with the new ones
    cu_seqlens: torch.Tensor     # [B + 1] int32: bounds of the new tokens
    slot_mapping: torch.Tensor   # [max_tokens] int64 pool rows, -1: none
    positions: torch.Tensor      # [max_tokens] int64
    free_count: torch.Tensor     # [1] int32: the stack's height afterwards
    reject: torch.Tensor         # [1] int32: 0, or 1 for a step that cannot be


def _state(page_table, slots, lens, free_pages, free_count):
    dev = page_table.device
    assert page_table.dtype == torch.int32 and page_table.dim() == 2
    assert page_table.is_contiguous()
    B = slots.shape[0]
    for t, d, name in ((slots, torch.int64, "slots"),
                       (lens, torch.int32, "lens")):
        assert t.dtype == d and t.shape == (B,), (name, t.dtype, t.shape)
        assert t.is_contiguous() and t.device == dev, name
    assert free_pages.dtype == torch.int32 and free_pages.dim() == 1
    assert free_pages.is_contiguous() and free_pages.device == dev
    assert free_count.dtype == torch.int32 and free_count.numel() == 1
    assert free_count.device == dev
    return dev, B


def plan_pages(page_table, slots, ctx_lens, new_lens, free_pages, free_count,
               max_tokens, width=None, out=None):
    """A step's PagePlan: request i holds ctx_lens[i] tokens in row slots[i]
    of page_table and gets new_lens[i] more (0: none; a negative slot:
    padding, a request without tokens).

    page_table [S, W] int32 (updated in place with the pages taken); slots [B]
    int64, each row at most once; ctx_lens, new_lens [B] int32; free_pages [F]
    int32 and free_count [1] int32, the stack of free pages (its height
    afterwards is the plan's free_count); max_tokens: the length of
    slot_mapping and positions, an upper bound of the step's new tokens;
    width: pages per row of the plan's block table (W if None).
    out: a PagePlan of the same sizes to write into; its free_count may be
    free_count and its seq_lens may be ctx_lens, so that a replayed graph
    steps on from where it was.
    A step that cannot be (a slot outside the table or named twice, negative
    lengths, a request past its row or past width, more than max_tokens
    tokens, too few free pages) gives reject = 1, takes no page and has no
    tokens: block table and slot mapping -1, cu_seqlens and positions 0,
    seq_lens the contexts. prefill_varlen and prefill_diff_varlen take reject
    as it is."""
    dev, B = _state(page_table, slots, ctx_lens, free_pages, free_count)
    S, W = page_table.shape
    assert new_lens.dtype == torch.int32 and new_lens.shape == (B,)
    assert new_lens.is_contiguous() and new_lens.device == dev
    T = int(max_tokens)
    width = W if width is None else int(width)
    if out is None:
        a = -(-B * width // 4) * 4       # 16-byte steps for what follows
        buf = torch.empty(a + 2 * B + 3, dtype=torch.int32, device=dev)
        rest = buf[a:]
        tok = torch.empty((2, T), dtype=torch.int64, device=dev)
        out = PagePlan(buf[:B * width].view(B, width), rest[:B],
                       rest[B:2 * B + 1], tok[0], tok[1],
                       rest[2 * B + 1:2 * B + 2], rest[2 * B + 2:])
    else:
        for t, d, shape in ((out.block_table, torch.int32, (B, width)),
                            (out.seq_lens, torch.int32, (B,)),
                            (out.cu_seqlens, torch.int32, (B + 1,)),
                            (out.slot_mapping, torch.int64, (T,)),
                            (out.positions, torch.int64, (T,)),
                            (out.free_count, torch.int32, (1,)),
                            (out.reject, torch.int32, (1,))):
            assert t.dtype == d and t.shape == shape, (t.dtype, t.shape, shape)
            assert t.is_contiguous() and t.device == dev
    _call(dev, "tmopt_plan_pages", page_table.data_ptr(), S, W, _ptr(slots),
          _ptr(ctx_lens), _ptr(new_lens), B, free_pages.data_ptr(),
          free_pages.shape[0], free_count.data_ptr(), T, width,
          _ptr(out.block_table), _ptr(out.seq_lens), _ptr(out.cu_seqlens),
          _ptr(out.slot_mapping), _ptr(out.positions), _ptr(out.free_count),
          _ptr(out.reject))
    return out


def release_pages(page_table, slots, lens, free_pages, free_count, out=None):
    """Push the ceil(lens[i] / 16) pages of page-table row slots[i] (negative:
    none) back onto the stack free_pages (in place), in order.

    Returns (free_count [1], reject [1]) int32: the stack's height
    afterwards, and 1 where nothing was done: a slot outside the table or
    named twice, a length that is negative or past the row, or a stack that
    would overflow. out: that pair to write into; its free_count may be
    free_count. The rows keep their entries; release a request once."""
    dev, B = _state(page_table, slots, lens, free_pages, free_count)
    if out is None:
        n = torch.empty(2, dtype=torch.int32, device=dev)
        out = n[:1], n[1:]
    else:
        for t in out:
            assert t.dtype == torch.int32 and t.shape == (1,)
            assert t.device == dev
    n = int(_lib.load().tmopt_release_pages_workspace_size(B))
    ws = torch.empty(max(n, 16), dtype=torch.uint8, device=dev)
    _call(dev, "tmopt_release_pages", page_table.data_ptr(),
          page_table.shape[0], page_table.shape[1], _ptr(slots), _ptr(lens),
          B, free_pages.data_ptr(), free_pages.shape[0],
          free_count.data_ptr(), _ptr(out[0]), _ptr(out[1]), ws.data_ptr(),
          ws.numel())
    return out
