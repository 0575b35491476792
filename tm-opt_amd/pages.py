"""The page plan of a serving step, made on the GPU from its requests' lengths
(plan_pages), and the way back of finished requests' pages (release_pages).

A cache keeps, on the device, a page table [S, W] int32 with one row per
request it can hold, and a stack of free pages: free_pages [F] int32, of which
the first free_count [1] int32 name pages (none negative). plan_pages takes the
pages a step's new tokens need off the stack into the requests' rows, and gives
the index tensors that decode_paged, decode_diff_paged, prefill_varlen,
prefill_diff_varlen, kv_write_slots and kv_write_paged take. Nothing is read
back to the host, so a whole step can be captured and replayed while the
requests grow.
"""
from typing import NamedTuple

import torch

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


def _check_state(dev, page_table, free_pages, free_count):
    assert page_table.dtype == torch.int32 and page_table.dim() == 2
    assert page_table.is_contiguous()
    assert free_pages.dtype == torch.int32 and free_pages.dim() == 1
    assert free_pages.is_contiguous() and free_pages.device == dev
    assert free_count.dtype == torch.int32 and free_count.numel() == 1
    assert free_count.device == dev


def _check_index(t, dtype, n, dev):
    assert t.dtype == dtype and t.dim() == 1 and t.numel() == n, \
        (t.dtype, tuple(t.shape), dtype, n)
    assert t.is_contiguous() and t.device == dev


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
    as it is, and their outputs are NaN whole then; a KV write of such a plan
    writes nothing, a decode gives zeros. (Their max_context keeps a few tokens
    under a wide block table to one launch.)"""
    dev, B, T = page_table.device, slots.numel(), int(max_tokens)
    _check_state(dev, page_table, free_pages, free_count)
    _check_index(slots, torch.int64, B, dev)
    _check_index(ctx_lens, torch.int32, B, dev)
    _check_index(new_lens, torch.int32, B, dev)
    S, W = page_table.shape
    width = W if width is None else int(width)
    if out is None:
        # two allocations, cut (a slice costs as much as an allocation)
        pad = -B * width % 4             # 16-byte steps for what follows
        buf = torch.empty(B * (width + 2) + pad + 3, dtype=torch.int32,
                          device=dev)
        block, _, seq, cu, count, reject = buf.split_with_sizes(
            (B * width, pad, B, B + 1, 1, 1))
        slot_mapping, positions = torch.empty(
            2 * T, dtype=torch.int64, device=dev).split_with_sizes((T, T))
        out = PagePlan(block.view(B, width), seq, cu, slot_mapping, positions,
                       count, reject)
    else:
        block, seq, cu, slot_mapping, positions, count, reject = out
        assert block.dtype == torch.int32 and block.shape == (B, width)
        assert block.is_contiguous() and block.device == dev
        _check_index(seq, torch.int32, B, dev)
        _check_index(cu, torch.int32, B + 1, dev)
        _check_index(slot_mapping, torch.int64, T, dev)
        _check_index(positions, torch.int64, T, dev)
        _check_index(count, torch.int32, 1, dev)
        _check_index(reject, torch.int32, 1, dev)
    _call(dev, "tmopt_plan_pages", page_table.data_ptr(), S, W,
          slots.data_ptr(), ctx_lens.data_ptr(), new_lens.data_ptr(), B,
          free_pages.data_ptr(), free_pages.numel(), free_count.data_ptr(), T,
          width, block.data_ptr(), seq.data_ptr(), cu.data_ptr(),
          slot_mapping.data_ptr(), positions.data_ptr(), count.data_ptr(),
          reject.data_ptr())
    return out


def release_pages(page_table, slots, lens, free_pages, free_count, out=None):
    """Push the pages that the first ceil(lens[i] / 16) entries of page-table
    row slots[i] (negative: none) name back onto the stack free_pages (in
    place), in order. Entries that name none (negative: of pages a windowed
    request gave back before) are left out.

    Returns (free_count [1], reject [1]) int32: the stack's height
    afterwards, and 1 where nothing was done: a slot outside the table or
    named twice, a length that is negative or past the row, or a stack that
    would overflow. out: that pair to write into; its free_count may be
    free_count. The rows keep their entries; release a request once."""
    dev, B = page_table.device, slots.numel()
    _check_state(dev, page_table, free_pages, free_count)
    _check_index(slots, torch.int64, B, dev)
    _check_index(lens, torch.int32, B, dev)
    S, W = page_table.shape
    # the pair and the scratch in one allocation (16-byte steps)
    n = -(-(B + 1) // 4) * 4
    ws, count, reject = torch.empty(n + 2, dtype=torch.int32,
                                    device=dev).split_with_sizes((n, 1, 1))
    if out is None:
        out = count, reject
    else:
        count, reject = out
        _check_index(count, torch.int32, 1, dev)
        _check_index(reject, torch.int32, 1, dev)
    _call(dev, "tmopt_release_pages", page_table.data_ptr(), S, W,
          slots.data_ptr(), lens.data_ptr(), B, free_pages.data_ptr(),
          free_pages.numel(), free_count.data_ptr(), count.data_ptr(),
          reject.data_ptr(), ws.data_ptr(), 4 * n)
    return out
