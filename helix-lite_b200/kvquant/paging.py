"""Block tables and slot maps built on the GPU from request lengths.

The pool and its kernels take block tables, sequence lengths, slots, positions
and query offsets; these functions make them without a host round trip, from a
stack of free pages, and take pages back when sequences shrink or end:

  extend_tables    new tokens for every sequence of a batch: pages popped off
                   the free stack into the tables, and the batch's
                   query_start, seq_lens, slot_mapping and positions
                   (what write_kv, prompt_attention, prefill and decode take)
  truncate_tables  sequences cut to a shorter length (0 releases them): pages
                   nobody holds any more go back on the stack

``page_refs`` (int32, one count per pool page) lets sequences share pages: an
extended page starts at one reference, a truncated entry gives one back, and a
page returns to the stack with its last reference. To share a prefix, copy
table entries and add to the counts with torch (``block_table[rows, :n] =
block_table[src, :n]``, ``page_refs[pages] += len(rows)``, cached length n *
page_size); the pages past it are each sequence's own.

Pages keep their statistics and outlier lists until they are emptied:
``CompactKVPool.reset_allocated`` empties, per layer, the pages that one
extend_tables call handed out. The reference leaves tables and slots to vLLM's
scheduler on the host (src/kvquant/compact_backend.py:137-168 takes them as
inputs).
"""
from __future__ import annotations

from dataclasses import dataclass

import torch

import hxlib
from hxlib import call, ptr, stream


@dataclass
class BatchTables:
    query_start: torch.Tensor   # (B + 1,) int32: first packed token of each sequence, and their number
    seq_lens: torch.Tensor      # (B,) int32: tokens per sequence, the new ones included
    slot_mapping: torch.Tensor  # (num_tokens,) int64 pool slots; -1 past the batch's tokens
    positions: torch.Tensor     # (num_tokens,) int64 positions in the sequence; 0 past the batch's tokens
    free_count: torch.Tensor    # (1,) int32: pages left on the free stack


def _check(block_table, page_size, num_pages, free_pages, free_count, page_refs, **vectors):
    if block_table.dim() != 2:
        raise ValueError(f"block_table should be (B, max_pages), got {tuple(block_table.shape)}")
    named = {"block_table": block_table, "free_pages": free_pages, "free_count": free_count, **vectors}
    if page_refs is not None:
        named["page_refs"] = page_refs
    hxlib.require_cuda(*named.values())
    for name, t in named.items():
        if t.dtype != torch.int32:
            raise TypeError(f"{name} must be int32, got {t.dtype}")
        if t.device != block_table.device:
            raise ValueError(f"{name} is on {t.device}, block_table on {block_table.device}")
        if name != "block_table" and not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous")
    B = block_table.shape[0]
    if block_table.numel() and (block_table.stride(1) != 1 or (B > 1 and block_table.stride(0) < block_table.shape[1])):
        raise ValueError("block_table rows must be contiguous and must not overlap")
    for name, t in vectors.items():
        if t.shape != (B,):
            raise ValueError(f"{name} should be ({B},), got {tuple(t.shape)}")
    if free_count.numel() != 1 or free_pages.dim() != 1:
        raise ValueError("free_pages should be one-dimensional and free_count one number")
    if int(page_size) < 1:
        raise ValueError("page_size must be at least 1")
    n = int(num_pages) if num_pages is not None else (page_refs if page_refs is not None else free_pages).numel()
    if page_refs is not None and (page_refs.dim() != 1 or page_refs.numel() < n):
        raise ValueError(f"page_refs should hold one count for each of {n} pages")
    return n


def _row_stride(block_table):
    B, W = block_table.shape
    return int(block_table.stride(0)) if B > 1 else W


def extend_tables(block_table: torch.Tensor, cached_lens: torch.Tensor, new_tokens: torch.Tensor,
                  free_pages: torch.Tensor, free_count: torch.Tensor, *, num_tokens: int, page_size: int = 16,
                  page_refs: torch.Tensor | None = None, num_pages: int | None = None,
                  out: BatchTables | None = None) -> BatchTables:
    """Room for ``new_tokens[b]`` more tokens in each sequence (one kernel).

    block_table (B, max_pages) int32 is updated in place: entries past the
    ceil(cached / page_size) pages a sequence holds, up to what it needs. The
    k-th new page of the call, sequence by sequence, is ``free_pages[free_count
    - 1 - k]``. ``num_tokens`` is the length of the slot map (the batch's token
    count on the host, or an upper bound for a captured graph). ``num_pages``
    (the pool's block count; default: the length of page_refs or free_pages)
    bounds the page ids. Inputs other than block_table and page_refs are not
    changed: carry ``seq_lens`` and ``free_count`` on to the next step. ``out``
    takes the results in existing tensors, which may not be the inputs.

    Too few free pages, a sequence past max_pages, more tokens than
    ``num_tokens`` or a negative length hand out nothing and flag a device
    error (CompactKVPool.check / hxlib.check_device_errors): all slots are -1
    and seq_lens and free_count stay as they were.
    """
    n_pages = _check(block_table, page_size, num_pages, free_pages, free_count, page_refs, cached_lens=cached_lens,
                     new_tokens=new_tokens)
    B, W = block_table.shape
    dev = block_table.device
    T = int(num_tokens)
    if T < 0:
        raise ValueError("num_tokens must not be negative")
    want = {"query_start": ((B + 1,), torch.int32), "seq_lens": ((B,), torch.int32), "slot_mapping": ((T,), torch.int64),
            "positions": ((T,), torch.int64), "free_count": ((1,), torch.int32)}
    if out is None:
        out = BatchTables(*(torch.empty(s, dtype=d, device=dev) for s, d in want.values()))
    else:
        ins = {t.data_ptr() for t in (cached_lens, new_tokens, free_count, free_pages, block_table) if t.numel()}
        for name, (shape, dt) in want.items():
            t = getattr(out, name)
            hxlib.require_cuda(t)
            if t.shape != shape or t.dtype != dt or t.device != dev or not t.is_contiguous():
                raise ValueError(f"out.{name} must be a contiguous {shape} {dt} tensor on {dev}")
            if t.numel() and t.data_ptr() in ins:
                raise ValueError(f"out.{name} must not be one of the inputs")
    with torch.cuda.device(dev):
        call("hx_tables_extend", stream(dev), ptr(block_table), _row_stride(block_table), B, W, int(page_size),
             ptr(cached_lens), ptr(new_tokens), ptr(free_pages), free_pages.numel(), ptr(free_count), ptr(page_refs),
             n_pages, ptr(out.query_start), ptr(out.seq_lens), ptr(out.slot_mapping), ptr(out.positions), T,
             ptr(out.free_count), ptr(hxlib.err_word(dev)))
    return out


def truncate_tables(block_table: torch.Tensor, seq_lens: torch.Tensor, keep_lens: torch.Tensor,
                    free_pages: torch.Tensor, free_count: torch.Tensor, *, page_size: int = 16,
                    page_refs: torch.Tensor | None = None, num_pages: int | None = None):
    """Cut each sequence to min(keep_lens, seq_lens) tokens (one kernel).

    The pages past the kept tokens go back on the stack ``free_pages`` (changed
    in place), last one first, so that truncating what extend_tables just
    added leaves the stack as it was. With ``page_refs`` (changed in place) an
    entry gives back one reference, and a page is pushed once, with its last
    reference, at the place of the call's last entry that names it. Table
    entries past the kept pages keep their old values. Returns (seq_lens,
    free_count) as new tensors. A stack without room, or a page without a
    reference to give back, flags a device error.
    """
    n_pages = _check(block_table, page_size, num_pages, free_pages, free_count, page_refs, seq_lens=seq_lens,
                     keep_lens=keep_lens)
    B, W = block_table.shape
    dev = block_table.device
    lens = torch.empty((B,), dtype=torch.int32, device=dev)
    count = torch.empty((1,), dtype=torch.int32, device=dev)
    with torch.cuda.device(dev):
        call("hx_tables_truncate", stream(dev), ptr(block_table), _row_stride(block_table), B, W, int(page_size),
             ptr(seq_lens), ptr(keep_lens), ptr(free_pages), free_pages.numel(), ptr(free_count), ptr(page_refs),
             n_pages, ptr(lens), ptr(count), ptr(hxlib.err_word(dev)))
    return lens, count
