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
page_size); the pages past it are each sequence's own. extend_tables refuses to
write into a page of several references.

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
from hxlib import call


@dataclass
class BatchTables:
    query_start: torch.Tensor   # (B + 1,) int32: first packed token of each sequence, and their number
    seq_lens: torch.Tensor      # (B,) int32: tokens per sequence, the new ones included
    slot_mapping: torch.Tensor  # (num_tokens,) int64 pool slots; -1 past the batch's tokens
    positions: torch.Tensor     # (num_tokens,) int64 positions in the sequence; 0 past the batch's tokens
    free_count: torch.Tensor    # (1,) int32: pages left on the free stack


def _check(block_table, page_size, num_pages, free_pages, free_count, page_refs, **vectors):
    """Shapes, types and places; returns the number of pool pages."""
    if block_table.dim() != 2:
        raise ValueError(f"block_table should be (B, max_pages), got {tuple(block_table.shape)}")
    dev = block_table.device
    if dev.type != "cuda":
        hxlib.require_cuda(block_table)
    B, W = block_table.shape
    if block_table.dtype != _I32:
        raise TypeError(f"block_table must be int32, got {block_table.dtype}")
    vectors["free_pages"], vectors["free_count"] = free_pages, free_count
    if page_refs is not None:
        vectors["page_refs"] = page_refs
    for name, t in vectors.items():
        if t.dtype != _I32 or t.device != dev or t.dim() != 1 or not t.is_contiguous() \
                or (name not in _SIZED and t.shape[0] != B):
            hxlib.require_cuda(t)
            if t.dtype != _I32:
                raise TypeError(f"{name} must be int32, got {t.dtype}")
            if t.device != dev:
                raise ValueError(f"{name} is on {t.device}, block_table on {dev}")
            raise ValueError(f"{name} must be contiguous and " +
                             ("one-dimensional" if name in _SIZED else f"({B},)") + f", got {tuple(t.shape)}")
    if B and W and (block_table.stride(1) != 1 or (B > 1 and block_table.stride(0) < W)):
        raise ValueError("block_table rows must be contiguous and must not overlap")
    if free_count.shape[0] != 1:
        raise ValueError("free_count should be one number")
    if not 1 <= page_size < 1 << 31:
        raise ValueError("page_size must be at least 1 and fit 32 bits")
    n = int(num_pages) if num_pages is not None else (page_refs if page_refs is not None else free_pages).shape[0]
    if page_refs is not None and page_refs.shape[0] < n:
        raise ValueError(f"page_refs should hold one count for each of {n} pages")
    return n


_I32 = torch.int32
_SIZED = ("free_pages", "free_count", "page_refs")


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
    takes the results in existing tensors, which may overlap neither the inputs
    nor each other.

    Too few free pages, a sequence past max_pages, more tokens than
    ``num_tokens``, a negative length or a page id outside the pool (on the
    stack among those to be popped, or in the table where a sequence goes on)
    hand out nothing and flag a device error (CompactKVPool.check /
    hxlib.check_device_errors): all slots are -1 and seq_lens and free_count
    stay as they were. With ``page_refs`` so does a
    sequence whose new tokens would begin inside a page of more than one
    reference (a shared prefix cut to a length inside a page): its other
    holders read that page. Copy its rows to a page of the sequence's own
    first (CompactKVPool.unpack_to_staging, then write_kv), or cut to whole
    pages.
    """
    n_pages = _check(block_table, page_size, num_pages, free_pages, free_count, page_refs, cached_lens=cached_lens,
                     new_tokens=new_tokens)
    B, W = block_table.shape
    dev = block_table.device
    T = int(num_tokens)
    if not 0 <= T <= 1 << 30:
        raise ValueError(f"num_tokens must lie in 0 .. 2^30, got {T}")
    if out is None:
        i32, i64 = free_count.new_empty, torch.int64
        out = BatchTables(i32(B + 1), i32(B), i32(T, dtype=i64), i32(T, dtype=i64), i32(1))
    else:
        taken = [(hxlib.span(t), "one of the inputs") for t in (cached_lens, new_tokens, free_count, free_pages, block_table,
                                                           page_refs) if t is not None and t.numel()]
        for name, n, dt in (("query_start", B + 1, torch.int32), ("seq_lens", B, torch.int32),
                            ("slot_mapping", T, torch.int64), ("positions", T, torch.int64),
                            ("free_count", 1, torch.int32)):
            t = getattr(out, name)
            hxlib.require_cuda(t)
            if t.shape != (n,) or t.dtype != dt or t.device != dev or not t.is_contiguous():
                raise ValueError(f"out.{name} must be a contiguous ({n},) {dt} tensor on {dev}")
            if n:
                lo, hi = hxlib.span(t)
                for (a, e), whose in taken:
                    if lo < e and a < hi:
                        raise ValueError(f"out.{name} must not overlap {whose}")
                taken.append(((lo, hi), f"out.{name}"))
    i = dev.index
    with hxlib.on(i):
        call("hx_tables_extend", hxlib.raw_stream(i), block_table.data_ptr(), _row_stride(block_table), B, W,
             int(page_size), cached_lens.data_ptr(), new_tokens.data_ptr(), free_pages.data_ptr(), free_pages.shape[0],
             free_count.data_ptr(), page_refs.data_ptr() if page_refs is not None else None, n_pages,
             out.query_start.data_ptr(), out.seq_lens.data_ptr(), out.slot_mapping.data_ptr(), out.positions.data_ptr(),
             T, out.free_count.data_ptr(), hxlib.err_ptr(i))
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
    free_count) as new tensors. A page without a reference to give back, or an
    entry outside the pool, flags a device error and gives nothing back; the
    other entries do. A stack without room flags one as well, and then the
    lengths, the counts and the stack stay as they were.
    """
    n_pages = _check(block_table, page_size, num_pages, free_pages, free_count, page_refs, seq_lens=seq_lens,
                     keep_lens=keep_lens)
    B, W = block_table.shape
    dev = block_table.device
    lens, count = seq_lens.new_empty(B), free_count.new_empty(1)
    i = dev.index
    with hxlib.on(i):
        call("hx_tables_truncate", hxlib.raw_stream(i), block_table.data_ptr(), _row_stride(block_table), B, W,
             int(page_size), seq_lens.data_ptr(), keep_lens.data_ptr(), free_pages.data_ptr(), free_pages.shape[0],
             free_count.data_ptr(), page_refs.data_ptr() if page_refs is not None else None, n_pages, lens.data_ptr(),
             count.data_ptr(), hxlib.err_ptr(i))
    return lens, count
