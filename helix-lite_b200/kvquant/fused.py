"""Quest page selection and fused-dequant decode attention over a CompactKVPool.

This is the B200 hot path that replaces, per layer and decode step,
``select_top_blocks_for_layer`` + ``unpack_to_staging`` + FlashAttention on a
fp16 staging buffer (src/kvquant/compact_backend.py:225-299):

  quest_select   page scores from the pool's fp16 K min / max (pinned fp32
                 arithmetic) and an exact per-(sequence, KV head) top-K
                 threshold: sinks + the best k pages, ties to the lower page
  decode         one decode token per sequence: the selected pages are read
                 as packed codes, dequantised on chip and attended; returns
                 normalised o (fp32) and lse (natural log)
  selected_lists the selection as ascending page lists (API / tests)
  prefill        causal attention of prompt chunks, read from the pool
  shared_prefix_decode  decode of a batch on one prefix, read once for many
  prompt_attention  causal attention of whole prompts from their own K and V

quest_select also returns, per (b, h), how many pages each slice of the
sequence contributes (the threshold kernel's blocks count them as they go),
and decode balances its splits over the selected pages with them: every CTA
gets the same number of selected pages however the selection clusters along
the sequence, and finds its pages by scanning the scores of its slices.

Everything is asynchronous on the current stream; scratch is cached per
device and left zeroed by the kernels.
"""
from __future__ import annotations

import math
from dataclasses import dataclass

import torch

import hxlib
from hxlib import SEL_DENSE, SEL_LIST, SEL_SLICES, SEL_THRESHOLD, call, ptr, stream

from .compact_pool import CompactKVPool, ctypes_ref

NUM_SMS = 148


@dataclass
class Selection:
    scores: torch.Tensor      # (B, H, max_pages) fp32
    thresh: torch.Tensor      # (B * H,) int64 holding uint64 thresholds
    seq_lens: torch.Tensor    # (B,) int32 tokens
    page_size: int
    max_pages: int
    sink_pages: int
    lists: torch.Tensor | None = None   # (B * H, max_pages) int32 ascending selected pages
    counts: torch.Tensor | None = None  # (B * H,) int32
    slice_off: torch.Tensor | None = None  # (B * H, slices + 1) int32 exclusive selected counts


def _i32(t, device):
    if t.dtype == torch.int32 and t.device == device and t.is_contiguous():
        return t
    return t.to(device=device, dtype=torch.int32).contiguous()


def page_scores(pool: CompactKVPool, layer_idx: int, q: torch.Tensor, bt: torch.Tensor, sl: torch.Tensor,
                max_pages: int, sink_pages: int, scores: torch.Tensor, hist: torch.Tensor | None = None,
                gqa: str = "sum"):
    """Quest bounds of every page of each sequence into ``scores`` (B, H,
    max_pages) fp32 (one kernel); with ``hist`` also the level-1 key histogram
    the threshold kernel starts from. q (B, Hq, D) fp16 and bt / sl int32 on
    the pool's device."""
    B, Hq, D = q.shape
    H = pool.num_kv_heads
    stats = pool.layers[layer_idx].stats
    call("hx_quest_scores", stream(pool.device), ptr(q), B, H, Hq // H, D, 0 if gqa == "sum" else 1, 1,
         ptr(stats), hxlib.ctypes.c_void_p(stats.data_ptr() + 2 * D), 2 * D, pool.num_blocks * 2 * D,
         ptr(bt), bt.shape[1], ptr(sl), pool.block_size, max_pages, sink_pages, ptr(scores),
         ptr(hist) if hist is not None else None)


def quest_select(pool: CompactKVPool, layer_idx: int, query: torch.Tensor, block_table: torch.Tensor,
                 seq_lens: torch.Tensor, *, top_k: int | None = None, top_frac=(1, 4), sink_pages: int = 4,
                 gqa: str = "sum", max_pages: int | None = None, scores: torch.Tensor | None = None,
                 thresh: torch.Tensor | None = None, lists: bool = False,
                 list_out: tuple[torch.Tensor, torch.Tensor] | None = None,
                 slice_out: torch.Tensor | None = None) -> Selection:
    """Score every page of each sequence and fix the exact top-K thresholds.

    query (B, Hq, D) fp16 with Hq = group * H; block_table (B, >= max_pages)
    logical -> pool page; seq_lens (B,) tokens; optional preallocated
    ``scores`` (B, H, max_pages) fp32 and ``thresh`` (B*H,) int64 outputs.
    k = top_k pages if given,
    else floor(n_pages * top_frac[0] / top_frac[1]); gqa "sum" adds the
    per-query-head bounds of a group, "mean" bounds the group's mean query
    (the reference hook, compact_backend.py:231). The per-slice counts the
    decode balances over land in ``slice_out`` ((B*H, slices + 1) int32,
    slices = hx_quest_slices(max_pages)) when given. ``lists`` also writes
    the ascending page lists, into ``list_out`` = ((B*H, max_pages) int32,
    (B*H,) int32) when given.
    """
    dev = pool.device
    q = query.to(device=dev, dtype=torch.float16).contiguous()
    B, Hq, D = q.shape
    H = pool.num_kv_heads
    S = pool.block_size
    if Hq % H:
        raise ValueError("query heads must be a multiple of KV heads")
    bt = _i32(block_table, dev)
    sl = _i32(seq_lens, dev)
    mp = int(max_pages if max_pages is not None else bt.shape[1])
    if scores is None:
        scores = torch.empty((B, H, max(mp, 1)), dtype=torch.float32, device=dev)
    if thresh is None:
        thresh = torch.empty((B * H,), dtype=torch.int64, device=dev)
    hist = hxlib.scratch(dev, "quest_hist", B * H * 2 * 4096 * 4)
    cand = hxlib.scratch(dev, "quest_cand", B * H * max(mp, 1) * 8)
    ctr = hxlib.scratch(dev, "quest_ctr", B * H * 2 * 4)
    with torch.cuda.device(dev):
        st = stream(dev)
        page_scores(pool, layer_idx, q, bt, sl, mp, sink_pages, scores, hist, gqa)
        kf, fn, fd = (int(top_k), 0, 0) if top_k is not None else (0, int(top_frac[0]), int(top_frac[1]))
        nsl = int(hxlib.lib().hx_quest_slices(mp))
        if slice_out is None:
            slice_out = torch.empty((B * H, nsl + 1), dtype=torch.int32, device=dev)
        if slice_out.shape != (B * H, nsl + 1) or slice_out.dtype != torch.int32:
            raise ValueError(f"slice_out must be ({B * H}, {nsl + 1}) int32")
        call("hx_quest_threshold_slices", st, ptr(scores), B, H, ptr(sl), S, mp, sink_pages, kf, fn, fd, 1,
             ptr(hist), ptr(cand), ptr(ctr), ptr(thresh), ptr(slice_out), ptr(hxlib.err_word(dev)))
        lst = cnt = None
        if lists or list_out is not None:
            mpl = max(mp, 1)
            if list_out is not None:
                lst, cnt = list_out
            else:
                lst = torch.empty((B * H, mpl), dtype=torch.int32, device=dev)
                cnt = torch.empty((B * H,), dtype=torch.int32, device=dev)
            if lst.shape != (B * H, mpl) or cnt.shape != (B * H,) or lst.dtype != torch.int32:
                raise ValueError("list_out must be ((B*H, max_pages) int32, (B*H,) int32)")
            nch = -(-mpl // 2048)
            chunks = hxlib.scratch(dev, "quest_chunks", B * H * nch * 4)
            call("hx_quest_lists", st, ptr(scores), ptr(thresh), B, H, ptr(sl), S, mp, sink_pages, mpl, ptr(lst),
                 ptr(cnt), ptr(chunks))
    return Selection(scores, thresh, sl, S, mp, sink_pages, lst, cnt, slice_out)


def selected_lists(sel: Selection, union: bool = False, max_out: int | None = None):
    """Ascending selected logical pages: (B, H, max_out) int32 + counts (B, H);
    with union=True the union over heads: (B, max_out) + (B,)."""
    B, H, mp = sel.scores.shape
    mo = int(max_out if max_out is not None else mp)
    dev = sel.scores.device
    rows = B if union else B * H
    out = torch.full((rows, max(mo, 1)), -1, dtype=torch.int32, device=dev)
    counts = torch.empty((rows,), dtype=torch.int32, device=dev)
    with torch.cuda.device(dev):
        call("hx_quest_compact", stream(dev), ptr(sel.scores), ptr(sel.thresh), B, H, ptr(sel.seq_lens),
             sel.page_size, sel.max_pages, sel.sink_pages, 1 if union else 0, mo, ptr(out), ptr(counts))
    if union:
        return out, counts
    return out.view(B, H, -1), counts.view(B, H)


def default_splits(B: int, H: int, max_pages: int) -> int:
    """Splits per (sequence, head): about one decode CTA (12 warps) per SM."""
    want = max(1, math.ceil(NUM_SMS / max(1, B * H)))
    return max(1, min(want, max(1, math.ceil(max_pages / 16))))


def decode(pool: CompactKVPool, layer_idx: int, query: torch.Tensor, block_table: torch.Tensor,
           seq_lens: torch.Tensor, selection: Selection | None = None, *, lists: torch.Tensor | None = None,
           list_counts: torch.Tensor | None = None, page_begin: int = 0, max_pages: int | None = None,
           n_splits: int | None = None, softmax_scale: float | None = None, out16: torch.Tensor | None = None,
           o: torch.Tensor | None = None, lse: torch.Tensor | None = None, v_pos: str = "logical",
           cores: str = "tensor"):
    """Fused-dequant decode attention; returns (o (B, Hq, D) fp32, lse (B, Hq)).

    Pages attended: every page (no selection), the Quest selection (split
    over its selected pages by the selection's slice counts, else by its
    lists when it has them, else over the sequence), or explicit per-(b, h)
    logical page lists (``lists`` (B, H, L) int32 with ``list_counts`` (B,
    H)). ``page_begin`` is the absolute logical page of this pool's page 0
    (split-KV shards), used for V's position clamp. ``cores="cuda"`` runs QK
    and PV as fp32 FFMA on the CUDA cores (the comparison variant) instead of
    mma.sync on the tensor cores.
    """
    if cores not in ("tensor", "cuda"):
        raise ValueError("cores must be 'tensor' or 'cuda'")
    dev = pool.device
    q = query.to(device=dev, dtype=torch.float16).contiguous()
    B, Hq, D = q.shape
    H = pool.num_kv_heads
    bt = _i32(block_table, dev)
    sl = _i32(seq_lens, dev)
    mp = int(max_pages if max_pages is not None else bt.shape[1])
    slice_off = None
    if selection is not None and selection.slice_off is not None and lists is None:
        mp = selection.max_pages
        slice_off = selection.slice_off
        mode = SEL_SLICES
    elif selection is not None and selection.lists is not None and lists is None:
        lists, list_counts = selection.lists, selection.counts
        mode = SEL_LIST
        selection = None
    elif selection is not None:
        mp = selection.max_pages  # the scores' row stride
        mode = SEL_THRESHOLD
    elif lists is not None:
        mode = SEL_LIST
    else:
        mode = SEL_DENSE
    ns = int(n_splits or default_splits(B, H, mp if mode != SEL_LIST else lists.shape[-1]))
    scale = float(softmax_scale if softmax_scale is not None else 1.0 / math.sqrt(D))
    if o is None:
        o = torch.empty((B, Hq, D), dtype=torch.float32, device=dev)
    if lse is None:
        lse = torch.empty((B, Hq), dtype=torch.float32, device=dev)
    nbytes = hxlib.lib().hx_decode_scratch_bytes(B, H, ns)
    scr = hxlib.scratch(dev, "decode", nbytes)
    st_scales, _keep = pool.scales.device_layer(layer_idx, dev)
    if mode == SEL_LIST:
        lists_c = _i32(lists, dev).view(B * H, -1)
        counts_c = _i32(list_counts, dev)
        lstride = lists_c.shape[1]
    elif mode == SEL_SLICES:
        lists_c, counts_c = slice_off, None
        lstride = slice_off.shape[1]
    else:
        lists_c = counts_c = None
        lstride = 0
    with torch.cuda.device(dev):
        call("hx_decode_attn", stream(dev), ctypes_ref(pool.layers[layer_idx].struct), ctypes_ref(st_scales),
             ptr(q), B, Hq // H, scale, ptr(bt), bt.shape[1], ptr(sl), int(page_begin), mp,
             mode | (hxlib.VPOS_PHYSICAL if v_pos == "physical" else 0)
             | (hxlib.DECODE_CUDA_CORES if cores == "cuda" else 0),
             ptr(selection.scores) if selection is not None else None,
             ptr(selection.thresh) if selection is not None else None,
             selection.sink_pages if selection is not None else 0,
             ptr(lists_c), lstride, ptr(counts_c), ns, ptr(scr), ptr(o), ptr(lse), ptr(out16),
             ptr(hxlib.err_word(dev)))
    return o, lse


FUSED_MAX_PAGES = 16384   # rows the decode can select for itself (hx_decode_attn_select)


def quest_decode(pool: CompactKVPool, layer_idx: int, query: torch.Tensor, block_table: torch.Tensor,
                 seq_lens: torch.Tensor, *, top_k: int | None = None, top_frac=(1, 4), sink_pages: int = 4,
                 gqa: str = "sum", max_pages: int | None = None, scores: torch.Tensor | None = None, **kw):
    """Quest selection and fused decode in two kernels: the page scores (with
    their level-1 histogram), then the decode, whose CTAs find their row's
    exact top-K threshold themselves (hx_decode_attn_select). Same selection
    and outputs as quest_select + decode, without the threshold kernel; rows
    of at most FUSED_MAX_PAGES pages. Keyword arguments of decode_select
    pass through. Returns (o, lse)."""
    dev = pool.device
    q = query.to(device=dev, dtype=torch.float16).contiguous()
    B, Hq, D = q.shape
    H = pool.num_kv_heads
    if Hq % H:
        raise ValueError("query heads must be a multiple of KV heads")
    bt = _i32(block_table, dev)
    sl = _i32(seq_lens, dev)
    mp = int(max_pages if max_pages is not None else bt.shape[1])
    if scores is None:
        scores = torch.empty((B, H, max(mp, 1)), dtype=torch.float32, device=dev)
    hist = hxlib.scratch(dev, "quest_hist", B * H * 2 * 4096 * 4)
    with torch.cuda.device(dev):
        page_scores(pool, layer_idx, q, bt, sl, mp, sink_pages, scores, hist, gqa)
    return decode_select(pool, layer_idx, q, bt, sl, scores, top_k=top_k, top_frac=top_frac, sink_pages=sink_pages,
                         max_pages=mp, **kw)


def decode_select(pool: CompactKVPool, layer_idx: int, q: torch.Tensor, bt: torch.Tensor, sl: torch.Tensor,
                  scores: torch.Tensor, *, top_k: int | None = None, top_frac=(1, 4), sink_pages: int = 4,
                  max_pages: int | None = None, page_begin: int = 0, n_splits: int | None = None,
                  softmax_scale: float | None = None, o: torch.Tensor | None = None,
                  lse: torch.Tensor | None = None, out16: torch.Tensor | None = None, v_pos: str = "logical",
                  cores: str = "tensor", thresh_out: torch.Tensor | None = None,
                  slice_out: torch.Tensor | None = None):
    """The decode half of quest_decode: ``scores`` and the level-1 histogram
    (the "quest_hist" scratch) from page_scores; q fp16, bt / sl int32 on the
    pool's device. thresh_out (B*H,) int64 and slice_out (B*H, slices + 1)
    int32 receive the rows' thresholds and slice offsets when given."""
    dev = pool.device
    B, Hq, D = q.shape
    H = pool.num_kv_heads
    if cores not in ("tensor", "cuda"):
        raise ValueError("cores must be 'tensor' or 'cuda'")
    mp = int(max_pages if max_pages is not None else bt.shape[1])
    if mp > FUSED_MAX_PAGES:
        raise ValueError(f"decode_select selects rows of at most {FUSED_MAX_PAGES} pages; use quest_select")
    hist = hxlib.scratch(dev, "quest_hist", B * H * 2 * 4096 * 4)
    kf, fn, fd = (int(top_k), 0, 0) if top_k is not None else (0, int(top_frac[0]), int(top_frac[1]))
    ns = int(n_splits or default_splits(B, H, mp))
    scale = float(softmax_scale if softmax_scale is not None else 1.0 / math.sqrt(D))
    if o is None:
        o = torch.empty((B, Hq, D), dtype=torch.float32, device=dev)
    if lse is None:
        lse = torch.empty((B, Hq), dtype=torch.float32, device=dev)
    scr = hxlib.scratch(dev, "decode", hxlib.lib().hx_decode_scratch_bytes(B, H, ns))
    st_scales, _keep = pool.scales.device_layer(layer_idx, dev)
    flags = (hxlib.VPOS_PHYSICAL if v_pos == "physical" else 0) | (hxlib.DECODE_CUDA_CORES if cores == "cuda" else 0)
    with torch.cuda.device(dev):
        call("hx_decode_attn_select", stream(dev), ctypes_ref(pool.layers[layer_idx].struct), ctypes_ref(st_scales),
             ptr(q), B, Hq // H, scale, ptr(bt), bt.shape[1], ptr(sl), int(page_begin), mp, flags, ptr(scores),
             ptr(hist), sink_pages, kf, fn, fd, ns, ptr(scr), ptr(o), ptr(lse), ptr(out16), ptr(thresh_out),
             ptr(slice_out), ptr(hxlib.err_word(dev)))
    return o, lse


def prefill(pool: CompactKVPool, layer_idx: int, query: torch.Tensor, query_start: torch.Tensor,
            block_table: torch.Tensor, seq_lens: torch.Tensor, *, max_query_len: int | None = None,
            softmax_scale: float | None = None, v_pos: str = "logical", out: torch.Tensor | None = None,
            lse: torch.Tensor | None = None, out32: torch.Tensor | None = None):
    """Chunked-prefill attention read from the compact pool (one kernel).

    query (Tq, Hq, D) fp16: sequence b's chunk is rows query_start[b] ..
    query_start[b + 1] - 1, the last tokens of its seq_lens[b], already
    written to the pool (write_kv); each query attends causally to every
    earlier token of its sequence and to itself. Returns (out (Tq, Hq, D)
    fp16, lse (Tq, Hq) fp32 natural log); ``out32`` (Tq, Hq, D) fp32, when
    given, receives the output before its fp16 rounding. The reference's prefill reads
    vLLM's fp16 cache instead (src/kvquant/compact_backend.py:12-15).
    """
    dev = pool.device
    q = query.to(device=dev, dtype=torch.float16).contiguous()
    Tq, Hq, D = q.shape
    H = pool.num_kv_heads
    if Hq % H:
        raise ValueError("query heads must be a multiple of KV heads")
    qs = _i32(query_start, dev)
    bt = _i32(block_table, dev)
    sl = _i32(seq_lens, dev)
    B = qs.shape[0] - 1
    if max_query_len is None:
        max_query_len = int((qs[1:] - qs[:-1]).max().item()) if B > 0 else 0
    scale = float(softmax_scale if softmax_scale is not None else 1.0 / math.sqrt(D))
    if out is None:
        out = torch.empty((Tq, Hq, D), dtype=torch.float16, device=dev)
    if lse is None:
        lse = torch.empty((Tq, Hq), dtype=torch.float32, device=dev)
    st_scales, _keep = pool.scales.device_layer(layer_idx, dev)
    with torch.cuda.device(dev):
        call("hx_prefill_attn", stream(dev), ctypes_ref(pool.layers[layer_idx].struct), ctypes_ref(st_scales),
             ptr(q), ptr(qs), B, Hq // H, scale, ptr(bt), bt.shape[1], ptr(sl), int(max_query_len),
             hxlib.VPOS_PHYSICAL if v_pos == "physical" else 0, ptr(out), ptr(out32), ptr(lse),
             ptr(hxlib.err_word(dev)))
    return out, lse


def shared_prefix_decode(pool: CompactKVPool, layer_idx: int, query: torch.Tensor, block_table: torch.Tensor,
                         seq_lens: torch.Tensor, prefix_len: int, *, softmax_scale: float | None = None,
                         v_pos: str = "logical", n_splits: int | None = None, out: torch.Tensor | None = None,
                         lse: torch.Tensor | None = None):
    """Decode attention of a batch whose sequences share a prefix (two kernels).

    query (B, Hq, 128) fp16, one token per sequence; block_table (B, max_pages)
    and seq_lens (B,) as for ``decode``, with the first prefix_len / 16 entries
    of every row naming the same pool pages (read from the first row with
    tokens). ``prefix_len`` is
    a host number of tokens, a multiple of the page size. The prefix's pages
    are read and dequantised once for up to 2 * floor(128 / group) sequences
    (again for each further block of so many) and meet all their query rows in
    matrix products on the tensor cores; each sequence's own pages follow, and
    the parts are joined by their (maximum, sum). Every page is attended (no
    Quest selection): ``decode`` without a selection, except that the
    probabilities enter the product with V as fp16 (``decode`` keeps 22 bits) and
    the output is fp16. A sequence's own pages go to one CTA a KV head, at
    1.6 us a 128 tokens: it pays where the prefix is long and the rest short (8
    sequences behind 2K tokens with 8K of their own: 118 us against decode's 70;
    behind 32K, 137 against 201). A sequence of
    length 0 is a padding row (out 0, lse -inf). Returns (out (B, Hq, D) fp16,
    lse (B, Hq) fp32 natural log).
    """
    dev = pool.device
    if query.dim() != 3:
        raise ValueError(f"query should be (B, Hq, D), got {tuple(query.shape)}")
    if v_pos not in ("logical", "physical"):
        raise ValueError("v_pos must be 'logical' or 'physical'")
    q = query.to(device=dev, dtype=torch.float16).contiguous()
    if q.data_ptr() % 16:
        q = q.clone()
    B, Hq, D = q.shape
    H, S = pool.num_kv_heads, pool.block_size
    if Hq % H or Hq == 0:
        raise ValueError("query heads must be a multiple of KV heads")
    if block_table.dim() != 2 or block_table.shape[0] < B or seq_lens.shape != (B,):
        raise ValueError(f"block_table {tuple(block_table.shape)} and seq_lens {tuple(seq_lens.shape)} should have a row "
                         f"for each of {B} sequences")
    prefix_len = int(prefix_len)
    if prefix_len < 0 or prefix_len % S or prefix_len // S > block_table.shape[1]:
        raise ValueError(f"prefix_len must be a multiple of {S} within the block table, got {prefix_len}")
    bt = _i32(block_table, dev)
    sl = _i32(seq_lens, dev)
    scale = float(softmax_scale if softmax_scale is not None else 1.0 / math.sqrt(D))
    if out is None:
        out = q.new_empty((B, Hq, D))
    elif out.shape != q.shape or out.dtype != torch.float16 or out.device != q.device or not out.is_contiguous() \
            or out.data_ptr() % 8:
        raise ValueError(f"out must be a contiguous {tuple(q.shape)} float16 tensor on {dev}")
    if lse is None:
        lse = q.new_empty((B, Hq), dtype=torch.float32)
    elif lse.shape != (B, Hq) or lse.dtype != torch.float32 or lse.device != q.device or not lse.is_contiguous():
        raise ValueError(f"lse must be a contiguous {(B, Hq)} float32 tensor on {dev}")
    L = hxlib.lib()
    i = q.device.index
    ns = int(n_splits) if n_splits is not None else L.hx_prefix_splits(B, H, Hq // H, prefix_len // S)
    # from torch's allocator, so calls on different streams or in different captured graphs never share it
    scr = q.new_empty(max(16, L.hx_prefix_scratch_bytes(B, H, Hq // H, ns)), dtype=torch.uint8)
    st_scales, _keep = pool.scales.device_layer(layer_idx, dev)
    with hxlib.on(i):
        call("hx_prefix_decode", hxlib.raw_stream(i), ctypes_ref(pool.layers[layer_idx].struct), ctypes_ref(st_scales),
             q.data_ptr(), B, Hq // H, scale, bt.data_ptr(), bt.shape[1], sl.data_ptr(), prefix_len // S,
             hxlib.VPOS_PHYSICAL if v_pos == "physical" else 0, ns, scr.data_ptr(), out.data_ptr(), lse.data_ptr(),
             hxlib.err_ptr(i))
    return out, lse


_PROMPT_DT = {torch.float16: 1, torch.bfloat16: 2}


def _rows(t: torch.Tensor):
    """A (T, heads, D) tensor and its token and head strides as hx_prompt_attn
    takes them; a copy where the layout does not fit (16-byte rows)."""
    T, n, D = t.shape
    st, sh, sd = t.stride()
    if sd != 1 or t.data_ptr() % 16 or (T > 1 and (st < D or st % 8)) or (n > 1 and (sh < D or sh % 8)):
        t = t.contiguous()
        st, sh, _ = t.stride()
        if t.data_ptr() % 16:
            t = t.clone()
    return t, (st if T > 1 else n * D), (sh if n > 1 else D)


def prompt_attention(query: torch.Tensor, key: torch.Tensor, value: torch.Tensor, query_start: torch.Tensor, *,
                     softmax_scale: float | None = None, out: torch.Tensor | None = None,
                     lse: torch.Tensor | None = None):
    """Causal attention over whole prompts at full precision (one kernel).

    query (T, Hq, D), key and value (T, H, D), fp16 or bf16, D 64 or 128, Hq =
    group * H: B prompts back to back, prompt b's tokens are rows
    query_start[b] .. query_start[b + 1] - 1 (query_start (B + 1,) int32 on the
    device, as paging.extend_tables makes it). Each token attends to its
    prompt's tokens up to itself. The three may be slices of one projection
    (last dimension contiguous, strides of 16 bytes; other layouts are
    copied). Returns (out (T, Hq, D) in the input type, lse (T, Hq) fp32 natural
    log); rows past the last prompt are not written. ``out`` may be ``query``
    itself, and overlaps no other input. ``prefill`` is the same
    attention read back from the pool's quantised pages; here the prompt's own
    K and V, before write_kv packs them, give the unquantised result. K and V
    are read as they are (infinities and NaN of tokens that a row does not see
    do not reach it). Reference: FlashAttention over vLLM's fp16 cache
    (src/kvquant/compact_backend.py:194-205).
    """
    if query.dim() != 3 or key.dim() != 3 or value.shape != key.shape:
        raise ValueError(f"expected (T, Hq, D), (T, H, D), (T, H, D), got {tuple(query.shape)}, {tuple(key.shape)}, "
                         f"{tuple(value.shape)}")
    T, Hq, D = query.shape
    H = key.shape[1]
    if key.shape[0] != T or key.shape[2] != D:
        raise ValueError(f"query {tuple(query.shape)} and key {tuple(key.shape)} differ in tokens or head size")
    if query.dtype not in _PROMPT_DT or key.dtype != query.dtype or value.dtype != query.dtype:
        raise TypeError(f"query, key and value must all be float16 or all bfloat16, got {query.dtype}, {key.dtype}, "
                        f"{value.dtype}")
    if H < 1 or Hq < 1 or Hq % H:
        raise ValueError("query heads must be a multiple of KV heads")
    if query_start.dim() != 1 or query_start.numel() < 1:
        raise ValueError("query_start should be (B + 1,)")
    hxlib.require_cuda(query, key, value, query_start, out, lse)
    dev = query.device
    if key.device != dev or value.device != dev:
        raise ValueError("query, key and value must be on one device")
    scale = float(softmax_scale if softmax_scale is not None else 1.0 / math.sqrt(D))
    inplace = out is not None and out.data_ptr() == query.data_ptr() and out.stride() == query.stride()
    for t in (out, lse):
        if t is not None and (any(hxlib.overlap(t, x) for x in (key, value, query_start))
                              or (hxlib.overlap(t, query) and not (t is out and inplace))):
            raise ValueError("out and lse must not overlap key, value, query_start, or a part of query")
    if out is not None and lse is not None and hxlib.overlap(out, lse):
        raise ValueError("out and lse must not overlap")
    if out is None:
        out = query.new_empty((T, Hq, D))
    elif out.shape != query.shape or out.dtype != query.dtype or out.device != dev or not out.is_contiguous() \
            or out.data_ptr() % 16:
        raise ValueError(f"out must be a contiguous {tuple(query.shape)} {query.dtype} tensor on {dev}")
    if lse is None:
        lse = query.new_empty((T, Hq), dtype=torch.float32)
    elif lse.shape != (T, Hq) or lse.dtype != torch.float32 or lse.device != dev or not lse.is_contiguous():
        raise ValueError(f"lse must be a contiguous {(T, Hq)} float32 tensor on {dev}")
    qs = _i32(query_start, dev)
    q, qt, qh = _rows(query)
    k, kt, kh = _rows(key)
    v, vt, vh = _rows(value)
    i = dev.index
    with hxlib.on(i):
        call("hx_prompt_attn", hxlib.raw_stream(i), _PROMPT_DT[query.dtype], q.data_ptr(), qt, qh, k.data_ptr(), kt, kh,
             v.data_ptr(), vt, vh, qs.data_ptr(), qs.shape[0] - 1, T, H, Hq // H, D, scale, out.data_ptr(),
             lse.data_ptr(), hxlib.err_ptr(i))
    return out, lse


def merge_partials(o_parts: torch.Tensor, lse_parts: torch.Tensor, out16: torch.Tensor | None = None):
    """Merge R shards' normalised (o, lse): (R, N, D), (R, N) -> (N, D), (N,)."""
    R, N, D = o_parts.shape
    dev = o_parts.device
    op = o_parts.to(torch.float32).contiguous()
    lp = lse_parts.to(torch.float32).contiguous()
    o = torch.empty((N, D), dtype=torch.float32, device=dev)
    lse = torch.empty((N,), dtype=torch.float32, device=dev)
    with torch.cuda.device(dev):
        call("hx_merge_partials", stream(dev), ptr(op), ptr(lp), R, N, D, ptr(o), ptr(lse), ptr(out16))
    return o, lse
