"""Workloads of the batch-serving operators around the compact KV pool.

Three operators are timed and compared here, each in a plain form of elementary
torch operations and through the framework's entry points:

  tables  ``kvquant.paging.extend_tables`` / ``truncate_tables``: block tables,
          slot map, positions and query offsets of a batch from its requests'
          lengths, with pages taken from a free stack and given back to it
  prompt  ``kvquant.fused.prompt_attention``: causal attention over whole
          prompts of different lengths packed back to back, grouped heads
  prefix  ``kvquant.fused.shared_prefix_decode``: one decode token per sequence
          of a batch whose sequences share a long prefix of pool pages; the
          prefix's codes are read and dequantised once for the whole batch

Model shapes are those of the framework's benchmark (28 query heads on 4 KV
heads, head size 128, 16-token pages, nuq2 / nuq4 codes with 5% / 1% outliers,
t_cal 4096); the 64-wide head with one query head per KV head stands for
smaller models.
"""
from __future__ import annotations

import math
import os
import sys

import torch

own = False

PAGE = 16
DEV = "cuda"
T_CAL = 4096


def _package():
    """The framework's packages, as a program beside the repository imports them."""
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "helix-lite_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    from kvquant import fused, paging
    return fused, paging


# ---- cases ---------------------------------------------------------------------

def _tables(name, batch, cached, shortest, longest, shared):
    return {"name": name, "op": "tables", "batch": batch, "cached": cached, "shortest": shortest, "longest": longest,
            "shared": shared}


def _prompt(name, batch, shortest, longest, heads, kv_heads, dim, kind):
    return {"name": name, "op": "prompt", "batch": batch, "shortest": shortest, "longest": longest, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "type": kind}


def _prefix(name, batch, prefix, suffix, bits_k, bits_v, group=7):
    return {"name": name, "op": "prefix", "batch": batch, "prefix": prefix, "suffix": suffix, "bits_k": bits_k,
            "bits_v": bits_v, "group": group}


def listed():
    return [
        # a decode step: 64 sequences of up to 32K cached tokens, one new token each; prefix pages shared
        _tables("tables-decode-64", 64, 32768, 1, 1, True),
        # verification of drafted tokens: 256 sequences, up to 8 tokens each, rejected ones given back
        _tables("tables-drafts-256", 256, 16384, 1, 8, False),
        # admission of 64 fresh prompts of up to 8K tokens
        _tables("tables-prompts-64", 64, 0, 1, 8192, False),
        # the smallest prompts: a few tokens each, latency alone
        _prompt("prompt-few-tokens", 16, 1, 8, 28, 4, 128, "fp16"),
        # a prefill batch of short, ragged chat prompts
        _prompt("prompt-ragged-64", 64, 1, 1021, 28, 4, 128, "fp16"),
        # a smaller model without grouped heads, head size 64
        _prompt("prompt-d64-mha", 4, 1000, 4001, 16, 16, 64, "bf16"),
        # one 8K prompt
        _prompt("prompt-8k", 1, 8192, 8192, 28, 4, 128, "bf16"),
        # one long prompt of an odd length
        _prompt("prompt-20k", 1, 20011, 20011, 28, 4, 128, "fp16"),
        # four sequences on a 2K system prompt
        _prefix("prefix-2k-4", 4, 2048, 64, 4, 4),
        # a full batch answering questions about one 32K document
        _prefix("prefix-32k-64", 64, 32768, 512, 4, 4),
        # 16 sequences on a 128K document in a nuq2 layer
        _prefix("prefix-128k-16", 16, 131072, 777, 2, 2),
        # 8 sequences on the benchmark's 1M-token context
        _prefix("prefix-1m-8", 8, 1048576, 300, 4, 4),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["tables", "prompt", "prefix"])
    if op == "tables":
        batch = _log(rng, 1, 512)
        cached = rng.choice([0, _log(rng, 1, 32768)])
        longest = _log(rng, 1, max(2, 400000 // batch // 2))
        c = _tables("", batch, cached, rng.choice([0, 1]), min(longest, 16384), rng.random() < 0.5)
    elif op == "prompt":
        heads, kv_heads, dim = rng.choice([(28, 4, 128), (32, 8, 128), (16, 16, 64), (14, 2, 64), (8, 1, 128)])
        batch = _log(rng, 1, 64)
        longest = _log(rng, 1, 16000 / math.sqrt(batch))
        c = _prompt("", batch, rng.choice([0, 1, longest]), longest, heads, kv_heads, dim, rng.choice(["fp16", "bf16"]))
    else:
        prefix = PAGE * _log(rng, 8, 32768)
        batch = _log(rng, 1, max(2, min(80, 4000000 // prefix)))
        c = _prefix("", batch, prefix, _log(rng, 1, 700), rng.choice([2, 4]), rng.choice([2, 4]), rng.choice([1, 4, 7, 8]))
    del c["name"]
    return c


def _lengths(n, shortest, longest):
    """n lengths spread over shortest .. longest (both met when n > 1), the same for every seed."""
    if n == 1:
        return [longest]
    inner = [shortest + int((longest - shortest + 1) * ((i * 0.6180339887498949) % 1.0)) for i in range(1, n - 1)]
    return [longest] + inner + [shortest]


def _cdiv(a, b):
    return -(-a // b)


def _tables_lengths(case):
    b = case["batch"]
    return _lengths(b, 0, case["cached"]) if case["cached"] else [0] * b, _lengths(b, case["shortest"], case["longest"])


def _outlier_cap(bits):
    # entries a (head, page) list of 2048 elements may hold: 5% of them at nuq2, 1% at nuq4, with room
    return 128 if bits == 2 else 32


def work(case):
    if case["op"] == "tables":
        cached, new = _tables_lengths(case)
        tokens = sum(new)
        pages = sum(_cdiv(c + n, PAGE) - _cdiv(c, PAGE) for c, n in zip(cached, new))
        # lengths in and out, the free stack's entries read and given back, table entries written, 16 bytes a token,
        # a reference count per page on either way
        return {"bytes": 6 * 4 * case["batch"] + 4 * 4 * pages + 16 * tokens + (16 * pages if case["shared"] else 0),
                "flops": 0}
    if case["op"] == "prompt":
        lens = _lengths(case["batch"], case["shortest"], case["longest"])
        t = sum(lens)
        hq, h, d = case["heads"], case["kv_heads"], case["dim"]
        return {"bytes": 2 * t * d * (2 * hq + 2 * h) + 4 * t * hq, "flops": 4 * d * hq * sum(n * (n + 1) // 2 for n in lens)}
    h, d, g = 4, 128, case["group"]
    suf = _lengths(case["batch"], 1, case["suffix"])
    pages = case["prefix"] // PAGE + sum(_cdiv(s, PAGE) for s in suf)
    page = PAGE * d * (case["bits_k"] + case["bits_v"]) // 8 + 32
    page += 4 * 3 * (_outlier_cap(case["bits_k"]) + _outlier_cap(case["bits_v"])) // 4
    rows = case["batch"] * h * g
    return {"bytes": h * pages * page + rows * (4 * d + 4), "flops": 4 * d * h * g * sum(case["prefix"] + s for s in suf)}


# ---- inputs ---------------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def prepare(case, seed):
    return {"tables": _prepare_tables, "prompt": _prepare_prompt, "prefix": _prepare_prefix}[case["op"]](case, seed)


def _prepare_tables(case, seed):
    """Cached sequences on pages in random order, a free stack with the rest. With ``shared``, the first half of every
    table's cached pages is the longest sequence's (reference-counted), as prefix sharing leaves them."""
    g = _gen(seed)
    cached, new = _tables_lengths(case)
    b = case["batch"]
    order = torch.randperm(b, generator=g, device=DEV)
    cached, new = _i32(cached)[order], _i32(new)[order]
    width = _cdiv(case["cached"] + case["longest"], PAGE) + 8
    have = (cached + PAGE - 1) // PAGE
    num_pages = b * width + 64
    perm = torch.randperm(num_pages, generator=g, device=DEV).to(torch.int32)
    table = perm[:b * width].view(b, width).clone()
    col = torch.arange(width, device=DEV)
    refs = None
    if case["shared"]:
        row = table[torch.argmax(have)]
        table = torch.where(col[None] < (have // 2)[:, None], row[None], table)
        refs = torch.zeros(num_pages, dtype=torch.int32, device=DEV)
        used = col[None] < have[:, None]
        refs.index_add_(0, table[used].long(), torch.ones(int(used.sum()), dtype=torch.int32, device=DEV))
    held = torch.zeros(num_pages, dtype=torch.bool, device=DEV)
    held[table[col[None] < have[:, None]].long()] = True
    table = torch.where(col[None] < have[:, None], table, -1).contiguous()
    free = perm[~held[perm.long()]]
    stack = torch.full((num_pages,), -1, dtype=torch.int32, device=DEV)
    stack[:free.numel()] = free
    return {"op": "tables", "table": table, "cached": cached, "new": new, "free": stack, "count": _i32([free.numel()]),
            "refs": refs, "num_tokens": int(new.sum())}


def _prepare_prompt(case, seed):
    """q, k and v as a model's fused projection leaves them: slices of one (tokens, heads) matrix; per-channel scales."""
    g = _gen(seed)
    lens = _lengths(case["batch"], case["shortest"], case["longest"])
    t, hq, h, d = sum(lens), case["heads"], case["kv_heads"], case["dim"]
    dt = torch.float16 if case["type"] == "fp16" else torch.bfloat16
    chan = torch.exp(torch.empty(hq + 2 * h, d, device=DEV).uniform_(-0.7, 0.7, generator=g))
    qkv = (torch.randn(t, hq + 2 * h, d, generator=g, device=DEV) * chan).to(dt)
    order = torch.randperm(case["batch"], generator=g, device=DEV)
    start = torch.zeros(case["batch"] + 1, dtype=torch.int32, device=DEV)
    start[1:] = torch.cumsum(_i32(lens)[order], 0)
    return {"op": "prompt", "q": qkv[:, :hq], "k": qkv[:, hq:hq + h], "v": qkv[:, hq + h:], "start": start,
            "longest": case["longest"]}


def _prepare_prefix(case, seed):
    """A layer of the compact pool: packed codes, sparse outliers, per-channel K and per-token V codebooks; a batch whose
    block tables share their first pages (pool pages in random order)."""
    g = _gen(seed)
    h, d, b = 4, 128, case["batch"]
    bk, bv = case["bits_k"], case["bits_v"]
    suf = _lengths(b, 1, case["suffix"])
    n_pre, width = case["prefix"] // PAGE, _cdiv(case["suffix"], PAGE)
    nb = n_pre + b * width + 5
    z = {n: torch.special.ndtri((torch.arange(n, device=DEV, dtype=torch.float64) + 0.5) / n).float() for n in (4, 16)}
    ks = torch.exp(torch.empty(h, d, device=DEV).uniform_(-1.2, 0.7, generator=g))
    vs = torch.exp(torch.empty(h, T_CAL, device=DEV).uniform_(-0.3, 0.3, generator=g))
    k_poles = (ks[..., None] * z[1 << bk]).half()
    v_poles = (vs[..., None] * z[1 << bv]).half()
    seg = PAGE * d * (bk + bv) // 8
    codes = torch.randint(0, 1 << 62, (h * nb * seg // 8,), generator=g, device=DEV, dtype=torch.int64).view(torch.uint8)
    codes = codes.view(h, nb, seg)
    # outlier lists: one entry at a random place of each of `cap` strata of the page, the first `cnt` of them kept
    offs, cnts, arena, top = [], [], [], 0
    for cap, scale in ((_outlier_cap(bk), ks), (_outlier_cap(bv), None)):
        cnt = torch.randint(cap // 2, cap + 1, (h, nb), generator=g, device=DEV)
        width_s = PAGE * d // cap
        at = torch.arange(cap, device=DEV) * width_s + torch.randint(0, width_s, (h, nb, cap), generator=g, device=DEV)
        slot, ch = at // d, at % d
        val = torch.randn((h, nb, cap), generator=g, device=DEV) * 3.0
        if scale is not None:
            val = val * torch.gather(scale[:, None].expand(h, nb, d), 2, ch)
        bits = val.half().view(torch.int16).int() & 0xFFFF
        arena.append((bits | (ch.int() << 16) | (slot.int() << 24)).reshape(-1))
        offs.append(top + torch.arange(h * nb, device=DEV).view(h, nb) * cap)
        cnts.append(cnt)
        top += h * nb * cap
    caps = [torch.full((h, nb), c, device=DEV) for c in (_outlier_cap(bk), _outlier_cap(bv))]
    rows = torch.full((h, nb), PAGE, device=DEV)
    directory = torch.stack([torch.stack([offs[i], caps[i], cnts[i], rows], -1) for i in range(2)], 2).int().contiguous()
    perm = torch.randperm(nb, generator=g, device=DEV).int()
    table = torch.cat([perm[:n_pre].expand(b, n_pre), perm[n_pre:n_pre + b * width].view(b, width)], 1).contiguous()
    order = torch.randperm(b, generator=g, device=DEV)
    seq_lens = (case["prefix"] + _i32(suf)[order]).int()
    q = torch.randn((b, h * case["group"], d), generator=g, device=DEV)
    q = (q / ks.repeat_interleave(case["group"], 0).clamp(min=0.7)).half()
    s = {"op": "prefix", "codes": codes, "dir": directory, "arena": torch.cat(arena), "k_poles": k_poles,
         "v_poles": v_poles, "bits": (bk, bv), "table": table, "seq_lens": seq_lens, "q": q, "prefix": case["prefix"]}
    if own:
        s["pool"] = _pool(s)
    return s


def _pool(s):
    """The pool handle that a user's program keeps, holding the same packed layer."""
    _package()
    from kvquant.compact_pool import CompactKVPool
    from kvquant.scales import KVScales, PerChannelScale, PerTokenScale
    h, nb, _ = s["codes"].shape
    d = s["k_poles"].shape[1]
    kp, vp = s["k_poles"], s["v_poles"]
    sc = KVScales([PerChannelScale(kp, kp[..., -1], kp[..., 0], s["bits"][0])],
                  [PerTokenScale(vp, vp[..., -1], vp[..., 0], s["bits"][1])])
    pool = CompactKVPool(1, nb, PAGE, h, d, sc, device=s["codes"].device, outlier_capacity=s["arena"].numel())
    lay = pool.layers[0]
    lay.codes.copy_(s["codes"])
    lay.dir.copy_(s["dir"])
    lay.arena.copy_(s["arena"])
    lay.arena_top.fill_(s["arena"].numel())
    return pool


# ---- one pass ---------------------------------------------------------------------

def run(state):
    return {"tables": _run_tables, "prompt": _run_prompt, "prefix": _run_prefix}[state["op"]](state)


def _run_tables(s):
    """A step's tables, then the step's tokens given back (a rejected draft): the free stack ends as it began."""
    if own:
        _, paging = _package()
        t = paging.extend_tables(s["table"], s["cached"], s["new"], s["free"], s["count"], num_tokens=s["num_tokens"],
                                 page_size=PAGE, page_refs=s["refs"])
        lens, count = paging.truncate_tables(s["table"], t.seq_lens, s["cached"], s["free"], t.free_count,
                                             page_size=PAGE, page_refs=s["refs"])
        out = [t.query_start, t.seq_lens, t.slot_mapping, t.positions, t.free_count, lens, count]
    else:
        out = _plain_extend(s) + _plain_truncate(s)
    return out + [s["table"], s["free"]] + ([] if s["refs"] is None else [s["refs"]])


def _plain_extend(s):
    table, cached, new, free, refs = s["table"], s["cached"].long(), s["new"].long(), s["free"], s["refs"]
    b, width = table.shape
    have, need = (cached + PAGE - 1) // PAGE, (cached + new + PAGE - 1) // PAGE
    first = torch.cumsum(need - have, 0) - (need - have)
    col = torch.arange(width, device=DEV)[None]
    fresh = (col >= have[:, None]) & (col < need[:, None])
    place = s["count"].long() - 1 - (first[:, None] + col - have[:, None])
    page = free[torch.where(fresh, place, 0)]
    table.copy_(torch.where(fresh, page, table))
    if refs is not None:
        mark = torch.zeros(refs.numel() + 1, dtype=torch.int32, device=DEV)
        mark[torch.where(fresh, page, refs.numel()).long()] = 1
        refs.copy_(torch.where(mark[:-1] > 0, mark[:-1], refs))
    start = torch.zeros(b + 1, dtype=torch.int64, device=DEV)
    start[1:] = torch.cumsum(new, 0)
    tok = torch.arange(s["num_tokens"], device=DEV)
    seq = torch.searchsorted(start[1:].contiguous(), tok, right=True).clamp(max=b - 1)
    pos = cached[seq] + tok - start[seq]
    slot = table[seq, pos // PAGE].long() * PAGE + pos % PAGE
    s["lens"] = (cached + new).int()
    s["left"] = s["count"] - (need - have).sum().int()
    return [start.int(), s["lens"], slot, pos, s["left"]]


def _plain_truncate(s):
    table, lens, keep, free, refs = s["table"], s["lens"].long(), s["cached"].long(), s["free"], s["refs"]
    b, width = table.shape
    keep = torch.minimum(keep, lens)
    col = torch.arange(width, device=DEV)[None]
    dropped = ((col >= ((keep + PAGE - 1) // PAGE)[:, None]) & (col < ((lens + PAGE - 1) // PAGE)[:, None])).view(-1)
    page = torch.where(dropped, table.view(-1), free.numel()).long()
    if refs is not None:
        left = torch.zeros(refs.numel() + 1, dtype=torch.int32, device=DEV)
        left[:-1] = refs
        left.index_add_(0, page, torch.full_like(page, -1, dtype=torch.int32))
        refs.copy_(left[:-1])
        entry = torch.arange(b * width, device=DEV)
        last = torch.full((refs.numel() + 1,), -1, dtype=torch.int64, device=DEV).scatter_reduce_(0, page, entry, "amax")
        dropped = dropped & (left[page] == 0) & (last[page] == entry)
    rank = torch.cumsum(dropped, 0) - 1
    total = dropped.sum()
    stack = torch.cat([free, free[:1]])
    stack[torch.where(dropped, s["left"].long() + total - 1 - rank, free.numel())] = torch.where(dropped, table.view(-1), free[0])
    free.copy_(stack[:-1])
    return [keep.int(), s["left"] + total.int()]


def _run_prompt(s):
    if own:
        fused, _ = _package()
        return list(fused.prompt_attention(s["q"], s["k"], s["v"], s["start"]))
    q, k, v, start, longest = s["q"], s["k"], s["v"], s["start"].long(), s["longest"]
    t, hq, d = q.shape
    h = k.shape[1]
    b = start.numel() - 1
    # padded (batch, heads, longest, dim) in 32 bits; blocks of queries bound the scores' memory
    tok = start[:-1, None] + torch.arange(longest, device=DEV)[None]
    inside = tok < start[1:, None]
    tok = torch.where(inside, tok, 0)
    qp = q[tok].float().view(b, longest, h, hq // h, d).permute(0, 2, 3, 1, 4)
    kp = k[tok].float().permute(0, 2, 3, 1).contiguous()
    vp = v[tok].float().permute(0, 2, 1, 3).contiguous()
    out = torch.empty((t, hq, d), dtype=q.dtype, device=DEV)
    lse = torch.empty((t, hq), dtype=torch.float32, device=DEV)
    step = max(1, min(longest, (1 << 30) // (b * hq * longest)))
    for i in range(0, longest, step):
        e = min(longest, i + step)
        rows = qp[:, :, :, i:e].reshape(b, h, -1, d)
        x = torch.matmul(rows, kp[..., :e]) * (1.0 / math.sqrt(d))
        x = x.view(b, h, hq // h, e - i, e)
        x.masked_fill_(torch.arange(e, device=DEV)[None] > torch.arange(i, e, device=DEV)[:, None], -math.inf)
        m = x.amax(-1, keepdim=True)
        x = x.sub_(m).exp_()
        l = x.sum(-1, keepdim=True)
        o = torch.matmul(x.view(b, h, -1, e), vp[:, :, :e]).view(b, h, hq // h, e - i, d) / l
        ok = inside[:, i:e]
        out[tok[:, i:e][ok]] = o.permute(0, 3, 1, 2, 4).reshape(b, e - i, hq, d)[ok].to(q.dtype)
        lse[tok[:, i:e][ok]] = (m + torch.log(l)).squeeze(-1).permute(0, 3, 1, 2).reshape(b, e - i, hq)[ok]
    return [out, lse]


def _plain_dequant(s, pages, pos, kv):
    """Dequantised K (kv 0) or V (kv 1) of pool pages: (heads, pages * 16, dim) in 32 bits."""
    h, _, seg = s["codes"].shape
    d = s["k_poles"].shape[1]
    bits = s["bits"][kv]
    base = 0 if kv == 0 else PAGE * d * s["bits"][0] // 8
    rows = s["codes"][:, pages, base:base + PAGE * d * bits // 8]
    shift = torch.arange(0, 8, bits, device=DEV, dtype=torch.uint8)
    code = ((rows[..., None] >> shift) & ((1 << bits) - 1)).view(h, -1, PAGE, d).int()
    head = torch.arange(h, device=DEV, dtype=torch.int32)[:, None, None, None]
    if kv == 0:
        row = head * d + torch.arange(d, device=DEV, dtype=torch.int32)
        x = s["k_poles"].float().view(-1)[row * (1 << bits) + code]
    else:
        row = head * T_CAL + pos.clamp(max=T_CAL - 1).int().view(1, -1, PAGE, 1)
        x = s["v_poles"].float().view(-1)[row * (1 << bits) + code]
    del code
    off, cnt = s["dir"][:, pages, kv, 0].long(), s["dir"][:, pages, kv, 2].long()
    slot = torch.arange(_outlier_cap(bits), device=DEV)
    ent = s["arena"][(off[..., None] + slot).clamp(max=s["arena"].numel() - 1)]
    hit = slot < cnt[..., None]
    val = (ent & 0xFFFF).to(torch.int16).view(torch.float16).float()
    page = torch.arange(h * pages.numel(), device=DEV).view(h, -1, 1)
    at = page * (PAGE * d) + ((ent >> 24) & 31) * d + ((ent >> 16) & 255)
    x = x.view(-1)
    x[at[hit]] = val[hit]
    return x.view(h, -1, d)


def _run_prefix(s):
    if own:
        fused, _ = _package()
        return list(fused.shared_prefix_decode(s["pool"], 0, s["q"], s["table"], s["seq_lens"], s["prefix"]))
    q, n = s["q"].float(), s["prefix"]
    b, hq, d = q.shape
    h = s["k_poles"].shape[0]
    g, n_pre = hq // h, n // PAGE
    table = s["table"].long()
    width = table.shape[1] - n_pre
    rows = q.view(b, h, g, d)
    pos = torch.arange(n, device=DEV)
    tail = n + torch.arange(width * PAGE, device=DEV)
    scale = 1.0 / math.sqrt(d)
    flat = rows.permute(1, 0, 2, 3).reshape(h, b * g, d)
    xp = torch.matmul(flat, _plain_dequant(s, table[0, :n_pre], pos, 0).transpose(1, 2)) * scale
    own_pages = table[:, n_pre:].reshape(-1)
    ks = _plain_dequant(s, own_pages, tail.repeat(b), 0).view(h, b, -1, d)
    xs = torch.matmul(rows.permute(1, 0, 2, 3), ks.transpose(2, 3)) * scale
    xs.masked_fill_((tail[None] >= s["seq_lens"][:, None])[None, :, None], -math.inf)
    xp = xp.view(h, b, g, n)
    m = torch.maximum(xp.amax(-1, keepdim=True), xs.amax(-1, keepdim=True))
    xp, xs = xp.sub_(m).exp_(), xs.sub_(m).exp_()
    l = xp.sum(-1, keepdim=True) + xs.sum(-1, keepdim=True)
    o = torch.matmul(xp.view(h, b * g, n), _plain_dequant(s, table[0, :n_pre], pos, 1)).view(h, b, g, d)
    o = o + torch.matmul(xs, _plain_dequant(s, own_pages, tail.repeat(b), 1).view(h, b, -1, d))
    out = (o / l).permute(1, 0, 2, 3).reshape(b, hq, d).half()
    return [out, (m + torch.log(l)).squeeze(-1).permute(1, 0, 2).reshape(b, hq).contiguous()]


# ---- from the definitions, in 64 bits ----------------------------------------------

def exact(case, seed):
    if case["op"] == "tables":
        return None  # whole numbers only
    s = prepare(case, seed)
    return _exact_prompt(s) if case["op"] == "prompt" else _exact_prefix(s)


def _softmax64(x, v):
    """softmax(x) v and the logarithm of the sum of exponentials, row by row; x (rows, keys), v (keys, dim), 64 bits."""
    z = torch.logsumexp(x, 1)
    return torch.exp(x - z[:, None]) @ v, z


def _exact_prompt(s):
    q, k, v = s["q"], s["k"], s["v"]
    t, hq, d = q.shape
    group = hq // k.shape[1]
    out = torch.zeros((t, hq, d), dtype=torch.float64, device=DEV)
    lse = torch.zeros((t, hq), dtype=torch.float64, device=DEV)
    start = s["start"].tolist()
    for a, e in zip(start[:-1], start[1:]):
        for head in range(hq):
            kh, vh = k[a:e, head // group].double(), v[a:e, head // group].double()
            for i in range(a, e, 8192):
                j = min(e, i + 8192)
                x = q[i:j, head].double() @ kh[:j - a].T / math.sqrt(d)
                seen = torch.arange(a, j, device=DEV)[None] <= torch.arange(i, j, device=DEV)[:, None]
                out[i:j, head], lse[i:j, head] = _softmax64(torch.where(seen, x, -math.inf), vh[:j - a])
    return [out, lse]


def _exact_tokens(s, head, pages, first, kv):
    """Dequantised tokens of one head in 64 bits, level by level: code -> level by comparison, outliers over them."""
    d, bits = s["k_poles"].shape[1], s["bits"][kv]
    begin = 0 if kv == 0 else PAGE * d * s["bits"][0] // 8
    byte = s["codes"][head, pages][:, begin:begin + PAGE * d * bits // 8].reshape(-1, d * bits // 8)
    code = torch.stack([(byte >> (bits * i)) % (1 << bits) for i in range(8 // bits)], 2).reshape(-1, d)
    n = code.shape[0]
    if kv == 0:
        levels = s["k_poles"][head].double()[None]
    else:
        levels = s["v_poles"][head].double()[(first + torch.arange(n, device=DEV)).clamp(max=T_CAL - 1)][:, None]
    x = torch.zeros((n, d), dtype=torch.float64, device=DEV)
    for c in range(1 << bits):
        x += torch.where(code == c, levels[..., c], 0.0)
    rec = s["dir"][head, pages, kv].long()
    own_page = torch.repeat_interleave(torch.arange(pages.numel(), device=DEV), rec[:, 2])
    nth = torch.arange(own_page.numel(), device=DEV) - (torch.cumsum(rec[:, 2], 0) - rec[:, 2])[own_page]
    ent = s["arena"][rec[own_page, 0] + nth].long() & 0xFFFFFFFF
    x[own_page * PAGE + (ent >> 24), (ent >> 16) & 0xFF] = (ent & 0xFFFF).to(torch.int16).view(torch.float16).double()
    return x


def _exact_prefix(s):
    q = s["q"].double()
    b, hq, d = q.shape
    h, n, n_pre = s["k_poles"].shape[0], s["prefix"], s["prefix"] // PAGE
    g = hq // h
    out, lse = torch.zeros_like(q), torch.zeros((b, hq), dtype=torch.float64, device=DEV)
    for head in range(h):
        pages = s["table"][0, :n_pre].long()
        kp, vp = _exact_tokens(s, head, pages, 0, 0), _exact_tokens(s, head, pages, 0, 1)
        for i, length in enumerate(s["seq_lens"].tolist()):
            tail = s["table"][i, n_pre:_cdiv(length, PAGE)].long()
            k1 = _exact_tokens(s, head, tail, n, 0)[:length - n]
            v1 = _exact_tokens(s, head, tail, n, 1)[:length - n]
            rows = slice(head * g, head * g + g)
            x = torch.cat([q[i, rows] @ kp.T, q[i, rows] @ k1.T], 1) / math.sqrt(d)
            z = torch.logsumexp(x, 1)
            p = torch.exp(x - z[:, None])
            out[i, rows], lse[i, rows] = p[:, :n] @ vp + p[:, n:] @ v1, z
    return [out, lse]
