"""GPU tests of the block-table kernels against a plain restatement on the
host: whole numbers, equal bit for bit."""
from __future__ import annotations

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def _i32(v):
    return torch.tensor(np.asarray(v), dtype=torch.int32, device="cuda")


def _extend(table, cached, new, free, count, num_tokens, S, refs=None):
    """The rule, one token at a time."""
    table, refs = table.copy(), None if refs is None else refs.copy()
    slots, pos = np.full(num_tokens, -1, np.int64), np.zeros(num_tokens, np.int64)
    start = [0]
    for b, (c, n) in enumerate(zip(cached, new)):
        for j in range(-(-c // S), -(-(c + n) // S)):
            count -= 1
            table[b, j] = free[count]
            if refs is not None:
                refs[free[count]] = 1
        for i in range(n):
            pos[start[-1] + i] = c + i
            slots[start[-1] + i] = int(table[b, (c + i) // S]) * S + (c + i) % S
        start.append(start[-1] + n)
    return table, np.array(start), np.asarray(cached) + np.asarray(new), slots, pos, count, refs


def _truncate(table, lens, keep, free, count, S, refs=None):
    free, refs = free.copy(), None if refs is None else refs.copy()
    keep = np.maximum(np.minimum(keep, lens), 0)
    ent = [int(table[b, j]) for b in range(len(lens)) for j in range(-(-keep[b] // S), -(-lens[b] // S))]
    if refs is not None:
        for p in ent:
            refs[p] -= 1
        last = {p: k for k, p in enumerate(ent)}
        ent = [p for k, p in enumerate(ent) if refs[p] == 0 and last[p] == k]
    for i, p in enumerate(ent):
        free[count + len(ent) - 1 - i] = p
    return keep, count + len(ent), free, refs


def _state(rng, B, cached_max, W, S, spare=40):
    num = B * W + spare
    perm = rng.permutation(num).astype(np.int32)
    cached = rng.integers(0, cached_max + 1, B)
    table = np.full((B, W), -7, np.int32)
    at = 0
    for b in range(B):
        n = -(-int(cached[b]) // S)
        table[b, :n] = perm[at:at + n]
        at += n
    free = np.full(num, -1, np.int32)
    free[:num - at] = perm[at:]
    refs = np.zeros(num, np.int32)
    refs[perm[:at]] = 1
    return table, cached, free, num - at, refs


@pytest.mark.parametrize("B,cached_max,new_max,S", [(1, 0, 1, 16), (1, 16, 1, 16), (3, 50, 40, 16), (64, 700, 1, 16),
                                                     (33, 100, 300, 16), (257, 64, 9, 32), (1500, 20, 5, 1),
                                                     (16384, 3, 2, 16), (5, 0, 9000, 16)])
@pytest.mark.parametrize("shared", [False, True])
def test_extend_then_truncate_match_the_rule(B, cached_max, new_max, S, shared):
    from kvquant import paging
    import hxlib
    rng = np.random.default_rng(B + new_max + S)
    W = -(-(cached_max + new_max) // S) + 1
    table, cached, free, count, refs = _state(rng, B, cached_max, W, S)
    new = rng.integers(0, new_max + 1, B)
    new[-1] = new_max
    pad = 5
    T = int(new.sum()) + pad
    # the table is a view of a wider one: rows apart, the rest untouched
    wide = torch.full((B, W + 3), -9, dtype=torch.int32, device="cuda")
    wide[:, :W] = _i32(table)
    g = wide[:, :W]
    gf, gc, gr = _i32(free), _i32([count]), _i32(refs) if shared else None
    out = paging.extend_tables(g, _i32(cached), _i32(new), gf, gc, num_tokens=T, page_size=S, page_refs=gr,
                               num_pages=len(free))
    wt, ws, wl, wslot, wpos, wc, wr = _extend(table, cached, new, free, count, T, S, refs if shared else None)
    hxlib.check_device_errors()
    assert np.array_equal(g.cpu().numpy(), wt) and bool((wide[:, W:] == -9).all())
    for got, want in ((out.query_start, ws), (out.seq_lens, wl), (out.slot_mapping, wslot), (out.positions, wpos),
                      (out.free_count, [wc]), (gf, free), (gc, [count])):
        assert np.array_equal(got.cpu().numpy(), want)
    if shared:
        assert np.array_equal(gr.cpu().numpy(), wr)
    keep = rng.integers(0, cached_max + new_max + 2, B)
    lens, left = paging.truncate_tables(g, out.seq_lens, _i32(keep), gf, out.free_count, page_size=S, page_refs=gr,
                                        num_pages=len(free))
    hxlib.check_device_errors()
    kl, kc, kf, kr = _truncate(wt, wl, keep, free, wc, S, wr)
    assert np.array_equal(lens.cpu().numpy(), kl) and int(left) == kc
    assert np.array_equal(gf.cpu().numpy(), kf)
    if shared:
        assert np.array_equal(gr.cpu().numpy(), kr)


def test_truncate_undoes_extend():
    from kvquant import paging
    rng = np.random.default_rng(5)
    table, cached, free, count, refs = _state(rng, 40, 90, 20, 16)
    g, gf, gc, gr = _i32(table), _i32(free), _i32([count]), _i32(refs)
    new = _i32(rng.integers(0, 100, 40))
    out = paging.extend_tables(g, _i32(cached), new, gf, gc, num_tokens=4000, page_refs=gr)
    lens, left = paging.truncate_tables(g, out.seq_lens, _i32(cached), gf, out.free_count, page_refs=gr)
    assert np.array_equal(gf.cpu().numpy(), free) and int(left) == count
    assert np.array_equal(lens.cpu().numpy(), cached) and np.array_equal(gr.cpu().numpy(), refs)


def test_shared_pages_come_back_with_their_last_reference():
    """Four sequences on one 30-page prefix plus their own pages: the first two
    released give back their own pages only; the last two, released in one
    call, give back every prefix page once."""
    from kvquant import paging
    import hxlib
    S, pre, own = 16, 30, 3
    num = pre + 4 * own + 10
    rng = np.random.default_rng(9)
    perm = rng.permutation(num).astype(np.int32)
    table = np.concatenate([np.tile(perm[:pre], (4, 1)), perm[pre:pre + 4 * own].reshape(4, own)], 1)
    refs = np.zeros(num, np.int32)
    refs[perm[:pre]], refs[perm[pre:pre + 4 * own]] = 4, 1
    free = np.full(num, -1, np.int32)
    free[:10] = perm[-10:]
    lens = np.full(4, (pre + own) * S)
    g, gf, gr, count = _i32(table), _i32(free), _i32(refs), 10
    gl, gc = _i32(lens), _i32([count])
    for keep in ([0, 0, 9999, 9999], [0, 0, 0, 0]):
        gl2, gc = paging.truncate_tables(g, gl, _i32(keep), gf, gc, page_refs=gr)
        lens2, count, free, refs = _truncate(table, gl.cpu().numpy(), np.array(keep), free, count, S, refs)
        gl = gl2
        assert np.array_equal(gl.cpu().numpy(), lens2) and int(gc) == count
        assert np.array_equal(gf.cpu().numpy(), free) and np.array_equal(gr.cpu().numpy(), refs)
    hxlib.check_device_errors()
    assert count == num and sorted(free.tolist()) == list(range(num))


def test_the_same_row_released_twice_is_an_error_and_frees_once():
    from kvquant import paging
    import hxlib
    g, gr = _i32([[3, 1], [3, 1]]), _i32([0, 1, 0, 1])
    gf, gc = _i32([0, 2, -1, -1]), _i32([2])
    lens, left = paging.truncate_tables(g, _i32([32, 32]), _i32([0, 0]), gf, gc, page_refs=gr)
    with pytest.raises(hxlib.HelixError, match="out of range"):
        hxlib.check_device_errors()
    assert int(left) == 4 and sorted(gf.tolist()) == [0, 1, 2, 3] and gr.tolist() == [0, 0, 0, 0]


@pytest.mark.parametrize("what,error", [("pages", "too few free pages"), ("rows", "out of range"),
                                        ("tokens", "out of range"), ("negative", "out of range")])
def test_extend_that_cannot_be_served_hands_out_nothing(what, error):
    from kvquant import paging
    import hxlib
    rng = np.random.default_rng(2)
    table, cached, free, count, refs = _state(rng, 6, 40, 8, 16)
    new, T = np.full(6, 17), 6 * 17
    if what == "pages":
        count = 3
    elif what == "rows":
        new[2] = 8 * 16 + 1 - cached[2]
        T = int(new.sum())
    elif what == "tokens":
        T -= 1
    else:
        new[4] = -1
    g, gr = _i32(table), _i32(refs)
    out = paging.extend_tables(g, _i32(cached), _i32(new), _i32(free), _i32([count]), num_tokens=T, page_refs=gr)
    with pytest.raises(hxlib.HelixError, match=error):
        hxlib.check_device_errors()
    assert np.array_equal(g.cpu().numpy(), table) and np.array_equal(gr.cpu().numpy(), refs)
    assert bool((out.slot_mapping == -1).all()) and int(out.free_count) == count
    assert np.array_equal(out.seq_lens.cpu().numpy(), cached) and bool((out.query_start == 0).all())


def test_captured_step_loop_and_empty_batch():
    """A decode step captured once and replayed: lengths and the free count
    carried on inside the graph; then a batch without sequences."""
    from kvquant import paging
    B, W, S = 7, 6, 16
    g = torch.full((B, W), -1, dtype=torch.int32, device="cuda")
    lens, count = _i32([0] * B), _i32([B * W])
    free, one = _i32(np.arange(B * W)), _i32([1] * B)
    out = paging.extend_tables(g, lens, one, free, count, num_tokens=B + 2)   # warm-up outside the capture
    lens.zero_()
    count.fill_(B * W)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        paging.extend_tables(g, lens, one, free, count, num_tokens=B + 2, out=out)
        lens.copy_(out.seq_lens)
        count.copy_(out.free_count)
    for step in range(40):
        graph.replay()
        want = g[:, step // S].long() * S + step % S
        assert torch.equal(out.slot_mapping[:B], want) and bool((out.positions[:B] == step).all())
        assert out.slot_mapping[B:].tolist() == [-1, -1]
    assert int(count) == B * W - 3 * B and lens.tolist() == [40] * B
    e = paging.extend_tables(g[:0], lens[:0], one[:0], free, count, num_tokens=3)
    assert e.query_start.tolist() == [0] and e.slot_mapping.tolist() == [-1] * 3 and int(e.free_count) == int(count)


def test_reset_allocated_empties_the_new_pages():
    from helpers import gpu_outlier_sets
    from kvquant import paging
    from kvquant.compact_pool import CompactKVPool
    from kvquant.synthetic import NUQ4, make_kv, make_scales
    H, D, S, NB = 2, 128, 16, 12
    sc = make_scales([NUQ4], H, D, t_cal=64, seed=1)
    pool = CompactKVPool(1, NB, S, H, D, sc)
    K, V = make_kv(NB * S, H, D, seed=2, chan_seed=1, outlier_frac=0.05)
    at = torch.arange(NB * S, device="cuda")
    pool.write_kv(0, K, V, at, at)
    g, free, count = torch.full((2, 4), -1, dtype=torch.int32, device="cuda"), _i32(np.arange(NB)), _i32([9])
    before = pool.k_min.clone()
    out = paging.extend_tables(g, _i32([0, 0]), _i32([20, 50]), free, count, num_tokens=70)
    pool.reset_allocated(0, free, count, out.free_count)
    pool.check()
    taken = sorted(range(9))[-6:]
    assert int(out.free_count) == 3
    lists = gpu_outlier_sets(pool, 0)
    assert all(b not in taken for (_, b, _) in lists) and any(b not in taken for (_, b, _) in lists)
    now = pool.k_min[0]
    assert bool(torch.isinf(now[taken]).all())
    rest = [b for b in range(NB) if b not in taken]
    assert torch.equal(now[rest], before[0][rest])
