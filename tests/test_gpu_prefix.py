"""GPU parity of the shared-prefix decode against float64 attention over the
oracle's dequantisation of the same pool.

Tolerance. With e = 2^-19 scale max_j sum_c |q_c k_jc| bounding what fp32
scores (128 exact products, eight accumulations of sixteen, the exponent's
argument) are off by, a probability moves by a factor of at most 1 + 2 e, then
by half an fp16 step u = 2^-11, and the result by half a step: with A the
softmax average of |v|, (u + 2 e + 2^-17) A + u |o|, plus the absolute step of
small fp16 probabilities, n 2^-25 max|v|, and of small outputs, 2^-25. lse moves by
at most e + 2^-18 + |lse| 2^-22.
"""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from helpers import make_pools, np16, write_both

pytestmark = pytest.mark.gpu

S, D = 16, 128


def _build(bits, prefix, suffixes, H=2, t_cal=64, seed=0, v_pos="logical", spare=6):
    """Pools with one prefix and a suffix per sequence on shuffled pages."""
    from kvquant.synthetic import NUQ2, NUQ4, make_kv, make_scales
    lay = {4: NUQ4, 2: NUQ2}
    sc = make_scales([lay[bits[0]]], H, D, t_cal=t_cal, seed=seed)
    if bits[1] != bits[0]:
        sc.per_layer_values = make_scales([lay[bits[1]]], H, D, t_cal=t_cal, seed=seed + 7).per_layer_values
    n_pre = prefix // S
    width = max((-(-s // S) for s in suffixes), default=0)
    nb = n_pre + sum(-(-s // S) for s in suffixes) + spare
    gpu, orc = make_pools(sc, nb, S, H, D)
    rng = np.random.default_rng(seed)
    perm = rng.permutation(nb)
    table = np.full((len(suffixes), n_pre + max(width, 1)), -1, np.int64)
    table[:, :n_pre] = perm[:n_pre]
    at = n_pre

    def write(pages, n, pos0, sd):
        if n == 0:
            return
        K, V = make_kv(n, H, D, seed=sd, outlier_frac=lay[bits[0]][1], chan_seed=seed)
        i = torch.arange(n, device="cuda")
        slots = torch.from_numpy(pages).cuda()[i // S] * S + i % S
        write_both(gpu, orc, 0, K, V, slots, slots if v_pos == "physical" else pos0 + i)

    write(perm[:n_pre], prefix, 0, seed + 1)
    for b, s in enumerate(suffixes):
        m = -(-s // S)
        table[b, n_pre:n_pre + m] = perm[at:at + m]
        write(perm[at:at + m], s, prefix, seed + 2 + b)
        at += m
    return gpu, orc, table


def _check(gpu, orc, table, lens, q, out, lse, scale, v_pos, skip=()):
    q64, H = np16(q).astype(np.float64), gpu.num_kv_heads
    got, gl = np16(out).astype(np.float64), np16(lse).astype(np.float64)
    g = q.shape[1] // H
    for b, n in enumerate(lens):
        if n == 0:
            assert not got[b].any() and np.isneginf(gl[b]).all()
            continue
        if b in skip:
            continue
        K, V = orc.dequant_sequence(0, np.where(table[b] < 0, 0, table[b]), n, v_pos=v_pos)
        K, V = np.asarray(K, np.float64), np.asarray(V, np.float64)
        for h in range(H):
            rows = q64[b, h * g:(h + 1) * g]
            s = rows @ K[:, h].T * scale
            z = np.log(np.exp(s - s.max(1, keepdims=True)).sum(1)) + s.max(1)
            p = np.exp(s - z[:, None])
            o, A = p @ V[:, h], p @ np.abs(V[:, h])
            e = 2.0 ** -19 * scale * (np.abs(rows) @ np.abs(K[:, h]).T).max(1)
            u = 2.0 ** -11
            tol = (u + 2 * e[:, None] + 2.0 ** -17) * A + u * np.abs(o) + n * 2.0 ** -25 * np.abs(V[:, h]).max() + 2.0 ** -25
            err = np.abs(got[b, h * g:(h + 1) * g] - o)
            assert (err <= tol).all(), f"sequence {b} head {h}: {(err - tol).max()} over"
            assert (np.abs(gl[b, h * g:(h + 1) * g] - z) <= e + 2.0 ** -18 + np.abs(z) * 2.0 ** -22).all()


def _q(B, Hq, seed, size=0.5):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn((B, Hq, D), generator=g, device="cuda") * size).half()


def _i32(v):
    return torch.tensor(np.asarray(v), dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("bits", [(4, 4), (2, 2), (4, 2), (2, 4)])
@pytest.mark.parametrize("prefix,suffixes,G", [(16, [1], 1), (128, [1, 16, 17], 7), (1040, [300, 1, 0, 129, 40], 4),
                                               (2048, [5 * i % 67 for i in range(40)], 7), (0, [200, 1, 31], 7),
                                               (384, [0, 0], 8)])
def test_matches_the_formula(bits, prefix, suffixes, G):
    from kvquant import fused
    gpu, orc, table = _build(bits, prefix, suffixes, seed=prefix + G + bits[0])
    lens = [prefix + s for s in suffixes]
    q = _q(len(lens), 2 * G, prefix + 1)
    out, lse = fused.shared_prefix_decode(gpu, 0, q, _i32(table), _i32(lens), prefix)
    gpu.check()
    _check(gpu, orc, table, lens, q, out, lse, 1 / math.sqrt(D), "logical")


@pytest.mark.parametrize("n_splits", [1, 2, 5, 9])
def test_splits_padding_rows_and_physical_positions(n_splits):
    """Any number of splits; rows of length 0 between live ones; V rows by the
    physical slot with t_cal inside the pool."""
    from kvquant import fused
    suffixes = [40, 7, 0, 100]
    gpu, orc, table = _build((4, 4), 1136, suffixes, seed=5, t_cal=700, v_pos="physical")
    lens = [1176, 0, 1136, 1236]
    q = _q(4, 14, 3)
    out, lse = fused.shared_prefix_decode(gpu, 0, q, _i32(table), _i32(lens), 1136, v_pos="physical", n_splits=n_splits,
                                          softmax_scale=0.05)
    gpu.check()
    _check(gpu, orc, table, lens, q, out, lse, 0.05, "physical")


@pytest.mark.parametrize("B,G", [(1, 1), (1, 7), (18, 7), (19, 7), (36, 7), (37, 7), (3, 64), (2, 128), (130, 1)])
def test_row_tiles(B, G):
    """Batches that just fill, and just pass, one and two tiles of query rows."""
    from kvquant import fused
    suffixes = [(3 * i) % 20 + 1 for i in range(B)]
    gpu, orc, table = _build((4, 4), 272, suffixes, H=1, seed=B + G)
    lens = [272 + s for s in suffixes]
    q = _q(B, G, B)
    out, lse = fused.shared_prefix_decode(gpu, 0, q, _i32(table), _i32(lens), 272)
    gpu.check()
    _check(gpu, orc, table, lens, q, out, lse, 1 / math.sqrt(D), "logical")


def test_equals_the_decode_of_every_sequence():
    """The same batch through the per-sequence decode, over tables made by paging."""
    from kvquant import fused, paging
    from kvquant.compact_pool import CompactKVPool
    from kvquant.synthetic import NUQ2, NUQ4, make_kv, make_scales
    H, G, B, pre, NB = 4, 7, 6, 4096, 400
    sc = make_scales([NUQ2, NUQ4], H, D, t_cal=512, seed=3)
    pool = CompactKVPool(2, NB, S, H, D, sc)
    bt = torch.full((B, 300), -1, dtype=torch.int32, device="cuda")
    free, count = torch.randperm(NB, device="cuda").int(), _i32([NB])
    refs = torch.zeros(NB, dtype=torch.int32, device="cuda")
    # the prefix as sequence 0, then shared by the others
    t = paging.extend_tables(bt[:1], _i32([0]), _i32([pre]), free, count, num_tokens=pre, page_refs=refs)
    for layer in range(2):
        pool.reset_allocated(layer, free, count, t.free_count)
        pool.write_kv(layer, *make_kv(pre, H, D, seed=layer, chan_seed=3 + 1000 * layer), t.slot_mapping, t.positions)
    bt[1:, :pre // S] = bt[:1, :pre // S]
    refs[bt[0, :pre // S].long()] += B - 1
    new = _i32([1, 50, 16, 333, 7, 128])
    t2 = paging.extend_tables(bt, _i32([pre] * B), new, free, t.free_count, num_tokens=int(new.sum()), page_refs=refs)
    for layer in range(2):
        pool.reset_allocated(layer, free, t.free_count, t2.free_count)
        pool.write_kv(layer, *make_kv(int(new.sum()), H, D, seed=9 + layer, chan_seed=3 + 1000 * layer), t2.slot_mapping,
                      t2.positions)
    q = _q(B, H * G, 4, 0.3)
    for layer in range(2):
        o, l0 = fused.decode(pool, layer, q, bt, t2.seq_lens)
        out, lse = fused.shared_prefix_decode(pool, layer, q, bt, t2.seq_lens, pre)
        pool.check()
        # the bound at the top of this file with A <= max|v|; the decode, whose probabilities keep 22 bits and whose
        # output is fp32, is off by at most (2 e + 2^-17) max|v| and adds that much
        ks, vs = (torch.empty((NB, S, H, D), dtype=torch.float16, device="cuda") for _ in range(2))
        at = torch.arange(NB, device="cuda")
        pool.unpack_to_staging(layer, at, torch.full_like(at, pre), ks, vs)
        pool.unpack_to_staging(layer, at, torch.zeros_like(at), ks, vs2 := torch.empty_like(vs))
        vmax = float(torch.maximum(vs.abs(), vs2.abs()).max()) * 1.5   # V rows between: levels scale with their row's spread
        kabs = ks.float().abs().permute(2, 0, 1, 3).reshape(H, -1, D)
        dots = torch.matmul(q.float().abs().view(B, H, G, D).permute(1, 0, 2, 3).reshape(H, -1, D), kabs.transpose(1, 2))
        e = 2.0 ** -19 / math.sqrt(D) * float(dots.max())
        u, n = 2.0 ** -11, int(t2.seq_lens.max())
        tol = (u + 4 * e + 2.0 ** -16 + n * 2.0 ** -25) * vmax + u * o.abs() + 2.0 ** -25
        assert bool(((out.float() - o).abs() <= tol).all())
        assert bool(((lse - l0).abs() <= 2 * e + 2.0 ** -17 + l0.abs() * 2.0 ** -21).all())
    lens, left = paging.truncate_tables(bt, t2.seq_lens, _i32([0] * B), free, t2.free_count, page_refs=refs)
    pool.check()
    assert int(left) == NB and int(refs.abs().sum()) == 0 and sorted(free.tolist()) == list(range(NB))


def test_stale_entries_behind_a_sequence_change_nothing():
    """Outliers left in slots past a sequence's end (infinite ones too) are masked."""
    from kvquant import fused
    gpu, orc, table = _build((4, 4), 160, [20, 3], seed=21)
    lens = [180, 163]
    q = _q(2, 14, 5)
    out, lse = fused.shared_prefix_decode(gpu, 0, q, _i32(table), _i32(lens), 160)
    big = torch.full((1, 2, D), float("inf"), dtype=torch.float16, device="cuda")
    pos = torch.tensor([181], device="cuda")
    slot = torch.tensor([int(table[0, 11]) * S + 5], device="cuda")
    gpu.write_kv(0, big, big, slot, pos)
    slot = torch.tensor([int(table[1, 10]) * S + 3], device="cuda")
    gpu.write_kv(0, big, big, slot, torch.tensor([163], device="cuda"))
    out2, lse2 = fused.shared_prefix_decode(gpu, 0, q, _i32(table), _i32(lens), 160)
    gpu.check()
    assert torch.equal(out, out2) and torch.equal(lse, lse2)


def test_bad_lengths_and_pages_are_flagged():
    import hxlib
    from kvquant import fused
    gpu, orc, table = _build((4, 4), 160, [20, 3, 9], seed=22)
    q = _q(3, 14, 6)
    good, _ = fused.shared_prefix_decode(gpu, 0, q, _i32(table), _i32([180, 163, 169]), 160)
    for lens in ([180, 159, 169], [180, 10_000, 169]):
        out, lse = fused.shared_prefix_decode(gpu, 0, q, _i32(table), _i32(lens), 160)
        with pytest.raises(hxlib.HelixError, match="out of range"):
            gpu.check()
        assert not out[1].any() and bool(torch.isneginf(lse[1]).all())
        assert torch.equal(out[0], good[0]) and torch.equal(out[2], good[2])
    for page in (-1, gpu.num_blocks):
        bad = table.copy()
        bad[0, 3] = page
        fused.shared_prefix_decode(gpu, 0, q, _i32(bad), _i32([180, 163, 169]), 160)
        with pytest.raises(hxlib.HelixError, match="out of range"):
            gpu.check()


def test_streams_graphs_and_repeats():
    import hxlib
    from kvquant import fused
    gpu, orc, table = _build((2, 2), 640, [30, 61, 2], seed=30)
    q, bt, sl = _q(3, 14, 7), _i32(table), _i32([670, 701, 642])
    out, lse = fused.shared_prefix_decode(gpu, 0, q, bt, sl, 640)
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(fused.shared_prefix_decode(gpu, 0, q, bt, sl, 640))
        graphs.append(g)
    for st in (a, b):
        st.wait_stream(torch.cuda.current_stream())
    for _ in range(20):   # two captured calls side by side on two streams
        with torch.cuda.stream(a):
            graphs[0].replay()
        with torch.cuda.stream(b):
            graphs[1].replay()
    torch.cuda.synchronize()
    for o, l in outs:
        assert torch.equal(o, out) and torch.equal(l, lse)
    sl.copy_(_i32([645, 0, 701 - 32]))
    graphs[0].replay()
    o2, l2 = fused.shared_prefix_decode(gpu, 0, q, bt, sl, 640)
    assert torch.equal(outs[0][0], o2) and torch.equal(outs[0][1], l2)
    with pytest.raises(hxlib.HelixError, match="out of range"):   # sequence 2 now runs into table entries of -1
        gpu.check()


def test_more_work_items_than_sms():
    """Blocks of query rows past one wave of CTAs, and one KV head with a full
    group of rows; a sample of the sequences is checked."""
    from kvquant import fused
    B, G, H = 700, 8, 8
    suffixes = [i % 4 for i in range(B)]
    gpu, orc, table = _build((4, 4), 48, suffixes, H=H, seed=40)
    lens = [48 + s for s in suffixes]
    q = _q(B, H * G, 41)
    out, lse = fused.shared_prefix_decode(gpu, 0, q, _i32(table), _i32(lens), 48)
    gpu.check()
    keep = set(range(0, B, 37)) | {15, 16, 31, 32, B - 1}
    _check(gpu, orc, table, lens, q, out, lse, 1 / math.sqrt(D), "logical", skip=set(range(B)) - keep)
