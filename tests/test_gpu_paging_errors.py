"""Table calls that cannot be served, or are given bad ids, counts and sizes:
what they flag, and the tables, stack, counts and lengths they leave."""
from __future__ import annotations

import subprocess
import sys
from pathlib import Path

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def _i32(v):
    return torch.tensor(np.asarray(v), dtype=torch.int32, device="cuda")


def _flagged(match):
    import hxlib
    with pytest.raises(hxlib.HelixError, match=match):
        hxlib.check_device_errors()


def _handed_out_nothing(out, table, was, cached, count, refs=None, refs_was=None):
    assert torch.equal(table, was) and int(out.free_count) == count
    assert bool((out.slot_mapping == -1).all()) and not out.query_start.any()
    assert out.seq_lens.tolist() == list(cached)
    if refs is not None:
        assert torch.equal(refs, refs_was)


# ---- a shared page is not written into

@pytest.mark.parametrize("cut", [1, 5, 15])
def test_extending_into_a_shared_page_hands_out_nothing(cut):
    """Two sequences on one 3-page prefix; the second is cut inside the shared
    third page. Its next tokens would fall into a page the first reads."""
    from kvquant import paging
    S, num = 16, 12
    table = _i32([[4, 7, 2, 9, -1, -1], [4, 7, 2, 5, -1, -1]])
    refs = torch.zeros(num, dtype=torch.int32, device="cuda")
    refs[[4, 7, 2]] = 2
    refs[[9, 5]] = 1
    free, count = _i32([0, 1, 3, 6, 8, 10, 11, -1, -1, -1, -1, -1]), _i32([7])
    lens, count = paging.truncate_tables(table, _i32([60, 60]), _i32([60, 3 * S - cut]), free, count, page_refs=refs)
    assert lens.tolist() == [60, 48 - cut] and int(count) == 8
    was, refs_was = table.clone(), refs.clone()
    out = paging.extend_tables(table, lens, _i32([2, 3]), free, count, num_tokens=5, page_refs=refs)
    _flagged("shared page")
    _handed_out_nothing(out, table, was, lens.tolist(), 8, refs, refs_was)
    # not extended, the same sequence stands in nobody's way
    out = paging.extend_tables(table, lens, _i32([2, 0]), free, count, num_tokens=2, page_refs=refs)
    import hxlib
    hxlib.check_device_errors()
    assert out.slot_mapping.tolist() == [9 * S + 12, 9 * S + 13]
    # a page of its own (the caller copies the rows), and it goes on there
    fresh = int(free[7])
    table[1, 2] = fresh
    refs[2] -= 1
    refs[fresh] += 1
    out = paging.extend_tables(table, lens, _i32([0, 3]), free, _i32([7]), num_tokens=3, page_refs=refs)
    hxlib.check_device_errors()
    assert out.slot_mapping.tolist()[0] == fresh * S + 16 - cut


def test_whole_shared_pages_are_extended_past():
    from kvquant import paging
    import hxlib
    table, refs = _i32([[3, 1, -1], [3, 1, -1]]), _i32([0, 2, 0, 2, 0])
    out = paging.extend_tables(table, _i32([32, 32]), _i32([1, 16]), _i32([0, 2, 4]), _i32([3]), num_tokens=17, page_refs=refs)
    hxlib.check_device_errors()
    assert table.tolist() == [[3, 1, 4], [3, 1, 2]] and refs.tolist() == [0, 2, 1, 2, 1]
    assert out.slot_mapping.tolist() == [64] + list(range(32, 48))


# ---- ids outside the pool

@pytest.mark.parametrize("bad", [-1, 64, 2 ** 31 - 1, -2 ** 31])
@pytest.mark.parametrize("counted", [False, True])
@pytest.mark.parametrize("where", ["stack", "table"])
def test_extend_with_a_bad_id_hands_out_nothing(bad, counted, where):
    """On the stack among the pages to be popped, or as the page that a
    sequence goes on filling: a row never ends up on a page it was not given."""
    from kvquant import paging
    rng = np.random.default_rng(3)
    num, B, W = 64, 5, 8
    perm = rng.permutation(num)
    table = np.full((B, W), 33, np.int64)        # stale entries name a page that another may hold
    cached = np.array([0, 5, 16, 31, 40])
    at = 0
    for b, c in enumerate(cached):
        n = -(-c // 16)
        table[b, :n] = perm[at:at + n]
        at += n
    refs = np.zeros(num, np.int64)
    refs[perm[:at]] = 1
    free = perm[at:].copy()
    if where == "stack":
        free[-7] = bad
    else:
        table[3, 1] = bad
    g, gr, gf, count = _i32(table), _i32(refs) if counted else None, _i32(free), _i32([len(free)])
    was, rw = g.clone(), gr.clone() if counted else None
    out = paging.extend_tables(g, _i32(cached), _i32([20, 30, 40, 50, 10]), gf, count, num_tokens=160, page_refs=gr,
                               num_pages=num)
    _flagged("out of range")
    _handed_out_nothing(out, g, was, cached, len(free), gr, rw)


@pytest.mark.parametrize("B,pages", [(4, 5), (64, 300)])
@pytest.mark.parametrize("counted", [False, True])
def test_truncate_gives_back_the_good_entries_only(B, pages, counted):
    """Bad entries among those dropped: flagged, and neither pushed nor counted
    (one CTA, and many)."""
    from kvquant import paging
    rng = np.random.default_rng(B)
    num = B * pages + 10
    perm = rng.permutation(num)
    table = perm[:B * pages].reshape(B, pages).copy()
    keep = rng.integers(0, pages * 16 + 1, B)
    keep[0], keep[1] = 0, 7
    bad = [(0, 0, -1), (0, pages - 1, num), (1, 1, 2 ** 31 - 1), (1, 0, -5)]   # the last one is kept, not dropped
    for b, j, e in bad:
        table[b, j] = e
    refs = np.zeros(num, np.int64)
    refs[table[(table >= 0) & (table < num)]] = 1
    ent = [int(table[b, j]) for b in range(B) for j in range(-(-keep[b] // 16), pages)]
    good = [p for p in ent if 0 <= p < num]
    assert len(good) == len(ent) - 3
    free = np.full(num, -1)
    free[:10] = perm[-10:]
    gf, gr = _i32(free), _i32(refs) if counted else None
    lens, count = paging.truncate_tables(_i32(table), _i32([pages * 16] * B), _i32(keep), gf, _i32([10]), page_refs=gr,
                                         num_pages=num)
    _flagged("out of range")
    assert int(count) == 10 + len(good) and lens.tolist() == keep.tolist()
    assert gf[:int(count)].tolist() == free[:10].tolist() + good[::-1]
    if counted:
        refs[good] = 0
        assert gr.tolist() == refs.tolist()


# ---- a stack without room

@pytest.mark.parametrize("twice", [False, True])
def test_truncate_with_counts_onto_a_full_stack_gives_back_nothing(twice):
    """Ten pages would come free (``twice``: nine, and some entries find no
    reference to give back) on a stack with room for eight: counts, stack and
    lengths stay as they were."""
    from kvquant import paging
    table = np.array([[3, 8, 5, 11], [3, 8, 5, 0], [3, 8, 2, 1], [13, 6, 4, 12]])
    refs = np.zeros(14, np.int64)
    for p in table.ravel():
        refs[p] += 1
    refs[3] = 5                                  # someone outside the batch holds it too
    if twice:
        refs[8], refs[5], refs[6] = 2, 1, 0      # fewer than the entries that name them
    free = np.full(11, -1)
    free[:3] = [7, 9, 10]
    g, gf, gr = _i32(table), _i32(free), _i32(refs)
    lens, count = paging.truncate_tables(g, _i32([64, 60, 50, 64]), _i32([0, 0, 0, 0]), gf, _i32([3]), page_refs=gr, num_pages=14)
    _flagged("out of range")
    assert gr.tolist() == refs.tolist() and gf.tolist() == free.tolist() and int(count) == 3
    assert lens.tolist() == [64, 60, 50, 64]


# ---- batch sizes whose lengths just fill the default shared memory

@pytest.mark.parametrize("call,B", [("extend", 6112), ("extend", 6144), ("truncate", 6112), ("truncate", 6144)])
def test_batches_around_the_default_shared_memory(call, B):
    """In a process of its own: a larger batch raises the kernel's limit for good."""
    code = f"""
import torch, hxlib
from kvquant import paging
B = {B}
z = lambda n: torch.zeros(n, dtype=torch.int32, device="cuda")
t, f = z((B, 1)), torch.arange(B, dtype=torch.int32, device="cuda")
if "{call}" == "extend":
    r = paging.extend_tables(t, z(B), z(B) + 1, f, z(1) + B, num_tokens=B)
    hxlib.check_device_errors()
    assert int(r.free_count) == 0 and torch.equal(r.slot_mapping, torch.arange(B - 1, -1, -1, device="cuda") * 16)
else:
    t[:, 0] = f
    lens, count = paging.truncate_tables(t, z(B) + 9, z(B), z(B), z(1))
    hxlib.check_device_errors()
    assert int(count) == B and not lens.any()
"""
    root = Path(__file__).resolve().parents[1] / "helix-lite_b200"
    r = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]


# ---- lengths at the border of 32 bits

def test_lengths_past_32_bits_are_refused():
    from kvquant import paging
    import hxlib
    S = 1 << 20
    table = torch.arange(2049, dtype=torch.int32, device="cuda")[None].contiguous()
    free, was = _i32([2049, 2050]), table.clone()
    for new, fits in ((8, False), (7, True)):
        out = paging.extend_tables(table, _i32([2 ** 31 - 8]), _i32([new]), free, _i32([2]), num_tokens=8, page_size=S,
                                   num_pages=3000)
        if fits:
            hxlib.check_device_errors()
            assert out.seq_lens.tolist() == [2 ** 31 - 1]
            assert out.slot_mapping.tolist() == [2047 * S + S - 8 + i for i in range(7)] + [-1]
        else:
            _flagged("out of range")
            _handed_out_nothing(out, table, was, [2 ** 31 - 8], 2)
    for kw in (dict(num_tokens=2 ** 30 + 1), dict(num_tokens=2 ** 32 + 8), dict(num_tokens=8, page_size=2 ** 32 + 16)):
        with pytest.raises(ValueError):
            paging.extend_tables(table, _i32([0]), _i32([8]), free, _i32([2]), **kw)


# ---- results in tensors that another argument or result also names

def test_outputs_that_alias_are_refused():
    from kvquant import paging
    table, cached, new = _i32([[-1, -1]]), _i32([0]), _i32([3])
    free, count, refs = _i32([0, 1, 2]), _i32([3]), _i32([0, 0, 0])

    def out(**kw):
        o = paging.BatchTables(_i32([0, 0]), _i32([0]), torch.zeros(3, dtype=torch.int64, device="cuda"),
                               torch.zeros(3, dtype=torch.int64, device="cuda"), _i32([0]))
        for k, t in kw.items():
            setattr(o, k, t)
        return o
    one = _i32([0])
    long = torch.zeros(4, dtype=torch.int64, device="cuda")
    for kw in (dict(free_count=one, seq_lens=one), dict(seq_lens=refs[1:2]), dict(free_count=free[2:]),
               dict(query_start=refs[1:]), dict(slot_mapping=long[1:], positions=long[:3])):
        with pytest.raises(ValueError, match="out"):
            paging.extend_tables(table, cached, new, free, count, num_tokens=3, page_refs=refs, out=out(**kw))
    ok = paging.extend_tables(table, cached, new, free, count, num_tokens=3, page_refs=refs,
                              out=out(slot_mapping=torch.cat([long, long])[:3], query_start=_i32([0, 0, 0, 0])[1:3]))
    assert ok.slot_mapping.tolist() == [32, 33, 34] and ok.seq_lens.tolist() == [3]


def test_a_shared_page_is_copied_by_hand_and_extended():
    """What the refusal asks for: the page's rows read back and written to a page
    of the sequence's own (levels and outliers quantise to themselves), then
    both sequences go on, each as if it had never shared."""
    from kvquant import paging
    from kvquant.compact_pool import CompactKVPool
    from kvquant.synthetic import NUQ4, make_kv, make_scales
    import hxlib
    H, D, S, NB = 2, 128, 16, 16
    sc = make_scales([NUQ4], H, D, t_cal=128, seed=5)
    pool, alone = CompactKVPool(1, NB, S, H, D, sc), CompactKVPool(1, NB, S, H, D, sc)
    K, V = make_kv(64, H, D, seed=6, chan_seed=5, outlier_frac=0.05)
    table = torch.full((2, 6), -1, dtype=torch.int32, device="cuda")
    free, refs, count = _i32(np.arange(NB)), torch.zeros(NB, dtype=torch.int32, device="cuda"), _i32([NB])
    t = paging.extend_tables(table[:1], _i32([0]), _i32([40]), free, count, num_tokens=40, page_refs=refs)
    pool.write_kv(0, K[:40], V[:40], t.slot_mapping, t.positions)
    table[1] = table[0]
    refs[table[0, :3].long()] += 1
    lens, count = paging.truncate_tables(table, _i32([40, 40]), _i32([40, 37]), free, t.free_count, page_refs=refs)
    assert lens.tolist() == [40, 37] and int(count) == NB - 3
    new = _i32([2, 3])
    paging.extend_tables(table, lens, new, free, count, num_tokens=5, page_refs=refs)
    _flagged("shared page")
    # sequence 1 takes a page of its own in place of the third, with the 5 tokens it keeps there
    old = table[1, 2].clone()
    sk, sv = (torch.empty((1, S, H, D), dtype=torch.float16, device="cuda") for _ in range(2))
    pool.unpack_to_staging(0, old[None], torch.tensor([32], device="cuda"), sk, sv)
    own = free[count.long() - 1]
    count -= 1
    at = torch.arange(5, device="cuda")
    pool.write_kv(0, sk[0, :5].contiguous(), sv[0, :5].contiguous(), own.long() * S + at, 32 + at)
    table[1, 2] = own[0]
    refs[old.long()] -= 1
    refs[own.long()] += 1
    t = paging.extend_tables(table, lens, new, free, count, num_tokens=5, page_refs=refs)
    hxlib.check_device_errors()
    # sequence 0 goes on with tokens 40, 41, sequence 1 with 50 .. 52
    pool.write_kv(0, K[[40, 41, 50, 51, 52]].contiguous(), V[[40, 41, 50, 51, 52]].contiguous(), t.slot_mapping, t.positions)
    for b, toks in ((0, list(range(42))), (1, list(range(37)) + [50, 51, 52])):
        n = len(toks)
        i = torch.arange(n, device="cuda")
        alone.reset_pages(0, torch.arange(3, dtype=torch.int32, device="cuda"))
        alone.write_kv(0, K[toks].contiguous(), V[toks].contiguous(), i, i)
        got, want = [], []
        for p, pages, out in ((pool, table[b, :3], got), (alone, torch.arange(3, device="cuda"), want)):
            k, v = (torch.empty((3, S, H, D), dtype=torch.float16, device="cuda") for _ in range(2))
            p.unpack_to_staging(0, pages, torch.arange(3, device="cuda") * S, k, v)
            p.check()
            out += [k.view(-1, H, D)[:n], v.view(-1, H, D)[:n]]
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
