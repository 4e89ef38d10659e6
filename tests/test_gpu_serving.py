"""A serving run end to end: tables built on the GPU, prompts attended at full
precision and packed, a system prompt shared by the batch, decode steps that
read it once; against the float64 oracle. And the vLLM hook's two options."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from helpers import np16, oracle_scales
from test_gpu_prefix import _check as check_prefix
from test_gpu_prefix import _i32, _q
from test_gpu_prompt import _check as check_prompt
from test_gpu_prompt import _formula

pytestmark = pytest.mark.gpu

H, G, D, S, NB = 2, 7, 128, 16, 64


def _pools(seed, t_cal=128):
    from kvquant.compact_pool import CompactKVPool
    from kvquant.synthetic import NUQ4, make_scales
    from oracle.pool import OraclePool
    sc = make_scales([NUQ4], H, D, t_cal=t_cal, seed=seed)
    return CompactKVPool(1, NB, S, H, D, sc), OraclePool(1, NB, S, H, D, oracle_scales(sc))


def test_prompts_then_decode_steps_on_a_shared_system_prompt():
    from kvquant import fused, paging
    from kvquant.synthetic import make_kv
    gpu, orc = _pools(3)

    def write(t, n, seed):
        K, V = make_kv(n, H, D, seed=seed, chan_seed=3)
        gpu.write_kv(0, K, V, t.slot_mapping, t.positions)
        orc.write_kv(0, np16(K), np16(V), np16(t.slot_mapping), np16(t.positions))
        return K, V

    B, pre = 3, 160
    bt = torch.full((B, 30), -1, dtype=torch.int32, device="cuda")
    free, refs, count = torch.randperm(NB, device="cuda").int(), torch.zeros(NB, dtype=torch.int32, device="cuda"), _i32([NB])
    # the system prompt: attended from its own K and V, then packed
    t = paging.extend_tables(bt[:1], _i32([0]), _i32([pre]), free, count, num_tokens=pre, page_refs=refs)
    K, V = write(t, pre, 5)
    q = _q(pre, H * G, 6, 0.2)
    out, lse = fused.prompt_attention(q, K, V, t.query_start)
    want, wl, mag = _formula(q, K, V, [0, pre], 1 / math.sqrt(D))
    check_prompt(out, lse, want, wl, mag, V, pre, torch.ones(pre, dtype=torch.bool, device="cuda"))
    # the batch shares it
    bt[1:, :pre // S] = bt[0, :pre // S]
    refs[bt[0, :pre // S].long()] += B - 1
    lens, new = _i32([pre] * B), _i32([40, 1, 17])
    for step in range(4):
        t = paging.extend_tables(bt, lens, new, free, t.free_count, num_tokens=int(new.sum()), page_refs=refs)
        write(t, int(new.sum()), 10 + step)
        lens, new = t.seq_lens, _i32([1] * B)
        q = _q(B, H * G, 20 + step)
        out, lse = fused.shared_prefix_decode(gpu, 0, q, bt, lens, pre)
        gpu.check()
        check_prefix(gpu, orc, np16(bt), lens.tolist(), q, out, lse, 1 / math.sqrt(D), "logical")
    lens, left = paging.truncate_tables(bt, lens, _i32([0] * B), free, t.free_count, page_refs=refs)
    gpu.check()
    assert int(left) == NB and not refs.any()


def test_hook_options(monkeypatch):
    """The hook's shared-prefix decode against its per-sequence decode, and its
    exact prompts against the formula."""
    import types

    from kvquant import compact_backend as cb
    from kvquant.synthetic import make_kv
    gpu, orc = _pools(7)
    pre, lens = 96, [130, 97, 111]
    rng = np.random.default_rng(1)
    perm = rng.permutation(NB)
    table = np.concatenate([np.tile(perm[:6], (3, 1)), perm[6:6 + 9].reshape(3, 3)], 1)
    for b, n in enumerate(lens):
        lo = 0 if b == 0 else pre
        K, V = make_kv(n - lo, H, D, seed=b, chan_seed=7)
        i = np.arange(lo, n)
        slots = torch.from_numpy(table[b, i // S] * S + i % S).cuda()
        gpu.write_kv(0, K, V, slots, slots)
        orc.write_kv(0, np16(K), np16(V), np16(slots), np16(slots))
    q = _q(3, H * G, 2)
    meta = types.SimpleNamespace(num_actual_tokens=3, block_table=_i32(table), seq_lens=_i32(lens), common_prefix_len=pre + 1)
    monkeypatch.setattr(cb, "_TOP_K", 0)
    monkeypatch.setattr(cb, "_SHARED_PREFIX", True)
    out = torch.zeros((3, H * G, D), dtype=torch.float16, device="cuda")
    cb.decode_into(gpu, 0, q, meta, out, scale=0.1)
    gpu.check()
    from kvquant import fused
    want, lse = fused.shared_prefix_decode(gpu, 0, q, _i32(table), _i32(lens), pre, softmax_scale=0.1, v_pos="physical")
    assert torch.equal(out, want)
    check_prefix(gpu, orc, table, lens, q, out, lse, 0.1, "physical")
    # prompts
    n = 37
    K, V = make_kv(2 * n, H, D, seed=9, chan_seed=7)
    q = _q(2 * n, H * G, 3, 0.2)
    meta = types.SimpleNamespace(num_actual_tokens=2 * n, max_query_len=n, max_seq_len=n, query_start_loc=_i32([0, n, 2 * n]))
    assert cb.whole_prompts(meta, q, K)
    out = torch.zeros((2 * n + 3, H * G, D), dtype=torch.float16, device="cuda")
    cb.prompts_into(q, K, V, meta, out, scale=0.1)
    want, wl, mag = _formula(q, K, V, [0, n, 2 * n], 0.1)
    check_prompt(out[:2 * n], wl.float(), want, wl, mag, V, n, torch.ones(2 * n, dtype=torch.bool, device="cuda"))
    assert not out[2 * n:].any()


def test_install_sets_the_options_and_defaults_leave_them_off():
    import types

    from kvquant import compact_backend as cb
    from kvquant import fused
    from kvquant.synthetic import NUQ4, make_kv, make_scales
    sc = make_scales([NUQ4], H, D, t_cal=64, seed=2)
    backend = type("Backend", (), {"get_impl_cls": None})
    base = type("Impl", (), {"do_kv_cache_update": lambda self, *a: None})
    kw = dict(num_layers=1, num_blocks=16, num_kv_heads=H, head_size=D, scales=sc, backend_cls=backend, impl_cls=base)
    layer = types.SimpleNamespace(layer_name="model.layers.0.self_attn.attn")
    K, V = make_kv(16 * S, H, D, seed=3, chan_seed=2)
    slots = torch.arange(16 * S, device="cuda")
    table = _i32([[0, 1, 2, 3], [0, 1, 4, 5]])
    q = _q(2, H * G, 4)
    meta = types.SimpleNamespace(max_query_len=1, num_actual_tokens=2, causal=True, block_table=table,
                                 seq_lens=_i32([50, 40]), common_prefix_len=32)
    got = {}
    for asked in (True, False):
        cb.install_compact_backend("", **kw, **({"shared_prefix": True, "exact_prompts": True} if asked else {}))
        assert cb._SHARED_PREFIX is asked and cb._EXACT_PROMPTS is asked
        impl = backend.get_impl_cls()()
        impl.scale, impl.sliding_window = 0.1, (-1, -1)
        impl.do_kv_cache_update(layer, K, V, None, slots)
        out = torch.zeros((2, H * G, D), dtype=torch.float16, device="cuda")
        impl.forward(layer, q, None, None, None, meta, out)
        cb.pool().check()
        if asked:
            want, _ = fused.shared_prefix_decode(cb.pool(), 0, q, table, meta.seq_lens, 32, softmax_scale=0.1, v_pos="physical")
        else:
            want, _ = fused.decode(cb.pool(), 0, q, table, meta.seq_lens, softmax_scale=0.1, v_pos="physical")
        assert torch.equal(out, want.half())
