"""Refusals of the prompt and shared-prefix attention that need no GPU."""
from __future__ import annotations

import pytest
import torch

import hxlib


def test_prompt_attention_refuses_on_the_host():
    L = hxlib.lib()
    a = hxlib.ctypes.c_void_p(256)  # never read: every call below is refused on the host
    odd = hxlib.ctypes.c_void_p(264)
    good = [None, 1, a, 512, 128, a, 512, 128, a, 512, 128, a, 1, 8, 4, 1, 128, 0.1, a, a, None]
    bad = [(1, 0), (1, 3), (2, odd), (2, None), (3, 511), (4, 64), (6, 516), (9, -8), (11, None), (12, -1), (13, -1),
           (14, 0), (15, 0), (15, 129), (16, 96), (17, 0.0), (17, -1.0), (17, float("nan")), (17, float("inf")), (18, odd)]
    for i, v in bad:
        args = list(good)
        args[i] = v
        assert L.hx_prompt_attn(*args) in (hxlib.HX_ERR_ARG, hxlib.HX_ERR_UNSUPPORTED), (i, v)
    for i in (12, 13):
        args = list(good)
        args[i] = 0          # no prompts, no tokens: nothing to do
        assert L.hx_prompt_attn(*args) == hxlib.HX_OK


def test_prefix_decode_refuses_on_the_host():
    L = hxlib.lib()
    a, odd = hxlib.ctypes.c_void_p(256), hxlib.ctypes.c_void_p(257)

    def pool(**kw):
        f = dict(codes=256, stats=256, dir=256, arena=256, arena_top=256, arena_capacity=64, num_blocks=8, block_size=16,
                 num_kv_heads=4, head_size=128, bits_k=4, bits_v=4)
        f.update(kw)
        return hxlib.ctypes.byref(hxlib.PoolLayer(**f))

    def scales(**kw):
        f = dict(k_poles=256, k_upper=256, k_lower=256, v_poles=256, v_upper=256, v_lower=256, levels_k=16, levels_v=16,
                 t_cal=4, reserved=0)
        f.update(kw)
        return hxlib.ctypes.byref(hxlib.LayerScales(**f))

    good = [None, pool(), scales(), a, 2, 7, 0.1, a, 20, a, 8, 0, 1, a, a, a, None]
    bad = [(1, None), (2, None), (3, None), (3, odd), (4, -1), (5, 0), (5, 129), (6, 0.0), (6, -1.0), (7, None), (8, 7),
           (9, None), (10, -1), (11, 1), (12, 0), (12, 2), (12, -1), (13, None), (13, odd), (14, None),
           (1, pool(head_size=64)), (1, pool(block_size=32)), (1, pool(bits_k=3)), (2, scales(levels_k=17)),
           (2, scales(t_cal=0)), (1, pool(codes=264))]
    for i, v in bad:
        args = list(good)
        args[i] = v
        assert L.hx_prefix_decode(*args) in (hxlib.HX_ERR_ARG, hxlib.HX_ERR_UNSUPPORTED), (i, v)
    args = list(good)
    args[4] = 0
    assert L.hx_prefix_decode(*args) == hxlib.HX_OK
    assert L.hx_prefix_splits(0, 4, 7, 8) == 0 and L.hx_prefix_splits(2, 4, 7, 0) == 0
    for B in (1, 18, 37, 200):
        for pages in (1, 8, 9, 65536):
            n = L.hx_prefix_splits(B, 4, 7, pages)
            assert 1 <= n <= -(-pages // 8)
            assert L.hx_prefix_scratch_bytes(B, 4, 7, n) == (n + 1) * B * 28 * 130 * 4


def test_shapes_and_types_are_refused():
    from kvquant import fused
    q, k = torch.zeros((4, 6, 128), dtype=torch.float16), torch.zeros((4, 2, 128), dtype=torch.float16)
    s = torch.tensor([0, 4], dtype=torch.int32)
    for args, err in (((q, k, k, s), hxlib.HelixError), ((q[0], k, k, s), ValueError), ((q, k, k[:3], s), ValueError),
                      ((q[:3], k, k, s), ValueError), ((q[:, :5], k, k, s), ValueError), ((q.float(), k, k, s), TypeError),
                      ((q, k, k.bfloat16(), s), TypeError), ((q, k, k, s[None]), ValueError),
                      ((q, k[..., :64], k[..., :64], s), ValueError)):
        with pytest.raises(err):
            fused.prompt_attention(*args)


def _hook(monkeypatch, **state):
    """The compact hook's module with recorders in place of the kernels."""
    import types

    from kvquant import compact_backend as cb
    calls = []

    def recorder(name, result):
        def f(*args, **kw):
            calls.append((name, args, kw))
            return result(*args, **kw)
        return f
    half = lambda pool, li, q, *a, **kw: (torch.full(q.shape, 0.5), None)  # noqa: E731
    prompt = lambda q, k, v, qs, out=None, **kw: (out.fill_(0.25) if out is not None else torch.full_like(q, 0.25), None)  # noqa: E731
    monkeypatch.setattr(cb, "fused", types.SimpleNamespace(
        decode=recorder("decode", half), shared_prefix_decode=recorder("shared", half),
        prefill=recorder("prefill", half), prompt_attention=recorder("prompt", prompt)))
    monkeypatch.setattr(cb, "_POOL", types.SimpleNamespace(num_layers=4, block_size=16))
    monkeypatch.setattr(cb, "_TOP_K", 0)
    for k, v in state.items():
        monkeypatch.setattr(cb, k, v)
    impl = cb.make_impl_cls(type("Base", (), {}))()
    impl.scale, impl.sliding_window = 0.125, (-1, -1)
    layer = types.SimpleNamespace(layer_name="model.layers.1.self_attn.attn")
    return cb, impl, layer, calls


def _meta(**kw):
    import types
    return types.SimpleNamespace(causal=True, **kw)


def test_hook_decodes_a_shared_prefix_once_when_asked(monkeypatch):
    bt, sl = torch.zeros((3, 9), dtype=torch.int32), torch.full((3,), 100, dtype=torch.int32)
    q = torch.randn(4, 28, 128)
    for asked, common, want in ((True, 70, "shared"), (True, 15, "decode"), (True, 0, "decode"), (False, 70, "decode")):
        cb, impl, layer, calls = _hook(monkeypatch, _SHARED_PREFIX=asked)
        out = torch.zeros(4, 28, 128, dtype=torch.float16)
        impl.forward(layer, q, None, None, None, _meta(max_query_len=1, num_actual_tokens=3, block_table=bt, seq_lens=sl,
                                                       common_prefix_len=common), out)
        assert [c[0] for c in calls] == [want]
        if want == "shared":
            assert calls[0][1][5] == 64 and calls[0][2]["v_pos"] == "physical"  # whole blocks of the prefix
        assert bool((out[:3] == 0.5).all()) and not out[3].any()


def test_hook_attends_whole_prompts_exactly_when_asked(monkeypatch):
    bt, q = torch.zeros((2, 9), dtype=torch.int32), torch.randn(12, 28, 128).half()
    k = torch.randn(12, 4, 128).half()

    def meta(n, longest, longest_seq):
        return _meta(max_query_len=longest, max_seq_len=longest_seq, num_actual_tokens=n, block_table=bt,
                     seq_lens=torch.tensor([5, 5]), query_start_loc=torch.tensor([0, 5, n]))
    for asked, m, want in ((True, meta(10, 5, 5), "prompt"), (False, meta(10, 5, 5), "prefill"),
                           (True, meta(10, 5, 9), "prefill"), (True, meta(9, 5, 5), "prefill")):
        cb, impl, layer, calls = _hook(monkeypatch, _EXACT_PROMPTS=asked, _FP16_CACHE=False)
        out = torch.zeros(12, 28, 128, dtype=torch.float16)
        impl.forward(layer, q, k, k, None, m, out)
        assert [c[0] for c in calls] == [want]
        if want == "prompt":
            assert bool((out[:10] == 0.25).all()) and not out[10:].any()


def test_hook_takes_an_output_off_the_kernels_alignment(monkeypatch):
    """prompt_attention writes 16-byte pieces; any other output is copied into."""
    bt, q, k = torch.zeros((2, 9), dtype=torch.int32), torch.randn(10, 28, 128).half(), torch.randn(10, 4, 128).half()
    m = _meta(max_query_len=5, max_seq_len=5, num_actual_tokens=10, block_table=bt, seq_lens=torch.tensor([5, 5]),
              query_start_loc=torch.tensor([0, 5, 10]))
    buf = torch.zeros(12 * 28 * 128 + 8, dtype=torch.float16)
    for shift, direct in ((0, True), (1, False), (4, False), (8, True)):
        cb, impl, layer, calls = _hook(monkeypatch, _EXACT_PROMPTS=True, _FP16_CACHE=False)
        out = buf.zero_()[shift:shift + 12 * 28 * 128].view(12, 28, 128)
        impl.forward(layer, q, k, k, None, m, out)
        assert [c[0] for c in calls] == ["prompt"] and (calls[0][2]["out"] is not None) == direct
        assert bool((out[:10] == 0.25).all()) and not out[10:].any()


def test_hook_attends_one_token_prompts_exactly_too(monkeypatch):
    """A batch of one-token prompts is a batch of whole prompts; one-token steps
    of longer sequences, or without the option, decode from the pool."""
    bt, q, k = torch.zeros((3, 9), dtype=torch.int32), torch.randn(3, 28, 128).half(), torch.randn(3, 4, 128).half()
    for asked, cache, longest, want in ((True, False, 1, "prompt"), (True, False, 2, "decode"), (False, False, 1, "decode"),
                                        (True, True, 1, "decode")):
        cb, impl, layer, calls = _hook(monkeypatch, _EXACT_PROMPTS=asked, _FP16_CACHE=cache)
        out = torch.zeros(3, 28, 128, dtype=torch.float16)
        m = _meta(max_query_len=1, max_seq_len=longest, num_actual_tokens=3, block_table=bt,
                  seq_lens=torch.full((3,), longest), query_start_loc=torch.tensor([0, 1, 2, 3]))
        impl.forward(layer, q, k, k, None, m, out)
        assert [c[0] for c in calls] == [want]


def test_hook_reads_a_shared_prefix_once_only_where_that_pays(monkeypatch):
    """A short common prefix before long sequences of their own goes to the
    per-sequence decode, which splits every sequence over the SMs."""
    bt, q = torch.zeros((64, 9), dtype=torch.int32), torch.randn(64, 28, 128)
    for B, H, common, longest, want in (
            (4, 4, 2048, 2048 + 300, "shared"), (4, 4, 2048, 2048 + 400, "decode"),       # 64 own <= H (B - 1) common
            (8, 4, 2048, 2048 + 32768, "decode"), (2, 4, 4096, 4096 + 131072, "decode"),
            (64, 4, 32768, 32768 + 512, "shared"), (64, 8, 2048, 2048 + 16000, "shared"), (8, 1, 2048, 2048 + 512, "decode"),
            (64, 4, 112, 112, "decode"), (64, 4, 128, 130, "shared"), (3, 4, 1024, 0, "shared")):  # no length known
        cb, impl, layer, calls = _hook(monkeypatch, _SHARED_PREFIX=True)
        cb._POOL.num_kv_heads = H
        out = torch.zeros(64, 28, 128, dtype=torch.float16)
        impl.forward(layer, q, None, None, None, _meta(max_query_len=1, num_actual_tokens=B, block_table=bt,
                                                       seq_lens=torch.full((64,), longest), common_prefix_len=common,
                                                       max_seq_len=longest), out)
        assert [c[0] for c in calls] == [want], (B, H, common, longest)
