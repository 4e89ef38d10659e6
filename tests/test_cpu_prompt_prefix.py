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
            assert L.hx_prefix_scratch_bytes(B, 4, 7, n) == (2 * n + 2) * B * 28 * 130 * 4


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
