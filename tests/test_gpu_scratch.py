"""Cached scratch under captured graphs: a larger eager call between capture and
replay takes a new buffer, and the graph's own stays its own."""
from __future__ import annotations

import pytest
import torch

from helpers import make_pools

pytestmark = pytest.mark.gpu


def test_a_larger_call_between_capture_and_replay(monkeypatch):
    import hxlib
    from kvquant import fused
    from kvquant.synthetic import NUQ4, make_kv, make_scales
    H, D, S, NB = 4, 128, 16, 64
    pool, _ = make_pools(make_scales([NUQ4], H, D, t_cal=64, seed=1), NB, S, H, D)
    K, V = make_kv(NB * S, H, D, seed=2, chan_seed=1)
    at = torch.arange(NB * S, device="cuda")
    pool.write_kv(0, K, V, at, at)
    q = torch.randn(64, 28, D, device="cuda").half() * 0.2
    bt = torch.arange(NB, dtype=torch.int32, device="cuda").expand(64, NB).contiguous()
    sl = torch.full((64,), NB * S, dtype=torch.int32, device="cuda")
    monkeypatch.setattr(hxlib, "_scratch", {})   # as in a new process
    want, wl = fused.decode(pool, 0, q[:1], bt[:1], sl[:1], n_splits=4)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        o, lse = fused.decode(pool, 0, q[:1], bt[:1], sl[:1], n_splits=4)
    small = hxlib._scratch[(0, "decode")].numel()
    fused.decode(pool, 0, q, bt, sl, n_splits=16)
    assert hxlib._scratch[(0, "decode")].numel() > small
    fills = [torch.full((small,), 7, dtype=torch.uint8, device="cuda") for _ in range(64)]
    for _ in range(5):
        g.replay()
    torch.cuda.synchronize()
    pool.check()
    assert torch.equal(o, want) and torch.equal(lse, wl)
    assert all(bool((f == 7).all()) for f in fills)
