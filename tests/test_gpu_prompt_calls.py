"""Calls of the whole-prompt attention that the documentation allows or
refuses by where its tensors lie."""
from __future__ import annotations

import math

import pytest
import torch

from test_gpu_prompt import _check, _formula, _make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D,dt", [(64, torch.bfloat16), (128, torch.float16)])
@pytest.mark.parametrize("Hq,H", [(7, 1), (8, 8)])
def test_output_in_place_of_the_queries(D, dt, Hq, H):
    """A work item reads its own rows of q before it writes them, and no other
    item reads them: the same bits as with an output of its own."""
    from kvquant import fused
    lens = [1, 300, 17, 0, 129]
    q, k, v, start = _make(lens, Hq, H, D, dt, seed=71)
    q = q.contiguous()
    qs = torch.tensor(start, dtype=torch.int32, device="cuda")
    want, wl, mag = _formula(q, k, v, start, 1 / math.sqrt(D))
    apart, lse = fused.prompt_attention(q, k, v, qs)
    out, lse2 = fused.prompt_attention(q, k, v, qs, out=q)
    assert out.data_ptr() == q.data_ptr() and torch.equal(out, apart) and torch.equal(lse, lse2)
    _check(out, lse2, want, wl, mag, v, max(lens), torch.ones(len(q), dtype=torch.bool, device="cuda"))


def test_outputs_over_inputs_are_refused():
    from kvquant import fused
    q, k, v, start = _make([40], 4, 4, 64, torch.float16, seed=72)
    q, k, v = (x.contiguous() for x in (q, k, v))
    qs = torch.tensor(start, dtype=torch.int32, device="cuda")
    both = torch.cat([q, q])
    words = torch.zeros(40 * 4 + 2, dtype=torch.int32, device="cuda")
    words[1] = 40
    for args, kw in (((q, k, v, qs), dict(out=k)), ((q, k, v, qs), dict(out=v)),
                     ((both[1:41], k, v, qs), dict(out=both[:40])),
                     ((q, k, v, qs), dict(lse=v.view(torch.float32).view(-1)[:160].view(40, 4))),
                     ((q, k, v, words[:2]), dict(lse=words[1:161].view(torch.float32).view(40, 4)))):
        with pytest.raises(ValueError, match="overlap"):
            fused.prompt_attention(*args, **kw)
    buf = torch.empty(q.numel() * 2 + 40 * 4 * 4, dtype=torch.uint8, device="cuda")
    out = buf[:q.numel() * 2].view(torch.float16).view(q.shape)
    with pytest.raises(ValueError, match="overlap"):
        fused.prompt_attention(q, k, v, qs, out=out, lse=buf[q.numel() * 2 - 16:-16].view(torch.float32).view(40, 4))
    o, l = fused.prompt_attention(q, k, v, qs, out=out, lse=buf[q.numel() * 2:].view(torch.float32).view(40, 4))
    w, wl = fused.prompt_attention(q, k, v, qs)
    assert torch.equal(o, w) and torch.equal(l, wl)


def test_same_attention_as_the_pool_prefill_on_what_the_pool_holds():
    """prompt_attention on the dequantised K and V, and prefill from the pool,
    both against the formula in 64 bits. Each query is a multiple of one visible
    token's key (score 12), so a wrong score, page or position shows.

    Tolerance: as in test_gpu_prompt for the first, with e = 2^-19 scale
    max_j sum_c |q_c k_jc| for what fp32 scores are off by (a probability moves
    by a factor of at most 1 + 2 e); prefill keeps 22 bits of its probabilities,
    so it has the rounding of its output (half a step u) and 2 e + 2^-17 of the
    softmax average of |v|."""
    from kvquant import fused
    from kvquant.compact_pool import CompactKVPool
    from kvquant.synthetic import NUQ4, make_kv, make_scales
    n, H, G, D = 333, 4, 7, 128
    sc = make_scales([NUQ4], H, D, t_cal=512, seed=81)
    pool = CompactKVPool(1, 32, 16, H, D, sc)
    K, V = make_kv(n, H, D, seed=82, chan_seed=81)
    g = torch.Generator(device="cuda").manual_seed(83)
    pages = torch.randperm(32, generator=g, device="cuda")[:21]
    at = torch.arange(n, device="cuda")
    slots = pages[at // 16] * 16 + at % 16
    pool.write_kv(0, K, V, slots, at)
    sk, sv = (torch.empty((21, 16, H, D), dtype=torch.float16, device="cuda") for _ in range(2))
    pool.unpack_to_staging(0, pages, torch.arange(21, device="cuda") * 16, sk, sv)
    k, v = sk.view(-1, H, D)[:n], sv.view(-1, H, D)[:n]
    assert float((k.float() - K.float()).norm() / K.float().norm()) < 0.5   # the pool's pages, in order
    seen = (torch.rand((n, H * G), generator=g, device="cuda") * (at[:, None] + 1)).long()
    kj = k.float()[seen, torch.arange(H * G, device="cuda") // G]
    q = (kj * (12 * math.sqrt(D) / kj.square().sum(-1, keepdim=True))).half()
    qs = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    want, wl, mag = _formula(q, k, v, [0, n], 1 / math.sqrt(D))
    dots = torch.einsum("thgd,khd->thgk", q.double().abs().view(n, H, G, D), k.double().abs())
    e = (2.0 ** -19 / math.sqrt(D)) * dots.amax(-1).view(n, H * G)
    u, vmax = 2.0 ** -11, float(v.abs().max())
    a, la = fused.prompt_attention(q, k, v, qs)
    b, lb = fused.prefill(pool, 0, q, qs, pages[None], torch.tensor([n], device="cuda"))
    pool.check()
    for got, lse, p_step, small in ((a, la, u, n * 2.0 ** -25 * vmax), (b, lb, 0.0, 0.0)):
        tol = (p_step + 2 * e[..., None] + 2.0 ** -17) * mag + u * want.abs() + small + 2.0 ** -25
        err = (got.double() - want).abs()
        assert bool((err <= tol).all()), f"worst {(err - tol).max()} over"
        assert bool(((lse.double() - wl).abs() <= e + 2.0 ** -18 + wl.abs() * 2.0 ** -22).all())


def test_hook_prompts_are_the_functions_and_its_lse_the_formulas():
    import types

    from kvquant import compact_backend as cb
    from kvquant import fused
    n, H, G, D = 70, 2, 7, 128
    q, k, v, start = _make([n, n, n], H * G, H, D, torch.bfloat16, seed=91)
    qs = torch.tensor(start, dtype=torch.int32, device="cuda")
    meta = types.SimpleNamespace(num_actual_tokens=3 * n, max_query_len=n, max_seq_len=n, query_start_loc=qs)
    buf = torch.zeros((3 * n + 2) * H * G * D + 1, dtype=torch.bfloat16, device="cuda")
    want, wl, mag = _formula(q, k, v, start, 0.07)
    o, lse = fused.prompt_attention(q, k, v, qs, softmax_scale=0.07)
    _check(o, lse, want, wl, mag, v, n, torch.ones(3 * n, dtype=torch.bool, device="cuda"))
    for shift in (0, 1):   # on and off the 16-byte alignment
        out = buf.zero_()[shift:shift + (3 * n + 2) * H * G * D].view(-1, H * G, D)
        cb.prompts_into(q, k, v, meta, out, scale=0.07)
        assert torch.equal(out[:3 * n], o) and not out[3 * n:].any()
