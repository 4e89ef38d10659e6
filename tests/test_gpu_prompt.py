"""GPU parity of the whole-prompt attention against the formula in 64 bits.

Tolerance. The inputs are exact and products are summed in fp32, so what is
left is one rounding of each probability to the input type and one of the
output, each at most half a step u = eps / 2 of the value. With p'_j = p_j (1 +
e_j), |e_j| <= u, the output moves by at most u * sum_j p_j |v_j| <= u * A, A
= the softmax average of |v|, and then by u |o| (1 + u). fp32 sums of up to n
terms, exp2 and the division add less than 2^-18 A here (scores below 2^6:
2^-24 * 2^6 each, averaged over the row), so the bound is
(u + 2^-17) A + u |o|. fp16 probabilities below 2^-14 of the row's maximum
have an absolute step of 2^-25 instead: at most n 2^-25 max|v| / l in all, l
>= 1 the sum of exponentials relative to the maximum; n 2^-25 max|v| covers
it, and the P in use may be relative to a maximum 2^8 smaller, which only
shrinks that share. lse: fp32 scores and sums, 2^-18 + |lse| 2^-22.
"""
from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def _formula(q, k, v, start, scale):
    """Row by row in 64 bits; a row outside every prompt stays None-like (NaN)."""
    T, Hq, D = q.shape
    g = Hq // k.shape[1]
    out = torch.full((T, Hq, D), math.nan, dtype=torch.float64, device="cuda")
    lse = torch.full((T, Hq), math.nan, dtype=torch.float64, device="cuda")
    mag = torch.zeros((T, Hq, D), dtype=torch.float64, device="cuda")
    for a, e in zip(start[:-1], start[1:]):
        n = e - a
        if n <= 0:
            continue
        keep = torch.ones((n, n), dtype=torch.bool, device="cuda").tril()
        for h in range(Hq):
            vv = v[a:e, h // g].double()
            s = torch.where(keep, q[a:e, h].double() @ k[a:e, h // g].double().T * scale, -math.inf)
            z = torch.logsumexp(s, 1)
            p = torch.exp(s - z[:, None])
            out[a:e, h], mag[a:e, h], lse[a:e, h] = p @ vv, p @ vv.abs(), z
    return out, lse, mag


def _check(got, lse, want, wl, mag, v, longest, inside):
    u = torch.finfo(got.dtype).eps / 2
    tiny = longest * 2.0 ** -25 * v.double().abs().max() if got.dtype == torch.float16 else 0.0
    tol = (u + 2.0 ** -17) * mag + u * want.abs() + tiny + (2.0 ** -25 if got.dtype == torch.float16 else 0.0)
    err = (got.double() - want).abs()
    assert bool((err[inside] <= tol[inside]).all()), f"worst {((err - tol)[inside]).max()} over"
    dl = (lse.double() - wl).abs()[inside]
    assert bool((dl <= 2.0 ** -18 + wl[inside].abs() * 2.0 ** -22).all()), f"lse off by {dl.max()}"


def _make(lens, Hq, H, D, dt, seed, lead=0, tail=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    T = lead + sum(lens) + tail
    qkv = torch.randn((T, Hq + 2 * H, D), generator=g, device="cuda").to(dt)
    start = [lead]
    for n in lens:
        start.append(start[-1] + n)
    return qkv[:, :Hq], qkv[:, Hq:Hq + H], qkv[:, Hq + H:], start


LENGTHS = [[1], [2], [17, 18, 19], [127, 128, 129], [1, 0, 5, 0, 0, 300, 1], [36, 37, 255, 256, 257], [1100], [0],
           [640, 1, 333]]


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("Hq,H,D", [(28, 4, 128), (3, 3, 128), (8, 1, 64), (16, 4, 64)])
@pytest.mark.parametrize("lens", LENGTHS)
def test_matches_the_formula(lens, Hq, H, D, dt):
    import hxlib
    from kvquant import fused
    q, k, v, start = _make(lens, Hq, H, D, dt, seed=sum(lens) + D, lead=3, tail=4)
    T = q.shape[0]
    out = torch.full((T, Hq, D), 7.0, dtype=dt, device="cuda")
    lse = torch.full((T, Hq), 9.0, device="cuda")
    qs = torch.tensor(start, dtype=torch.int32, device="cuda")
    got, gl = fused.prompt_attention(q, k, v, qs, out=out, lse=lse)
    hxlib.check_device_errors()
    assert got is out and gl is lse
    want, wl, mag = _formula(q, k, v, start, 1 / math.sqrt(D))
    inside = torch.zeros(T, dtype=torch.bool, device="cuda")
    inside[start[0]:start[-1]] = True
    # rows outside every prompt are left as they were
    assert bool((out[~inside] == 7).all()) and bool((lse[~inside] == 9).all())
    _check(out, lse, want, wl, mag, v, max(lens), inside)


@pytest.mark.parametrize("Hq,H", [(128, 1), (96, 1), (130, 2), (5, 1)])
def test_group_sizes(Hq, H):
    import hxlib
    from kvquant import fused
    q, k, v, start = _make([70, 9], Hq, H, 64, torch.float16, seed=Hq)
    out, lse = fused.prompt_attention(q, k, v, torch.tensor(start, dtype=torch.int32, device="cuda"), softmax_scale=0.2)
    hxlib.check_device_errors()
    want, wl, mag = _formula(q, k, v, start, 0.2)
    _check(out, lse, want, wl, mag, v, 70, torch.ones(79, dtype=torch.bool, device="cuda"))


def test_many_prompts_of_every_length():
    import hxlib
    from kvquant import fused
    lens = [(7 * i) % 90 for i in range(300)]
    q, k, v, start = _make(lens, 7, 1, 128, torch.bfloat16, seed=1)
    out, lse = fused.prompt_attention(q, k, v, torch.tensor(start, dtype=torch.int32, device="cuda"))
    hxlib.check_device_errors()
    want, wl, mag = _formula(q, k, v, start, 1 / math.sqrt(128))
    _check(out, lse, want, wl, mag, v, 90, torch.ones(q.shape[0], dtype=torch.bool, device="cuda"))


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
def test_maximum_that_keeps_rising(dt):
    """Scores that rise along the row by far more than the rescale slack, and
    rows with large negative scores."""
    import hxlib
    from kvquant import fused
    n, D = 900, 128
    g = torch.Generator(device="cuda").manual_seed(3)
    q = torch.randn((n, 2, D), generator=g, device="cuda")
    k = torch.randn((n, 1, D), generator=g, device="cuda") * 0.05
    q[..., 0], k[..., 0] = 4.0, torch.arange(n, device="cuda")[:, None] / 16.0
    q[:, 1, 0] = -4.0
    q, k = q.to(dt), k.to(dt)
    v = torch.randn((n, 1, D), generator=g, device="cuda").to(dt)
    out, lse = fused.prompt_attention(q, k, v, torch.tensor([0, n], dtype=torch.int32, device="cuda"))
    hxlib.check_device_errors()
    want, wl, mag = _formula(q, k, v, [0, n], 1 / math.sqrt(D))
    _check(out, lse, want, wl, mag, v, n, torch.ones(n, dtype=torch.bool, device="cuda"))


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_masked_places_may_hold_anything(dt, value):
    """A token's K and V reach only the rows that see it, whatever they hold:
    the prompts before it, the tokens before it and the rows past the last
    prompt stay as without it; V's value reaches the rows that do see it."""
    import hxlib
    from kvquant import fused
    lens, D = [150, 90, 200], 128
    q, k, v, start = _make(lens, 14, 2, D, dt, seed=8, tail=50)
    qs = torch.tensor(start, dtype=torch.int32, device="cuda")
    clean, cl = fused.prompt_attention(q, k, v, qs)
    v2, k2 = v.clone(), k.clone()
    at = start[1] + 40
    v2[at, 0, 5] = value
    k2[start[2] + 170], v2[start[2] + 170] = value, value
    k2[start[3]:], v2[start[3]:] = value, value
    out, lse = fused.prompt_attention(q, k2, v2, qs)
    hxlib.check_device_errors()
    n = start[3]
    same = torch.ones((n, 14, D), dtype=torch.bool, device="cuda")
    same[at:start[2], :7, 5] = False
    same[start[2] + 170:] = False
    assert torch.equal(out[:n][same], clean[:n][same])
    assert torch.equal(lse[:start[2] + 170], cl[:start[2] + 170])
    hit = out[at:start[2], :7, 5].float()
    assert bool((torch.isnan(hit) if math.isnan(value) else hit == value).all())
    late = out[start[2] + 170:n].float()
    assert bool((~torch.isfinite(late)).all())


def test_layouts_streams_and_repeats():
    """Contiguous, sliced, transposed and misaligned layouts give the same bits, and so do
    a second run, another stream and a captured graph."""
    from kvquant import fused
    q, k, v, start = _make([333, 64], 8, 2, 64, torch.float16, seed=4)
    qs = torch.tensor(start, dtype=torch.int32, device="cuda")
    out, lse = fused.prompt_attention(q, k, v, qs)
    heads_first = [t.permute(1, 0, 2).contiguous().permute(1, 0, 2) for t in (q, k, v)]
    odd = torch.zeros((q.shape[0], 12, 67), dtype=torch.float16, device="cuda")
    odd[:, :8, 3:] = q
    forms = [(q.contiguous(), k.contiguous(), v.contiguous()), heads_first, (odd[:, :8, 3:], k, v), (q, k, v)]
    for a, b, c in forms:
        o2, l2 = fused.prompt_attention(a, b, c, qs)
        assert torch.equal(o2, out) and torch.equal(l2, lse)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        o3, l3 = fused.prompt_attention(q, k, v, qs)
    side.synchronize()
    assert torch.equal(o3, out) and torch.equal(l3, lse)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o4, l4 = fused.prompt_attention(q, k, v, qs)
    qs2 = torch.tensor([0, 64, q.shape[0]], dtype=torch.int32, device="cuda")
    graph.replay()
    assert torch.equal(o4, out) and torch.equal(l4, lse)
    qs.copy_(qs2)          # other lengths of the same total, in the captured call
    graph.replay()
    o5, l5 = fused.prompt_attention(q, k, v, qs2)
    assert torch.equal(o4, o5) and torch.equal(l4, l5)


def test_query_start_out_of_range_is_flagged():
    import hxlib
    from kvquant import fused
    q, k, v, _ = _make([50], 4, 2, 64, torch.float16, seed=6)
    fused.prompt_attention(q, k, v, torch.tensor([0, 51], dtype=torch.int32, device="cuda"))
    with pytest.raises(hxlib.HelixError, match="out of range"):
        hxlib.check_device_errors()
    fused.prompt_attention(q, k, v, torch.tensor([30, 20], dtype=torch.int32, device="cuda"))
    with pytest.raises(hxlib.HelixError, match="out of range"):
        hxlib.check_device_errors()


def test_close_to_the_pool_prefill():
    """The same prompt through the pool (nuq4) differs from the unquantised
    result by the quantisation, a few per cent of its norm."""
    from kvquant import fused
    from kvquant.compact_pool import CompactKVPool
    from kvquant.synthetic import NUQ4, make_kv, make_scales
    n, H = 200, 4
    sc = make_scales([NUQ4], H, 128, t_cal=256, seed=11)
    pool = CompactKVPool(1, 16, 16, H, 128, sc)
    K, V = make_kv(n, H, 128, seed=12, chan_seed=11)
    at = torch.arange(n, device="cuda")
    pool.write_kv(0, K, V, at, at)
    g = torch.Generator(device="cuda").manual_seed(13)
    q = (torch.randn((n, 28, 128), generator=g, device="cuda") * 0.1).half()
    qs = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    bt = torch.arange(13, dtype=torch.int32, device="cuda")[None]
    a, _ = fused.prompt_attention(q, K, V, qs)
    b, _ = fused.prefill(pool, 0, q, qs, bt, torch.tensor([n], device="cuda"))
    pool.check()
    assert float((a.float() - b.float()).norm() / a.float().norm()) < 0.25


def test_thousands_of_one_token_prompts():
    """Each token sees itself alone: the output is its V, the lse its score."""
    import hxlib
    from kvquant import fused
    n = 3001
    q, k, v, start = _make([1] * n, 4, 2, 64, torch.float16, seed=31)
    out, lse = fused.prompt_attention(q, k, v, torch.tensor(start, dtype=torch.int32, device="cuda"))
    hxlib.check_device_errors()
    assert torch.equal(out, v.repeat_interleave(2, 1))
    s = (q.double() * k.double().repeat_interleave(2, 1)).sum(-1) / 8
    assert bool(((lse.double() - s).abs() <= 2.0 ** -18 + s.abs() * 2.0 ** -22).all())
