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
