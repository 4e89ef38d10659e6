"""Shared-prefix decode where the sequences' own pages outweigh the prefix: many
key tiles a suffix, on both streams, against the float64 oracle."""
from __future__ import annotations

import math

import pytest

from test_gpu_prefix import D, _build, _check, _i32, _q

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits,prefix,suffixes,G", [((4, 4), 32, [2500, 1, 0, 1281, 640], 7),
                                                    ((2, 2), 16, [1919, 2048], 4), ((4, 4), 0, [3000, 5], 8),
                                                    ((2, 4), 144, [1000] * 40, 4)])
def test_long_suffixes(bits, prefix, suffixes, G):
    from kvquant import fused
    gpu, orc, table = _build(bits, prefix, suffixes, seed=61, t_cal=700)
    lens = [prefix + s for s in suffixes]
    q = _q(len(lens), 2 * G, 62)
    out, lse = fused.shared_prefix_decode(gpu, 0, q, _i32(table), _i32(lens), prefix)
    gpu.check()
    _check(gpu, orc, table, lens, q, out, lse, 1 / math.sqrt(D), "logical")


def test_padding_rows_before_the_first_sequence():
    """The first rows have ended: length 0, their table rows cleared. The prefix
    is read from the first row that has a sequence; with none, nothing is read."""
    import torch
    from kvquant import fused
    gpu, orc, table = _build((4, 4), 400, [50, 7, 300, 20], seed=63)
    q = _q(4, 14, 64)
    for ended in (1, 2, 3, 4):
        t = table.copy()
        t[:ended] = -1
        lens = [0] * ended + [450, 407, 700, 420][ended:]
        out, lse = fused.shared_prefix_decode(gpu, 0, q, _i32(t), _i32(lens), 400)
        gpu.check()
        _check(gpu, orc, table, lens, q, out, lse, 1 / math.sqrt(D), "logical")
        assert bool(torch.isfinite(out).all())
