"""The first call of a process made inside a graph capture: the error word it
creates belongs to the process, not to the graph, and no replay clears it."""
from __future__ import annotations

import subprocess
import sys
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu

CODE = """
import torch, hxlib
from kvquant import fused, paging
i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
table, lens, new, free, count = i32([[-1, -1]]), i32([0]), i32([3]), i32([0, 1]), i32([2])
q = torch.randn(3, 2, 64, device="cuda").half()
start = i32([0, 3])
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    if "CALL" == "tables":
        out = paging.extend_tables(table, lens, new, free, count, num_tokens=3)
    else:
        out, lse = fused.prompt_attention(q, q, q, start)
g.replay()
hxlib.check_device_errors()
bad = new if "CALL" == "tables" else start
was = bad.clone()
bad[-1] = 50          # more tokens than the slot map has, or than there are
g.replay()
bad.copy_(was)
g.replay()            # a good replay after the bad one
try:
    hxlib.check_device_errors()
except hxlib.HelixError as e:
    assert "out of range" in str(e)
else:
    raise SystemExit("the error was lost")
hxlib.check_device_errors()
del g
torch.cuda.empty_cache()
x = torch.full((1 << 20,), 7, dtype=torch.int32, device="cuda")
hxlib.check_device_errors()
"""


@pytest.mark.parametrize("call", ["tables", "prompt"])
def test_errors_survive_replays(call):
    root = Path(__file__).resolve().parents[1] / "helix-lite_b200"
    r = subprocess.run([sys.executable, "-c", CODE.replace("CALL", call)], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout[-500:] + r.stderr[-1500:]
