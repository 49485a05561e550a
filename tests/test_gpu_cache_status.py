"""What a graph's kernels report, and the scratch that calls keep."""
import math
import os
import subprocess
import sys

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def in_a_new_process(code, word):
    res = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert word in res.stdout, res.stderr[-2000:]


def test_a_graph_captured_before_any_other_call_reports_what_its_replays_meet():
    """Positions and lengths that go out of range only at a replay."""
    in_a_new_process("""
import torch
from topk_attn_b200 import capi, ops
cache = ops.quantized_kv_cache(8, 2, "int8", batch=3)
rows = torch.randn(3, 2, 2, 128, device="cuda", dtype=torch.float16)
q = torch.randn(3, 4, 128, device="cuda", dtype=torch.float16)
at, lens = (torch.zeros(3, device="cuda", dtype=torch.int32) for _ in range(2))
graphs = []
torch.cuda.synchronize()
for call in (lambda: ops.kv_append_quantized(cache, rows, rows, at), lambda: ops.kv_dequantize(cache, at, 2),
             lambda: ops.flash_decoding_quantized(q, cache, 0.1, lens)):
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call()
    graphs.append(g)
for g in graphs:
    g.replay()
ops.check_status()
for g, bad in zip(graphs, (at, at, lens)):
    for value in (9, -1):
        bad.fill_(value)
        g.replay()
        try:
            ops.check_status()
        except capi.RaError:
            ops.clear_status()
        else:
            raise SystemExit("nothing reported")
    bad.zero_()
    g.replay()
    ops.check_status()
print("all reported")
""", "all reported")
