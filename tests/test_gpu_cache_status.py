"""What a graph's kernels report, and the scratch that calls keep."""
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
    assert word in res.stdout and res.returncode == 0, res.stderr[-2000:]


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


def test_scratch_of_a_growing_batch_is_bounded():
    """A batch that grows row by row keeps one buffer of at most twice what the largest call needs."""
    in_a_new_process("""
import torch
from topk_attn_b200 import capi, ops
k, v = (torch.randn(160, 100, 8, 128, device="cuda", dtype=torch.bfloat16) for _ in range(2))
q = torch.randn(160, 32, 128, device="cuda", dtype=torch.bfloat16)
out = torch.empty_like(q)
for b in range(1, 161):
    ops.shared_prefix_attention(q[:b], None, (k[:b], v[:b]), 0.1, out=out[:b])
    if b == 1:
        torch.cuda.synchronize()
        start = torch.cuda.memory_allocated()
torch.cuda.synchronize()
need = max(capi.lib().ra_cache_attention_workspace_bytes(b, 32, 8, 0, 100) for b in range(1, 161))
grown = torch.cuda.memory_allocated() - start
assert grown <= 2 * need + (1 << 20), (grown, need)
for i in (0, 80, 159):
    alone = ops.shared_prefix_attention(q[i:i + 1], None, (k[i:i + 1], v[i:i + 1]), 0.1)
    assert (out[i].double() - alone[0].double()).abs().max() <= 2.0 ** -7 * alone.double().abs().max()
print("bounded")
""", "bounded")


def test_scratch_that_is_replaced_while_launches_use_it():
    """Calls that need ever more scratch behind one another without a pause, on two streams, with other tensors taken
    and given back between them, give what each gives alone."""
    from topk_attn_b200 import ops
    g = torch.Generator(device=DEV).manual_seed(3)
    pk, pv = (torch.randn(3000, 4, 128, generator=g, device=DEV).half() for _ in range(2))
    q = torch.randn(300, 16, 128, generator=g, device=DEV).half()
    sizes = [1, 2, 5, 9, 17, 40, 70, 129, 200, 300]
    want = [ops.shared_prefix_attention(q[:b].clone(), (pk, pv), None, 0.1) for b in reversed(sizes)][::-1]
    torch.cuda.synchronize()
    for _ in range(3):
        stream = torch.cuda.Stream()          # with a small buffer to begin with, whatever came before
        got = []
        with torch.cuda.stream(stream):
            for b in sizes:
                got.append(ops.shared_prefix_attention(q[:b], (pk, pv), None, 0.1))
                torch.empty(1 << 21, dtype=torch.uint8, device=DEV).fill_(255)
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, want))
