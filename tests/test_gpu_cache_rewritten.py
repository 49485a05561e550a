"""Tokens that are written again and again while the kernels that read them are launched early: every call sees what
the call before it wrote."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
SM = 1.0 / math.sqrt(128)


@pytest.mark.parametrize("kind", ["int8", "fp8", "int4"])
@pytest.mark.parametrize("B,N,H", [(4, 96, 8), (2, 2000, 4)])
def test_read_back_after_writing_the_same_tokens(kind, B, N, H):
    """Read back, write other values, read back, without a pause; the new rows are written by the kernel before too."""
    from topk_attn_b200 import ops
    g = torch.Generator(device=DEV).manual_seed(1)
    base = [torch.randn(B, N, H, 128, generator=g, device=DEV).half() for _ in range(4)]
    cache = ops.quantized_kv_cache(N, H, kind, batch=B, device=DEV)
    want = []
    for x in base:
        ops.kv_append_quantized(cache, x, -x, 0)
        torch.cuda.synchronize()
        want.append(ops.kv_dequantize(cache))
        torch.cuda.synchronize()
    rows = torch.empty_like(base[0])
    got = []
    for i in range(60):
        rows.copy_(base[i % 4])
        ops.kv_append_quantized(cache, rows, base[i % 4].neg(), 0)
        got.append((i, ops.kv_dequantize(cache), ops.kv_dequantize(cache)))
    for i, *pairs in got:
        for k, v in pairs:
            assert torch.equal(k, want[i % 4][0]) and torch.equal(v, want[i % 4][1])
    ops.check_status(torch.device(DEV))


@pytest.mark.parametrize("kind", ["int8", "fp8", "int4"])
@pytest.mark.parametrize("B,G", [(3, 4), (40, 4)])
def test_attention_after_writing_the_same_tokens(kind, B, G):
    """A prefix and own caches that are written between two calls, and queries that are computed just before."""
    from topk_attn_b200 import ops
    H, Np, N = 2, 700, 50
    g = torch.Generator(device=DEV).manual_seed(2)
    sets = [(torch.randn(B, G * H, 128, generator=g, device=DEV).half(), torch.randn(Np, H, 128, generator=g, device=DEV).half(),
             torch.randn(B, N, H, 128, generator=g, device=DEV).half()) for _ in range(4)]
    prefix = ops.quantized_kv_cache(Np, H, kind, device=DEV)
    cache = ops.quantized_kv_cache(N, H, kind, batch=B, device=DEV)

    def step(i, pause):
        q, p, o = sets[i % 4]
        ops.kv_append_quantized(prefix, p, p.neg(), 0)
        if pause:
            torch.cuda.synchronize()
        ops.kv_append_quantized(cache, o, o.neg(), 0)
        q = q * 2
        if pause:
            torch.cuda.synchronize()
        return ops.shared_prefix_attention(q, prefix, cache, SM)
    want = [step(i, True) for i in range(4)]
    torch.cuda.synchronize()
    got = [step(i, False) for i in range(60)]
    assert all(torch.equal(x, want[i % 4]) for i, x in enumerate(got))
    ops.check_status(torch.device(DEV))
