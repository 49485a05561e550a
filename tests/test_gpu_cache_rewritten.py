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


@pytest.mark.parametrize("kind", ["", "int8", "int4"])
def test_a_call_behind_an_event_of_another_stream(kind):
    """Between two calls on one stream it waits for another stream that writes the queries, the lengths and the caches: the
    second call's first kernel, though launched early, starts behind that."""
    from topk_attn_b200 import ops
    B, H, Np, N = 20, 2, 600, 40
    g = torch.Generator(device=DEV).manual_seed(5)
    sets = [(torch.randn(B, 4 * H, 128, generator=g, device=DEV).half(), torch.randn(Np, H, 128, generator=g, device=DEV).half(),
             torch.randn(B, N, H, 128, generator=g, device=DEV).half(),
             torch.randint(0, N + 1, (B,), generator=g, device=DEV, dtype=torch.int32)) for _ in range(3)]
    q, lens = torch.empty_like(sets[0][0]), torch.empty_like(sets[0][3])
    if kind:
        prefix, cache = ops.quantized_kv_cache(Np, H, kind, device=DEV), ops.quantized_kv_cache(N, H, kind, batch=B, device=DEV)
    else:
        prefix, cache = ((torch.empty_like(sets[0][i]), torch.empty_like(sets[0][i])) for i in (1, 2))

    def write(i):
        q.copy_(sets[i][0])
        lens.copy_(sets[i][3])
        for c, x in ((prefix, sets[i][1]), (cache, sets[i][2])):
            if kind:
                ops.kv_append_quantized(c, x, x.neg(), 0)
            else:
                c[0].copy_(x)
                c[1].copy_(x.neg())
    want = []
    for i in range(3):
        write(i)
        torch.cuda.synchronize()
        want.append(ops.shared_prefix_attention(q, prefix, cache, SM, lens))
        torch.cuda.synchronize()
    one, other = torch.cuda.Stream(), torch.cuda.Stream()
    got = []
    for i in range(12):
        with torch.cuda.stream(other):
            other.wait_stream(one)
            torch.cuda._sleep(100000)
            write(i % 3)
        with torch.cuda.stream(one):
            ops.shared_prefix_attention(sets[0][0], (sets[0][1], sets[0][1]), None, SM)      # what comes before, on one
            one.wait_stream(other)
            got.append(ops.shared_prefix_attention(q, prefix, cache, SM, lens))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want[i % 3]) for i, x in enumerate(got))
