"""Writing rows into a quantised cache and reading them back, against the 64-bit restatement: codes and
scales are equal, bit for bit, at the sizes, strides and values where a quantiser can go wrong."""
import math

import pytest
import torch

from oracle import cache_oracle as O

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
KINDS = ["int8", "fp8", "int4"]
DTYPES = [torch.float16, torch.bfloat16]


def rows(shape, dtype, seed, spread=True):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g)
    if spread:   # magnitudes over many binades, row by row
        x = x * torch.exp2(torch.randint(-8, 8, shape[:-1] + (1,), generator=g).float())
    return x.to(dtype)


def held(cache):
    """(codes float64, scales) of a cache's k or v as the restatement lays them out."""
    out = []
    for c, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
        c, s = c.cpu(), s.cpu()
        if cache.kind == "int4":
            c = torch.stack(((c & 15).double() - 8, (c >> 4).double() - 8), -1).flatten(-2)
            s = s.transpose(-3, -2)
        else:
            c = c.double()
            s = s.transpose(-2, -1).unsqueeze(-1)
        out.append((c, s))
    return out


def check(cache, at, x, which, counts=None):
    """Cache rows at the tokens at[b].. hold x [B,T,H,128]; all others are as they were (zeros)."""
    codes, scales = held(cache)[which]
    if not cache.per_row:
        codes, scales = codes[None], scales[None]
    want_c, want_s = torch.zeros_like(codes), torch.zeros_like(scales)
    if cache.kind == "int4":
        want_c -= 8          # untouched bytes are zero
    rc, rs, _ = O.quantize(x, cache.kind)
    for b in range(x.size(0)):
        n = x.size(1) if counts is None else max(0, min(x.size(1), int(counts[b])))
        want_c[b, at[b]:at[b] + n] = rc[b, :n]
        want_s[b, at[b]:at[b] + n] = rs[b, :n]
    assert torch.equal(codes, want_c)
    assert torch.equal(torch.nan_to_num(scales, nan=-1.0), torch.nan_to_num(want_s, nan=-1.0))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,T,H", [(1, 1, 1), (3, 1, 5), (2, 77, 8), (1, 1000, 2), (5, 33, 32)])
def test_append_holds_the_defined_codes(kind, dtype, B, T, H):
    from topk_attn_b200 import ops
    k, v = rows((B, T, H, 128), dtype, T + H), rows((B, T, H, 128), dtype, T + H + 1)
    cache = ops.quantized_kv_cache(T + 9, H, kind, batch=B, device=DEV)
    at = torch.arange(B, dtype=torch.int32) % 9
    ops.kv_append_quantized(cache, k.to(DEV), v.to(DEV), at.to(DEV))
    ops.check_status(torch.device(DEV))
    check(cache, at.tolist(), k, 0)
    check(cache, at.tolist(), v, 1)
    for out_type in DTYPES:
        kb, vb = ops.kv_dequantize(cache, at.to(DEV), T, out_type)
        for back, x in ((kb, k), (vb, v)):
            want = O.quantize(x, kind)[2]
            # one fp32 rounding of code * scale, one of the result's type, half a step each
            rel = 2.0 ** -24 + torch.finfo(out_type).eps / 2 * (1 + 2.0 ** -24)
            far = (back.cpu().double() - want).abs()
            assert (far <= rel * want.abs() + 2.0 ** -25).all()


@pytest.mark.parametrize("kind", KINDS)
def test_ties_and_their_neighbours_round_to_even_of_the_exact_quotient(kind):
    """Values at and next to the borders between codes: every border of a row whose scale is a power of
    two is a tie, and the neighbours of the borders are the values a rounded quotient gets wrong."""
    from topk_attn_b200 import ops
    top = {"int8": 127.0, "fp8": 448.0, "int4": 7.0}[kind]
    out = []
    for amax in (top, top * 2.0 ** -3, 1.0, 100.0, 3.140625):
        step = amax / top
        border = (torch.arange(42).double() * (3 if kind == "int8" else 0.16) + 0.5) * step
        near = torch.stack((border, border * (1 + 2.0 ** -10), border * (1 - 2.0 ** -10)), 1).flatten()
        row = torch.cat((near, torch.tensor([0.0, amax]))).clamp(max=amax)
        out.append(row * torch.where(torch.arange(128) % 2 == 0, 1.0, -1.0))
    x = torch.stack(out).half()
    if kind == "int4":
        x[:, 31::32] = torch.tensor([7.0, 0.875, 1.0, 100.0, 3.140625]).half()[:, None]
        x = torch.minimum(x.abs(), x[:, 31:32].abs()) * torch.sign(x)
    x = x.view(1, -1, 1, 128)
    cache = ops.quantized_kv_cache(x.size(1), 1, kind, batch=1, device=DEV)
    ops.kv_append_quantized(cache, x.to(DEV), x.to(DEV), 0)
    check(cache, [0], x, 0)


@pytest.mark.parametrize("kind", KINDS)
def test_special_rows(kind):
    """All zeros, tiny, subnormal, huge, infinite and NaN rows; only the row (int4: group) concerned is
    spoilt."""
    from topk_attn_b200 import ops
    x = rows((1, 10, 2, 128), torch.bfloat16, 3, spread=False)
    x[0, 0] = 0
    x[0, 1] *= 2.0 ** -110
    x[0, 2] *= 2.0 ** -96
    x[0, 3] *= 2.0 ** 120
    x[0, 4, 0, 5] = math.inf
    x[0, 5, 1, 70] = math.nan
    x[0, 6, 0, 127] = -math.inf
    x[0, 7] = 2.0 ** -133
    x[0, 8, :, 1:] = 0
    cache = ops.quantized_kv_cache(10, 2, kind, batch=1, device=DEV)
    ops.kv_append_quantized(cache, x.to(DEV), x.to(DEV), 0)
    ops.check_status(torch.device(DEV))
    check(cache, [0], x, 0)
    check(cache, [0], x, 1)
    kb, _ = ops.kv_dequantize(cache, 0, 10, torch.bfloat16)
    want = O.quantize(x, kind)[2]
    assert torch.equal(torch.isnan(kb.cpu()), torch.isnan(want))
    kb, vb = ops.kv_dequantize(cache, 4, dtype=torch.bfloat16)
    assert kb.shape == (1, 6, 2, 128)


@pytest.mark.parametrize("kind", KINDS)
def test_padded_batch_counts_and_rows_behind_are_left_alone(kind):
    from topk_attn_b200 import ops
    B, T, H = 6, 40, 3
    k, v = rows((B, T, H, 128), torch.float16, 1), rows((B, T, H, 128), torch.float16, 2)
    counts = torch.tensor([0, 1, 39, 40, -3, 1000], dtype=torch.int32)
    at = torch.tensor([0, 5, 60, 24, 1, 0], dtype=torch.int32)
    cache = ops.quantized_kv_cache(100, H, kind, batch=B, device=DEV)
    ops.kv_append_quantized(cache, k.to(DEV), v.to(DEV), at.to(DEV), counts.to(DEV))
    ops.check_status(torch.device(DEV))
    check(cache, at.tolist(), k, 0, counts)
    check(cache, at.tolist(), v, 1, counts)


def test_a_padded_batch_may_reach_over_the_end_of_the_cache():
    """With an int position the rows that counts leaves out need no room."""
    from topk_attn_b200 import ops
    k = rows((2, 8, 3, 128), torch.float16, 1)
    counts = torch.tensor([2, 0], dtype=torch.int32)
    cache = ops.quantized_kv_cache(10, 3, "fp8", batch=2, device=DEV)
    ops.kv_append_quantized(cache, k.to(DEV), k.to(DEV), 8, counts.to(DEV))
    ops.check_status(torch.device(DEV))
    check(cache, [8, 8], k, 0, counts)


def test_rows_outside_the_cache_are_left_out_and_reported():
    from topk_attn_b200 import capi, ops
    dev = torch.device(DEV)
    B, T, H = 3, 4, 2
    k = rows((B, T, H, 128), torch.float16, 1)
    cache = ops.quantized_kv_cache(8, H, "int8", batch=B, device=DEV)
    at = torch.tensor([6, -2, 2], dtype=torch.int32, device=DEV)
    try:
        ops.kv_append_quantized(cache, k.to(DEV), k.to(DEV), at)
        with pytest.raises(capi.RaError):
            ops.check_status(dev)
        ops.clear_status(dev)
        ops.check_status(dev)
        full = O.quantize(k, "int8")[0]
        got = held(cache)[0][0]
        assert torch.equal(got[0, 6:], full[0, :2]) and not got[0, :6].any()
        assert torch.equal(got[1, :2], full[1, 2:]) and not got[1, 2:].any()
        assert torch.equal(got[2, 2:6], full[2])
        kb, _ = ops.kv_dequantize(cache, at, T)
        assert not kb[0, 2:].any() and not kb[1, :2].any() and kb[0, 1].any()
        with pytest.raises(capi.RaError):
            ops.check_status(dev)
    finally:
        ops.clear_status(dev)


def test_strided_rows_strided_caches_and_one_shared_cache():
    from topk_attn_b200 import ops
    B, T, H = 2, 19, 4
    qkv = rows((B, T, 3 * H, 128), torch.bfloat16, 5)
    k, v = qkv[:, :, H:2 * H], qkv[:, :, 2 * H:]
    big = ops.quantized_kv_cache(64, 2 * H, "fp8", batch=B, device=DEV)
    part = ops.QuantizedKV(big.k[:, 8:40, H:], big.v[:, 8:40, H:], big.k_scale[:, H:, 8:40], big.v_scale[:, H:, 8:40])
    d = qkv.to(DEV)
    ops.kv_append_quantized(part, d[:, :, H:2 * H], d[:, :, 2 * H:], 13)
    check(part, [13] * B, k, 0)
    check(part, [13] * B, v, 1)
    whole = held(big)[0][0]
    assert not whole[:, :21].any() and not whole[:, :, :H].any()
    shared = ops.quantized_kv_cache(30, H, "int4", device=DEV)
    ops.kv_append_quantized(shared, d[0, :, H:2 * H], d[0, :, 2 * H:], torch.tensor([7], dtype=torch.int32, device=DEV))
    check(shared, [7], k[:1], 0)
    kb, vb = ops.kv_dequantize(shared.first(9), 7)
    assert kb.shape == (2, H, 128)
    ops.check_status(torch.device(DEV))


def test_refusals():
    from topk_attn_b200 import capi, ops
    cache = ops.quantized_kv_cache(8, 2, "int8", batch=2, device=DEV)
    good = torch.zeros(2, 3, 2, 128, dtype=torch.float16, device=DEV)
    for k, v in [(good.float(), good.float()), (good.cpu(), good.cpu()), (good[:1], good[:1]), (good, good[:, :2]),
                 (good[..., :64], good[..., :64]), (good, good.bfloat16()), (good[:, :, :1], good[:, :, :1]),
                 (good.transpose(2, 3).contiguous().transpose(2, 3), good)]:
        with pytest.raises(ValueError):
            ops.kv_append_quantized(cache, k, v, 0)
    with pytest.raises(ValueError):
        ops.kv_append_quantized(cache, good, good, torch.zeros(2, dtype=torch.int64, device=DEV))
    with pytest.raises(ValueError):
        ops.kv_append_quantized(cache, good, good, 0, torch.zeros(3, dtype=torch.int32, device=DEV))
    off = torch.zeros(good.numel() + 1, dtype=torch.float16, device=DEV)[1:].view(good.shape)
    for args in [(good, good, 6), (good, good, -1), (off, good, 0)]:
        with pytest.raises(capi.RaError):
            ops.kv_append_quantized(cache, *args)
    with pytest.raises(ValueError):
        ops.kv_dequantize(cache, 0, 3, torch.float32)
    with pytest.raises(ValueError):
        ops.kv_dequantize(cache, torch.zeros(2, dtype=torch.int32, device=DEV))
    with pytest.raises(capi.RaError):
        ops.kv_dequantize(cache, 5, 4)
    with pytest.raises(ValueError):
        ops.quantized_kv_cache(8, 2, "int3")
    ops.kv_append_quantized(cache, good[:, :0], good[:, :0], 0)
    assert ops.kv_dequantize(cache, 8)[0].shape == (2, 0, 2, 128)
    ops.check_status(torch.device(DEV))
