"""Random shapes, formats, storages and lengths in one run each: attention at the element-by-element bound, appended and
read-back rows bit for bit."""
import math
import random

import pytest
import torch

from oracle import cache_oracle as O

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
SM = 1.0 / math.sqrt(128)


def stored(x, how):
    """The same values in another storage: dense, heads before tokens, a slice of a larger tensor, tokens before rows."""
    if how == 1:
        return x.transpose(-3, -2).contiguous().transpose(-3, -2)
    if how == 2:
        raw = x.contiguous().view(torch.uint8)
        big = torch.full((*raw.shape[:-3], raw.size(-3) + 3, raw.size(-2) + 2, raw.size(-1)), 0x7f, device=DEV, dtype=torch.uint8)
        big[..., 2:2 + raw.size(-3), 1:1 + raw.size(-2), :] = raw
        return big.view(x.dtype)[..., 2:2 + raw.size(-3), 1:1 + raw.size(-2), :]
    if how == 3 and x.dim() == 4:
        return x.transpose(0, 1).contiguous().transpose(0, 1)
    return x.contiguous()


def decoded(codes, scales, kind):
    scales = scales.double()
    if kind == "int4":
        x = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).double() - 8
        return (x.unflatten(-1, (4, 32)) * scales.transpose(-3, -2)[..., None]).flatten(-2)
    return codes.double() * scales.transpose(-2, -1)[..., None]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("kind", ["", "int8", "fp8", "int4"])
def test_attention_over_random_shapes(kind, dtype):
    from topk_attn_b200 import ops
    rng, g = random.Random(7), torch.Generator(device=DEV).manual_seed(7)
    for _ in range(40):
        H, G, B = rng.choice([1, 2, 3, 8]), rng.choice([1, 2, 3, 5, 7, 8, 9, 12, 17, 40]), rng.randrange(1, 60)
        Np, N = rng.choice([0, rng.randrange(1, 900)]), rng.choice([0, rng.randrange(1, 300)])
        q = (torch.randn(B, H * G, 128, generator=g, device=DEV) * rng.choice([0.05, 0.5, 2.0])).to(dtype)
        args, vals, scales = [], [], []
        for shape in ((Np, H, 128), (B, N, H, 128)):
            if shape[-3] == 0:
                args.append(None), vals.append(None), scales.append(None)
                continue
            how = rng.randrange(4)
            pair = [(torch.randn(shape, generator=g, device=DEV) * torch.exp2(torch.randint(
                -4, 3, shape[:-1] + (1,), generator=g, device=DEV).float())).to(dtype) for _ in range(2)]
            if kind:
                c = ops.quantized_kv_cache(shape[-3], H, kind, batch=B if len(shape) == 4 else None)
                ops.kv_append_quantized(c, *pair, 0)
                vals.append((decoded(c.k, c.k_scale, kind), decoded(c.v, c.v_scale, kind)))
                scales.append(c.k_scale.transpose(-3, -2).amax(-1) if kind == "int4" else c.k_scale.transpose(-2, -1))
                args.append(ops.QuantizedKV(stored(c.k, how), stored(c.v, how), c.k_scale, c.v_scale))
            else:
                vals.append(tuple(pair)), scales.append(None)
                args.append(tuple(stored(x, how) for x in pair))
        if args == [None, None]:
            continue
        lens = torch.randint(0, N + 1, (B,), generator=g, device=DEV, dtype=torch.int32) if N and rng.random() < 0.7 else None
        given = q.clone()
        out = ops.shared_prefix_attention(given, *args, SM, lens, given if rng.random() < 0.3 else None)
        ref, mass, reach = O.attention_terms(q, SM, *vals, lens, scales, kind)
        # fp16 weights are 2^10 at least for the largest of a row, and their rests off by half of 2^-24 at most
        least = (Np + N) * 2.0 ** -35 * max(float(v[1].abs().max()) for v in vals if v) if kind or dtype == torch.float16 else 0.0
        assert ((out.double() - ref).abs() <= O.bound(ref, mass, reach, Np + N, dtype) + least).all(), (B, H, G, Np, N)
    ops.check_status(torch.device(DEV))


@pytest.mark.parametrize("kind", ["int8", "fp8", "int4"])
def test_rows_of_random_shapes_at_random_places(kind):
    """Positions and counts in and out of range, rows and caches in other storages; everything else stays as it was."""
    from topk_attn_b200 import capi, ops
    rng, g = random.Random(11), torch.Generator(device=DEV).manual_seed(11)
    for _ in range(60):
        B, T, H, N = rng.randrange(1, 8), rng.randrange(1, 120), rng.choice([1, 2, 3, 8, 33]), rng.randrange(1, 200)
        dtype, how = rng.choice([torch.float16, torch.bfloat16]), rng.randrange(4)
        k, v = ((torch.randn(B, T, H, 128, generator=g, device=DEV) * 4).to(dtype) for _ in range(2))
        big = ops.quantized_kv_cache(N + 3, H + 2, kind, batch=B)
        for x in (big.k, big.v):
            x.view(torch.uint8).random_(0, 120, generator=g)
        for x in (big.k_scale, big.v_scale):
            x.uniform_(0.1, 1, generator=g)
        cache = ops.QuantizedKV(big.k[:, 1:1 + N, 1:1 + H], big.v[:, 1:1 + N, 1:1 + H],
                                big.k_scale[:, 1:1 + H, 1:1 + N], big.v_scale[:, 1:1 + H, 1:1 + N])
        at = torch.randint(-T - 1, N + 2, (B,), generator=g, device=DEV, dtype=torch.int32)
        counts = torch.randint(-2, T + 3, (B,), generator=g, device=DEV, dtype=torch.int32)
        want = [x.clone() for x in (big.k, big.v, big.k_scale, big.v_scale)]
        outside = False
        for i, x in enumerate((k, v)):
            codes, scales = (y.to(DEV) for y in O.pack(*O.quantize(x.cpu(), kind)[:2], kind))
            for b, (p, c) in enumerate(zip(at.tolist(), counts.clamp(0, T).tolist())):
                outside |= c > 0 and (p < 0 or p + c > N)
                lo, hi = max(0, -p), min(c, N - p)
                if hi > lo:
                    want[i].view(torch.uint8)[b, 1 + p + lo:1 + p + hi, 1:1 + H] = codes.view(torch.uint8)[b, lo:hi]
                    want[2 + i][b, 1:1 + H, 1 + p + lo:1 + p + hi] = scales[b, :, lo:hi]
        try:
            ops.kv_append_quantized(cache, stored(k, how), stored(v, rng.randrange(4)), at, counts)
            if outside:
                with pytest.raises(capi.RaError):
                    ops.check_status(torch.device(DEV))
            else:
                ops.check_status(torch.device(DEV))
            for got, x in zip((big.k, big.v, big.k_scale, big.v_scale), want):
                assert torch.equal(got.view(torch.uint8), x.view(torch.uint8)), (B, T, H, N)
            back = ops.kv_dequantize(cache, at, T, dtype)
            for got, codes, scales in zip(back, want[:2], want[2:]):
                val = decoded(codes[:, 1:1 + N, 1:1 + H], scales[:, 1:1 + H, 1:1 + N], kind).float().to(dtype)
                for b, p in enumerate(at.tolist()):
                    lo, hi = min(T, max(0, -p)), max(0, min(T, N - p))
                    assert torch.equal(got[b, lo:hi], val[b, p + lo:p + hi] if hi > lo else got[b, :0])
                    assert not got[b, :lo].any() and not got[b, max(hi, 0):].any()
        finally:
            ops.clear_status(torch.device(DEV))
