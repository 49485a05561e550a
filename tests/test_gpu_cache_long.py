"""Long contexts of which every tile counts, offsets beyond 32 bits and decode loops, held to the bound that tells a
wrong answer from a right one."""
import math

import pytest
import torch

from oracle import cache_oracle as O

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
SM = 1.0 / math.sqrt(128)
FORMS = [("", torch.float16), ("", torch.bfloat16), ("int8", torch.float16), ("int8", torch.bfloat16),
         ("fp8", torch.float16), ("fp8", torch.bfloat16), ("int4", torch.float16), ("int4", torch.bfloat16)]


def hold(rows, kind):
    """(cache argument, its exact values, its K scales [..., N, H]) of rows k, v as a cache of a kind holds them."""
    from topk_attn_b200 import ops
    if not kind:
        return tuple(rows), tuple(rows), None
    vals, parts, scale = [], [], None
    for x in rows:
        c, s, val = O.quantize(x.cpu(), kind)
        parts.append([t.to(DEV) for t in O.pack(c, s, kind)])
        vals.append(val.to(DEV))
        scale = s.amax(-1).to(DEV) if scale is None else scale
    return ops.QuantizedKV(parts[0][0], parts[1][0], parts[0][1], parts[1][1]), tuple(vals), scale


def hold_to(out, q, prefix, own, lens, kind, tokens):
    ref, mass, reach = O.attention_terms(q, SM, prefix and prefix[1], own and own[1], lens,
                                         [prefix and prefix[2], own and own[2]], kind)
    most = O.bound(ref, mass, reach, tokens, q.dtype)
    assert (ref.abs() > 4 * most).double().mean() > 0.5          # zeros would be seen
    assert ((out.double() - ref).abs() <= most).all()


@pytest.mark.parametrize("kind,dtype", FORMS)
@pytest.mark.parametrize("B,Np", [(3, 50001), (16, 30016), (24, 61441), (131, 49152), (300, 20011)])
def test_every_tile_of_a_long_prefix_counts(B, Np, kind, dtype):
    from topk_attn_b200 import ops
    g = torch.Generator(device=DEV).manual_seed(B)
    q, k, v = O.planted(B, Np, dtype, g)
    prefix = hold((k, v), kind)
    out = ops.shared_prefix_attention(q[:, None], prefix[0], None, SM)
    ops.check_status(torch.device(DEV))
    hold_to(out, q[:, None], prefix, None, None, kind, Np)


@pytest.mark.parametrize("kind,dtype", FORMS)
@pytest.mark.parametrize("G", [1, 8, 12])
def test_every_tile_of_long_caches_of_different_lengths_counts(G, kind, dtype):
    from topk_attn_b200 import ops
    g = torch.Generator(device=DEV).manual_seed(G)
    N, lens = 30011, torch.tensor([30011, 0, 12345, 64, 1, 30010], dtype=torch.int32, device=DEV)
    rows = [O.planted(G, N, dtype, g) for _ in range(6)]
    q, k, v = (torch.stack([r[i] for r in rows]) for i in range(3))
    own = hold((k, v), kind)
    out = ops.shared_prefix_attention(q, None, own[0], SM, lens)
    ops.check_status(torch.device(DEV))
    assert not out[1].any()
    hold_to(out[[0, 2, 3, 4, 5]], q[[0, 2, 3, 4, 5]], None, [own[0]] + [None if x is None else tuple(y[[0, 2, 3, 4, 5]] for y in x)
            if isinstance(x, tuple) else x[[0, 2, 3, 4, 5]] for x in own[1:]], lens[[0, 2, 3, 4, 5]], kind, N)


def test_offsets_beyond_32_bits_reach_the_token_that_counts():
    """Caches whose codes take 3.2 GB each: the last token of every row, which takes nine tenths of the weight and more,
    written, read back and attended to, as own caches and as a prefix shared by 24 queries a key."""
    from topk_attn_b200 import ops
    B, N, H, G = 3, 1 << 20, 8, 8
    g = torch.Generator(device=DEV).manual_seed(1)
    k, v = (torch.empty(B, N, H, 128, dtype=torch.int8, device=DEV).random_(-127, 128, generator=g) for _ in range(2))
    ks, vs = (torch.rand(B, H, N, generator=g, device=DEV) * 0.01 + 0.01 for _ in range(2))
    cache = ops.QuantizedKV(k, v, ks, vs)
    u = torch.randn(B, H, 128, generator=g, device=DEV)
    last = torch.randn(B, 1, H, 128, generator=g, device=DEV).half()
    key = (u * (17.0 * math.sqrt(128) / u.square().sum(-1, keepdim=True))).half()[:, None]
    ops.kv_append_quantized(cache, key, last, torch.full((B,), N - 1, dtype=torch.int32, device=DEV))
    for back, rows in zip(ops.kv_dequantize(cache, N - 1, 1), (key, last)):
        want = O.quantize(rows.cpu(), "int8")[2]
        assert ((back.cpu().double() - want).abs() <= O.half_step(want, torch.float16) + want.abs() * 2.0 ** -24).all()
    q = u.half()[:, :, None].expand(B, H, G, 128).reshape(B, H * G, 128).contiguous()
    outs = [(ops.flash_decoding_quantized(q, cache, SM), range(B))]
    one = ops.QuantizedKV(k[2], v[2], ks[2], vs[2])
    outs.append((ops.shared_prefix_attention(q[2:].expand(B, -1, -1).contiguous(), one, None, SM), [2] * B))
    ops.check_status(torch.device(DEV))
    for out, rows in outs:
        for b, r in enumerate(rows):
            for h in (0, H - 1):
                kd, vd = (c[r, :, h].double() * s[r, h].double()[:, None] for c, s in ((k, ks), (v, vs)))
                qh = q[r:r + 1, h * G:(h + 1) * G]
                w = torch.softmax(qh[0, 0].double() @ kd.T * SM, -1)
                assert w[-1] > 0.9
                ref, mass = w @ vd, w @ vd.abs()
                reach = (qh[0, 0].double().abs() @ (kd.abs() + 128 * ks[r, h].double()[:, None]).T).amax() * SM
                most = O.bound(ref, mass, reach[None], N, torch.float16)
                assert (ref.abs() > 4 * most).double().mean() > 0.5
                assert ((out[b, h * G:(h + 1) * G].double() - ref).abs() <= most).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("kind", ["int8", "fp8", "int4"])
@pytest.mark.parametrize("B,G", [(3, 4), (24, 2)])
def test_a_decode_loop_sees_what_is_held(B, G, kind, dtype):
    """Append and attend, step by step, against the codes that the rows have by definition; the newest tokens carry
    weight, so a step that leaves its own cache out is seen."""
    from topk_attn_b200 import ops
    H, Np, T, steps = 2, 333, 6, 4
    g = torch.Generator().manual_seed(3)

    def some(*shape):
        return torch.randn(shape, generator=g).to(dtype)
    prompt = some(Np, H, 128), some(Np, H, 128)
    prefix = ops.quantized_kv_cache(Np, H, kind, device=DEV)
    ops.kv_append_quantized(prefix, *(x.to(DEV) for x in prompt), 0)
    cache = ops.quantized_kv_cache(T + steps, H, kind, batch=B, device=DEV)
    all_rows = [torch.zeros(B, T + steps, H, 128, dtype=dtype) for _ in range(2)]
    lens = torch.tensor([i % (T + 1) for i in range(B)], dtype=torch.int32)
    start = some(B, T, H, 128), some(B, T, H, 128)
    for x, y in zip(all_rows, start):
        for b in range(B):
            x[b, :lens[b]] = y[b, :lens[b]]
    ops.kv_append_quantized(cache, *(x.to(DEV) for x in start), 0, lens.to(DEV))
    held = hold(prompt, kind)
    for _ in range(steps):
        q = some(B, H * G, 128)
        new = (q.view(B, H, G, 128)[:, :, 0].float() * 0.4).to(dtype)[:, None], some(B, 1, H, 128)
        ops.kv_append_quantized(cache, *(x.to(DEV) for x in new), lens.to(DEV))
        for x, y in zip(all_rows, new):
            x[torch.arange(B), lens.long()] = y[:, 0]
        lens += 1
        out = ops.shared_prefix_attention(q.to(DEV), prefix, cache, SM, lens.to(DEV))
        hold_to(out, q.to(DEV), held, hold(all_rows, kind), lens, kind, Np + T + steps)
    ops.check_status(torch.device(DEV))
