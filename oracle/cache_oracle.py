"""Quantised caches and attention behind a shared prefix, restated in 64 bits on the CPU.

Formats (rows of 128 values): int8 s = fp32(amax/127), code = rne(x/s); fp8 s = the least power of
two with amax <= 448 s, code = e4m3(x/s); int4 for each 32 values s = fp32(amax/7), code = rne(x/s).
A row (a group of 32) with amax < 2**-100 is zeros with s = 0; one that is not finite has s = NaN."""
import math

import torch

GROUP = {"int8": 128, "fp8": 128, "int4": 32}


def quantize(x, kind):
    """x [..., 128] -> (codes float64 [..., 128], scales fp32 [..., 1 or 4], values float64)."""
    y = x.double().unflatten(-1, (-1, GROUP[kind]))
    amax = y.abs().amax(-1)
    ok = torch.isfinite(amax) & (amax >= 2.0 ** -100)
    top = {"int8": 127.0, "fp8": 448.0, "int4": 7.0}[kind]
    safe = torch.where(ok, amax, 1.0)
    if kind == "fp8":
        m, e = torch.frexp(safe / 448.0)
        scale = torch.exp2(torch.where(m == 0.5, e - 1, e).double())
    else:
        scale = (safe / top).float().double()
    u = torch.where(ok[..., None], y, 0.0) / scale[..., None]
    if kind == "fp8":
        q = torch.exp2(torch.floor(torch.log2(u.abs().clamp_min(2.0 ** -6))) - 3)
        codes = torch.round(u / q) * q
    else:
        codes = torch.round(u).clamp(-top, top)
    scale = torch.where(ok, scale, torch.where(torch.isfinite(amax), 0.0, math.nan))
    return codes.flatten(-2), scale.float(), (codes * scale[..., None]).flatten(-2)


def pack(codes, scales, kind):
    """Codes and scales of rows [..., N, H, 128] in the layout of a cache."""
    if kind == "int8":
        c = codes.to(torch.int8)
    elif kind == "fp8":
        c = codes.float().to(torch.float8_e4m3fn)
    else:
        n = (codes + 8).to(torch.uint8)
        c = n[..., 0::2] | (n[..., 1::2] << 4)
    s = scales.transpose(-3, -2)
    return c.contiguous(), (s if kind == "int4" else s.squeeze(-1)).contiguous()


def attention(q, sm_scale, prefix=None, own=None, lens=None):
    """q [B,Hq,128]; prefix (k, v) [Np,Hkv,128]; own (k, v) [B,N,Hkv,128]; float64 [B,Hq,128]."""
    B, Hq, D = q.shape
    heads = (prefix or own)[0].size(-2)
    g = Hq // heads
    out = torch.zeros(B, Hq, D, dtype=torch.float64)
    for b in range(B):
        ks, vs = [], []
        if prefix is not None:
            ks.append(prefix[0].double())
            vs.append(prefix[1].double())
        if own is not None:
            n = own[0].size(1) if lens is None else max(0, min(own[0].size(1), int(lens[b])))
            ks.append(own[0][b, :n].double())
            vs.append(own[1][b, :n].double())
        k, v = torch.cat(ks), torch.cat(vs)
        if k.size(0) == 0:
            continue
        qb = q[b].double().view(heads, g, D)
        s = torch.einsum("hgd,nhd->hgn", qb, k) * sm_scale
        out[b] = torch.einsum("hgn,nhd->hgd", torch.softmax(s, -1), v).reshape(Hq, D)
    return out


def tolerance(ref, q, sm_scale, ks, vs, total, dtype, kind=""):
    """Bound on |kernel - ref| for outputs of ``dtype``: what each rounding can contribute at worst.

    fp32 sums of 128 exact products: 2^-24 * 130 of sum |q||k| in every score, and a score's error
    is a relative error of its weight; exp2 in hardware 2^-22; weights rounded for the matrix
    product, half a step relative (plus 2^-25 absolute for each token where fp16 weights turn
    subnormal); for int4 two half steps of fp16 in the scores and the values, which a kernel that
    dequantised them in fp16 would need; fp32 sums over the tokens 2^-24 each; the output's own half step.
    A relative weight error d moves the output by at most 2 d max |v|.

    A coarse bound, wider than the answer itself for int4 and for long contexts: ``bound`` is the one that tells a
    wrong result from a right one."""
    half = torch.finfo(dtype).eps / 2
    kmax = torch.stack([k.abs().double().flatten(0, -2).amax(0) for k in ks]).amax(0)
    vmax = max(float(v.abs().max()) for v in vs)
    score = float((q.abs().double() @ kmax).max()) * sm_scale
    weight = 2.0 ** -8 if (dtype == torch.bfloat16 and not kind) else 2.0 ** -11
    d = score * (130 * 2.0 ** -24 + (2.0 ** -10 if kind == "int4" else 0.0)) + 2.0 ** -22 + weight
    d += total * (2.0 ** -25 + 2.0 ** -24)
    return 2 * d * vmax + (2.0 ** -10 * vmax if kind == "int4" else 0.0) + half * ref.abs()


#: What a kernel may add to a code while it multiplies it: int8 codes go through as code + 128, int4 ones as code + 8.
LIFT = {"int8": 128.0, "int4": 8.0}


def attention_terms(q, sm_scale, prefix=None, own=None, lens=None, scales=None, kind=""):
    """What an error bound needs beside the result: (out, mass, reach), float64 on q's device.  mass = sum w |v| of each
    element; reach [B,Hq] = sm_scale * the largest sum |q| (|k| + LIFT s) of any token, s its K scale.  ``scales``: the K
    scales [..., N, H] (int4: the largest of a row's four) of the prefix and of the own caches, where kind has them."""
    B, Hq, D = q.shape
    heads = (prefix or own)[0].size(-2)
    g = Hq // heads
    out, mass = (torch.zeros(B, Hq, D, dtype=torch.float64, device=q.device) for _ in range(2))
    reach = torch.zeros(B, Hq, dtype=torch.float64, device=q.device)
    for b in range(B):
        ks, vs, lift = [], [], []
        for i, part in enumerate((prefix, own)):
            if part is None:
                continue
            n = part[0].size(-3) if i == 0 or lens is None else max(0, min(part[0].size(1), int(lens[b])))
            k, v = (x[:n] if i == 0 else x[b, :n] for x in part)
            ks.append(k.double())
            vs.append(v.double())
            s = torch.zeros(n, heads, device=q.device) if kind not in LIFT else (scales[i][:n] if i == 0 else scales[i][b, :n]).abs() * LIFT[kind]
            lift.append(s.double())
        k, v, lift = torch.cat(ks), torch.cat(vs), torch.cat(lift)
        if k.size(0) == 0:
            continue
        qb = q[b].double().view(heads, g, D)
        w = torch.softmax(torch.einsum("hgd,nhd->hgn", qb, k) * sm_scale, -1)
        out[b] = torch.einsum("hgn,nhd->hgd", w, v).reshape(Hq, D)
        mass[b] = torch.einsum("hgn,nhd->hgd", w, v.abs()).reshape(Hq, D)
        far = torch.einsum("hgd,nhd->hgn", qb.abs(), k.abs() + lift[..., None])
        reach[b] = far.amax(-1).reshape(Hq) * sm_scale
    return out, mass, reach


def half_step(ref, dtype):
    """Half a step of dtype at ref: what rounding alone may be off by."""
    info = torch.finfo(dtype)
    _, e = torch.frexp(ref.abs().clamp_min(info.tiny))
    return torch.ldexp(torch.full_like(ref, info.eps / 2), e - 1)


def bound(ref, mass, reach, tokens, dtype):
    """The most that a result may be off: half a step of its type, and what its terms' roundings contribute.

    A weight is held as a 16-bit value, cut off, and the 16-bit rest of it, rounded: a step of the one times half a
    step of the other, 2^-7 2^-8 = 2^-15 (bf16) or 2^-10 2^-11 = 2^-21 (fp16).  Its score is an fp32 sum of 8 products of 16
    dims, each at most 2^-23 of the terms' magnitude off, and a few more roundings: 2^-19 reach, which is a relative
    error of the weight.  The hardware's exp2 adds 2^-22, the argument's rounding as much.  All of these enter the sum of
    the values and the sum of the weights: twice.  Sums over the tokens take two steps for every 16 of them, each at
    most 2^-23 of the magnitude; joining parts takes fewer."""
    weight = 2.0 ** -15 if dtype == torch.bfloat16 else 2.0 ** -21
    d = 2 * (weight + 2.0 ** -19 * reach[..., None] + 2.0 ** -21) + (tokens / 8 + 64) * 2.0 ** -23
    return half_step(ref, dtype) + d * mass


def moved(out, ref):
    """Share of the elements that are not the correctly rounded result."""
    return float((out != ref.to(out.dtype)).double().mean())


def planted(queries, tokens, dtype, gen):
    """Queries [R,128] and rows k, v [N,1,128] of which every tile of 64 tokens counts: one key of each points along a query
    (the tiles take the queries in turn) with a score of 9, the others' scores are near 0."""
    dev = gen.device
    q = torch.randn(queries, 128, generator=gen, device=dev).to(dtype)
    k = torch.randn(tokens, 128, generator=gen, device=dev) * 0.05
    v = torch.randn(tokens, 128, generator=gen, device=dev)
    tiles = torch.arange(0, tokens, 64, device=dev)
    at = tiles + (torch.rand(tiles.numel(), generator=gen, device=dev) * (tokens - tiles).clamp(max=64)).long()
    to = q.float()[torch.arange(tiles.numel(), device=dev) % queries]
    k[at] = to * (9.0 * math.sqrt(128) / to.square().sum(-1, keepdim=True))
    return q, k.to(dtype)[:, None], v.to(dtype)[:, None]
