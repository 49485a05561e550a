"""The quantised key/value cache and the shared-prefix attention, as a user's program calls them.

Three operators, each in its plain form (elementary torch operations) and, with ``own`` set, by the
package's own entry points:

* ``kv_quant``   quantising key/value rows as they are written into a cache, and reading them back;
* ``quant_attn`` decode attention that reads the quantised cache directly, one query token per row;
* ``prefix``     decode attention of a batch whose sequences share a long prefix, in front of a
                 cache of their own.

The formats hold one fp32 scale for each (token, head) row of 128 values ("int8": amax/127; "fp8":
e4m3 with the least power of two that brings amax to 448 or less), or for each 32 of them ("int4":
amax/7, two codes in a byte, the code plus 8, the even value in the low half).  Codes are token-major
[.., N, H, 128] ([.., N, H, 64] for int4), scales head-major [.., H, N] ([.., H, N, 4] for int4).
"""
import math

import torch

own = False

D = 128
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
CODE_BYTES = {"int8": 128, "fp8": 128, "int4": 64}     # of one row of 128 values
SCALES = {"int8": 1, "fp8": 1, "int4": 4}
SM_SCALE = 1.0 / math.sqrt(D)


# ------------------------------------------------------------------------------------- the cases
def listed():
    return [
        # one decode step of a serving batch: every sequence writes one token (launch latency)
        {"name": "write_token_int8", "op": "kv_quant", "kind": "int8", "dtype": "fp16", "batch": 64, "tokens": 1,
         "heads": 8, "ragged": False, "fused": False},
        # a long prompt's rows, as views of one fused k/v projection
        {"name": "write_prompt_fp8", "op": "kv_quant", "kind": "fp8", "dtype": "bf16", "batch": 2, "tokens": 16384,
         "heads": 8, "ragged": False, "fused": True},
        # a padded batch of prompts of odd length, one kv head for each query head
        {"name": "write_padded_int4", "op": "kv_quant", "kind": "int4", "dtype": "fp16", "batch": 16, "tokens": 1001,
         "heads": 32, "ragged": True, "fused": False},
        # one sequence at a 4096-token context, 32 heads: the smallest decode step of the benchmark
        {"name": "attn_one_int8", "op": "quant_attn", "kind": "int8", "dtype": "fp16", "batch": 1, "hq": 32, "hkv": 32,
         "tokens": 4096, "ragged": False},
        # the benchmark's dense decode: 8 sequences at 32768 tokens, 32 query and 8 kv heads
        {"name": "attn_batch_int8", "op": "quant_attn", "kind": "int8", "dtype": "fp16", "batch": 8, "hq": 32, "hkv": 8,
         "tokens": 32768, "ragged": False},
        # a serving batch of very different lengths, an empty sequence among them, groups of 8
        {"name": "attn_ragged_fp8", "op": "quant_attn", "kind": "fp8", "dtype": "bf16", "batch": 32, "hq": 32, "hkv": 4,
         "tokens": 32768, "ragged": True},
        # the benchmark's 1 Mi-token context in 4 bits
        {"name": "attn_long_int4", "op": "quant_attn", "kind": "int4", "dtype": "fp16", "batch": 1, "hq": 32, "hkv": 8,
         "tokens": 1048576, "ragged": False},
        # two short chats behind a short common prompt of odd length (launch latency)
        {"name": "prefix_small_fp16", "op": "prefix", "kind": "", "dtype": "fp16", "batch": 2, "hq": 8, "hkv": 8,
         "prefix": 777, "tokens": 64, "ragged": True},
        # a serving batch behind one system prompt
        {"name": "prefix_chat_bf16", "op": "prefix", "kind": "", "dtype": "bf16", "batch": 32, "hq": 32, "hkv": 8,
         "prefix": 2048, "tokens": 1024, "ragged": True},
        # questions about one long document: the benchmark's 131072 tokens and 32 heads
        {"name": "prefix_document_fp16", "op": "prefix", "kind": "", "dtype": "fp16", "batch": 16, "hq": 32, "hkv": 32,
         "prefix": 131072, "tokens": 512, "ragged": True},
        # many samples from one long prompt: enough queries for each key to be bound by arithmetic
        {"name": "prefix_wide_bf16", "op": "prefix", "kind": "", "dtype": "bf16", "batch": 256, "hq": 32, "hkv": 8,
         "prefix": 32768, "tokens": 256, "ragged": True},
        # a batch behind a prompt whose cache, and the sequences' own, are held in 8 bits
        {"name": "prefix_int8", "op": "prefix", "kind": "int8", "dtype": "fp16", "batch": 32, "hq": 32, "hkv": 8,
         "prefix": 16385, "tokens": 512, "ragged": True},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["kv_quant", "quant_attn", "quant_attn", "prefix", "prefix"])
    dtype = rng.choice(["fp16", "bf16"])
    ragged = rng.random() < 0.5
    if op == "kv_quant":
        heads = rng.choice([1, 2, 4, 8, 32])
        tokens = _log_int(rng, 1, 16384)
        batch = _log_int(rng, 1, max(1, min(256, 32768 * 8 // (tokens * heads))))
        return {"op": op, "kind": rng.choice(["int8", "fp8", "int4"]), "dtype": dtype, "batch": batch,
                "tokens": tokens, "heads": heads, "ragged": ragged, "fused": rng.random() < 0.5}
    hkv = rng.choice([1, 2, 4, 8, 32])
    group = rng.choice([1, 2, 4, 8] if hkv < 32 else [1])
    if op == "quant_attn":
        tokens = _log_int(rng, 1, 524288)
        batch = _log_int(rng, 1, max(1, min(256, 4 * 1048576 // (tokens * hkv))))
        return {"op": op, "kind": rng.choice(["int8", "fp8", "int4"]), "dtype": dtype, "batch": batch,
                "hq": hkv * group, "hkv": hkv, "tokens": tokens, "ragged": ragged}
    prefix = _log_int(rng, 1, 131072)
    batch = _log_int(rng, 1, max(1, min(256, 256 * 32 * 32768 // (prefix * hkv * group))))
    tokens = _log_int(rng, 1, max(1, min(4096, 1048576 // (batch * hkv))))
    return {"op": op, "kind": rng.choice(["", "", "int8", "fp8", "int4"]), "dtype": dtype, "batch": batch,
            "hq": hkv * group, "hkv": hkv, "prefix": prefix, "tokens": tokens, "ragged": ragged}


# ------------------------------------------------------------------------------------- the inputs
def _lengths(case):
    """Lengths of a padded batch: spread over their logarithm from the full one down to 0 or 1."""
    n, b = case["tokens"], case["batch"]
    if not case["ragged"]:
        return [n] * b
    return [n if i == 0 else int(math.exp(math.log(n + 1) * (b - 1 - i) / max(1, b - 1))) - 1 for i in range(b)]


def _rows(gen, shape, dtype):
    """Key rows as models have them: a few channels of every head much larger than the others."""
    x = torch.randn(shape, generator=gen, device="cuda", dtype=dtype)
    chan = torch.ones(shape[-2:], device="cuda", dtype=dtype)
    chan[torch.rand(shape[-2:], generator=gen, device="cuda") < 0.03] = 4.0
    return x.mul_(chan)


def _coded(gen, shape, kind):
    """Codes and scales of a cache that has been filled before: [.., N, H] rows of 128 values."""
    *lead, n, h = shape
    scale = torch.rand(*lead, h, n, *([4] if kind == "int4" else []), generator=gen, device="cuda") + 0.5
    if kind == "int8":
        x = torch.empty(*shape, D, dtype=torch.int8, device="cuda").random_(-127, 128, generator=gen)
        return x, scale.mul_(2.0 / 127)
    if kind == "fp8":
        x = torch.randn(*shape, D, generator=gen, device="cuda", dtype=torch.float16).mul_(96.0).clamp_(-448, 448)
        return x.to(torch.float8_e4m3fn), torch.exp2(torch.floor(scale.mul_(2)) - 8)
    x = torch.empty(*shape, D // 2, dtype=torch.uint8, device="cuda").random_(0, 256, generator=gen)
    x = torch.where(x & 15 == 0, x + 1, x)
    x = torch.where(x >> 4 == 0, x + 16, x)
    return x, scale.mul_(2.0 / 7)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype, b, n = DTYPES[case["dtype"]], case["batch"], case["tokens"]
    lens = torch.tensor(_lengths(case), dtype=torch.int32)
    lens = lens[torch.randperm(b, generator=torch.Generator().manual_seed(seed))].to("cuda")
    s = {"case": case, "lens": lens if case["ragged"] else None}
    if case["op"] == "kv_quant":
        h, kind = case["heads"], case["kind"]
        if case["fused"]:
            kv = _rows(gen, (b, n, 2, h, D), dtype)
            s["new_k"], s["new_v"] = kv[:, :, 0], kv[:, :, 1]
        else:
            s["new_k"], s["new_v"] = _rows(gen, (b, n, h, D), dtype), _rows(gen, (b, n, h, D), dtype)
        s["at"] = torch.randint(0, 64, (b,), generator=gen, device="cuda", dtype=torch.int32)
        code = {"int8": torch.int8, "fp8": torch.float8_e4m3fn, "int4": torch.uint8}[kind]
        for x in ("k", "v"):
            s[x] = torch.zeros(b, n + 64, h, CODE_BYTES[kind], dtype=torch.uint8, device="cuda").view(code)
            s[x + "_scale"] = torch.zeros(b, h, n + 64, *([4] if kind == "int4" else []), device="cuda")
        return s
    hq, hkv, kind = case["hq"], case["hkv"], case["kind"]
    s["q"] = torch.randn(b, hq, D, generator=gen, device="cuda").mul_(1.5).to(dtype)
    for x in ("k", "v"):
        if kind:
            s[x], s[x + "_scale"] = _coded(gen, (b, n, hkv), kind)
        else:
            s[x] = _rows(gen, (b, n, hkv, D), dtype)
        if case["op"] == "prefix":
            if kind:
                s["p" + x], s["p" + x + "_scale"] = _coded(gen, (case["prefix"], hkv), kind)
            else:
                s["p" + x] = _rows(gen, (case["prefix"], hkv, D), dtype)
    return s


# --------------------------------------------------------------------------------- the operators
def _own(s):
    from topk_attn_b200 import ops
    case = s["case"]
    if case["op"] == "kv_quant":
        cache = ops.QuantizedKV(s["k"], s["v"], s["k_scale"], s["v_scale"])
        ops.kv_append_quantized(cache, s["new_k"], s["new_v"], s["at"], s["lens"])
        return ops.kv_dequantize(cache, s["at"], case["tokens"], DTYPES[case["dtype"]])
    if case["kind"]:
        cache = ops.QuantizedKV(s["k"], s["v"], s["k_scale"], s["v_scale"])
    else:
        cache = (s["k"], s["v"])
    if case["op"] == "quant_attn":
        return ops.flash_decoding_quantized(s["q"], cache, SM_SCALE, s["lens"])
    if case["kind"]:
        prefix = ops.QuantizedKV(s["pk"], s["pv"], s["pk_scale"], s["pv_scale"])
    else:
        prefix = (s["pk"], s["pv"])
    return ops.shared_prefix_attention(s["q"], prefix, cache, SM_SCALE, s["lens"])


def _requantised(x, kind):
    """fp32 values that the codes of the rows x [.., 128] stand for."""
    x = x.float()
    if kind == "int4":
        x = x.unflatten(-1, (4, 32))
    amax = x.abs().amax(-1, keepdim=True)
    if kind == "fp8":
        frac, exp = torch.frexp(amax)
        shift = torch.where(frac <= 0.875, exp - 9, exp - 8)
        y = torch.ldexp(torch.ldexp(x, -shift).to(torch.float8_e4m3fn).float(), shift)
    else:
        top = 127 if kind == "int8" else 7
        scale = (amax.double() / top).float()        # a quotient next to a border needs 64 bits
        y = torch.round(x.double() / scale.double()).clamp(-top, top).float() * scale
    y = torch.where(amax < 2.0 ** -100, 0.0, y)
    return y.flatten(-2) if kind == "int4" else y


def _values(x, scale, kind):
    """fp32 [.., N, H, 128] of codes and their scales."""
    scale = scale.transpose(-3, -2) if kind == "int4" else scale.transpose(-2, -1)
    if kind != "int4":
        return x.float() * scale.unsqueeze(-1)
    x = torch.stack((x & 15, x >> 4), -1).flatten(-2).float() - 8.0
    return (x.unflatten(-1, (4, 32)) * scale.unsqueeze(-1)).flatten(-2)


def _cache(s, x, lead=""):
    kind = s["case"]["kind"]
    return _values(s[lead + x], s[lead + x + "_scale"], kind) if kind else s[lead + x].float()


def _plain(s):
    case = s["case"]
    dtype, b, n = DTYPES[case["dtype"]], case["batch"], case["tokens"]
    live = None
    if s["lens"] is not None:
        live = torch.arange(n, device="cuda") < s["lens"].unsqueeze(1)          # [B, N]
    if case["op"] == "kv_quant":
        k, v = _requantised(s["new_k"], case["kind"]), _requantised(s["new_v"], case["kind"])
        if live is not None:
            k, v = torch.where(live[..., None, None], k, 0.0), torch.where(live[..., None, None], v, 0.0)
        return k.to(dtype), v.to(dtype)
    hq, hkv = case["hq"], case["hkv"]
    g = hq // hkv
    q = s["q"].float().view(b, hkv, g, D) * SM_SCALE
    k, v = _cache(s, "k").transpose(1, 2), _cache(s, "v").transpose(1, 2)       # [B, Hkv, N, 128]
    x = q @ k.transpose(2, 3)                                                   # [B, Hkv, G, N]
    if live is not None:
        x = torch.where(live[:, None, None], x, -math.inf)
    top = x.amax(-1, keepdim=True)
    if case["op"] == "prefix":
        pk, pv = _cache(s, "k", "p").transpose(0, 1), _cache(s, "v", "p").transpose(0, 1)
        px = q.transpose(0, 1).reshape(hkv, b * g, D) @ pk.transpose(1, 2)      # [Hkv, B*G, Np]
        px = px.view(hkv, b, g, -1).transpose(0, 1)
        top = torch.maximum(top, px.amax(-1, keepdim=True))
    top = torch.where(top == -math.inf, 0.0, top)                               # nothing to attend to
    w = torch.exp(x - top)
    total, out = w.sum(-1, keepdim=True), w @ v
    if case["op"] == "prefix":
        pw = torch.exp(px - top)
        total = total + pw.sum(-1, keepdim=True)
        out = out + (pw.transpose(0, 1).reshape(hkv, b * g, -1) @ pv).view(hkv, b, g, D).transpose(0, 1)
    out = torch.where(total > 0, out / total, 0.0)
    return out.reshape(b, hq, D).to(dtype)


def run(state):
    return _own(state) if own else _plain(state)


def work(case):
    lens = sum(_lengths(case))
    if case["op"] == "kv_quant":
        rows = 2 * case["heads"] * lens
        held = CODE_BYTES[case["kind"]] + 4 * SCALES[case["kind"]]
        back = 2 * case["heads"] * case["batch"] * case["tokens"]
        return {"bytes": rows * (2 * D + held) + back * 2 * D, "flops": 3 * rows * D}
    row = CODE_BYTES[case["kind"]] + 4 * SCALES[case["kind"]] if case["kind"] else 2 * D
    tokens = lens + case.get("prefix", 0)
    seen = lens + case["batch"] * case.get("prefix", 0)
    return {"bytes": 2 * tokens * case["hkv"] * row + 4 * case["batch"] * case["hq"] * D,
            "flops": 4 * D * (case["hq"] // case["hkv"]) * case["hkv"] * seen}


# ------------------------------------------------------------------------- the definition, 64 bits
def _decoded(codes, scales, kind):
    """float64 values [N, 128] of one head's codes and scales."""
    if kind == "int4":
        vals = torch.empty(codes.size(0), D, dtype=torch.float64, device=codes.device)
        vals[:, 0::2] = codes.bitwise_and(15).double() - 8
        vals[:, 1::2] = codes.bitwise_right_shift(4).double() - 8
        return vals * scales.double().repeat_interleave(32, dim=1)
    return codes.double() * scales.double()[:, None]


def _defined_codes(x, kind):
    """What the rows x (float64, [rows, 128]) are stored as."""
    if kind == "int4":
        x = x.reshape(-1, 32)
    peak = x.abs().max(dim=1).values
    if kind == "fp8":
        step = torch.zeros_like(peak)
        ok = peak > 0
        step[ok] = torch.ceil(torch.log2(peak[ok] / 448.0))
        scale = torch.exp2(step)
        y = x / scale[:, None]
        binade = torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -6)))
        quantum = torch.exp2(binade - 3)
        y = torch.round(y / quantum) * quantum
    else:
        m = 127.0 if kind == "int8" else 7.0
        scale = (peak / m).to(torch.float32).double()
        y = torch.round(x / scale.where(scale > 0, 1.0)[:, None])
    y = y * scale[:, None]
    y[peak < 2.0 ** -100] = 0.0
    return y.reshape(-1, D)


def exact(case, seed):
    s = prepare(case, seed)
    b, n = case["batch"], case["tokens"]
    lens = s["lens"].tolist() if s["lens"] is not None else [n] * b
    if case["op"] == "kv_quant":
        res = []
        for x in (s["new_k"], s["new_v"]):
            y = torch.zeros(x.shape, dtype=torch.float64, device="cuda")
            for i in range(b):
                if lens[i]:
                    rows = x[i, :lens[i]].double()
                    y[i, :lens[i]] = _defined_codes(rows.reshape(-1, D), case["kind"]).view(rows.shape)
            res.append(y)
        return tuple(res)
    hkv, kind = case["hkv"], case["kind"]
    g = case["hq"] // hkv
    out = torch.zeros(b, case["hq"], D, dtype=torch.float64, device="cuda")

    def head(x, lead, h, i=None):
        codes = s[lead + x] if i is None else s[lead + x][i]
        if not kind:
            return codes[:, h].double()
        sc = s[lead + x + "_scale"] if i is None else s[lead + x + "_scale"][i]
        return _decoded(codes[:, h], sc[h], kind)

    for h in range(hkv):
        if case["op"] == "prefix":
            pk, pv = head("k", "p", h), head("v", "p", h)
        else:
            pk = pv = torch.zeros(0, D, dtype=torch.float64, device="cuda")
        q = s["q"][:, h * g:(h + 1) * g].double()
        far = (q.reshape(b * g, D) @ pk.T * SM_SCALE).view(b, g, -1)
        near = torch.full((b, g, n), -math.inf, dtype=torch.float64, device="cuda")
        vals = []
        for i in range(b):
            m = lens[i]
            near[i, :, :m] = q[i] @ head("k", "", h, i)[:m].T * SM_SCALE
            vals.append(head("v", "", h, i)[:m])
        lse = torch.logsumexp(torch.cat((far, near), -1), -1)                   # [B, G]
        lse = torch.where(torch.isinf(lse), 0.0, lse)[..., None]
        res = (torch.exp(far - lse).view(b * g, -1) @ pv).view(b, g, D)
        for i in range(b):
            res[i] += torch.exp(near[i, :, :lens[i]] - lse[i]) @ vals[i]
        out[:, h * g:(h + 1) * g] = res
    return out
