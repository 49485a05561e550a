"""Decode attention over a quantised cache and behind a shared prefix, against 64-bit attention."""
import math

import pytest
import torch

from oracle import cache_oracle as O

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
SM = 1.0 / math.sqrt(128)


def make(B, Hq, Hkv, Np, N, kind, dtype, seed=0):
    """(q, prefix, own) on the CPU: fp16/bf16 tensors, and for a kind the codes' values beside them."""
    g = torch.Generator().manual_seed(seed)
    q = (torch.randn(B, Hq, 128, generator=g) * 2).to(dtype)
    res = []
    for shape in ((Np, Hkv, 128), (B, N, Hkv, 128)):
        if shape[-3] == 0 and shape[0] == Np:
            res.append(None)
            continue
        pair = [(torch.randn(shape, generator=g) * torch.exp2(torch.randint(-2, 3, shape[-2:-1] + (1,), generator=g).float())).to(dtype)
                for _ in range(2)]
        if kind:
            coded = [O.quantize(x, kind) for x in pair]
            vals = tuple((c.unflatten(-1, (s.size(-1), -1)) * s.double()[..., None]).flatten(-2) for c, s, _ in coded)
            res.append((vals, [O.pack(c, s, kind) for c, s, _ in coded]))
        else:
            res.append((tuple(pair), pair))
    return q, res[0], res[1]


def device_cache(held, kind):
    from topk_attn_b200 import ops
    if held is None:
        return None
    if kind:
        (kc, ks), (vc, vs) = held[1]
        return ops.QuantizedKV(kc.to(DEV), vc.to(DEV), ks.to(DEV), vs.to(DEV))
    return tuple(x.to(DEV) for x in held[1])


def check(q, prefix, own, kind, lens=None, dtype=None, call=None):
    from topk_attn_b200 import ops
    ref = O.attention(q, SM, prefix and prefix[0], own and own[0], lens)
    dl = lens.to(DEV) if lens is not None else None
    out = ops.shared_prefix_attention(q.to(DEV), device_cache(prefix, kind), device_cache(own, kind), SM, dl)
    ops.check_status(torch.device(DEV))
    parts = [p[0] for p in (prefix, own) if p is not None]
    total = sum(p[0].size(-3) for p in parts)
    tol = O.tolerance(ref, q, SM, [p[0] for p in parts if p[0].numel()], [p[1] for p in parts if p[1].numel()], total,
                      q.dtype, kind)
    far = (out.cpu().double() - ref).abs()
    assert out.dtype == q.dtype
    worst = float((far / tol).max())
    assert worst <= 1.0
    return out


KINDS = ["", "int8", "fp8", "int4"]
DTYPES = [torch.float16, torch.bfloat16]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("B,Hq,Hkv,N", [(1, 1, 1, 1), (1, 4, 4, 129), (2, 8, 2, 1000), (3, 32, 4, 300), (2, 6, 1, 2049),
                                        (1, 24, 2, 515), (1, 40, 1, 131)])
def test_own_caches_without_a_prefix(B, Hq, Hkv, N, kind, dtype):
    q, _, own = make(B, Hq, Hkv, 0, N, kind, dtype, N)
    check(q, None, own, kind)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("B,Hq,Hkv,Np,N", [
    (1, 1, 1, 1, 1), (2, 8, 8, 777, 64), (5, 8, 2, 128, 1), (3, 12, 4, 1025, 130), (9, 16, 2, 515, 33),
    (40, 8, 2, 300, 20), (70, 4, 1, 2000, 5), (33, 32, 8, 640, 17), (140, 2, 2, 260, 3)])
def test_prefix_and_own_caches(B, Hq, Hkv, Np, N, kind, dtype):
    q, prefix, own = make(B, Hq, Hkv, Np, N, kind, dtype, Np + N)
    lens = torch.tensor([(7 * i) % (N + 1) for i in range(B)], dtype=torch.int32)
    check(q, prefix, own, kind, lens)


@pytest.mark.parametrize("kind,dtype", [("", torch.float16), ("", torch.bfloat16), ("int8", torch.float16),
                                        ("fp8", torch.bfloat16), ("int4", torch.float16)])
@pytest.mark.parametrize("B,Np", [(24, 123457), (131, 98304)])
def test_many_tiles_for_each_part(kind, dtype, B, Np):
    """One kv head, so that every CTA walks a long run of tiles: one and two tiles of queries."""
    q, prefix, own = make(B, 1, 1, Np, 2, kind, dtype, 5)
    check(q, prefix, own, kind)


@pytest.mark.parametrize("kind", KINDS)
def test_prefix_alone_and_a_shared_quantised_cache(kind):
    from topk_attn_b200 import ops
    q, prefix, _ = make(3, 8, 4, 600, 1, kind, torch.float16, 4)
    out = check(q, prefix, None, kind)
    if kind:
        again = ops.flash_decoding_quantized(q.to(DEV), device_cache(prefix, kind), SM)
        assert torch.equal(out, again)
        cut = device_cache(prefix, kind).first(599)
        ref = O.attention(q, SM, tuple(x[:599] for x in prefix[0]))
        far = (ops.flash_decoding_quantized(q.to(DEV), cut, SM).cpu().double() - ref).abs()
        assert (far <= O.tolerance(ref, q, SM, [prefix[0][0]], [prefix[0][1]], 599, q.dtype, kind)).all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_what_lies_behind_a_length_is_not_looked_at(kind, dtype):
    """Garbage, infinities and NaN behind each row's length, rows of length zero, lengths out of range."""
    from topk_attn_b200 import capi, ops
    B, N = 6, 300
    q, _, own = make(B, 8, 2, 0, N, kind, dtype, 9)
    lens = torch.tensor([0, 1, 128, 129, 255, 300], dtype=torch.int32)
    clean = ops.shared_prefix_attention(q.to(DEV), None, device_cache(own, kind), SM, lens.to(DEV))
    cache = device_cache(own, kind)
    for b in range(B):
        n = int(lens[b])
        if kind:
            cache.k.view(torch.uint8)[b, n:] = 0x7f
            cache.v.view(torch.uint8)[b, n:] = 0x7f
            cache.k_scale[b, :, n:] = math.nan
            cache.v_scale[b, :, n:] = math.inf
        else:
            cache[0][b, n:] = math.nan
            cache[1][b, n:] = math.inf if b % 2 else math.nan
    out = ops.shared_prefix_attention(q.to(DEV), None, cache, SM, lens.to(DEV))
    assert torch.equal(out, clean) and not out[0].any() and torch.isfinite(out).all()
    check(q, None, own, kind, lens)
    ops.check_status(torch.device(DEV))
    try:
        wild = lens.clone()
        wild[0], wild[5] = -7, 2 ** 31 - 1
        out = ops.shared_prefix_attention(q.to(DEV), None, cache, SM, wild.to(DEV))
        assert torch.equal(out, clean)
        with pytest.raises(capi.RaError):
            ops.check_status(torch.device(DEV))
    finally:
        ops.clear_status(torch.device(DEV))


@pytest.mark.parametrize("kind", KINDS)
def test_a_nan_that_is_attended_to_shows(kind):
    from topk_attn_b200 import ops
    q, prefix, own = make(40, 4, 2, 200, 130, kind, torch.float16, 2)
    cache, pre = device_cache(own, kind), device_cache(prefix, kind)
    lens = torch.full((40,), 130, dtype=torch.int32, device=DEV)
    if kind:
        cache.k_scale[0, 0, 129] = math.nan
        cache.v_scale[1, 1, 0] = math.nan
    else:
        cache[0][0, 129, 0, 3] = math.nan
        cache[1][1, 0, 1] = math.nan
    out = ops.shared_prefix_attention(q.to(DEV), pre, cache, SM, lens)
    nan = torch.isnan(out)
    assert nan[0, :2].all() and nan[1, 2:].all()
    if kind != "int4":
        assert not nan[0, 2:].any() and not nan[1, :2].any()
    assert not nan[2:].any()


def test_empty_parts():
    from topk_attn_b200 import ops
    q, prefix, own = make(2, 4, 2, 50, 40, "", torch.float16, 1)
    pre, cache = device_cache(prefix, ""), device_cache(own, "")
    a = ops.shared_prefix_attention(q.to(DEV), pre, None, SM)
    b = ops.shared_prefix_attention(q.to(DEV), pre, tuple(x[:, :0] for x in cache), SM)
    c = ops.shared_prefix_attention(q.to(DEV), pre, cache, SM, torch.zeros(2, dtype=torch.int32, device=DEV))
    tol = O.tolerance(a.cpu().double(), q, SM, [prefix[0][0]], [prefix[0][1]], 50, torch.float16)
    for x in (b, c):
        assert ((x.double() - a.double()).abs().cpu() <= 2 * tol).all()
    z = ops.shared_prefix_attention(q.to(DEV), tuple(x[:0] for x in pre), tuple(x[:, :0] for x in cache), SM)
    assert not z.any()
    d = ops.shared_prefix_attention(q.to(DEV), tuple(x[:0] for x in pre), cache, SM)
    e = ops.shared_prefix_attention(q.to(DEV), None, cache, SM)
    assert torch.equal(d, e)


@pytest.mark.parametrize("scale", [0.05, 60.0])
@pytest.mark.parametrize("B", [2, 80])
def test_flat_and_peaked_scores(scale, B):
    """Scores that are all alike, and scores whose maximum keeps rising from tile to tile."""
    q, prefix, own = make(B, 4, 2, 1500, 260, "", torch.float16, 6)
    ramp = torch.linspace(0.1, 1.0, 1500)[:, None, None]
    (pk, pv), (k, v) = prefix[0], own[0]
    pk = (pk.float() * ramp * scale / 8).half()
    k = (k.float() * scale / 8).half()
    check(q, ((pk, pv), [pk, pv]), ((k, v), [k, v]), "")


def test_repeated_calls_give_the_same_bits_and_strided_caches_work():
    from topk_attn_b200 import ops
    q, prefix, own = make(4, 16, 4, 900, 400, "", torch.bfloat16, 8)
    first = check(q, prefix, own, "")
    for _ in range(3):
        assert torch.equal(first, check(q, prefix, own, ""))
    wide = torch.zeros(4, 512, 6, 128, dtype=torch.bfloat16, device=DEV)
    wk, wv = wide.clone(), wide.clone()
    wk[:, 50:450, 1:5], wv[:, 50:450, 1:5] = own[1][0].to(DEV), own[1][1].to(DEV)
    out = ops.shared_prefix_attention(q.to(DEV), device_cache(prefix, ""), (wk[:, 50:450, 1:5], wv[:, 50:450, 1:5]), SM)
    assert torch.equal(out, first)
    hm = tuple(x.to(DEV).transpose(1, 2).contiguous().transpose(1, 2) for x in own[1])   # head-major storage
    assert torch.equal(ops.shared_prefix_attention(q.to(DEV), device_cache(prefix, ""), hm, SM), first)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("B,Hkv,Np,N", [(32, 8, 16385, 200), (150, 2, 9000, 70), (3, 4, 6000, 900)])
def test_calls_behind_one_another_give_the_same_bits(kind, B, Hkv, Np, N):
    """Many calls without a pause, on two sets of inputs in turn, all of them in L2: a tile that is overwritten
    too early, or a call that overlaps the next one's memory, shows as another result."""
    from topk_attn_b200 import ops
    g = torch.Generator(device=DEV).manual_seed(7)
    sets = []
    for _ in range(2):
        q = torch.randn(B, 4 * Hkv, 128, generator=g, device=DEV).half()
        rows = [torch.randn(Np, Hkv, 128, generator=g, device=DEV).half() for _ in range(2)]
        own = [torch.randn(B, N, Hkv, 128, generator=g, device=DEV).half() for _ in range(2)]
        if kind:
            pre = ops.quantized_kv_cache(Np, Hkv, kind, device=DEV)
            ops.kv_append_quantized(pre, *rows, 0)
            cache = ops.quantized_kv_cache(N, Hkv, kind, batch=B, device=DEV)
            ops.kv_append_quantized(cache, *own, 0)
        else:
            pre, cache = tuple(rows), tuple(own)
        lens = torch.randint(0, N + 1, (B,), generator=g, device=DEV, dtype=torch.int32)
        torch.cuda.synchronize()
        sets.append((q, pre, cache, SM, lens))
    want = []
    for s in sets:
        want.append(ops.shared_prefix_attention(*s))
        torch.cuda.synchronize()
    for _ in range(6):
        got = [ops.shared_prefix_attention(*sets[i % 2]) for i in range(60)]
        assert all(torch.equal(x, want[i % 2]) for i, x in enumerate(got))
    ops.check_status(torch.device(DEV))


def test_offsets_beyond_32_bits():
    """The last tokens of the last row of a cache whose codes take 3.2 GB each: written, read back and attended
    to; and as a shared prefix seen by 24 queries per key."""
    from topk_attn_b200 import ops
    B, N, H = 3, 1 << 20, 8
    g = torch.Generator(device=DEV).manual_seed(1)
    k, v = (torch.empty(B, N, H, 128, dtype=torch.int8, device=DEV).random_(-127, 128, generator=g) for _ in range(2))
    ks, vs = (torch.rand(B, H, N, generator=g, device=DEV) * 0.01 + 0.01 for _ in range(2))
    cache = ops.QuantizedKV(k, v, ks, vs)
    rows = torch.randn(B, 3, H, 128, generator=g, device=DEV).half()
    ops.kv_append_quantized(cache, rows, -rows, N - 3)
    kb, vb = ops.kv_dequantize(cache, N - 4, 4)
    want = O.quantize(rows.cpu(), "int8")[2]
    assert (kb[:, 1:].cpu().double() - want).abs().max() <= want.abs().max() * 2.0 ** -11
    assert torch.equal(kb[:, 1:], -vb[:, 1:])
    q = torch.randn(B, 8 * H, 128, generator=g, device=DEV).half()
    q[2, -8:, :] = rows[2, 2, -1] * 0.5        # the last head's queries look at its last token
    out = ops.flash_decoding_quantized(q, cache, SM)
    one = ops.QuantizedKV(k[2], v[2], ks[2], vs[2])
    shared = ops.shared_prefix_attention(q, one, None, SM)
    ops.check_status(torch.device(DEV))
    kd, vd = (c[2, :, H - 1].double() * s[2, H - 1].double()[:, None] for c, s in ((k, ks), (v, vs)))
    for b, got in ((2, out), (2, shared), (0, shared)):
        ref = torch.softmax(q[b, -8:].double() @ kd.T * SM, -1) @ vd
        qb = q[b:b + 1, -8:].cpu()
        tol = O.tolerance(ref.cpu(), qb, SM, [kd[:, None].cpu()], [vd[:, None].cpu()], N, torch.float16, "int8")
        assert ((got[b, -8:].double() - ref).abs().cpu() <= tol).all()


def test_a_decode_loop_over_a_quantised_prefix_and_cache():
    """The operators together: a prompt is quantised once into a shared cache, then every step appends one
    token to each row's own cache and attends over both; and reading the caches back gives what the
    attention saw."""
    from topk_attn_b200 import ops
    B, Hq, Hkv, Np, steps = 3, 8, 2, 333, 5
    g = torch.Generator().manual_seed(3)
    for kind in ("int8", "fp8", "int4"):
        prompt = [torch.randn(Np, Hkv, 128, generator=g).half() for _ in range(2)]
        prefix = ops.quantized_kv_cache(Np, Hkv, kind, device=DEV)
        ops.kv_append_quantized(prefix, prompt[0].to(DEV), prompt[1].to(DEV), 0)
        cache = ops.quantized_kv_cache(16, Hkv, kind, batch=B, device=DEV)
        pos = torch.tensor([0, 2, 5], dtype=torch.int32, device=DEV)
        start = [torch.randn(B, 5, Hkv, 128, generator=g).half().to(DEV) for _ in range(2)]
        ops.kv_append_quantized(cache, *start, 0, pos)
        pk, pv = (O.quantize(x, kind)[2] for x in prompt)
        for _ in range(steps):
            q = torch.randn(B, Hq, 128, generator=g).half()
            new = [torch.randn(B, 1, Hkv, 128, generator=g).half().to(DEV) for _ in range(2)]
            ops.kv_append_quantized(cache, *new, pos)
            pos += 1
            out = ops.shared_prefix_attention(q.to(DEV), prefix, cache, SM, pos)
            kb, vb = (x.cpu() for x in ops.kv_dequantize(cache, 0, 16))
            ref = O.attention(q, SM, (pk, pv), (kb, vb), pos.cpu())
            # the read-back values are rounded to fp16 once more: half a step in scores and values
            tol = O.tolerance(ref, q, SM, [pk, kb], [pv, vb], Np + 16, torch.float16, "int4")
            assert ((out.cpu().double() - ref).abs() <= tol).all()
        ops.check_status(torch.device(DEV))


def test_captured_graphs_replayed_at_the_same_time_and_other_streams():
    """Two captured steps replayed on two streams at once, mixed with an eager call on a third: each has
    scratch of its own."""
    from topk_attn_b200 import ops
    cases, graphs = [], []
    for i, (B, Np, N) in enumerate(((8, 4000, 700), (6, 5000, 900))):
        q, prefix, own = make(B, 16, 4, Np, N, "", torch.float16, 20 + i)
        dq, dp, do = q.to(DEV), device_cache(prefix, ""), device_cache(own, "")
        lens = torch.full((B,), N, dtype=torch.int32, device=DEV)
        ref = ops.shared_prefix_attention(dq, dp, do, SM, lens)
        out = torch.empty_like(dq)
        gr = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(gr):
            ops.shared_prefix_attention(dq, dp, do, SM, lens, out=out)
        cases.append((dq, dp, do, lens, ref, out))
        graphs.append(gr)
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    extra = []
    for _ in range(20):
        for gr, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                gr.replay()
        with torch.cuda.stream(streams[2]):
            dq, dp, do, lens, _, _ = cases[0]
            extra.append(ops.shared_prefix_attention(dq, dp, do, SM, lens))
    torch.cuda.synchronize()
    for *_, ref, out in cases:
        assert torch.equal(ref, out)
    assert all(torch.equal(x, cases[0][4]) for x in extra)
    cases[0][3].fill_(3)          # lengths are read at replay
    want = ops.shared_prefix_attention(*cases[0][:3], SM, cases[0][3])
    graphs[0].replay()
    torch.cuda.synchronize()
    assert torch.equal(cases[0][5], want)
    ops.check_status(torch.device(DEV))


def test_first_calls_of_a_process_inside_a_capture():
    """A process whose very first calls are captured: scratch and status come from the graph's memory."""
    import subprocess
    import sys
    code = """
import torch
from topk_attn_b200 import ops
torch.manual_seed(0)
q = torch.randn(40, 8, 128, device="cuda", dtype=torch.float16)
pk, pv = (torch.randn(300, 2, 128, device="cuda", dtype=torch.float16) for _ in range(2))
cache = ops.quantized_kv_cache(64, 2, "int8", batch=40)
rows = torch.randn(40, 9, 2, 128, device="cuda", dtype=torch.float16)
lens = torch.full((40,), 9, device="cuda", dtype=torch.int32)
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    ops.kv_append_quantized(cache, rows, rows, 0)
    a = ops.flash_decoding_quantized(q, cache, 0.1, lens)
    b = ops.shared_prefix_attention(q, (pk, pv), None, 0.1)
for _ in range(3):
    g.replay()
torch.cuda.synchronize()
assert torch.equal(a, ops.flash_decoding_quantized(q, cache, 0.1, lens))
assert torch.equal(b, ops.shared_prefix_attention(q, (pk, pv), None, 0.1))
ops.check_status()
print("captured first")
"""
    import os
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    res = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert "captured first" in res.stdout, res.stderr[-2000:]


def test_output_in_place_of_the_queries_and_another_stream():
    from topk_attn_b200 import ops
    q, prefix, own = make(20, 8, 2, 700, 90, "", torch.float16, 11)
    pre, cache = device_cache(prefix, ""), device_cache(own, "")
    ref = ops.shared_prefix_attention(q.to(DEV), pre, cache, SM)
    dq = q.to(DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = ops.shared_prefix_attention(dq, pre, cache, SM, out=dq)
    torch.cuda.synchronize()
    assert out.data_ptr() == dq.data_ptr() and torch.equal(dq, ref)


def test_refusals():
    from topk_attn_b200 import capi, ops
    q, prefix, own = make(2, 8, 2, 50, 40, "", torch.float16, 1)
    dq, pre, cache = q.to(DEV), device_cache(prefix, ""), device_cache(own, "")
    lens = torch.full((2,), 3, dtype=torch.int32, device=DEV)
    quant = ops.quantized_kv_cache(40, 2, "int8", batch=2, device=DEV)
    shared = ops.quantized_kv_cache(40, 2, "int8", device=DEV)
    f = ops.shared_prefix_attention
    bad = [(dq, None, None, SM), (q, pre, cache, SM), (dq.float(), pre, cache, SM), (dq[..., :64], pre, cache, SM),
           (dq, cache, pre, SM), (dq, pre, tuple(x[:1] for x in cache), SM), (dq, pre, cache, SM, lens[:1]),
           (dq, pre, cache, SM, lens.long()), (dq, pre, None, SM, lens), (dq, pre, (cache[0], cache[1][:, :3]), SM),
           (dq, pre, (cache[0], cache[1].bfloat16()), SM), (dq, (pre[0][:, :1], pre[1][:, :1]), cache, SM),
           (dq, pre, cache, SM, lens, dq.bfloat16()), (dq, pre, tuple(x.cpu() for x in cache), SM),
           (dq.transpose(0, 1).contiguous().transpose(0, 1), pre, cache, SM)]
    for args in bad:
        with pytest.raises(ValueError):
            f(*args)
    wrong = [(dq, pre, quant, SM), (dq, pre, cache, 0.0), (dq, pre, cache, math.nan), (dq.bfloat16(), pre, cache, SM),
             (dq[:, :7].contiguous(), pre, cache, SM),
             (dq, pre, tuple(x.new_zeros(2, 40, 260)[..., :256].unflatten(-1, (2, 128)) for x in cache), SM)]
    for args in wrong:
        with pytest.raises(capi.RaError):
            f(*args)
    with pytest.raises(ValueError):
        ops.flash_decoding_quantized(dq, cache, SM)
    with pytest.raises(ValueError):
        ops.flash_decoding_quantized(dq, shared, SM, lens)
    with pytest.raises(ValueError):
        ops.flash_decoding_quantized(dq, ops.QuantizedKV(quant.k, quant.v, quant.k_scale[:, :, :9], quant.v_scale), SM)
    ops.check_status(torch.device(DEV))
