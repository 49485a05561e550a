"""CPU checks of the quantised-cache and shared-prefix entry points: struct mirrors, refusals that need no
device, workspace sizes, and the restatement's own properties."""
import ctypes as C
import math

import pytest
import torch

from oracle import cache_oracle as O
from test_abi_cpu import struct_fields


@pytest.mark.parametrize("cname,pyname", [("ra_kv_cache", "RaKvCache"), ("ra_kv_rows_params", "RaKvRowsParams"),
                                          ("ra_cache_attention_params", "RaCacheAttentionParams")])
def test_ctypes_mirrors_match_header(cname, pyname):
    from topk_attn_b200 import capi
    assert [f[0] for f in getattr(capi, pyname)._fields_] == struct_fields(cname)


def a_cache(capi, fmt, n=100, heads=2):
    c = capi.RaKvCache()
    c.k, c.v, c.format, c.num_tokens = 4096, 8192, fmt, n
    row = 64 if fmt == capi.RA_CACHE_INT4 else 128
    c.head_stride, c.token_stride, c.batch_stride = row, heads * row, n * heads * row
    if fmt >= capi.RA_CACHE_INT8:
        w = 4 if fmt == capi.RA_CACHE_INT4 else 1
        c.k_scale, c.v_scale = 4096, 8192
        c.scale_head_stride, c.scale_batch_stride = w * n, w * n * heads
    return c


def some_rows(capi, fmt):
    p = capi.RaKvRowsParams()
    p.cache, p.caches, p.num_kv_heads, p.head_dim = a_cache(capi, fmt), 3, 2, 128
    p.k_rows, p.v_rows, p.num_rows, p.status = 4096, 8192, 5, 256
    p.k_batch_stride = p.v_batch_stride = 5 * 256
    p.k_token_stride = p.v_token_stride = 256
    p.k_head_stride = p.v_head_stride = 128
    return p


def test_row_refusals_without_a_device():
    from topk_attn_b200 import capi
    lib = capi.lib()
    changes = [("head_dim", 64, 2), ("caches", 0, 1), ("num_kv_heads", 0, 1), ("num_rows", -1, 1), ("row_type", 2, 1),
               ("k_rows", None, 1), ("v_rows", 4104, 1), ("status", None, 1), ("k_token_stride", 250, 1),
               ("v_head_stride", -128, 1), ("position", 96, 1), ("position", -1, 1), ("position", 2 ** 31 - 1, 1)]
    inner = [("k", None), ("v", 4104), ("format", capi.RA_CACHE_FP16), ("format", 7), ("num_tokens", 0),
             ("token_stride", 64), ("token_stride", 264), ("head_stride", 0), ("batch_stride", 0), ("batch_stride", -256),
             ("k_scale", None), ("v_scale", 4098), ("scale_head_stride", 99), ("scale_batch_stride", 0)]
    for fn in (lib.ra_kv_append_quantized, lib.ra_kv_dequantize):
        assert fn(None) == capi.RA_ERR_INVALID_ARGUMENT
        for name, value, code in changes:
            p = some_rows(capi, capi.RA_CACHE_INT8)
            setattr(p, name, value)
            assert fn(C.byref(p)) == code, name
        for name, value in inner:
            p = some_rows(capi, capi.RA_CACHE_INT8)
            setattr(p.cache, name, value)
            assert fn(C.byref(p)) == capi.RA_ERR_INVALID_ARGUMENT, (name, value)
        p = some_rows(capi, capi.RA_CACHE_FP8)
        p.num_rows = 0
        assert fn(C.byref(p)) == capi.RA_OK


def test_attention_refusals_without_a_device():
    from topk_attn_b200 import capi
    lib = capi.lib()

    def params():
        p = capi.RaCacheAttentionParams()
        p.q, p.out, p.status, p.workspace = 4096, 8192, 256, 4096
        p.batch, p.num_q_heads, p.num_kv_heads, p.head_dim, p.sm_scale = 3, 8, 2, 128, 1.0
        p.prefix, p.cache = a_cache(capi, capi.RA_CACHE_FP16, 50), a_cache(capi, capi.RA_CACHE_FP16)
        p.workspace_bytes = 1 << 40
        return p
    assert lib.ra_cache_attention(None) == capi.RA_ERR_INVALID_ARGUMENT
    for name, value, code in [("head_dim", 64, 2), ("batch", 0, 1), ("num_q_heads", 7, 1), ("num_kv_heads", 0, 1),
                              ("type", 5, 1), ("type", 1, 1), ("sm_scale", 0.0, 1), ("sm_scale", -1.0, 1),
                              ("sm_scale", math.nan, 1), ("q", None, 1), ("out", 8200, 1), ("status", None, 1),
                              ("workspace", None, 3), ("workspace", 4100, 3), ("workspace_bytes", 255, 3)]:
        p = params()
        setattr(p, name, value)
        assert lib.ra_cache_attention(C.byref(p)) == code, name
    for name, value in [("num_tokens", -1), ("k", None), ("format", capi.RA_CACHE_BF16), ("format", capi.RA_CACHE_INT8),
                        ("token_stride", 132), ("batch_stride", 0)]:
        p = params()
        setattr(p.cache, name, value)
        assert lib.ra_cache_attention(C.byref(p)) == capi.RA_ERR_INVALID_ARGUMENT, name


def test_workspace_sizes():
    from topk_attn_b200 import capi
    f = capi.lib().ra_cache_attention_workspace_bytes
    assert f(0, 8, 2, 1, 1) == 0 and f(1, 8, 2, -1, 1) == 0
    assert f(1, 8, 2, 0, 0) >= 256
    assert f(4, 32, 8, 4096, 1024) > f(4, 32, 8, 0, 1024) >= 4 * 32 * 130 * 4


@pytest.mark.parametrize("kind", ["int8", "fp8", "int4"])
def test_restated_formats_are_as_near_as_they_should_be(kind):
    x = torch.randn(50, 3, 128, generator=torch.Generator().manual_seed(0)).half()
    codes, scales, values = O.quantize(x, kind)
    g = O.GROUP[kind]
    amax = x.double().abs().unflatten(-1, (-1, g)).amax(-1)
    step = (scales.double()[..., None] * torch.ones(g)).flatten(-2)
    err = (values - x.double()).abs()
    if kind == "fp8":
        assert (amax <= 448 * scales.double()).all() and (amax > 224 * scales.double()).all()
        # half a step: 2^-4 relative, and half of 2^-9 scales where e4m3 is subnormal
        assert (err <= torch.maximum(x.double().abs() * 2.0 ** -4, step * 2.0 ** -10)).all()
    else:
        assert (err <= step * (0.5 + 1e-6)).all()
    packed, _ = O.pack(codes, scales, kind)
    assert packed.shape[-1] == (64 if kind == "int4" else 128)
    if kind == "fp8":
        assert torch.equal(packed.double(), codes)


def test_tensors_off_the_gpu_are_refused():
    from topk_attn_b200 import ops
    cache = ops.quantized_kv_cache(4, 2, "int8", batch=1, device="cpu")
    rows = torch.zeros(1, 1, 2, 128, dtype=torch.float16)
    with pytest.raises(ValueError):
        ops.kv_append_quantized(cache, rows, rows, 0)
    with pytest.raises(ValueError):
        ops.kv_dequantize(cache)
    with pytest.raises(ValueError):
        ops.flash_decoding_quantized(rows[0], cache, 1.0)
    with pytest.raises(ValueError):
        ops.shared_prefix_attention(rows[0], None, cache, 1.0)
    with pytest.raises(ValueError):
        cache.first(5)
