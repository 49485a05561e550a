"""Rules of the cache operators that need no device: what their sources may not do, sizes that have to be refused."""
import ctypes as C
import os

import pytest
import torch

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "topk_attn_b200", "csrc")


@pytest.mark.parametrize("name", ["quant_cache.cu", "cache_attend.cu", "prefix_attend.cu"])
def test_kernels_that_are_launched_early_do_not_load_through_the_read_only_path(name):
    """Such a load is defined only for data that nobody writes as long as the kernel lives, and these kernels are
    resident while the kernel before them still writes what they read."""
    with open(os.path.join(CSRC, name)) as f:
        source = f.read()
    assert "griddepcontrol.wait" in source
    for word in ("__ldg", "ldg128_nc", "global.nc"):
        assert word not in source, word


@pytest.mark.parametrize("where", ["prefix", "cache"])
@pytest.mark.parametrize("missing", ["k", "v"])
def test_half_a_cache_is_refused(where, missing):
    from topk_attn_b200 import ops
    q = torch.zeros(2, 4, 128, dtype=torch.float16)
    x = torch.zeros((5, 2, 128) if where == "prefix" else (2, 5, 2, 128), dtype=torch.float16)
    half = (None, x) if missing == "k" else (x, None)
    with pytest.raises(ValueError, match="both k and v"):
        ops.shared_prefix_attention(q, *((half, None) if where == "prefix" else (None, half)), 1.0)


@pytest.mark.parametrize("missing", ["k_scale", "v_scale"])
def test_a_quantised_cache_without_a_scale_is_refused(missing):
    from topk_attn_b200 import ops
    cache = ops.quantized_kv_cache(5, 2, "int8", batch=2, device="cpu")
    setattr(cache, missing, None)
    with pytest.raises(ValueError, match="both scales"):
        ops.flash_decoding_quantized(torch.zeros(2, 4, 128, dtype=torch.float16), cache, 1.0)
    rows = torch.zeros(2, 1, 2, 128, dtype=torch.float16)
    for call in (lambda: ops.kv_append_quantized(cache, rows, rows, 0), lambda: ops.kv_dequantize(cache)):
        with pytest.raises((ValueError, TypeError)):
            call()


def test_more_rows_than_tiles_can_be_counted_are_refused():
    """Rows with a token stride of zero can be as many as an int32 holds; their tiles are counted rounding up."""
    from test_cache_abi_cpu import some_rows
    from topk_attn_b200 import capi
    for fn in (capi.lib().ra_kv_append_quantized, capi.lib().ra_kv_dequantize):
        p = some_rows(capi, capi.RA_CACHE_INT8)
        p.num_rows, p.k_token_stride, p.v_token_stride, p.positions = 2 ** 31 - 1, 0, 0, 4096
        assert fn(C.byref(p)) == capi.RA_ERR_UNSUPPORTED


def test_workspace_of_refused_sizes_is_zero():
    """Products that pass 32 bits ended the process in a division by zero."""
    from topk_attn_b200 import capi
    f = capi.lib().ra_cache_attention_workspace_bytes
    top = 2 ** 31 - 1
    for sizes in [(1000, 1 << 30, 1 << 30, 128, 0), (top, top, 1, 128, 0), (1, top, top, 1, 1), (8, 32, 8, top, 0),
                  (8, 32, 8, 0, top), (2, 7, 2, 5, 5), (1 << 20, 32, 8, 64, 64)]:
        assert f(*sizes) == 0, sizes
    assert f(1 << 19, 32, 8, 64, 64) > 0 and f(1, 1, 1, top - 4095, top - 4095) > 0
