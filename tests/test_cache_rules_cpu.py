"""Rules of the cache operators that need no device: what their sources may not do, sizes that have to be refused."""
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
