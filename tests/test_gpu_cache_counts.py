"""Counts of a padded batch that are no counts."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("kind", ["int8", "fp8", "int4"])
def test_the_least_int32_as_a_count_writes_nothing(kind):
    """It is below zero like any other, also for the tiles whose first row is taken from it."""
    from topk_attn_b200 import ops
    T, H = 300, 2
    rows = torch.randn(2, T, H, 128, device=DEV, dtype=torch.float16)
    cache = ops.quantized_kv_cache(T, H, kind, batch=2, device=DEV)
    counts = torch.tensor([-2 ** 31, 2 ** 31 - 1], dtype=torch.int32, device=DEV)
    ops.kv_append_quantized(cache, rows, rows, 0, counts)
    ops.check_status(torch.device(DEV))
    for x in (cache.k, cache.v):
        assert not x.view(torch.uint8)[0].any() and x.view(torch.uint8)[1].any(-1).all()
    for s in (cache.k_scale, cache.v_scale):
        assert not s[0].any() and s[1].all()
