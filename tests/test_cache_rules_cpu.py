"""Rules of the cache operators that need no device: what their sources may not do, sizes that have to be refused."""
import os

import pytest

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
