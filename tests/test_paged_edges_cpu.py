"""Refusals and out-of-the-ordinary calls of ops.paged on its CPU path."""
import pytest
import torch

from nano_gpic_b200.ops import paged as P
from test_paged_cpu import _cache, _i32


def test_scale_pools_of_odd_alignment_are_refused():
    kv, table = _cache([4], 1, 64, 8, "e4m3")
    odd = torch.zeros(kv.k_sf.numel() + 1, dtype=torch.uint8)[1:].view(kv.k_sf.shape)
    x = torch.randn(4, 64).bfloat16()
    for sf in ((odd, kv.v_sf), (kv.k_sf, odd)):
        bad = P.PagedKV(kv.k, kv.v, *sf)
        for call in (lambda: P.cache_write(bad, x, x, table, _i32([0]), _i32([0, 4])),
                     lambda: P.cache_read(bad, table, _i32([0]), _i32([0, 4]), 4),
                     lambda: P.paged_attn(x, bad, table, _i32([4]), _i32([0, 4]), 4, 4)):
            with pytest.raises(RuntimeError, match="paged: scale pools"):
                call()


SCALES = [0.0, -0.1, float("nan"), float("inf"), 1e-50, 1e39]


@pytest.mark.parametrize("scale", SCALES)
def test_scales_that_are_no_positive_fp32_are_refused(scale):
    kv, table = _cache([4], 1, 64, 8, "bf16")
    x = torch.randn(4, 64).bfloat16()
    P.cache_write(kv, x, x, table, _i32([0]), _i32([0, 4]))
    with pytest.raises(RuntimeError, match="paged: scale"):
        P.paged_attn(x, kv, table, _i32([4]), _i32([0, 4]), 4, 4, scale=scale)
