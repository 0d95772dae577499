"""Calls around the routed experts at the borders of what they document."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def test_a_sort_whose_counts_no_array_can_hold_is_refused():
    """before anything is made: the ids are one element seen 671 million times"""
    from nestquant_b200 import routing
    from nestquant_b200.capi import NestQuantError
    sel = torch.zeros(1, 1, dtype=torch.int64, device="cuda").expand(1 << 27, 5)
    before = torch.cuda.memory_allocated()
    with pytest.raises(NestQuantError, match="more than an array can hold"):
        routing.sort_picks(sel, 1024)
    assert torch.cuda.memory_allocated() == before
