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


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("E,topk", [(5, 2), (64, 8), (255, 3), (1000, 32)])
@pytest.mark.parametrize("score,renorm", [("sigmoid", True), ("sigmoid", False), ("softmax", True), ("softmax", False)])
def test_the_gradient_of_a_row_with_nothing_left_is_zero(E, topk, dtype, score, renorm):
    """weights of 0 whatever the logits are; the other rows' gradients are those that they have without it"""
    from nestquant_b200 import routing
    g = torch.Generator("cuda").manual_seed(E)
    l = torch.randn(9, E, generator=g, device="cuda").to(dtype)
    drw = torch.randn(9, topk, generator=g, device="cuda")
    empty = [0, 4, 5, 8]
    l[empty] = -math.inf
    l[4] = math.nan
    l[5, ::2] = math.nan
    l.requires_grad_(True)
    sel, rw = routing.route(l, topk, score=score, renorm=renorm, scale=2.5, dtype=F32)
    got, = torch.autograd.grad(rw, l, drw)
    assert (sel[empty] == -1).all() and (rw[empty] == 0).all()
    assert (got[empty] == 0).all() and not got.isnan().any()
    rest = [t for t in range(9) if t not in empty]
    alone = l.detach()[rest].requires_grad_(True)
    want, = torch.autograd.grad(routing.route(alone, topk, score=score, renorm=renorm, scale=2.5, dtype=F32)[1], alone, drw[rest])
    assert torch.equal(got[rest], want)
