"""Calls around the routed experts at the borders of what they document."""
import math

import pytest
import torch

from .test_routing_gpu import choice

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


@pytest.mark.parametrize("topk", [1, 2, 8, 31, 32])
@pytest.mark.parametrize("E", [40, 64, 256, 700])
def test_a_tie_at_the_last_pick_does_not_hide_a_better_expert_behind_it(E, topk):
    """the last pick and the next expert have the same logit and bias, and one behind them a score that only 64 bits tell from theirs"""
    from nestquant_b200 import routing
    l, b = torch.full((6, E), -4.0, device="cuda"), torch.zeros(E, device="cuda")
    b[:topk - 1] = 2 - torch.arange(topk - 1, device="cuda") / 64          # what is ahead of them for sure
    at = topk - 1
    l[0, at:at + 3] = torch.tensor([17.0, 17.0, 18.0])
    l[1, [at, at + 1, E - 1]] = torch.tensor([17.0, 17.0, 17.5], device="cuda")
    l[2, at:] = 17
    l[2, E - 1] = 19                                                      # more than a warp has lanes
    l[3, at:] = 17                                                        # nothing better
    l[4, at:at + 3] = torch.tensor([17.0, 17.0, 16.5])                    # worse
    l[5, at:at + 4] = torch.tensor([17.0, 17.0, 18.0, 18.0])              # better ones tie too
    want = choice(l, b, topk)
    assert want[:3, -1].tolist() == [at + 2, E - 1, E - 1] and want[3:, -1].tolist() == [at, at, at + 2]
    for dtype in (F32, BF16, F16):
        assert torch.equal(routing.route(l.to(dtype), topk, bias=b, dtype=F32)[0].cpu(), want)


@pytest.mark.parametrize("E,topk", [(8, 1), (33, 8), (128, 8), (256, 8), (256, 32), (1000, 6)])
def test_16_bit_logits_whose_sigmoids_are_1_in_32_bits(E, topk):
    """scores that tie often, at the last pick too, among others that 32 bits cannot tell from them"""
    from nestquant_b200 import routing
    g = torch.Generator("cuda").manual_seed(E + topk)
    l = (15 + torch.randint(0, 24, (300, E), generator=g, device="cuda") / 4).bfloat16()
    l[::7, : E // 2] = -2
    b = torch.zeros(E, device="cuda")
    assert torch.equal(routing.route(l, topk, bias=b)[0].cpu(), choice(l, b, topk))
    b[::3] = 2.0 ** -26
    assert torch.equal(routing.route(l, topk, bias=b)[0].cpu(), choice(l, b, topk))


def test_inputs_with_tangents_are_refused():
    """no forward-mode derivative is built, and none is dropped without a word"""
    import torch.autograd.forward_ad as ad
    from nestquant_b200 import routing, w4
    from nestquant_b200.capi import NestQuantError
    l, b, x, y, rw = (torch.randn(s, device="cuda") for s in ((6, 16), (16,), (6, 128), (12, 128), (6, 2)))
    o = routing.sort_picks(routing.route(l, 2)[0], 16)
    q = torch.randint(0, 256, (32, 64), device="cuda", dtype=torch.uint8)
    w = w4.W4(q, torch.ones(32, 1, device="cuda", dtype=F16))
    calls = {
        "logits": (l, lambda t: routing.route(t, 2)), "bias": (b, lambda t: routing.route(l, 2, bias=t)), "x": (x, lambda t: routing.dispatch(t, o)),
        "y": (y, lambda t: routing.combine(t, o, rw)), "rw": (rw, lambda t: routing.combine(y, o, t)), "4-bit x": (x.half(), lambda t: w(t)),
    }
    for name, (t, call) in calls.items():
        call(t)
        with ad.dual_level():
            for leaf in (t, t.clone().requires_grad_(True)):
                dual = ad.make_dual(leaf, torch.ones_like(t))
                with pytest.raises(NestQuantError):
                    call(dual)
                with torch.no_grad(), pytest.raises(NestQuantError):
                    call(dual)
            call(ad.unpack_dual(dual).primal.detach())
        with pytest.raises(RuntimeError):
            torch.func.jvp(call, (t,), (torch.ones_like(t),))


@pytest.mark.parametrize("part", ["pos", "start"])
def test_an_order_that_changed_before_its_backward_pass_is_refused(part):
    from nestquant_b200 import routing
    sel = torch.randint(0, 8, (20, 3), generator=torch.Generator("cuda").manual_seed(1), device="cuda")
    x, y, rw = (torch.randn(s, device="cuda", requires_grad=True) for s in ((20, 16), (60, 16), (20, 3)))
    def both():
        o = routing.sort_picks(sel, 8)
        return o, (routing.dispatch(x, o), x), (routing.combine(y, o, rw), y), (routing.combine(y, o, rw), rw)
    o, *calls = both()
    for out, leaf in calls:
        torch.autograd.grad(out.sum(), leaf)
    o, *calls = both()
    if part == "pos":
        o.pos.copy_(o.pos.flip(0))                             # (a permutation still)
    else:
        o.start[-1] -= 1
    for out, leaf in calls:
        with pytest.raises(RuntimeError, match="changed"):
            torch.autograd.grad(out.sum(), leaf)
    with torch.inference_mode():
        o = routing.sort_picks(sel, 8)                         # (a tensor without a version)
    out = routing.dispatch(x, o)
    for _ in range(2):
        torch.autograd.grad(out, x, torch.ones_like(out), retain_graph=True)
    out = routing.dispatch(x, routing.sort_picks(sel, 8)) + 0
    torch.autograd.grad(out.sum(), x)


@pytest.mark.parametrize("T", [2, 8, 16, 40, 64, 150])
def test_a_rows_bits_do_not_depend_on_the_values_of_other_rows(T):
    """how a row's sums are cut goes by the call's sizes; with one matrix and with one per expert"""
    from nestquant_b200 import w4
    N, K, E, g = 272, 1024, 4, 64
    gen = torch.Generator("cuda").manual_seed(T)
    q = torch.randint(0, 256, (E, N, K // 2), generator=gen, device="cuda", dtype=torch.uint8)
    s = (0.01 * torch.randn(E, N, K // g, generator=gen, device="cuda")).half()
    start = torch.tensor([0, T // 2, T // 2, T - 1, T], dtype=torch.int32, device="cuda")
    x, other = (torch.randn(T, K, generator=gen, device="cuda").half() for _ in range(2))
    for call in (w4.W4(q[0], s[0]), lambda x, dtype: w4.W4(q, s)(x, start=start, dtype=dtype)):
        y = call(x, dtype=F32)
        for r in (0, T // 2, T - 1):
            mixed = other.clone()
            mixed[r] = x[r]
            got = call(mixed, dtype=F32)
            assert torch.equal(got[r], y[r]) and not torch.equal(got, y)


@pytest.mark.parametrize("T,topk,E", [(1, 1, 1), (40, 3, 9), (3000, 4, 200), (9000, 8, 300)])
def test_experts_and_tokens_of_the_sorted_places(T, topk, E):
    """the arrays that nq_sort_picks writes for callers in other languages, in the form of one launch and in that of three"""
    from nestquant_b200 import capi, routing
    g = torch.Generator("cuda").manual_seed(T)
    sel = torch.randint(-1, E + 1, (T, topk), generator=g, device="cuda")
    P, L = T * topk, capi.lib()
    pe, pt, pos = (torch.full((P + 1,), -7, dtype=torch.int32, device="cuda") for _ in range(3))
    start = torch.full((E + 3,), -7, dtype=torch.int32, device="cuda")
    ints = L.nq_pf_sort_scratch_ints(P, E)
    scratch = torch.empty(ints, dtype=torch.int32, device="cuda")
    capi.check(L.nq_sort_picks(*map(capi.ptr, (sel,)), T, topk, E, *map(capi.ptr, (pe, pt, pos, start, scratch)), ints, capi.current_stream()))
    o = routing.sort_picks(sel, E)
    assert torch.equal(pe[:P], o.expert) and torch.equal(pt[:P], o.token) and torch.equal(pos[:P], o.pos.flatten()) and torch.equal(start[:E + 1], o.start)
    flat = sel.flatten().tolist()
    order = sorted(range(P), key=lambda i: (flat[i] if 0 <= flat[i] < E else E, i))
    assert pe[:P].tolist() == [flat[i] if 0 <= flat[i] < E else E for i in order] and pt[:P].tolist() == [i // topk for i in order]
    assert int(start[E + 1]) == P and all(int(t[-1]) == -7 for t in (pe, pt, pos, start))
