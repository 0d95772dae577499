"""The router's choice and rows sorted by expert and back (nestquant_b200.routing) against the definitions in 64 bits, and their gradients against the
formulas and against differences.

Tolerances: a result is off by its rounding, eps / 2 of its type, and by what 32-bit arithmetic loses on the way, 2^-24 of each intermediate
value: counted below where a test says so."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
U = 2.0 ** -24


def half_step(t):
    return torch.finfo(t).eps / 2


def close(got, want, tol, what=""):
    """|got - want| <= tol (a tensor or number), element by element, plus half a step of got's type"""
    w = want.to(got.device).double()
    bad = ~((got.double() - w).abs() <= tol + half_step(got.dtype) * w.abs() * (1 + 1e-6) + torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps)
    assert not bad.any(), (what, int(bad.sum()), got[bad][:4], w[bad][:4])


# ---- route ----------------------------------------------------------------------------------------------------------------------

def choice(logits, bias, topk):
    """ids by the exact scores, on the host, sorted with Python's integers and floats"""
    l = logits.double().cpu()
    b = None if bias is None else bias.double().cpu()
    out = []
    for t in range(l.shape[0]):
        row = l[t].tolist()
        rank = []
        for e, v in enumerate(row):
            if math.isnan(v) or v == -math.inf or (b is not None and (math.isnan(b[e]) or b[e] == -math.inf)):
                continue
            s = v if b is None else (1 / (1 + math.exp(-v)) if v > -700 else 0.0) + float(b[e])
            rank.append((-s, e))
        ids = [e for _, e in sorted(rank)[:topk]]
        out.append(ids + [-1] * (topk - len(ids)))
    return torch.tensor(out, dtype=torch.int64).view(l.shape[0], topk)


def weights(logits, sel, score, renorm, scale):
    l = logits.double()
    have = sel >= 0
    p = torch.sigmoid(l)
    if score == "softmax":
        ok = ~l.isnan()
        p = torch.softmax(torch.where(ok, l, -math.inf), 1)
    w = torch.where(have, p.gather(1, sel.clamp(min=0)), 0)
    if renorm:
        lg = torch.where(have, l.gather(1, sel.clamp(min=0)), -math.inf)
        f = torch.nn.functional.logsigmoid(lg) if score == "sigmoid" else lg
        w = torch.where(have, torch.softmax(f, 1), 0)         # p / sum p through the logarithms
    return scale * w


def logits_of(T, E, dtype=F32, seed=1, spread=1.5):
    g = torch.Generator("cuda").manual_seed(seed)
    return (spread * torch.randn(T, E, generator=g, device="cuda")).to(dtype)


@pytest.mark.parametrize("T,E,topk,dtype,out,score,renorm,bias", [
    (1, 1, 1, F32, F16, "sigmoid", True, True),
    (5, 8, 8, F32, F32, "sigmoid", True, True),            # every expert
    (33, 64, 4, BF16, F16, "softmax", True, False),
    (7, 33, 3, F16, BF16, "sigmoid", False, True),         # one expert more than lanes
    (130, 160, 6, F32, F32, "softmax", False, False),
    (257, 256, 8, F32, F16, "sigmoid", True, True),
    (64, 255, 9, BF16, F32, "sigmoid", True, False),       # rows that start off 16 bytes
    (3, 1024, 32, F32, F32, "sigmoid", True, True),        # the largest
    (9, 1001, 32, F16, F32, "softmax", True, False),
])
def test_route_matches_the_definition(T, E, topk, dtype, out, score, renorm, bias):
    from nestquant_b200 import routing
    l = logits_of(T, E, dtype, seed=T + E)
    b = 0.2 * torch.randn(E, generator=torch.Generator("cuda").manual_seed(E), device="cuda") if bias else None
    sel, rw = routing.route(l, topk, score=score, bias=b, renorm=renorm, scale=2.5, dtype=out)
    assert sel.dtype == torch.int64 and rw.dtype == out and sel.shape == rw.shape == (T, topk)
    want = choice(l, b, topk)
    assert torch.equal(sel.cpu(), want)
    # exponentials of 2 ulp, a sum of up to topk (renormalised) or of a lane's 32 and five more, a quotient, two products
    close(rw, weights(l, sel, score, renorm, 2.5), 2.5 * (4 + 2 + topk + 40) * U * weights(l, sel, score, renorm, 1.0), "weights")


def test_route_equal_scores_go_to_the_lowest_id():
    from nestquant_b200 import routing
    for E in (5, 40, 256, 700):
        k = min(8, E)
        for l in (torch.zeros(3, E, device="cuda"), torch.full((3, E), -0.0, device="cuda")):
            l[1, ::2] = 0.0                                    # both zeros are one value
            for b in (None, torch.zeros(E, device="cuda")):
                sel, rw = routing.route(l, k, bias=b, dtype=F32)
                assert torch.equal(sel.cpu(), torch.arange(k).expand(3, k))
                close(rw, torch.full((3, k), 1 / k), 8 * U)


def test_route_order_of_scores_that_32_bits_cannot_tell_apart():
    """sigmoids within a rounding of one another, whose order the bias or the next digit decides; equal pairs among them"""
    from nestquant_b200 import routing
    E, T = 96, 64
    g = torch.Generator("cuda").manual_seed(3)
    l = 9 + torch.rand(T, E, generator=g, device="cuda") * 6               # 1 - sigmoid down to 3e-7: steps of 6e-8 are coarse
    l[:, 50:60] = l[:, 40:50]
    b = torch.zeros(E, device="cuda")
    b[::3] = 2.0 ** -25
    b[50:60] = b[40:50]
    sel, _ = routing.route(l, 20, bias=b, dtype=F32)
    want = choice(l, b, 20)
    near = torch.sigmoid(l.float()).cpu().gather(1, want)
    assert (near[:, :-1] == near[:, 1:]).float().mean() > 0.05           # the case is what it says
    assert torch.equal(sel.cpu(), want)
    large = torch.full((E,), 3e7, device="cuda")                         # a bias beside which sigmoids vanish in 32 bits
    sel, _ = routing.route(l, 20, bias=large, dtype=F32)
    assert torch.equal(sel.cpu(), choice(l, large, 20))
    sel, _ = routing.route(l[:, :32].contiguous(), 32, bias=large[:32], dtype=F32)
    assert torch.equal(sel.cpu(), choice(l[:, :32], large[:32], 32))


@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
def test_route_masked_experts_and_rows(score):
    from nestquant_b200 import routing
    T, E, k = 8, 70, 6
    l = logits_of(T, E)
    l[0] = -math.inf                         # nothing left
    l[1, 3:] = -math.inf                     # three left
    l[2, ::2] = math.nan
    l[3] = math.nan
    l[4, 1:] = torch.finfo(F32).min          # the lowest value is not a mask
    l[5, 10:] = -300.0                       # sigmoids that 32 bits do not hold
    l[5, :10] = -math.inf
    b = None
    if score == "sigmoid":
        b = torch.zeros(E, device="cuda")
        b[20:25] = -math.inf
        b[25] = math.nan
    for renorm in (True, False):
        sel, rw = routing.route(l, k, score=score, bias=b, renorm=renorm, scale=1.0, dtype=F32)
        assert torch.equal(sel.cpu(), choice(l, b, k))
        w = weights(torch.where(l == torch.finfo(F32).min, -3e38, l.double()), sel, score, renorm, 1.0)
        close(rw, w, 64 * U * w.abs() + 1e-37, (score, renorm))          # (what is below 32 bits' range is 0 there)
        assert (rw[0] == 0).all() and (sel[0] == -1).all() and (sel[3] == -1).all() and (sel[1, 3:] == -1).all()


def test_route_strides_streams_and_empty_calls():
    from nestquant_b200 import routing
    wide = logits_of(40, 300, seed=5)
    for l in (wide[:, 7:200], wide[::3, :128], wide.t()[:64], wide[:1, :5], wide[0:1].expand(4, 300)):
        sel, rw = routing.route(l, 4, dtype=F32)
        assert torch.equal(sel.cpu(), choice(l, None, 4))
    sel, rw = routing.route(wide[:0], 4)
    assert sel.shape == rw.shape == (0, 4)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        sel, _ = routing.route(wide, 8, dtype=F32)
        got = sel.clone()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got.cpu(), choice(wide, None, 8))


@pytest.mark.parametrize("T,E,topk,dtype,score,renorm,bias", [
    (4, 1, 1, F32, "sigmoid", False, False), (17, 40, 8, F32, "sigmoid", True, True), (31, 256, 8, BF16, "sigmoid", True, False), (9, 120, 6, F16, "softmax", False, False),
    (5, 500, 32, F32, "softmax", True, False), (3, 1000, 10, F32, "softmax", False, False), (33, 64, 4, F32, "sigmoid", False, True),
])
def test_route_gradient(T, E, topk, dtype, score, renorm, bias):
    from nestquant_b200 import routing
    l = logits_of(T, E, dtype, seed=T).requires_grad_(True)
    if E > 4:
        with torch.no_grad():
            l[1, 2:] = -math.inf                              # a row with two experts left
    b = 0.1 * torch.randn(E, device="cuda") if bias else None
    drw = torch.randn(T, topk, generator=torch.Generator("cuda").manual_seed(7), device="cuda")
    sel, rw = routing.route(l, topk, score=score, bias=b, renorm=renorm, scale=2.5, dtype=F32)
    got, = torch.autograd.grad(rw, l, drw)
    assert got.dtype == dtype and not sel.requires_grad
    wide = l.detach().double().requires_grad_(True)
    w = weights(wide, sel, score, renorm, 2.5)
    want, = torch.autograd.grad(w, wide, drw.double())
    want = torch.where(l.detach() == -math.inf, 0, want.nan_to_num())
    # differences g - sum of g r of size max|g|, everything else relative to p: some 60 roundings in the longest chain
    size = 2.5 * drw.abs().amax(1, keepdim=True).double()
    close(got, want, 64 * U * size, "formula")
    if dtype == F32:                                          # and differences of the weights themselves, the choice held
        step, v = 1e-4, torch.randn(T, E, device="cuda").double()
        at = lambda h: (weights(l.detach().double().masked_fill(l.detach() == -math.inf, -1e30) + h * v, sel, score, renorm, 2.5) * drw.double()).sum()
        d = (at(step) - at(-step)) / (2 * step)
        assert abs(float(d - (got.double() * v).sum())) <= 1e-5 * (1 + abs(float(d))) + 64 * U * float((size * v.abs()).sum())


# ---- rows by expert and back ----------------------------------------------------------------------------------------------------

def picks(T, E, topk, seed=1, holes=True):
    g = torch.Generator("cuda").manual_seed(seed)
    sel = torch.rand(T, max(E, topk), generator=g, device="cuda").argsort(1)[:, :topk].contiguous()
    if E < topk:
        sel = torch.randint(0, E, (T, topk), generator=g, device="cuda")
    if holes and T > 2:
        sel[torch.rand(T, topk, generator=g, device="cuda") < 0.1] = -1
        sel[1] = -1                              # a token without any expert
        sel[2, 0] = E                            # one that is not here
        sel[0, -1] = 1 << 40
    return sel


def places(sel, E):
    """sorted (expert, pick) of the live picks, then the others; by Python's sort"""
    flat = sel.flatten().tolist()
    order = sorted(range(len(flat)), key=lambda i: (flat[i] if 0 <= flat[i] < E else E, i))
    live = sum(0 <= e < E for e in flat)
    start = [sum(1 for e in flat if 0 <= e < E and e < x) for x in range(E + 1)]
    return torch.tensor(order, dtype=torch.int64), live, torch.tensor(start, dtype=torch.int32)


@pytest.mark.parametrize("T,E,topk", [(1, 1, 1), (3, 5, 2), (40, 64, 4), (2000, 7, 4), (32, 256, 8), (300, 1024, 31), (3000, 200, 3), (64, 33, 4), (65, 33, 4), (8191, 17, 8), (20000, 300, 4)])
def test_sort_picks(T, E, topk):
    from nestquant_b200 import routing
    sel = picks(T, E, topk)
    o = routing.sort_picks(sel, E)
    order, live, start = places(sel, E)
    assert torch.equal(o.start.cpu(), start) and int(o.start[-1]) == live
    pos = torch.empty(T * topk, dtype=torch.int32)
    pos[order] = torch.arange(T * topk, dtype=torch.int32)
    assert torch.equal(o.pos.cpu(), pos.view(T, topk))
    assert torch.equal(o.token.cpu().long(), order // topk)
    e = sel.flatten().cpu()[order]
    assert torch.equal(o.expert.cpu().long(), torch.where((e >= 0) & (e < E), e, E))


SHAPES = [(1, 3, 1, 8), (5, 4, 2, 1), (33, 16, 8, 1000), (9, 256, 8, 6144), (70, 12, 3, 77), (64, 9, 10, 130), (130, 5, 17, 64), (3, 2, 33, 24)]


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("T,E,topk,H", SHAPES)
def test_dispatch_and_its_gradient(T, E, topk, H, dtype):
    from nestquant_b200 import routing
    g = torch.Generator("cuda").manual_seed(T)
    sel = picks(T, E, topk, holes=T > 3)
    o = routing.sort_picks(sel, E)
    order, live, _ = places(sel, E)
    x = torch.randn(T, H, generator=g, device="cuda").to(dtype).requires_grad_(True)
    xs = routing.dispatch(x, o)
    want = x.detach()[(order // topk).cuda()]
    want[live:] = 0
    assert torch.equal(xs, want)
    d = torch.randn(T * topk, H, generator=g, device="cuda").to(dtype)
    d[live:] = math.nan                          # what comes in for picks without an expert does not count
    got, = torch.autograd.grad(xs, x, d)
    add = lambda v: torch.zeros(T, H, dtype=torch.float64, device="cuda").index_add_(0, (order[:live] // topk).cuda(), v[:live].double())
    close(got, add(d), topk * U * add(d.abs()), "dx")         # topk additions in 32 bits
    if T > 3:
        assert (got[1] == 0).all()


@pytest.mark.parametrize("dtype,out,wt", [(F32, F32, F32), (F16, F16, F16), (F16, F32, F16), (BF16, BF16, F32), (BF16, F32, BF16)])
@pytest.mark.parametrize("T,E,topk,H", SHAPES)
def test_combine_and_its_gradients(T, E, topk, H, dtype, out, wt):
    from nestquant_b200 import routing
    g = torch.Generator("cuda").manual_seed(T + 1)
    sel = picks(T, E, topk, holes=T > 3)
    o = routing.sort_picks(sel, E)
    order, live, _ = places(sel, E)
    y = torch.randn(T * topk, H, generator=g, device="cuda").to(dtype)
    y[live:] = math.nan                          # rows that nobody computed
    y.requires_grad_(True)
    rw = torch.randn(T, topk, generator=g, device="cuda").to(wt)
    rw[0, 0] = 0                                 # a weight of 0 has a gradient
    rw.requires_grad_(True)
    got = routing.combine(y, o, rw, dtype=out)
    assert got.dtype == out
    token, at = (order // topk).cuda()[:live], order.cuda()[:live]
    yd, wd = y.detach().double()[:live], rw.detach().double().flatten()[at]
    add = lambda v: torch.zeros(T, H, dtype=torch.float64, device="cuda").index_add_(0, token, v)
    close(got, add(yd * wd[:, None]), 2 * topk * U * add((yd * wd[:, None]).abs()), "out")
    d = torch.randn(T, H, generator=g, device="cuda").to(out)
    dy, drw = torch.autograd.grad(got, (y, rw), d)
    want = torch.zeros(T * topk, H, dtype=torch.float64, device="cuda")
    want[:live] = d.double()[token] * wd[:, None]
    close(dy, want, U * want.abs(), "dy")        # one product
    assert (dy[live:] == 0).all()
    dot, size = (torch.zeros(T * topk, dtype=torch.float64, device="cuda") for _ in range(2))
    dot[at] = (yd * d.double()[token]).sum(1)
    size[at] = (yd * d.double()[token]).abs().sum(1)
    # a product, a thread's share of the additions, eight of the warp and the CTA
    close(drw, dot.view(T, topk), (H // 32 + 16 + 2) * 2 * U * size.view(T, topk), "drw")
    only, = torch.autograd.grad(routing.combine(y.detach(), o, rw, dtype=out), rw, d)          # one gradient alone
    assert torch.equal(only, drw)
    only, = torch.autograd.grad(routing.combine(y, o, rw.detach(), dtype=out), y, d)
    assert torch.equal(only, dy)


def test_rows_off_16_bytes_and_with_strides():
    from nestquant_b200 import routing
    T, E, topk, H = 21, 8, 3, 64
    sel = picks(T, E, topk)
    o = routing.sort_picks(sel, E)
    order, live, _ = places(sel, E)
    token = (order // topk).cuda()
    buf = torch.randn(T * 3, 200, device="cuda").half()
    for x in (buf[:T, 1:65], buf[:T, 4:68], buf[::3, 8:72], buf.t()[:T, :64], buf[:1, :64].expand(T, 64)):
        xs = routing.dispatch(x, o)
        want = x[token].clone()
        want[live:] = 0
        assert torch.equal(xs, want)
    flat = torch.randn(T * topk * H + 1, device="cuda").bfloat16()
    y = flat[1:].view(T * topk, H)               # contiguous, two bytes off
    rw = torch.rand(T, topk, device="cuda")
    aligned = routing.combine(y.clone(), o, rw)
    assert torch.equal(routing.combine(y, o, rw), aligned)
    assert torch.equal(routing.combine(y, o, rw.t().contiguous().t()), aligned)


def test_rows_past_32_bit_offsets():
    from nestquant_b200 import routing
    T, topk, H, E = 36000, 8, 8192, 16                        # 2.4e9 elements
    sel = torch.arange(T * topk, device="cuda").view(T, topk) % E
    o = routing.sort_picks(sel, E)
    x = torch.randn(T, 1, device="cuda").bfloat16() + torch.arange(H, device="cuda").bfloat16()
    xs = routing.dispatch(x, o)
    for p in (0, T * topk // 2, T * topk - 1):
        assert torch.equal(xs[p], x[int(o.token[p])])
    out = routing.combine(xs, o, torch.full((T, topk), 0.125, device="cuda"))
    assert torch.equal(out[-1], x[-1]) and torch.equal(out[0], x[0])     # 8 x 1/8 of the same row: exact
    del xs, out
    torch.cuda.empty_cache()


def test_a_training_step_captured_and_replayed():
    """route -> sort -> dispatch -> an elementwise stand-in for the experts -> combine with its backward pass in one CUDA graph, on inputs that change"""
    from nestquant_b200 import routing
    T, E, topk, H = 50, 24, 4, 136
    g = torch.Generator("cuda").manual_seed(11)
    x = torch.randn(T, H, generator=g, device="cuda").bfloat16().requires_grad_(True)
    l = logits_of(T, E, seed=8).requires_grad_(True)
    d = torch.randn(T, H, generator=g, device="cuda")

    def step():
        sel, rw = routing.route(l, topk, dtype=F32, scale=2.5)
        o = routing.sort_picks(sel, E)
        y = torch.tanh(routing.dispatch(x, o)) * (1 + o.expert[:, None] % 3)
        out = routing.combine(y, o, rw, dtype=F32)
        return (out.detach(),) + torch.autograd.grad(out, (x, l), d)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for seed in (1, 2):
        with torch.no_grad():
            x.copy_(torch.randn(T, H, generator=g, device="cuda"))
            l.copy_(logits_of(T, E, seed=seed))
        graph.replay()
        got = [t.clone() for t in held]
        for a, b in zip(got, step()):
            assert torch.equal(a, b)


def test_gradients_cannot_be_differentiated_again():
    from nestquant_b200 import routing
    l = logits_of(6, 16).requires_grad_(True)
    x = torch.randn(6, 32, device="cuda", requires_grad=True)
    sel, rw = routing.route(l, 2, dtype=F32)
    o = routing.sort_picks(sel, 16)
    out = routing.combine(routing.dispatch(x, o).square(), o, rw)
    gl, gx = torch.autograd.grad(out.square().sum(), (l, x), create_graph=True)
    once = torch.autograd.grad(routing.combine(routing.dispatch(x, o).square(), o, routing.route(l, 2, dtype=F32)[1]).square().sum(), (l, x))
    assert torch.equal(gl, once[0]) and torch.equal(gx, once[1])
    for g in (gl, gx):
        with pytest.raises(RuntimeError):
            g.sum().backward(retain_graph=True)


def test_unused_outputs_and_frozen_inputs():
    from nestquant_b200 import routing
    l = logits_of(6, 16).requires_grad_(True)
    sel, rw = routing.route(l, 2, dtype=F32)
    assert not sel.requires_grad and rw.requires_grad
    with torch.no_grad():
        assert not routing.route(l, 2)[1].requires_grad
    o = routing.sort_picks(sel, 16)
    y = torch.randn(12, 8, device="cuda")
    out = routing.combine(y, o, rw)
    out.sum().backward()
    assert l.grad is not None and y.grad is None
    l2 = logits_of(6, 16).requires_grad_(True)
    _, rw2 = routing.route(l2, 2, dtype=F32)
    l2.data.add_(0)
    with torch.no_grad():
        l2.add_(1)                                             # changed behind the backward pass: torch says so
    with pytest.raises(RuntimeError):
        rw2.sum().backward()


def test_repeats_have_the_same_bits():
    from nestquant_b200 import routing
    T, E, topk, H = 900, 64, 8, 1000
    sel = picks(T, E, topk)
    y = torch.randn(T * topk, H, device="cuda").bfloat16().requires_grad_(True)
    rw = torch.rand(T, topk, device="cuda").requires_grad_(True)
    d = torch.randn(T, H, device="cuda").bfloat16()
    once = None
    for _ in range(4):
        o = routing.sort_picks(sel, E)
        out = routing.combine(y, o, rw)
        all_ = (o.pos, out, *torch.autograd.grad(out, (y, rw), d))
        once = once or all_
        assert all(torch.equal(a, b) for a, b in zip(once, all_))


def test_refusals():
    from nestquant_b200 import routing
    from nestquant_b200.capi import NestQuantError
    l = torch.zeros(4, 16, device="cuda")
    b = torch.zeros(16, device="cuda")
    o = routing.sort_picks(torch.zeros(4, 2, dtype=torch.int64, device="cuda"), 16)
    x, y, rw = torch.zeros(4, 32, device="cuda"), torch.zeros(8, 32, device="cuda"), torch.zeros(4, 2, device="cuda")
    for call in (
        lambda: routing.route(l, 0), lambda: routing.route(l, 17), lambda: routing.route(torch.zeros(2, 1025, device="cuda"), 2), lambda: routing.route(l.double(), 2),
        lambda: routing.route(torch.zeros(2, 64, device="cuda"), 33), lambda: routing.route(l, 2, score="relu"), lambda: routing.route(l, 2, score="softmax", bias=b),
        lambda: routing.route(l, 2, bias=b.half()), lambda: routing.route(l, 2, bias=b[:8]), lambda: routing.route(l, 2, bias=b.cpu()), lambda: routing.route(l[0], 2),
        lambda: routing.route(l, 2, dtype=torch.float64), lambda: routing.route(l, 2, bias=b.clone().requires_grad_(True)), lambda: routing.route(l.cpu(), 2),
        lambda: routing.sort_picks(torch.zeros(4, 2, dtype=torch.int32, device="cuda"), 16), lambda: routing.sort_picks(torch.zeros(4, 2, dtype=torch.int64, device="cuda"), 1025),
        lambda: routing.sort_picks(torch.zeros(8, dtype=torch.int64, device="cuda"), 16), lambda: routing.sort_picks(torch.zeros(4, 0, dtype=torch.int64, device="cuda"), 16),
        lambda: routing.dispatch(x[:3], o), lambda: routing.dispatch(x.double(), o), lambda: routing.dispatch(x.cpu(), o), lambda: routing.dispatch(x[:, :0], o),
        lambda: routing.combine(y[:7], o, rw), lambda: routing.combine(y, o, rw[:, :1]), lambda: routing.combine(y, o, rw, dtype=F16),
        lambda: routing.combine(y.half(), o, rw, dtype=BF16), lambda: routing.combine(y, o, rw.cpu()), lambda: routing.combine(y, o, rw.double()),
    ):
        with pytest.raises(NestQuantError):
            call()
    out, = torch.autograd.grad(routing.route(l.requires_grad_(True), 2, dtype=F32)[1].sum(), l)
    assert out.shape == l.shape
