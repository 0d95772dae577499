"""The router's choice, and tokens' rows sorted by expert and back: what stands around the experts of a layer, with the gradients that a router
needs when it is trained.

    sel, rw = routing.route(logits, 8, bias=bias, scale=2.5)      # ids and weights as MoELayer takes them
    order = routing.sort_picks(sel, E)                            # for experts that are not this library's planes:
    xs = routing.dispatch(x, order)                               #   rows sorted by expert, order.start = where each expert's begin
    out = routing.combine(experts(xs, order.start), order, rw)    #   weighted sums of the picks' rows

Everything is enqueued on the current stream of the tensors' device without a host sync, can be captured in a CUDA graph, and gives the same
bits every time.  route, dispatch and combine are differentiable (once) in logits, x, y and rw; a call whose tensors need no gradient does not enter
autograd.  To capture a backward pass, use torch.autograd.grad, or leaves that no eager graph still holds: the engine joins the stream
on which a leaf's gradient was first accumulated, which a capture forbids.  Errors are NestQuantError, raised before anything is enqueued.
"""
import torch

from .capi import NestQuantError, element_types, launch, lib

_TYPE = element_types()
_SCORES = {"sigmoid": 0, "softmax": 1}


def _rows(t, name, types=_TYPE):
    if not (isinstance(t, torch.Tensor) and t.is_cuda and t.dim() == 2 and t.dtype in types):
        raise NestQuantError(f"{name}: expected a CUDA tensor of two dimensions, {' / '.join(str(d)[6:] for d in types)}")
    return t


def _same_device(a, b, name):
    if a.get_device() != b.get_device():
        raise NestQuantError(f"{name}: tensors on different devices")


def _strided(t):
    """t, or a copy, whose rows are contiguous and do not overlap"""
    return t if t.stride(1) == 1 and t.stride(0) >= t.shape[1] or t.numel() == 0 else t.contiguous()


def _stride(t):
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _once(grad):
    if torch.is_grad_enabled() and grad is not None and grad.requires_grad:
        raise NestQuantError("gradients of gradients: not built")


# ---- route ----------------------------------------------------------------------------------------------------------------------

def route(logits, topk, score="sigmoid", bias=None, renorm=True, scale=1.0, dtype=torch.float16):
    """Router logits [T,E] (fp32, fp16 or bf16; E <= 1024) -> (sel int64 [T,topk], rw [T,topk] of `dtype`), topk <= 32.

    Chosen are the topk experts with the largest sigmoid(logit) + bias (bias: fp32 [E], sees the choice only), without a bias those with the largest
    logits; ids in falling order of the score, equal scores by the lowest id.  The order is that of the exact scores, not of their
    roundings.  Experts whose logit or bias is -inf or NaN are never chosen; where fewer than topk are left, the last ids are -1 and
    their weights 0, picks that every call of this library skips.
    rw = scale * p, divided by the sum of the chosen p if renorm; p = sigmoid(logit), or with score="softmax" the softmax over all
    experts (no bias).  Differentiable in logits through rw."""
    _rows(logits, "route: logits")
    T, E = logits.shape
    if score not in _SCORES or dtype not in _TYPE:
        raise NestQuantError(f"route: score {score!r} (sigmoid, softmax), weights of {dtype}")
    if not 1 <= topk <= min(E, 32) or E > 1024:
        raise NestQuantError(f"route: {topk} picks of {E} experts (to 32 of 1024)")
    if bias is not None:
        if score != "sigmoid":
            raise NestQuantError("route: a bias goes with sigmoid scores")
        if not (isinstance(bias, torch.Tensor) and bias.is_cuda and bias.dtype == torch.float32 and bias.shape == (E,) and bias.is_contiguous()):
            raise NestQuantError(f"route: bias, expected a contiguous CUDA tensor of torch.float32 [{E}]")
        if bias.requires_grad and torch.is_grad_enabled():
            raise NestQuantError("route: the bias has no gradient (detach it)")
        _same_device(logits, bias, "route")
    logits = _strided(logits)
    if logits.requires_grad and torch.is_grad_enabled():
        return _Route.apply(logits, bias, topk, _SCORES[score], bool(renorm), float(scale), dtype)
    return _route(logits, bias, topk, _SCORES[score], bool(renorm), float(scale), dtype)


def _route(logits, bias, topk, score, renorm, scale, dtype):
    T, E = logits.shape
    sel = torch.empty(T, topk, dtype=torch.int64, device=logits.device)
    rw = torch.empty(T, topk, dtype=dtype, device=logits.device)
    launch("route", lib().nq_route, logits, logits.data_ptr(), _TYPE[logits.dtype], _stride(logits), None if bias is None else bias.data_ptr(), T, E, topk,
           score, renorm, scale, sel.data_ptr(), rw.data_ptr(), _TYPE[dtype])
    return sel, rw


class _Route(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, bias, topk, score, renorm, scale, dtype):
        sel, rw = _route(logits, bias, topk, score, renorm, scale, dtype)
        ctx.save_for_backward(logits, sel)
        ctx.how = topk, score, renorm, scale
        ctx.mark_non_differentiable(sel)
        ctx.set_materialize_grads(False)             # (zeros for sel would be a launch)
        return sel, rw

    @staticmethod
    def backward(ctx, _, drw):
        _once(drw)
        if drw is None:
            return (None,) * 7
        logits, sel = ctx.saved_tensors
        topk, score, renorm, scale = ctx.how
        drw = drw.contiguous()
        T, E = logits.shape
        grad = torch.empty(T, E, dtype=logits.dtype, device=logits.device)
        launch("route backward", lib().nq_route_bwd, logits, logits.data_ptr(), _TYPE[logits.dtype], _stride(logits), sel.data_ptr(), drw.data_ptr(),
               _TYPE[drw.dtype], T, E, topk, score, renorm, scale, grad.data_ptr())
        return grad, None, None, None, None, None, None


# ---- rows by expert and back ----------------------------------------------------------------------------------------------------

class Order:
    """The picks of a call sorted by expert (sort_picks).  int32 tensors on the device: start [E+1], first place of each expert's picks (start[E]:
    where the picks without an expert begin); pos [T,topk], place of each pick; expert [P] (E: none) and token [P] of each place, P = T * topk."""

    def __init__(s, T, topk, E, buf):
        s.T, s.topk, s.E, s.P = T, topk, E, T * topk
        s._buf, s._ptr = buf, buf.data_ptr()         # start [E + 2], then pos, expert, token [P] each

    def _part(s, i):
        at = s.E + 2 + i * s.P
        return s._buf[at:at + s.P]

    start = property(lambda s: s._buf[:s.E + 1])
    pos = property(lambda s: s._part(0).view(s.T, s.topk))
    expert = property(lambda s: s._part(1))
    token = property(lambda s: s._part(2))
    # addresses for the calls below
    _live = property(lambda s: s._ptr + 4 * s.E)
    _pos = property(lambda s: s._ptr + 4 * (s.E + 2))


def sort_picks(sel, E):
    """Expert ids int64 [T,topk] -> their Order: a stable sort by expert, picks whose id is outside [0, E) behind all others.  E <= 1024."""
    _rows(sel, "sort_picks: sel", (torch.int64,))
    T, topk = sel.shape
    P = T * topk
    if not 1 <= E <= 1024 or topk < 1 or 3 * P + E + 2 > 0x7fffffff:
        raise NestQuantError(f"sort_picks: {T} x {topk} picks of {E} experts (to 1024)")
    sel = sel.contiguous()
    ints = int(lib().nq_pf_sort_scratch_ints(P, E))
    buf = torch.empty(E + 2 + 3 * P + max(ints, 1), dtype=torch.int32, device=sel.device)       # (the scratch behind the arrays)
    o = Order(T, topk, E, buf)
    at = lambda i: o._pos + 4 * i * P
    launch("sort_picks", lib().nq_sort_picks, sel, sel.data_ptr(), T, topk, E, at(1), at(2), at(0), o._ptr, at(3), max(ints, 1))
    return o


def dispatch(x, order):
    """Rows [T,H] (fp32, fp16, bf16) -> [T*topk,H]: each token's row at the places of its picks, rows sorted by expert (order.start); zeros
    at the places of picks without an expert.  Differentiable in x: the gradient adds up the token's rows, in pick order and 32 bits; what comes in for
    picks without an expert is not read."""
    _rows(x, "dispatch: x")
    if x.shape[0] != order.T or x.shape[1] < 1:
        raise NestQuantError(f"dispatch: x {tuple(x.shape)}, an order of {order.T} tokens")
    _same_device(x, order._buf, "dispatch")
    x = _strided(x)
    if x.requires_grad and torch.is_grad_enabled():
        return _Dispatch.apply(x, order)
    return _dispatch(x, order)


def _dispatch(x, order):
    H = x.shape[1]
    xs = torch.empty(order.P, H, dtype=x.dtype, device=x.device)
    launch("dispatch", lib().nq_dispatch, x, x.data_ptr(), _TYPE[x.dtype], _stride(x), order._pos, order._live, order.T, order.topk, H, xs.data_ptr())
    return xs


class _Dispatch(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, order):
        ctx.order = order
        return _dispatch(x, order)

    @staticmethod
    def backward(ctx, dxs):
        _once(dxs)
        o = ctx.order
        dxs = dxs.contiguous()
        H = dxs.shape[1]
        dx = torch.empty(o.T, H, dtype=dxs.dtype, device=dxs.device)
        launch("dispatch backward", lib().nq_dispatch_bwd, dxs, dxs.data_ptr(), _TYPE[dxs.dtype], o._pos, o._live, o.T, o.topk, H, dx.data_ptr())
        return dx, None


def combine(y, order, rw, dtype=None):
    """The picks' rows y [T*topk,H], in the order's places, and weights rw [T,topk] -> [T,H]: sums over each token's picks of rw * y, in pick order
    and 32 bits, as `dtype` (y's own, or fp32).  Rows of picks without an expert are not read; a token with none gets zeros.  Differentiable
    in y and rw (both 0 for picks without an expert)."""
    _rows(y, "combine: y"); _rows(rw, "combine: rw")
    dtype = dtype or y.dtype
    if y.shape[0] != order.P or y.shape[1] < 1 or rw.shape != (order.T, order.topk):
        raise NestQuantError(f"combine: y {tuple(y.shape)}, rw {tuple(rw.shape)}, an order of {order.T} x {order.topk} picks")
    if dtype not in (y.dtype, torch.float32):
        raise NestQuantError(f"combine: {y.dtype} rows as {dtype} (their own type, or fp32)")
    _same_device(y, order._buf, "combine"); _same_device(y, rw, "combine")
    y, rw = y.contiguous(), rw.contiguous()
    if (y.requires_grad or rw.requires_grad) and torch.is_grad_enabled():
        return _Combine.apply(y, rw, order, dtype)
    return _combine(y, rw, order, dtype)


def _combine(y, rw, order, dtype):
    H = y.shape[1]
    out = torch.empty(order.T, H, dtype=dtype, device=y.device)
    launch("combine", lib().nq_combine, y, y.data_ptr(), _TYPE[y.dtype], rw.data_ptr(), _TYPE[rw.dtype], order._pos, order._live, order.T, order.topk, H,
           out.data_ptr(), _TYPE[dtype])
    return out


class _Combine(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y, rw, order, dtype):
        ctx.save_for_backward(y, rw)
        ctx.order = order
        return _combine(y, rw, order, dtype)

    @staticmethod
    def backward(ctx, dout):
        _once(dout)
        y, rw = ctx.saved_tensors
        o, dout = ctx.order, dout.contiguous()
        dy = torch.empty_like(y) if ctx.needs_input_grad[0] else None
        drw = torch.empty_like(rw) if ctx.needs_input_grad[1] else None
        launch("combine backward", lib().nq_combine_bwd, y, dout.data_ptr(), _TYPE[dout.dtype], y.data_ptr(), _TYPE[y.dtype], rw.data_ptr(), _TYPE[rw.dtype],
               o._pos, o._live, o.T, o.topk, y.shape[1], None if dy is None else dy.data_ptr(), None if drw is None else drw.data_ptr())
        return dy, drw, None, None
