"""The router's choice, and tokens' rows sorted by expert and back: what stands around the experts of a layer, with the gradients that a router
needs when it is trained.

    sel, rw = routing.route(logits, 8, bias=bias, scale=2.5)      # ids and weights as MoELayer takes them
    order = routing.sort_picks(sel, E)                            # for experts that are not this library's planes:
    xs = routing.dispatch(x, order)                               #   rows sorted by expert, order.start = where each expert's begin
    out = routing.combine(experts(xs, order.start), order, rw)    #   weighted sums of the picks' rows

Everything is enqueued on the current stream of the tensors' device without a host sync, can be captured in a CUDA graph, and gives the same
bits every time.  route, dispatch and combine are differentiable (once, in backward mode; dual tensors are refused) in logits, x, y and rw; a call whose tensors
need no gradient does not enter autograd.  To capture a backward pass, use torch.autograd.grad, or leaves that no eager graph still holds: the engine joins the stream
on which a leaf's gradient was first accumulated, which a capture forbids.  Errors are NestQuantError, raised before anything is enqueued.
"""
import torch

from .capi import torch_ops

_ops = torch_ops()
Order = _ops.Order


def route(logits, topk, score="sigmoid", bias=None, renorm=True, scale=1.0, dtype=torch.float16):
    """Router logits [T,E] (fp32, fp16 or bf16; E <= 1024) -> (sel int64 [T,topk], rw [T,topk] of `dtype`), topk <= 32.

    Chosen are the topk experts with the largest sigmoid(logit) + bias (bias: fp32 [E], sees the choice only), without a bias those with the largest
    logits; ids in falling order of the score, equal scores by the lowest id.  The order is that of the exact scores, not of their
    roundings.  Experts whose logit or bias is -inf or NaN are never chosen; where fewer than topk are left, the last ids are -1 and
    their weights 0, picks that every call of this library skips.
    rw = scale * p, divided by the sum of the chosen p if renorm; p = sigmoid(logit), or with score="softmax" the softmax over all
    experts (no bias).  Differentiable in logits through rw."""
    return _ops.route(logits, topk, score, bias, renorm, scale, dtype)


def sort_picks(sel, E):
    """Expert ids int64 [T,topk] -> their Order: a stable sort by expert, picks whose id is outside [0, E) behind all others.  E <= 1024; somewhat
    fewer than 2^30 picks, with 1,024 experts half as many (E + 1 counts for every 256 picks stand in one array)."""
    return _ops.sort_picks(sel, E)


def dispatch(x, order):
    """Rows [T,H] (fp32, fp16, bf16) -> [T*topk,H]: each token's row at the places of its picks, rows sorted by expert (order.start); zeros
    at the places of picks without an expert.  Differentiable in x: the gradient adds up the token's rows, in pick order and 32 bits; what comes in for
    picks without an expert is not read."""
    return _ops.dispatch(x, order)


def combine(y, order, rw, dtype=None):
    """The picks' rows y [T*topk,H], in the order's places, and weights rw [T,topk] -> [T,H]: sums over each token's picks of rw * y, in pick order
    and 32 bits, as `dtype` (y's own, or fp32).  Rows of picks without an expert are not read; a token with none gets zeros.  Differentiable
    in y and rw (both 0 for picks without an expert)."""
    return _ops.combine(y, order, rw, dtype)
