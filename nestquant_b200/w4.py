"""Products with plain 4-bit weights: the matrices of a layer that are not trellis planes (a shared expert, projections), or experts that a checkpoint
has in 4 bits with a scale, and perhaps a zero point, per row and group of columns.

    up = w4.W4(q, scales, zeros)              # once, when the weights are loaded
    y = up(x)                                 # x [T,K] -> [T,N]
    ys = experts(xs, start=order.start)       # one matrix per expert, rows sorted by expert (routing.dispatch)
"""
from .capi import torch_ops

_ops = torch_ops()


class W4:
    """Matrices N x K of weights (q - zero) * scale, q in 0 .. 15, laid out for the kernel (the arguments are not kept).

    q       uint8 [N,K/2], or [E,N,K/2] for one matrix per expert: two columns a byte, the even one in the low half
    scales  fp16 or bf16 [..,N,K/group], group 32, 64 or 128
    zeros   uint8 [..,N,K/group], 0 .. 15 (the low four bits count); None: 8 everywhere

    A call takes x [T,K] (fp16 or bf16) to W x as `dtype` (x's own, or fp32), every product and sum in 32 bits: the only rounding is the result's.
    With one matrix per expert, `start` (int32 [E+1] on the device, as Order.start) says whose rows are whose, start[0] = 0; rows from start[E] on give
    zeros.  Enqueued on the current stream of x's device, no host sync, bitwise repeatable.  There is no gradient: the weights are frozen, and an x that
    needs one, or has a tangent, is refused."""

    def __init__(s, q, scales, zeros=None):
        s._planes = p = _ops.w4_planes(q, scales, zeros)
        s.E, s.N, s.K, s.group, s.experts = p.E, p.N, p.K, p.group, p.E if p.experts else None

    def __call__(s, x, start=None, dtype=None):
        return _ops.w4_matmul(s._planes, x, start, dtype)

    def status(s):
        """0; 1 if a device-side wait of a call has run out (its results are then invalid); 2 if a call was given a start that falls (its rows
        are then zeros).  Synchronises."""
        return int(s._planes.status.item())

    def nbytes(s):
        """bytes of the planes on the device"""
        return sum(t.numel() * t.element_size() for t in (s._planes.qw, s._planes.sc, s._planes.zp) if t is not None)
