"""Products with plain 4-bit weights: the matrices of a layer that are not trellis planes (a shared expert, projections), or experts that a checkpoint
has in 4 bits with a scale, and perhaps a zero point, per row and group of columns.

    up = w4.W4(q, scales, zeros)              # once, when the weights are loaded
    y = up(x)                                 # x [T,K] -> [T,N]
    ys = experts(xs, start=order.start)       # one matrix per expert, rows sorted by expert (routing.dispatch)
"""
import ctypes as C

import torch

from .capi import NestQuantError, check, element_types, launch, lib

_TYPE = element_types()
_HALVES = (torch.float16, torch.bfloat16)


def _device(t, dtypes, name):
    if not (isinstance(t, torch.Tensor) and t.is_cuda and t.dtype in dtypes):
        raise NestQuantError(f"W4: {name}: expected a CUDA tensor of {' / '.join(str(d) for d in dtypes)}")


class W4:
    """Matrices N x K of weights (q - zero) * scale, q in 0 .. 15, laid out for the kernel (the arguments are not kept).

    q       uint8 [N,K/2], or [E,N,K/2] for one matrix per expert: two columns a byte, the even one in the low half
    scales  fp16 or bf16 [..,N,K/group], group 32, 64 or 128
    zeros   uint8 [..,N,K/group], 0 .. 15 (the low four bits count); None: 8 everywhere

    A call takes x [T,K] (fp16 or bf16) to W x as `dtype` (x's own, or fp32), every product and sum in 32 bits: the only rounding is the result's.
    With one matrix per expert, `start` (int32 [E+1] on the device, as Order.start) says whose rows are whose, start[0] = 0; rows from start[E] on give
    zeros.  Enqueued on the current stream of x's device, no host sync, bitwise repeatable.  There is no gradient: the weights are frozen, and an x that
    needs one is refused."""

    def __init__(s, q, scales, zeros=None):
        _device(q, (torch.uint8,), "q")
        _device(scales, _HALVES, "scales")
        if q.dim() not in (2, 3) or scales.dim() != q.dim() or q.shape[:-1] != scales.shape[:-1] or q.numel() == 0 or scales.shape[-1] == 0:
            raise NestQuantError(f"W4: q {tuple(q.shape)}, scales {tuple(scales.shape)}: expected [..,N,K/2] and [..,N,K/group]")
        s.experts = q.shape[0] if q.dim() == 3 else None
        s.E, s.N, s.K = s.experts or 1, q.shape[-2], 2 * q.shape[-1]
        s.group = s.K // scales.shape[-1]
        if s.group not in (32, 64, 128) or s.group * scales.shape[-1] != s.K:
            raise NestQuantError(f"W4: {s.K} columns with {scales.shape[-1]} scales a row: groups are of 32, 64 or 128 columns")
        if zeros is not None:
            _device(zeros, (torch.uint8,), "zeros")
            if zeros.shape != scales.shape:
                raise NestQuantError(f"W4: zeros {tuple(zeros.shape)}, scales {tuple(scales.shape)}")
        if any(t.get_device() != q.get_device() for t in (scales, zeros) if t is not None):
            raise NestQuantError("W4: tensors on different devices")
        n = C.c_int64()
        check(lib().nq_w4_units(s.E, s.N, s.K, C.byref(n)), "W4")
        per = 16 * (128 // s.group)
        s.device = q.device
        s._qw = torch.empty(n.value * 1024, dtype=torch.uint8, device=q.device)
        s._sc = torch.empty(n.value * per, dtype=scales.dtype, device=q.device)
        s._zp = None if zeros is None else torch.empty(n.value * per, dtype=torch.uint8, device=q.device)
        q, scales, zeros = q.contiguous(), scales.contiguous(), None if zeros is None else zeros.contiguous()
        # addresses of the planes, for the calls
        s._status = torch.zeros(1, dtype=torch.int32, device=q.device)
        s._planes = s._qw.data_ptr(), s._sc.data_ptr(), _TYPE[scales.dtype], None if zeros is None else s._zp.data_ptr(), s._status.data_ptr()
        s._index = q.get_device()
        launch("W4", lib().nq_w4_layout, q, q.data_ptr(), scales.data_ptr(), None if zeros is None else zeros.data_ptr(), s.E, s.N, s.K, s.group,
               s._planes[0], s._planes[1], s._planes[3])

    def status(s):
        """0, or 1 if a device-side wait of a call has run out (its results are then invalid).  Synchronises."""
        return int(s._status.item())

    def nbytes(s):
        """bytes of the planes on the device"""
        return sum(t.numel() * t.element_size() for t in (s._qw, s._sc, s._zp) if t is not None)

    def __call__(s, x, start=None, dtype=None):
        if not (isinstance(x, torch.Tensor) and x.is_cuda and x.dim() == 2 and x.dtype in _HALVES):
            raise NestQuantError("W4: x, expected a CUDA tensor [T,K] of torch.float16 / torch.bfloat16")
        T, K = x.shape
        own = x.dtype
        dtype = dtype or own
        if K != s.K or dtype is not own and dtype is not torch.float32:
            raise NestQuantError(f"W4: x {tuple(x.shape)} of {own} as {dtype}, a matrix of {s.K} columns (result in x's own type, or fp32)")
        if x.get_device() != s._index:
            raise NestQuantError("W4: x and the weights are on different devices")
        if x.requires_grad and torch.is_grad_enabled():
            raise NestQuantError("W4: no gradient (detach x, or call under torch.no_grad)")
        if (s.experts is None) != (start is None):
            raise NestQuantError("W4: start goes with one matrix per expert, and only with that")
        if start is not None and not (isinstance(start, torch.Tensor) and start.is_cuda and start.dtype == torch.int32 and start.is_contiguous() and
                                      start.numel() > s.E and start.get_device() == s._index):
            raise NestQuantError(f"W4: start, expected a contiguous CUDA tensor of torch.int32 [{s.E + 1}]")
        rows, cols = x.stride()
        if T <= 1:
            rows = K
        if cols != 1 or rows < K or rows % 8 or x.data_ptr() % 16:
            x, rows = x.clone(memory_format=torch.contiguous_format), K      # rows that the kernel reads start on 16 bytes
        out = torch.empty((T, s.N), dtype=dtype, device=s.device)
        qw, sc, sc_type, zp, status = s._planes
        launch("W4", lib().nq_w4_matmul, x, x.data_ptr(), _TYPE[own], rows, qw, sc, sc_type, zp, None if start is None else start.data_ptr(), T, s.E, s.N, K,
               s.group, out.data_ptr(), _TYPE[dtype], s.N, status)
        return out
