"""What the calls around the routed experts refuse before anything is enqueued.  The C entry points check sizes, types and pointers without looking at
the device, the Python ones refuse tensors that are not there."""
import ctypes as C

import pytest
import torch

from nestquant_b200 import capi
from nestquant_b200.capi import NQ_BF16, NQ_F16, NQ_F32, NestQuantError

P = 4096        # stands for an address
ARG = -1


def _with(call, base, **over):
    a = dict(base, **over)
    return call(*a.values())


ROUTE = dict(logits=P, type=NQ_F32, row_stride=16, bias=P, T=4, E=16, topk=2, score=0, renorm=1, scale=1.0, sel=P, rw=P, rw_type=NQ_F16, stream=None)
ROUTE_BWD = dict(logits=P, type=NQ_F32, row_stride=16, sel=P, drw=P, rw_type=NQ_F16, T=4, E=16, topk=2, score=0, renorm=1, scale=1.0, dlogits=P, stream=None)
SORT = dict(sel=P, T=4, topk=2, E=16, pe=P, pt=P, pos=P, start=P, scratch=P, ints=1 << 20, stream=None)
DISPATCH = dict(x=P, type=NQ_F16, row_stride=64, pos=P, live=P, T=4, topk=2, H=64, xs=P, stream=None)
DISPATCH_BWD = dict(dxs=P, type=NQ_F16, pos=P, live=P, T=4, topk=2, H=64, dx=P, stream=None)
COMBINE = dict(y=P, type=NQ_F16, rw=P, rw_type=NQ_F32, pos=P, live=P, T=4, topk=2, H=64, out=P, out_type=NQ_F32, stream=None)
COMBINE_BWD = dict(dout=P, out_type=NQ_F16, y=P, type=NQ_F16, rw=P, rw_type=NQ_F32, pos=P, live=P, T=4, topk=2, H=64, dy=P, drw=P, stream=None)
LAYOUT = dict(q=P, scales=P, zeros=P, E=2, N=64, K=256, group=64, qw=P, sc=P, zp=P, stream=None)
MATMUL = dict(x=P, type=NQ_F16, x_stride=256, qw=P, sc=P, sc_type=NQ_F16, zp=P, start=P, rows=4, E=2, N=64, K=256, group=64, out=P, out_type=NQ_F32, out_stride=64, status=P, stream=None)


@pytest.mark.skipif(torch.cuda.is_available(), reason="the arguments are not device addresses")
@pytest.mark.parametrize("name,base,over", [(n, b, o) for n, b, overs in [
    ("nq_route", ROUTE, [dict(type=3), dict(rw_type=-1), dict(T=-1), dict(E=0), dict(E=1025, row_stride=1025), dict(topk=0), dict(topk=17), dict(E=64, row_stride=64, topk=33),
                         dict(row_stride=15), dict(score=2), dict(score=1), dict(logits=None), dict(sel=None), dict(rw=None)]),
    ("nq_route_bwd", ROUTE_BWD, [dict(type=3), dict(T=-1), dict(topk=17), dict(row_stride=15), dict(score=-1), dict(logits=None), dict(sel=None), dict(drw=None), dict(dlogits=None)]),
    ("nq_sort_picks", SORT, [dict(T=-1), dict(topk=0), dict(E=0), dict(E=1025), dict(T=1 << 30, topk=4), dict(sel=None), dict(pos=None), dict(start=None), dict(scratch=None), dict(ints=0)]),
    ("nq_dispatch", DISPATCH, [dict(type=5), dict(T=-1), dict(topk=0), dict(H=0), dict(row_stride=63), dict(T=1 << 30, topk=2), dict(x=None), dict(pos=None), dict(live=None), dict(xs=None),
                               dict(x=P + 1)]),
    ("nq_dispatch_bwd", DISPATCH_BWD, [dict(type=5), dict(T=-1), dict(topk=0), dict(H=0), dict(dxs=None), dict(pos=None), dict(live=None), dict(dx=None)]),
    ("nq_combine", COMBINE, [dict(type=7), dict(rw_type=9), dict(out_type=NQ_BF16), dict(T=-1), dict(topk=0), dict(H=0), dict(y=None), dict(rw=None), dict(out=None)]),
    ("nq_combine_bwd", COMBINE_BWD, [dict(type=7), dict(rw_type=9), dict(out_type=NQ_BF16), dict(T=-1), dict(H=0), dict(dout=None), dict(y=None), dict(rw=None), dict(pos=None)]),
    ("nq_w4_layout", LAYOUT, [dict(group=16), dict(group=256), dict(K=96, group=64), dict(K=0), dict(N=0), dict(E=0), dict(q=None), dict(zp=None), dict(zeros=None), dict(qw=P + 8), dict(q=P + 1)]),
    ("nq_w4_matmul", MATMUL, [dict(type=NQ_F32), dict(sc_type=NQ_F32), dict(out_type=NQ_BF16), dict(group=48), dict(K=320, group=128), dict(rows=-1), dict(start=None), dict(x_stride=255),
                              dict(x_stride=260), dict(out_stride=63), dict(x=P + 8), dict(x=None), dict(qw=None), dict(sc=None), dict(out=None), dict(status=None), dict(E=0), dict(E=1025)]),
] for o in overs], ids=lambda v: v if isinstance(v, str) else ",".join(f"{a}={b}" for a, b in v.items()) if len(v) < 4 else "")
def test_c_entry_points_refuse(name, base, over):
    assert _with(getattr(capi.lib(), name), base, **over) == ARG
    assert capi.lib().nq_last_error()


def test_nothing_to_do_is_done():
    """no tokens, no rows: no pointer is needed"""
    L = capi.lib()
    assert _with(L.nq_route, ROUTE, T=0, logits=None, sel=None, rw=None) == 0
    assert _with(L.nq_route_bwd, ROUTE_BWD, T=0, logits=None) == 0
    assert _with(L.nq_dispatch, DISPATCH, T=0, x=None, xs=None) == 0 and _with(L.nq_dispatch_bwd, DISPATCH_BWD, T=0, dxs=None) == 0
    assert _with(L.nq_combine, COMBINE, T=0, y=None) == 0 and _with(L.nq_combine_bwd, COMBINE_BWD, T=0, dout=None) == 0
    assert _with(L.nq_combine_bwd, COMBINE_BWD, dy=None, drw=None, dout=None) == 0
    assert _with(L.nq_w4_matmul, MATMUL, rows=0, x=None, out=None) == 0


def test_units():
    n = C.c_int64()
    for E, N, K, want in ((1, 16, 128, 1), (1, 17, 129, 4), (3, 4096, 6144, 3 * 256 * 48), (1, 1, 32, 1), (200, 12288, 12288, 200 * 768 * 96)):
        assert capi.lib().nq_w4_units(E, N, K, C.byref(n)) == (0 if K % 32 == 0 else ARG)
        if K % 32 == 0:
            assert n.value == want
    assert capi.lib().nq_w4_units(1, 16, 128, None) == ARG


def test_python_entry_points_refuse_host_tensors():
    from nestquant_b200 import routing, w4
    for call in (lambda: routing.route(torch.zeros(4, 16), 2), lambda: routing.sort_picks(torch.zeros(4, 2, dtype=torch.int64), 16),
                 lambda: w4.W4(torch.zeros(16, 64, dtype=torch.uint8), torch.zeros(16, 1, dtype=torch.float16))):
        with pytest.raises(NestQuantError):
            call()
