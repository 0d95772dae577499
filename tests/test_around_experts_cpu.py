"""Calls around the routed experts that their C entry points have to refuse by sizes and addresses alone, before any launch (without a device a call that goes
on ends with NQ_ERR_CUDA)."""
import ctypes as C

import pytest
import torch

from nestquant_b200 import capi

P = 4096        # stands for an address
no_device = pytest.mark.skipif(torch.cuda.is_available(), reason="the arguments are not device addresses")


def refused(rc):
    return rc == capi.NQ_ERR_ARG and capi.lib().nq_last_error()


@no_device
@pytest.mark.parametrize("T,topk,E", [(150_000_000, 4, 1024), ((2 ** 31 - 1) // 8, 8, 1024), (70_000_000, 8, 1000), (2 ** 31 - 1, 1, 255)])
def test_a_sort_whose_counts_no_array_can_hold_is_refused(T, topk, E):
    """a count per slice of 256 picks and bin, 2^31 - 1 at most: there is no size to ask for, so no array is large enough"""
    L = capi.lib()
    assert -(-T * topk // 256) * (E + 1) > 2 ** 31 - 1 and L.nq_pf_sort_scratch_ints(T * topk, E) == 0
    for ints in (0, 1, 2 ** 31 - 1):
        assert refused(L.nq_sort_picks(P, T, topk, E, None, None, P, P, P, ints, None))
        assert refused(L.nq_pf_sort(P, P, P, T, topk, E, P, P, P, P, None, P, ints, None))
        a = capi.NqPrefill()
        for n, t in a._fields_:
            setattr(a, n, P if t is C.c_void_p else 0)
        a.peer_x = a.hits = a.hit_counts = None
        a.T, a.topk, a.E, a.H, a.I, a.R, a.nm_gu, a.nm_dn = T, topk, E, 256, 128, 256, 2, 1
        a.plan_ints, a.sort_scratch_ints = 1 << 20, ints
        assert refused(L.nq_prefill(C.byref(a), None))


@no_device
def test_a_sort_of_more_picks_than_its_slices_can_count_is_refused():
    L = capi.lib()
    for T in (2 ** 31 - 1, 2 ** 31 - 255):
        assert refused(L.nq_sort_picks(P, T, 1, 1, None, None, P, P, P, 2 ** 31 - 1, None))


@no_device
@pytest.mark.parametrize("group,needs", [(32, 8), (64, 4), (128, 4)])
def test_zero_points_off_their_copies_alignment_are_refused(group, needs):
    """the products copy zero points 8 (groups of 32) or 4 bytes at a time; what suffices goes on to the device that is not there"""
    L = capi.lib()
    for zp in range(P, P + 17):
        fits = zp % needs == 0
        rc = (L.nq_w4_layout(P, P, P, 2, 64, 256, group, P, P, zp, None),
              L.nq_w4_matmul(P, capi.NQ_F16, 256, P, P, capi.NQ_F16, zp, P, 4, 2, 64, 256, group, P, capi.NQ_F32, 64, P, None),
              L.nq_w4_matmul(P, capi.NQ_F16, 256, P, P, capi.NQ_F16, zp, None, 40, 1, 64, 256, group, P, capi.NQ_F32, 64, P, None))
        assert all(r == (capi.NQ_ERR_CUDA if fits else capi.NQ_ERR_ARG) for r in rc), (zp, rc)


ENTRIES = {      # entry point: its arguments, and the element size of each pointer among them
    "nq_route": (dict(logits=P, type=capi.NQ_F32, row_stride=16, bias=P, T=4, E=16, topk=2, score=0, renorm=1, scale=1.0, sel=P, rw=P, rw_type=capi.NQ_F16, stream=None),
                 dict(logits=4, bias=4, sel=8, rw=2)),
    "nq_route_bwd": (dict(logits=P, type=capi.NQ_BF16, row_stride=16, sel=P, drw=P, rw_type=capi.NQ_F32, T=4, E=16, topk=2, score=0, renorm=1, scale=1.0, dlogits=P, stream=None),
                     dict(logits=2, sel=8, drw=4, dlogits=2)),
    "nq_sort_picks": (dict(sel=P, T=4, topk=2, E=16, pe=P, pt=P, pos=P, start=P, scratch=P, ints=1 << 20, stream=None), dict(sel=8, pe=4, pt=4, pos=4, start=4, scratch=4)),
    "nq_dispatch": (dict(x=P, type=capi.NQ_F32, row_stride=64, pos=P, live=P, T=4, topk=2, H=64, xs=P, stream=None), dict(x=4, pos=4, live=4, xs=4)),
    "nq_dispatch_bwd": (dict(dxs=P, type=capi.NQ_F16, pos=P, live=P, T=4, topk=2, H=64, dx=P, stream=None), dict(dxs=2, pos=4, live=4, dx=2)),
    "nq_combine": (dict(y=P, type=capi.NQ_F16, rw=P, rw_type=capi.NQ_F32, pos=P, live=P, T=4, topk=2, H=64, out=P, out_type=capi.NQ_F32, stream=None),
                   dict(y=2, rw=4, pos=4, live=4, out=4)),
    "nq_combine_bwd": (dict(dout=P, out_type=capi.NQ_F32, y=P, type=capi.NQ_F16, rw=P, rw_type=capi.NQ_F16, pos=P, live=P, T=4, topk=2, H=64, dy=P, drw=P, stream=None),
                       dict(dout=4, y=2, rw=2, pos=4, live=4, dy=2, drw=2)),
    "nq_w4_layout": (dict(q=P, scales=P, zeros=P, E=2, N=64, K=256, group=64, qw=P, sc=P, zp=P, stream=None), dict(q=2, scales=2)),
    "nq_w4_matmul": (dict(x=P, type=capi.NQ_F16, x_stride=256, qw=P, sc=P, sc_type=capi.NQ_F16, zp=P, start=P, rows=4, E=2, N=64, K=256, group=64, out=P, out_type=capi.NQ_F32,
                          out_stride=64, status=P, stream=None), dict(start=4, out=4, status=4)),
}


@no_device
@pytest.mark.parametrize("name,pointer,size", [(n, p, s) for n, (_, sizes) in ENTRIES.items() for p, s in sizes.items()])
def test_addresses_off_their_elements_are_refused(name, pointer, size):
    """a kernel would fault on them; whole elements further on the call goes on to the device that is not there"""
    entry, base = getattr(capi.lib(), name), ENTRIES[name][0]
    for off in range(1, 2 * size + 1):
        rc = entry(*dict(base, **{pointer: P + off}).values())
        assert rc == (capi.NQ_ERR_ARG if off % size else capi.NQ_ERR_CUDA), off
