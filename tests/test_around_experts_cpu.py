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
