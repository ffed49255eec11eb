"""Arguments of the 4-bit cache and the eviction that would make workgroups race or read outside a tensor, on the CPU: they
are turned away before a kernel is launched."""
import ctypes as C

import pytest

from glake_amd import _C
from test_small_cache_refusals import P, evict, refused, weigh

N = C.c_void_p(0)


def evict_strides(slot, head, **kw):
    a = dict(ns=4, hk=2, m=64)
    a.update(kw)
    return _C.lib().vtkv_evict_rows(P, P, P, slot, head, a["ns"], P, P, P, 0, a["hk"], 128, _C.BF16, 10, 5, a["m"], P, 1 << 20, N)


@pytest.mark.parametrize("slot,head", [(0, 64), (128, 0), (0, 0), (127, 64), (128, 63), (64, 64), (-128, 64), (63, 1 << 20)])
def test_overlapping_weights_are_refused(slot, head):
    refused(weigh(ss=slot, hs=head, b=0), "overlap")
    refused(evict_strides(slot, head), "overlap")


@pytest.mark.parametrize("kw,slot,head", [({}, 128, 64), ({}, 64, 256), ({}, 1 << 40, 1 << 30), (dict(ns=1), 0, 64), (dict(hk=1), 64, 0),
                                          (dict(ns=1, hk=1), 0, 0)])
def test_weights_in_any_order_that_keeps_them_apart(kw, slot, head):
    assert weigh(ss=slot, hs=head, b=0, **kw) == 0
    assert evict_strides(slot, head, **kw) == 0


def test_lengths_that_overlap_in_part_are_refused():
    at = lambda n: C.c_void_p(4096 + n)  # noqa: E731
    for n in (4, 12, -4, -12):
        refused(evict(sl=P, nl=at(n), b=4), "apart")
    # (apart or the same: refused only for the workspace that is missing here)
    for n in (0, 16, -16):
        assert evict(sl=P, nl=at(n), b=4, ws=N) == _C.ENOMEM
