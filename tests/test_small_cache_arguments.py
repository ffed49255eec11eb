"""Arguments of the 4-bit cache and the eviction that would make workgroups race or read outside a tensor, on the CPU: they
are turned away before a kernel is launched."""
import ctypes as C

import pytest
import torch

from glake_amd import _C, _custom_ops as ops
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


def rows(tokens=4, values=4, batch=4, lens=4, starts=4, most=3, offsets=None):
    key, value = torch.zeros(tokens, 2, 64), torch.zeros(values, 2, 64)
    i64, i32 = torch.zeros(batch, dtype=torch.int64), torch.zeros(16, dtype=torch.int32)
    return ops._int4_rows(key, value, i64 if offsets is None else torch.zeros(offsets, dtype=torch.int64), i64,
                          None if lens is None else i32[:lens], None if starts is None else i32[:starts], most, 2, 64)


@pytest.mark.parametrize("kw", [dict(lens=3), dict(starts=3), dict(lens=None), dict(starts=None), dict(values=3), dict(tokens=3),
                                dict(offsets=3), dict(most=1, tokens=3, values=3)])
def test_rows_without_an_entry_for_every_sequence_are_refused(kw):
    with pytest.raises(_C.VtkvError):
        rows(**kw)


@pytest.mark.parametrize("kw", [{}, dict(lens=9, starts=5), dict(tokens=100, values=100), dict(most=1, lens=None, starts=None),
                                dict(most=1, tokens=6, values=6, lens=1), dict(batch=0, lens=0, starts=0), dict(tokens=2, values=2)])
def test_rows_with_an_entry_for_every_sequence(kw):
    key, value = rows(**kw)
    assert key.shape[1:] == value.shape[1:] == (2, 64)


def test_more_units_than_a_launch_can_number():
    from test_small_cache_refusals import decode

    refused(decode(h=17, hk=17, qs=17 * 128, m=0x7fffffff), "max_seq_len")
    assert decode(h=17, hk=17, qs=17 * 128, m=1 << 30) == _C.ENOMEM  # (only the workspace is missing)


def test_more_rows_than_the_weights_can_number():
    one = dict(h=1, hk=1, ss=1 << 40, hs=1 << 40, ns=1)
    refused(weigh(m=0x7fffffff, b=0, **one), "max_seq_len")
    assert weigh(m=1 << 30, b=0, **one) == 0
