"""Refusals of the beam and page-pool entry points at their edges, without a GPU."""
import ctypes as C
import types

import pytest
import torch

from adi_amd import hip
from test_beam_cpu import batch, fork, pool, refused


def test_a_fork_of_no_rows_checks_what_it_reads():
    lib = hip.load()
    check = lambda **change: lib.adi_hip_paged_fork_check(  # noqa: E731
        C.byref(pool()), C.byref(batch(sequences=0)), C.byref(fork(parents=None, lengths=None, table=None, **change)))
    assert check() == hip.OK and check(references=None) == hip.OK
    refused(check(references=2), "unaligned")


@pytest.mark.parametrize("shape", [(2, 3, 0), (2, 3, 4, 0), (2, 3, 0, 4), (2, 0, 5), (0, 3, 2, 4)])
def test_state_rows_of_nothing(shape):
    """Tensors without elements are rows of no bytes, or no rows."""
    ctx = types.SimpleNamespace(device=-1)
    rows = hip.StateRows(ctx, [torch.empty(shape)])
    assert (rows.requests, rows.beams) == shape[:2]
    size = 4
    for n in shape[2:]:
        size *= n
    assert rows.struct[0].row_bytes == size
    with pytest.raises(hip.HipError, match="contiguous"):
        hip.StateRows(ctx, [torch.empty(2, 3, 4, 4).transpose(2, 3)])


@pytest.mark.parametrize("array,requests,ok", [
    ((1 << 20, 1 << 45, (1 << 45) + 100, 100), (1 << 19) + 1, False),  # 2^19 strides of 2^45 are 2^64
    ((1 << 20, 1 << 45, (1 << 46) - 1, 100), (1 << 19) + 2, False),
    ((1 << 20, 1 << 45, 1 << 20, 100), (1 << 19) + 1, True),           # requests outermost
    ((1 << 20, 100, 100 << 10, 100), 1 << 10, True),
    ((1 << 20, 100, (100 << 10) - 1, 100), 1 << 10, False),
    ((1 << 20, 101, 101 * 1023 + 100, 100), 1 << 10, True),
    ((1 << 20, 101, 101 * 1023 + 99, 100), 1 << 10, False),
    ((1 << 20, 100, 99, 100), 2, False)])
def test_rows_of_requests_that_overlap(array, requests, ok):
    """Beams outermost: all requests' rows between two of a request's."""
    rows = (hip.RowArray * 1)(hip.RowArray(*array))
    status = hip.load().adi_hip_reorder_check(rows, 1, requests, 2, 1 << 30)
    if ok:
        assert status == hip.OK
    else:
        refused(status, "overlap")


class Untouched:
    """A library of which nothing may be called."""

    def __getattr__(self, name):
        raise AssertionError(f"{name} was called")


def meta(*shape, dtype=torch.int32):
    return torch.empty(shape, dtype=dtype, device="meta")


HUGE = (1 << 32) + 1  # 1 in 32 bits


def test_sizes_past_32_bits_are_refused():
    """None is cut to 32 bits on its way into the library, and none ends in another
    error than a refusal's."""
    ctx = types.SimpleNamespace(device=-1, lib=Untouched(), handle=None)
    space = types.SimpleNamespace(handle=None)
    held = types.SimpleNamespace(pages=4, references=meta(4), struct=None)
    calls = [
        lambda: hip.StateRows(ctx, [meta(HUGE, 2, 3)]),
        lambda: hip.StateRows(ctx, [meta(1, HUGE, 3)]),
        lambda: hip.paged_copy(ctx, held, held, meta(HUGE), meta(HUGE)),
        lambda: hip.beam_select(ctx, meta(1, 1, HUGE, dtype=torch.float16), meta(1, 1, dtype=torch.float32),
                                meta(1, 1, dtype=torch.float32), meta(1, 1), meta(1, 1), space),
        lambda: hip.beam_select(ctx, meta(HUGE, 1, 5, dtype=torch.float16), meta(HUGE, 1, dtype=torch.float32),
                                meta(HUGE, 1, dtype=torch.float32), meta(HUGE, 1), meta(HUGE, 1), space),
        lambda: hip.paged_fork(ctx, held, types.SimpleNamespace(lengths=meta(1), table=meta(1, HUGE), struct=None),
                               meta(1, 1), space),
        lambda: hip.paged_fork(ctx, held, types.SimpleNamespace(lengths=meta(HUGE), table=meta(HUGE, 1), struct=None),
                               meta(1, HUGE), space),
        lambda: hip.paged_compact(ctx, held, meta(HUGE), meta(HUGE, 1), meta(1), space),
        lambda: hip.paged_compact(ctx, held, meta(1), meta(1, HUGE), meta(1), space)]
    for call in calls:
        with pytest.raises(hip.HipError):
            call()
