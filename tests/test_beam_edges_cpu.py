"""Refusals of the beam and page-pool entry points at their edges, without a GPU."""
import ctypes as C

from adi_amd import hip
from test_beam_cpu import batch, fork, pool, refused


def test_a_fork_of_no_rows_checks_what_it_reads():
    lib = hip.load()
    check = lambda **change: lib.adi_hip_paged_fork_check(  # noqa: E731
        C.byref(pool()), C.byref(batch(sequences=0)), C.byref(fork(parents=None, lengths=None, table=None, **change)))
    assert check() == hip.OK and check(references=None) == hip.OK
    refused(check(references=2), "unaligned")
