"""The beam and page-pool entry points without a GPU: their structures against
the header, the packed arguments, and the refusals of every call."""
import ctypes as C
import os
import subprocess

import pytest

from adi_amd import hip

HEADER = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "adi_hip.h")

STRUCTS = {
    "adi_hip_beam_arguments": hip.BeamArguments,
    "adi_hip_row_array": hip.RowArray,
    "adi_hip_paged_pool": hip.PagedPoolStruct,
    "adi_hip_paged_fork_arguments": hip.PagedForkArguments,
    "adi_hip_paged_compact_arguments": hip.PagedCompactArguments,
}


def test_struct_layouts_match_header(tmp_path):
    lines = ["#include <stdio.h>", "#include <stddef.h>", '#include "adi_hip.h"', "int main(void) {"]
    for cname, ctype in STRUCTS.items():
        lines.append(f'printf("{cname} size %zu\\n", sizeof({cname}));')
        for field, _ in ctype._fields_:
            lines.append(f'printf("{cname} {field} %zu\\n", offsetof({cname}, {field}));')
    src = tmp_path / "layout.c"
    src.write_text("\n".join(lines + ["return 0;", "}"]))
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-std=c11", "-Wall", "-Werror", "-I", os.path.dirname(HEADER), str(src), "-o", str(exe)],
                   check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split("\n")
    want = {tuple(line.split()[:2]): int(line.split()[2]) for line in out if line}
    for cname, ctype in STRUCTS.items():
        assert want[(cname, "size")] == C.sizeof(ctype), cname
        for field, _ in ctype._fields_:
            assert want[(cname, field)] == getattr(ctype, field).offset, (cname, field)


def test_packed_arguments_are_the_structures():
    beam = list(range(1, 17))
    assert hip._pack_beam(*beam) == bytes(hip.BeamArguments(*beam))
    fork = list(range(21, 27))
    assert hip._pack_fork(*fork) == bytes(hip.PagedForkArguments(*fork))
    compact = list(range(31, 38))
    assert hip._pack_compact(*compact) == bytes(hip.PagedCompactArguments(*compact))


def refused(status, message):
    assert status == hip.INVALID_ARGUMENT
    assert message in hip.load().adi_hip_last_error(None).decode()


# ---- beam select -----------------------------------------------------------------

def beam(**change):
    held = dict(type=0, logits=1 << 20, request_stride=400, beam_stride=100, requests=2, beams=4, vocabulary=100,
                choices=8, scores=1 << 21, weights=None, ended=None, ended_token=0, settle=0, out_scores=1 << 22,
                parents=1 << 23, tokens=1 << 24)
    held.update(change)
    return hip.BeamArguments(**held)


@pytest.mark.parametrize("change", [
    {}, {"beams": 1}, {"beams": 64}, {"choices": 1}, {"choices": 128}, {"vocabulary": 1}, {"vocabulary": 1 << 24},
    {"requests": 1 << 20}, {"requests": 0, "logits": None, "scores": None}, {"type": 1, "logits": (1 << 20) + 2},
    {"settle": 1, "choices": 4}, {"weights": 1 << 25, "ended": 1 << 26}])
def test_beam_check_accepts(change):
    assert hip.load().adi_hip_beam_check(C.byref(beam(**change))) == hip.OK


@pytest.mark.parametrize("change,message", [
    ({"type": 3}, "unknown type"), ({"beams": 0}, "beams must be"), ({"beams": 65}, "beams must be"),
    ({"choices": 0}, "choices must be"), ({"choices": 129}, "choices must be"),
    ({"vocabulary": 0}, "vocabulary must be"), ({"vocabulary": (1 << 24) + 1}, "vocabulary must be"),
    ({"requests": (1 << 20) + 1}, "requests"), ({"settle": 2}, "settle must be"),
    ({"settle": 1}, "as many as beams"), ({"logits": None}, "null"), ({"scores": None}, "null"),
    ({"out_scores": None}, "null"), ({"parents": None}, "null"), ({"tokens": None}, "null"),
    ({"logits": (1 << 20) + 2}, "unaligned"), ({"type": 2, "logits": (1 << 20) + 1}, "unaligned"),
    ({"scores": (1 << 21) + 1}, "unaligned"), ({"weights": 2}, "unaligned"), ({"ended": 2}, "unaligned"),
    ({"tokens": 6}, "unaligned"), ({"parents": 6}, "unaligned"), ({"out_scores": 6}, "unaligned"),
    ({"out_scores": 1 << 21}, "overlap")])
def test_beam_refusals(change, message):
    refused(hip.load().adi_hip_beam_check(C.byref(beam(**change))), message)


def test_null_contexts_and_descriptors():
    lib = hip.load()
    refused(lib.adi_hip_beam_check(None), "null")
    refused(lib.adi_hip_paged_fork_check(None, None, None), "null")
    refused(lib.adi_hip_paged_copy_check(None, None, None, None, None, 0), "null")
    refused(lib.adi_hip_paged_compact_check(None, None), "null")
    assert lib.adi_hip_beam_select(None, None, None) == hip.INVALID_ARGUMENT
    assert lib.adi_hip_reorder_rows(None, None, 0, 0, 1, None) == hip.INVALID_ARGUMENT
    assert lib.adi_hip_paged_fork(None, None, None, None, None) == hip.INVALID_ARGUMENT
    assert lib.adi_hip_paged_copy(None, None, None, None, None, None, 0) == hip.INVALID_ARGUMENT
    assert lib.adi_hip_paged_compact(None, None, None, None) == hip.INVALID_ARGUMENT


# ---- reorder rows -----------------------------------------------------------------

@pytest.mark.parametrize("array,requests,beams,ok", [
    ((1 << 20, 400, 100, 100), 3, 4, True),
    ((1 << 20, 100, 300, 100), 3, 4, True),      # beams outermost
    ((1 << 20, 0, 100, 100), 1, 4, True),
    ((1 << 20, 7, 0, 7), 3, 1, True),
    ((None, 0, 0, 0), 3, 4, True),               # rows of no bytes
    ((1 << 20, 400, 99, 100), 3, 4, False),
    ((1 << 20, 399, 100, 100), 3, 4, False),
    ((1 << 20, 100, 299, 100), 3, 4, False),
    ((1 << 20, 0, 100, 100), 3, 4, False),       # one request's rows for all
    ((1 << 20, 100, 0, 100), 3, 4, False),
])
def test_reorder_arrays(array, requests, beams, ok):
    rows = (hip.RowArray * 1)(hip.RowArray(*array))
    status = hip.load().adi_hip_reorder_check(rows, 1, requests, beams, 1 << 30)
    if ok:
        assert status == hip.OK
    else:
        refused(status, "overlap")


def test_reorder_refusals():
    lib = hip.load()
    rows = (hip.RowArray * 1)(hip.RowArray(1 << 20, 400, 100, 100))
    for count, requests, beams, parents, message in [
            (1, 2, 0, 4, "beams must be"), (1, 2, 65, 4, "beams must be"), (1, (1 << 20) + 1, 4, 4, "requests"),
            ((1 << 16) + 1, 2, 4, 4, "arrays"), (1, 2, 4, None, "null"), (1, 2, 4, 2, "unaligned")]:
        refused(lib.adi_hip_reorder_check(rows, count, requests, beams, parents), message)
    refused(lib.adi_hip_reorder_check(None, 1, 2, 4, 4), "null")
    refused(lib.adi_hip_reorder_check((hip.RowArray * 1)(hip.RowArray(None, 400, 100, 100)), 1, 2, 4, 4), "null array")
    refused(lib.adi_hip_reorder_check((hip.RowArray * 1)(hip.RowArray(4, 0, 1 << 46, 1 << 36)), 1, 1, 4, 4), "2^36")
    # (a block moves 4 KB of 64 rows, 16 of four; all are checked before any is moved)
    small, large = hip.RowArray(4, 1 << 30, 1 << 20, 16), hip.RowArray(4, 1 << 30, 1 << 20, 1 << 16)
    both = (hip.RowArray * 2)(small, large)
    refused(lib.adi_hip_reorder_check(both, 2, 1 << 19, 64, 4), "too many rows")
    assert lib.adi_hip_reorder_check(both, 2, (1 << 19) - 1, 64, 4) == hip.OK
    assert lib.adi_hip_reorder_check(both, 2, 1 << 19, 4, 4) == hip.OK
    assert lib.adi_hip_reorder_check(None, 0, 2, 4, None) == hip.OK


# ---- pools ------------------------------------------------------------------------

def cache(**change):
    held = dict(type=0, heads=2, head_size=64, page_size=16, pages=100, keys=1 << 20, values=1 << 21,
                page_stride=2048, entry_stride=128, head_stride=64)
    held.update(change)
    return hip.PagedCacheStruct(**held)


def pool(caches=None, count=None, references=1 << 22, lacking=None):
    array = (hip.PagedCacheStruct * 2)(*(caches or [cache(), cache(keys=1 << 23, values=1 << 24)]))
    p = hip.PagedPoolStruct(2 if count is None else count, array, references, lacking)
    p.held = array
    return p


def batch(**change):
    held = dict(sequences=8, tokens=8, max_tokens=1, max_length=160, offsets=1 << 25, lengths=1 << 26,
                table=1 << 27, table_stride=10)
    held.update(change)
    return hip.PagedBatchStruct(**held)


def fork(**change):
    held = dict(beams=4, parents=1 << 28, lengths=1 << 26, table=1 << 27, table_stride=10, references=1 << 22)
    held.update(change)
    return hip.PagedForkArguments(**held)


POOLS = [
    (dict(count=0), "caches must be"), (dict(count=1025), "caches must be"),
    (dict(caches=[cache(), cache(type=2)]), "one type and layout"),
    (dict(caches=[cache(), cache(pages=99)]), "one type and layout"),
    (dict(caches=[cache(), cache(heads=1)]), "one type and layout"),
    (dict(caches=[cache(), cache(head_size=128)]), "one type and layout"),
    (dict(caches=[cache(), cache(page_size=8)]), "one type and layout"),
    (dict(caches=[cache(), cache(page_stride=4096)]), "one type and layout"),
    (dict(caches=[cache(pages=(1 << 22) + 1)] * 2), "2^22 pages"),
    (dict(caches=[cache(head_size=48)] * 2), "head size"),
    (dict(caches=[cache(keys=(1 << 20) + 4)] * 2), "16-byte"),
    (dict(caches=[cache(heads=4096, page_size=4096)] * 2), "2^30 elements"),
]


@pytest.mark.parametrize("change,message", POOLS + [
    (dict(references=None), "references"), (dict(references=(1 << 22) + 2), "references"),
    (dict(lacking=2), "references")])
def test_counted_pool_refusals(change, message):
    lib = hip.load()
    p = pool(**change)
    refused(lib.adi_hip_paged_fork_check(C.byref(p), C.byref(batch()), C.byref(fork())), message)
    compact = hip.PagedCompactArguments(1 << 22, 8, 1 << 26, 1 << 27, 1 << 27, 10, 1 << 28)
    refused(lib.adi_hip_paged_compact_check(C.byref(p), C.byref(compact)), message)


@pytest.mark.parametrize("change,message", POOLS)
def test_copied_pool_refusals(change, message):
    lib = hip.load()
    p = pool(**change)
    good = pool()
    for a, b in [(p, good), (good, p), (p, p)]:
        refused(lib.adi_hip_paged_copy_check(C.byref(a), C.byref(b), 4, 4, None, 3), message)


@pytest.mark.parametrize("to,args,message", [
    ({}, (4, 4, None, (1 << 22) + 1), "2^22"), ({}, (None, 4, None, 1), "null"), ({}, (4, None, None, 1), "null"),
    ({}, (2, 4, None, 1), "unaligned"), ({}, (4, 2, None, 1), "unaligned"), ({}, (4, 4, 2, 1), "unaligned"),
    (dict(count=1), (4, 4, None, 1), "different caches"),
    (dict(caches=[cache(type=2)] * 2), (4, 4, None, 1), "different caches"),
    (dict(caches=[cache(heads=1)] * 2), (4, 4, None, 1), "different caches"),
    (dict(caches=[cache(head_size=128)] * 2), (4, 4, None, 1), "different caches"),
    (dict(caches=[cache(page_size=8)] * 2), (4, 4, None, 1), "different caches")])
def test_copy_refusals(to, args, message):
    refused(hip.load().adi_hip_paged_copy_check(C.byref(pool()), C.byref(pool(**to)), *args), message)


def test_copy_accepts():
    lib = hip.load()
    other = pool(caches=[cache(pages=7, entry_stride=64, head_stride=1024)] * 2, references=None)
    assert lib.adi_hip_paged_copy_check(C.byref(pool()), C.byref(other), 4, 4, 4, 1 << 22) == hip.OK
    assert lib.adi_hip_paged_copy_check(C.byref(pool()), C.byref(other), None, None, None, 0) == hip.OK


@pytest.mark.parametrize("change,arguments,message", [
    ({}, dict(beams=0), "beams must be"), ({}, dict(beams=65), "beams must be"), ({}, dict(beams=3), "multiple"),
    ({}, dict(parents=None), "null"), ({}, dict(lengths=None), "null"), ({}, dict(table=None), "null"),
    ({}, dict(references=None), "null"), ({}, dict(parents=2), "unaligned"), ({}, dict(lengths=2), "unaligned"),
    ({}, dict(table=2), "unaligned"), ({}, dict(references=2), "unaligned"), ({}, dict(table_stride=0), "null"),
    ({}, dict(table_stride=11), "different strides"),
    ({"table_stride": 9}, {}, "shorter than max_length"), ({"max_length": 1 << 28}, {}, "2^28"),
    ({"max_length": 0, "table": None}, {}, "null"), ({"offsets": None}, {}, "null offsets"),
    ({"max_tokens": 9}, {}, "max_tokens"), ({"table_stride": (1 << 30) + 1000}, dict(table=4), "too large")])
def test_fork_refusals(change, arguments, message):
    lib = hip.load()
    refused(lib.adi_hip_paged_fork_check(C.byref(pool()), C.byref(batch(**change)), C.byref(fork(**arguments))), message)


def test_fork_accepts():
    lib = hip.load()
    for change, arguments in [({}, {}), ({}, dict(beams=1)), ({}, dict(beams=8)), ({}, dict(table=1 << 29)),
                              ({}, dict(table=1 << 29, table_stride=3)),
                              ({"sequences": 0}, dict(parents=None, lengths=None, table=None))]:
        assert lib.adi_hip_paged_fork_check(C.byref(pool()), C.byref(batch(**change)),
                                            C.byref(fork(**arguments))) == hip.OK
    refused(lib.adi_hip_paged_fork_check(C.byref(pool()), C.byref(batch()), None), "null arguments")
    refused(lib.adi_hip_paged_fork_check(C.byref(pool()), None, C.byref(fork())), "null")


def test_compact_refusals():
    lib = hip.load()
    p = pool()
    good = dict(references=1 << 22, rows=8, lengths=1 << 26, table=1 << 27, next_table=1 << 27, table_stride=10,
                live=1 << 28)
    check = lambda **change: lib.adi_hip_paged_compact_check(  # noqa: E731
        C.byref(p), C.byref(hip.PagedCompactArguments(**{**good, **change})))
    assert check() == hip.OK
    assert check(rows=0, lengths=None, table=None, next_table=None, table_stride=0) == hip.OK
    for change, message in [(dict(references=None), "null"), (dict(live=None), "null"), (dict(live=2), "unaligned"),
                            (dict(references=2), "unaligned"), (dict(rows=(1 << 20) + 1), "rows"),
                            (dict(lengths=None), "null or unaligned table"), (dict(table=None), "table"),
                            (dict(next_table=None), "table"), (dict(table_stride=0), "table"),
                            (dict(lengths=2), "table"), (dict(table=2), "table"), (dict(next_table=2), "table")]:
        refused(check(**change), message)
