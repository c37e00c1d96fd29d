"""The rotary and paged-cache entry points without a GPU: their structures
against the header, the frequencies of every scaling against their formulas in
double, the refusals of both, and adi_hip_paged_check over host arrays."""
import concurrent.futures
import ctypes as C
import math
import os
import subprocess

import numpy as np
import pytest

from adi_amd import hip

HEADER = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "adi_hip.h")

STRUCTS = {
    "adi_hip_rope_options": hip.RopeOptions,
    "adi_hip_rows": hip.Rows,
    "adi_hip_paged_cache": hip.PagedCacheStruct,
    "adi_hip_paged_batch": hip.PagedBatchStruct,
    "adi_hip_paged_append_arguments": hip.PagedAppendArguments,
    "adi_hip_paged_attention_arguments": hip.PagedAttentionArguments,
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
    rows = [(i, 10 * i + 1, 10 * i + 2, 10 * i + 3) for i in range(5)]
    assert hip._pack_rows(*rows[1]) == bytes(hip.Rows(*rows[1]))
    assert hip._pack_append(77, *rows[0], *rows[1], 78, 79, *rows[2], *rows[3], 80, 1.5, 2.5) == bytes(
        hip.PagedAppendArguments(77, hip.Rows(*rows[0]), hip.Rows(*rows[1]), 78, 79, hip.Rows(*rows[2]),
                                 hip.Rows(*rows[3]), 80, 1.5, 2.5))
    assert hip._pack_attention(9, *rows[1], *rows[2], *rows[3], 0.5, 6) == bytes(
        hip.PagedAttentionArguments(9, hip.Rows(*rows[1]), hip.Rows(*rows[2]), hip.Rows(*rows[3]), 0.5, 6))


# ---- frequencies --------------------------------------------------------------

def close(got, want):
    # pow, log and the ramp are a few roundings of 2^-53 each; log(theta) in the
    # exponent multiplies them by at most 20
    np.testing.assert_allclose(got, want, rtol=1e-13, atol=0)


@pytest.mark.parametrize("rotary", [2, 6, 64, 128, 1024])
@pytest.mark.parametrize("theta", [1e4, 1e7])
def test_plain_linear_and_ntk(rotary, theta):
    i = np.arange(rotary // 2)
    base = theta ** (-2.0 * i / rotary)
    f, m = hip.rope_frequencies(rotary, theta=theta)
    close(f, base)
    assert m == 1.0
    close(hip.rope_frequencies(rotary, theta=theta, scaling="linear", factor=8.0)[0], base / 8)
    if rotary > 2:
        f, _ = hip.rope_frequencies(rotary, theta=theta, scaling="ntk", factor=8.0)
        close(f[0], 1.0)
        close(f[-1], base[-1] / 8)
    assert hip.rope_frequencies(rotary, theta=theta, magnitude=0.5)[1] == 0.5


@pytest.mark.parametrize("fast,slow", [(0.0, 0.0), (16.0, 2.0)])
def test_yarn(fast, slow):
    rotary, theta, factor, original = 64, 1e4, 4.0, 4096.0
    i = np.arange(rotary // 2)
    base = theta ** (-2.0 * i / rotary)
    f, m = hip.rope_frequencies(rotary, theta=theta, scaling="yarn", factor=factor, original=original, fast=fast,
                                slow=slow)
    a, b = (fast, slow) if fast else (32.0, 1.0)
    # the pair that turns t times over the original context
    pair = [rotary * math.log(original / (t * 2 * math.pi)) / (2 * math.log(theta)) for t in (a, b)]
    low, high = max(math.floor(pair[0]), 0), min(math.ceil(pair[1]), rotary - 1)
    ramp = np.clip((i - low) / (high - low), 0, 1)
    close(f, base * (1 - ramp) + base / factor * ramp)
    assert f[0] == base[0] and abs(m - (0.1 * math.log(factor) + 1)) < 1e-15


@pytest.mark.parametrize("fast,slow", [(0.0, 0.0), (8.0, 2.0)])
def test_bands(fast, slow):
    rotary, theta, factor, original = 128, 5e5, 8.0, 8192.0
    base = theta ** (-2.0 * np.arange(rotary // 2) / rotary)
    f, m = hip.rope_frequencies(rotary, theta=theta, scaling="bands", factor=factor, original=original, fast=fast,
                                slow=slow)
    a, b = (fast, slow) if fast else (4.0, 1.0)
    for got, plain in zip(f, base):
        turns = original * plain / (2 * math.pi)
        if turns >= a:
            want = plain
        elif turns <= b:
            want = plain / factor
        else:
            part = (turns - b) / (a - b)
            want = plain * part + plain / factor * (1 - part)
        close(got, want)
    assert m == 1.0


@pytest.mark.parametrize("options,message", [
    (dict(rotary=0), "rotary must be even"),
    (dict(rotary=7), "rotary must be even"),
    (dict(rotary=1026), "rotary must be even"),
    (dict(rotary=64, theta=1.0), "theta"),
    (dict(rotary=64, theta=float("nan")), "theta"),
    (dict(rotary=64, scaling="linear", factor=0.5), "factor"),
    (dict(rotary=64, scaling="yarn", factor=float("inf"), original=4096.0), "factor"),
    (dict(rotary=64, scaling="yarn", factor=2.0), "original"),
    (dict(rotary=64, scaling="bands", factor=2.0, original=4096.0, fast=1.0, slow=2.0), "fast must be above slow"),
    (dict(rotary=64, scaling="bands", factor=2.0, original=4096.0, fast=2.0, slow=0.0), "slow above 0"),
    (dict(rotary=2, scaling="ntk", factor=2.0), "NTK"),
    (dict(rotary=64, magnitude=-1.0), "magnitude"),
    (dict(rotary=64, layout="thirds"), "layout"),
])
def test_frequency_refusals(options, message):
    with pytest.raises(hip.HipError, match=message) as info:
        hip.rope_frequencies(**options)
    assert info.value.status == hip.INVALID_ARGUMENT


def test_unknown_codes_are_refused():
    lib = hip.load()
    for layout, scaling in ((2, 0), (0, 5)):
        o = hip.RopeOptions(64, layout, scaling, 1e4, 1.0, 1.0, 0.0, 0.0, 0.0)
        assert lib.adi_hip_rope_frequencies(C.byref(o), None, None) == hip.INVALID_ARGUMENT
        assert b"unknown" in lib.adi_hip_last_error(None)
    assert lib.adi_hip_rope_frequencies(None, None, None) == hip.INVALID_ARGUMENT


# ---- descriptors and batches -----------------------------------------------------

POOL = np.zeros(4096, np.uint8)
ALIGNED = POOL.ctypes.data + (-POOL.ctypes.data) % 64


def cache(**change):
    fields = dict(type=hip.BF16, heads=2, head_size=64, page_size=16, pages=10, keys=ALIGNED, values=ALIGNED,
                  page_stride=2048, entry_stride=128, head_stride=64)
    fields.update(change)
    return hip.PagedCacheStruct(**fields)


def batch(**change):
    fields = dict(offsets=np.array([0, 3, 3, 4]), lengths=np.array([40, 0, 16]),
                  table=np.array([[7, 0, 9], [-1, -1, -1], [3, -1, -1]]), tokens=6, max_tokens=3, max_length=48)
    fields.update(change)
    return fields


def test_check_accepts():
    hip.paged_check(cache(), **batch())
    hip.paged_check(cache(), **batch(offsets=np.array([0]), lengths=np.zeros(0, int), table=np.zeros((0, 0), int),
                                     tokens=0, max_tokens=0, max_length=0))
    # one shared page, front padding (more rows than entries)
    hip.paged_check(cache(), **batch(table=np.array([[7, 0, 9], [7, 0, 9], [7, 0, 9]]), lengths=np.array([2, 0, 16])))


@pytest.mark.parametrize("change,message", [
    (dict(type=3), "unknown type"),
    (dict(heads=0), "heads"),
    (dict(head_size=96), "head size"),
    (dict(page_size=24), "page size"),
    (dict(page_size=4), "page size"),
    (dict(page_size=8192), "page size"),
    (dict(pages=0), "no pages"),
    (dict(keys=None), "aligned"),
    (dict(values=ALIGNED + 8), "aligned"),
    (dict(entry_stride=132), "aligned"),
    (dict(head_stride=68), "aligned"),
    (dict(page_stride=2052), "aligned"),
])
def test_cache_refusals(change, message):
    with pytest.raises(hip.HipError, match=message) as info:
        hip.paged_check(cache(**change), **batch())
    assert info.value.status == hip.INVALID_ARGUMENT


@pytest.mark.parametrize("change,message", [
    (dict(max_length=64), "page table is shorter"),
    (dict(max_length=1 << 28), "max_length"),
    (dict(max_tokens=7), "max_tokens must be at most tokens"),
    (dict(offsets=np.array([0, 3, 2, 4])), "sequence 1's rows do not ascend"),
    (dict(offsets=np.array([0, 3, 3, 7])), "sequence 2's rows do not ascend"),
    (dict(offsets=np.array([0, 2, 2, 6])), "sequence 2 has more than max_tokens"),
    (dict(lengths=np.array([40, 49, 16])), "sequence 1 has more than max_length"),
    (dict(table=np.array([[7, 10, 9], [-1, -1, -1], [3, -1, -1]])), "sequence 0's page 1 "),
    (dict(lengths=np.array([40, 0, 17])), "sequence 2's page 1 "),
    (dict(lengths=np.array([40, 1, 16])), "sequence 1's page 0 "),
])
def test_batch_refusals(change, message):
    with pytest.raises(hip.HipError, match=message) as info:
        hip.paged_check(cache(), **batch(**change))
    assert info.value.status == hip.INVALID_ARGUMENT


def test_null_context_and_descriptors():
    lib = hip.load()
    assert lib.adi_hip_paged_check(None, None) == hip.INVALID_ARGUMENT
    assert lib.adi_hip_paged_append(None, None, None, None) == hip.INVALID_ARGUMENT
    assert lib.adi_hip_paged_attention(None, None, None, None, None) == hip.INVALID_ARGUMENT
    assert lib.adi_hip_rope_rows(None, None, None, 0, 0, 0, None, None) == hip.INVALID_ARGUMENT
    lib.adi_hip_rope_destroy(None)
    lib.adi_hip_paged_workspace_destroy(None)


def test_threads_keep_their_own_messages():
    """Two threads whose checks fail differently, one of them many times while
    the other holds its message's address."""
    raw = C.CDLL(hip.load()._name)
    raw.adi_hip_last_error.restype = C.c_void_p
    raw.adi_hip_last_error.argtypes = [C.c_void_p]
    address = []

    def fail(change, message):
        with pytest.raises(hip.HipError, match=message):
            hip.paged_check(cache(**change), **batch())

    def other():
        for heads in (0, 70000):
            for _ in range(200):
                fail(dict(heads=heads), "heads must be")
                assert C.string_at(raw.adi_hip_last_error(None)).endswith(b"heads must be 1 to 65536")

    fail(dict(page_size=24), "page size")
    address.append(raw.adi_hip_last_error(None))
    held = C.string_at(address[0])
    assert b"page size" in held
    with concurrent.futures.ThreadPoolExecutor(3) as pool:
        for done in [pool.submit(other) for _ in range(3)]:
            done.result()
    assert C.string_at(address[0]) == held and raw.adi_hip_last_error(None) == address[0]


def test_a_thread_without_a_message_reads_the_last_failed_creation():
    lib = hip.load()
    with concurrent.futures.ThreadPoolExecutor(1) as pool:
        assert pool.submit(lib.adi_hip_context_create, 4096, None).result() == hip.INVALID_ARGUMENT
    with concurrent.futures.ThreadPoolExecutor(1) as pool:
        assert pool.submit(lib.adi_hip_last_error, None).result() == b"adi_hip_context_create: null output pointer"


@pytest.mark.parametrize("change,message", [
    (dict(tokens=(1 << 32) + 6), "out of range"),
    (dict(max_tokens=(1 << 32) + 3), "out of range"),
    (dict(max_length=(1 << 32) + 48), "out of range"),
    (dict(offsets=np.array([0, 3, 3, (1 << 32) + 4])), "32-bit"),
    (dict(lengths=np.array([40, 1 << 40, 16])), "32-bit"),
    (dict(table=np.array([[7, 1 << 32, 9], [-1, -1, -1], [3, -1, -1]])), "32-bit"),
    (dict(lengths=np.array([40.5, 0, 16])), "32-bit"),
])
def test_check_refuses_what_32_bits_cannot_hold(change, message):
    """Each of these, cut to 32 bits, is the accepted batch."""
    with pytest.raises(hip.HipError, match=message) as info:
        hip.paged_check(cache(), **batch(**change))
    assert info.value.status == hip.INVALID_ARGUMENT


def test_rotary_dimensions_past_32_bits():
    with pytest.raises(hip.HipError, match="rotary") as info:
        hip.rope_frequencies((1 << 32) + 64)
    assert info.value.status == hip.INVALID_ARGUMENT


@pytest.mark.parametrize("magnitude", [1e39, 1e300, 1e-46, float("inf"), float("nan"), -0.5])
def test_magnitudes_that_a_float_cannot_hold(magnitude):
    with pytest.raises(hip.HipError, match="magnitude") as info:
        hip.rope_frequencies(64, magnitude=magnitude)
    assert info.value.status == hip.INVALID_ARGUMENT
