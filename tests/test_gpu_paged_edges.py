"""Paged attention at the edges of what its documentation allows.

Where scores are far from 0, results have the same bounds as for scores near it,
as long as a score stays within a float.

The scores of these cases are exact in a float, so a weight's error is that of
its exponent. An exponent passes at most four roundings (from its score, to a
new level, to its part's level, to the row's), each half a step of at most 64
(what lies below weighs less than 2^-64): 4 * 64 * 2^-24 * ln 2 < 2^-16. The
exponential and the joins' factors add at most 16 half steps of a float, and a
16-bit weight half a step of its type, in the numerator and (k_paged_chunk) in the
denominator."""
import math

import numpy as np
import pytest
import torch

from adi_amd import hip
from test_gpu_paged import PAIRS, TYPES, U, Pool, attention, check_attention, half_step, normal, within

pytestmark = pytest.mark.gpu

STEP = [1, 1, 3]            # rows of k_paged_step (8 query heads on 2)
CHUNK = [40, 1, 9]          # k_paged_chunk
LENGTHS = [130, 1, 3000]    # one part and several


@pytest.fixture(scope="module")
def workspace(gpu):
    w = hip.PagedWorkspace(gpu)
    yield w
    gpu.synchronize()
    w.close()


def weighted(pool, scores, counts, lengths, heads, values, kind, scale):
    """(outputs, bound) [tokens, heads, size] in double of exact scores
    scores(row, entries) -> [heads, entries]."""
    out, bound = [], []
    for s, (a, length) in enumerate(zip(pool.offsets, lengths)):
        at = np.arange(length)
        pages = torch.tensor(pool.table[s, at // pool.page], device="cuda")
        v = values[pages, torch.tensor(at % pool.page, device="cuda")].double()
        v = v.repeat_interleave(heads // v.shape[1], 1).permute(1, 0, 2)  # [heads, entries, size]
        for i in range(counts[s]):
            n = max(length - counts[s] + i + 1, 0)
            w = torch.softmax(scores(a + i, s)[:, :n] * scale, -1)
            o = torch.bmm(w[:, None], v[:, :n].contiguous())[:, 0] if n else torch.zeros_like(v[:, 0])
            spread = torch.bmm(w[:, None], v[:, :n].abs().contiguous())[:, 0] if n else torch.zeros_like(o)
            error = 2 * (2.0 ** -16 + 16 * U) + (0 if kind == "f32" else 2 * half_step(kind)) + 3 * (n + 16) * U
            out.append(o)
            bound.append(spread * error + half_step(kind) * (o.abs() + spread * error) + torch.finfo(TYPES[kind]).tiny)
    return torch.stack(out), torch.stack(bound)


FAR = {  # far, near dimensions of a query and a key's far one; the near ones' unit; scale
    # scores near 2^26 with steps of 8, 2^23 scaled: weights within a few of each other
    "f16": [(2048.0, 1.0, 32960.0, 16.0, 1 / 8), (32768.0, 2.0, 32768.0, 64.0, 2.0 ** -7),
            # near 2^31 in steps of 256, scaled 2^28: all of the weight on the largest
            (49152.0, 1.0, 49152.0, 256.0, 1 / 8)],
    "bf16": [(2.0 ** 20, 1.0, 2.0 ** 20, 2.0 ** 17, 2.0 ** -17), (2.0 ** 40, 2.0 ** 40, 2.0 ** 40, 2.0 ** 17, 2.0 ** -57),
             (2.0 ** 50, 2.0 ** 50, 2.0 ** 50, 2.0 ** 27, 1 / 8)],
}
FAR["f32"] = FAR["bf16"]


@pytest.mark.parametrize("rows,kind", PAIRS)
@pytest.mark.parametrize("which", range(3))
@pytest.mark.parametrize("counts", [STEP, CHUNK])
@pytest.mark.parametrize("size", [64, 128, 256])
def test_exact_scores_far_from_zero(gpu, workspace, rows, kind, which, counts, size):
    """Scores a b + c u: a b (or its negative, or 0, by row) beside which a float
    has few bits left, u from 0 to 7."""
    far, near, key, unit, scale = FAR[rows][which]
    heads, kv = 8, 2
    pool = Pool(5 + which, LENGTHS, 16, kv, size, kind)
    batch = pool.batch(gpu, counts)
    n = pool.tokens
    rng = np.random.default_rng(which)
    small = [torch.tensor(rng.integers(0, 8, length), device="cuda").double() for length in LENGTHS]
    for s, length in enumerate(LENGTHS):
        for p in range(-(-length // 16)):
            page, held = int(pool.table[s, p]), min(16, length - 16 * p)
            pool.keys[page, :held] = 0
            pool.keys[page, :held, :, 3] = key
            pool.keys[page, :held, :, size - 5] = (small[s][16 * p:16 * p + held] * unit)[:, None].to(pool.keys.dtype)
    sign = torch.tensor(rng.choice([1.0, 1.0, -1.0, 0.0], (n, heads)), device="cuda")
    q = torch.zeros(n, heads, size, dtype=TYPES[rows], device="cuda")
    q[..., 3] = (sign * far).to(q.dtype)
    q[..., size - 5] = near
    assert torch.equal(q[..., 3].double(), sign * far) and float(pool.keys[int(pool.table[0, 0]), 0, 0, 3]) == key

    def scores(row, s):
        score = sign[row][:, None] * (far * key) + near * unit * small[s][None, :]
        assert torch.equal(score.float().double(), score)
        return score

    out = torch.empty_like(q)
    hip.paged_attention(gpu, pool.cache(gpu), batch, q, out, workspace, scale=scale)
    want, bound = weighted(pool, scores, counts, LENGTHS, heads, pool.values, rows, scale)
    within(out, want, bound)


@pytest.mark.parametrize("rows,kind", PAIRS)
@pytest.mark.parametrize("magnitude", [300.0, 5000.0, 20000.0])
@pytest.mark.parametrize("counts", [STEP, CHUNK])
@pytest.mark.parametrize("heads", [8, 64])
def test_equal_keys_of_any_magnitude_weigh_the_same(gpu, workspace, rows, kind, magnitude, counts, heads):
    """Every key of a head the same random row, so that its scores, however
    rounded, are one number: outputs are the values' means, one entry's its value."""
    size, kv = 64, 2
    pool = Pool(9, LENGTHS, 16, kv, size, kind)
    # (f16's largest is 65504)
    key = normal(4, kv, size, scale=magnitude).clamp(-60000, 60000).to(TYPES[kind])
    for s, length in enumerate(LENGTHS):
        for p in range(-(-length // 16)):
            pool.keys[int(pool.table[s, p]), :min(16, length - 16 * p)] = key
    batch = pool.batch(gpu, counts)
    q = normal(5, pool.tokens, heads, size, scale=magnitude).clamp(-60000, 60000).to(TYPES[rows])
    out = torch.empty_like(q)
    hip.paged_attention(gpu, pool.cache(gpu), batch, q, out, workspace)
    even = [torch.zeros(heads, length, dtype=torch.float64, device="cuda") for length in LENGTHS]
    want, bound = weighted(pool, lambda row, s: even[s], counts, LENGTHS, heads, pool.values, rows, 1.0)
    within(out, want, bound)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("up,down", [(115, -115), (-100, 100), (-115, 115), (105, -112), (-125, 10)])
@pytest.mark.parametrize("counts,lengths", [([1], [100]), ([33], [100]), ([33, 2], [90, 2000])])
def test_queries_and_keys_at_both_ends_of_a_float(gpu, workspace, kind, up, down, counts, lengths):
    """f32 queries of 2^up and keys of 2^down: ordinary scores, or nothing."""
    def bend(pool, q):
        pool.keys.mul_(2.0 ** down)
        q.mul_(2.0 ** up)

    for size in (64, 128, 256):
        check_attention(gpu, workspace, "f32", kind, size, 4, 2, 32, counts, lengths, bend=bend)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("counts", [[1], [33]])
def test_large_queries_across_large_keys(gpu, workspace, kind, counts):
    """Queries and keys whose largest elements' product is past a float while their
    scores are 0, and keys whose elements are 2^220 apart."""
    def across(pool, q):
        pool.keys[..., 32:].mul_(2.0 ** 110)
        pool.keys[..., :32] = 0
        q[..., :32].mul_(2.0 ** 110)
        q[..., 32:] = 0

    def apart(pool, q):
        pool.keys[..., :32].mul_(2.0 ** -110)
        pool.keys[..., 32:].mul_(2.0 ** 110)
        q[..., :32] = 0
        q[..., 32:].mul_(2.0 ** -100)
        q.mul_(2.0 ** -10)

    for b in (across, apart):
        check_attention(gpu, workspace, "f32", kind, 64, 4, 2, 32, counts, [100], bend=b)


@pytest.mark.parametrize("rows,kind", PAIRS)
@pytest.mark.parametrize("heads", [4, 64])
@pytest.mark.parametrize("junk", [math.nan, math.inf, -math.inf])
def test_rows_that_see_nothing_are_zero_whatever_they_hold(gpu, workspace, rows, kind, heads, junk):
    """Front padding and empty sequences whose queries and gates were never
    written: 0, and the other rows as with ordinary padding."""
    counts, lengths = [3, 4, 2, 40], [1, 0, 50, 37]
    pool = Pool(3, lengths, 16, 2, 64, kind)
    batch = pool.batch(gpu, counts)
    q, gate = (normal(i, pool.tokens, heads, 64, kind=rows) for i in (1, 2))
    blank = torch.zeros(pool.tokens, dtype=torch.bool, device="cuda")
    for a, n, length in zip(pool.offsets, counts, lengths):
        blank[a:a + max(n - length, 0)] = True
    assert int(blank.sum()) == 2 + 4 + 3
    out = torch.empty_like(q), torch.empty_like(q)
    hip.paged_attention(gpu, pool.cache(gpu), batch, q, out[0], workspace, gate=gate)
    q[blank], gate[blank] = junk, junk
    hip.paged_attention(gpu, pool.cache(gpu), batch, q, out[1], workspace, gate=gate)
    assert bool((out[1][blank] == 0).all()) and torch.equal(*out)
    assert bool((out[1][~blank] != 0).any(-1).all())


def test_a_step_of_more_than_2_to_32_entries(gpu, workspace):
    """Twenty histories of 2^28 - 1 entries among 43 of one, all of one page, on 8
    heads: one block more than sequences, so a part is a whole history. Value
    (e, head, d) is head + 1 where e % 64 = d, so every sum is exact."""
    n, page, heads, size, longest = 63, 4096, 8, 64, (1 << 28) - 1
    lengths = [longest if s % 3 == 1 and s < 60 else 1 for s in range(n)]
    keys = torch.zeros(1, page, heads, size, dtype=torch.bfloat16, device="cuda")
    values = torch.eye(size, dtype=torch.bfloat16, device="cuda").repeat(page // size, 1)[None, :, None, :]
    values = values * torch.arange(1, heads + 1, device="cuda").to(torch.bfloat16)[:, None]
    table = torch.zeros(n, 1 << 16, dtype=torch.int32, device="cuda")
    batch = hip.PagedBatch(gpu, torch.arange(n + 1, dtype=torch.int32, device="cuda"),
                           torch.tensor(lengths, dtype=torch.int32, device="cuda"), table, n, 1, longest)
    q = normal(1, n, heads, size, kind="bf16")
    out = torch.full_like(q, 7.0)
    hip.paged_attention(gpu, hip.PagedCache(gpu, keys, values), batch, q, out, workspace)
    scale = torch.arange(1, heads + 1, device="cuda").double()[:, None]
    at = torch.arange(size, device="cuda")
    for s, length in enumerate(lengths):
        want = scale * ((length - at + size - 1) // size).double() / length
        within(out[s], want, want * (half_step("bf16") + 16 * U), s)
    # the workspace as it was: a call after it gives what it gives alone
    check_attention(gpu, workspace, "bf16", "bf16", 64, 8, 8, 16, [1] * 8, [4000] * 8)


def test_a_refused_layer_call_appends_nothing(gpu, workspace):
    """More sequences than the attention takes (the append takes them)."""
    from adi_amd import synthetic as syn
    rng = syn.rng_for(40, 256)
    tlut = syn.ne_tlut(rng)
    layer = hip.upload_full_attention(gpu, syn.full_attention(rng, 256, tlut), gpu.ne_codebook(tlut))
    keys = normal(1, 2, 16, 2, 256)
    before, x = keys.clone(), normal(2, 1, 256)
    n = 1 << 16
    offsets, lengths = (torch.ones(k, dtype=torch.int32, device="cuda") for k in (n + 1, n))
    offsets[0] = 0
    batch = hip.PagedBatch(gpu, offsets, lengths, torch.zeros(n, 1, dtype=torch.int32, device="cuda"), 1, 1, 16)
    cache = hip.PagedCache(gpu, keys, keys.clone())
    with pytest.raises(hip.HipError, match="65535") as info:
        hip.full_attention_paged(gpu, layer, cache, batch, x, torch.empty_like(x), workspace)
    assert info.value.status == hip.INVALID_ARGUMENT
    gpu.synchronize()
    assert torch.equal(keys, before)


def test_numbers_past_a_float_are_refused(gpu, workspace):
    pool = Pool(1, [20], 16, 2, 64, "bf16", junk=None)
    q, k = normal(1, 1, 4, 64, kind="bf16"), normal(2, 1, 2, 64, kind="bf16")
    cache, batch = pool.cache(gpu), pool.batch(gpu, [1])
    for call in (lambda: hip.paged_attention(gpu, cache, batch, q, torch.empty_like(q), workspace, scale=1e39),
                 lambda: hip.paged_append(gpu, cache, batch, k, k, epsilon=1e39),
                 lambda: hip.paged_append(gpu, cache, batch, k, k, weight_offset=-1e39)):
        with pytest.raises(hip.HipError, match="past a float") as info:
            call()
        assert info.value.status == hip.INVALID_ARGUMENT


def test_a_float_step_is_as_near_as_float_sums_are(gpu, workspace):
    """One token of 16 f32 heads on 2 of 256 behind 1,999 entries, the error's mean
    square rather than its bound. A rounding's is (0.6 * 2^-24)^2 of the square of what
    is rounded. A score sums 256 products of deviation 2, in four sums of 64: its error
    has the mean square (0.6 * 2^-24)^2 * 4 * 64^2 / 2 * 2^2, so a sixteenth (the scale)
    of its root is 4.0e-7; a weight is off by as much of itself, and an output, a sum of
    weights times values of random sign, by as much of its own size. The exponentials,
    the sums of products and the quotient are under ten roundings of 0.6 * 2^-24 more:
    sqrt(4.0^2 + 10 * 0.36^2) = 4.2; half as much again for eight draws."""
    error = size = 0.0
    for seed in range(8):
        pool = Pool(100 + 10 * seed, [2000], 16, 2, 256, "f32")
        q = normal(seed, 1, 16, 256, scale=2.0)
        out = torch.empty_like(q)
        hip.paged_attention(gpu, pool.cache(gpu), pool.batch(gpu, [1]), q, out, workspace)
        want, _, _ = attention(q, pool.keys, pool.values, pool.offsets, [2000], pool.table, 16, 1 / 16, 0, "f32")
        error += float((out.double() - want).square().sum())
        size += float(want.square().sum())
    assert math.sqrt(error / size) <= 1.5 * 4.2e-7, math.sqrt(error / size)
