"""The choice of a beam search's step and the states that follow it on the GPU,
against the definitions in double: every type, one token to the checkpoint's
vocabulary and odd ones, ties, masked tokens, beams that are dead, ended, NaN or
all alike, ranks next to each other, strides, captured and concurrent calls.

A score's bound: half a step of the float it is rounded to, and 2^-32 for the
logarithm of the sum (exponentials good to 2^-33 of theirs, sums in double)."""
import math

import numpy as np
import pytest
import torch

from adi_amd import hip

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
U = 2.0 ** -24
NONE = -1


def normal(seed, *shape, kind="f32", scale=1.0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return (torch.randn(*shape, device="cuda", generator=g) * scale).to(TYPES[kind])


def ints(values):
    return torch.tensor(np.asarray(values), dtype=torch.int32, device="cuda")


@pytest.fixture(scope="module")
def workspace(gpu):
    w = hip.PagedWorkspace(gpu)
    yield w
    gpu.synchronize()
    w.close()


def chosen(logits, scores, choices, weights=None, ended=None, ended_token=0, settle=False):
    """The definition, request by request: (scores, parents, tokens) in double."""
    n, k, v = logits.shape
    out = np.full((n, choices), -np.inf), np.full((n, choices), NONE), np.full((n, choices), NONE)
    scores = scores.double().cpu().numpy()
    weights = np.ones((n, k)) if weights is None else weights.double().cpu().numpy()
    ended = np.zeros((n, k)) if ended is None else ended.cpu().numpy()
    for r in range(n):
        found, bad = [], False
        for b in range(k):
            s, w = scores[r, b], weights[r, b]
            if s == -math.inf:
                continue
            bad |= not (math.isfinite(s) and 0 < w < math.inf)
            if ended[r, b]:
                found.append((-s * w, b, 0, ended_token, s))
                continue
            x = logits[r, b].double()
            bad |= bool(torch.isnan(x).any()) or bool((x == math.inf).any())
            if bad or bool((x == -math.inf).all()):
                continue
            most = x.max()
            lse = float(most + torch.log(torch.exp(x - most).sum()))
            x = x.cpu().numpy()
            for t in np.argsort(-x, kind="stable")[:choices]:
                if x[t] != -math.inf:
                    found.append((-(s + (x[t] - lse)) * w, b, -x[t], int(t), s + (x[t] - lse)))
        if bad:
            out[0][r] = np.nan
            continue
        found.sort()
        places = list(range(choices))
        best = found[:choices]
        if settle:
            parents = [f[1] for f in best]
            free = iter([i for i in range(k) if i not in parents])
            places = [f if parents.index(f) == i else next(free) for i, f in enumerate(parents)]
            places += list(free)
        for i, f in zip(places, best):
            out[0][r, i], out[1][r, i], out[2][r, i] = f[4], f[1], f[3]
    return out


def check(gpu, workspace, logits, scores, choices, **more):
    n = logits.shape[0]
    out = (torch.full((n, choices), 5.0, device="cuda"), ints(np.full((n, choices), 99)), ints(np.full((n, choices), 99)))
    hip.beam_select(gpu, logits, scores, *out, workspace, **more)
    want = chosen(logits, scores, choices, **more)
    got = [t.cpu().numpy() for t in out]
    assert np.array_equal(got[1], want[1]), (got[1], want[1])
    assert np.array_equal(got[2], want[2]), (got[2], want[2])
    fine = np.isfinite(want[0])
    assert np.array_equal(np.isnan(got[0]), np.isnan(want[0]))
    assert np.array_equal(got[0][~fine & ~np.isnan(want[0])], want[0][~fine & ~np.isnan(want[0])])
    bound = U * np.abs(want[0][fine]) + 2.0 ** -32
    assert (np.abs(got[0][fine].astype(np.float64) - want[0][fine]) <= bound).all()
    return out


def running(seed, n, k):
    return normal(seed, n, 1) * 3 - 20 + normal(seed + 1, n, k)


SIZES = [(1, 1, 1, 1), (2, 1, 1, 3), (1, 4, 17, 8), (3, 3, 513, 7), (2, 5, 2048, 10), (2, 2, 2049, 4), (1, 2, 8192, 128),
         (2, 2, 8193, 5), (5, 8, 50257, 16), (1, 64, 1000, 128), (3, 64, 33, 64), (1, 4, 248320, 8),
         (2, 16, 30001, 32), (17, 3, 4100, 6), (1, 1, 131072, 100), (300, 2, 100, 4)]


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n,k,v,choices", SIZES)
def test_sizes_and_types(gpu, workspace, kind, n, k, v, choices):
    check(gpu, workspace, normal(v + k, n, k, v, kind=kind, scale=3.0), running(v, n, k), choices)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("settle", [False, True])
@pytest.mark.parametrize("n,k,v", [(4, 4, 1000), (3, 8, 20000), (2, 64, 700), (5, 1, 300), (6, 5, 9)])
def test_weights_ended_beams_and_places(gpu, workspace, kind, settle, n, k, v):
    g = np.random.default_rng(k + v)
    ended = ints(g.random((n, k)) < 0.3) * ints(g.integers(1, 1 << 30, (n, k)))
    weights = torch.tensor(g.uniform(0.01, 2.0, (n, k)), dtype=torch.float32, device="cuda")
    logits = normal(k, n, k, v, kind=kind, scale=4.0)
    logits[ended != 0] = math.nan  # not read
    check(gpu, workspace, logits, running(9, n, k), k if settle else min(2 * k, 128), weights=weights, ended=ended,
          ended_token=3, settle=settle)


@pytest.mark.parametrize("v", [40, 5000, 248320])
def test_a_first_step_and_beams_all_alike(gpu, workspace, v):
    logits = normal(v, 2, 1, v, kind="bf16", scale=2.0).expand(2, 4, v).contiguous()
    scores = torch.tensor([[0.0, -math.inf, -math.inf, -math.inf]] * 2, device="cuda")
    for settle in (False, True):
        check(gpu, workspace, logits, scores, 4, settle=settle)
    # every candidate four times: the lower beam first
    check(gpu, workspace, logits, torch.full((2, 4), -7.25, device="cuda"), 16)
    check(gpu, workspace, logits.float(), torch.zeros(2, 4, device="cuda"), 7)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("v,choices", [(6, 6), (300, 7), (8192, 33), (20011, 128)])
@pytest.mark.parametrize("values", [1, 2, 5])
def test_equal_logits(gpu, workspace, kind, v, choices, values):
    """A handful of values (-0 and 0 among them) at all the tokens."""
    levels = torch.tensor([0.0, -0.0, -1.5, -2.0, 0.25][:values], device="cuda", dtype=TYPES[kind])
    g = torch.Generator(device="cuda")
    g.manual_seed(v + values)
    logits = levels[torch.randint(0, values, (3, 3, v), device="cuda", generator=g)]
    check(gpu, workspace, logits, running(1, 3, 3), choices)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("fill", ["lowest", "-inf"])
@pytest.mark.parametrize("left", [0, 1, 5, 300])
def test_masked_tokens(gpu, workspace, kind, fill, left):
    """All but `left` tokens at the type's lowest value or -infinity."""
    v = 20000
    logits = normal(3, 2, 3, v, kind=kind)
    value = -math.inf if fill == "-inf" else torch.finfo(TYPES[kind]).min
    g = np.random.default_rng(left)
    keep = torch.zeros(2, 3, v, dtype=torch.bool, device="cuda")
    for r in range(2):
        for b in range(3):
            keep[r, b, torch.tensor(g.permutation(v)[:left], device="cuda", dtype=torch.long)] = True
    logits = torch.where(keep, logits, torch.full_like(logits, value))
    check(gpu, workspace, logits, running(2, 2, 3), 16)
    logits[0, 1] = -math.inf  # and a beam with nothing at all
    check(gpu, workspace, logits, running(2, 2, 3), 16)


def test_sorted_logits_and_spikes(gpu, workspace):
    """A row's best all in one place, at either end, and apart from the others."""
    v = 70001
    ramp = torch.linspace(-5, 5, v, device="cuda")
    logits = torch.stack([ramp, ramp.flip(0), torch.roll(ramp, 8000), ramp * 0 - 3])[None].contiguous()
    check(gpu, workspace, logits, torch.tensor([[-3.0, -3.5, -2.5, -1.0]], device="cuda"), 128)
    logits[0, 3, 65536:65600] = 2.0
    check(gpu, workspace, logits, torch.tensor([[-3.0, -3.5, -2.5, -1.0]], device="cuda"), 100)
    far = normal(8, 1, 2, 9000, scale=1e4)
    check(gpu, workspace, far, torch.tensor([[-3.0, -3.5]], device="cuda"), 20)


@pytest.mark.parametrize("v", [300, 9000, 70001])
def test_logits_far_from_0(gpu, workspace, v):
    """Every float is a logit: large ones of both signs, rows around the edges of what
    the kernel's own exponentials take (65536), parts of a row on either side of it."""
    for shift, scale in [(65536.0, 3.0), (-65536.0, 3.0), (7e4, 3.0), (-7e4, 3.0), (0.0, 3e4), (0.0, 1e30), (1e38, 1e37),
                         (-1e38, 1e37)]:
        logits = normal(v, 2, 2, v) * scale + shift
        check(gpu, workspace, logits, running(4, 2, 2), 9)
    half = normal(v, 1, 2, v)
    half[:, :, v // 2:] += 65536.0
    half[:, 1] -= 65530.0
    check(gpu, workspace, half, running(4, 1, 2), 9)
    for kind, shift in (("f16", 65000.0), ("f16", -65000.0), ("bf16", 3e38), ("bf16", -3e38)):
        check(gpu, workspace, (normal(v, 2, 2, v, scale=2.0) + shift).to(TYPES[kind]), running(4, 2, 2), 9)
    tiny = (normal(v, 2, 2, v) * 1e-39)  # below the normal floats
    check(gpu, workspace, tiny, running(4, 2, 2), 9)


def test_many_requests_of_few_tokens(gpu, workspace):
    n = 70000  # more than a launch takes
    out = torch.zeros(n, 2, device="cuda"), ints(np.zeros((n, 2))), ints(np.zeros((n, 2)))
    logits, scores = normal(1, n, 2, 5), running(1, n, 2)
    hip.beam_select(gpu, logits, scores, *out, workspace)
    x = (scores[..., None].double() + torch.log_softmax(logits.double(), -1)).reshape(n, 10)
    best = x.topk(2, -1)
    assert torch.equal(out[1], (best.indices // 5).int()) and torch.equal(out[2], (best.indices % 5).int())
    assert bool(((out[0].double() - best.values).abs() <= U * best.values.abs() + 2.0 ** -32).all())


def test_wrong_logits_and_scores(gpu, workspace):
    """A NaN or +infinity makes its request NaN, and no other; what a dead beam
    holds does not matter."""
    for v in (50, 9000):
        base = normal(v, 8, 3, v)
        scores = running(5, 8, 3)
        base[0, 1, v // 2] = math.nan
        base[1, 2, v - 1] = math.inf
        base[2, 0, 0] = -math.nan
        scores[3, 1] = math.nan
        scores[4, 1] = math.inf
        base[5, 0] = math.nan
        scores[5, 0] = -math.inf
        base[6, 2, 3] = -math.inf
        weights = torch.ones(8, 3, device="cuda")
        weights[5, 0] = math.nan  # of the dead beam
        check(gpu, workspace, base, scores, 6, weights=weights)
        for wrong in (0.0, -1.0, math.inf, math.nan):
            weights[7, 1] = wrong
            check(gpu, workspace, base, scores, 6, weights=weights)
        ended = torch.zeros(8, 3, dtype=torch.int32, device="cuda")
        ended[4, 1] = 1  # +infinity
        ended[3, 1] = 1
        ended[5, 0] = 1  # dead all the same
        check(gpu, workspace, base, scores, 6, ended=ended)
    dead = torch.full((2, 3), -math.inf, device="cuda")
    check(gpu, workspace, normal(1, 2, 3, 40), dead, 3)
    check(gpu, workspace, normal(1, 2, 3, 40), dead, 3, settle=True)


def test_ranks_next_to_each_other(gpu, workspace):
    """Candidates of two beams whose ranks differ by 1e-10 to 1e-8 only, through their
    scores or through one far logit of many."""
    v = 30000
    row = normal(4, v, scale=2.0)
    for gap in (1, 2, -1):
        logits = row.expand(1, 2, v).contiguous()
        a = np.float32(-1e-3)
        b = a
        for _ in range(abs(gap)):
            b = np.nextafter(b, np.float32(gap), dtype=np.float32)
        check(gpu, workspace, logits, torch.tensor([[a, b]], device="cuda"), 12)
    for change in (1.0, -1.0, 2.0):
        logits = row.expand(1, 2, v).contiguous()
        low = int(row.argmin())
        logits[0, 1, low] += change  # e^-8 of a sum of some 10^5
        check(gpu, workspace, logits, torch.full((1, 2), -2.5, device="cuda"), 12)


def test_strides_and_addresses(gpu, workspace):
    for kind in TYPES:
        for shift in (0, 1, 3):
            whole = normal(6, 4, 7, 5003, kind=kind, scale=2.0)
            check(gpu, workspace, whole[1:, 1:6, shift:shift + 4990], running(3, 3, 5), 10)
            check(gpu, workspace, whole.transpose(0, 1)[:, :3, shift:shift + 100], running(3, 7, 3), 3, settle=True)
    # a broadcast row of logits
    check(gpu, workspace, normal(6, 3, 1, 600).expand(3, 4, 600), running(3, 3, 4), 8)


def test_small_workspace_takes_requests_in_turn(gpu):
    w = hip.PagedWorkspace(gpu, 1 << 20)
    check(gpu, w, normal(1, 40, 4, 30000, kind="f16", scale=2.0), running(1, 40, 4), 64)
    check(gpu, w, normal(1, 40, 4, 30000, scale=2.0), running(1, 40, 4), 4, settle=True,
          weights=normal(3, 40, 4).abs() + 0.1, ended=ints(np.arange(160).reshape(40, 4) % 5 == 0))
    # 64 rows of 31 tiles of 12 + 8 * 128 bytes are 2 MiB
    with pytest.raises(hip.HipError, match="workspace") as e:
        check(gpu, w, normal(1, 1, 64, 248320), running(1, 1, 64), 128)
    assert e.value.status == hip.OUT_OF_MEMORY
    gpu.synchronize()
    w.close()


def test_logits_past_32_bits(gpu, workspace):
    """A vocabulary whose rows begin beyond 2^32 bytes."""
    rows = normal(1, 3, 2, 1000, kind="bf16", scale=2.0)
    whole = torch.empty((1 << 31) + 100000, dtype=torch.bfloat16, device="cuda")
    view = whole.as_strided((3, 2, 1000), (1 << 30, 50000, 1))
    view.copy_(rows)
    check(gpu, workspace, view, running(1, 3, 2), 8)


def test_captured_calls_replay(gpu, workspace):
    logits = normal(1, 6, 4, 40000, scale=2.0)
    scores = running(1, 6, 4)
    out = torch.zeros(6, 4, device="cuda"), ints(np.zeros((6, 4))), ints(np.zeros((6, 4)))
    stream = torch.cuda.Stream()
    ctx = hip.Context(0)
    ctx.use_stream(stream)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        hip.beam_select(ctx, logits, scores, *out, workspace, settle=True)
    for seed in range(4):
        logits.copy_(normal(seed, 6, 4, 40000, scale=2.0))
        scores.copy_(running(seed + 50, 6, 4))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        held = [t.clone() for t in out]
        want = check(gpu, workspace, logits, scores, 4, settle=True)
        assert all(torch.equal(a, b) for a, b in zip(held, want))
    ctx.synchronize()
    ctx.close()


def test_two_contexts_on_two_streams(gpu):
    """Calls that may run at once, each with a workspace of its own."""
    made = []
    for i in range(2):
        stream = torch.cuda.Stream()
        ctx = hip.Context(0)
        ctx.use_stream(stream)
        made.append((ctx, hip.PagedWorkspace(ctx), normal(i, 8, 4, 60000, scale=2.0), running(i, 8, 4),
                     (torch.zeros(8, 8, device="cuda"), ints(np.zeros((8, 8))), ints(np.zeros((8, 8))))))
    torch.cuda.synchronize()
    for _ in range(20):
        for ctx, w, logits, scores, out in made:
            hip.beam_select(ctx, logits, scores, *out, w)
    torch.cuda.synchronize()
    for ctx, w, logits, scores, out in made:
        want = check(gpu, w, logits, scores, 8)
        assert all(torch.equal(a, b) for a, b in zip(out, want))
        w.close()
        ctx.close()


def test_select_refusals(gpu, workspace):
    n, k, v = 2, 3, 50
    good = dict(logits=normal(1, n, k, v), scores=running(1, n, k), out_scores=torch.zeros(n, 4, device="cuda"),
                parents=ints(np.zeros((n, 4))), tokens=ints(np.zeros((n, 4))), workspace=workspace)
    hip.beam_select(gpu, **good)
    for change in [dict(logits=normal(1, n, k, v).double()), dict(logits=normal(1, n * k, v)),
                   dict(logits=normal(1, n, k, v).cpu()), dict(logits=normal(1, n, v, k).transpose(1, 2)),
                   dict(logits=normal(1, n, 65, v)), dict(scores=running(1, n, k + 1)),
                   dict(scores=running(1, n, k).double()), dict(scores=running(1, n, k).cpu()),
                   dict(out_scores=torch.zeros(n, device="cuda")), dict(out_scores=torch.zeros(n + 1, 4, device="cuda")),
                   dict(parents=ints(np.zeros((n, 3)))), dict(parents=ints(np.zeros((n, 4))).long()),
                   dict(tokens=ints(np.zeros((n, 4))).cpu()), dict(settle=True), dict(ended_token=1 << 32),
                   dict(ended_token=-1), dict(weights=torch.ones(n, k, device="cuda").half()),
                   dict(weights=torch.ones(n, k + 1, device="cuda")), dict(ended=torch.ones(n, k, device="cuda")),
                   dict(logits=normal(1, n, k, 0)),
                   dict(out_scores=torch.zeros(n, 129, device="cuda"), parents=ints(np.zeros((n, 129))),
                        tokens=ints(np.zeros((n, 129))))]:
        with pytest.raises(hip.HipError) as e:
            hip.beam_select(gpu, **{**good, **change})
        assert e.value.status == hip.INVALID_ARGUMENT
    hip.beam_select(gpu, **{**good, "logits": normal(1, 0, k, v), "scores": running(1, 0, k),
                            "out_scores": torch.zeros(0, 4, device="cuda"), "parents": ints(np.zeros((0, 4))),
                            "tokens": ints(np.zeros((0, 4)))})
    gpu.synchronize()


# ---- states that follow their parents -----------------------------------------------

def reordered(t, parents):
    """What the rows become: parents that are no beam leave the row."""
    k = t.shape[1]
    p = parents.long().cpu().numpy()
    own = np.broadcast_to(np.arange(k), p.shape)
    p = np.where((p >= 0) & (p < k), p, own)
    return t[torch.arange(t.shape[0], device="cuda")[:, None], torch.tensor(p, device="cuda")]


def parent_maps(n, k, seed):
    g = np.random.default_rng(seed)
    yield g.integers(0, k, (n, k))
    yield np.stack([g.permutation(k) for _ in range(n)])          # cycles
    yield np.tile(np.arange(k), (n, 1))                           # nothing moves
    yield np.tile((np.arange(k) + 1) % k, (n, 1))
    yield np.where(g.random((n, k)) < 0.3, -1, g.integers(0, k + 2, (n, k)))  # parents that are none


@pytest.mark.parametrize("k", [1, 2, 3, 4, 5, 8, 16, 17, 33, 64])
@pytest.mark.parametrize("n", [1, 5])
def test_reorder_maps(gpu, n, k):
    for seed, parents in enumerate(parent_maps(n, k, k)):
        arrays = [normal(1, n, k, 300), normal(2, n, k, 7, 5, kind="bf16"), normal(3, n, k, 1, kind="f16"),
                  torch.randint(0, 1 << 30, (n, k, 1001), dtype=torch.int32, device="cuda"), normal(4, n, k, 2048)]
        want = [reordered(t, ints(parents)) for t in arrays]
        hip.reorder_rows(gpu, hip.StateRows(gpu, arrays), ints(parents))
        for got, w in zip(arrays, want):
            assert torch.equal(got, w), (seed, got.shape)


@pytest.mark.parametrize("dtype,row", [(torch.uint8, 1), (torch.uint8, 3), (torch.uint8, 4097), (torch.int16, 5),
                                       (torch.int64, 1), (torch.float64, 33), (torch.int32, 3), (torch.uint8, 70003)])
def test_reorder_rows_of_any_size(gpu, dtype, row):
    n, k = 3, 6
    t = torch.randint(0, 100, (n, k, row), device="cuda").to(dtype)
    for parents in parent_maps(n, k, 1):
        want = reordered(t, ints(parents))
        hip.reorder_rows(gpu, hip.StateRows(gpu, [t]), ints(parents))
        assert torch.equal(t, want)


def test_reorder_strides_and_what_lies_between(gpu):
    n, k = 4, 5
    for shift, size in [(0, 64), (1, 61), (3, 17), (4, 60)]:
        for order in (False, True):
            whole = normal(1, n, k, 100) if not order else normal(1, k, n, 100)
            view = whole[:, :, shift:shift + size]
            view = view.transpose(0, 1) if order else view
            keep = whole.clone()
            parents = ints(np.random.default_rng(2).integers(0, k, (n, k)))
            want = reordered(view, parents)
            hip.reorder_rows(gpu, hip.StateRows(gpu, [view]), parents)
            assert torch.equal(view, want)
            kept = keep[:, :, shift:shift + size]
            (kept.transpose(0, 1) if order else kept).copy_(want)
            assert torch.equal(whole, keep)


def test_reorder_many_arrays_and_none(gpu):
    n, k = 2, 4
    parents = ints([[1, 1, 0, 3], [2, 2, 2, 2]])
    arrays = [normal(i, n, k, 10 + i) for i in range(150)] + [normal(1, n, k, 0)]
    want = [reordered(t, parents) for t in arrays]
    hip.reorder_rows(gpu, hip.StateRows(gpu, arrays), parents)
    assert all(torch.equal(a, b) for a, b in zip(arrays, want))
    hip.reorder_rows(gpu, hip.StateRows(gpu, []), ints(np.zeros((0, 1))))
    empty = torch.zeros(0, 4, 10, device="cuda")
    hip.reorder_rows(gpu, hip.StateRows(gpu, [empty]), ints(np.zeros((0, 4))))
    gpu.synchronize()


def test_reorder_past_32_bits(gpu):
    """Rows more than 2^32 bytes apart."""
    whole = torch.empty((1 << 31) * 3 + 4096, dtype=torch.uint8, device="cuda")
    view = whole.as_strided((1, 3, 3000), (0, 1 << 31, 1))
    view.copy_(torch.randint(0, 255, (1, 3, 3000), device="cuda"))
    want = reordered(view, ints([[2, 0, 1]]))
    hip.reorder_rows(gpu, hip.StateRows(gpu, [view]), ints([[2, 0, 1]]))
    assert torch.equal(view, want)


def test_reorder_captured(gpu):
    arrays = [normal(1, 3, 4, 5000), normal(2, 3, 4, 33, kind="bf16")]
    parents = ints(np.zeros((3, 4)))
    stream = torch.cuda.Stream()
    ctx = hip.Context(0)
    ctx.use_stream(stream)
    rows = hip.StateRows(ctx, arrays)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        hip.reorder_rows(ctx, rows, parents)
    for seed in range(4):
        parents.copy_(ints(np.random.default_rng(seed).integers(0, 4, (3, 4))))
        for i, t in enumerate(arrays):
            t.copy_(normal(seed + i, *t.shape).to(t.dtype))
        want = [reordered(t, parents) for t in arrays]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(arrays, want))
    ctx.close()


def test_reorder_refusals(gpu):
    t = normal(1, 2, 4, 10)
    for arrays in ([t, normal(1, 2, 3, 10)], [normal(1, 8)], [t.cpu()], [normal(1, 2, 4, 10, 10).transpose(2, 3)]):
        with pytest.raises(hip.HipError):
            hip.StateRows(gpu, arrays)
    rows = hip.StateRows(gpu, [t])
    for parents in (ints(np.zeros((2, 3))), ints(np.zeros((2, 4))).long(), ints(np.zeros((2, 4))).cpu()):
        with pytest.raises(hip.HipError):
            hip.reorder_rows(gpu, rows, parents)
    for broadcast in (normal(1, 2, 1, 10).expand(2, 4, 10), normal(1, 1, 4, 10).expand(2, 4, 10)):
        with pytest.raises(hip.HipError, match="overlap"):
            hip.reorder_rows(gpu, hip.StateRows(gpu, [broadcast]), ints(np.zeros((2, 4))))
    with pytest.raises(hip.HipError, match="beams"):
        hip.reorder_rows(gpu, hip.StateRows(gpu, [normal(1, 1, 65, 3)]), ints(np.zeros((1, 65))))
