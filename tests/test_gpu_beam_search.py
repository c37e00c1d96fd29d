"""A beam search's steps as they are used together: over the whole model
(selection, states that follow their parents, decoding, direct and replayed), and
over the paged full-attention layer (admission, fork, append and attention, a
pool compacted and a request moved to another between steps).

The model's search is compared with the same search in numpy over states that are
copied row by row: the same decode calls on the same states give the same bits,
so parents, tokens and lengths are equal; scores are sums of floats each rounded once
a step (half a step of the running sum) behind logarithms good to 2^-32."""
import math

import numpy as np
import pytest
import torch

import small_model
from adi_amd import hip, serving
from conftest import max_rel_error
from test_gpu_pages import ints, pool_of

pytestmark = pytest.mark.gpu

VOCAB = small_model.VOCAB


@pytest.fixture(scope="module")
def parts(gpu):
    return small_model.build(gpu, seed=72)


def plain_search(gpu, model, prompt, steps, beams, penalty, stop, masked, capacity):
    """(hypotheses as (tokens, sum, score, ended), best first) with every state
    copied and every candidate compared on the host, in double."""
    states = hip.BeamStates(gpu, model, beams, capacity)
    logits = torch.empty((beams, VOCAB), device="cuda")
    hip.prefill(gpu, model, prompt, states.sequences[0], logits[0])
    rows = [dict(tokens=[], total=0.0, ended=False)] + [None] * (beams - 1)
    position = len(prompt)
    for n in range(1, steps + 1):
        logits[:, masked] = torch.finfo(torch.float32).min
        x = logits.double().cpu().numpy()
        found = []
        for b, r in enumerate(rows):
            if r is None:
                continue
            if r["ended"]:
                found.append((-r["total"] * np.float32(len(r["tokens"])) ** -penalty, b, 0, None, r["total"]))
                continue
            lse = x[b].max() + math.log(np.exp(x[b] - x[b].max()).sum())
            for t in np.argsort(-x[b], kind="stable")[:beams]:
                total = r["total"] + (x[b, t] - lse)
                found.append((-total * n ** -penalty, b, -x[b, t], int(t), total))
        found.sort()
        best = found[:beams]
        parents = [f[1] for f in best]
        free = iter([b for b in range(beams) if b not in parents])
        new = [None] * beams
        source = list(range(beams))
        for i, f in enumerate(best):
            place = f[1] if parents.index(f[1]) == i else next(free)
            r = rows[f[1]]
            total = float(np.float32(f[4]))
            new[place] = r if f[3] is None else dict(tokens=r["tokens"] + [f[3]], total=total, ended=f[3] in stop)
            source[place] = f[1]
        rows = new
        for t in states.arrays:
            t.copy_(t[:, source].clone())
        if n == steps or all(r is None or r["ended"] for r in rows):
            break
        for s in states.sequences:
            s.struct.position = position
        tokens = [0 if r is None else (stop[0] if r["ended"] else r["tokens"][-1]) for r in rows]
        hip.decode_batch(gpu, model, tokens, states.sequences, logits)
        position += 1
    out = [(r["tokens"][:-1] if r["ended"] else r["tokens"], r["total"], r["total"] / len(r["tokens"]) ** penalty,
            r["ended"]) for r in rows if r is not None]
    return sorted(out, key=lambda h: -h[2])


@pytest.mark.parametrize("replay", [False, True])
@pytest.mark.parametrize("beams,penalty,stop,masked", [
    (1, 0.0, [], []), (4, 0.0, [], [0, 5, 511]), (4, 1.0, [3, 77, 200, 301, 410], [1]), (7, 0.6, list(range(0, 512, 9)), [])])
def test_search_over_the_model(gpu, parts, replay, beams, penalty, stop, masked):
    capacity, steps = 24, 9
    search = serving.BeamSearch(gpu, parts["two"], beams, capacity, penalty, stop, masked, replay_steps=replay)
    try:
        for prompt in ([3, 9, 40], [7], [5, 1, 4, 1, 5, 9, 2, 6]):
            got = search.search(prompt, steps)
            want = plain_search(gpu, parts["two"], prompt, steps, beams, penalty, stop, masked, capacity)
            assert [h.tokens for h in got] == [w[0] for w in want]
            assert [h.finish_reason == "stop_token" for h in got] == [w[3] for w in want]
            for h, w in zip(got, want):
                # the sums differ by their logarithms, 2^-32 each (the tokens' own
                # may be far smaller: sums of 1e-6 occur), and by a rounding where
                # that decides one: a step of the sum each; the score's quotient
                # adds its own
                bound = steps * (2.0 ** -23 * abs(w[1]) + 2.0 ** -32)
                assert abs(h.log_probability - w[1]) <= bound
                assert abs(h.score - w[2]) <= bound + 2.0 ** -23 * abs(w[2])
            assert not set(masked) & {t for h in got for t in h.tokens}
    finally:
        search.close()


def test_search_scores_are_the_oracles(gpu, oracle, parts):
    """The hypotheses' log-probabilities from the oracle, run token by token: logits
    within 1e-3 of their largest, so a token's log-probability within twice that."""
    search = serving.BeamSearch(gpu, parts["one"], 3, 16)
    try:
        for h in search.search([3, 9, 40], 4):
            o = small_model.OracleSequence(parts, 16)
            for t in [3, 9, 40]:
                logits = o.step(oracle, t)
            total, bound = 0.0, 0.0
            for t in h.tokens:
                x = logits.astype(np.float64)
                total += x[t] - (x.max() + math.log(np.exp(x - x.max()).sum()))
                bound += 2e-3 * np.abs(x).max()
                logits = o.step(oracle, t)
            assert abs(h.log_probability - total) <= bound
    finally:
        search.close()


def test_one_beam_is_the_greedy_choice(gpu, parts):
    model = parts["one"]
    search = serving.BeamSearch(gpu, model, 1, 16)
    s, logits, tokens = hip.Sequence(model, 16), torch.empty(1, VOCAB, device="cuda"), []
    hip.prefill(gpu, model, [3, 9], s, logits[0])
    for _ in range(6):
        picked = torch.empty(1, dtype=torch.int32, device="cuda")
        hip.argmax_rows(gpu, logits, 1, VOCAB, picked)
        tokens.append(int(picked))
        hip.decode_batch(gpu, model, tokens[-1:], [s], logits)
    assert [h.tokens for h in search.search([3, 9], 6)] == [tokens]
    search.close()


def test_search_refusals(gpu, parts):
    model = parts["one"]
    for change in [dict(beams=0), dict(beams=65), dict(capacity=0), dict(capacity=1 << 30), dict(stop_tokens=[VOCAB]),
                   dict(masked_tokens=[-1])]:
        with pytest.raises(serving.GenerationError):
            serving.BeamSearch(gpu, model, **{**dict(beams=2, capacity=8), **change})
    search = serving.BeamSearch(gpu, model, 2, 8)
    for prompt, steps in (([], 2), ([1, 2], 0), ([1] * 7, 2)):
        with pytest.raises(serving.GenerationError):
            search.search(prompt, steps)
    assert len(search.search([1] * 7, 1)) == 2
    search.close()


# ---- the paged layer -------------------------------------------------------------------

@pytest.fixture(scope="module")
def layer(gpu):
    from adi_amd import synthetic as syn
    rng = syn.rng_for(44, 256)
    tlut = syn.ne_tlut(rng)
    host = syn.full_attention(rng, 256, tlut)
    return hip.upload_full_attention(gpu, host, gpu.ne_codebook(tlut))


def test_search_over_the_paged_layer(gpu, layer):
    """Two requests of three beams over two layers' caches that share a pool (the
    second layer reads the first's rows), each step compared with the layer over every
    beam's own contiguous cache: outputs to 1e-4 of the largest, the layer tests'
    own bound. Between steps the pool is compacted, and once moved to another."""
    page, pages, columns, beams, requests = 16, 60, 6, 3, 2
    rows, hidden = beams * requests, 256
    workspace = hip.PagedWorkspace(gpu)
    g = np.random.default_rng(5)

    def made():
        return [torch.full((pages, page, 2, 256), math.nan, device="cuda") for _ in range(4)]

    tensors, count, live = made(), ints(np.zeros(pages)), ints([0])
    lengths, table = ints(np.zeros(rows)), ints(np.full((rows, columns), -1))
    # every row's own caches, [layer][row] of keys and values
    own = [[[torch.zeros(96, 2, 256, device="cuda") for _ in range(2)] for _ in range(rows)] for _ in range(2)]
    held = np.zeros(rows, int)

    def step(parents, added):
        nonlocal own, held
        parents, added = np.asarray(parents), np.asarray(added)
        pool = pool_of(gpu, tensors, count)
        offsets = np.concatenate([[0], np.cumsum(added)])
        total = int(offsets[-1])
        batch = hip.PagedBatch(gpu, ints(offsets), lengths, table, total, int(added.max()), columns * page)
        hip.paged_fork(gpu, pool, batch, ints(parents).view(requests, beams), workspace)
        source = [s // beams * beams + p if p >= 0 else None for s, p in enumerate(parents)]
        held = np.array([0 if q is None else held[q] for q in source])
        own = [[[t.clone() for t in each[q]] if q is not None else [torch.zeros_like(t) for t in each[0]]
                for q in source] for each in own]
        x = torch.tensor(g.normal(size=(total, hidden)), dtype=torch.float32, device="cuda")
        mine = theirs = x / x.square().mean(-1, keepdim=True).sqrt()
        for i in range(2):
            out = torch.empty_like(mine)
            hip.full_attention_paged(gpu, layer, pool.caches[i], batch, mine, out, workspace)
            want = torch.empty_like(theirs)
            for s in range(rows):
                if added[s]:
                    a, b = offsets[s], offsets[s + 1]
                    to = torch.empty(b - a, hidden, device="cuda")
                    hip.full_attention_prefill(gpu, layer, int(held[s]), int(added[s]), theirs[a:b].contiguous(), to,
                                               *own[i][s], 96)
                    want[a:b] = to
            assert max_rel_error(out.cpu().numpy(), want.cpu().numpy()) <= 1e-4, i
            mine = theirs = want  # (so that a layer's differences do not add up)
        held = held + added

    step([-1] * 6, [37, 0, 0, 16, 0, 0])
    step([0] * 6, [1] * 6)
    for i in range(14):
        step(g.integers(0, beams, rows), [1] * 6)
        if i % 4 == 2:
            hip.paged_compact(gpu, pool_of(gpu, tensors, count), lengths, table, live, workspace)
            n = int(live)
            assert int((count[:n] > 0).sum()) == n and int(count[n:].abs().sum()) == 0
        if i == 6:  # to another pool, the pages renumbered
            numbers = g.permutation(pages)
            fresh, moved = made(), torch.zeros_like(count)
            hip.paged_copy(gpu, pool_of(gpu, tensors), pool_of(gpu, fresh), ints(np.arange(pages)), ints(numbers))
            renamed = ints(numbers)
            moved[renamed.long()] = count
            table = torch.where(table >= 0, renamed[table.clamp(min=0).long()], table)
            tensors, count = fresh, moved
    step([-1, -1, -1, 0, 1, 2], [20, 0, 0, 1, 1, 1])  # one request ends, another begins in its rows
    step([0, 0, -1, 2, 2, 2], [1, 1, 0, 1, 1, 1])
    hip.paged_fork(gpu, pool_of(gpu, tensors, count), hip.PagedBatch(gpu, ints(np.zeros(7)), lengths, table, 0, 0, 96),
                   ints(np.full((2, 3), -1)), workspace)
    assert int(count.abs().sum()) == 0 and int(lengths.abs().sum()) == 0
    gpu.synchronize()
    workspace.close()
