"""serving.BeamSearch where a call can go wrong beside its own sizes: streams other than
the current one, threads, more beams than tokens, many beams, and positions past those
that a recorded step covers (512)."""
import math
import threading

import pytest
import torch

import small_model
from adi_amd import hip, serving
from test_gpu_beam_search import plain_search

pytestmark = pytest.mark.gpu

VOCAB = small_model.VOCAB
PROMPTS = ([3, 9, 40], [7], [5, 1, 4, 1, 5, 9, 2, 6])


@pytest.fixture(scope="module")
def parts(gpu):
    return small_model.build(gpu, seed=72)


def searched(ctx, model, replay, **change):
    search = serving.BeamSearch(ctx, model, 4, 24, replay_steps=replay, **change)
    try:
        return [search.search(p, 8) for p in PROMPTS]
    finally:
        search.close()


@pytest.mark.parametrize("replay", [False, True])
def test_search_on_a_stream_of_its_own(gpu, parts, replay):
    """A context of another stream than the thread's current one, in this thread and
    in a worker's, gives what the current one's gives."""
    change = dict(length_penalty=0.7, stop_tokens=[3, 77, 200, 301, 410], masked_tokens=[0, 5])
    want = searched(gpu, parts["two"], replay, **change)
    ctx = hip.Context(0)
    ctx.use_stream(torch.cuda.Stream())
    torch.cuda.synchronize()
    assert searched(ctx, parts["two"], replay, **change) == want
    with torch.cuda.stream(torch.cuda.Stream()):
        assert searched(ctx, parts["two"], replay, **change) == want
    found = []
    worker = threading.Thread(target=lambda: found.append(searched(ctx, parts["two"], replay, **change)))
    worker.start()
    worker.join()
    assert found == [want]
    ctx.close()


@pytest.mark.parametrize("replay", [False, True])
def test_search_after_the_context_changed_its_stream(gpu, parts, replay):
    ctx = hip.Context(0)
    search = serving.BeamSearch(ctx, parts["one"], 3, 16, replay_steps=replay)
    want = search.search([3, 9], 6)
    for _ in range(2):
        ctx.use_stream(torch.cuda.Stream())
        assert search.search([3, 9], 6) == want
    ctx.use_stream(torch.cuda.default_stream())
    assert search.search([3, 9], 6) == want
    search.close()
    ctx.close()


@pytest.mark.parametrize("replay", [False, True])
@pytest.mark.parametrize("beams,allowed,steps", [(4, [9], 5), (4, [9, 200], 1), (4, [9, 200], 5), (7, [1, 2, 300], 2),
                                                 (64, [1, 2, 300], 3)])
def test_more_beams_than_allowed_tokens(gpu, parts, replay, beams, allowed, steps):
    """Masked tokens are never chosen: as many hypotheses as the others make, all
    different, and where those are all there are, their probabilities sum to 1."""
    masked = [t for t in range(VOCAB) if t not in allowed]
    search = serving.BeamSearch(gpu, parts["two"], beams, 24, masked_tokens=masked, replay_steps=replay)
    found = search.search([3, 9, 40], steps)
    search.close()
    assert len(found) == min(beams, len(allowed) ** steps)
    assert all(len(h.tokens) == steps and set(h.tokens) <= set(allowed) for h in found)
    assert len({tuple(h.tokens) for h in found}) == len(found)
    if len(allowed) == 1:
        # one token has all of the probability: a sum of logarithms good to 2^-32
        assert abs(found[0].log_probability) <= steps * 2.0 ** -32
    elif beams >= len(allowed) ** steps:
        # all sequences there are: their probabilities sum to 1, each score a sum of
        # floats rounded once a step (2^-24 of it) behind logarithms good to 2^-32
        total = sum(math.exp(h.log_probability) for h in found)
        worst = max(abs(h.log_probability) for h in found)
        assert abs(total - 1.0) <= 2.0 * steps * (2.0 ** -24 * worst + 2.0 ** -32)


@pytest.mark.parametrize("penalty", [42.0, -42.0])
def test_penalties_at_a_floats_edge(gpu, parts, penalty):
    """8^42 is 2^126; one token more is refused before the prompt is run."""
    search = serving.BeamSearch(gpu, parts["one"], 4, 24, penalty, stop_tokens=list(range(0, VOCAB, 5)))
    found = search.search([3, 9], 8)
    assert len(found) == 4
    for h in found:
        length = len(h.tokens) + (h.finish_reason == "stop_token")
        assert h.score == h.log_probability / float(length) ** penalty
    with pytest.raises(serving.GenerationError, match="length_penalty"):
        search.search([3, 9], 9)
    search.close()


@pytest.mark.parametrize("replay", [False, True])
@pytest.mark.parametrize("beams,prompt,steps,penalty,stop", [(4, 507, 12, 0.0, []), (3, 1021, 8, 1.0, [3, 77, 200]),
                                                             (64, 5, 6, 0.5, list(range(0, VOCAB, 9)))])
def test_long_prompts_and_many_beams(gpu, parts, replay, beams, prompt, steps, penalty, stop):
    """The same as the search on the host; scores as there."""
    tokens = [(7 * i * i + 3 * i) % VOCAB for i in range(prompt)]
    capacity = prompt + steps
    search = serving.BeamSearch(gpu, parts["one"], beams, capacity, penalty, stop, replay_steps=replay)
    got = search.search(tokens, steps)
    search.close()
    want = plain_search(gpu, parts["one"], tokens, steps, beams, penalty, stop, [], capacity)
    assert [h.tokens for h in got] == [w[0] for w in want]
    assert [h.finish_reason == "stop_token" for h in got] == [w[3] for w in want]
    for h, w in zip(got, want):
        bound = steps * (2.0 ** -23 * abs(w[1]) + 2.0 ** -32)
        assert abs(h.log_probability - w[1]) <= bound
        assert abs(h.score - w[2]) <= bound + 2.0 ** -23 * abs(w[2])
