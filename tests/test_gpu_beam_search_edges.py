"""serving.BeamSearch where a call can go wrong beside its own sizes: streams other than
the current one, threads."""
import threading

import pytest
import torch

import small_model
from adi_amd import hip, serving

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
