"""serving.BeamSearch without a GPU: stand-ins for the library's calls and for torch's
streams, over torch's own operations on the CPU."""
import contextlib
import types

import pytest
import torch

from adi_amd import hip, serving

VOCAB, BEAMS, CAPACITY = 11, 3, 16


class Stream:
    def __init__(self, name):
        self.name, self.waits = name, []

    def wait_stream(self, other):
        self.waits.append(other.name)


class Torch:
    """torch with streams that only note which is the current one, every use of it
    noted with its stream, and tensors on the CPU."""

    def __init__(self):
        self.default, self.uses = Stream("default"), []
        self.current = self.default
        self.cuda = types.SimpleNamespace(current_stream=lambda device=None: self.current, stream=self._stream)

    @contextlib.contextmanager
    def _stream(self, stream):
        before, self.current = self.current, stream
        try:
            yield
        finally:
            self.current = before

    def note(self, what):
        self.uses.append((what, self.current.name))

    def __getattr__(self, name):
        held = getattr(torch, name)
        if not callable(held) or isinstance(held, type):
            return held

        def call(*args, **kind):
            self.note(name)
            kind.pop("device", None)
            return held(*args, **kind)
        return call


class Search:
    """A search whose model gives the same logits everywhere."""

    def __init__(self, monkeypatch, stream="side", logits=None):
        self.torch = Torch()
        self.ctx = types.SimpleNamespace(torch=self.torch, device=0, stream=Stream(stream), handle=None)
        self.model = types.SimpleNamespace(struct=types.SimpleNamespace(context=1 << 20), vocabulary=VOCAB)
        self.logits = torch.linspace(0, 1, VOCAB) if logits is None else logits
        self.prefills = self.steps = 0
        note = self.torch.note

        class States:
            def __init__(own, ctx, model, beams, capacity, more=()):
                note("states")
                own.sequences, own.more = [None] * beams, more

            def start(own):
                note("start")

            def follow(own, parents, position):
                note("follow")
                rows = [p if p >= 0 else b for b, p in enumerate(parents[0].tolist())]
                for t in own.more:
                    t[0] = t[0, rows].clone()

        def prefill(ctx, model, prompt, sequence, logits, ubatch):
            note("prefill")
            self.prefills += 1
            logits.copy_(self.logits)

        def decode(ctx, model, tokens, sequences, logits):
            note("decode")
            self.steps += 1
            logits.copy_(self.logits.expand_as(logits))

        def select(ctx, logits, scores, out_scores, parents, tokens, workspace, weights=None, ended=None,
                   ended_token=0, settle=False):
            note("select")
            self.weights = weights
            found = []
            for b in range(BEAMS):
                if scores[0, b] == -torch.inf:
                    continue
                w = 1.0 if weights is None else float(weights[0, b])
                if ended is not None and ended[0, b]:
                    found.append((-w * float(scores[0, b]), b, ended_token, float(scores[0, b])))
                    continue
                each = scores[0, b].double() + logits[0, b].double().log_softmax(0)
                found += [(-w * float(each[v]), b, v, float(each[v])) for v in range(VOCAB)
                          if logits[0, b, v] > -torch.inf]
            found.sort()
            for i in range(BEAMS):
                _, b, v, s = found[i] if i < len(found) else (0, -1, -1, -torch.inf)
                out_scores[0, i], parents[0, i], tokens[0, i] = s, b, v

        monkeypatch.setattr(hip, "BeamStates", States)
        monkeypatch.setattr(hip, "PagedWorkspace", lambda ctx: types.SimpleNamespace(close=lambda: None))
        monkeypatch.setattr(hip, "prefill", prefill)
        monkeypatch.setattr(hip, "decode_batch", decode)
        monkeypatch.setattr(hip, "beam_select", select)

    def make(self, **change):
        return serving.BeamSearch(self.ctx, self.model, **{**dict(beams=BEAMS, capacity=CAPACITY, replay_steps=False),
                                                           **change})


def test_all_work_is_on_the_contexts_stream(monkeypatch):
    """Whichever stream the thread's current one is: the constructor's fills, the
    search's own operations and the library's calls, behind the caller's work."""
    s = Search(monkeypatch)
    search = s.make(stop_tokens=[4], masked_tokens=[2], length_penalty=0.7)
    assert s.torch.uses and {stream for _, stream in s.torch.uses} == {"side"}
    assert s.ctx.stream.waits == ["default"]
    s.torch.uses.clear()
    with s.torch.cuda.stream(Stream("worker")):
        assert len(search.search([1, 2], 4)) == BEAMS
        assert s.torch.current.name == "worker"
    assert {"start", "prefill", "select", "follow", "decode"} <= {what for what, _ in s.torch.uses}
    assert {stream for _, stream in s.torch.uses} == {"side"}
    assert s.ctx.stream.waits == ["default", "worker"]


def test_a_context_given_another_stream(monkeypatch):
    """The search goes to the new stream, behind what the old one holds."""
    s = Search(monkeypatch)
    search = s.make()
    s.ctx.stream = Stream("other")
    s.torch.uses.clear()
    search.search([1], 2)
    assert {stream for _, stream in s.torch.uses} == {"other"}
    assert sorted(s.ctx.stream.waits) == ["default", "side"]


def test_one_stream_waits_for_nothing(monkeypatch):
    s = Search(monkeypatch)
    s.ctx.stream = s.torch.default
    search = s.make()
    search.search([1], 2)
    assert s.torch.default.waits == []
    assert {stream for _, stream in s.torch.uses} == {"default"}


@pytest.mark.parametrize("allowed,steps", [([5], 3), ([5, 9], 1), ([1, 2], 2), ([], 2)])
def test_masked_tokens_are_never_chosen(monkeypatch, allowed, steps):
    """Also where fewer are left than there are beams: as many hypotheses as the tokens
    make."""
    s = Search(monkeypatch)
    found = s.make(masked_tokens=[t for t in range(VOCAB) if t not in allowed]).search([1], steps)
    assert len(found) == min(BEAMS, len(allowed) ** steps)
    assert all(len(h.tokens) == steps and set(h.tokens) <= set(allowed) for h in found)
    assert len({tuple(h.tokens) for h in found}) == len(found)


@pytest.mark.parametrize("penalty", [float("nan"), float("inf"), -float("inf")])
def test_penalties_that_are_not_finite_are_refused(monkeypatch, penalty):
    with pytest.raises(serving.GenerationError, match="finite"):
        Search(monkeypatch).make(length_penalty=penalty)


@pytest.mark.parametrize("sign", [1, -1])
def test_penalties_that_no_float_holds_are_refused(monkeypatch, sign):
    """Before the prompt is run, and only for as many tokens as make them so: 8^42 is
    2^126, of which a float and its inverse are normal numbers."""
    s = Search(monkeypatch)
    search = s.make(length_penalty=42.0 * sign)
    with pytest.raises(serving.GenerationError, match="length_penalty"):
        search.search([1], 9)
    assert s.prefills == 0
    assert len(search.search([1], 8)) == BEAMS
    assert s.prefills == 1 and bool(torch.isfinite(s.weights).all()) and bool((s.weights >= 2.0 ** -126).all())
    assert len(s.make(length_penalty=1e30 * sign).search([1], 1)) == BEAMS


def test_a_closed_search_is_refused(monkeypatch):
    s = Search(monkeypatch)
    search = s.make()
    search.close()
    with pytest.raises(serving.GenerationError, match="closed"):
        search.search([1], 2)
    assert s.prefills == 0
    search.close()
