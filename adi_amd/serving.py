"""Continuous batching on the device: the reference's ContinuousBatcher
(src/generation.cpp:343-660, include/adi/generation.hpp:75-95) over the
library's adi_hip_batcher, with token ids in place of text (the tokenizer
and chat template stay with the caller).

A worker thread runs the loop: while requests are pending or active it calls
adi_hip_batcher_step, one iteration of the reference's loop (admit the oldest
pending request by prefilling its prompt, sample every active sequence,
finish on a stop token or the output limit, decode the rest in one batched
step). While the same sequences keep stepping, their decode step is
recorded once as a HIP graph and replayed (replay_steps=False launches every
step directly; both give the same bits). generate() submits a request and blocks until it finishes, passing
each new token to `token_callback` as it appears and cancelling the request
when `cancelled()` turns true, as generate_from_prompt does. The worker owns
the context while the batcher runs: other work must not use it meanwhile."""
from __future__ import annotations

import contextlib
import ctypes as C
import math
import threading
import time
from dataclasses import dataclass
from functools import partial
from typing import Callable, Optional, Sequence

from . import hip

PENDING, RUNNING, STOP_TOKEN, LENGTH, FAILED = 0, 1, 2, 3, 4


@dataclass
class GenerationResult:
    """adi::GenerationResult (include/adi/generation.hpp:29-38) with token
    ids in place of text."""
    tokens: list
    input_tokens: int
    output_tokens: int
    finish_reason: str  # "stop_token" or "length"
    prefill_seconds: float
    decode_seconds: float


class GenerationError(RuntimeError):
    pass


class ContinuousBatcher(hip._Owner):
    def __init__(self, ctx: hip.Context, model: hip.Model, max_batch: int = 16,
                 capacity: int = 4096, prefill_ubatch: int = 128,
                 stop_tokens: Sequence[int] = (), masked_tokens: Sequence[int] = (),
                 start: bool = True, replay_steps: bool = True):
        self.handle, self._thread = None, None
        self.ctx, self.model = ctx, model
        hip.release_dropped()
        stop = (hip.u32 * max(len(stop_tokens), 1))(*stop_tokens)
        masked = (hip.u32 * max(len(masked_tokens), 1))(*masked_tokens)
        options = hip.BatcherOptions(max_batch, capacity, prefill_ubatch, stop, len(stop_tokens),
                                     masked, len(masked_tokens), 0 if replay_steps else 1)
        handle = hip.vp()
        ctx.check(ctx.lib.adi_hip_batcher_create(ctx.handle, C.byref(model.struct),
                                                 C.byref(options), C.byref(handle)))
        self.handle = handle
        ctx._users.add(handle.value)
        self._cond = threading.Condition()
        self._stop = False
        self._work = 0          # requests pending or active, as of the last step
        self._submitted = 0     # submissions so far
        self._steps = 0
        self._failure: Optional[hip.HipError] = None
        if start:
            self._thread = threading.Thread(target=self._run, name="adi-batcher", daemon=True)
            self._thread.start()

    # -- the worker loop (Impl::run, src/generation.cpp:540-660) --
    def _run(self):
        while True:
            with self._cond:
                idle = self._work == 0
                while not self._stop and self._work == 0:
                    self._cond.wait()
                if self._stop:
                    return
            if idle:
                # a short window makes simultaneous arrivals deterministic
                # without imposing meaningful latency on a lone request
                time.sleep(0.002)
            try:
                self.step()
            except hip.HipError as error:  # the decode step failed its requests
                self._failure = error
            with self._cond:
                self._cond.notify_all()

    def step(self) -> int:
        """One loop iteration; returns the requests still pending or active."""
        remaining = hip.u32()
        with self._cond:
            seen = self._submitted
        status = self.ctx.lib.adi_hip_batcher_step(self.handle, C.byref(remaining))
        with self._cond:
            # a request submitted during the step may be missing from its count
            self._work = remaining.value if self._submitted == seen else max(remaining.value, 1)
            self._steps += 1
            self._cond.notify_all()
        self.ctx.check(status)
        return remaining.value

    # -- requests --
    def submit(self, prompt: Sequence[int], max_output_tokens: Optional[int] = None,
               temperature: float = 0.7, top_p: float = 0.9, seed: int = 0) -> int:
        if max_output_tokens is not None and max_output_tokens <= 0:
            raise GenerationError("max_output_tokens must be positive")
        toks = (hip.u32 * max(len(prompt), 1))(*[int(t) for t in prompt])
        opts = hip.GenerationOptions(0 if max_output_tokens is None else max_output_tokens,
                                     temperature, top_p, seed)
        request = hip.u64()
        self.ctx.check(self.ctx.lib.adi_hip_batcher_submit(self.handle, toks, len(prompt),
                                                           C.byref(opts), C.byref(request)))
        with self._cond:
            self._submitted += 1
            self._work += 1
            self._cond.notify_all()
        return request.value

    def cancel(self, request: int) -> None:
        self.ctx.check(self.ctx.lib.adi_hip_batcher_cancel(self.handle, request))

    def status(self, request: int):
        """(state, tokens so far, RequestStatus)."""
        st = hip.RequestStatus()
        cap = 1 << 16
        buf = (hip.u32 * cap)()
        self.ctx.check(self.ctx.lib.adi_hip_batcher_status(self.handle, request, C.byref(st), buf,
                                                           cap))
        return st.state, list(buf[:min(st.output_tokens, cap)]), st

    def result(self, request: int) -> GenerationResult:
        """The finished request's result (its error raised if it failed);
        the request is released."""
        state, tokens, st = self.status(request)
        if state in (PENDING, RUNNING):
            raise GenerationError("request has not finished")
        error = self.ctx.lib.adi_hip_batcher_request_error(self.handle, request).decode()
        self.ctx.lib.adi_hip_batcher_release(self.handle, request)
        if state == FAILED:
            raise GenerationError(error)
        return GenerationResult(tokens, st.input_tokens, st.output_tokens,
                                "stop_token" if state == STOP_TOKEN else "length",
                                st.prefill_seconds, st.decode_seconds)

    def generate(self, prompt: Sequence[int], max_output_tokens: Optional[int] = None,
                 temperature: float = 0.7, top_p: float = 0.9, seed: int = 0,
                 token_callback: Optional[Callable[[int], None]] = None,
                 cancelled: Optional[Callable[[], bool]] = None) -> GenerationResult:
        """generate_from_prompt (src/generation.cpp:662-676) on token ids."""
        if self._thread is None:
            raise GenerationError("the batcher was created without its worker thread")
        request = self.submit(prompt, max_output_tokens, temperature, top_p, seed)
        sent = 0
        while True:
            with self._cond:
                self._cond.wait(timeout=0.05)
            state, tokens, _ = self.status(request)
            if token_callback is not None:
                try:
                    for t in tokens[sent:]:
                        token_callback(t)
                except BaseException:
                    self.cancel(request)  # Request::callback_failed
                    raise
                sent = len(tokens)
            if cancelled is not None and state in (PENDING, RUNNING) and cancelled():
                self.cancel(request)
            if state not in (PENDING, RUNNING):
                return self.result(request)
            if self._thread is not None and not self._thread.is_alive():
                raise GenerationError("continuous batcher stopped")

    def close(self) -> None:
        if self._thread is not None:
            with self._cond:
                self._stop = True
                self._cond.notify_all()
            self._thread.join()
            self._thread = None
        super().close()

    def _take(self) -> list:
        handle, self.handle = self.handle, None
        if not handle:
            return []
        return [partial(self.ctx.lib.adi_hip_batcher_destroy, handle), partial(self.ctx._users.discard, handle.value)]


@dataclass
class Hypothesis:
    """One result of a beam search: its tokens without the stop token, the sum of
    their log-probabilities (the stop token's included), and that divided by
    length^length_penalty, which results are ordered by."""
    tokens: list
    log_probability: float
    score: float
    finish_reason: str  # "stop_token" or "length"


class BeamSearch:
    """Beam search over the model, with token ids, beside the batcher's one token a
    row (sample_token, src/generation.cpp:161-225): each step takes the best
    `beams` of beams x vocabulary on the device (hip.beam_select), the decoder
    states follow their parents in place (hip.BeamStates), and the beams decode
    as a batch, recorded once as a HIP graph and replayed (replay_steps=False
    launches every step directly; both give the same bits). Beams that have ended stay as
    one candidate each; candidates are compared by sum / length^length_penalty. All
    work runs on the context's stream, whichever torch's current one is, behind what
    the caller's holds. One search at a time; the context must not be used otherwise
    meanwhile."""

    def __init__(self, ctx: hip.Context, model: hip.Model, beams: int = 4, capacity: int = 4096,
                 length_penalty: float = 0.0, stop_tokens: Sequence[int] = (), masked_tokens: Sequence[int] = (),
                 prefill_ubatch: int = 128, replay_steps: bool = True):
        if not 1 <= beams <= 64:
            raise GenerationError("beams must be 1 to 64")
        if not 1 <= capacity <= model.struct.context:
            raise GenerationError("capacity exceeds model context")
        if any(not 0 <= t < model.vocabulary for t in (*stop_tokens, *masked_tokens)):
            raise GenerationError("a stop or masked token is outside the vocabulary")
        if not math.isfinite(length_penalty):
            raise GenerationError("length_penalty must be finite")
        torch = ctx.torch
        self.ctx, self.model, self.beams, self.capacity = ctx, model, beams, capacity
        self.length_penalty, self.ubatch, self.replay_steps = float(length_penalty), prefill_ubatch, replay_steps
        self._graph: Optional[hip.DecodeGraph] = None
        self._made: Optional[object] = None  # the stream of the last work on what follows
        with self._on_stream():
            device = f"cuda:{ctx.device}"
            self._stop = torch.tensor(list(stop_tokens), dtype=torch.int32, device=device)
            self._ended_token = int(stop_tokens[0]) if len(stop_tokens) else 0
            self._masked = torch.tensor(list(masked_tokens), dtype=torch.int64, device=device)
            self._logits = torch.empty((1, beams, model.vocabulary), dtype=torch.float32, device=device)
            self._history = torch.zeros((1, beams, capacity), dtype=torch.int32, device=device)
            self._tokens = torch.zeros((1, beams), dtype=torch.int32, device=device)
            self._parents = torch.zeros((1, beams), dtype=torch.int32, device=device)
            self._scores = [torch.zeros((1, beams), dtype=torch.float32, device=device) for _ in range(2)]
            self._workspace = hip.PagedWorkspace(ctx)
            self._states = hip.BeamStates(ctx, model, beams, capacity, more=[self._history])

    @contextlib.contextmanager
    def _on_stream(self):
        """torch's current stream is the context's."""
        cuda, stream = self.ctx.torch.cuda, self.ctx.stream
        for before in (cuda.current_stream(self.ctx.device), self._made):
            if before is not None and before != stream:
                stream.wait_stream(before)
        self._made = stream
        with cuda.stream(stream):
            yield

    def _decode(self) -> None:
        if not self.replay_steps:
            hip.decode_batch(self.ctx, self.model, self._tokens[0].tolist(), self._states.sequences, self._logits)
            return
        if self._graph is None:
            self._graph = hip.DecodeGraph(self.ctx, self.model, self._states.sequences, self._tokens, self._logits)
        self._graph.launch()

    def search(self, prompt: Sequence[int], max_output_tokens: int) -> list:
        """The beams' hypotheses, best first: fewer than the beams where the tokens that are
        not masked make no more."""
        if self._workspace is None:
            raise GenerationError("the search is closed")
        if max_output_tokens < 1:
            raise GenerationError("max_output_tokens must be positive")
        if len(prompt) < 1 or len(prompt) + max_output_tokens > self.capacity:
            raise GenerationError("the prompt and its output exceed the capacity")
        # (length^-length_penalty is held in a float)
        if abs(self.length_penalty) * math.log2(max_output_tokens) > 126:
            raise GenerationError("length_penalty is too large for so many tokens")
        with self._on_stream():
            return self._search(prompt, max_output_tokens)

    def _search(self, prompt: Sequence[int], max_output_tokens: int) -> list:
        torch, states = self.ctx.torch, self._states
        scores, other = self._scores
        states.start()
        hip.prefill(self.ctx, self.model, prompt, states.sequences[0], self._logits[0, 0], ubatch=self.ubatch)
        # the prompt is one beam; the first step's children are all its own
        scores.fill_(-torch.inf)
        scores[0, 0] = 0.0
        ended = torch.zeros_like(self._tokens)
        lengths = torch.zeros_like(scores)
        position = len(prompt)
        for n in range(1, max_output_tokens + 1):
            if self._masked.numel():
                self._logits.index_fill_(2, self._masked, -torch.inf)
            # (a live beam's candidates have n tokens)
            lengths = torch.where(ended != 0, lengths, float(n))
            hip.beam_select(self.ctx, self._logits, scores, other, self._parents, self._tokens, self._workspace,
                            weights=lengths.pow(-self.length_penalty) if self.length_penalty else None, ended=ended,
                            ended_token=self._ended_token, settle=True)
            scores, other = other, scores
            states.follow(self._parents, position)
            self._history[:, :, n - 1] = self._tokens
            # (rows without a beam, of a vocabulary smaller than the beams, have no parent)
            parents = self._parents.clamp(min=0).long()
            lengths = lengths.gather(1, parents)
            ended = ended.gather(1, parents)
            if self._stop.numel():
                ended = ((ended != 0) | torch.isin(self._tokens, self._stop)).int()
            done, wrong = torch.stack([((ended != 0) | torch.isneginf(scores)).all(), scores.isnan().any()]).tolist()
            if wrong:
                raise GenerationError("the model's logits hold a NaN or an infinity")
            if n == max_output_tokens or done:
                break
            self._tokens.clamp_(min=0)  # (of rows without a beam)
            self._decode()
            position += 1
        found = []
        for row, total, length, gone in zip(self._history[0].tolist(), scores[0].tolist(), lengths[0].tolist(),
                                            ended[0].tolist()):
            if total == float("-inf"):
                continue
            length = int(length)
            found.append(Hypothesis(row[:length - 1 if gone else length], total, total / length ** self.length_penalty,
                                    "stop_token" if gone else "length"))
        return sorted(found, key=lambda h: -h.score)

    def close(self) -> None:
        if getattr(self, "_graph", None) is not None:
            self._graph.close()
            self._graph = None
        if getattr(self, "_workspace", None) is not None:
            self._workspace.close()
            self._workspace = None
