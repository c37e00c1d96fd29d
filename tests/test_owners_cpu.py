"""Objects that own handles of the library and are dropped without close(): their
finalizers must not touch the device (a capture on any stream would end), so the
handles wait for the next call that does. Without a GPU: a stand-in for the
library records the calls."""
import ctypes as C
import gc

import pytest
import torch

from adi_amd import hip, serving


class Library:
    """Every function of the library: records its name and first argument."""

    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        def call(handle=None, *rest):
            self.calls.append((name, getattr(handle, "value", handle)))
            return hip.OK
        return call


@pytest.fixture
def lib():
    gc.collect()
    hip._dropped.clear()
    yield Library()
    hip._dropped.clear()


def context(lib, handle=1, books=()):
    ctx = hip.Context.__new__(hip.Context)
    ctx.lib, ctx.handle, ctx._books, ctx.device = lib, C.c_void_p(handle), [C.c_void_p(b) for b in books], 0
    ctx._users = set()
    return ctx


def rope(lib, handle=2):
    r = hip.Rope.__new__(hip.Rope)
    r.lib, r.handle = lib, C.c_void_p(handle)
    return r


def workspace(lib, handle=3):
    w = hip.PagedWorkspace.__new__(hip.PagedWorkspace)
    w.lib, w.handle = lib, C.c_void_p(handle)
    return w


def used(ctx, kind, handle):
    """A graph or a batcher of a context."""
    o = kind.__new__(kind)
    o.ctx, o.handle, o._thread = ctx, C.c_void_p(handle), None
    ctx._users.add(handle)
    return o


def weights(lib, kind, handle=4):
    fields = {"struct": None, "weights": handle, "lib": lib}
    if kind is hip.GgufMoeLayer:
        fields.update(experts=8, hidden=64)
    if kind is hip.GgufHead:
        fields.update(final_norm=0)
    return kind(**fields)


MADE = {
    "context": (context, "adi_hip_context_destroy"),
    "rope": (rope, "adi_hip_rope_destroy"),
    "workspace": (workspace, "adi_hip_paged_workspace_destroy"),
    "moe": (lambda lib: weights(lib, hip.GgufMoeLayer), "adi_hip_weights_destroy"),
    "embedding": (lambda lib: weights(lib, hip.GgufEmbedding), "adi_hip_weights_destroy"),
    "layer": (lambda lib: weights(lib, hip.GgufDecoderLayer), "adi_hip_weights_destroy"),
    "head": (lambda lib: weights(lib, hip.GgufHead), "adi_hip_weights_destroy"),
    "graph": (lambda lib: used(context(lib), hip.DecodeGraph, 5), "adi_hip_decode_graph_destroy"),
    "batcher": (lambda lib: used(context(lib), serving.ContinuousBatcher, 6), "adi_hip_batcher_destroy"),
}


@pytest.mark.parametrize("cycle", [False, True])
@pytest.mark.parametrize("kind", MADE)
def test_dropped_objects_wait(lib, kind, cycle):
    make, destroy = MADE[kind]
    held = [make(lib)]
    if cycle:
        held.append(held)
    del held
    gc.collect()
    assert lib.calls == []
    hip.release_dropped()
    gc.collect()
    hip.release_dropped()
    assert [name for name, _ in lib.calls][0] == destroy
    assert [name for name, _ in lib.calls].count(destroy) == 1
    hip.release_dropped()
    assert len(lib.calls) == (2 if kind in ("graph", "batcher") else 1)  # (and its context, after it)


@pytest.mark.parametrize("kind", MADE)
def test_close_frees_at_once(lib, kind):
    make, destroy = MADE[kind]
    held = make(lib)
    held.close()
    assert [name for name, _ in lib.calls] == [destroy]
    held.close()
    assert len(lib.calls) == 1
    del held
    gc.collect()
    assert [name for name, _ in lib.calls].count(destroy) == 1


def test_the_pattern_of_a_refused_call(lib):
    """A temporary in a call that raises: exception -> traceback -> frame -> exception."""
    def refuse(r):
        raise hip.HipError(hip.INVALID_ARGUMENT, "no")

    def body():
        with pytest.raises(hip.HipError) as info:
            refuse(rope(lib))
        assert info
    body()
    gc.collect()
    assert lib.calls == []
    hip.release_dropped()
    assert lib.calls == [("adi_hip_rope_destroy", 2)]


@pytest.mark.parametrize("kind", [hip.DecodeGraph, serving.ContinuousBatcher])
@pytest.mark.parametrize("first", [0, 1])
def test_a_context_waits_for_what_uses_it(lib, kind, first):
    """In a cycle the collector runs finalizers in any order; here in both."""
    ctx = context(lib, 1, books=[7, 8])
    o = used(ctx, kind, 5)
    for held in [(ctx, o), (o, ctx)][first]:
        held.__del__()
    assert lib.calls == []
    hip.release_dropped()
    assert [handle for _, handle in lib.calls] == [5, 7, 8, 1]
    assert not hip._dropped


def test_a_context_alone_waits(lib):
    ctx = context(lib)
    o = used(ctx, hip.DecodeGraph, 5)
    ctx.__del__()
    hip.release_dropped()
    assert lib.calls == [] and len(hip._dropped) == 1
    o.close()
    hip.release_dropped()
    assert [handle for _, handle in lib.calls] == [5, 1]


def test_what_an_object_held_lives_until_it_is_freed(lib):
    """A graph's weights and context go after it."""
    o = used(context(lib), hip.DecodeGraph, 5)
    o.model = weights(lib, hip.GgufHead)
    del o
    gc.collect()
    hip.release_dropped()
    gc.collect()
    hip.release_dropped()
    assert [handle for _, handle in lib.calls][0] == 5
    assert sorted(handle for _, handle in lib.calls) == [1, 4, 5]


def test_nothing_is_freed_while_the_stream_captures(lib, monkeypatch):
    r = rope(lib)
    del r
    monkeypatch.setattr(torch.cuda, "is_initialized", lambda: True)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    hip.release_dropped()
    assert lib.calls == [] and len(hip._dropped) == 1
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    hip.release_dropped()
    assert lib.calls == [("adi_hip_rope_destroy", 2)]


def drop(lib):
    rope(lib, 99)
    assert ("adi_hip_rope_destroy", 99) not in lib.calls


def test_calls_that_touch_the_device_free_what_was_dropped(lib):
    ctx, file = context(lib), type("File", (), {"handle": None})()
    book = hip.np.zeros(4, hip.np.float32)
    calls = [
        lambda: hip.Rope(ctx, 64), lambda: hip.PagedWorkspace(ctx), workspace(lib).close,
        lambda: ctx.expert_codebook(book), lambda: ctx.ne_codebook(book),
        lambda: hip.upload_codebooks_gguf(ctx, file), lambda: hip.upload_moe_layer_gguf(ctx, file, 0, 0, 0),
        lambda: hip.upload_decoder_layer_gguf(ctx, file, 0, 0, 0), lambda: hip.upload_head_gguf(ctx, file),
        lambda: hip.upload_embedding_gguf(ctx, file)]
    for call in calls:
        lib.calls.clear()
        drop(lib)
        held = call()
        assert ("adi_hip_rope_destroy", 99) in lib.calls
        del held


def test_synchronize_frees_nothing(lib):
    """It waits for one stream, which another thread's capture survives."""
    drop(lib)
    context(lib).synchronize()
    assert [name for name, _ in lib.calls] == ["adi_hip_synchronize"]


def test_a_dropped_search_does_not_touch_the_device(lib):
    search = serving.BeamSearch.__new__(serving.BeamSearch)
    search._graph, search._workspace = used(context(lib), hip.DecodeGraph, 5), workspace(lib)
    del search
    gc.collect()
    assert lib.calls == []
    hip.release_dropped()
    gc.collect()
    hip.release_dropped()
    assert sorted(handle for _, handle in lib.calls) == [1, 3, 5]


@pytest.mark.parametrize("kind", [hip.DecodeGraph, serving.ContinuousBatcher])
@pytest.mark.parametrize("how", ["close", "drop"])
def test_a_closed_context_outlives_what_uses_it(lib, kind, how):
    """Freeing a graph or a batcher waits for the context's stream, so the context
    goes after it."""
    ctx = context(lib, 1, books=[7])
    o = used(ctx, kind, 5)
    ctx.close()
    assert lib.calls == []
    if how == "close":
        o.close()
    del o
    hip.release_dropped()
    assert [handle for _, handle in lib.calls] == [5, 7, 1]
    ctx.close()
    assert len(lib.calls) == 3
