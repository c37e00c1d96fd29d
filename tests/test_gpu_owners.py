"""Objects dropped without close() while a graph is captured: the capture goes on,
its replays give what eager calls give, and the objects are freed afterwards."""
import gc

import numpy as np
import pytest
import torch

from adi_amd import hip

pytestmark = pytest.mark.gpu


def ints(values):
    return torch.as_tensor(np.asarray(values, np.int32)).cuda()


def dropped(gpu):
    """Objects that only the collector finds."""
    held = [hip.Rope(gpu, 64), hip.PagedWorkspace(gpu, 1 << 20), hip.Context(0)]
    held[2].ne_codebook(np.linspace(-1.0, 1.0, 1024, dtype=np.float32))
    held.append(held)


def test_objects_collected_during_a_capture(gpu):
    gc.collect()
    hip.release_dropped()
    rope, positions = hip.Rope(gpu, 128, "pairs", 1e4), ints([3, 70, 5000])
    x = torch.randn(3, 4, 128, device="cuda")
    out, eager = torch.empty_like(x), torch.empty_like(x)
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    hip.rope_rows(gpu, rope, x, positions, eager)
    torch.cuda.synchronize()
    gc.disable()
    try:
        dropped(gpu)
        with torch.cuda.graph(graph, stream=stream):
            gpu.use_stream(torch.cuda.current_stream())
            gc.collect()  # as it may run anywhere
            waiting = len(hip._dropped)
            hip.release_dropped()
            assert len(hip._dropped) == waiting
            hip.rope_rows(gpu, rope, x, positions, out)
    finally:
        gc.enable()
        gpu.use_stream(torch.cuda.default_stream())
    assert waiting == 3
    hip.release_dropped()
    assert not hip._dropped
    for i in range(3):
        x.normal_()
        positions.add_(i)
        out.zero_()
        hip.rope_rows(gpu, rope, x, positions, eager)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager)
    rope.close()


def test_dropped_memory_comes_back(gpu):
    """Sixteen workspaces of 1 GiB, one after another, each dropped in a cycle: the
    next one's creation frees those before."""
    gc.collect()
    hip.release_dropped()
    free = torch.cuda.mem_get_info()[0]
    for _ in range(16):
        held = [hip.PagedWorkspace(gpu, 1 << 30)]
        held.append(held)
        del held
        gc.collect()
    assert torch.cuda.mem_get_info()[0] > free - (2 << 30)
    hip.release_dropped()
    assert torch.cuda.mem_get_info()[0] > free - (1 << 30)
