"""Forks at the edge of what a call holds: batches of no rows."""
import numpy as np
import pytest
import torch

from adi_amd import hip
from test_gpu_pages import ints, made_caches, pool_of, words

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def workspace(gpu):
    w = hip.PagedWorkspace(gpu)
    yield w
    gpu.synchronize()
    w.close()


def no_rows(gpu, columns=4):
    empty = torch.empty(0, dtype=torch.int32, device="cuda")
    return hip.PagedBatch(gpu, ints([0]), empty, torch.empty((0, columns), dtype=torch.int32, device="cuda"), 0, 0, 64)


@pytest.mark.parametrize("pages", [5, 256, 257, 5000])
@pytest.mark.parametrize("in_place", [True, False])
def test_a_fork_of_no_rows(gpu, workspace, pages, in_place):
    """The counts are the old ones, and the number of pages that lack is 0, as after
    any call, whatever the step before left there."""
    old = np.arange(pages) % 3
    count, lacking = ints(old), ints([17])
    pool = pool_of(gpu, made_caches(1, 1, pages, 16, 1, 64, "bf16"), count, lacking)
    given = None if in_place else ints(old + 5)
    hip.paged_fork(gpu, pool, no_rows(gpu), torch.empty((0, 4), dtype=torch.int32, device="cuda"), workspace,
                   references=given)
    assert words(lacking).tolist() == [0]
    assert np.array_equal(words(count), old if in_place else old + 5)


def test_a_pool_that_ran_out_and_emptied(gpu, workspace):
    """Rows that lack pages, given back, then a step of no rows."""
    count, lacking = ints(np.zeros(3)), ints([0])
    pool = pool_of(gpu, made_caches(2, 1, 3, 16, 1, 64, "f32"), count, lacking)
    lengths, table = ints([0, 0]), ints(np.full((2, 4), -1))
    batch = hip.PagedBatch(gpu, ints([0, 40, 80]), lengths, table, 80, 40, 64)
    hip.paged_fork(gpu, pool, batch, ints([[-1], [-1]]), workspace)
    assert words(lacking).tolist() == [3]
    hip.paged_fork(gpu, pool, no_rows(gpu), torch.empty((0, 1), dtype=torch.int32, device="cuda"), workspace)
    assert words(lacking).tolist() == [0] and words(count).tolist() == [1, 1, 1]


def test_a_fork_of_no_rows_without_anything_to_write(gpu, workspace):
    count = ints([1, 2, 0])
    pool = pool_of(gpu, made_caches(3, 1, 3, 16, 1, 64, "f32"), count)
    hip.paged_fork(gpu, pool, no_rows(gpu), torch.empty((0, 1), dtype=torch.int32, device="cuda"), workspace)
    assert words(count).tolist() == [1, 2, 0]
