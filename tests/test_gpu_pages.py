"""Tables that are forked, grown and given back, pages copied and pools compacted on
the GPU, against the same kept in lists on the host: pages shared and not, last
pages that are full, partly filled and shared, requests that begin and end, pools
that run out, bounds and page numbers that are wrong, every layout and type, in
place and not, captured calls, and a beam search's steps over the paged layer."""
import numpy as np
import pytest
import torch

from adi_amd import hip

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
NONE = 0xFFFFFFFF


def ints(values):
    """Whole numbers below 2^32 (or negative ones) as the 32 bits they are."""
    held = np.asarray(values).astype(np.int64) & 0xFFFFFFFF
    return torch.tensor(held.astype(np.uint32).view(np.int32), device="cuda")


def words(t):
    return t.cpu().numpy().astype(np.int64) & 0xFFFFFFFF


@pytest.fixture(scope="module")
def workspace(gpu):
    w = hip.PagedWorkspace(gpu)
    yield w
    gpu.synchronize()
    w.close()


def made_caches(seed, count, pages, page, heads, size, kind, heads_first=False, wide=0):
    """Keys, values, keys, ... of `count` caches; `wide`: elements between pages."""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    out = []
    for _ in range(2 * count):
        whole = torch.randn(pages, heads * page * size + wide, device="cuda", generator=g).to(TYPES[kind])
        t = whole[:, :heads * page * size]
        out.append(t.view(pages, heads, page, size).transpose(1, 2) if heads_first else t.view(pages, page, heads, size))
    return out


def pool_of(gpu, tensors, references=None, lacking=None):
    return hip.PagedPool(gpu, [hip.PagedCache(gpu, tensors[i], tensors[i + 1]) for i in range(0, len(tensors), 2)],
                         references, lacking)


def moved(tensors, moves, source=None):
    """The tensors after moves (from page, to page, entries)."""
    out = [t.clone() for t in tensors]
    for new, old in zip(out, source or tensors):
        for a, b, n in moves:
            new[b, :n] = old[a, :n]
    return out


def ceil(a, b):
    return -(-a // b)


def forked(parents, beams, added, lengths, table, count, page, pages, columns, max_length, max_tokens):
    """The definition in lists: (lengths, {(row, column): page}, counts, lacking, moves)."""
    free = iter([p for p in range(pages) if count[p] == 0])
    held = [[int(p) for p in table[i, :min(ceil(int(n), page), table.shape[1])]] for i, n in enumerate(lengths)]
    after = count.copy()
    for pages_of in held:
        for p in pages_of:
            if p < pages:
                after[p] -= 1
    new_lengths, new_table, moves, lacking = [], {}, [], 0

    def take():
        nonlocal lacking
        p = next(free, NONE)
        lacking += p == NONE
        return p

    for s, parent in enumerate(parents):
        group = s // beams * beams
        mine, n = ([], 0) if not 0 <= parent < beams else (list(held[group + parent]), int(lengths[group + parent]))
        over = added[s] > max_tokens or n + added[s] > max_length
        if not over and n % page and added[s] and n // page < table.shape[1]:
            last = mine[-1]
            eldest = parent not in list(parents[group:s])
            if last < pages and not (eldest and count[last] == 1):
                mine[-1] = take()
                if mine[-1] != NONE:
                    moves.append((last, mine[-1], n % page))
        want = min(ceil(n + added[s], page), columns)
        while len(mine) < want:
            mine.append(NONE if over else take())
        new_lengths.append(n + added[s])
        for c, p in enumerate(mine[:columns]):
            new_table[s, c] = p
            if p < pages:
                after[p] += 1
    return new_lengths, new_table, after, lacking, moves


class Books:
    """A server's tables on the host, and the device's next to them."""

    def __init__(self, gpu, workspace, rows, beams, columns, pages, page, seed=1, caches=2, heads=2, size=64, kind="bf16",
                 **layout):
        self.gpu, self.workspace = gpu, workspace
        self.rows, self.beams, self.columns, self.pages, self.page = rows, beams, columns, pages, page
        self.lengths = np.zeros(rows, np.int64)
        self.table = np.full((rows, columns), NONE, np.int64)
        self.count = np.zeros(pages, np.int64)
        self.tensors = made_caches(seed, caches, pages, page, heads, size, kind, **layout)
        self.device()

    def device(self):
        self.d_lengths, self.d_table, self.d_count = ints(self.lengths), ints(self.table), ints(self.count)
        self.d_lacking = ints([77])
        self.pool = pool_of(self.gpu, self.tensors, self.d_count, self.d_lacking)

    def step(self, parents, added, max_tokens=None, max_length=None, in_place=True, tokens=None):
        parents, added = np.asarray(parents).reshape(-1), np.asarray(added).reshape(-1)
        max_tokens = int(added.max(initial=0)) if max_tokens is None else max_tokens
        max_length = self.columns * self.page if max_length is None else max_length
        want = forked(parents, self.beams, added, self.lengths, self.table, self.count, self.page, self.pages,
                      self.columns, max_length, max_tokens)
        data = moved(self.tensors, want[4])
        offsets = ints(np.concatenate([[0], np.cumsum(added)]))
        old = {}
        if not in_place:
            old = dict(lengths=self.d_lengths, table=self.d_table, references=self.d_count)
            held = [t.clone() for t in old.values()]
            self.d_lengths, self.d_table, self.d_count = (torch.full_like(t, 12345) for t in old.values())
            self.d_table.copy_(old["table"])
            self.pool = pool_of(self.gpu, self.tensors, self.d_count, self.d_lacking)
        batch = hip.PagedBatch(self.gpu, offsets, self.d_lengths, self.d_table,
                               max(int(added.sum()), max_tokens) if tokens is None else tokens, max_tokens, max_length)
        hip.paged_fork(self.gpu, self.pool, batch, ints(parents).view(-1, self.beams), self.workspace, **old)
        for (s, c), p in want[1].items():
            self.table[s, c] = p
        self.lengths, self.count = np.array(want[0], np.int64), want[2]
        assert np.array_equal(words(self.d_lengths), self.lengths)
        assert np.array_equal(words(self.d_table), self.table)
        assert np.array_equal(words(self.d_count), self.count & NONE)
        assert int(self.d_lacking) == want[3]
        for t, w in zip(self.tensors, data):
            assert torch.equal(t, w)
        if not in_place:
            assert all(torch.equal(a, b) for a, b in zip(held, old.values()))
        return batch


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("page,heads,size,layout", [
    (8, 1, 64, {}), (16, 2, 256, {}), (64, 3, 128, dict(heads_first=True)), (16, 5, 64, dict(wide=8)),
    (32, 2, 64, dict(heads_first=True, wide=64)), (256, 1, 64, {})])
def test_a_search_from_prompt_to_end(gpu, workspace, kind, page, heads, size, layout):
    """Admission, the first step's fork of all from one, steps that fork and drop,
    and the end of a request, three requests of four beams."""
    b = Books(gpu, workspace, 12, 4, 12, 120, page, heads=heads, size=size, kind=kind, **layout)
    g = np.random.default_rng(page)
    prompt = np.array([3 * page + 5, page, 1])
    first = np.zeros((3, 4), int)
    first[:, 0] = prompt
    b.step(np.full((3, 4), -1), first)
    b.step(np.zeros((3, 4)).astype(int), np.ones((3, 4), int))
    for i in range(2 * page if page < 64 else 5):
        b.step(g.integers(0, 4, (3, 4)), np.ones((3, 4), int), in_place=i % 2 == 0)
    b.step([[-1] * 4, [0, 1, 2, 3], [2, 2, -1, 9]], [[0] * 4, [1, 0, 2, page], [0, 1, 1, 0]])
    b.step(np.full((3, 4), -1), np.zeros((3, 4), int))
    assert (b.count == 0).all() and (b.lengths == 0).all()


@pytest.mark.parametrize("beams,requests", [(1, 1), (1, 300), (2, 7), (3, 5), (4, 64), (8, 3), (16, 2), (17, 3), (64, 2)])
@pytest.mark.parametrize("in_place", [True, False])
def test_beams_and_requests(gpu, workspace, beams, requests, in_place):
    rows = beams * requests
    b = Books(gpu, workspace, rows, beams, 6, 6 * rows + 40, 8, caches=1, heads=1)
    g = np.random.default_rng(beams)
    b.step(np.full(rows, -1), g.integers(0, 30, rows))
    for _ in range(4):
        added = g.integers(0, 4, rows) * (g.random(rows) < 0.7)
        parents = np.where(g.random(rows) < 0.1, -1, g.integers(0, beams, rows))
        grown = np.where(parents < 0, 0, b.lengths[np.arange(rows) // beams * beams + parents.clip(0)])
        b.step(parents, np.minimum(added, 6 * 8 - grown), in_place=in_place)


@pytest.mark.parametrize("pages", [4095, 4096, 4097, 30011, 140001])
def test_pools_of_many_segments(gpu, workspace, pages):
    """The lowest free pages, wherever in a long pool they lie."""
    b = Books(gpu, workspace, 8, 4, 400, pages, 8, caches=1, heads=1)
    g = np.random.default_rng(pages)
    # a sequence of its own that holds most pages, in no order
    others = g.permutation(pages)[:pages * 9 // 10]
    b.count[others] = 1
    b.device()
    b.step(np.full(8, -1), [290 * 8 + 3, 0, 0, 0, 1, 0, 0, 0])
    for i in range(3):
        b.step(np.where(np.arange(8) < 4, 0, g.integers(0, 4, 8)) if i == 0 else g.integers(0, 4, 8),
               np.ones(8, int), in_place=i != 1)
    b.step(np.full(8, -1), np.zeros(8, int))
    assert b.count.sum() == others.size


def test_a_pool_that_runs_out(gpu, workspace):
    b = Books(gpu, workspace, 8, 4, 8, 20, 8, caches=1, heads=1)
    b.step(np.full(8, -1), [20, 0, 0, 0, 60, 0, 0, 0])  # 3 and 8 of 20
    b.step([0] * 8, [1] * 8)                            # 6 copies, 9 free: three left
    b.step([0, 0, 1, 1, 0, 1, 1, 1], [1] * 8)           # 4 copies, one cannot be had
    assert int(b.d_lacking) == 1
    # rows without a page go on without one, and give back only what they hold
    b.step([0, 1, 2, 3, 0, 1, 2, 3], [1] * 8)
    b.step(np.full(8, -1), [0] * 8)
    assert (b.count == 0).all()
    b.step(np.full(8, -1), [64] * 8)
    assert int(b.d_lacking) == 64 - 20
    b.step(np.full(8, -1), [0] * 8)
    assert (b.count == 0).all()


def test_bounds_and_wrong_page_numbers(gpu, workspace):
    b = Books(gpu, workspace, 8, 2, 6, 60, 8, caches=1, heads=1)
    b.step(np.full(8, -1), [20, 0, 33, 0, 40, 0, 8, 0])
    # more new tokens, and more entries, than the batch allows
    b.step([0, 0, 0, 0, 0, 0, 0, 0], [1, 5, 1, 1, 1, 1, 1, 1], max_tokens=2, max_length=40)
    b.step([0, 1, 0, 1, 0, 1, 0, 1], [1] * 8, max_tokens=2, max_length=40)
    # numbers that are no pages, in the middle and last
    b.table[0, 1], b.table[6, 1] = 60, NONE
    b.count[words(b.d_table)[0, 1]] -= 1
    if words(b.d_table)[6, 1] < 60:
        b.count[words(b.d_table)[6, 1]] -= 1
    b.device()
    b.step([0, 0, 1, 1, 0, 0, 0, 0], [1] * 8)
    b.step(np.full(8, -1), [0] * 8)


def test_shared_last_pages(gpu, workspace):
    """Forks without new tokens share a partly filled page; the next token copies
    it for all but none where others hold it too."""
    b = Books(gpu, workspace, 8, 4, 4, 40, 16, caches=1, heads=1)
    b.step(np.full(8, -1), [21, 0, 0, 0, 32, 0, 0, 0])
    b.step([0] * 8, [0] * 8)                       # shared, no copy
    assert b.count.max() == 4
    b.step([0, 1, 2, 3] * 2, [1, 0, 0, 1, 1, 1, 0, 0])
    b.step([0, 1, 2, 3] * 2, [1] * 8)
    b.step([3, 3, 1, 0] * 2, [16] * 8)
    # a page that a row outside holds too
    b.count[b.table[0, 0]] += 1
    b.device()
    b.step([0, 1, 2, 3] * 2, [0] * 8)
    b.step([1, 0, 3, 2] * 2, [1] * 8)


def test_tables_of_other_widths(gpu, workspace):
    """From a narrow table into a wider one and back."""
    tensors = made_caches(1, 1, 50, 8, 1, 64, "f16")
    g = np.random.default_rng(4)
    lengths, table = np.array([20, 7, 0, 24]), np.full((4, 3), NONE, np.int64)
    order = g.permutation(50)
    count = np.zeros(50, np.int64)
    at = 0
    for s, n in enumerate(lengths):
        k = ceil(n, 8)
        table[s, :k] = order[at:at + k]
        at += k
    count[order[:at]] = 1
    for columns, max_length in ((7, 56), (9, 50), (4, 26), (3, 24)):
        want = forked([0, 0, 1, 1], 2, [3, 1, 5, 1], lengths, table, count, 8, 50, columns, max_length, 5)
        data = moved(tensors, want[4])
        d_table, d_lengths, d_count = ints(np.full((4, columns), 4242)), ints([9] * 4), ints([0] * 50)
        batch = hip.PagedBatch(gpu, ints([0, 3, 4, 9, 10]), d_lengths, d_table, 10, 5, max_length)
        hip.paged_fork(gpu, pool_of(gpu, tensors, d_count), batch, ints([[0, 0], [1, 1]]), workspace, ints(lengths),
                       ints(table), ints(count))
        expected = np.full((4, columns), 4242)
        for (s, c), p in want[1].items():
            expected[s, c] = p
        assert np.array_equal(words(d_table), expected)
        assert np.array_equal(words(d_lengths), want[0]) and np.array_equal(words(d_count), want[2])
        assert all(torch.equal(a, w) for a, w in zip(tensors, data))


def test_more_caches_than_a_launch_takes(gpu, workspace):
    b = Books(gpu, workspace, 4, 4, 4, 30, 8, caches=70, heads=1)
    b.step(np.full(4, -1), [13, 0, 0, 0])
    b.step([0] * 4, [1] * 4)
    sources, targets = [1, 2], [25, 24]
    want = moved(b.tensors, [(1, 25, 8), (2, 24, 8)])
    hip.paged_copy(gpu, b.pool, b.pool, ints(sources), ints(targets))
    assert all(torch.equal(a, w) for a, w in zip(b.tensors, want))


@pytest.mark.parametrize("pages", [1023, 1024, 1025])
@pytest.mark.parametrize("beams,requests,columns", [(4, 1, 700), (4, 3, 200), (1, 12, 40), (1, 13, 40), (16, 1, 60), (64, 1, 256),
                                                    (64, 1, 257)])
@pytest.mark.parametrize("in_place", [True, False])
def test_forks_in_one_launch_and_two(gpu, workspace, pages, beams, requests, columns, in_place):
    """At the borders between them, the first columns and the last, to the last page."""
    rows = beams * requests
    b = Books(gpu, workspace, rows, beams, columns, pages, 8, caches=1, heads=1)
    g = np.random.default_rng(pages + rows + columns)
    first = np.zeros((requests, beams), int)
    first[:, 0] = min(columns - 3, (pages - 30) // requests) * 8 - 5
    b.step(np.full(rows, -1), first)
    b.step(np.zeros(rows, int), np.ones(rows, int), in_place=in_place)
    for i in range(3):
        b.step(g.integers(0, beams, rows), g.integers(0, 8, rows), in_place=in_place)
    # more than there are pages
    b.step(g.integers(0, beams, rows), np.where(np.arange(rows) % 2 == 0, 16, 1), in_place=in_place, max_length=columns * 8)


@pytest.mark.parametrize("own", [(1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 1, 0), (1, 0, 1), (0, 1, 1)])
def test_fork_of_arrays_partly_in_place(gpu, workspace, own):
    b = Books(gpu, workspace, 8, 4, 12, 100, 8)
    b.step(np.full(8, -1), [21, 0, 0, 0, 9, 0, 0, 0])
    b.step([0] * 8, [1] * 8)
    parents, added = np.array([3, 1, 1, 0, 2, 2, 7, 0]), np.array([1, 1, 2, 0, 1, 9, 3, 1])
    want = forked(parents, 4, added, b.lengths, b.table, b.count, 8, 100, 12, 96, 9)
    data = moved(b.tensors, want[4])
    old = [b.d_lengths, b.d_table, b.d_count]
    new = [t if o else t.clone() for t, o in zip(old, own)]
    pool = pool_of(gpu, b.tensors, new[2], b.d_lacking)
    batch = hip.PagedBatch(gpu, ints(np.concatenate([[0], np.cumsum(added)])), new[0], new[1], int(added.sum()), 9, 96)
    hip.paged_fork(gpu, pool, batch, ints(parents).view(2, 4), workspace, lengths=old[0], table=old[1], references=old[2])
    for (s, c), p in want[1].items():
        b.table[s, c] = p
    assert np.array_equal(words(new[0]), want[0]) and np.array_equal(words(new[1]), b.table)
    assert np.array_equal(words(new[2]), want[2]) and int(b.d_lacking) == want[3]
    assert all(torch.equal(t, w) for t, w in zip(b.tensors, data))


def test_one_workspace_for_calls_of_all_kinds(gpu):
    """Selection, forks and compactions behind one another, of sizes that join through
    the workspace's tickets and of others."""
    space = hip.PagedWorkspace(gpu)
    b = Books(gpu, space, 4, 4, 12, 60, 8, caches=1, heads=1)
    b.step(np.full(4, -1), [21, 0, 0, 0])
    g = torch.Generator(device="cuda").manual_seed(4)
    for i, v in enumerate((500, 9000, 33, 100000, 500)):
        logits = torch.randn((1, 4, v), generator=g, device="cuda")
        scores = torch.randn((1, 4), generator=g, device="cuda")
        out = torch.empty((1, 4), device="cuda")
        parents, tokens = ints(np.zeros((1, 4))), ints(np.zeros((1, 4)))
        hip.beam_select(gpu, logits, scores, out, parents, tokens, space)
        rank = (scores.double()[..., None] + torch.log_softmax(logits.double(), -1)).view(-1)
        best = torch.argsort(rank, descending=True, stable=True)[:4]
        assert torch.equal(parents[0].long(), best // v) and torch.equal(tokens[0].long(), best % v)
        b.step(words(parents), [1] * 4, in_place=i % 2 == 0)
        live, table, count, moves = compacted(b.count, b.lengths, b.table, 8)
        data, d_live = moved(b.tensors, moves), ints([0])
        hip.paged_compact(gpu, b.pool, b.d_lengths, b.d_table, d_live, space)
        b.table, b.count = table, count
        assert int(d_live) == live and np.array_equal(words(b.d_table), table)
        assert np.array_equal(words(b.d_count), count)
        assert all(torch.equal(t, w) for t, w in zip(b.tensors, data))


def test_fork_captured(gpu, workspace):
    """A step recorded once, replayed with new parents over what it wrote itself."""
    b = Books(gpu, workspace, 8, 4, 12, 150, 8, caches=2)
    b.step(np.full(8, -1), [21, 0, 0, 0, 9, 0, 0, 0])
    b.step([0] * 8, [1] * 8)
    stream = torch.cuda.Stream()
    ctx = hip.Context(0)
    ctx.use_stream(stream)
    parents, offsets = ints(np.zeros((2, 4))), ints(np.arange(9))
    batch = hip.PagedBatch(ctx, offsets, b.d_lengths, b.d_table, 8, 1, 96)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        hip.paged_fork(ctx, b.pool, batch, parents, workspace)
    g = np.random.default_rng(3)
    for _ in range(6):
        p = g.integers(0, 4, (2, 4))
        parents.copy_(ints(p))
        want = forked(p.reshape(-1), 4, [1] * 8, b.lengths, b.table, b.count, 8, 150, 12, 96, 1)
        data = moved(b.tensors, want[4])
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for (s, c), q in want[1].items():
            b.table[s, c] = q
        b.lengths, b.count = np.array(want[0]), want[2]
        assert np.array_equal(words(b.d_table), b.table) and np.array_equal(words(b.d_count), b.count)
        assert all(torch.equal(t, w) for t, w in zip(b.tensors, data))
    ctx.close()


def test_fork_of_small_workspaces(gpu):
    w = hip.PagedWorkspace(gpu, 1 << 20)
    b = Books(gpu, w, 4, 4, 4, 30, 8, caches=1, heads=1)
    b.step(np.full(4, -1), [13, 0, 0, 0])
    tensors = [torch.zeros(300000, 8, 1, 64, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    count = ints(np.zeros(300000))
    batch = hip.PagedBatch(gpu, ints([0, 1]), ints([0]), ints([[0]]), 1, 1, 8)
    for call in (lambda: hip.paged_fork(gpu, pool_of(gpu, tensors, count), batch, ints([[-1]]), w),
                 lambda: hip.paged_compact(gpu, pool_of(gpu, tensors, count), batch.lengths, batch.table, ints([0]), w)):
        with pytest.raises(hip.HipError, match="workspace") as e:
            call()
        assert e.value.status == hip.OUT_OF_MEMORY
    w.close()


def test_fork_refusals(gpu, workspace):
    b = Books(gpu, workspace, 4, 2, 4, 30, 8, caches=1, heads=1)
    batch = hip.PagedBatch(gpu, ints(np.arange(5)), b.d_lengths, b.d_table, 4, 1, 32)
    good = dict(pool=b.pool, batch=batch, parents=ints(np.zeros((2, 2))), workspace=workspace)
    for change in [dict(parents=ints(np.zeros(4))), dict(parents=ints(np.zeros((2, 3)))),
                   dict(parents=ints(np.zeros((2, 2))).long()), dict(parents=ints(np.zeros((2, 2))).cpu()),
                   dict(lengths=ints([0] * 3)), dict(table=ints(np.zeros((3, 4)))), dict(references=ints([0] * 29)),
                   dict(references=ints([0] * 30).long()), dict(pool=pool_of(gpu, b.tensors)),
                   dict(pool=pool_of(gpu, b.tensors), references=ints([0] * 30))]:
        with pytest.raises(hip.HipError) as e:
            hip.paged_fork(gpu, **{**good, **change})
        assert e.value.status == hip.INVALID_ARGUMENT
    for args in [([],), ([hip.PagedCache(gpu, *b.tensors)], ints([0] * 29)),
                 ([hip.PagedCache(gpu, *b.tensors)], ints([0] * 30), ints([0, 0]))]:
        with pytest.raises(hip.HipError):
            hip.PagedPool(gpu, *args)
    empty = hip.PagedBatch(gpu, ints([0]), ints([]), ints(np.zeros((0, 3))), 0, 0, 0)
    hip.paged_fork(gpu, b.pool, empty, ints(np.zeros((0, 2))), workspace)
    gpu.synchronize()


# ---- copies --------------------------------------------------------------------------

@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("page,heads,size", [(8, 1, 64), (16, 2, 256), (64, 3, 128), (32, 7, 64), (1024, 1, 128)])
@pytest.mark.parametrize("first,second", [({}, None), (dict(heads_first=True), None), ({}, dict(heads_first=True)),
                                          (dict(heads_first=True, wide=8), dict(wide=16))])
def test_copies(gpu, kind, page, heads, size, first, second):
    a = made_caches(1, 2, 30, page, heads, size, kind, **first)
    b = a if second is None else made_caches(2, 2, 40, page, heads, size, kind, **second)
    g = np.random.default_rng(page)
    order = g.permutation(30)
    sources, targets = order[:9], order[9:18] if second is None else g.permutation(40)[:9]
    entries = np.array([1, page, page - 1, 0, 3, page + 5, NONE, page // 2, 7])
    for some in (None, entries):
        n = [page] * 9 if some is None else [min(int(x), page) for x in some]
        want = moved(b, list(zip(sources, targets, n)), a)
        hip.paged_copy(gpu, pool_of(gpu, a), pool_of(gpu, b), ints(sources), ints(targets),
                       None if some is None else ints(some))
        assert all(torch.equal(t, w) for t, w in zip(b, want))


def test_copies_of_wrong_pages_and_none(gpu):
    a = made_caches(1, 1, 30, 8, 2, 64, "f16")
    b = made_caches(2, 1, 20, 8, 2, 64, "f16")
    want = moved(b, [(3, 4, 8), (29, 19, 8)], a)
    hip.paged_copy(gpu, pool_of(gpu, a), pool_of(gpu, b), ints([3, 30, 5, NONE, 29, 1]), ints([4, 5, 20, 6, 19, NONE]))
    assert all(torch.equal(t, w) for t, w in zip(b, want))
    hip.paged_copy(gpu, pool_of(gpu, a), pool_of(gpu, b), ints([]), ints([]))
    hip.paged_copy(gpu, pool_of(gpu, a), pool_of(gpu, a), ints([3, 4]), ints([3, 4]))  # onto themselves
    for change in [dict(targets=ints([1, 2])), dict(sources=ints([1]).long()), dict(entries=ints([1, 2])),
                   dict(targets=ints([1]).cpu()), dict(target=pool_of(gpu, made_caches(1, 2, 30, 8, 2, 64, "f16"))),
                   dict(target=pool_of(gpu, made_caches(1, 1, 30, 8, 2, 64, "bf16")))]:
        with pytest.raises(hip.HipError) as e:
            hip.paged_copy(gpu, **{**dict(source=pool_of(gpu, a), target=pool_of(gpu, b), sources=ints([1]),
                                          targets=ints([2])), **change})
        assert e.value.status == hip.INVALID_ARGUMENT
    gpu.synchronize()


def test_copies_past_32_bits(gpu):
    """Pages more than 2^32 bytes into a pool."""
    pages = 9000
    t = [torch.empty(pages, 4096, 2, 64, dtype=torch.float16, device="cuda") for _ in range(2)]
    for x in t:
        x[3].normal_()
        x[-1].zero_()
        x[4200].zero_()
    hip.paged_copy(gpu, pool_of(gpu, t), pool_of(gpu, t), ints([3, 3]), ints([pages - 1, 4200]), ints([4096, 77]))
    for x in t:
        assert torch.equal(x[-1], x[3]) and torch.equal(x[4200, :77], x[3, :77]) and not bool(x[4200, 77:].any())


# ---- compaction ------------------------------------------------------------------------

def compacted(count, lengths, table, page):
    live = int((count > 0).sum())
    movers = [p for p in range(live, count.size) if count[p] > 0]
    holes = [p for p in range(live) if count[p] == 0]
    name = dict(zip(movers, holes))
    new, after = table.copy(), count.copy()
    for i, n in enumerate(lengths):
        for c in range(min(ceil(int(n), page), table.shape[1])):
            new[i, c] = name.get(int(table[i, c]), table[i, c])
    for a, b in name.items():
        after[b], after[a] = count[a], 0
    return live, new, after, [(a, b, page) for a, b in name.items()]


@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("pages,rows,page,share,layout", [
    (1, 1, 8, 1.0, {}), (1, 1, 8, 0.0, {}), (7, 2, 16, 0.5, {}), (100, 5, 8, 0.3, dict(heads_first=True)),
    (2047, 20, 8, 0.7, {}), (2048, 20, 8, 0.5, {}), (2049, 30, 8, 0.02, {}), (4096, 30, 8, 1.0, {}),
    (9001, 100, 8, 0.4, dict(wide=8)), (6000, 3, 8, 0.999, {}), (140001, 90, 8, 0.6, {})])
def test_compaction(gpu, workspace, in_place, pages, rows, page, share, layout):
    g = np.random.default_rng(pages + rows)
    live = int(pages * share)
    held = g.permutation(pages)[:live]
    columns = max(ceil(live, rows), 1) + 2
    table = np.full((rows, columns), 7, np.int64)
    lengths, count = np.zeros(rows, np.int64), np.zeros(pages, np.int64)
    for i, part in enumerate(np.array_split(held, rows)):
        table[i, :part.size] = part
        lengths[i] = max(part.size * page - g.integers(0, page), 0)
        count[part] = 1
    # and pages that several hold
    if rows > 1 and lengths[0] > page:
        table[1, :1] = table[0, :1]
        lengths[1] = max(lengths[1], 1)
        count = np.zeros(pages, np.int64)
        for i in range(rows):
            for c in range(ceil(int(lengths[i]), page)):
                count[table[i, c]] += 1
    tensors = made_caches(1, 2, pages, page, 1, 64, "bf16", **layout)
    want_live, want_table, want_count, moves = compacted(count, lengths, table, page)
    data = moved(tensors, moves)
    d_table, d_count, d_live = ints(table), ints(count), ints([-3])
    if in_place:
        hip.paged_compact(gpu, pool_of(gpu, tensors, d_count), ints(lengths), d_table, d_live, workspace)
    else:
        old_table, old_count = d_table, d_count
        d_table, d_count = d_table.clone(), torch.full_like(d_count, 55)
        hip.paged_compact(gpu, pool_of(gpu, tensors, d_count), ints(lengths), d_table, d_live, workspace, old_table,
                          old_count)
        assert np.array_equal(words(old_table), table) and np.array_equal(words(old_count), count)
    assert int(d_live) == want_live
    assert np.array_equal(words(d_table), want_table) and np.array_equal(words(d_count), want_count)
    assert all(torch.equal(t, w) for t, w in zip(tensors, data))


@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("pages,rows,share", [(2, 1, 0.5), (3, 2, 0.7), (16, 3, 0.5), (255, 9, 0.4), (256, 9, 1.0), (256, 9, 0.5),
                                              (257, 9, 0.6), (700, 40, 0.05), (1023, 33, 0.5), (1024, 33, 0.97),
                                              (1024, 33, 1.0), (1025, 33, 0.5)])
def test_compaction_of_tiny_pools(gpu, workspace, in_place, pages, rows, share):
    test_compaction(gpu, workspace, in_place, pages, rows, 8, share, {})


def test_compaction_in_place_again_and_again(gpu):
    # one workspace, calls behind one another with nothing between them
    space = hip.PagedWorkspace(gpu, 1 << 20)
    g = np.random.default_rng(3)
    cases = []
    for pages in (40, 64, 7, 40, 900):
        table = g.permutation(pages)[:pages // 2][None, :]
        count = np.zeros(pages, np.int64)
        count[table[0]] = 1
        tensors = made_caches(pages, 1, pages, 8, 1, 64, "bf16")
        lengths = np.array([8 * table.shape[1]])
        live, new, after, moves = compacted(count, lengths, table, 8)
        cases.append((pool_of(gpu, tensors, ints(count)), ints(lengths), ints(table), ints([0]), tensors,
                      moved(tensors, moves), live, new, after))
    for pool, lengths, table, live, *_ in cases:
        hip.paged_compact(gpu, pool, lengths, table, live, space)
    for pool, _, table, live, tensors, data, want_live, want_table, want_count in cases:
        assert int(live) == want_live
        assert np.array_equal(words(table), want_table) and np.array_equal(words(pool.references), want_count)
        assert all(torch.equal(t, w) for t, w in zip(tensors, data))


@pytest.mark.parametrize("pages", [50, 5000])
def test_compaction_of_more_caches_than_a_launch_takes(gpu, workspace, pages):
    table = np.array([[pages - 1, 3, pages // 2]])
    lengths, count = np.array([20]), np.zeros(pages, np.int64)
    count[table[0]] = 1
    tensors = made_caches(9, 70, pages, 8, 1, 64, "bf16")
    live, want_table, want_count, moves = compacted(count, lengths, table, 8)
    data = moved(tensors, moves)
    d_table, d_count, d_live = ints(table), ints(count), ints([0])
    # (the table in place, the counts not; then all of it again, in place and with none to move)
    after = torch.full_like(d_count, 9)
    hip.paged_compact(gpu, pool_of(gpu, tensors, after), ints(lengths), d_table, d_live, workspace, references=d_count)
    hip.paged_compact(gpu, pool_of(gpu, tensors, after), ints(lengths), d_table, d_live, workspace)
    assert int(d_live) == live == 3
    assert np.array_equal(words(d_table), want_table) and np.array_equal(words(after), want_count)
    assert all(torch.equal(t, w) for t, w in zip(tensors, data))


def test_compaction_of_wrong_numbers_and_no_rows(gpu, workspace):
    """A table that names pages counted as free, and numbers that are no pages."""
    tensors = made_caches(1, 1, 40, 8, 1, 64, "f16")
    count = np.zeros(40, np.int64)
    count[[0, 30, 31]] = 1
    table = np.array([[0, 30, 35, 40, NONE, 31]])
    live, new, after, moves = compacted(count, [48], table, 8)
    data = moved(tensors, moves)
    d_table, d_count, d_live = ints(table), ints(count), ints([0])
    hip.paged_compact(gpu, pool_of(gpu, tensors, d_count), ints([48]), d_table, d_live, workspace)
    assert int(d_live) == 3 and words(d_table).tolist() == [[0, 1, 35, 40, NONE, 2]] and new.tolist() == words(d_table).tolist()
    assert all(torch.equal(t, w) for t, w in zip(tensors, data))
    d_count = ints(count)
    hip.paged_compact(gpu, pool_of(gpu, tensors, d_count), ints([]), ints(np.zeros((0, 3))), d_live, workspace)
    assert np.array_equal(words(d_count), after)
    d_count = ints(np.full(40, 1))  # a length past the table
    d_table = ints([[5, 6]])
    hip.paged_compact(gpu, pool_of(gpu, tensors, d_count), ints([1 << 27]), d_table, d_live, workspace)
    assert int(d_live) == 40 and words(d_table).tolist() == [[5, 6]]
    for change in [dict(lengths=ints([1, 2])), dict(live=ints([1, 2])), dict(next_table=ints([[1, 2, 3]])),
                   dict(references=ints([1])), dict(pool=pool_of(gpu, tensors))]:
        with pytest.raises(hip.HipError) as e:
            hip.paged_compact(gpu, **{**dict(pool=pool_of(gpu, tensors, d_count), lengths=ints([8]), live=d_live,
                                             next_table=d_table, table=ints([[1, 2]]), workspace=workspace), **change})
        assert e.value.status == hip.INVALID_ARGUMENT


def test_compaction_captured(gpu, workspace):
    tensors = made_caches(1, 1, 3000, 8, 1, 64, "f32")
    stream = torch.cuda.Stream()
    ctx = hip.Context(0)
    ctx.use_stream(stream)
    d_count, d_table, d_lengths, d_live = ints(np.zeros(3000)), ints(np.zeros((1, 3000))), ints([0]), ints([0])
    pool = pool_of(ctx, tensors, d_count)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        hip.paged_compact(ctx, pool, d_lengths, d_table, d_live, workspace)
    for seed in range(4):
        g = np.random.default_rng(seed)
        held = g.permutation(3000)[:g.integers(0, 3000)]
        count, table = np.zeros(3000, np.int64), np.full((1, 3000), 5, np.int64)
        count[held] = 1
        table[0, :held.size] = held
        d_count.copy_(ints(count))
        d_table.copy_(ints(table))
        d_lengths.copy_(ints([held.size * 8]))
        live, new, after, moves = compacted(count, [held.size * 8], table, 8)
        data = moved(tensors, moves)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert int(d_live) == live
        assert np.array_equal(words(d_table), new) and np.array_equal(words(d_count), after)
        assert all(torch.equal(t, w) for t, w in zip(tensors, data))
    ctx.close()
