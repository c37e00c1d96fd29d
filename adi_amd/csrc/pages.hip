// pages.hip -- the pages of a paged cache: tables forked, grown and given back
// with their reference counts, pages copied, and a pool compacted.
//
// Nothing here reads a count on the host: pages are found, counted and moved by
// the kernels, the lowest free ones first, so results do not depend on the order
// of blocks and a captured call replays with the tables it finds.
#include "paged_attention.hpp"

#include <algorithm>

namespace adi_hip {
namespace {

constexpr uint32_t kThreads = 256;
constexpr uint32_t kWaves = kThreads / kWave;
constexpr uint32_t kNone = 0xFFFFFFFFu;
constexpr uint32_t kMaxBeams = 64;
constexpr uint32_t kCaches = 64, kMaxCaches = 1024;  // of a launch, of a pool
constexpr uint32_t kMaxPages = 1u << 22;
// pages of a segment: what a block counts
constexpr uint32_t kSegment = 2048, kSegments = kMaxPages / kSegment;
constexpr uint32_t kOwn = kSegment / kThreads;  // pages of a thread
// Pools of which one block finds the free pages (fork), or every block counts all
// live ones (compaction): a compaction saves a launch (4,096 pages 9.4 us on the device
// and 13.2), a fork its second kernel's search for a segment (4 rows 7.8 and 8.4, 128
// rows over two segments 13.4 either way). At 8,192 the registers for a thread's pages
// cost smaller pools a microsecond.
constexpr uint32_t kSmallPages = 4096;
// Pools that a compaction takes in one launch, and its blocks a CU that copy: those
// whose old counts stay (1 cache of 100 pages of 32 KB 9.9 us in two launches and 7.0, of
// 1,000 12.2 and 8.8, 10 caches 67.5 and 67.1, 30 184 and 190; of 4,096 34 and 39, as
// every block reads all counts), and in place where no more than a block a CU copies
// (9.7 and 6.7; a thousand blocks wait at their ticket for 10 us).
constexpr uint32_t kTinyPages = 1024, kTinyCopiers = 4;
// A fork does so with up to 256 rows, by the same number of blocks that copy, where the
// one that writes the tables has so many runs of 256 columns to go through, or one
// request's (4 beams of 2,005 entries 9.8 us in two launches and 6.9, 8 of 1,000 10.7 and
// 8.1, 16 of 300 14.8 and 11.9; 4 requests of 4 beams, 16 runs, 9.5 and 11.4; 8 rows without
// beams 9.8 and 8.8). In place the tables wait for the last block's arrival: 1 row without
// beams 9.9 and 6.9, 4 rows 9.6 and 8.8, 4 beams of 2,005 entries 11.2 and 9.2, but 8 rows
// without beams 9.6 and 12.8, 10 of them 9.6 and 14.8, for which the bound is too high.
constexpr uint32_t kTinyTables = 12;

using u32x4 = uint32_t __attribute__((ext_vector_type(4)));

// ---- copies of pages ---------------------------------------------------------

// The keys and values of every cache of a pool, and how a page of them lies: its
// first n entries are `heads` runs of n entries (heads outermost) or n runs of
// `heads`, in units of 16 bytes.
struct CachesView {
    char *data[2u * kCaches];  // keys, values, keys, ...
    uint64_t page_stride, entry_stride, head_stride;  // bytes
    uint32_t arrays, heads, head_shift, page_size, pages;  // head_shift: log2 of a head's units
    uint32_t heads_first;
};

CachesView caches_view(const adi_hip_paged_pool &pool, uint32_t first) {
    CachesView v{};
    const adi_hip_paged_cache *const caches = pool.cache + first;
    const uint32_t count = std::min(pool.caches - first, kCaches);
    const adi_hip_paged_cache &c = caches[0];
    const uint32_t size = type_bytes(c.type);
    for (uint32_t i = 0; i < count; ++i) {
        v.data[2u * i] = static_cast<char *>(caches[i].keys);
        v.data[2u * i + 1u] = static_cast<char *>(caches[i].values);
    }
    v.page_stride = c.page_stride * size;
    v.entry_stride = c.entry_stride * size;
    v.head_stride = c.head_stride * size;
    v.arrays = 2u * count;
    v.heads = c.heads;
    v.head_shift = log2_of(c.head_size * size / 16u);
    v.page_size = c.page_size;
    v.pages = c.pages;
    v.heads_first = c.entry_stride < c.head_stride ? 1u : 0u;
    return v;
}

// Where unit u of a page's first `entries` lies: vectors of a head counted entry by
// entry, or head by head where `heads_first` (the order of the copy's source).
__device__ __forceinline__ uint64_t unit_at(const CachesView &v, uint32_t heads_first, uint32_t entries, uint32_t u) {
    const uint32_t run = heads_first != 0u ? entries : v.heads;
    const uint32_t vector = u >> v.head_shift, d = u - (vector << v.head_shift);
    const uint32_t outer = run == 1u ? vector : vector / run, inner = vector - outer * run;
    return outer * (heads_first != 0u ? v.head_stride : v.entry_stride) +
           inner * (heads_first != 0u ? v.entry_stride : v.head_stride) + d * 16u;
}

// Units of 16 bytes that a thread copies at once. Whole pages go in pieces of two
// (256 pages of 128 KB in ten caches, 1.34 GB: 253 us, 5.3 TB/s; in four 265, in
// sixteen 269), parts of pages in four, as fewer blocks find nothing to do (290 of up
// to 32 KB: 46 and 51 us).
constexpr uint32_t kAhead = 4, kWholeAhead = 2;

// Piece `piece` of the first `entries` of a page of array n.
template <uint32_t AHEAD>
struct PieceOfPage {
    static constexpr uint32_t kPiece = kThreads * AHEAD;
    u32x4 x[AHEAD];

    __device__ __forceinline__ void load(const CachesView &from, uint32_t n, uint32_t page, uint32_t entries,
                                         uint32_t piece) {
        const uint32_t units = entries * from.heads << from.head_shift;
        const char *const a = from.data[n] + page * from.page_stride;
#pragma unroll
        for (uint32_t i = 0; i < AHEAD; ++i) {
            const uint32_t u = piece * kPiece + i * kThreads + threadIdx.x;
            if (u < units) {
                x[i] = *reinterpret_cast<const u32x4 *>(a + unit_at(from, from.heads_first, entries, u));
            }
        }
    }
    // (in the order of the source's)
    __device__ __forceinline__ void store(const CachesView &from, const CachesView &to, uint32_t n, uint32_t page,
                                          uint32_t entries, uint32_t piece) const {
        const uint32_t units = entries * from.heads << from.head_shift;
        char *const b = to.data[n] + page * to.page_stride;
#pragma unroll
        for (uint32_t i = 0; i < AHEAD; ++i) {
            const uint32_t u = piece * kPiece + i * kThreads + threadIdx.x;
            if (u < units) {
                *reinterpret_cast<u32x4 *>(b + unit_at(to, from.heads_first, entries, u)) = x[i];
            }
        }
    }
};

struct CopyArgs {
    CachesView from, to;
    const uint32_t *sources, *targets, *entries;
    uint32_t pieces;
};

template <uint32_t AHEAD>
__global__ __launch_bounds__(kThreads) void k_paged_copy(CopyArgs args) {
    const uint32_t piece = blockIdx.x % args.pieces, rest = blockIdx.x / args.pieces;
    const uint32_t n = rest % args.from.arrays, i = rest / args.from.arrays;
    const uint32_t source = args.sources[i], target = args.targets[i];
    uint32_t entries = args.from.page_size;
    if (args.entries != nullptr) {
        entries = min(entries, args.entries[i]);
    }
    if (source < args.from.pages && target < args.to.pages) {
        PieceOfPage<AHEAD> x;
        x.load(args.from, n, source, entries, piece);
        x.store(args.from, args.to, n, target, entries, piece);
    }
}

// ---- counts of a pool's segments -----------------------------------------------

// The sum of `own` over the threads below this one, and in `all` over the block.
// `sums`: kWaves words of LDS, free for use when every thread is here.
__device__ __forceinline__ uint32_t block_before(uint32_t own, uint32_t *sums, uint32_t &all) {
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x / kWave;
    uint32_t sum = own;
#pragma unroll
    for (uint32_t step = 1; step < 64u; step <<= 1) {
        const uint32_t below = static_cast<uint32_t>(__shfl_up(static_cast<int>(sum), step));
        sum += lane >= step ? below : 0u;
    }
    __syncthreads();
    if (lane == 63u) {
        sums[wave] = sum;
    }
    __syncthreads();
    uint32_t before = sum - own;
    all = 0u;
    for (uint32_t w = 0; w < kWaves; ++w) {
        before += w < wave ? sums[w] : 0u;
        all += sums[w];
    }
    return before;
}

// What a fork's first launch leaves for its second, of each row: the entries that
// it and its parent held (0: no parent), its new ones, the parent's row; the page
// of which the first entries are copied (kNone: none), and how many pages rows
// before it take.
struct RowPlan {
    uint32_t held, parents, added, parent;
    uint32_t source, before, demand, over;
};

struct ForkArgs {
    const uint32_t *old_lengths, *old_table, *old_references;
    uint32_t old_stride;
    uint32_t *lengths, *table, *references;
    uint32_t stride, max_length;
    const uint32_t *offsets, *parents;
    uint32_t rows, beams, page_shift, pages, segments;
    uint32_t tokens, max_tokens;
    uint32_t *lacking;
    // workspace
    RowPlan *plan;
    uint32_t *free_count, *free_page;  // [segments], [segments][kSegment]; in a small pool [1], [pages]
    uint32_t *demand;                  // of all rows
    uint32_t small;
    uint32_t *ticket;  // of a tiny pool, zero between calls
};

__device__ __forceinline__ uint32_t pages_of(uint32_t entries, uint32_t shift) {
    return (entries >> shift) + ((entries & ((1u << shift) - 1u)) != 0u ? 1u : 0u);
}

// A row's plan, but for the pages that rows before it take (no row: one that takes none).
__device__ __forceinline__ RowPlan plan_of(const ForkArgs &args, uint32_t row) {
    RowPlan plan{0u, 0u, 0u, kNone, kNone, 0u, 0u, 0u};
    if (row >= args.rows) {
        return plan;
    }
    const uint32_t page_mask = (1u << args.page_shift) - 1u;
    const uint32_t group = row / args.beams * args.beams, parent = args.parents[row];
    const uint32_t a = min(args.offsets[row], args.tokens), b = min(args.offsets[row + 1u], args.tokens);
    plan.held = args.old_lengths[row];
    plan.added = b > a ? b - a : 0u;
    if (parent < args.beams) {
        plan.parent = group + parent;
        plan.parents = args.old_lengths[plan.parent];
    }
    const uint64_t next = static_cast<uint64_t>(plan.parents) + plan.added;
    plan.over = plan.added > args.max_tokens || next > args.max_length ? 1u : 0u;
    if (plan.over == 0u) {
        plan.demand = pages_of(plan.parents + plan.added, args.page_shift) -
                      pages_of(plan.parents, args.page_shift);
        const uint32_t last = plan.parents >> args.page_shift;
        if ((plan.parents & page_mask) != 0u && plan.added != 0u && last < args.old_stride) {
            const uint32_t page = args.old_table[static_cast<uint64_t>(plan.parent) * args.old_stride + last];
            bool eldest = true;
            for (uint32_t others = group; others < row; others += 8u) {
                uint32_t of_others[8];
#pragma unroll
                for (uint32_t i = 0; i < 8u; ++i) {
                    of_others[i] = args.parents[min(others + i, row)];
                }
#pragma unroll
                for (uint32_t i = 0; i < 8u; ++i) {
                    eldest = eldest && (others + i >= row || of_others[i] != parent);
                }
            }
            if (page < args.pages && !(eldest && args.old_references[page] == 1u)) {
                plan.source = page;
                plan.demand += 1u;
            }
        }
    }
    return plan;
}

// The rows' plans by the first block (bound by its chain of loads: a row's parent, its
// length, its last page, the page's count: 4 rows 3.7 us, 128 5.2; one block, so that a
// row's place among those that take pages is a sum within it). Of a small pool
// (kSmallPages) it counts the free pages too, a run of them a thread, and lists the first
// of them, as many as rows take; of others every block but the first lists a segment's.
// The others copy the counts, where the new ones are apart from the old.
__global__ __launch_bounds__(kThreads) void k_fork_plan(ForkArgs args) {
    __shared__ uint32_t sums[kWaves];
    const uint32_t t = threadIdx.x;
    if (blockIdx.x != 0u) {
        const uint32_t segment = blockIdx.x - 1u, first = segment * kSegment + t * kOwn;
        uint32_t count[kOwn], own = 0u;
#pragma unroll
        for (uint32_t i = 0; i < kOwn; ++i) {
            count[i] = first + i < args.pages ? args.old_references[first + i] : 1u;
            own += count[i] == 0u ? 1u : 0u;
        }
        if (args.references != args.old_references) {
#pragma unroll
            for (uint32_t i = 0; i < kOwn; ++i) {
                if (first + i < args.pages) {
                    args.references[first + i] = count[i];
                }
            }
        }
        if (args.small != 0u) {
            return;
        }
        uint32_t all = 0u, at = block_before(own, sums, all);
        uint32_t *const list = args.free_page + segment * kSegment;
#pragma unroll
        for (uint32_t i = 0; i < kOwn; ++i) {
            if (count[i] == 0u) {
                list[at++] = first + i;
            }
        }
        if (t == 0u) {
            args.free_count[segment] = all;
        }
        return;
    }
    // (on its way while the rows are planned; a run past the pool's end has no free ones)
    constexpr uint32_t kRun = kSmallPages / kThreads;
    uint32_t count[kRun];
    const uint32_t run = (args.pages + kThreads - 1u) / kThreads;
    if (args.small != 0u) {
#pragma unroll
        for (uint32_t i = 0; i < kRun; ++i) {
            if (i < run) {
                count[i] = args.old_references[min(t * run + i, args.pages - 1u)];
            }
        }
    }
    uint32_t taken = 0u;
    for (uint32_t base = 0; base < args.rows; base += kThreads) {
        const uint32_t row = base + t;
        RowPlan plan = plan_of(args, row);
        uint32_t all = 0u;
        plan.before = taken + block_before(plan.demand, sums, all);
        taken += all;
        if (row < args.rows) {
            args.plan[row] = plan;
        }
    }
    if (t == 0u) {
        *args.demand = taken;
    }
    if (args.small == 0u) {
        return;
    }
    uint32_t own = 0u;
#pragma unroll
    for (uint32_t i = 0; i < kRun; ++i) {
        if (i < run) {
            count[i] = t * run + i < args.pages ? count[i] : 1u;
            own += count[i] == 0u ? 1u : 0u;
        }
    }
    uint32_t all = 0u, at = block_before(own, sums, all);
#pragma unroll
    for (uint32_t i = 0; i < kRun; ++i) {
        if (i < run && count[i] == 0u) {
            if (at < taken) {
                args.free_page[at] = t * run + i;
            }
            ++at;
        }
    }
    if (t == 0u) {
        args.free_count[0] = all;
    }
}

// A pool's free pages as a wave finds them: a lane counts those of a run of
// segments, and knows the number up to its run's end.
struct FreePages {
    uint32_t up_to, run, all;

    __device__ __forceinline__ explicit FreePages(const ForkArgs &args) {
        const uint32_t lane = threadIdx.x & 63u;
        if (args.small != 0u) {
            run = 1u;
            up_to = all = args.free_count[0];
            return;
        }
        run = (args.segments + kWave - 1u) / kWave;
        up_to = 0u;
        for (uint32_t s = lane * run; s < min(lane * run + run, args.segments); ++s) {
            up_to += args.free_count[s];
        }
#pragma unroll
        for (uint32_t step = 1; step < kWave; step <<= 1) {
            const uint32_t below = static_cast<uint32_t>(__shfl_up(static_cast<int>(up_to), step));
            up_to += lane >= step ? below : 0u;
        }
        all = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(up_to), kWave - 1));
    }
    // The n-th of them, kNone where there are not as many. Every lane is here.
    __device__ __forceinline__ uint32_t nth(const ForkArgs &args, uint32_t n) const {
        if (args.small != 0u) {
            return n < all ? args.free_page[n] : kNone;
        }
        // the first lane whose run ends beyond it
        uint32_t owner = 0u;
#pragma unroll
        for (uint32_t step = kWave / 2u; step != 0u; step >>= 1) {
            const uint32_t end = static_cast<uint32_t>(__shfl(static_cast<int>(up_to), static_cast<int>(owner + step - 1u)));
            owner += end <= n ? step : 0u;
        }
        const uint32_t before = static_cast<uint32_t>(__shfl(static_cast<int>(up_to), static_cast<int>(owner == 0u ? 0u : owner - 1u)));
        if (n >= all) {
            return kNone;
        }
        uint32_t left = n - (owner == 0u ? 0u : before), s = owner * run;
        while (run > 1u && left >= args.free_count[s]) {
            left -= args.free_count[s];
            ++s;
        }
        return args.free_page[s * kSegment + left];
    }
};

struct ForkCopyArgs {
    CachesView caches;
    uint32_t pieces, table_blocks, column_blocks;
    uint64_t work;  // pieces of all rows and arrays
    uint32_t in_place;
};

// Column c of a request's rows (its first is `group`), parent by parent: each entry is
// read before any is written, so that the old table may be the new one. Counts change by take(page), a
// page's first holder, and add(page, change); nth(n) is the n-th free page. Every
// thread of the block is here.
template <uint32_t K, typename Nth, typename Take, typename Add>
__device__ __forceinline__ void fork_column(const ForkArgs &args, const RowPlan *plans, uint32_t group, uint32_t c,
                                            Nth &&nth, Take &&take, Add &&add) {
    uint32_t x[K], kept[K];
#pragma unroll
    for (uint32_t q = 0; q < K; ++q) {
        x[q] = kNone;
        kept[q] = 0u;
        if (q < args.beams && c < min(pages_of(plans[q].held, args.page_shift), args.old_stride)) {
            x[q] = args.old_table[static_cast<uint64_t>(group + q) * args.old_stride + c];
        }
    }
    // a lane's row, read from there by its number
    const uint32_t lane = threadIdx.x & 63u;
    const RowPlan own = plans[min(lane, args.beams - 1u)];
    const auto of_row = [](uint32_t v, uint32_t row) {
        return static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v), static_cast<int>(row)));
    };
    const auto child = [&](uint32_t s, uint32_t parents_page, uint32_t &keeps) {
        const uint32_t parents = of_row(own.parents, s), added = of_row(own.added, s);
        const bool has_source = of_row(own.source, s) != kNone;
        const uint32_t held = pages_of(parents, args.page_shift);
        const uint32_t end = static_cast<uint32_t>(
            min((static_cast<uint64_t>(parents) + added + (1u << args.page_shift) - 1u) >> args.page_shift,
                static_cast<uint64_t>(args.stride)));
        const bool copies = c < end && has_source && c == parents >> args.page_shift;
        const bool takes = copies || (c < end && c >= held && of_row(own.over, s) == 0u);
        uint32_t page = !takes && c < held ? parents_page : kNone;
        keeps += c < end && !takes && c < held ? 1u : 0u;
        if (__ballot(takes) != 0u) {
            const uint32_t n = of_row(own.before, s) + (copies ? 0u : c - held + (has_source ? 1u : 0u));
            const uint32_t taken = nth(takes ? n : kNone);
            if (takes && taken != kNone) {
                page = taken;
                take(page);
            }
        }
        if (c < end) {
            args.table[static_cast<uint64_t>(group + s) * args.stride + c] = page;
        }
        if (c == 0u) {
            args.lengths[group + s] =
                static_cast<uint32_t>(min(static_cast<uint64_t>(parents) + added, uint64_t(kNone)));
        }
    };
    const uint32_t parent = lane < args.beams ? own.parent - group : K;
#pragma unroll
    for (uint32_t q = 0; q < K; ++q) {
        for (uint64_t left = __ballot(parent == q); left != 0u; left &= left - 1u) {
            child(static_cast<uint32_t>(__builtin_ctzll(left)), x[q], kept[q]);
        }
    }
    uint32_t none = 0u;
    for (uint64_t left = __ballot(lane < args.beams && own.parent == kNone); left != 0u; left &= left - 1u) {
        child(static_cast<uint32_t>(__builtin_ctzll(left)), kNone, none);
    }
    // a page's holders of the request, counted once where they follow each other
    uint32_t page = kNone, change = 0u;
#pragma unroll
    for (uint32_t q = 0; q < K; ++q) {
        if (x[q] < args.pages) {
            if (x[q] != page) {
                if (change != 0u) {
                    add(page, change);
                }
                page = x[q];
                change = 0u;
            }
            change += kept[q] - 1u;
        }
    }
    if (change != 0u) {
        add(page, change);
    }
}

// The tables, a column of a request's rows a thread, and the copies: what a block
// copies is on its way before it knows where it goes. (Bound by a chain of
// four loads, 4.2 us for 4 rows in ten caches, and by a request's rows one after another
// where they take pages, half a microsecond each; 32 requests of 4, half of whose rows
// copy parts of pages, 22 MB in all, 8.0 us.)
template <uint32_t K>
__global__ __launch_bounds__(kThreads) void k_fork_apply(ForkArgs args, ForkCopyArgs copy) {
    __shared__ RowPlan plans[K];
    const uint32_t t = threadIdx.x;
    if (blockIdx.x >= copy.table_blocks) {
        for (uint64_t w = blockIdx.x - copy.table_blocks; w < copy.work; w += gridDim.x - copy.table_blocks) {
            const uint32_t piece = static_cast<uint32_t>(w % copy.pieces);
            const uint64_t rest = w / copy.pieces;
            const uint32_t n = static_cast<uint32_t>(rest % copy.caches.arrays);
            const RowPlan plan = args.plan[rest / copy.caches.arrays];
            const uint32_t entries = plan.parents & ((1u << args.page_shift) - 1u);
            if (plan.source != kNone) {
                PieceOfPage<kAhead> x;
                x.load(copy.caches, n, plan.source, entries, piece);
                const uint32_t target = FreePages(args).nth(args, plan.before);
                if (target != kNone) {
                    x.store(copy.caches, copy.caches, n, target, entries, piece);
                }
            }
        }
        return;
    }
    const FreePages free(args);
    if (blockIdx.x == 0u && t == 0u && args.lacking != nullptr) {
        *args.lacking = *args.demand > free.all ? *args.demand - free.all : 0u;
    }
    const uint32_t group = blockIdx.x / copy.column_blocks * args.beams;
    const uint32_t c = blockIdx.x % copy.column_blocks * kThreads + t;
    if (t < args.beams) {
        plans[t] = args.plan[group + t];
    }
    __syncthreads();
    fork_column<K>(
        args, plans, group, c, [&](uint32_t n) { return free.nth(args, n); },
        [&](uint32_t page) { args.references[page] = 1u; },
        [&](uint32_t page, uint32_t change) { atomicAdd(&args.references[page], change); });
}

// Tiny pools and few rows in one launch: every block plans all rows and finds the free
// pages, and takes its share of the copies. One block writes the tables, lengths and
// counts (counted in LDS): the first, which copies nothing, or where any of them are the
// old ones too the last through the ticket, when all have read them. (Bound by its
// chain: the plan's four loads, the sums' barriers, the tables: 5.6 us for 4 rows, where
// two launches take 8.)
template <uint32_t K>
__global__ __launch_bounds__(kThreads) void k_fork_tiny(ForkArgs args, ForkCopyArgs copy) {
    constexpr uint32_t kRun = kTinyPages / kThreads;
    __shared__ RowPlan plans[kThreads];
    __shared__ uint32_t counts[kTinyPages];
    __shared__ uint16_t free[kTinyPages];
    __shared__ uint32_t sums[kWaves];
    __shared__ uint32_t arrived;
    const uint32_t t = threadIdx.x, run = (args.pages + kThreads - 1u) / kThreads, first = t * run;
    uint32_t count[kRun], own = 0u;
#pragma unroll
    for (uint32_t i = 0; i < kRun; ++i) {
        count[i] = i < run ? args.old_references[min(first + i, args.pages - 1u)] : 1u;
    }
    RowPlan plan = plan_of(args, t);
    uint32_t demand = 0u, all = 0u;
    plan.before = block_before(plan.demand, sums, demand);
    plans[t] = plan;
#pragma unroll
    for (uint32_t i = 0; i < kRun; ++i) {
        count[i] = i < run && first + i < args.pages ? count[i] : 1u;
        own += count[i] == 0u ? 1u : 0u;
    }
    uint32_t at = block_before(own, sums, all);
#pragma unroll
    for (uint32_t i = 0; i < kRun; ++i) {
        if (count[i] == 0u) {
            free[at++] = static_cast<uint16_t>(first + i);
        }
    }
    if (t == 0u && copy.in_place != 0u) {
        arrived = coherent_add(args.ticket, 1u);
    }
    __syncthreads();
    const uint32_t copiers = copy.in_place != 0u ? gridDim.x : gridDim.x - 1u;
    if (copy.in_place != 0u || blockIdx.x != 0u) {
        for (uint32_t w = blockIdx.x - (gridDim.x - copiers); w < copy.work; w += copiers) {
            const uint32_t piece = w % copy.pieces, rest = w / copy.pieces;
            const uint32_t n = rest % copy.caches.arrays;
            const RowPlan row = plans[rest / copy.caches.arrays];
            if (row.source != kNone && row.before < all) {
                const uint32_t entries = row.parents & ((1u << args.page_shift) - 1u);
                PieceOfPage<kAhead> x;
                x.load(copy.caches, n, row.source, entries, piece);
                x.store(copy.caches, copy.caches, n, free[row.before], entries, piece);
            }
        }
    }
    if (copy.in_place != 0u ? arrived != gridDim.x - 1u : blockIdx.x != 0u) {
        return;
    }
#pragma unroll
    for (uint32_t i = 0; i < kRun; ++i) {
        if (i < run && first + i < args.pages) {
            counts[first + i] = count[i];
        }
    }
    __syncthreads();
    for (uint32_t b = 0; b < copy.table_blocks; ++b) {
        const uint32_t group = b / copy.column_blocks * args.beams;
        fork_column<K>(
            args, plans + group, group, b % copy.column_blocks * kThreads + t,
            [&](uint32_t n) { return n < all ? static_cast<uint32_t>(free[n]) : kNone; },
            [&](uint32_t page) { counts[page] = 1u; },
            [&](uint32_t page, uint32_t change) { atomicAdd(&counts[page], change); });
    }
    __syncthreads();
#pragma unroll
    for (uint32_t i = 0; i < kRun; ++i) {
        if (i < run && first + i < args.pages) {
            args.references[first + i] = counts[first + i];
        }
    }
    if (t == 0u) {
        if (args.lacking != nullptr) {
            *args.lacking = demand > all ? demand - all : 0u;
        }
        if (copy.in_place != 0u) {
            coherent_store(args.ticket, 0u);
        }
    }
}

// A batch of no rows: the counts as they were, and no page lacks.
__global__ __launch_bounds__(kThreads) void k_fork_none(const uint32_t *old_references, uint32_t *references,
                                                        uint32_t pages, uint32_t *lacking) {
    const uint32_t i = blockIdx.x * kThreads + threadIdx.x;
    if (i < pages) {
        references[i] = old_references[i];
    }
    if (i == 0u && lacking != nullptr) {
        *lacking = 0u;
    }
}

// ---- compaction -----------------------------------------------------------------

struct CompactArgs {
    const uint32_t *old_references, *old_table, *lengths;
    uint32_t *references, *table;
    uint32_t rows, stride, columns, page_shift, pages, segments;
    uint32_t *live;
    // workspace
    uint32_t *count;                     // live pages of each segment
    uint32_t *sources, *targets, *rank;  // [pages / 2] twice, [pages]
    uint32_t *moves;
    uint32_t *ticket;  // of a tiny pool, zero between calls
};

// The free and live pages of long pools, a segment a block.
__global__ __launch_bounds__(kThreads) void k_compact_count(CompactArgs args) {
    __shared__ uint32_t sums[kWaves];
    const uint32_t first = blockIdx.x * kSegment + threadIdx.x * kOwn;
    uint32_t own = 0u;
#pragma unroll
    for (uint32_t i = 0; i < kOwn; ++i) {
        own += first + i < args.pages && args.old_references[first + i] != 0u ? 1u : 0u;
    }
    uint32_t all = 0u;
    (void)block_before(own, sums, all);
    if (threadIdx.x == 0u) {
        args.count[blockIdx.x] = all;
    }
}

// The live pages before every segment's, in LDS (`before`, kSegments + 1 words).
__device__ __forceinline__ void segments_before(const uint32_t *count, uint32_t segments, uint32_t *before,
                                                uint32_t *sums) {
    uint32_t done = 0u;
    for (uint32_t base = 0; base < segments; base += kThreads) {
        const uint32_t s = base + threadIdx.x;
        uint32_t all = 0u;
        const uint32_t at = done + block_before(s < segments ? count[s] : 0u, sums, all);
        if (s < segments) {
            before[s] = at;
        }
        done += all;
    }
    if (threadIdx.x == 0u) {
        before[segments] = done;
    }
    __syncthreads();
}

// The n-th live page behind the first `live` moves to the n-th free one below it.
// (Of a small pool every block reads all counts, so that no launch before it has to.
// Bound by its loads and block-wide sums, one after another: 100 pages 4.3 us, 4,096
// 6.)
__global__ __launch_bounds__(kThreads) void k_compact_plan(CompactArgs args) {
    constexpr uint32_t kSmall = kSmallPages / kSegment;
    __shared__ uint32_t before[kSegments + 1u];
    __shared__ uint32_t sums[kWaves];
    const uint32_t t = threadIdx.x;
    // of each segment, a bit for each of the thread's pages that is held
    uint32_t holds = 0u, first_below = 0u, border = 0u;
    uint32_t mine[kOwn];
    const uint32_t first = blockIdx.x * kSegment + t * kOwn;
    if (args.pages <= kSmallPages) {
        uint32_t held[kSmall], count[kSmall][kOwn];
#pragma unroll
        for (uint32_t s = 0; s < kSmall; ++s) {
#pragma unroll
            for (uint32_t i = 0; i < kOwn; ++i) {
                count[s][i] = args.old_references[min(s * kSegment + t * kOwn + i, args.pages - 1u)];
            }
        }
        uint32_t done = 0u;
#pragma unroll
        for (uint32_t s = 0; s < kSmall; ++s) {
            held[s] = 0u;
#pragma unroll
            for (uint32_t i = 0; i < kOwn; ++i) {
                held[s] |= s * kSegment + t * kOwn + i < args.pages && count[s][i] != 0u ? 1u << i : 0u;
            }
            uint32_t all = 0u;
            (void)block_before(static_cast<uint32_t>(__popc(held[s])), sums, all);
            if (t == 0u) {
                before[s] = done;
            }
            done += all;
        }
        if (t == 0u) {
            before[kSmall] = done;
            before[args.segments] = done;
        }
        border = done / kSegment;
#pragma unroll
        for (uint32_t s = 0; s < kSmall; ++s) {
            holds = s == blockIdx.x ? held[s] : holds;
            first_below = s == border ? held[s] : first_below;
#pragma unroll
            for (uint32_t i = 0; i < kOwn; ++i) {
                mine[i] = s == blockIdx.x ? count[s][i] : mine[i];
            }
        }
        __syncthreads();
    } else {
        segments_before(args.count, args.segments, before, sums);
        border = before[args.segments] / kSegment;
#pragma unroll
        for (uint32_t i = 0; i < kOwn; ++i) {
            mine[i] = first + i < args.pages ? args.old_references[first + i] : 0u;
            holds |= mine[i] != 0u ? 1u << i : 0u;
            const uint32_t edge = border * kSegment + t * kOwn + i;
            first_below |= edge < args.pages && args.old_references[edge] != 0u ? 1u << i : 0u;
        }
    }
    const uint32_t live = before[args.segments];
    if (args.references != args.old_references) {
#pragma unroll
        for (uint32_t i = 0; i < kOwn; ++i) {
            if (first + i < args.pages) {
                args.references[first + i] = mine[i];
            }
        }
    }
    uint32_t all = 0u, at = before[blockIdx.x] + block_before(static_cast<uint32_t>(__popc(holds)), sums, all);
    // live pages below `live`: of the segments before its own, and in that
    uint32_t below = 0u;
#pragma unroll
    for (uint32_t i = 0; i < kOwn; ++i) {
        below += border * kSegment + t * kOwn + i < live ? first_below >> i & 1u : 0u;
    }
    uint32_t in_border = 0u;
    (void)block_before(below, sums, in_border);
    const uint32_t kept = before[border] + in_border;
#pragma unroll
    for (uint32_t i = 0; i < kOwn; ++i) {
        const uint32_t page = first + i;
        const bool lives = (holds >> i & 1u) != 0u;
        if (page < args.pages) {
            if (page >= live) {
                // (held, but counted as free: it has no new number)
                args.rank[page] = lives ? at - kept : kNone;
                if (lives) {
                    args.sources[at - kept] = page;
                }
            } else if (!lives) {
                args.targets[page - at] = page;
            }
        }
        at += lives ? 1u : 0u;
    }
    if (blockIdx.x == 0u && t == 0u) {
        *args.moves = live - kept;
        *args.live = live;
    }
}

struct CompactCopyArgs {
    CachesView caches;
    uint32_t pieces, table_blocks;
    uint32_t counts;  // 1: the counts are written too
};

// The moves and the tables: blocks in turn over what the plan counted, as the host does
// not know how much it is (908 of 4,096 pages of 16 KB in ten caches' keys and values,
// 595 MB read and written: 121.6 us, 4.9 TB/s, HBM's rate for a copy).
__global__ __launch_bounds__(kThreads) void k_compact_apply(CompactArgs args, CompactCopyArgs copy) {
    const uint32_t moves = *args.moves, live = *args.live;
    if (blockIdx.x >= copy.table_blocks) {
        const uint64_t work = static_cast<uint64_t>(moves) * copy.caches.arrays * copy.pieces;
        for (uint64_t w = blockIdx.x - copy.table_blocks; w < work; w += gridDim.x - copy.table_blocks) {
            const uint32_t piece = static_cast<uint32_t>(w % copy.pieces);
            const uint64_t rest = w / copy.pieces;
            const uint32_t n = static_cast<uint32_t>(rest % copy.caches.arrays);
            const uint64_t i = rest / copy.caches.arrays;
            const uint32_t source = args.sources[i], target = args.targets[i];
            PieceOfPage<kAhead> x;
            x.load(copy.caches, n, source, 1u << args.page_shift, piece);
            x.store(copy.caches, copy.caches, n, target, 1u << args.page_shift, piece);
        }
        return;
    }
    const uint32_t step = copy.table_blocks * kThreads;
    for (uint32_t i = blockIdx.x * kThreads + threadIdx.x; i < moves; i += step) {
        const uint32_t source = args.sources[i], target = args.targets[i];
        args.references[target] = args.references[source];
        args.references[source] = 0u;
    }
    for (uint64_t i = blockIdx.x * kThreads + threadIdx.x; i < static_cast<uint64_t>(args.rows) * args.columns;
         i += step) {
        const uint32_t row = static_cast<uint32_t>(i / args.columns), c = static_cast<uint32_t>(i % args.columns);
        if (c < pages_of(args.lengths[row], args.page_shift)) {
            const uint64_t at = static_cast<uint64_t>(row) * args.stride + c;
            const uint32_t page = args.old_table[at];
            const uint32_t rank = page >= live && page < args.pages ? args.rank[page] : kNone;
            args.table[at] = rank != kNone ? args.targets[rank] : page;
        }
    }
}

// A tiny pool in one launch: every block reads all counts and finds all moves, and
// takes its share of them and of the tables. The counts are written by one block: the
// first, or where they are the old ones too, the last through the ticket, when all
// have read them. (100 pages: 4.9 us, two launches 7.8.)
__global__ __launch_bounds__(kThreads) void k_compact_tiny(CompactArgs args, CompactCopyArgs copy) {
    constexpr uint32_t kRun = kTinyPages / kThreads;
    __shared__ uint32_t sums[kWaves];
    __shared__ uint16_t sources[kTinyPages / 2u], targets[kTinyPages / 2u], name[kTinyPages];
    __shared__ uint32_t kept_below, arrived;
    const uint32_t t = threadIdx.x, run = (args.pages + kThreads - 1u) / kThreads, first = t * run;
    const bool in_place = args.references == args.old_references;
    uint32_t count[kRun], held = 0u;
#pragma unroll
    for (uint32_t i = 0; i < kRun; ++i) {
        count[i] = i < run ? args.old_references[min(first + i, args.pages - 1u)] : 0u;
    }
#pragma unroll
    for (uint32_t i = 0; i < kRun; ++i) {
        count[i] = i < run && first + i < args.pages ? count[i] : 0u;
        held |= count[i] != 0u ? 1u << i : 0u;
    }
    uint32_t live = 0u;
    const uint32_t before = block_before(static_cast<uint32_t>(__popc(held)), sums, live);
    if (live - first < run) {
        kept_below = before + static_cast<uint32_t>(__popc(held & ((1u << (live - first)) - 1u)));
    } else if (t == 0u && live == kThreads * run) {
        kept_below = live;
    }
    if (t == 0u && in_place && copy.counts != 0u) {
        arrived = coherent_add(args.ticket, 1u);
    }
    __syncthreads();
    const uint32_t kept = kept_below, moves = live - kept;
    uint32_t at = before;
#pragma unroll
    for (uint32_t i = 0; i < kRun; ++i) {
        const bool lives = (held >> i & 1u) != 0u;
        const uint32_t page = first + i;
        if (i < run && page < args.pages) {
            if (lives && page >= live) {
                sources[at - kept] = static_cast<uint16_t>(page);
            } else if (!lives && page < live) {
                targets[page - at] = static_cast<uint16_t>(page);
            }
        }
        at += lives ? 1u : 0u;
    }
    __syncthreads();
    if (blockIdx.x >= copy.table_blocks) {
        // (pieces of 16 KB of memory that exists: their number fits)
        const uint32_t work = moves * copy.caches.arrays * copy.pieces;
        for (uint32_t w = blockIdx.x - copy.table_blocks; w < work; w += gridDim.x - copy.table_blocks) {
            const uint32_t piece = w % copy.pieces, rest = w / copy.pieces;
            const uint32_t n = rest % copy.caches.arrays, i = rest / copy.caches.arrays;
            PieceOfPage<kAhead> x;
            x.load(copy.caches, n, sources[i], 1u << args.page_shift, piece);
            x.store(copy.caches, copy.caches, n, targets[i], 1u << args.page_shift, piece);
        }
    } else {
        at = before;
#pragma unroll
        for (uint32_t i = 0; i < kRun; ++i) {
            const bool lives = (held >> i & 1u) != 0u;
            const uint32_t page = first + i;
            if (i < run && page < args.pages) {
                name[page] = lives && page >= live ? targets[at - kept] : static_cast<uint16_t>(page);
            }
            at += lives ? 1u : 0u;
        }
        __syncthreads();
        const uint32_t step = copy.table_blocks * kThreads;
        for (uint64_t i = blockIdx.x * kThreads + t; i < static_cast<uint64_t>(args.rows) * args.columns; i += step) {
            const uint32_t row = static_cast<uint32_t>(i / args.columns), c = static_cast<uint32_t>(i % args.columns);
            if (c < pages_of(args.lengths[row], args.page_shift)) {
                const uint64_t place = static_cast<uint64_t>(row) * args.stride + c;
                const uint32_t page = args.old_table[place];
                args.table[place] = page < args.pages ? name[page] : page;
            }
        }
    }
    if (blockIdx.x == 0u && t == 0u) {
        *args.live = live;
    }
    if (copy.counts == 0u || (in_place ? arrived != gridDim.x - 1u : blockIdx.x != 0u)) {
        return;
    }
    at = before;
#pragma unroll
    for (uint32_t i = 0; i < kRun; ++i) {
        const bool lives = (held >> i & 1u) != 0u;
        const uint32_t page = first + i;
        if (i < run && page < args.pages) {
            if (page >= live) {
                count[i] = 0u;
            } else if (!lives) {
                count[i] = args.old_references[sources[page - at]];
            }
        }
        at += lives ? 1u : 0u;
    }
    __syncthreads();
#pragma unroll
    for (uint32_t i = 0; i < kRun; ++i) {
        if (i < run && first + i < args.pages) {
            args.references[first + i] = count[i];
        }
    }
    if (t == 0u && in_place) {
        coherent_store(args.ticket, 0u);
    }
}

// ---- checks and launches ----------------------------------------------------------

void require_caches(const adi_hip_paged_cache *caches, uint32_t count) {
    require(caches != nullptr && count >= 1 && count <= kMaxCaches, "paged pool: caches must be 1 to 1024");
    adi_hip_paged_batch none{};
    for (uint32_t i = 0; i < count; ++i) {
        require_paged(&caches[i], &none);
        const adi_hip_paged_cache &a = caches[0], &b = caches[i];
        require(a.type == b.type && a.heads == b.heads && a.head_size == b.head_size && a.page_size == b.page_size &&
                    a.pages == b.pages && a.page_stride == b.page_stride && a.entry_stride == b.entry_stride &&
                    a.head_stride == b.head_stride,
                "paged pool: the caches of a pool must be of one type and layout");
    }
    require(caches[0].pages <= kMaxPages, "paged pool: more than 2^22 pages");
    // (a page's units are counted in 32 bits)
    require(uint64_t(caches[0].heads) * caches[0].head_size * caches[0].page_size < (1u << 30),
            "paged pool: a page of 2^30 elements or more");
}

void require_pool(const adi_hip_paged_pool *pool) {
    require(pool != nullptr, "paged pool: null descriptor");
    require_caches(pool->cache, pool->caches);
}

void require_counted(const adi_hip_paged_pool *pool) {
    require_pool(pool);
    require(pool->references != nullptr && aligned_to(pool->references, 4) && aligned_to(pool->lacking, 4),
            "paged pool: null or unaligned references");
}

uint32_t pieces_of(const adi_hip_paged_cache &c, uint32_t entries, uint32_t ahead) {
    return ceil_div(uint64_t(entries) * c.heads * c.head_size * type_bytes(c.type) / 16u, kThreads * ahead);
}

void require_fork(const adi_hip_paged_pool *pool, const adi_hip_paged_batch *batch,
                  const adi_hip_paged_fork_arguments *a) {
    require_counted(pool);
    require_paged(&pool->cache[0], batch);
    require(a != nullptr, "paged fork: null arguments");
    require(a->beams >= 1 && a->beams <= kMaxBeams && batch->sequences % a->beams == 0,
            "paged fork: beams must be 1 to 64, and sequences a multiple of them");
    if (batch->sequences == 0) {
        require(aligned_to(a->references, 4), "paged fork: unaligned argument");
        return;
    }
    require(a->parents != nullptr && a->lengths != nullptr && a->table != nullptr && a->references != nullptr &&
                batch->table != nullptr && batch->table_stride >= 1 && a->table_stride >= 1,
            "paged fork: null argument");
    require(aligned_to(a->parents, 4) && aligned_to(a->lengths, 4) && aligned_to(a->table, 4) &&
                aligned_to(a->references, 4),
            "paged fork: unaligned argument");
    require(a->table != batch->table || a->table_stride == batch->table_stride,
            "paged fork: the tables overlap with different strides");
    require(uint64_t(batch->sequences / a->beams) * ceil_div(std::max(a->table_stride, batch->table_stride), kThreads) <
                (1u << 22),
            "paged fork: the tables are too large");
}

struct Scratch {
    char *at;
    uint64_t left;
    template <typename T>
    T *take(uint64_t count) {
        const uint64_t bytes = (count * sizeof(T) + 255u) & ~uint64_t(255);
        if (bytes > left) {
            fail(ADI_HIP_OUT_OF_MEMORY, "paged pool: the workspace is too small for the pool's pages and rows");
        }
        T *const p = reinterpret_cast<T *>(at);
        at += bytes;
        left -= bytes;
        return p;
    }
};

Scratch scratch_of(adi_hip_context *ctx, const adi_hip_paged_workspace *workspace) {
    require(workspace != nullptr, "paged pool: null workspace");
    require(workspace->device == ctx->device, "paged pool: the workspace is on another device");
    return {static_cast<char *>(workspace->base) + kTickets * sizeof(uint32_t),
            workspace->bytes - kTickets * sizeof(uint32_t)};
}

void paged_fork(adi_hip_context *ctx, const adi_hip_paged_pool *pool, const adi_hip_paged_batch *batch,
                const adi_hip_paged_fork_arguments *a, const adi_hip_paged_workspace *workspace) {
    require_fork(pool, batch, a);
    Scratch scratch = scratch_of(ctx, workspace);
    const adi_hip_paged_cache &c = pool->cache[0];
    if (batch->sequences == 0) {
        const uint32_t copied = a->references != nullptr && a->references != pool->references ? c.pages : 0u;
        if (copied != 0u || pool->lacking != nullptr) {
            launch(ctx, "fork_none", k_fork_none, dim3(std::max(ceil_div(copied, kThreads), 1u)), dim3(kThreads), 0,
                   a->references, pool->references, copied, pool->lacking);
        }
        return;
    }
    ForkArgs args{};
    args.old_lengths = a->lengths;
    args.old_table = a->table;
    args.old_references = a->references;
    args.old_stride = a->table_stride;
    args.lengths = const_cast<uint32_t *>(batch->lengths);
    args.table = const_cast<uint32_t *>(batch->table);
    args.references = pool->references;
    args.stride = batch->table_stride;
    args.max_length = batch->max_length;
    args.offsets = batch->offsets;
    args.parents = a->parents;
    args.rows = batch->sequences;
    args.beams = a->beams;
    args.page_shift = log2_of(c.page_size);
    args.pages = c.pages;
    args.segments = ceil_div(c.pages, kSegment);
    args.tokens = batch->tokens;
    args.max_tokens = batch->max_tokens;
    args.lacking = pool->lacking;
    ForkCopyArgs copy{};
    copy.pieces = pieces_of(c, c.page_size - 1u, kAhead);
    copy.column_blocks = ceil_div(std::max(args.old_stride, args.stride), kThreads);
    copy.table_blocks = args.rows / args.beams * copy.column_blocks;
    copy.work = uint64_t(args.rows) * 2u * std::min(pool->caches, kCaches) * copy.pieces;
    copy.in_place = args.lengths == args.old_lengths || args.table == args.old_table ||
                    args.references == args.old_references;
    const auto of_beams = [&](auto &&go) {
        if (args.beams <= 4) {
            go(std::integral_constant<uint32_t, 4>());
        } else if (args.beams <= 16) {
            go(std::integral_constant<uint32_t, 16>());
        } else {
            go(std::integral_constant<uint32_t, 64>());
        }
    };
    if (c.pages <= kTinyPages && args.rows <= kThreads && pool->caches <= kCaches && (copy.table_blocks == 1u || copy.table_blocks * args.beams <= kTinyTables) &&
        copy.work <= (copy.in_place != 0u ? 1u : kTinyCopiers) * ctx->cu_count) {
        args.ticket = static_cast<uint32_t *>(workspace->base);
        copy.caches = caches_view(*pool, 0);
        const dim3 grid(static_cast<uint32_t>(copy.work) + (copy.in_place != 0u ? 0u : 1u)), block(kThreads);
        of_beams([&](auto k) {
            launch(ctx, "fork_tiny", k_fork_tiny<decltype(k)::value>, grid, block, 0, args, copy);
        });
        return;
    }
    args.plan = scratch.take<RowPlan>(args.rows);
    args.free_count = scratch.take<uint32_t>(args.segments);
    args.free_page = scratch.take<uint32_t>(uint64_t(args.segments) * kSegment);
    args.demand = scratch.take<uint32_t>(1);
    args.small = c.pages <= kSmallPages ? 1u : 0u;
    const uint32_t others = args.small != 0u && args.references == args.old_references ? 0u : args.segments;
    launch(ctx, "fork_plan", k_fork_plan, dim3(1u + others), dim3(kThreads), 0, args);
    for (uint32_t first = 0; first < pool->caches; first += kCaches) {
        copy.caches = caches_view(*pool, first);
        copy.work = uint64_t(args.rows) * copy.caches.arrays * copy.pieces;
        const uint32_t copiers = static_cast<uint32_t>(std::min<uint64_t>(copy.work, 16u * ctx->cu_count));
        const dim3 grid(copy.table_blocks + copiers), block(kThreads);
        of_beams([&](auto k) {
            launch(ctx, "fork_apply", k_fork_apply<decltype(k)::value>, grid, block, 0, args, copy);
        });
        copy.table_blocks = 0;
    }
}

void require_copy(const adi_hip_paged_pool *from, const adi_hip_paged_pool *to, const uint32_t *sources,
                  const uint32_t *targets, const uint32_t *entries, uint32_t count) {
    require_pool(from);
    require_pool(to);
    const adi_hip_paged_cache &a = from->cache[0], &b = to->cache[0];
    require(from->caches == to->caches && a.type == b.type && a.heads == b.heads && a.head_size == b.head_size &&
                a.page_size == b.page_size,
            "paged copy: pools of different caches");
    require(count <= kMaxPages, "paged copy: more than 2^22 pages");
    require(count == 0 || (sources != nullptr && targets != nullptr && aligned_to(sources, 4) &&
                           aligned_to(targets, 4) && aligned_to(entries, 4)),
            "paged copy: null or unaligned argument");
}

void paged_copy(adi_hip_context *ctx, const adi_hip_paged_pool *from, const adi_hip_paged_pool *to,
                const uint32_t *sources, const uint32_t *targets, const uint32_t *entries, uint32_t count) {
    require_copy(from, to, sources, targets, entries, count);
    CopyArgs args{};
    args.pieces = pieces_of(from->cache[0], from->cache[0].page_size, entries != nullptr ? kAhead : kWholeAhead);
    for (uint32_t first = 0; first < from->caches; first += kCaches) {
        args.from = caches_view(*from, first);
        args.to = caches_view(*to, first);
        const uint64_t each = uint64_t(args.from.arrays) * args.pieces;
        const uint64_t at_once = std::max<uint64_t>((1u << 23) / each, 1u);
        for (uint64_t done = 0; done < count; done += at_once) {
            const uint64_t n = std::min<uint64_t>(at_once, count - done);
            args.sources = sources + done;
            args.targets = targets + done;
            args.entries = entries != nullptr ? entries + done : nullptr;
            const dim3 grid(static_cast<uint32_t>(n * each)), block(kThreads);
            if (entries != nullptr) {
                launch(ctx, "paged_copy", k_paged_copy<kAhead>, grid, block, 0, args);
            } else {
                launch(ctx, "paged_copy", k_paged_copy<kWholeAhead>, grid, block, 0, args);
            }
        }
    }
}

void require_compact(const adi_hip_paged_pool *pool, const adi_hip_paged_compact_arguments *a) {
    require_counted(pool);
    require(a != nullptr && a->references != nullptr && a->live != nullptr && aligned_to(a->references, 4) &&
                aligned_to(a->live, 4),
            "paged compact: null or unaligned argument");
    require(a->rows <= (1u << 20), "paged compact: more than 2^20 rows");
    require(a->rows == 0 || (a->lengths != nullptr && a->table != nullptr && a->next_table != nullptr &&
                             a->table_stride >= 1 && aligned_to(a->lengths, 4) && aligned_to(a->table, 4) &&
                             aligned_to(a->next_table, 4)),
            "paged compact: null or unaligned table");
}

void paged_compact(adi_hip_context *ctx, const adi_hip_paged_pool *pool, const adi_hip_paged_compact_arguments *a,
                   const adi_hip_paged_workspace *workspace) {
    require_compact(pool, a);
    Scratch scratch = scratch_of(ctx, workspace);
    const adi_hip_paged_cache &c = pool->cache[0];
    CompactArgs args{};
    args.old_references = a->references;
    args.old_table = a->table;
    args.lengths = a->lengths;
    args.references = pool->references;
    args.table = a->next_table;
    args.rows = a->rows;
    args.stride = a->table_stride;
    args.columns = a->table_stride;
    args.page_shift = log2_of(c.page_size);
    args.pages = c.pages;
    args.segments = ceil_div(c.pages, kSegment);
    args.live = a->live;
    CompactCopyArgs copy{};
    copy.pieces = pieces_of(c, c.page_size, kAhead);
    const uint64_t work = uint64_t(c.pages / 2u) * 2u * std::min(pool->caches, kCaches) * copy.pieces;
    const bool tiny = c.pages <= kTinyPages && (work <= ctx->cu_count || args.references != args.old_references);
    const uint64_t words = std::max<uint64_t>(uint64_t(a->rows) * args.columns, tiny ? 1u : c.pages / 2u + 1u);
    const uint32_t table_blocks =
        static_cast<uint32_t>(std::min<uint64_t>((words + kThreads - 1) / kThreads, ctx->cu_count));
    const auto copiers = [&](uint32_t a_cu) {
        return static_cast<uint32_t>(std::min<uint64_t>(uint64_t(c.pages / 2u) * copy.caches.arrays * copy.pieces,
                                                        a_cu * ctx->cu_count));
    };
    if (tiny) {
        args.ticket = static_cast<uint32_t *>(workspace->base);
        for (uint32_t first = 0; first < pool->caches; first += kCaches) {
            // the tables and counts are the last launch's, as they may be the old ones
            const bool last = pool->caches - first <= kCaches;
            copy.caches = caches_view(*pool, first);
            copy.table_blocks = last ? table_blocks : 0u;
            copy.counts = last ? 1u : 0u;
            const uint32_t blocks = copy.table_blocks + copiers(kTinyCopiers);
            if (blocks != 0) {
                launch(ctx, "compact_tiny", k_compact_tiny, dim3(blocks), dim3(kThreads), 0, args, copy);
            }
        }
        return;
    }
    args.count = scratch.take<uint32_t>(args.segments);
    args.sources = scratch.take<uint32_t>(c.pages / 2u);
    args.targets = scratch.take<uint32_t>(c.pages / 2u);
    args.rank = scratch.take<uint32_t>(c.pages);
    args.moves = scratch.take<uint32_t>(1);
    if (c.pages > kSmallPages) {
        launch(ctx, "compact_count", k_compact_count, dim3(args.segments), dim3(kThreads), 0, args);
    }
    launch(ctx, "compact_plan", k_compact_plan, dim3(args.segments), dim3(kThreads), 0, args);
    copy.table_blocks = table_blocks;
    for (uint32_t first = 0; first < pool->caches; first += kCaches) {
        copy.caches = caches_view(*pool, first);
        launch(ctx, "compact_apply", k_compact_apply, dim3(copy.table_blocks + copiers(16u)), dim3(kThreads), 0, args,
               copy);
        copy.table_blocks = 0;
    }
}

}  // namespace
}  // namespace adi_hip

using namespace adi_hip;

extern "C" {

int adi_hip_paged_fork(adi_hip_context *ctx, const adi_hip_paged_pool *pool, const adi_hip_paged_batch *batch,
                       const adi_hip_paged_fork_arguments *arguments, adi_hip_paged_workspace *workspace) {
    return guarded(ctx, [&] { paged_fork(ctx, pool, batch, arguments, workspace); });
}

int adi_hip_paged_copy(adi_hip_context *ctx, const adi_hip_paged_pool *from, const adi_hip_paged_pool *to,
                       const uint32_t *sources, const uint32_t *targets, const uint32_t *entries, uint32_t count) {
    return guarded(ctx, [&] { paged_copy(ctx, from, to, sources, targets, entries, count); });
}

int adi_hip_paged_compact(adi_hip_context *ctx, const adi_hip_paged_pool *pool,
                          const adi_hip_paged_compact_arguments *arguments, adi_hip_paged_workspace *workspace) {
    return guarded(ctx, [&] { paged_compact(ctx, pool, arguments, workspace); });
}

int adi_hip_paged_fork_check(const adi_hip_paged_pool *pool, const adi_hip_paged_batch *batch,
                             const adi_hip_paged_fork_arguments *arguments) {
    return guarded_host([&] { require_fork(pool, batch, arguments); });
}

int adi_hip_paged_copy_check(const adi_hip_paged_pool *from, const adi_hip_paged_pool *to, const uint32_t *sources,
                             const uint32_t *targets, const uint32_t *entries, uint32_t count) {
    return guarded_host([&] { require_copy(from, to, sources, targets, entries, count); });
}

int adi_hip_paged_compact_check(const adi_hip_paged_pool *pool, const adi_hip_paged_compact_arguments *arguments) {
    return guarded_host([&] { require_compact(pool, arguments); });
}

}  // extern "C"
