// paged.hip -- the paged cache of many sequences: its checks on the host, the
// append of new keys and values, and the workspace of its attention
// (paged_attention.hip).
//
// Append: per head of a new token an RMS norm (where weighted), the rotation
// to the token's position, and one rounding into the cache's type, with the
// queries' norm and rotation in the same launch (normalize_head and apply_rope,
// src/executor.cpp:25-72, and the cache writes of 392-400, for many sequences).
#include "paged.hpp"

#include "paged_attention.hpp"

namespace adi_hip {

void require_paged(const adi_hip_paged_cache *cache, const adi_hip_paged_batch *batch) {
    require(cache != nullptr && batch != nullptr, "paged cache: null descriptor");
    require(known_type(cache->type), "paged cache: unknown type");
    require(cache->heads >= 1 && cache->heads <= 65536, "paged cache: heads must be 1 to 65536");
    require(cache->head_size == 64 || cache->head_size == 128 || cache->head_size == 256,
            "paged cache: head size must be 64, 128 or 256");
    require(is_power_of_two(cache->page_size) && cache->page_size >= 8 && cache->page_size <= 4096,
            "paged cache: page size must be a power of two, 8 to 4096");
    require(cache->pages >= 1, "paged cache: no pages");
    const uint64_t step = 16u / type_bytes(cache->type);
    require(cache->keys != nullptr && cache->values != nullptr && aligned_to(cache->keys, 16) &&
                aligned_to(cache->values, 16) && cache->page_stride % step == 0 && cache->entry_stride % step == 0 &&
                cache->head_stride % step == 0,
            "paged cache: keys, values and strides must be 16-byte aligned");
    require(batch->max_length < (1u << 28), "paged batch: max_length must be below 2^28");
    require(batch->max_tokens <= batch->tokens && batch->tokens < (1u << 30),
            "paged batch: max_tokens must be at most tokens, tokens below 2^30");
    require(batch->sequences <= (1u << 20), "paged batch: more than 2^20 sequences");
    require(batch->sequences == 0 || (batch->offsets != nullptr && batch->lengths != nullptr),
            "paged batch: null offsets or lengths");
    require(batch->sequences == 0 || batch->max_length == 0 ||
                (batch->table != nullptr &&
                 batch->table_stride >= (batch->max_length + cache->page_size - 1) / cache->page_size),
            "paged batch: the page table is shorter than max_length");
}

PagedView paged_view(const adi_hip_paged_cache &cache, const adi_hip_paged_batch &batch) {
    return {static_cast<char *>(cache.keys), static_cast<char *>(cache.values), cache.page_stride, cache.entry_stride,
            cache.head_stride, log2_of(cache.page_size), cache.pages, cache.heads, batch.offsets, batch.lengths,
            batch.table, batch.table_stride, batch.sequences, batch.tokens, batch.max_tokens, batch.max_length};
}

namespace {

constexpr uint32_t kThreads = 256;

struct AppendArgs {
    PagedView c;
    RowsView keys, values, queries, queries_out;
    const uint16_t *key_norm, *query_norm;
    const double *turns;       // [half], or
    const float *sines;        // [position][half cosines, half sines], or neither
    uint32_t half, pairs;      // rotary / 2; whether 2 i and 2 i + 1 turn together
    float magnitude;
    uint32_t query_heads, parts;
    uint32_t run;              // tokens of a block, one after another
    float weight_offset, epsilon;
};

// Sum over the L lanes of a row (a power of two, aligned).
template <uint32_t L>
__device__ __forceinline__ float row_sum(float v) {
    v += lane_xor<1>(v);
    v += lane_xor<2>(v);
    v += lane_xor<4>(v);
    if constexpr (L > 8) {
        v += lane_xor<8>(v);
    }
    if constexpr (L > 16) {
        v += lane_xor<16>(v);
    }
    if constexpr (L > 32) {
        v += lane_xor<32>(v);
    }
    return v;
}

template <typename T, uint32_t N>
struct alignas(sizeof(T) * N < 16u ? sizeof(T) * N : 16u) Vector {
    T v[N];
};

constexpr uint32_t kAhead = 2;  // tokens whose rows are on their way

// A part of the heads (queries, then keys, then values) of a run of tokens, D / N
// lanes a head of N = 16 bytes of input each, so a head stays within a wave.
// The token's sequence is the number of sequences that end at or before it,
// counted 64 at a time with what is needed of them; its sines go through LDS once
// a block, a head's partner dimensions through the wave's own piece of LDS.
//
// Bound by a block's chain of loads (offsets and lengths, page, store) where the
// tokens are few (3.8 us for one, 4.3 for 32), by the rows' bytes where they are
// many: 2,919 tokens of 32 + 8 + 8 heads of 128 in bf16, 72 MB, take 16.1 us, 4.5
// TB/s (19 where none of it is in the last-level cache). A block a token and part waited out that chain and its sines for every
// one, and read its partners from LDS by the element: 28.9.
template <typename R, typename C, uint32_t D>
__global__ __launch_bounds__(kThreads) void k_paged_append(AppendArgs args) {
    constexpr uint32_t N = 16u / sizeof(R), L = D / N, kRows = kThreads / L;
    __shared__ __align__(16) float cosine[D / 2u], sine[D / 2u];
    __shared__ __align__(16) float turned[kThreads * N];
    const PagedView &c = args.c;
    const uint32_t t = threadIdx.x, lane = t & 63u, at = (t % L) * N;
    const uint32_t rows = args.query_heads + 2u * c.heads;
    const bool whole = args.half % (args.pairs != 0u ? N / 2u : N) == 0u;
    // (at most D / 2 of them, so one a thread)
    const double turns = args.turns != nullptr && t < args.half ? args.turns[t] : 0.0;
    const uint32_t row = blockIdx.x % args.parts * kRows + t / L;
    const bool live = row < rows;
    // 0 queries, 1 keys, 2 values
    const uint32_t kind = row < args.query_heads ? 0u : row < args.query_heads + c.heads ? 1u : 2u;
    const uint32_t head = kind == 0u ? row : (row - args.query_heads) - (kind - 1u) * c.heads;
    const RowsView &source = kind == 0u ? args.queries : kind == 1u ? args.keys : args.values;
    const R *const in = reinterpret_cast<const R *>(source.data) + head * source.head_stride + at;
    const uint64_t in_stride = source.token_stride;
    R *const out = reinterpret_cast<R *>(args.queries_out.data) + head * args.queries_out.head_stride + at;
    C *const pool = reinterpret_cast<C *>(kind == 1u ? c.keys : c.values) + head * c.head_stride + at;
    const uint16_t *const norm = kind == 0u ? args.query_norm : kind == 1u ? args.key_norm : nullptr;
    const bool norms = args.query_norm != nullptr || args.key_norm != nullptr;
    float weight[N];
    if (norms) {
#pragma unroll
        for (uint32_t k = 0; k < N; ++k) {
            weight[k] = norm != nullptr ? args.weight_offset + bf16_of(norm[at + k]) : 1.0f;
        }
    }
    const uint32_t from = blockIdx.x / args.parts * args.run, to = min(from + args.run, c.tokens);
    using V = Vector<R, N>;
    V next[kAhead] = {};
#pragma unroll
    for (uint32_t u = 0; u < kAhead; ++u) {
        if (live && from + u < to) {
            next[u] = *reinterpret_cast<const V *>(in + (from + u) * in_stride);
        }
    }
    uint32_t sequence = ~0u, page = ~0u, page_index = ~0u;
    SequenceRows rows_of{};
    for (uint32_t token = from; token < to; ++token) {
        float x[N];
#pragma unroll
        for (uint32_t k = 0; k < N; ++k) {
            x[k] = static_cast<float>(next[0].v[k]);
        }
#pragma unroll
        for (uint32_t u = 0; u + 1u < kAhead; ++u) {
            next[u] = next[u + 1u];
        }
        if (live && token + kAhead < to) {
            next[kAhead - 1u] = *reinterpret_cast<const V *>(in + (token + kAhead) * in_stride);
        }
        if (sequence == ~0u || token - rows_of.first >= rows_of.count) {
            sequence = ~0u;
            page_index = ~0u;
            for (uint32_t s = 0; s < c.sequences; s += 64u) {
                const uint32_t own = min(s + lane, c.sequences - 1u);
                const uint32_t a = min(c.offsets[own], c.tokens), b = min(c.offsets[own + 1u], c.tokens);
                const uint32_t length = c.lengths[own];
                const uint32_t ended =
                    static_cast<uint32_t>(__popcll(__ballot(s + lane < c.sequences && b <= token)));
                if (ended < 64u) {
                    if (s + ended < c.sequences) {
                        const auto of = [&](uint32_t v) {
                            return static_cast<uint32_t>(
                                __builtin_amdgcn_readlane(static_cast<int>(v), static_cast<int>(ended)));
                        };
                        const uint32_t first = of(a), end = of(b);
                        sequence = s + ended;
                        rows_of.first = first;
                        rows_of.count = end > first ? end - first : 0u;
                        rows_of.length = of(length);
                        rows_of.over = rows_of.count > c.max_tokens || rows_of.length > c.max_length;
                    }
                    break;
                }
            }
        }
        // (uniform over the block)
        if (sequence == ~0u || token < rows_of.first || token - rows_of.first >= rows_of.count) {
            continue;
        }
        const int64_t place = static_cast<int64_t>(rows_of.length) - rows_of.count + (token - rows_of.first);
        const bool held = !rows_of.over && place >= 0;
        const uint32_t position = held ? static_cast<uint32_t>(place) : 0u;
        if (!held) {
            page = ~0u;
            page_index = ~0u;
        } else if (position >> c.page_shift != page_index) {
            page_index = position >> c.page_shift;
            page = c.table[static_cast<uint64_t>(sequence) * c.table_stride + page_index];
        }
        if (norms) {
            float squares = 0.0f;
#pragma unroll
            for (uint32_t k = 0; k < N; ++k) {
                squares += x[k] * x[k];
            }
            squares = row_sum<L>(squares);
            const float scale = norm != nullptr ? 1.0f / sqrtf(squares / static_cast<float>(D) + args.epsilon) : 1.0f;
#pragma unroll
            for (uint32_t k = 0; k < N; ++k) {
                x[k] *= scale * weight[k];
            }
        }
        if (args.half != 0u) {
            if (token != from) {
                __syncthreads();  // the last token's sines are used
            }
            if (t < args.half) {
                if (args.sines != nullptr) {
                    const float *values = args.sines + static_cast<uint64_t>(position) * 2u * args.half;
                    cosine[t] = values[t];
                    sine[t] = values[args.half + t];
                } else {
                    const Turn turn = turn_of(position, turns);
                    cosine[t] = turn.cosine * args.magnitude;
                    sine[t] = turn.sine * args.magnitude;
                }
            }
            float *const own = turned + t / L * D;
            if (args.pairs == 0u) {
                // (read back behind the barrier)
                store_values<float, N>(own + at, x);
            }
            __syncthreads();
            if (kind != 2u && at < 2u * args.half) {
                float y[N] = {};
                if (whole) {
                    // the lane's dimensions are all first or all second ones of
                    // their pairs, or whole pairs: LDS in 16 bytes (by the
                    // element, lanes 32 bytes apart meet on eight banks)
                    using F = Vector<float, N>;
                    using H = Vector<float, N / 2u>;
                    if (args.pairs != 0u) {
                        const H w = *reinterpret_cast<const H *>(cosine + at / 2u);
                        const H z = *reinterpret_cast<const H *>(sine + at / 2u);
#pragma unroll
                        for (uint32_t k = 0; k < N; ++k) {
                            y[k] = k & 1u ? x[k] * w.v[k / 2u] + x[k ^ 1u] * z.v[k / 2u]
                                          : x[k] * w.v[k / 2u] - x[k ^ 1u] * z.v[k / 2u];
                        }
                    } else {
                        const bool second = at >= args.half;
                        const uint32_t pair = second ? at - args.half : at;
                        const F w = *reinterpret_cast<const F *>(cosine + pair);
                        const F z = *reinterpret_cast<const F *>(sine + pair);
                        const F other = *reinterpret_cast<const F *>(own + (second ? pair : pair + args.half));
                        const float sign = second ? 1.0f : -1.0f;
#pragma unroll
                        for (uint32_t k = 0; k < N; ++k) {
                            y[k] = x[k] * w.v[k] + other.v[k] * (sign * z.v[k]);
                        }
                    }
                } else {
#pragma unroll 1
                    for (uint32_t k = 0; k < N; ++k) {
                        const uint32_t d = at + k;
                        float value = x[0];
#pragma unroll
                        for (uint32_t i = 1; i < N; ++i) {
                            value = i == k ? x[i] : value;
                        }
                        if (d < 2u * args.half) {
                            float beside = 0.0f;
#pragma unroll
                            for (uint32_t i = 0; i < N; ++i) {
                                beside = (i ^ 1u) == k ? x[i] : beside;
                            }
                            const bool second = args.pairs != 0u ? (k & 1u) != 0u : d >= args.half;
                            const uint32_t pair = args.pairs != 0u ? d >> 1 : second ? d - args.half : d;
                            const float other = args.pairs != 0u ? beside : own[second ? pair : d + args.half];
                            value = value * cosine[pair] + (second ? other : -other) * sine[pair];
                        }
#pragma unroll
                        for (uint32_t i = 0; i < N; ++i) {
                            y[i] = i == k ? value : y[i];
                        }
                    }
                }
#pragma unroll
                for (uint32_t k = 0; k < N; ++k) {
                    x[k] = y[k];
                }
            }
        }
        if (live && kind == 0u) {
            if (rows_of.over) {
#pragma unroll
                for (uint32_t k = 0; k < N; ++k) {
                    x[k] = __builtin_nanf("");
                }
            }
            store_values<R, N>(out + token * args.queries_out.token_stride, x);
        } else if (live && page < c.pages) {
            store_values<C, N>(pool + page * c.page_stride + (position & ((1u << c.page_shift) - 1u)) * c.entry_stride,
                               x);
        }
    }
}

template <typename R, typename C, uint32_t D>
void launch_append(adi_hip_context *ctx, AppendArgs args) {
    constexpr uint32_t kRows = kThreads / (D / (16u / sizeof(R)));
    args.parts = ceil_div(args.query_heads + 2u * args.c.heads, kRows);
    // runs of tokens where there are more than six blocks a CU, what their registers
    // let it hold (2,919 tokens, of an earlier form: 17.6 us; 3, 4, 8 and 12 blocks 19.4, 17.8, 18.8, 19.0)
    const uint64_t jobs = static_cast<uint64_t>(args.c.tokens) * args.parts;
    args.run = std::max(ceil_div(jobs, 6u * static_cast<uint64_t>(ctx->cu_count)), 1u);
    const uint64_t grid = static_cast<uint64_t>(ceil_div(args.c.tokens, args.run)) * args.parts;
    require(grid < (1u << 23), "paged append: too many heads");
    launch(ctx, "paged_append", k_paged_append<R, C, D>, dim3(static_cast<uint32_t>(grid)), dim3(kThreads), 0, args);
}

template <typename R, typename C>
void launch_append(adi_hip_context *ctx, const AppendArgs &args, uint32_t head_size) {
    if (head_size == 64) {
        launch_append<R, C, 64>(ctx, args);
    } else if (head_size == 128) {
        launch_append<R, C, 128>(ctx, args);
    } else {
        launch_append<R, C, 256>(ctx, args);
    }
}

}  // namespace

void paged_append(adi_hip_context *ctx, const adi_hip_paged_cache *cache, const adi_hip_paged_batch *batch,
                  const adi_hip_paged_append_arguments *a, const float *sines, uint32_t sines_half) {
    require_paged(cache, batch);
    require(a != nullptr, "paged append: null arguments");
    const uint32_t type = a->keys.type;
    require(known_type(type) && (type == cache->type || (type == ADI_HIP_F32 && cache->type == ADI_HIP_BF16)),
            "paged append: f32 rows go into an f32 or bf16 cache, others into their own type");
    require(a->query_heads <= 65536, "paged append: more than 65536 query heads");
    require(a->rope == nullptr || (a->rope->device == ctx->device && a->rope->rotary <= cache->head_size),
            "paged append: the rotation has more dimensions than a head, or is on another device");
    require(std::isfinite(a->weight_offset) && std::isfinite(a->epsilon) && a->epsilon >= 0.0f,
            "paged append: weight offset or epsilon is not valid");
    if (batch->tokens == 0 || batch->sequences == 0) {
        return;
    }
    require_rows(a->keys, type, "paged append: keys must be 16-byte aligned rows");
    require_rows(a->values, type, "paged append: values must be 16-byte aligned rows of the keys' type");
    require(aligned_to(a->key_norm, 2) && aligned_to(a->query_norm, 2), "paged append: unaligned norm weight");
    if (a->query_heads != 0) {
        require_rows(a->queries, type, "paged append: queries must be 16-byte aligned rows of the keys' type");
        require_rows(a->queries_out, type, "paged append: query outputs must be 16-byte aligned rows of the keys' type");
        require(same_rows(a->queries, a->queries_out) || a->queries.data != a->queries_out.data,
                "paged append: the query outputs overlap the queries");
    }
    const bool weighted = a->query_heads != 0;
    AppendArgs args{paged_view(*cache, *batch), rows_view(a->keys), rows_view(a->values), rows_view(a->queries),
                    rows_view(a->queries_out), a->key_norm, weighted ? a->query_norm : nullptr, nullptr, sines,
                    sines_half, 0, 1.0f, a->query_heads, 0, 1, a->weight_offset, a->epsilon};
    if (a->rope != nullptr) {
        args.turns = a->rope->turns;
        args.half = a->rope->rotary / 2;
        args.pairs = a->rope->layout == ADI_HIP_ROPE_PAIRS ? 1u : 0u;
        args.magnitude = a->rope->magnitude;
    }
    if (type == ADI_HIP_F32 && cache->type == ADI_HIP_F32) {
        launch_append<float, float>(ctx, args, cache->head_size);
    } else if (type == ADI_HIP_F32) {
        launch_append<float, __bf16>(ctx, args, cache->head_size);
    } else if (type == ADI_HIP_F16) {
        launch_append<_Float16, _Float16>(ctx, args, cache->head_size);
    } else {
        launch_append<__bf16, __bf16>(ctx, args, cache->head_size);
    }
}

}  // namespace adi_hip

using namespace adi_hip;

extern "C" {

int adi_hip_paged_check(const adi_hip_paged_cache *cache, const adi_hip_paged_batch *batch) {
    return guarded_host([&] {
        require_paged(cache, batch);
        for (uint32_t s = 0; s < batch->sequences; ++s) {
            const std::string name = "paged batch: sequence " + std::to_string(s);
            const uint32_t begin = batch->offsets[s], end = batch->offsets[s + 1];
            if (end < begin || end > batch->tokens) {
                fail(ADI_HIP_INVALID_ARGUMENT, name + "'s rows do not ascend within the batch's");
            }
            if (end - begin > batch->max_tokens) {
                fail(ADI_HIP_INVALID_ARGUMENT, name + " has more than max_tokens rows");
            }
            if (batch->lengths[s] > batch->max_length) {
                fail(ADI_HIP_INVALID_ARGUMENT, name + " has more than max_length entries");
            }
            for (uint32_t p = 0; p * cache->page_size < batch->lengths[s]; ++p) {
                if (batch->table[static_cast<size_t>(s) * batch->table_stride + p] >= cache->pages) {
                    fail(ADI_HIP_INVALID_ARGUMENT, name + "'s page " + std::to_string(p) + " is not one of the cache's");
                }
            }
        }
    });
}

int adi_hip_paged_append(adi_hip_context *ctx, const adi_hip_paged_cache *cache, const adi_hip_paged_batch *batch,
                         const adi_hip_paged_append_arguments *arguments) {
    return guarded(ctx, [&] { paged_append(ctx, cache, batch, arguments, nullptr, 0); });
}

int adi_hip_paged_workspace_create(adi_hip_context *ctx, size_t bytes, adi_hip_paged_workspace **out) {
    return guarded(ctx, [&] {
        require(out != nullptr, "paged workspace: null output");
        *out = nullptr;
        bytes = bytes == 0 ? size_t(64) << 20 : bytes;
        require(bytes >= size_t(1) << 20, "paged workspace: at least 1 MiB");
        void *base = nullptr;
        check_hip(hipMalloc(&base, bytes), "paged workspace allocation");
        hipError_t error = hipMemset(base, 0, kTickets * sizeof(uint32_t));
        if (error == hipSuccess) {
            error = hipDeviceSynchronize();
        }
        if (error != hipSuccess) {
            (void)hipFree(base);
            check_hip(error, "paged workspace tickets");
        }
        auto *workspace = new (std::nothrow) adi_hip_paged_workspace{ctx->device, base, bytes};
        if (workspace == nullptr) {
            (void)hipFree(base);
            throw std::bad_alloc();
        }
        *out = workspace;
    });
}

void adi_hip_paged_workspace_destroy(adi_hip_paged_workspace *workspace) {
    if (workspace == nullptr) {
        return;
    }
    int previous = 0;
    (void)hipGetDevice(&previous);
    (void)hipSetDevice(workspace->device);
    (void)hipDeviceSynchronize();
    (void)hipFree(workspace->base);
    (void)hipSetDevice(previous);
    delete workspace;
}

int adi_hip_paged_attention(adi_hip_context *ctx, const adi_hip_paged_cache *cache, const adi_hip_paged_batch *batch,
                            const adi_hip_paged_attention_arguments *arguments, adi_hip_paged_workspace *workspace) {
    return guarded(ctx, [&] { paged_attention(ctx, cache, batch, arguments, workspace); });
}

}  // extern "C"
