// paged_attention.hip -- causal grouped attention of new tokens of many
// sequences over a paged cache (grouped_query_online_attention,
// src/attention.cpp:40, for ragged batches).
//
// A row is a query head of a new token; the rows of a KV head, (token, query
// head of the group) in order, read the same entries. Scores are formed
// transposed, S^T = K Q^T, and so is the output, O^T += V^T P^T: a lane of S^T's
// result holds some keys of one row, and that is the second product's operand as
// it stands, with the values taken in the same order of keys. A row's maximum
// and sum live in the lanes of its column.
//
// Two kernels. k_paged_step: up to 16 rows a KV head (a decode step's tokens):
// a wave streams its tiles from the cache straight into operands, the waves of
// a block and the blocks of a long history are joined. k_paged_chunk: more rows,
// 128 a block, over tiles staged in LDS.
//
// Floats on the 16-bit matrix cores: an f32 value is the exact sum of three bf16
// pieces, each the leading 8 bits of what is left (truncated, so that none
// overflows), and a product is the sum of the piece products down to 2^-16 of
// it; what is left out is below 2^-22 of the largest.
#include "paged_attention.hpp"

#include <type_traits>

namespace adi_hip {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

constexpr uint32_t kThreads = 256;
constexpr uint32_t kStepRows = 16;    // of a KV head, k_paged_step
constexpr uint32_t kStepKeys = 32;    // a wave's tile
constexpr uint32_t kChunkRows = 128;  // of a block, k_paged_chunk
constexpr uint32_t kChunkKeys = 32;   // a block's tile
constexpr uint32_t kSpanUnit = 128;   // parts of a history are multiples of this
constexpr float kNegative = -__builtin_huge_valf();

struct AttendArgs {
    PagedView c;
    RowsView queries, outputs, gate;
    float log2_scale;     // scale log2 e
    uint32_t window;
    uint32_t group;       // query heads of a KV head
    uint32_t span, parts; // entries of a part of a history, parts at most
    uint32_t tiles;       // k_paged_chunk: row tiles of a sequence at most
    float *partial;       // [part][token][head][D + 4]: sums, maximum, denominator (parts > 1)
};

// A part's row in the workspace.
template <uint32_t D>
__device__ __forceinline__ float *partial_row(const AttendArgs &a, uint32_t part, uint32_t token, uint32_t head) {
    const uint64_t heads = static_cast<uint64_t>(a.c.heads) * a.group;
    return a.partial + ((static_cast<uint64_t>(part) * a.c.tokens + token) * heads + head) * (D + 4u);
}

// Where a sequence's parts begin: 0, or with a window at or before the first
// entry its first row sees.
__device__ __forceinline__ int32_t base_of(const AttendArgs &a, int32_t first_position) {
    const int32_t first = first_position - static_cast<int32_t>(a.window) + 1;
    return a.window == 0u || first <= 0 ? 0 : first & ~static_cast<int32_t>(kSpanUnit - 1u);
}

// exp2(log2_scale (s - m)), s not above m: for f32 rows the difference is taken
// first, so that its rounding is relative to it; for 16-bit rows in one
// multiply-add.
template <bool EXACT>
__device__ __forceinline__ float weight_of(float s, float m, float log2_scale) {
    if constexpr (EXACT) {
        return __builtin_amdgcn_exp2f((s - m) * log2_scale);
    } else {
        return __builtin_amdgcn_exp2f(fmaf(s, log2_scale, -m * log2_scale));
    }
}

template <typename T>
__device__ __forceinline__ uint32_t pack(float x, float y) {
    const f32x2 v = {x, y};
    if constexpr (std::is_same_v<T, _Float16>) {
        return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, f16x2));
    } else {
        return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, bf16x2));
    }
}

// Two floats as pairs of 16-bit pieces: one, rounded to nearest, or three whose
// sum they are, exactly (an infinity or NaN is its first piece).
template <typename T, uint32_t N>
__device__ __forceinline__ void split(float x, float y, uint32_t (&out)[N]) {
    if constexpr (N == 1) {
        out[0] = pack<T>(x, y);
    } else {
#pragma unroll
        for (uint32_t i = 0; i < N; ++i) {
            const uint32_t a = __float_as_uint(x), b = __float_as_uint(y);
            out[i] = __builtin_amdgcn_perm(b, a, 0x07060302u);
            const float ra = x - __uint_as_float(a & 0xFFFF0000u), rb = y - __uint_as_float(b & 0xFFFF0000u);
            x = (a & 0x7F800000u) == 0x7F800000u ? 0.0f : ra;
            y = (b & 0x7F800000u) == 0x7F800000u ? 0.0f : rb;
        }
    }
}

template <typename T>
__device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
    if constexpr (std::is_same_v<T, _Float16>) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0,
                                                      0, 0);
    } else {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c,
                                                       0, 0, 0);
    }
}
template <typename T>
__device__ __forceinline__ f32x16 mfma(u32x4 a, u32x4 b, f32x16 c) {
    if constexpr (std::is_same_v<T, _Float16>) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0,
                                                      0, 0);
    } else {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c,
                                                       0, 0, 0);
    }
}

// The piece products of a K step, smallest first.
template <typename T, uint32_t A, uint32_t B, typename C>
__device__ __forceinline__ C product(const u32x4 (&a)[A], const u32x4 (&b)[B], C c) {
#pragma unroll
    for (int32_t order = 2; order >= 0; --order) {
#pragma unroll
        for (int32_t i = 0; i < static_cast<int32_t>(A); ++i) {
            const int32_t j = order - i;
            if (j >= 0 && j < static_cast<int32_t>(B)) {
                c = mfma<T>(a[i], b[j], c);
            }
        }
    }
    return c;
}

// Whether either 16-bit value of a pair is an infinity or NaN.
template <typename T>
__device__ __forceinline__ bool odd_pair(uint32_t v) {
    constexpr uint32_t kOnes = std::is_same_v<T, _Float16> ? 0x7C00u : 0x7F80u;
    return (v & kOnes) == kOnes || ((v >> 16) & kOnes) == kOnes;
}
template <typename T>
__device__ __forceinline__ uint32_t clean_pair(uint32_t v) {
    constexpr uint32_t kOnes = std::is_same_v<T, _Float16> ? 0x7C00u : 0x7F80u;
    v = (v & kOnes) == kOnes ? v & 0xFFFF0000u : v;
    return ((v >> 16) & kOnes) == kOnes ? v & 0x0000FFFFu : v;
}
__device__ __forceinline__ bool odd_float(float v) { return (__float_as_uint(v) & 0x7F800000u) == 0x7F800000u; }

// An entry's page: its first element's offset, and whether there is such a page
// (if not, page 0 stands in, which is always there to be read).
struct Page {
    uint64_t at;
    bool bad;
};
__device__ __forceinline__ Page page_of(const PagedView &c, const uint32_t *table, uint32_t entry) {
    const uint32_t page = table[entry >> c.page_shift];
    const bool bad = page >= c.pages;
    return {(bad ? 0u : page) * c.page_stride + (entry & ((1u << c.page_shift) - 1u)) * c.entry_stride, bad};
}

// N consecutive outputs of a row, gated.
template <typename R, uint32_t N>
__device__ __forceinline__ void store_output(const AttendArgs &a, uint32_t token, uint32_t head, uint32_t at,
                                             float (&v)[N]) {
    struct alignas(sizeof(R) * N) Vector {
        R v[N];
    };
    if (a.gate.data != nullptr) {
        const Vector g = *reinterpret_cast<const Vector *>(reinterpret_cast<const R *>(a.gate.data) +
                                                           token * a.gate.token_stride + head * a.gate.head_stride +
                                                           at);
#pragma unroll
        for (uint32_t k = 0; k < N; ++k) {
            v[k] *= 1.0f / (1.0f + expf(-static_cast<float>(g.v[k])));
        }
    }
    Vector out;
#pragma unroll
    for (uint32_t k = 0; k < N; ++k) {
        out.v[k] = static_cast<R>(v[k]);
    }
    *reinterpret_cast<Vector *>(reinterpret_cast<R *>(a.outputs.data) + token * a.outputs.token_stride +
                                head * a.outputs.head_stride + at) = out;
}

// Rows of a sequence that nothing is computed for: NaN where it is over the
// batch's bounds, 0 where it has no entries. By one block, for a KV head.
template <typename R, uint32_t D>
__device__ __forceinline__ void fill_rows(const AttendArgs &a, const SequenceRows &s, uint32_t kv) {
    const uint64_t items = static_cast<uint64_t>(s.count) * a.group * (D / 4u);
    for (uint64_t i = threadIdx.x; i < items; i += kThreads) {
        const uint32_t row = static_cast<uint32_t>(i / (D / 4u)), at = static_cast<uint32_t>(i % (D / 4u)) * 4u;
        const float v = s.over ? __builtin_nanf("") : 0.0f;
        float out[4] = {v, v, v, v};
        store_output<R, 4>(a, s.first + row / a.group, kv * a.group + row % a.group, at, out);
    }
}

// ---- up to 16 rows a KV head --------------------------------------------------

template <uint32_t D>
struct StepLds {
    __align__(16) float sums[4][kStepRows][D + 4u];
    float maximum[4][kStepRows], denominator[4][kStepRows];
};

// Block (KV head, part, sequence): its four waves take the part's tiles in turn.
// Lane l is column c = l % 16 (a row), quarter g = l / 16.
template <typename T, typename R, uint32_t D>
__global__ __launch_bounds__(kThreads, 1) void k_paged_step(AttendArgs args) {
    constexpr bool kFloat = std::is_same_v<T, float>;  // the cache's type
    constexpr uint32_t P = std::is_same_v<R, float> ? 3u : 1u;
    // a wave's tile, and the keys of a tile that a lane holds: kKeys / 4 in a row
    constexpr uint32_t kKeys = kFloat ? 16u : 32u, kHeld = kKeys / 4u;
    // dimensions of a value row that a lane holds side by side, and groups of 16 lanes' worth
    constexpr uint32_t kSide = kFloat ? 4u : D == 64u ? 4u : 8u, kGroups = D / (16u * kSide);
    __shared__ StepLds<D> lds;
    const PagedView &cache = args.c;
    const uint32_t kv = blockIdx.x % cache.heads, part = blockIdx.x / cache.heads, sequence = blockIdx.y;
    const uint32_t t = threadIdx.x, lane = t & 63u, wave = t >> 6;
    const uint32_t c = lane & 15u, g = lane >> 4;
    const SequenceRows s = sequence_rows(cache, sequence);
    if (s.count == 0u) {
        return;
    }
    if (s.over || s.length == 0u) {
        if (part == 0u) {
            fill_rows<R, D>(args, s, kv);
        }
        return;
    }
    const uint32_t rows = s.count * args.group;  // at most kStepRows
    const int32_t first_position = static_cast<int32_t>(s.length) - static_cast<int32_t>(s.count);
    const uint32_t row = min(c, rows - 1u);
    const uint32_t token = s.first + row / args.group, head = kv * args.group + row % args.group;
    const int32_t position = first_position + static_cast<int32_t>(row / args.group);
    const int32_t window = static_cast<int32_t>(args.window);
    const int32_t oldest = window == 0 ? 0 : max(0, position - window + 1);  // the row's first entry
    const int32_t begin = base_of(args, first_position) + static_cast<int32_t>(part * args.span);
    const int32_t end = min(begin + static_cast<int32_t>(args.span), static_cast<int32_t>(s.length));
    if (begin >= end) {
        return;
    }
    // entries that some row sees, and those that every row sees
    const int32_t seen_from = window == 0 ? 0 : max(0, first_position - window + 1);
    const int32_t all_from = window == 0 ? 0 : max(0, static_cast<int32_t>(s.length) - window);
    const uint32_t *const table = cache.table + static_cast<uint64_t>(sequence) * cache.table_stride;
    const T *const keys = reinterpret_cast<const T *>(cache.keys) + kv * cache.head_stride;
    const T *const values = reinterpret_cast<const T *>(cache.values) + kv * cache.head_stride;

    // the row's query as the products take it
    const R *const query = reinterpret_cast<const R *>(args.queries.data) + token * args.queries.token_stride +
                           head * args.queries.head_stride;
    f32x4 query_float[kFloat ? D / 16u : 1u];
    u32x4 query_pieces[kFloat ? 1u : D / 32u][P];
    if constexpr (kFloat) {
#pragma unroll
        for (uint32_t j = 0; j < D / 16u; ++j) {
            query_float[j] = *reinterpret_cast<const f32x4 *>(query + 16u * j + 4u * g);
        }
    } else if constexpr (P == 1) {
#pragma unroll
        for (uint32_t j = 0; j < D / 32u; ++j) {
            query_pieces[j][0] = *reinterpret_cast<const u32x4 *>(query + 32u * j + 8u * g);
        }
    } else {
#pragma unroll
        for (uint32_t j = 0; j < D / 32u; ++j) {
            const f32x4 lo = *reinterpret_cast<const f32x4 *>(query + 32u * j + 8u * g);
            const f32x4 hi = *reinterpret_cast<const f32x4 *>(query + 32u * j + 8u * g + 4u);
#pragma unroll
            for (uint32_t k = 0; k < 4u; ++k) {
                uint32_t pieces[P];
                k < 2u ? split<T>(lo[2u * k], lo[2u * k + 1u], pieces)
                       : split<T>(hi[2u * k - 4u], hi[2u * k - 3u], pieces);
#pragma unroll
                for (uint32_t p = 0; p < P; ++p) {
                    query_pieces[j][p][k] = pieces[p];
                }
            }
        }
    }

    f32x4 sums[kGroups][kSide];
#pragma unroll
    for (uint32_t i = 0; i < kGroups; ++i) {
#pragma unroll
        for (uint32_t k = 0; k < kSide; ++k) {
            sums[i][k] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        }
    }
    float maximum = kNegative, denominator = 0.0f;

    for (int32_t first = begin + static_cast<int32_t>(wave * kKeys); first < end; first += 4 * kKeys) {
        // Key operands: row i of A is key first + kHeld (i / 4) + i % 4 (+ 4
        // in the second of two products with 32 keys), so that register r of
        // the results is key first + kHeld g + r. Groups of 8 entries from a
        // multiple of 8 share a page.
        const int32_t key_group = first + static_cast<int32_t>((kHeld * (c >> 2)) & ~7u);
        const int32_t value_group = first + static_cast<int32_t>((kHeld * g) & ~7u);
        Page key_page{0, false}, value_page{0, false};
        if (key_group < end) {
            key_page = page_of(cache, table, key_group);
        }
        if (value_group < end) {
            value_page = page_of(cache, table, value_group);
        }
        const uint32_t key_at = (kHeld * (c >> 2) & 7u) + (c & 3u);
        const T *const key = keys + key_page.at + key_at * cache.entry_stride;
        const T *const value = values + value_page.at + ((kHeld * g) & 7u) * cache.entry_stride;
        float score[kHeld];
        if constexpr (kFloat) {
            f32x4 k[D / 16u];
#pragma unroll
            for (uint32_t j = 0; j < D / 16u; ++j) {
                k[j] = *reinterpret_cast<const f32x4 *>(key + 16u * j + 4u * g);
            }
            f32x4 acc[2] = {{0.0f, 0.0f, 0.0f, 0.0f}, {0.0f, 0.0f, 0.0f, 0.0f}};
#pragma unroll
            for (uint32_t j = 0; j < D / 16u; ++j) {
#pragma unroll
                for (uint32_t i = 0; i < 4u; ++i) {
                    acc[j & 1u] =
                        __builtin_amdgcn_mfma_f32_16x16x4f32(k[j][i], query_float[j][i], acc[j & 1u], 0, 0, 0);
                }
            }
#pragma unroll
            for (uint32_t r = 0; r < 4u; ++r) {
                score[r] = acc[0][r] + acc[1][r];
            }
        } else {
            u32x4 k[2][D / 32u][1];
#pragma unroll
            for (uint32_t h = 0; h < 2u; ++h) {
#pragma unroll
                for (uint32_t j = 0; j < D / 32u; ++j) {
                    k[h][j][0] =
                        *reinterpret_cast<const u32x4 *>(key + 4u * h * cache.entry_stride + 32u * j + 8u * g);
                }
            }
#pragma unroll
            for (uint32_t h = 0; h < 2u; ++h) {
                f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (uint32_t j = 0; j < D / 32u; ++j) {
                    acc = product<T>(k[h][j], query_pieces[j], acc);
                }
#pragma unroll
                for (uint32_t r = 0; r < 4u; ++r) {
                    score[4u * h + r] = acc[r];
                }
            }
        }
        // values: kHeld entries of the lane's quarter, kSide dimensions of each group
        using Chunk = std::conditional_t<kFloat, f32x4, std::conditional_t<kSide == 8u, u32x4, u32x2>>;
        Chunk held[kGroups][kHeld];
#pragma unroll
        for (uint32_t i = 0; i < kGroups; ++i) {
#pragma unroll
            for (uint32_t k = 0; k < kHeld; ++k) {
                held[i][k] = *reinterpret_cast<const Chunk *>(value + k * cache.entry_stride + 16u * kSide * i +
                                                              kSide * c);
            }
        }
        const int32_t own_first = first + static_cast<int32_t>(kHeld * g);  // the lane's keys
        // a tile that some row does not see whole (uniform but for bad pages)
        const bool edge = first + static_cast<int32_t>(kKeys) > first_position + 1 || first < all_from;
        bool careful = false;
        if (__any(edge || value_page.bad)) {
            bool odd = false;
#pragma unroll
            for (uint32_t k = 0; k < kHeld; ++k) {
                const int32_t entry = own_first + static_cast<int32_t>(k);
                const bool visible = entry <= position && entry >= oldest;
                score[k] = !visible ? kNegative : value_page.bad ? __builtin_nanf("") : score[k];
                // (what no row sees is whatever the page held before)
                const bool any = entry < static_cast<int32_t>(s.length) && entry >= seen_from && !value_page.bad;
#pragma unroll
                for (uint32_t i = 0; i < kGroups; ++i) {
                    constexpr uint32_t kWords = sizeof(Chunk) / 4u;
#pragma unroll
                    for (uint32_t w = 0; w < kWords; ++w) {
                        held[i][k][w] = any ? held[i][k][w] : 0;
                        if constexpr (kFloat) {
                            odd |= odd_float(held[i][k][w]);
                        } else {
                            odd |= odd_pair<T>(held[i][k][w]);
                        }
                    }
                }
            }
            // with one token every row sees the same entries
            careful = s.count > 1u && __any(odd);
        }
        float top = score[0];
#pragma unroll
        for (uint32_t k = 1; k < kHeld; ++k) {
            top = fmaxf(top, score[k]);
        }
        top = fmaxf(top, lane_xor<16>(top));
        top = fmaxf(top, lane_xor<32>(top));
        if (__any(top > maximum)) {
            const float next = fmaxf(maximum, top);
            const float factor = next == kNegative ? 1.0f : weight_of<P == 3>(maximum, next, args.log2_scale);
            maximum = next;
            denominator *= factor;
#pragma unroll
            for (uint32_t i = 0; i < kGroups; ++i) {
#pragma unroll
                for (uint32_t k = 0; k < kSide; ++k) {
                    sums[i][k] *= factor;
                }
            }
        }
        const float level = maximum == kNegative ? 0.0f : maximum;
#pragma unroll
        for (uint32_t k = 0; k < kHeld; ++k) {
            score[k] = weight_of<P == 3>(score[k], level, args.log2_scale);
            denominator += score[k];
        }
        if (careful) {
            // Entries with infinities or NaN of which some rows see only a
            // part: their values are taken out of the products and added for the
            // rows that see them.
            for (uint32_t from = 0; from < 4u; ++from) {
#pragma unroll
                for (uint32_t k = 0; k < kHeld; ++k) {
                    const int32_t entry = first + static_cast<int32_t>(kHeld * from + k);
                    const float weight = __shfl(score[k], static_cast<int>(from * 16u + c));
                    const bool visible = entry <= position && entry >= oldest;
#pragma unroll
                    for (uint32_t i = 0; i < kGroups; ++i) {
#pragma unroll
                        for (uint32_t n = 0; n < kSide; ++n) {
#pragma unroll
                            for (uint32_t r = 0; r < 4u; ++r) {
                                // row r of the lane's results is the chunk of lane 4 g + r
                                const int source = static_cast<int>(from * 16u + 4u * g + r);
                                float v;
                                if constexpr (kFloat) {
                                    v = __shfl(held[i][k][n], source);
                                } else {
                                    const uint32_t pair = __shfl(held[i][k][n / 2u], source);
                                    const uint16_t bits = static_cast<uint16_t>(n & 1u ? pair >> 16 : pair);
                                    v = static_cast<float>(__builtin_bit_cast(T, bits));
                                }
                                sums[i][n][r] += visible && odd_float(v) ? v * weight : 0.0f;
                            }
                        }
                    }
                }
            }
#pragma unroll
            for (uint32_t i = 0; i < kGroups; ++i) {
#pragma unroll
                for (uint32_t k = 0; k < kHeld; ++k) {
                    constexpr uint32_t kWords = sizeof(Chunk) / 4u;
#pragma unroll
                    for (uint32_t w = 0; w < kWords; ++w) {
                        if constexpr (kFloat) {
                            held[i][k][w] = odd_float(held[i][k][w]) ? 0.0f : held[i][k][w];
                        } else {
                            held[i][k][w] = clean_pair<T>(held[i][k][w]);
                        }
                    }
                }
            }
        }
        if constexpr (kFloat) {
#pragma unroll
            for (uint32_t r = 0; r < 4u; ++r) {
#pragma unroll
                for (uint32_t i = 0; i < kGroups; ++i) {
#pragma unroll
                    for (uint32_t n = 0; n < 4u; ++n) {
                        sums[i][n] =
                            __builtin_amdgcn_mfma_f32_16x16x4f32(held[i][r][n], score[r], sums[i][n], 0, 0, 0);
                    }
                }
            }
        } else {
            u32x4 weights[P];
#pragma unroll
            for (uint32_t k = 0; k < 4u; ++k) {
                uint32_t pieces[P];
                split<T>(score[2u * k], score[2u * k + 1u], pieces);
#pragma unroll
                for (uint32_t p = 0; p < P; ++p) {
                    weights[p][k] = pieces[p];
                }
            }
#pragma unroll
            for (uint32_t i = 0; i < kGroups; ++i) {
#pragma unroll
                for (uint32_t n = 0; n < kSide; ++n) {
                    u32x4 v[1];
#pragma unroll
                    for (uint32_t k = 0; k < 4u; ++k) {
                        v[0][k] = __builtin_amdgcn_perm(held[i][2u * k + 1u][n / 2u], held[i][2u * k][n / 2u],
                                                        n & 1u ? 0x07060302u : 0x05040100u);
                    }
                    sums[i][n] = product<T>(v, weights, sums[i][n]);
                }
            }
        }
    }

    // the row's lanes' parts of the denominator, then the waves
    denominator += lane_xor<16>(denominator);
    denominator += lane_xor<32>(denominator);
    if (g == 0u) {
        lds.maximum[wave][c] = maximum;
        lds.denominator[wave][c] = denominator;
    }
    __syncthreads();
    {
        float top = lds.maximum[0][c];
#pragma unroll
        for (uint32_t w = 1; w < 4u; ++w) {
            top = fmaxf(top, lds.maximum[w][c]);
        }
        const float factor = maximum == kNegative && top == kNegative ? 1.0f
                                                                        : weight_of<P == 3>(maximum, top, args.log2_scale);
        if (c < rows) {
#pragma unroll
            for (uint32_t i = 0; i < kGroups; ++i) {
#pragma unroll
                for (uint32_t r = 0; r < 4u; ++r) {
#pragma unroll
                    for (uint32_t n = 0; n < kSide; n += 4u) {
                        *reinterpret_cast<f32x4 *>(&lds.sums[wave][c][16u * kSide * i + kSide * (4u * g + r) + n]) =
                            f32x4{sums[i][n][r], sums[i][n + 1u][r], sums[i][n + 2u][r], sums[i][n + 3u][r]} * factor;
                    }
                }
            }
        }
    }
    __syncthreads();
    const bool whole = args.parts == 1u;
    for (uint32_t i = t; i < rows * (D / 4u); i += kThreads) {
        const uint32_t r = i / (D / 4u), at = i % (D / 4u) * 4u;
        float top = kNegative;
#pragma unroll
        for (uint32_t w = 0; w < 4u; ++w) {
            top = fmaxf(top, lds.maximum[w][r]);
        }
        float total = 0.0f;
        f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (uint32_t w = 0; w < 4u; ++w) {
            const float m = lds.maximum[w][r];
            total += lds.denominator[w][r] *
                     (m == kNegative && top == kNegative ? 1.0f : weight_of<P == 3>(m, top, args.log2_scale));
            sum += *reinterpret_cast<const f32x4 *>(&lds.sums[w][r][at]);
        }
        const uint32_t row_token = s.first + r / args.group, row_head = kv * args.group + r % args.group;
        if (whole) {
            const bool none = first_position + static_cast<int32_t>(r / args.group) < 0;
            float out[4];
#pragma unroll
            for (uint32_t k = 0; k < 4u; ++k) {
                out[k] = none ? 0.0f : sum[k] / total;
            }
            store_output<R, 4>(args, row_token, row_head, at, out);
        } else {
            float *to = partial_row<D>(args, part, row_token, row_head);
            *reinterpret_cast<f32x4 *>(to + at) = sum;
            if (at == 0u) {
                to[D] = top;
                to[D + 1u] = total;
            }
        }
    }
}

// ---- joining the parts of a history -------------------------------------------

// Block (token, query head), a thread a dimension.
template <typename R, uint32_t D, bool EXACT>
__global__ __launch_bounds__(D) void k_paged_join(AttendArgs args) {
    const PagedView &cache = args.c;
    const uint32_t heads = cache.heads * args.group;
    const uint64_t rows = static_cast<uint64_t>(cache.tokens) * heads;
    for (uint64_t row = blockIdx.x; row < rows; row += gridDim.x) {
        const uint32_t token = static_cast<uint32_t>(row / heads), head = static_cast<uint32_t>(row % heads);
        uint32_t sequence = 0;
        for (uint32_t s = 0; s < cache.sequences; s += 64u) {
            const uint32_t lane = threadIdx.x & 63u;
            const bool before = s + lane < cache.sequences && cache.offsets[s + lane + 1u] <= token;
            const uint32_t ended = static_cast<uint32_t>(__popcll(__ballot(before)));
            sequence += ended;
            if (ended < 64u) {
                break;
            }
        }
        if (sequence >= cache.sequences) {
            continue;
        }
        const SequenceRows s = sequence_rows(cache, sequence);
        if (token < s.first || token - s.first >= s.count || s.over || s.length == 0u) {
            continue;  // (filled by the attention itself)
        }
        const int32_t first_position = static_cast<int32_t>(s.length) - static_cast<int32_t>(s.count);
        const int32_t position = first_position + static_cast<int32_t>(token - s.first);
        const int32_t base = base_of(args, first_position);
        const int32_t window = static_cast<int32_t>(args.window);
        const int32_t oldest = window == 0 ? 0 : max(0, position - window + 1);
        float sum = 0.0f, total = 0.0f, top = kNegative;
        if (position >= 0) {
            const uint32_t from = static_cast<uint32_t>(oldest - base) / args.span;
            const uint32_t to = static_cast<uint32_t>(position - base) / args.span;
            for (uint32_t p = from; p <= to; ++p) {
                top = fmaxf(top, partial_row<D>(args, p, token, head)[D]);
            }
            for (uint32_t p = from; p <= to; ++p) {
                const float *part = partial_row<D>(args, p, token, head);
                const float factor =
                    part[D] == kNegative && top == kNegative ? 1.0f : weight_of<EXACT>(part[D], top, args.log2_scale);
                total += part[D + 1u] * factor;
                sum += part[threadIdx.x] * factor;
            }
        }
        float out[1] = {position < 0 ? 0.0f : sum / total};
        store_output<R, 1>(args, token, head, threadIdx.x, out);
    }
}

// ---- more rows ----------------------------------------------------------------

// LDS places: 16-byte pieces of a row of D 16-bit values are permuted so that
// the reads of a phase fall on different banks: keys, where 16 rows are read at
// one piece, by the row; values, where four rows are read at 64 bytes, by four
// pieces. A row of 64 values is half the banks, so two rows share a turn.
template <uint32_t D>
__device__ __forceinline__ uint32_t key_place(uint32_t row, uint32_t piece) {
    const uint32_t turn = D == 64u ? (row >> 1) & 7u : row & 15u;
    return row * (D * 2u) + ((piece ^ turn) << 4);
}
template <uint32_t D>
__device__ __forceinline__ uint32_t value_place(uint32_t row, uint32_t piece) {
    const uint32_t turn = D == 64u ? (row & 2u) << 1 : (row & 3u) << 2;
    return row * (D * 2u) + ((piece ^ turn) << 4);
}

// Block (row tile, KV head, part, sequence): 128 rows, 32 a wave, lane l row
// l % 32 and half h = l / 32.
template <typename T, typename R, uint32_t D>
__global__ __launch_bounds__(kThreads, 1) void k_paged_chunk(AttendArgs args) {
    constexpr bool kFloat = std::is_same_v<T, float>;
    using M = std::conditional_t<kFloat, __bf16, T>;  // the matrix cores' type
    constexpr uint32_t P = std::is_same_v<R, float> ? 3u : 1u;
    constexpr uint32_t Q = kFloat ? 3u : 1u;
    constexpr uint32_t kPlane = kChunkKeys * D * 2u;
    constexpr uint32_t kPieces = D / 8u;                                // of a row
    constexpr uint32_t kLoads = kChunkKeys * kPieces / kThreads;        // a thread's pieces of a tile
    static_assert(kChunkKeys * kPieces % kThreads == 0 || D == 32u);
    extern __shared__ __align__(16) unsigned char lds[];
    unsigned char *const key_lds = lds;
    unsigned char *const value_lds = lds + Q * kPlane;
    // the last tile with a value that is not finite, and with a bad page
    volatile uint32_t *const odd = reinterpret_cast<volatile uint32_t *>(lds + 2u * Q * kPlane);
    volatile uint32_t *const bad_key = odd + 4u;  // [kChunkKeys]
    const PagedView &cache = args.c;
    // the blocks of one (KV head, part, sequence) read the same entries: their
    // number is a multiple of 8 or the group's, so they share an XCD (block b
    // runs on XCD b % 8); the tiles with the longest histories come first
    const uint32_t groups = cache.heads * args.parts * cache.sequences;
    const uint32_t padded = groups < 8u ? groups : (groups + 7u) & ~7u;
    const uint32_t which = blockIdx.x % padded, tile = args.tiles - 1u - blockIdx.x / padded;
    if (which >= groups) {
        return;
    }
    const uint32_t kv = which % cache.heads, part = which / cache.heads % args.parts;
    const uint32_t sequence = which / (cache.heads * args.parts);
    const SequenceRows s = sequence_rows(cache, sequence);
    if (s.count == 0u) {
        return;
    }
    if (s.over || s.length == 0u) {
        if (part == 0u && tile == 0u) {
            fill_rows<R, D>(args, s, kv);
        }
        return;
    }
    const uint32_t rows = s.count * args.group;
    if (tile * kChunkRows >= rows) {
        return;
    }
    const uint32_t t = threadIdx.x, lane = t & 63u;
    const uint32_t wave = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(t >> 6)));
    const uint32_t column = lane & 31u, half = lane >> 5;
    const int32_t first_position = static_cast<int32_t>(s.length) - static_cast<int32_t>(s.count);
    const int32_t window = static_cast<int32_t>(args.window);
    const auto place = [&](uint32_t row) { return first_position + static_cast<int32_t>(row / args.group); };
    const auto from = [&](int32_t position) { return window == 0 ? 0 : max(0, position - window + 1); };
    const uint32_t block_last = min((tile + 1u) * kChunkRows, rows) - 1u;
    const int32_t block_low = place(tile * kChunkRows), block_high = place(block_last);
    const uint32_t wave_row = tile * kChunkRows + wave * 32u;
    const bool wave_live = wave_row < rows;
    const int32_t wave_low = place(min(wave_row, rows - 1u)), wave_high = place(min(wave_row + 31u, rows - 1u));
    const uint32_t row = min(wave_row + column, rows - 1u);
    const uint32_t token = s.first + row / args.group, head = kv * args.group + row % args.group;
    const int32_t position = place(row), oldest = from(position);
    // entries of the part that some row of the block sees
    int32_t begin = base_of(args, first_position) + static_cast<int32_t>(part * args.span);
    const int32_t end = min(begin + static_cast<int32_t>(args.span), block_high + 1);
    begin = max(begin, from(block_low) & ~static_cast<int32_t>(kChunkKeys - 1u));
    const bool whole = args.parts == 1u;
    if (begin >= end && !whole) {
        return;
    }
    const uint32_t *const table = cache.table + static_cast<uint64_t>(sequence) * cache.table_stride;
    const T *const keys = reinterpret_cast<const T *>(cache.keys) + kv * cache.head_stride;
    const T *const values = reinterpret_cast<const T *>(cache.values) + kv * cache.head_stride;
    if (t < 2u) {
        odd[t] = ~0u;
    }

    // the row's query: step j holds dimensions 16 j + 8 half + 0 .. 7
    u32x4 query_pieces[D / 16u][P];
    {
        const R *const query = reinterpret_cast<const R *>(args.queries.data) + token * args.queries.token_stride +
                               head * args.queries.head_stride + 8u * half;
#pragma unroll
        for (uint32_t j = 0; j < D / 16u; ++j) {
            if constexpr (P == 1) {
                query_pieces[j][0] = *reinterpret_cast<const u32x4 *>(query + 16u * j);
            } else {
                const f32x4 lo = *reinterpret_cast<const f32x4 *>(query + 16u * j);
                const f32x4 hi = *reinterpret_cast<const f32x4 *>(query + 16u * j + 4u);
#pragma unroll
                for (uint32_t k = 0; k < 4u; ++k) {
                    uint32_t pieces[P];
                    k < 2u ? split<M>(lo[2u * k], lo[2u * k + 1u], pieces)
                           : split<M>(hi[2u * k - 4u], hi[2u * k - 3u], pieces);
#pragma unroll
                    for (uint32_t p = 0; p < P; ++p) {
                        query_pieces[j][p][k] = pieces[p];
                    }
                }
            }
        }
    }

    // A tile passes through registers: piece t + 256 i of it, of row piece /
    // kPieces.
    using Piece = std::conditional_t<kFloat, f32x4, u32x4>;
    constexpr uint32_t kWide = kFloat ? 2u : 1u;
    Piece key_in[kLoads][kWide], value_in[kLoads][kWide];
    uint32_t bad_in = 0;
    const auto load = [&](int32_t first) {
        bad_in = 0;
#pragma unroll
        for (uint32_t i = 0; i < kLoads; ++i) {
            const uint32_t piece = t + kThreads * i, at = piece % kPieces * 8u;
            const int32_t entry = first + static_cast<int32_t>(piece / kPieces);
            Page page{0, false};
            if (entry < end) {
                page = page_of(cache, table, entry);
            }
            bad_in |= page.bad ? 1u << i : 0u;
#pragma unroll
            for (uint32_t w = 0; w < kWide; ++w) {
                key_in[i][w] = reinterpret_cast<const Piece *>(keys + page.at + at)[w];
                value_in[i][w] = reinterpret_cast<const Piece *>(values + page.at + at)[w];
            }
        }
    };
    const auto stage = [&](int32_t first, bool edge) {
        if (edge || bad_in != 0u) {
#pragma unroll
            for (uint32_t i = 0; i < kLoads; ++i) {
                const uint32_t piece = t + kThreads * i;
                const int32_t entry = first + static_cast<int32_t>(piece / kPieces);
                const bool bad = (bad_in >> i & 1u) != 0u;
                const bool any = entry < end && entry >= from(block_low) && !bad;
                bool seen = false;
#pragma unroll
                for (uint32_t w = 0; w < kWide; ++w) {
#pragma unroll
                    for (uint32_t k = 0; k < 4u; ++k) {
                        value_in[i][w][k] = any ? value_in[i][w][k] : 0;
                        if constexpr (kFloat) {
                            seen |= odd_float(value_in[i][w][k]);
                            value_in[i][w][k] = odd_float(value_in[i][w][k]) ? 0.0f : value_in[i][w][k];
                        } else {
                            seen |= odd_pair<T>(value_in[i][w][k]);
                            value_in[i][w][k] = clean_pair<T>(value_in[i][w][k]);
                        }
                    }
                }
                if (seen) {
                    odd[0] = static_cast<uint32_t>(first);
                }
                if (bad) {
                    odd[1] = static_cast<uint32_t>(first);
                }
                if (piece % kPieces == 0u) {
                    bad_key[piece / kPieces] = bad ? static_cast<uint32_t>(first) : ~0u;
                }
            }
        }
#pragma unroll
        for (uint32_t i = 0; i < kLoads; ++i) {
            const uint32_t piece = t + kThreads * i, entry = piece / kPieces, at = piece % kPieces;
            if constexpr (kFloat) {
                u32x4 k[Q], v[Q];
#pragma unroll
                for (uint32_t n = 0; n < 4u; ++n) {
                    uint32_t pieces[Q];
                    split<M>(key_in[i][n / 2u][2u * n % 4u], key_in[i][n / 2u][2u * n % 4u + 1u], pieces);
#pragma unroll
                    for (uint32_t p = 0; p < Q; ++p) {
                        k[p][n] = pieces[p];
                    }
                    split<M>(value_in[i][n / 2u][2u * n % 4u], value_in[i][n / 2u][2u * n % 4u + 1u], pieces);
#pragma unroll
                    for (uint32_t p = 0; p < Q; ++p) {
                        v[p][n] = pieces[p];
                    }
                }
#pragma unroll
                for (uint32_t p = 0; p < Q; ++p) {
                    *reinterpret_cast<u32x4 *>(key_lds + p * kPlane + key_place<D>(entry, at)) = k[p];
                    *reinterpret_cast<u32x4 *>(value_lds + p * kPlane + value_place<D>(entry, at)) = v[p];
                }
            } else {
                *reinterpret_cast<u32x4 *>(key_lds + key_place<D>(entry, at)) = key_in[i][0];
                *reinterpret_cast<u32x4 *>(value_lds + value_place<D>(entry, at)) = value_in[i][0];
            }
        }
    };

    f32x16 sums[D / 32u];
#pragma unroll
    for (uint32_t m = 0; m < D / 32u; ++m) {
#pragma unroll
        for (uint32_t r = 0; r < 16u; ++r) {
            sums[m][r] = 0.0f;
        }
    }
    float maximum = kNegative, denominator = 0.0f;
    // register r of a score tile is key 8 (r / 4) + 4 half + r % 4
    const auto key_of = [&](uint32_t r) { return static_cast<int32_t>(8u * (r / 4u) + 4u * half + r % 4u); };

    if (begin < end) {
        load(begin);
    }
    for (int32_t first = begin; first < end; first += static_cast<int32_t>(kChunkKeys)) {
        const bool edge = first + static_cast<int32_t>(kChunkKeys) > block_low + 1 || first < from(block_high);
        __syncthreads();  // the last tile's reads (and the first's marks) are done
        stage(first, edge);
        __syncthreads();
        if (first + static_cast<int32_t>(kChunkKeys) < end) {
            load(first + static_cast<int32_t>(kChunkKeys));
        }
        if (!wave_live || first > wave_high || first + static_cast<int32_t>(kChunkKeys) <= from(wave_low)) {
            continue;  // nothing of the tile is seen by the wave's rows
        }
        f32x16 score;
#pragma unroll
        for (uint32_t r = 0; r < 16u; ++r) {
            score[r] = 0.0f;
        }
#pragma unroll
        for (uint32_t j = 0; j < D / 16u; ++j) {
            u32x4 k[Q];
#pragma unroll
            for (uint32_t p = 0; p < Q; ++p) {
                k[p] = *reinterpret_cast<const u32x4 *>(key_lds + p * kPlane + key_place<D>(column, 2u * j + half));
            }
            score = product<M>(k, query_pieces[j], score);
        }
        const bool bad_tile = odd[1] == static_cast<uint32_t>(first);
        if (bad_tile || first + static_cast<int32_t>(kChunkKeys) > wave_low + 1 || first < from(wave_high)) {
#pragma unroll
            for (uint32_t r = 0; r < 16u; ++r) {
                const int32_t entry = first + key_of(r);
                const bool visible = entry <= position && entry >= oldest;
                const bool bad = bad_tile && bad_key[key_of(r)] == static_cast<uint32_t>(first);
                score[r] = !visible ? kNegative : bad ? __builtin_nanf("") : score[r];
            }
        }
        float top = score[0];
#pragma unroll
        for (uint32_t r = 1; r < 16u; ++r) {
            top = fmaxf(top, score[r]);
        }
        top = fmaxf(top, lane_xor<32>(top));
        if (__any(top > maximum)) {
            const float next = fmaxf(maximum, top);
            const float factor = next == kNegative ? 1.0f : weight_of<P == 3>(maximum, next, args.log2_scale);
            maximum = next;
            denominator *= factor;
#pragma unroll
            for (uint32_t m = 0; m < D / 32u; ++m) {
                sums[m] *= factor;
            }
        }
        const float level = maximum == kNegative ? 0.0f : maximum;
#pragma unroll
        for (uint32_t r = 0; r < 16u; ++r) {
            score[r] = weight_of<P == 3>(score[r], level, args.log2_scale);
            denominator += score[r];
        }
#pragma unroll
        for (uint32_t u = 0; u < 2u; ++u) {
            u32x4 weights[P];
#pragma unroll
            for (uint32_t k = 0; k < 4u; ++k) {
                uint32_t pieces[P];
                split<M>(score[8u * u + 2u * k], score[8u * u + 2u * k + 1u], pieces);
#pragma unroll
                for (uint32_t p = 0; p < P; ++p) {
                    weights[p][k] = pieces[p];
                }
            }
            // lane i of 16 takes row i / 4 of four entries at 4 (i % 4), and
            // gets dimension i of the four
            const uint32_t entry = 16u * u + 4u * half + (lane & 15u) / 4u;
            const uint32_t side = (lane >> 4 & 1u) * 16u + (lane & 3u) * 4u;
#pragma unroll
            for (uint32_t m = 0; m < D / 32u; ++m) {
                u32x4 v[Q];
#pragma unroll
                for (uint32_t p = 0; p < Q; ++p) {
                    const uint32_t d = 32u * m + side;
                    const auto read = [&](uint32_t e) {
                        auto *at = (__attribute__((address_space(3))) s16x4 *)(value_lds + p * kPlane +
                                                                              value_place<D>(e, d / 8u) + d % 8u * 2u);
                        return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(at));
                    };
                    const u32x2 lo = read(entry), hi = read(entry + 8u);
                    v[p] = u32x4{lo.x, lo.y, hi.x, hi.y};
                }
                sums[m] = product<M>(v, weights, sums[m]);
            }
        }
        if (odd[0] == static_cast<uint32_t>(first)) {
            // Values that are not finite, which the products left out, for the
            // rows that see them.
            for (int32_t k = 0; k < static_cast<int32_t>(kChunkKeys); ++k) {
                const int32_t entry = first + k;
                if (entry >= end) {
                    break;
                }
                const Page page = page_of(cache, table, entry);
                if (page.bad) {
                    continue;  // (its score is NaN already)
                }
                float weight = 0.0f;
#pragma unroll
                for (uint32_t r = 0; r < 16u; ++r) {
                    weight = key_of(r) == k ? score[r] : weight;
                }
                const float other = lane_xor<32>(weight);
                weight = static_cast<uint32_t>(k >> 2 & 1) == half ? weight : other;
                const bool visible = entry <= position && entry >= oldest;
                const T *const value = values + page.at + 4u * half;
#pragma unroll
                for (uint32_t m = 0; m < D / 32u; ++m) {
#pragma unroll
                    for (uint32_t r = 0; r < 16u; ++r) {
                        const float v = static_cast<float>(value[32u * m + 8u * (r / 4u) + r % 4u]);
                        sums[m][r] += visible && odd_float(v) ? v * weight : 0.0f;
                    }
                }
            }
        }
    }

    denominator += lane_xor<32>(denominator);
    if (!wave_live || wave_row + column >= rows) {
        return;
    }
    if (!whole && (position < begin || oldest >= end)) {
        return;  // the part holds nothing the row sees
    }
    float *const to = whole ? nullptr : partial_row<D>(args, part, token, head);
#pragma unroll
    for (uint32_t m = 0; m < D / 32u; ++m) {
#pragma unroll
        for (uint32_t q = 0; q < 4u; ++q) {
            const uint32_t at = 32u * m + 8u * q + 4u * half;
            f32x4 v = {sums[m][4u * q], sums[m][4u * q + 1u], sums[m][4u * q + 2u], sums[m][4u * q + 3u]};
            if (whole) {
                float out[4];
#pragma unroll
                for (uint32_t k = 0; k < 4u; ++k) {
                    out[k] = position < 0 ? 0.0f : v[k] / denominator;
                }
                store_output<R, 4>(args, token, head, at, out);
            } else {
                *reinterpret_cast<f32x4 *>(to + at) = v;
            }
        }
    }
    if (!whole && half == 0u) {
        to[D] = maximum;
        to[D + 1u] = denominator;
    }
}

// ---- host ---------------------------------------------------------------------

template <typename T, typename R, uint32_t D>
void launch_attention(adi_hip_context *ctx, AttendArgs args, const adi_hip_paged_workspace *workspace) {
    const PagedView &c = args.c;
    const uint32_t heads = c.heads * args.group;
    const bool step = uint64_t(c.max_tokens) * args.group <= kStepRows;
    // entries a row tile may see, its base rounded down with a window
    uint64_t extent = c.max_length;
    if (args.window != 0) {
        extent = std::min<uint64_t>(extent, uint64_t(args.window) + c.max_tokens + kSpanUnit);
    }
    const uint64_t row_tiles =
        step ? c.sequences
             : std::min<uint64_t>(ceil_div(uint64_t(c.max_tokens) * args.group, kChunkRows) * uint64_t(c.sequences),
                                  uint64_t(c.tokens) * args.group / kChunkRows + c.sequences);
    // parts: as many as give two blocks a CU, within the workspace
    const uint64_t blocks = row_tiles * c.heads;
    const uint64_t part_bytes = uint64_t(c.tokens) * heads * (D + 4u) * sizeof(float);
    uint64_t parts = std::max<uint64_t>(2u * ctx->cu_count / blocks, 1u);
    parts = std::min<uint64_t>({parts, workspace->bytes / part_bytes, (extent + kSpanUnit - 1) / kSpanUnit, 1024u});
    parts = std::max<uint64_t>(parts, 1u);
    const uint64_t span = (ceil_div(extent, parts) + kSpanUnit - 1) / kSpanUnit * kSpanUnit;
    args.span = static_cast<uint32_t>(std::max<uint64_t>(span, kSpanUnit));
    args.parts = std::max(ceil_div(extent, args.span), 1u);
    args.partial = static_cast<float *>(workspace->base);
    if (step) {
        require(uint64_t(args.parts) * c.heads < (1u << 24) && c.sequences < 65536u,
                "paged attention: too many heads or sequences");
        launch(ctx, "paged_step", k_paged_step<T, R, D>, dim3(args.parts * c.heads, c.sequences), dim3(kThreads), 0,
               args);
    } else {
        constexpr uint32_t Q = std::is_same_v<T, float> ? 3u : 1u;
        constexpr size_t lds = 2u * Q * kChunkKeys * D * 2u + 16u + kChunkKeys * 4u;
        static const bool raised = set_lds_limit(reinterpret_cast<const void *>(k_paged_chunk<T, R, D>), lds);
        (void)raised;
        args.tiles = ceil_div(uint64_t(c.max_tokens) * args.group, kChunkRows);
        const uint64_t groups = uint64_t(c.heads) * args.parts * c.sequences;
        const uint64_t grid = (groups < 8u ? groups : (groups + 7u) / 8u * 8u) * args.tiles;
        require(grid < (1u << 24), "paged attention: too many rows");
        launch(ctx, "paged_chunk", k_paged_chunk<T, R, D>, dim3(static_cast<uint32_t>(grid)), dim3(kThreads), lds,
               args);
    }
    if (args.parts > 1) {
        const uint64_t rows = uint64_t(c.tokens) * heads;
        launch(ctx, "paged_join", k_paged_join<R, D, std::is_same_v<R, float>>,
               dim3(static_cast<uint32_t>(std::min<uint64_t>(rows, 1u << 20))), dim3(D), 0, args);
    }
}

template <typename T, typename R>
void launch_attention(adi_hip_context *ctx, const AttendArgs &args, const adi_hip_paged_workspace *workspace,
                      uint32_t head_size) {
    if (head_size == 64) {
        launch_attention<T, R, 64>(ctx, args, workspace);
    } else if (head_size == 128) {
        launch_attention<T, R, 128>(ctx, args, workspace);
    } else {
        launch_attention<T, R, 256>(ctx, args, workspace);
    }
}

}  // namespace

void paged_attention(adi_hip_context *ctx, const adi_hip_paged_cache *cache, const adi_hip_paged_batch *batch,
                     const adi_hip_paged_attention_arguments *a, adi_hip_paged_workspace *workspace) {
    require_paged(cache, batch);
    require(a != nullptr && workspace != nullptr, "paged attention: null argument");
    require(workspace->device == ctx->device, "paged attention: the workspace is on another device");
    const uint32_t type = a->queries.type;
    require(known_type(type) && (type == cache->type || (type == ADI_HIP_F32 && cache->type == ADI_HIP_BF16)),
            "paged attention: f32 rows read an f32 or bf16 cache, others their own type");
    require(a->query_heads >= 1 && a->query_heads % cache->heads == 0 && a->query_heads / cache->heads <= 256,
            "paged attention: query heads must be 1 to 256 times the cache's");
    require(std::isfinite(a->scale) && a->scale >= 0.0f, "paged attention: scale must be positive, or 0");
    if (batch->tokens == 0 || batch->sequences == 0 || batch->max_tokens == 0) {
        return;
    }
    require_rows(a->queries, type, "paged attention: queries must be 16-byte aligned rows");
    require_rows(a->outputs, type, "paged attention: outputs must be 16-byte aligned rows of the queries' type");
    require(a->outputs.data != a->queries.data && a->outputs.data != a->gate.data,
            "paged attention: the outputs overlap the queries or the gate");
    if (a->gate.data != nullptr) {
        require_rows(a->gate, type, "paged attention: the gate must be 16-byte aligned rows of the queries' type");
    }
    const double scale = a->scale == 0.0f ? 1.0 / std::sqrt(double(cache->head_size)) : double(a->scale);
    const uint32_t window = std::min(a->window, 1u << 30);
    const AttendArgs args{paged_view(*cache, *batch), rows_view(a->queries), rows_view(a->outputs), rows_view(a->gate),
                          static_cast<float>(scale * 1.4426950408889634), window, a->query_heads / cache->heads, 0, 0,
                          0, nullptr};
    if (type == ADI_HIP_F32 && cache->type == ADI_HIP_F32) {
        launch_attention<float, float>(ctx, args, workspace, cache->head_size);
    } else if (type == ADI_HIP_F32) {
        launch_attention<__bf16, float>(ctx, args, workspace, cache->head_size);
    } else if (type == ADI_HIP_F16) {
        launch_attention<_Float16, _Float16>(ctx, args, workspace, cache->head_size);
    } else {
        launch_attention<__bf16, __bf16>(ctx, args, workspace, cache->head_size);
    }
}

}  // namespace adi_hip
