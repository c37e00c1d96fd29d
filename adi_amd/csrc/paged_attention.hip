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
// 64 to 256 a block, over tiles staged in LDS, a long history's parts joined by
// k_paged_join.
//
// Floats on the 16-bit matrix cores (k_paged_chunk; the step's f32 products over
// an f32 cache are the f32 ones): an f32 value is the exact sum of three bf16
// pieces, each the leading 8 bits of what is left (truncated, so that none
// overflows), and a product is the sum of the piece products down to 2^-16 of
// it; what is left out is below 2^-22 of the largest. Scores over f32 keys take
// two f16 pieces of 11 bits each instead, of queries and keys scaled by powers of
// two that bring a row's or a key's largest element to 2^14 .. 2^15: three
// products for six, and elements down to 2^-16 of the largest keep 22 bits.
//
// Rounding: scores, levels, sums and denominators are 32 bits. 16-bit rows'
// weights are rounded once to the rows' type, as the products take them (in
// k_paged_chunk the denominator is the sum of the rounded ones, which cancels a
// part of it), and outputs once at the end.
#include "paged_attention.hpp"

#include <atomic>
#include <cmath>
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

constexpr uint32_t kSpanUnit = 128;   // parts of a history are multiples of this
constexpr float kNegative = -__builtin_huge_valf();

struct AttendArgs {
    PagedView c;
    RowsView queries, outputs, gate;
    float log2_scale;     // scale log2 e
    float slack, far;     // kSlack, kFar / log2_scale
    uint32_t window;
    uint32_t group;       // query heads of a KV head
    uint32_t span, parts; // entries of a part of a history, parts at most
    uint32_t mixed;       // nonzero: k_paged_step takes the sequences of few rows, k_paged_chunk the others
    uint32_t slots;       // k_paged_step: blocks of a KV head that the sequences share by their lengths; 0: `parts` each
    uint32_t *tickets;    // [sequence][KV head], zero between calls (k_paged_step)
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

// How far (in powers of two of a weight) a row's scores may pass the level its
// sums are held at before they are rescaled to a new one: random scores pass
// their running maximum every few tiles, so the rescaling would be a third of the
// vector work; a weight of 2^8 is as exact as one of 1.
constexpr float kSlack = 8.0f;

// How far from 0 (in powers of two of a weight) a row's level may lie for that
// slack, and for a 16-bit row's exponents in one multiply-add: beyond it a
// float's step at the level (2^-3 here) comes near the slack, and passes it.
constexpr float kFar = 1048576.0f;

__device__ __forceinline__ bool far_level(const AttendArgs &a, float m) { return fabsf(m) > a.far; }

// exp2(log2_scale (s - m)): what sums at level s are multiplied by at level m.
__device__ __forceinline__ float factor_of(const AttendArgs &a, float s, float m) {
    return __builtin_amdgcn_exp2f((s - m) * a.log2_scale);
}

// A score s has the exponent log2_scale (s - minus) + offset at a row's level m. f32
// rows take the difference first (minus = m), so that its rounding is relative to
// it. 16-bit rows do with one multiply-add, and -m log2_scale rounded once as
// the offset: as good as exact, as their sums are held at the level of that
// offset, until settle_of takes them to m's. Far levels take the difference.
// f16 rows' exponents are 7 more (sums and denominators alike, so outputs are
// not): weights are up to 2^15 with the slack, and down to 2^-31 of the level
// before one is rounded to nothing, so that it takes a history of 2^20 such
// entries to matter; bf16 has the range as it is.
struct Level {
    float minus, offset;
};
template <typename R>
constexpr float kLift = std::is_same_v<R, _Float16> ? 7.0f : 0.0f;
template <typename R>
__device__ __forceinline__ Level near_level_of(const AttendArgs &a, float maximum) {
    const float m = maximum == kNegative ? 0.0f : maximum;
    if constexpr (std::is_same_v<R, float>) {
        return {m, 0.0f};
    } else {
        return {0.0f, fmaf(-m, a.log2_scale, kLift<R>)};
    }
}
template <typename R>
__device__ __forceinline__ Level level_of(const AttendArgs &a, float maximum) {
    if constexpr (!std::is_same_v<R, float>) {
        if (maximum != kNegative && far_level(a, maximum)) {
            return {maximum, kLift<R>};
        }
    }
    return near_level_of<R>(a, maximum);
}

// The exponent of a score that `minus` is taken from already.
template <typename R>
__device__ __forceinline__ float exponent_of(const AttendArgs &a, float s, const Level &level) {
    return std::is_same_v<R, float> ? s * a.log2_scale : fmaf(s, a.log2_scale, level.offset);
}
template <typename R>
__device__ __forceinline__ float weight_of(const AttendArgs &a, float s, const Level &level) {
    return __builtin_amdgcn_exp2f(exponent_of<R>(a, s, level));
}

// What a row's sums are multiplied by when its level rises from `from` to `to`.
template <typename R>
__device__ __forceinline__ float raise_of(const AttendArgs &a, float from, float to) {
    if constexpr (std::is_same_v<R, float>) {
        return factor_of(a, from, to);
    } else {
        const Level was = level_of<R>(a, from), is = level_of<R>(a, to);
        return from == kNegative ? 0.0f
                                 : __builtin_amdgcn_exp2f(exponent_of<R>(a, to - is.minus, is) -
                                                          exponent_of<R>(a, to - was.minus, was));
    }
}

// What takes a row's sums from its offset's level to `maximum` itself, by which
// they are joined with others.
template <typename R>
__device__ __forceinline__ float settle_of(const AttendArgs &a, float maximum) {
    if constexpr (std::is_same_v<R, float>) {
        return 1.0f;
    } else {
        const Level level = level_of<R>(a, maximum);
        const float m = maximum == kNegative ? 0.0f : maximum;
        return __builtin_amdgcn_exp2f(kLift<R> - exponent_of<R>(a, m - level.minus, level));
    }
}

// Two floats as pairs of 16-bit pieces: one, rounded to nearest; three bf16
// pieces whose sum they are, exactly (an infinity gives NaN); or two f16 pieces,
// 22 bits, of values scaled to f16's range.
template <typename T, uint32_t N>
__device__ __forceinline__ void split(float x, float y, uint32_t (&out)[N]) {
    if constexpr (N == 1) {
        out[0] = pack<T>(x, y);
    } else if constexpr (N == 2) {
        const f32x2 v = {x, y};
        const f16x2 hi = __builtin_convertvector(v, f16x2);
        out[0] = __builtin_bit_cast(uint32_t, hi);
        out[1] = pack<T>(x - static_cast<float>(hi.x), y - static_cast<float>(hi.y));
    } else {
#pragma unroll
        for (uint32_t i = 0; i < N; ++i) {
            const uint32_t a = __float_as_uint(x), b = __float_as_uint(y);
            out[i] = __builtin_amdgcn_perm(b, a, 0x07060302u);
            x -= __uint_as_float(a & 0xFFFF0000u);
            y -= __uint_as_float(b & 0xFFFF0000u);
        }
    }
}

// The power of two that brings values of a largest magnitude of these float bits
// to 2^14 .. 2^15, as an exponent (2^126 at most), and the power that takes it
// back. A score's two powers are added before they are applied: by itself either
// may pass a float's range where the score does not.
__device__ __forceinline__ uint32_t scale_exponent(uint32_t largest) { return min(268u - (largest >> 23), 253u); }
__device__ __forceinline__ float scale_of(uint32_t exponent) { return __uint_as_float(exponent << 23); }
__device__ __forceinline__ int32_t unscale_of(uint32_t exponent) { return 127 - static_cast<int32_t>(exponent); }
__device__ __forceinline__ uint32_t magnitude(uint32_t largest, float v) {
    return max(largest, __float_as_uint(v) & 0x7FFFFFFFu);
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

// The piece products of a K step, smallest first: all down to 2^-16 of a product
// of three pieces (of 8 bits), or 2^-11 of two (of 11).
template <typename T, uint32_t A, uint32_t B, typename C>
__device__ __forceinline__ C product(const u32x4 (&a)[A], const u32x4 (&b)[B], C c) {
#pragma unroll
    for (int32_t order = A == 2u ? 1 : 2; order >= 0; --order) {
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

// The same for X sums at once, turn by turn: a product that adds to the one
// before it waits twice its own time.
template <typename T, uint32_t X, uint32_t A, uint32_t B, typename C>
__device__ __forceinline__ void products(const u32x4 (&a)[X][A], const u32x4 (&b)[B], C *(&c)[X]) {
#pragma unroll
    for (int32_t order = A == 2u ? 1 : 2; order >= 0; --order) {
#pragma unroll
        for (int32_t i = 0; i < static_cast<int32_t>(A); ++i) {
            const int32_t j = order - i;
            if (j >= 0 && j < static_cast<int32_t>(B)) {
#pragma unroll
                for (uint32_t x = 0; x < X; ++x) {
                    *c[x] = mfma<T>(a[x][i], b[j], *c[x]);
                }
            }
        }
    }
}

// sum plus both values of a pair, in 32 bits.
template <typename T>
__device__ __forceinline__ float pair_sum(uint32_t pair, float sum) {
    if constexpr (std::is_same_v<T, _Float16>) {
        const f16x2 one = {1.0f, 1.0f};
        return __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, pair), one, sum, false);
    } else {
        const bf16x2 one = {1.0f, 1.0f};
        return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, pair), one, sum, false);
    }
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

// The weight of an entry for a row at its maximum so far, outside the tiles' way:
// for the few entries that hold values that are not finite.
template <typename T, typename R, uint32_t D>
__device__ __forceinline__ float odd_weight(const AttendArgs &a, const uint32_t *table, const T *keys, const R *query,
                                         uint32_t entry, float maximum) {
    const T *const key = keys + page_of(a.c, table, entry).at;
    float score = 0.0f;
    for (uint32_t d = 0; d < D; ++d) {
        score = fmaf(static_cast<float>(query[d]), static_cast<float>(key[d]), score);
    }
    const Level level = level_of<R>(a, maximum);
    return weight_of<R>(a, score - level.minus, level);
}

// N consecutive outputs of a row, gated unless the row sees nothing (whose gate
// may be whatever a padded row holds).
template <typename R, uint32_t N>
__device__ __forceinline__ void store_output(const AttendArgs &a, uint32_t token, uint32_t head, uint32_t at,
                                             float (&v)[N], bool none = false) {
    struct alignas(sizeof(R) * N) Vector {
        R v[N];
    };
    if (a.gate.data != nullptr && !none) {
        const Vector g = *reinterpret_cast<const Vector *>(reinterpret_cast<const R *>(a.gate.data) +
                                                           token * a.gate.token_stride + head * a.gate.head_stride +
                                                           at);
#pragma unroll
        for (uint32_t k = 0; k < N; ++k) {
            v[k] *= 1.0f / (1.0f + expf(-static_cast<float>(g.v[k])));
        }
    }
    store_values<R, N>(reinterpret_cast<R *>(a.outputs.data) + token * a.outputs.token_stride +
                           head * a.outputs.head_stride + at,
                       v);
}

// Rows of a sequence that nothing is computed for: NaN where it is over the
// batch's bounds, 0 where it has no entries. By one block, for a KV head.
template <typename R, uint32_t D>
__device__ __forceinline__ void fill_rows(const AttendArgs &a, const SequenceRows &s, uint32_t kv) {
    const uint64_t items = static_cast<uint64_t>(s.count) * a.group * (D / 4u);
    for (uint64_t i = threadIdx.x; i < items; i += blockDim.x) {
        const uint32_t row = static_cast<uint32_t>(i / (D / 4u)), at = static_cast<uint32_t>(i % (D / 4u)) * 4u;
        const float v = s.over ? __builtin_nanf("") : 0.0f;
        float out[4] = {v, v, v, v};
        store_output<R, 4>(a, s.first + row / a.group, kv * a.group + row % a.group, at, out, true);
    }
}

// LDS places: the 16-byte pieces of an entry's D 16-bit values are permuted so
// that the reads of a phase fall on different banks. Keys: the 16 entries that a
// phase's lanes read at one piece get different turns. Values: the entries that
// a transposing read's half wave reads side by side, four at 64 bytes (32
// rows a wave) or eight at 32 bytes (16). A row of 64 values is half the banks,
// so two rows share a turn.
template <uint32_t D, uint32_t ROWS>
__device__ __forceinline__ uint32_t key_place(uint32_t row, uint32_t piece) {
    uint32_t turn;
    if constexpr (ROWS == 32) {
        turn = D == 64u ? (row >> 1) & 7u : row & 15u;
    } else {
        turn = D == 64u ? (row >> 1 & 1u) | (row >> 3 & 3u) << 1 : (row & 3u) | (row >> 3 & 3u) << 2;
    }
    return row * (D * 2u) + ((piece ^ turn) << 4);
}
template <uint32_t D, uint32_t ROWS>
__device__ __forceinline__ uint32_t value_place(uint32_t row, uint32_t piece) {
    uint32_t turn;
    if constexpr (ROWS == 32) {
        turn = D == 64u ? (row & 2u) << 1 : (row & 3u) << 2;
    } else {
        turn = D == 64u ? (row & 2u) | (row >> 3 & 1u) << 2 : (row & 3u) << 1 | (row >> 3 & 1u) << 3;
    }
    return row * (D * 2u) + ((piece ^ turn) << 4);
}

// ---- up to 16 rows a KV head --------------------------------------------------

constexpr uint32_t kStepParts = 128;  // parts of a history at most

// Used one after another: the rows' queries, the waves' sums, the parts to join.
template <uint32_t D>
struct StepLds {
    union {
        __align__(16) unsigned char query[kStepRows * D * 6u];
        __align__(16) float sums[4][kStepRows][D + 4u];
        struct {
            // (a row's parts lie in as many banks)
            float factor[kStepParts][kStepRows + 1u], total[kStepParts][kStepRows + 1u];
            __align__(16) f32x4 group[kThreads];
        } parts;
    };
    float maximum[4][kStepRows], denominator[4][kStepRows];
    uint32_t last;
};

// 16 bytes written through to memory, and read past the caches that another
// XCD's writes do not reach.
__device__ __forceinline__ void store_through(float *base, uint32_t at, f32x4 v) {
    const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(base, 0, 0x7FFFFFFF, 0x00020000);
    __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, v), rs, at * 4u, 0, 16 /* sc1 */);
}
__device__ __forceinline__ f32x4 load_through(const float *base, uint32_t at) {
    const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(const_cast<float *>(base), 0, 0x7FFFFFFF, 0x00020000);
    return __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rs, at * 4u, 0, 16 /* sc1 */));
}

// Whether a tile's values are on their way beside its keys, or take the keys'
// registers when its scores are done; and the blocks a CU holds, by registers
// (which at heads of 64 and 128 have room for three or four: more than two have
// been timed at 256 only).
template <typename T, typename R, uint32_t D>
constexpr bool step_eager() {
    return D < 256u || sizeof(R) > sizeof(T);
}
template <typename T, typename R, uint32_t D>
constexpr uint32_t step_blocks() {
    return D == 256u ? (step_eager<T, R, D>() ? 1u : 2u) : 2u;
}

// Bound by the entries' bytes where there are many: two sequences behind 131,071
// entries, 8 heads of 128 in bf16, 832 MB in 148 us, 5.6 TB/s, above a large copy's
// 5.1; 32 sequences of up to 4,096 entries, 153 MB, 40 us from HBM, 3.8 TB/s (a
// block's start and end are some 8 us; 34 where the last call left them in the
// last-level cache). Where there are few,
// by its chain of latencies: one token behind 1,999 entries of 2 heads of 256 in
// f32, 8.2 MB, 18 us: some 4 to start, page numbers, a tile's loads and products
// 3, the join of 32 parts 7.
//
// Block (KV head, part, sequence), the parts of 2 to 64 sequences by their lengths,
// of others by max_length: its four waves take the part's tiles in turn,
// each straight from the cache into operands, the next tile's keys on their way
// from the end of this one's scores and its values from the end of their
// products. Lane l is column c = l % 16 (a row), quarter g = l / 16. The blocks
// of a history of several parts leave theirs in the workspace, a region of
// kStepRows rows of D + 4 each (whole cache lines, so that no two blocks write
// one), and the last through the ticket joins them.
template <typename T, typename R, uint32_t D>
__global__ __launch_bounds__(kThreads, (step_blocks<T, R, D>())) void k_paged_step(AttendArgs args) {
    constexpr bool kFloat = std::is_same_v<T, float>;  // the cache's type
    constexpr uint32_t P = std::is_same_v<R, float> ? 3u : 1u;
    // a wave's tile, and the keys of a tile that a lane holds: kKeys / 4 in a row
    constexpr uint32_t kKeys = kFloat ? 16u : 32u, kHeld = kKeys / 4u;
    // dimensions of a value row that a lane holds side by side, and groups of 16 lanes' worth
    constexpr uint32_t kSide = kFloat ? 4u : D == 64u ? 4u : 8u, kGroups = D / (16u * kSide);
    constexpr uint32_t kRegion = kStepRows * (D + 4u);
    constexpr bool kEager = step_eager<T, R, D>();
    constexpr int32_t kTurn = 4 * kKeys;  // entries of the four waves' tiles
    static_assert(kRegion * sizeof(float) % 128u == 0u);
    __shared__ StepLds<D> lds;
    const PagedView &cache = args.c;
    const uint32_t kv = blockIdx.x % cache.heads;
    const uint32_t t = threadIdx.x, lane = t & 63u, wave = t >> 6;
    const uint32_t c = lane & 15u, g = lane >> 4;
    const auto takes = [&](const SequenceRows &of) {
        return of.count != 0u && (args.mixed == 0u || of.count * args.group <= kStepRows);
    };
    SequenceRows s;
    uint32_t part = blockIdx.x / cache.heads, sequence = blockIdx.y, span = args.span;
    // the regions of the workspace of this (sequence, KV head): the first, and
    // how many lie from one part's to the next's
    uint32_t region_base = (sequence * cache.heads + kv) * args.parts, region_step = 1u;
    if (args.slots != 0u) {
        // Up to 64 sequences, one a lane: a span with which their parts fit the
        // slots. A sequence's last part is half empty on the average, so total /
        // (slots - sequences / 2) entries; where that is too short total / (slots -
        // sequences), which always fits, as a sequence has less than one part more
        // than its share.
        const SequenceRows own =
            lane < cache.sequences ? sequence_rows(cache, lane) : SequenceRows{0u, 0u, 0u, false};
        const bool taken = takes(own);
        const int32_t own_first = static_cast<int32_t>(own.length) - static_cast<int32_t>(own.count);
        const uint32_t extent = !taken                          ? 0u
                                : own.over || own.length == 0u ? 1u
                                                               : own.length - static_cast<uint32_t>(base_of(args, own_first));
        float total = static_cast<float>(extent);
        total += lane_xor<1>(total);
        total += lane_xor<2>(total);
        total += lane_xor<4>(total);
        total += lane_xor<8>(total);
        total += lane_xor<16>(total);
        total += lane_xor<32>(total);
        const float live_sequences = static_cast<float>(__popcll(__ballot(taken)));
        uint32_t parts = 0, sum = 0;
#pragma unroll 1
        for (uint32_t attempt = 0; attempt < 2u; ++attempt) {
            // (more slots than sequences; the sums' roundings are below 2^-17)
            const float left = static_cast<float>(args.slots) - live_sequences * (attempt == 0u ? 0.5f : 1.0f);
            // (2^28 entries hold any history whole, and are an integer that has room
            // to be rounded up)
            const float wanted = fminf(total * 1.0001f / left, 268435456.0f);
            span = max(args.span, (static_cast<uint32_t>(wanted) + kTurn) & ~(static_cast<uint32_t>(kTurn) - 1u));
            parts = (extent + span - 1u) / span;
            sum = parts;
#pragma unroll
            for (uint32_t d = 1; d < 64u; d *= 2u) {
                const uint32_t below = __shfl_up(sum, d);
                sum += lane >= d ? below : 0u;
            }
            if (__shfl(sum, 63) <= args.slots) {
                break;
            }
        }
        const uint64_t past = __ballot(sum > part);
        if (past == 0u) {
            return;
        }
        const int at = __ffsll(static_cast<unsigned long long>(past)) - 1;
        const auto of = [&](uint32_t v) {
            return static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v), at));
        };
        sequence = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(at));
        const uint32_t before = of(sum) - of(parts);
        part -= before;
        region_base = before * cache.heads + kv;
        region_step = cache.heads;
        s = {of(own.first), of(own.count), of(own.length), of(own.over ? 1u : 0u) != 0u};
        span = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(span)));
    } else {
        s = sequence_rows(cache, sequence);
        if (!takes(s)) {
            return;
        }
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
    const int32_t base = base_of(args, first_position);
    const int32_t begin = base + static_cast<int32_t>(part * span);
    const int32_t end = static_cast<int32_t>(min(static_cast<uint32_t>(begin) + span, s.length));
    if (begin >= end) {
        return;
    }
    const uint32_t live = (s.length - static_cast<uint32_t>(base) + span - 1u) / span;
    // entries that some row sees, and those that every row sees
    const int32_t seen_from = window == 0 ? 0 : max(0, first_position - window + 1);
    const int32_t all_from = window == 0 ? 0 : max(0, static_cast<int32_t>(s.length) - window);
    const uint32_t *const table = cache.table + static_cast<uint64_t>(sequence) * cache.table_stride;
    const T *const keys = reinterpret_cast<const T *>(cache.keys) + kv * cache.head_stride;
    const T *const values = reinterpret_cast<const T *>(cache.values) + kv * cache.head_stride;

    // Key operands: row i of A is key first + kHeld (i / 4) + i % 4 (+ 4 in the
    // second of two products with 32 keys), so that register r of the results
    // is key first + kHeld g + r. Groups of 8 entries from a multiple of 8 share a
    // page: this lane's for the keys it reads and for the values.
    const uint32_t key_group = (kHeld * (c >> 2)) & ~7u, value_group = (kHeld * g) & ~7u;
    const uint64_t key_at = ((kHeld * (c >> 2) & 7u) + (c & 3u)) * cache.entry_stride;
    const uint64_t value_at = ((kHeld * g) & 7u) * cache.entry_stride;
    struct Numbers {
        uint32_t key, value;
    };
    const auto numbers_of = [&](int32_t first) {
        const uint32_t last = static_cast<uint32_t>(end - 1);
        return Numbers{table[min(first + key_group, last) >> cache.page_shift],
                       table[min(first + value_group, last) >> cache.page_shift]};
    };
    const uint32_t page_mask = (1u << cache.page_shift) - 1u;
    // (a page that there is not: page 0 stands in, which is always there to be read)
    const auto place_of = [&](uint32_t number, uint32_t entry) {
        return (number >= cache.pages ? 0u : number) * cache.page_stride + (entry & page_mask) * cache.entry_stride;
    };

    f32x4 key_float[kFloat ? D / 16u : 1u];
    u32x4 key_half[kFloat ? 1u : 2u][kFloat ? 1u : D / 32u][1];
    using Chunk = std::conditional_t<kFloat, f32x4, std::conditional_t<kSide == 8u, u32x4, u32x2>>;
    Chunk held[kGroups][kHeld];
    const auto load_keys = [&](const Numbers &n, int32_t first) {
        const T *const key = keys + place_of(n.key, first + key_group) + key_at;
        if constexpr (kFloat) {
#pragma unroll
            for (uint32_t j = 0; j < D / 16u; ++j) {
                key_float[j] = *reinterpret_cast<const f32x4 *>(key + 16u * j + 4u * g);
            }
        } else {
#pragma unroll
            for (uint32_t h = 0; h < 2u; ++h) {
#pragma unroll
                for (uint32_t j = 0; j < D / 32u; ++j) {
                    key_half[h][j][0] =
                        *reinterpret_cast<const u32x4 *>(key + 4u * h * cache.entry_stride + 32u * j + 8u * g);
                }
            }
        }
    };
    const auto load_values = [&](const Numbers &n, int32_t first) {
        const T *const value = values + place_of(n.value, first + value_group) + value_at;
#pragma unroll
        for (uint32_t i = 0; i < kGroups; ++i) {
#pragma unroll
            for (uint32_t k = 0; k < kHeld; ++k) {
                held[i][k] = *reinterpret_cast<const Chunk *>(value + k * cache.entry_stride + 16u * kSide * i +
                                                              kSide * c);
            }
        }
    };

    int32_t first = begin + static_cast<int32_t>(wave * kKeys);
    Numbers now{0, 0}, next{0, 0};
    if (first < end) {
        now = numbers_of(first);
        load_keys(now, first);
        if constexpr (kEager) {
            load_values(now, first);
        }
        next = numbers_of(first + kTurn);
    }

    // the row's query as the products take it
    const R *const query = reinterpret_cast<const R *>(args.queries.data) + token * args.queries.token_stride +
                           head * args.queries.head_stride;
    // (f32 rows through LDS: as floats or in three pieces they are a quarter of the
    // registers, which then hold two blocks a CU)
    constexpr uint32_t kPlane = kStepRows * D * 2u;
    const auto query_place = [&](uint32_t piece) {
        if constexpr (kFloat) {
            return c * (D * 4u) + ((piece ^ c) << 4);
        } else {
            return key_place<D, 32>(c, piece);
        }
    };
    u32x4 query_pieces[P == 1u ? D / 32u : 1u][1];
    if constexpr (P == 1) {
#pragma unroll
        for (uint32_t j = 0; j < D / 32u; ++j) {
            query_pieces[j][0] = *reinterpret_cast<const u32x4 *>(query + 32u * j + 8u * g);
        }
    } else {
        if constexpr (kFloat) {
#pragma unroll
            for (uint32_t j = 0; j < D / 64u; ++j) {
                const uint32_t piece = 4u * (4u * j + wave) + g;
                *reinterpret_cast<f32x4 *>(lds.query + query_place(piece)) =
                    *reinterpret_cast<const f32x4 *>(query + 4u * piece);
            }
        } else {
            for (uint32_t j = wave; j < D / 32u; j += 4u) {
                const f32x4 lo = *reinterpret_cast<const f32x4 *>(query + 32u * j + 8u * g);
                const f32x4 hi = *reinterpret_cast<const f32x4 *>(query + 32u * j + 8u * g + 4u);
                u32x4 out[P];
#pragma unroll
                for (uint32_t k = 0; k < 4u; ++k) {
                    uint32_t pieces[P];
                    k < 2u ? split<T>(lo[2u * k], lo[2u * k + 1u], pieces)
                           : split<T>(hi[2u * k - 4u], hi[2u * k - 3u], pieces);
#pragma unroll
                    for (uint32_t p = 0; p < P; ++p) {
                        out[p][k] = pieces[p];
                    }
                }
#pragma unroll
                for (uint32_t p = 0; p < P; ++p) {
                    *reinterpret_cast<u32x4 *>(lds.query + p * kPlane + query_place(4u * j + g)) = out[p];
                }
            }
        }
        __syncthreads();
    }

    f32x4 sums[kGroups][kSide];
#pragma unroll
    for (uint32_t i = 0; i < kGroups; ++i) {
#pragma unroll
        for (uint32_t k = 0; k < kSide; ++k) {
            sums[i][k] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        }
    }
    // the level of the row's weights (kNegative before its first score), and the
    // score from which it is raised
    float maximum = kNegative, limit = kNegative, denominator = 0.0f;
    bool far = false;  // some row's level is
    // a tile that some row does not see whole
    const auto edge_tile = [&](int32_t at) {
        return at + static_cast<int32_t>(kKeys) > first_position + 1 || at < all_from;
    };
    bool odd_tile = false;

    for (; first < end; first += kTurn) {
        float score[kHeld];
        if constexpr (kFloat) {
            // (four sums of 64 dimensions at most: with two the scores' roundings were twice
            // those of a plain 32-bit product)
            f32x4 acc[4] = {};
#pragma unroll
            for (uint32_t j = 0; j < D / 16u; ++j) {
                const f32x4 q = *reinterpret_cast<const f32x4 *>(lds.query + query_place(4u * j + g));
#pragma unroll
                for (uint32_t i = 0; i < 4u; ++i) {
                    acc[j & 3u] =
                        __builtin_amdgcn_mfma_f32_16x16x4f32(key_float[j][i], q[i], acc[j & 3u], 0, 0, 0);
                }
            }
#pragma unroll
            for (uint32_t r = 0; r < 4u; ++r) {
                score[r] = (acc[0][r] + acc[1][r]) + (acc[2][r] + acc[3][r]);
            }
        } else {
            f32x4 acc[2] = {{0.0f, 0.0f, 0.0f, 0.0f}, {0.0f, 0.0f, 0.0f, 0.0f}};
#pragma unroll
            for (uint32_t j = 0; j < D / 32u; ++j) {
                u32x4 q[P];
#pragma unroll
                for (uint32_t p = 0; p < P; ++p) {
                    if constexpr (P == 1u) {
                        q[p] = query_pieces[j][p];
                    } else {
                        q[p] = *reinterpret_cast<const u32x4 *>(lds.query + p * kPlane + query_place(4u * j + g));
                    }
                }
                u32x4 k[2][1] = {{key_half[0][j][0]}, {key_half[1][j][0]}};
                f32x4 *to[2] = {&acc[0], &acc[1]};
                products<T>(k, q, to);
            }
#pragma unroll
            for (uint32_t h = 0; h < 2u; ++h) {
#pragma unroll
                for (uint32_t r = 0; r < 4u; ++r) {
                    score[4u * h + r] = acc[h][r];
                }
            }
        }
        const bool bad = now.value >= cache.pages;
        if constexpr (!kEager) {
            load_values(now, first);
        }
        now = next;
        if (kEager && first + kTurn < end) {
            load_keys(now, first + kTurn);
        }
        if (first + 2 * kTurn < end) {
            next = numbers_of(first + 2 * kTurn);
        }
        const int32_t own_first = first + static_cast<int32_t>(kHeld * g);  // the lane's keys
        if (__any(edge_tile(first) || bad)) {
            bool odd = false;
#pragma unroll
            for (uint32_t k = 0; k < kHeld; ++k) {
                const int32_t entry = own_first + static_cast<int32_t>(k);
                const bool visible = entry <= position && entry >= oldest;
                score[k] = !visible ? kNegative : bad ? __builtin_nanf("") : score[k];
                // (what no row sees is whatever the page held before)
                const bool any = entry < end && entry >= seen_from && !bad;
#pragma unroll
                for (uint32_t i = 0; i < kGroups; ++i) {
                    constexpr uint32_t kWords = sizeof(Chunk) / 4u;
#pragma unroll
                    for (uint32_t w = 0; w < kWords; ++w) {
                        held[i][k][w] = any ? held[i][k][w] : 0;
                        // (with one token every row sees the same entries)
                        if (s.count > 1u) {
                            if constexpr (kFloat) {
                                odd |= odd_float(held[i][k][w]);
                                held[i][k][w] = odd_float(held[i][k][w]) ? 0.0f : held[i][k][w];
                            } else {
                                odd |= odd_pair<T>(held[i][k][w]);
                                held[i][k][w] = clean_pair<T>(held[i][k][w]);
                            }
                        }
                    }
                }
            }
            odd_tile |= __any(odd) != 0;
        }
        float top = score[0];
#pragma unroll
        for (uint32_t k = 1; k < kHeld; ++k) {
            top = fmaxf(top, score[k]);
        }
        top = fmaxf(top, lane_xor<16>(top));
        top = fmaxf(top, lane_xor<32>(top));
        if (__any(top > limit)) {
            // (a row's level does not depend on the wave's other rows)
            const bool raised = top > limit;
            const float factor = raised ? raise_of<R>(args, maximum, top) : 1.0f;
            maximum = raised ? top : maximum;
            limit = raised ? top + (far_level(args, top) ? 0.0f : args.slack) : limit;
            far = __any(maximum != kNegative && far_level(args, maximum)) != 0;
            denominator *= factor;
#pragma unroll
            for (uint32_t i = 0; i < kGroups; ++i) {
#pragma unroll
                for (uint32_t k = 0; k < kSide; ++k) {
                    sums[i][k] *= factor;
                }
            }
        }
        Level level = near_level_of<R>(args, maximum);
        if (P == 1u && far) {
            level = level_of<R>(args, maximum);
#pragma unroll
            for (uint32_t k = 0; k < kHeld; ++k) {
                score[k] -= level.minus;
            }
        }
#pragma unroll
        for (uint32_t k = 0; k < kHeld; ++k) {
            score[k] = weight_of<R>(args, P == 3u ? score[k] - level.minus : score[k], level);
            denominator += score[k];
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
        if (first + kTurn < end) {
            if constexpr (kEager) {
                load_values(now, first + kTurn);
            } else {
                load_keys(now, first + kTurn);
            }
        }
    }

    if (odd_tile) {
        // Values that are not finite, in tiles of which some rows see only a
        // part: the products left them out, the rows that see them get them.
        for (int32_t at = begin + static_cast<int32_t>(wave * kKeys); at < end; at += kTurn) {
            for (int32_t entry = at; edge_tile(at) && entry < min(at + static_cast<int32_t>(kKeys), end); ++entry) {
                const float weight = odd_weight<T, R, D>(args, table, keys, query, entry, maximum);
                const bool visible = entry <= position && entry >= oldest;
                const Page page = page_of(cache, table, entry);
                const T *const value = values + page.at;
#pragma unroll
                for (uint32_t i = 0; i < kGroups; ++i) {
#pragma unroll
                    for (uint32_t n = 0; n < kSide; ++n) {
#pragma unroll
                        for (uint32_t r = 0; r < 4u; ++r) {
                            const float v = static_cast<float>(value[16u * kSide * i + kSide * (4u * g + r) + n]);
                            sums[i][n][r] += visible && !page.bad && odd_float(v) ? v * weight : 0.0f;
                        }
                    }
                }
            }
        }
    }

    // the row's lanes' parts of the denominator, then the waves
    denominator += lane_xor<16>(denominator);
    denominator += lane_xor<32>(denominator);
    const float settle = settle_of<R>(args, maximum);
    denominator *= settle;
    if (g == 0u) {
        lds.maximum[wave][c] = maximum;
        lds.denominator[wave][c] = denominator;
    }
    __syncthreads();
    const auto join_factor = [&](float m, float top) {
        return m == kNegative && top == kNegative ? 1.0f : factor_of(args, m, top);
    };
    const auto top_of = [&](uint32_t r) {
        return fmaxf(fmaxf(lds.maximum[0][r], lds.maximum[1][r]), fmaxf(lds.maximum[2][r], lds.maximum[3][r]));
    };
    if (c < rows) {
        const float factor = join_factor(maximum, top_of(c)) * settle;
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
    __syncthreads();
    const auto store_row = [&](uint32_t r, uint32_t at, f32x4 sum, float total) {
        const bool none = first_position + static_cast<int32_t>(r / args.group) < 0;
        float out[4];
#pragma unroll
        for (uint32_t k = 0; k < 4u; ++k) {
            out[k] = none ? 0.0f : sum[k] / total;
        }
        store_output<R, 4>(args, s.first + r / args.group, kv * args.group + r % args.group, at, out, none);
    };
    float *const joint = args.partial + static_cast<uint64_t>(region_base) * kRegion;
    const uint32_t part_step = region_step * kRegion;
    for (uint32_t i = t; i < rows * (D / 4u); i += kThreads) {
        const uint32_t r = i / (D / 4u), at = i % (D / 4u) * 4u;
        const float top = top_of(r);
        float total = 0.0f;
        f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (uint32_t w = 0; w < 4u; ++w) {
            total += lds.denominator[w][r] * join_factor(lds.maximum[w][r], top);
            sum += *reinterpret_cast<const f32x4 *>(&lds.sums[w][r][at]);
        }
        if (live == 1u) {
            store_row(r, at, sum, total);
            continue;
        }
        float *const region = joint + static_cast<uint64_t>(part) * part_step;
        store_through(region, r * (D + 4u) + at, sum);
        if (at == 0u) {
            store_through(region, r * (D + 4u) + D, f32x4{top, total, 0.0f, 0.0f});
        }
    }
    if (live == 1u) {
        return;
    }
    wait_stores();
    __syncthreads();
    uint32_t *const ticket = args.tickets + static_cast<uint64_t>(sequence) * cache.heads + kv;
    if (t == 0u) {
        lds.last = coherent_add(ticket, 1u) + 1u == live ? 1u : 0u;
    }
    __syncthreads();
    if (lds.last == 0u) {
        return;
    }
    if (t == 0u) {
        coherent_store(ticket, 0u);
    }
    // the parts' levels and denominators, all on their way at once, then a row's
    // top, factors and total by a wave
    for (uint32_t i = t; i < live * rows; i += kThreads) {
        const uint32_t p = i / rows, r = i % rows;
        const f32x4 v = load_through(joint, p * part_step + r * (D + 4u) + D);
        lds.parts.factor[p][r] = v[0];
        lds.parts.total[p][r] = v[1];
    }
    __syncthreads();
    for (uint32_t r = wave; r < rows; r += 4u) {
        float m[kStepParts / 64u], top = kNegative, total = 0.0f;
#pragma unroll
        for (uint32_t i = 0; i < kStepParts / 64u; ++i) {
            m[i] = 64u * i + lane < live ? lds.parts.factor[64u * i + lane][r] : kNegative;
            top = fmaxf(top, m[i]);
        }
        top = fmaxf(top, lane_xor<1>(top));
        top = fmaxf(top, lane_xor<2>(top));
        top = fmaxf(top, lane_xor<4>(top));
        top = fmaxf(top, lane_xor<8>(top));
        top = fmaxf(top, lane_xor<16>(top));
        top = fmaxf(top, lane_xor<32>(top));
#pragma unroll
        for (uint32_t i = 0; i < kStepParts / 64u; ++i) {
            if (64u * i + lane < live) {
                const float factor = join_factor(m[i], top);
                total += lds.parts.total[64u * i + lane][r] * factor;
                lds.parts.factor[64u * i + lane][r] = factor;
            }
        }
        total += lane_xor<1>(total);
        total += lane_xor<2>(total);
        total += lane_xor<4>(total);
        total += lane_xor<8>(total);
        total += lane_xor<16>(total);
        total += lane_xor<32>(total);
        if (lane == 0u) {
            lds.denominator[0][r] = total;
        }
    }
    __syncthreads();
    // then their sums, four dimensions of a row a thread; where that leaves
    // threads over, groups of them take the parts in turn
    const uint32_t items = rows * (D / 4u), groups = max(kThreads / items, 1u);
    const auto sum_of = [&](uint32_t i, uint32_t from, uint32_t step) {
        const uint32_t r = i / (D / 4u), at = r * (D + 4u) + i % (D / 4u) * 4u;
        f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
        constexpr uint32_t kAhead = 16;  // loads on their way at once
        for (uint32_t p = from; p < live; p += kAhead * step) {
            f32x4 v[kAhead];
#pragma unroll
            for (uint32_t u = 0; u < kAhead; ++u) {
                v[u] = load_through(joint, min(p + u * step, live - 1u) * part_step + at);
            }
#pragma unroll
            for (uint32_t u = 0; u < kAhead; ++u) {
                if (p + u * step < live) {
                    sum += v[u] * lds.parts.factor[p + u * step][r];
                }
            }
        }
        return sum;
    };
    if (groups == 1u) {
        for (uint32_t i = t; i < items; i += kThreads) {
            const uint32_t r = i / (D / 4u);
            store_row(r, i % (D / 4u) * 4u, sum_of(i, 0u, 1u), lds.denominator[0][r]);
        }
        return;
    }
    f32x4 *const parts = lds.parts.group;
    if (t < groups * items) {
        parts[t] = sum_of(t % items, t / items, groups);
    }
    __syncthreads();
    if (t < items) {
        f32x4 sum = parts[t];
        for (uint32_t q = 1; q < groups; ++q) {
            sum += parts[q * items + t];
        }
        const uint32_t r = t / (D / 4u);
        store_row(r, t % (D / 4u) * 4u, sum, lds.denominator[0][r]);
    }
}

// ---- joining the parts of a history -------------------------------------------

// A wave a row (token, query head) of more than one part: lane l takes the
// factors of parts l, l + 64, ... and dimensions D / 64 l .. of every part. Bound
// by the parts' bytes, which the chunks have just written: 8,192 rows of four
// parts of 256, 34 MB, 12.5 us.
template <typename R, uint32_t D>
__global__ __launch_bounds__(kThreads) void k_paged_join(AttendArgs args) {
    constexpr uint32_t kSide = D / 64u;
    const PagedView &cache = args.c;
    const uint32_t heads = cache.heads * args.group, lane = threadIdx.x & 63u;
    const uint64_t rows = static_cast<uint64_t>(cache.tokens) * heads;
    for (uint64_t row = blockIdx.x * 4ull + (threadIdx.x >> 6); row < rows; row += gridDim.x * 4ull) {
        const uint32_t token = static_cast<uint32_t>(row / heads), head = static_cast<uint32_t>(row % heads);
        uint32_t sequence = 0;
        for (uint32_t s = 0; s < cache.sequences; s += 64u) {
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
        if (token < s.first || token - s.first >= s.count || s.over || s.length == 0u ||
            (args.mixed != 0u && s.count * args.group <= kStepRows)) {
            continue;  // (filled by the attention itself, or joined there)
        }
        const int32_t first_position = static_cast<int32_t>(s.length) - static_cast<int32_t>(s.count);
        const int32_t position = first_position + static_cast<int32_t>(token - s.first);
        const int32_t base = base_of(args, first_position);
        const int32_t window = static_cast<int32_t>(args.window);
        const int32_t oldest = window == 0 ? 0 : max(0, position - window + 1);
        const uint32_t from = static_cast<uint32_t>(oldest - base) / args.span;
        const uint32_t to = position < 0 ? from : static_cast<uint32_t>(position - base) / args.span;
        if (from == to) {
            continue;  // (written by its one part)
        }
        float top = kNegative;
        for (uint32_t p = from + lane; p <= to; p += 64u) {
            top = fmaxf(top, partial_row<D>(args, p, token, head)[D]);
        }
        top = fmaxf(top, lane_xor<1>(top));
        top = fmaxf(top, lane_xor<2>(top));
        top = fmaxf(top, lane_xor<4>(top));
        top = fmaxf(top, lane_xor<8>(top));
        top = fmaxf(top, lane_xor<16>(top));
        top = fmaxf(top, lane_xor<32>(top));
        float total = 0.0f, sum[kSide];
#pragma unroll
        for (uint32_t k = 0; k < kSide; ++k) {
            sum[k] = 0.0f;
        }
        struct alignas(4u * kSide) Side {
            float v[kSide];
        };
#pragma unroll 8
        for (uint32_t p = from; p <= to; ++p) {
            const float *part = partial_row<D>(args, p, token, head);
            const float m = part[D], d = part[D + 1u];
            const Side v = *reinterpret_cast<const Side *>(part + kSide * lane);
            const float factor = m == kNegative && top == kNegative ? 1.0f : factor_of(args, m, top);
            total += d * factor;
#pragma unroll
            for (uint32_t k = 0; k < kSide; ++k) {
                sum[k] += v.v[k] * factor;
            }
        }
        const float scale = 1.0f / total;
#pragma unroll
        for (uint32_t k = 0; k < kSide; ++k) {
            sum[k] *= scale;
        }
        store_output<R, kSide>(args, token, head, kSide * lane, sum);
    }
}

// ---- more rows ----------------------------------------------------------------

// The shapes of k_paged_chunk: rows of a wave (the columns of its matrix
// products, 32 or 16), waves, keys of a tile, tiles in LDS at once, blocks a CU.
// A wave alone issues a vector instruction every 7 cycles or so and two fill the
// vector unit (16 multiply-adds a wave: 49 ns alone, 55 ns for both), so a SIMD
// gets two waves at least. 32 rows a wave read half as much LDS for a product,
// but a row's sums and queries then take D * 3 / 4 registers. Of what the
// registers and the 160 KB of LDS leave room for, the fastest of a sweep; in us of
// the kernels as they were then (10 to 15% above the present ones'), rows x
// keys (waves, tiles, blocks a CU), the kept one first:
//   16 bits,  64, a prompt of 8192:  32x64 (4, 1, 3) 424, 16x128 (8, 1, 2) 428,
//                                    16x64 (8, 1, 2) 482, 32x64 (8, 1, 1) 500
//   16 bits, 128, 5 ragged chunks:   32x64 (8, 2, 1) 165, 32x64 (8, 1, 1) 170,
//                                    32x32 (8, 2, 1) 186, 16x64 (8, 2, 1) 201
// and for a chunk of 2048 behind 2048, 16 heads:
//   16 bits, 256:         16x64 (8, 1, 1) 195, 16x32 (4, 1, 2) 220, 32x32 (4, 2, 1) 286
//   f32 and f32,  64:     16x64 (4, 1, 2) 191, 16x64 (8, 1, 1) 197, 16x32 (8, 1, 1) 248
//   f32 and f32, 128:     16x64 (8, 1, 1) 308, 16x32 (8, 1, 1) 348, 16x64 (4, 1, 2) 424
//   f32 and bf16,  64:    16x64 (4, 1, 2) 113, 16x64 (8, 1, 1) 127, 16x32 (8, 1, 1) 169
//   f32 and bf16, 128:    16x64 (4, 1, 2) 169, 16x64 (8, 1, 1) 185, 16x32 (8, 1, 1) 216
//   f32 and bf16, 256:    16x32 (8, 1, 1) 367, 16x64 (8, 1, 1) 372, 16x32 (4, 1, 2) 477
// f32 and f32 at 256 has LDS for one tile of 32 keys only (80 KB). Both shapes of f32
// rows at 256 are short of registers by 14 and 16 a lane, some of which are
// read back from memory (60 and 68 bytes a lane) for every tile.
template <uint32_t ROWS, uint32_t WAVES, uint32_t KEYS, uint32_t BUFFERS, uint32_t BLOCKS>
struct ChunkShape {
    static constexpr uint32_t kRows = ROWS, kWaves = WAVES, kKeys = KEYS, kBuffers = BUFFERS, kBlocks = BLOCKS;
};
template <typename T, typename R, uint32_t D>
struct ChunkOf {
    using Shape = std::conditional_t<
        D == 64, ChunkShape<32, 4, 64, 1, 3>,
        std::conditional_t<D == 128, ChunkShape<32, 8, 64, 2, 1>, ChunkShape<16, 8, 64, 1, 1>>>;
};
template <typename T, uint32_t D>
struct ChunkOf<T, float, D> {
    using Shape = std::conditional_t<
        D == 256, ChunkShape<16, 8, 32, 1, 1>,
        std::conditional_t<D == 128 && std::is_same_v<T, float>, ChunkShape<16, 8, 64, 1, 1>, ChunkShape<16, 4, 64, 1, 2>>>;
};
template <typename T, typename R, uint32_t D>
constexpr uint32_t chunk_rows() {
    using Shape = typename ChunkOf<T, R, D>::Shape;
    return Shape::kRows * Shape::kWaves;
}

template <typename T, typename R, uint32_t D>
constexpr size_t chunk_lds() {
    using Shape = typename ChunkOf<T, R, D>::Shape;
    constexpr size_t pieces = std::is_same_v<T, float> ? 5 : 2;
    return pieces * Shape::kBuffers * Shape::kKeys * D * 2 + 16 + 4 * Shape::kKeys * 4 +
           Shape::kWaves * 64 * 4;
}

// Bound by matrix and vector phases that overlap in part: 8192 f16 tokens, 32
// heads of 64 on 4, 275 GFLOP, 374 us (0.73 PFLOP/s; a large library product
// reaches 1.29): the matrix cores are busy 36% of the cycles, the vector units
// (a third of it exponentials) 58%, at a clock that such work takes down to 1.8
// GHz. Ragged chunks of 5 sequences in bf16, 32 heads of 128 on 8, 145 us (35%
// and 46%); 512 f32 tokens behind 3584 over f32 heads of 256, 153 us and a join
// of 12 (three products of pieces for a score's, six for a value's: 44% and 42%).
// Tried without gain on earlier forms of the kernel: the waves' halves
// a phase apart over two buffers of keys and three of values (165 -> 185 us for
// the ragged chunks), the next tile's scores among a tile's exponentials over three
// buffers (165 -> 209, the prompt 424 -> 562), wave priorities for either phase
// (165 -> 170 and 175), weights kept apart from the products by scheduling
// barriers (171); 16-bit denominators as a row of ones on the matrix cores (165, now
// 161; the prompt 424 -> 415).
//
// Block (row tile, KV head, part, sequence). Lane l of a wave is row l % ROWS
// of the wave's and piece l / ROWS of its keys.
template <typename T, typename R, uint32_t D>
__global__ __launch_bounds__((ChunkOf<T, R, D>::Shape::kWaves * 64u), (ChunkOf<T, R, D>::Shape::kBlocks *
                                                                     ChunkOf<T, R, D>::Shape::kWaves / 4u))
void k_paged_chunk(AttendArgs args) {
    using Shape = typename ChunkOf<T, R, D>::Shape;
    constexpr bool kFloat = std::is_same_v<T, float>;
    using M = std::conditional_t<kFloat, __bf16, T>;  // the matrix cores' type
    constexpr uint32_t P = std::is_same_v<R, float> ? 3u : 1u;
    constexpr uint32_t Q = kFloat ? 3u : 1u;
    // f32 keys: two f16 pieces of each, scaled by a power of two a row and a key
    // (three products instead of six, and a query in two thirds of the registers)
    using N = std::conditional_t<kFloat, _Float16, M>;
    constexpr uint32_t QP = kFloat ? 2u : P, KP = kFloat ? 2u : 1u;
    constexpr uint32_t W = Shape::kRows, kKeys = Shape::kKeys, kBlock = Shape::kWaves * 64u, kBuffers = Shape::kBuffers;
    constexpr uint32_t kBlockRows = W * Shape::kWaves;
    constexpr uint32_t kSub = kKeys / 32u;             // 32 keys at a time through the products
    constexpr uint32_t kHeld = W == 32u ? 16u : 8u;    // a lane's keys of 32
    constexpr uint32_t kStepDims = W == 32u ? 16u : 32u;
    using Acc = std::conditional_t<W == 32u, f32x16, f32x4>;
    constexpr uint32_t kRegisters = W == 32u ? 16u : 4u;
    constexpr uint32_t kPlane = kKeys * D * 2u, kBuffer = (KP + Q) * kPlane;
    constexpr uint32_t kPieces = D / 8u;                              // of an entry's key or value
    constexpr uint32_t kLoads = (kKeys * kPieces + kBlock - 1u) / kBlock;  // a thread's pieces of a tile's keys
    extern __shared__ __align__(16) unsigned char lds[];
    // whether a tile had a value that is not finite; each buffer's last tile with
    // a bad page, and its entries
    // (plain LDS accesses, ordered by the barriers: volatile ones through a generic
    // pointer waited for every load in flight)
    uint32_t *const marks = reinterpret_cast<uint32_t *>(lds + kBuffers * kBuffer);
    uint32_t *const bad_key = marks + 4u;                             // [2][kKeys]
    // the power of two that takes the scores of a key back from its scale
    int32_t *const key_unscale = reinterpret_cast<int32_t *>(lds + kBuffers * kBuffer) + 4u + 2u * kKeys;  // [2][kKeys]
    uint32_t *const page_ids = reinterpret_cast<uint32_t *>(key_unscale + 2u * kKeys);
    const PagedView &cache = args.c;
    // the blocks of one (KV head, part) of a sequence read the same entries: where
    // there are 8 or more such pairs their number is rounded up to a multiple
    // of 8, so that each stays on one XCD (block b runs on XCD b % 8)
    const uint32_t pairs = cache.heads * args.parts;
    const uint32_t padded = pairs < 8u ? pairs : (pairs + 7u) & ~7u;
    const uint32_t which = blockIdx.x % padded;
    if (which >= pairs) {
        return;
    }
    const uint32_t kv = which % cache.heads, part = which / cache.heads;
    // the row tiles of all sequences in order, those of a sequence from its last
    // (the longest histories) on: this block's is found by a running sum over
    // 64 sequences at a time (a block for each tile that max_tokens allows
    // instead: 6144 of them for one chunk of 512 tokens beside 31 single ones,
    // of which 5766 only wait for a CU)
    uint32_t sequence = ~0u, tile = blockIdx.x / padded;
    for (uint32_t first = 0; first < cache.sequences; first += 64u) {
        const uint32_t own = first + (threadIdx.x & 63u);
        uint32_t tiles = 0;
        if (own < cache.sequences) {
            const uint32_t a = min(cache.offsets[own], cache.tokens), b = min(cache.offsets[own + 1u], cache.tokens);
            const uint32_t count = min(b > a ? b - a : 0u, cache.max_tokens);
            tiles = args.mixed != 0u && count * args.group <= kStepRows
                        ? 0u
                        : (count * args.group + kBlockRows - 1u) / kBlockRows;
        }
        uint32_t sum = tiles;
#pragma unroll
        for (uint32_t d = 1; d < 64u; d *= 2u) {
            const uint32_t below = __shfl_up(sum, d);
            sum += (threadIdx.x & 63u) >= d ? below : 0u;
        }
        const uint64_t past = __ballot(sum > tile);
        if (past != 0u) {
            const int lane = __ffsll(static_cast<unsigned long long>(past)) - 1;
            sequence = first + static_cast<uint32_t>(lane);
            tile = __shfl(sum, lane) - 1u - tile;
            break;
        }
        tile -= __shfl(sum, 63);
    }
    if (sequence == ~0u) {
        return;
    }
    sequence = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(sequence)));
    tile = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(tile)));
    const SequenceRows s = sequence_rows(cache, sequence);
    if (s.over || s.length == 0u) {
        if (part == 0u && tile == 0u) {
            fill_rows<R, D>(args, s, kv);
        }
        return;
    }
    const uint32_t rows = s.count * args.group;
    if (tile * kBlockRows >= rows) {
        return;
    }
    const uint32_t t = threadIdx.x, lane = t & 63u;
    const uint32_t wave = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(t >> 6)));
    const uint32_t column = lane % W, side = lane / W;
    const int32_t first_position = static_cast<int32_t>(s.length) - static_cast<int32_t>(s.count);
    const int32_t window = static_cast<int32_t>(args.window);
    const auto place = [&](uint32_t row) { return first_position + static_cast<int32_t>(row / args.group); };
    const auto from = [&](int32_t position) { return window == 0 ? 0 : max(0, position - window + 1); };
    const uint32_t block_last = min((tile + 1u) * kBlockRows, rows) - 1u;
    const int32_t block_low = place(tile * kBlockRows), block_high = place(block_last);
    const int32_t block_from = from(block_low), block_all = from(block_high);
    const uint32_t wave_row = tile * kBlockRows + wave * W;
    const bool wave_live = wave_row < rows;
    const int32_t wave_low = place(min(wave_row, rows - 1u)), wave_high = place(min(wave_row + W - 1u, rows - 1u));
    const uint32_t row = min(wave_row + column, rows - 1u);
    const uint32_t token = s.first + row / args.group, head = kv * args.group + row % args.group;
    const int32_t position = place(row), oldest = from(position);
    // entries of the part that some row of the block sees
    const int32_t base = base_of(args, first_position);
    int32_t begin = base + static_cast<int32_t>(part * args.span);
    const int32_t end = min(begin + static_cast<int32_t>(args.span), block_high + 1);
    begin = max(begin, block_from & ~static_cast<int32_t>(kKeys - 1u));
    if (begin >= end && (part != 0u || block_high >= 0)) {
        return;
    }
    const uint32_t *const table = cache.table + static_cast<uint64_t>(sequence) * cache.table_stride;
    const T *const keys = reinterpret_cast<const T *>(cache.keys) + kv * cache.head_stride;
    const T *const values = reinterpret_cast<const T *>(cache.values) + kv * cache.head_stride;
    const R *const query = reinterpret_cast<const R *>(args.queries.data) + token * args.queries.token_stride +
                           head * args.queries.head_stride;
    if (t < 4u) {
        marks[t] = ~0u;
    }

    // the numbers of kBlock pages at a time
    uint32_t first_page = 0;
    const auto fill_pages = [&](int32_t entry) {
        first_page = static_cast<uint32_t>(entry) >> cache.page_shift;
        const uint32_t id = first_page + t;
        uint32_t page = ~0u;
        if (id <= static_cast<uint32_t>(end - 1) >> cache.page_shift) {
            page = table[id];
        }
        page_ids[t] = page < cache.pages ? page : ~0u;
    };

    // A tile's keys and its values pass through registers: pieces t + kBlock i of
    // either, piece p of entry p / kPieces.
    using Piece = std::conditional_t<kFloat, f32x4, u32x4>;
    constexpr uint32_t kWide = kFloat ? 2u : 1u;
    struct Held {
        Piece piece[kLoads][kWide];
        uint32_t bad;
    };
    const auto entry_of = [&](uint32_t i) { return (t + kBlock * i) / kPieces; };
    // (with few pieces some threads have none)
    const bool loads = kKeys * kPieces >= kBlock || t < kKeys * kPieces;
    const uint32_t page_mask = (1u << cache.page_shift) - 1u;
    // Where a page holds whole tiles (its size and the tiles' are powers of
    // two), a tile's page is one number and a thread's places in it are fixed.
    const bool paged_tiles = page_mask >= kKeys - 1u;
    uint64_t fixed[kLoads];
#pragma unroll
    for (uint32_t i = 0; i < kLoads; ++i) {
        fixed[i] = loads ? t % kPieces * 8u + entry_of(i) * cache.entry_stride : 0u;
    }
    const auto load = [&](Held &held, const T *from_pool, int32_t first) {
        held.bad = 0;
        const auto take = [&](uint32_t i, uint64_t at) {
            const Piece *const piece = reinterpret_cast<const Piece *>(from_pool + at);
#pragma unroll
            for (uint32_t w = 0; w < kWide; ++w) {
                held.piece[i][w] = piece[w];
            }
        };
        if (paged_tiles) {
            const uint32_t id = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(
                static_cast<int>(page_ids[(static_cast<uint32_t>(first) >> cache.page_shift) - first_page])));
            held.bad = id == ~0u ? (1u << kLoads) - 1u : 0u;
            const uint64_t tile_at = (id == ~0u ? 0u : id) * cache.page_stride + (first & page_mask) * cache.entry_stride;
#pragma unroll
            for (uint32_t i = 0; i < kLoads; ++i) {
                take(i, tile_at + fixed[i]);
            }
            return;
        }
#pragma unroll
        for (uint32_t i = 0; i < kLoads; ++i) {
            const int32_t entry = first + static_cast<int32_t>(entry_of(i));
            uint64_t at = t % kPieces * 8u;
            if (entry < end && loads) {
                const uint32_t page = page_ids[(static_cast<uint32_t>(entry) >> cache.page_shift) - first_page];
                held.bad |= page == ~0u ? 1u << i : 0u;
                at += (page == ~0u ? 0u : page) * cache.page_stride + (entry & page_mask) * cache.entry_stride;
            }
            take(i, at);
        }
    };
    const auto edge_tile = [&](int32_t first) {
        return first + static_cast<int32_t>(kKeys) > block_low + 1 || first < block_all;
    };
    // `turn` is the tile's of two that marks of bad pages are kept for
    const auto stage_keys = [&](Held &held, int32_t first, uint32_t buffer, uint32_t turn) {
        unsigned char *const to = lds + buffer * kBuffer;
        if ((edge_tile(first) || held.bad != 0u) && loads) {
#pragma unroll
            for (uint32_t i = 0; i < kLoads; ++i) {
                const bool bad = (held.bad >> i & 1u) != 0u;
                if (bad) {
                    marks[1u + turn] = static_cast<uint32_t>(first);
                }
                if (t % kPieces == 0u) {
                    bad_key[turn * kKeys + entry_of(i)] = bad ? static_cast<uint32_t>(first) : ~0u;
                }
            }
        }
#pragma unroll
        for (uint32_t i = 0; i < kLoads; ++i) {
            const uint32_t entry = entry_of(i), piece = t % kPieces;
            const uint32_t at = key_place<D, W>(entry, piece);
            if constexpr (kFloat) {
                uint32_t largest = 0;
#pragma unroll
                for (uint32_t w = 0; w < kWide; ++w) {
#pragma unroll
                    for (uint32_t k = 0; k < 4u; ++k) {
                        largest = magnitude(largest, held.piece[i][w][k]);
                    }
                }
                largest = max(largest, lane_xor_bits<1>(largest));
                largest = max(largest, lane_xor_bits<2>(largest));
                largest = max(largest, lane_xor_bits<4>(largest));
                if constexpr (kPieces > 8u) {
                    largest = max(largest, lane_xor_bits<8>(largest));
                }
                if constexpr (kPieces > 16u) {
                    largest = max(largest, lane_xor_bits<16>(largest));
                }
                const uint32_t exponent = scale_exponent(largest);
                const float scale = scale_of(exponent);
                if (piece == 0u && loads) {
                    key_unscale[buffer * kKeys + entry] = unscale_of(exponent);
                }
                u32x4 out[KP];
#pragma unroll
                for (uint32_t n = 0; n < 4u; ++n) {
                    uint32_t pieces[KP];
                    split<N>(held.piece[i][n / 2u][2u * n % 4u] * scale, held.piece[i][n / 2u][2u * n % 4u + 1u] * scale,
                             pieces);
#pragma unroll
                    for (uint32_t p = 0; p < KP; ++p) {
                        out[p][n] = pieces[p];
                    }
                }
                if (loads) {
#pragma unroll
                    for (uint32_t p = 0; p < KP; ++p) {
                        *reinterpret_cast<u32x4 *>(to + p * kPlane + at) = out[p];
                    }
                }
            } else if (loads) {
                *reinterpret_cast<u32x4 *>(to + at) = held.piece[i][0];
            }
        }
    };
    const auto stage_values = [&](Held &held, int32_t first, uint32_t buffer) {
        unsigned char *const to = lds + buffer * kBuffer + KP * kPlane;
        if (edge_tile(first) || held.bad != 0u) {
#pragma unroll
            for (uint32_t i = 0; i < kLoads; ++i) {
                const int32_t entry = first + static_cast<int32_t>(entry_of(i));
                // (what no row sees is whatever the page held before)
                const bool any = entry < end && entry >= block_from && (held.bad >> i & 1u) == 0u;
                bool seen = false;
#pragma unroll
                for (uint32_t w = 0; w < kWide; ++w) {
#pragma unroll
                    for (uint32_t k = 0; k < 4u; ++k) {
                        held.piece[i][w][k] = any ? held.piece[i][w][k] : 0;
                        if constexpr (kFloat) {
                            seen |= odd_float(held.piece[i][w][k]);
                            held.piece[i][w][k] = odd_float(held.piece[i][w][k]) ? 0.0f : held.piece[i][w][k];
                        } else {
                            seen |= odd_pair<T>(held.piece[i][w][k]);
                            held.piece[i][w][k] = clean_pair<T>(held.piece[i][w][k]);
                        }
                    }
                }
                if (seen && loads) {
                    marks[0] = 1u;
                }
            }
        }
        if (!loads) {
            return;
        }
#pragma unroll
        for (uint32_t i = 0; i < kLoads; ++i) {
            const uint32_t at = value_place<D, W>(entry_of(i), t % kPieces);
            if constexpr (kFloat) {
                u32x4 out[Q];
#pragma unroll
                for (uint32_t n = 0; n < 4u; ++n) {
                    uint32_t pieces[Q];
                    split<M>(held.piece[i][n / 2u][2u * n % 4u], held.piece[i][n / 2u][2u * n % 4u + 1u], pieces);
#pragma unroll
                    for (uint32_t p = 0; p < Q; ++p) {
                        out[p][n] = pieces[p];
                    }
                }
#pragma unroll
                for (uint32_t p = 0; p < Q; ++p) {
                    *reinterpret_cast<u32x4 *>(to + p * kPlane + at) = out[p];
                }
            } else {
                *reinterpret_cast<u32x4 *>(to + at) = held.piece[i][0];
            }
        }
    };

    // the row's query: step j holds dimensions kStepDims j + 8 side + 0 .. 7
    u32x4 query_pieces[D / kStepDims][QP];
    float query_scale = 1.0f;
    int32_t query_unscale = 0;
    if constexpr (kFloat) {
        uint32_t largest = 0;
#pragma unroll
        for (uint32_t j = 0; j < D / kStepDims; ++j) {
#pragma unroll
            for (uint32_t k = 0; k < 8u; ++k) {
                largest = magnitude(largest, query[kStepDims * j + 8u * side + k]);
            }
        }
        static_assert(!kFloat || W == 16u);
        largest = max(largest, lane_xor_bits<16>(largest));
        largest = max(largest, lane_xor_bits<32>(largest));
        query_scale = scale_of(scale_exponent(largest));
        query_unscale = unscale_of(scale_exponent(largest));
    }
#pragma unroll
    for (uint32_t j = 0; j < D / kStepDims; ++j) {
        const R *const at = query + kStepDims * j + 8u * side;
        if constexpr (P == 1) {
            query_pieces[j][0] = *reinterpret_cast<const u32x4 *>(at);
        } else {
            const f32x4 lo = *reinterpret_cast<const f32x4 *>(at) * query_scale;
            const f32x4 hi = *reinterpret_cast<const f32x4 *>(at + 4u) * query_scale;
#pragma unroll
            for (uint32_t k = 0; k < 4u; ++k) {
                uint32_t pieces[QP];
                k < 2u ? split<N>(lo[2u * k], lo[2u * k + 1u], pieces)
                       : split<N>(hi[2u * k - 4u], hi[2u * k - 3u], pieces);
#pragma unroll
                for (uint32_t p = 0; p < QP; ++p) {
                    query_pieces[j][p][k] = pieces[p];
                }
            }
        }
    }

    Acc sums[D / W];
#pragma unroll
    for (uint32_t m = 0; m < D / W; ++m) {
#pragma unroll
        for (uint32_t r = 0; r < kRegisters; ++r) {
            sums[m][r] = 0.0f;
        }
    }
    // the level of the row's weights (kNegative before its first score), and the
    // score from which it is raised
    float maximum = kNegative, limit = kNegative, denominator = 0.0f;
    bool far = false;  // some row's level is
    // a lane's keys of 32, and register r of sums[m]
    const auto key_of = [&](uint32_t r) {
        return W == 32u ? 8u * (r / 4u) + 4u * side + r % 4u : 8u * side + r;
    };
    const auto dimension_of = [&](uint32_t m, uint32_t r) {
        return W == 32u ? 32u * m + 8u * (r / 4u) + 4u * side + r % 4u : 16u * m + 4u * side + r;
    };

    // (a wave whose rows see nothing of a tile passes it by)
    const auto sees = [&](int32_t first) {
        return wave_live && first <= wave_high && first + static_cast<int32_t>(kKeys) > from(wave_low);
    };
    const auto scores = [&](uint32_t buffer, float (&score)[kSub][kHeld]) {
        const unsigned char *const key_lds = lds + buffer * kBuffer;
        // with 16 rows a wave two products of 16 keys for every 32, interleaved so that
        // a lane's eight results are eight keys in a row; a tile's turn by turn, as
        // a product that adds to the one before it waits for it
        constexpr uint32_t kHalves = W == 32u ? 1u : 2u, kProducts = kHalves * kSub;
        Acc acc[kProducts], *to[kProducts];
#pragma unroll
        for (uint32_t h = 0; h < kProducts; ++h) {
#pragma unroll
            for (uint32_t r = 0; r < kRegisters; ++r) {
                acc[h][r] = 0.0f;
            }
            to[h] = &acc[h];
        }
        u32x4 k[2][kProducts][KP];
        const auto read = [&](uint32_t j) {
#pragma unroll
            for (uint32_t h = 0; h < kProducts; ++h) {
                const uint32_t entry = 32u * (h / kHalves) +
                                       (W == 32u ? column : 8u * (column / 4u) + 4u * (h % 2u) + column % 4u);
#pragma unroll
                for (uint32_t p = 0; p < KP; ++p) {
                    k[j & 1u][h][p] = *reinterpret_cast<const u32x4 *>(
                        key_lds + p * kPlane + key_place<D, W>(entry, kStepDims / 8u * j + side));
                }
            }
        };
        read(0u);
#pragma unroll
        for (uint32_t j = 0; j < D / kStepDims; ++j) {
            if (j + 1u < D / kStepDims) {
                read(j + 1u);
            }
            products<N>(k[j & 1u], query_pieces[j], to);
            if constexpr (P == 3u) {
                __builtin_amdgcn_sched_barrier(0);
            }
        }
#pragma unroll
        for (uint32_t h = 0; h < kProducts; ++h) {
            const uint32_t sub = h / kHalves, at = h % kHalves * kRegisters;
#pragma unroll
            for (uint32_t r = 0; r < kRegisters; ++r) {
                score[sub][at + r] = acc[h][r];
                if constexpr (kFloat) {
                    score[sub][at + r] =
                        ldexpf(acc[h][r], query_unscale + key_unscale[buffer * kKeys + 32u * sub + key_of(at + r)]);
                }
            }
        }
    };
    const auto attend = [&](int32_t first, uint32_t buffer, uint32_t turn, float (&score)[kSub][kHeld]) {
        const unsigned char *const value_lds = lds + buffer * kBuffer + KP * kPlane;
        const bool bad_tile = marks[1u + turn] == static_cast<uint32_t>(first);
        if (bad_tile || first + static_cast<int32_t>(kKeys) > wave_low + 1 || first < from(wave_high)) {
#pragma unroll
            for (uint32_t b = 0; b < kSub; ++b) {
#pragma unroll
                for (uint32_t r = 0; r < kHeld; ++r) {
                    const uint32_t key = 32u * b + key_of(r);
                    const int32_t entry = first + static_cast<int32_t>(key);
                    const bool visible = entry <= position && entry >= oldest;
                    const bool bad = bad_tile && bad_key[turn * kKeys + key] == static_cast<uint32_t>(first);
                    score[b][r] = !visible ? kNegative : bad ? __builtin_nanf("") : score[b][r];
                }
            }
        }
        float top = score[0][0];
#pragma unroll
        for (uint32_t b = 0; b < kSub; ++b) {
#pragma unroll
            for (uint32_t r = 0; r < kHeld; ++r) {
                top = fmaxf(top, score[b][r]);
            }
        }
        if constexpr (W == 16u) {
            top = fmaxf(top, lane_xor<16>(top));
        }
        top = fmaxf(top, lane_xor<32>(top));
        if (__any(top > limit)) {
            // (a row's level does not depend on the wave's other rows)
            const bool raised = top > limit;
            const float factor = raised ? raise_of<R>(args, maximum, top) : 1.0f;
            maximum = raised ? top : maximum;
            limit = raised ? top + (far_level(args, top) ? 0.0f : args.slack) : limit;
            far = __any(maximum != kNegative && far_level(args, maximum)) != 0;
            denominator *= factor;
#pragma unroll
            for (uint32_t m = 0; m < D / W; ++m) {
                sums[m] *= factor;
            }
        }
        Level level = near_level_of<R>(args, maximum);
        if (P == 1u && far) {
            level = level_of<R>(args, maximum);
#pragma unroll
            for (uint32_t b = 0; b < kSub; ++b) {
#pragma unroll
                for (uint32_t r = 0; r < kHeld; ++r) {
                    score[b][r] -= level.minus;
                }
            }
        }
#pragma unroll
        for (uint32_t b = 0; b < kSub; ++b) {
#pragma unroll
            for (uint32_t r = 0; r < kHeld; ++r) {
                score[b][r] = weight_of<R>(args, P == 3u ? score[b][r] - level.minus : score[b][r], level);
                if constexpr (P == 3u) {
                    denominator += score[b][r];
                }
            }
            // steps of 16 keys (32 rows a wave) or 32
#pragma unroll
            for (uint32_t u = 0; u < kHeld / 8u; ++u) {
                u32x4 weights[P];
#pragma unroll
                for (uint32_t k = 0; k < 4u; ++k) {
                    uint32_t pieces[P];
                    split<M>(score[b][8u * u + 2u * k], score[b][8u * u + 2u * k + 1u], pieces);
#pragma unroll
                    for (uint32_t p = 0; p < P; ++p) {
                        weights[p][k] = pieces[p];
                    }
                }
                if constexpr (P == 1u) {
#pragma unroll
                    for (uint32_t k = 0; k < 4u; ++k) {
                        denominator = pair_sum<M>(weights[0][k], denominator);
                    }
                }
                // the values transposed: lane i of 16 takes row i / 4 of four
                // entries at dimension 4 (i % 4), and gets dimension i of the four
                const uint32_t entry = 32u * b + (lane & 15u) / 4u + (W == 32u ? 16u * u + 4u * side : 8u * side);
                const uint32_t next = entry + (W == 32u ? 8u : 4u);
                const uint32_t dimension = (W == 32u ? (lane >> 4 & 1u) * 16u : 0u) + (lane & 3u) * 4u;
                // (two at a time, the next two on their way)
                u32x4 v[2][2][Q];
                const auto read = [&](uint32_t i) {
#pragma unroll
                    for (uint32_t x = 0; x < 2u; ++x) {
#pragma unroll
                        for (uint32_t p = 0; p < Q; ++p) {
                            const uint32_t d = W * (2u * i + x) + dimension;
                            const auto four = [&](uint32_t e) {
                                auto *at = (__attribute__((address_space(3))) s16x4 *)(
                                    value_lds + p * kPlane + value_place<D, W>(e, d / 8u) + d % 8u * 2u);
                                return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(at));
                            };
                            const u32x2 lo = four(entry), hi = four(next);
                            v[i & 1u][x][p] = u32x4{lo.x, lo.y, hi.x, hi.y};
                        }
                    }
                };
                read(0u);
#pragma unroll
                for (uint32_t i = 0; i < D / W / 2u; ++i) {
                    if (i + 1u < D / W / 2u) {
                        read(i + 1u);
                    }
                    Acc *to[2] = {&sums[2u * i], &sums[2u * i + 1u]};
                    products<M>(v[i & 1u], weights, to);
                    if constexpr (P == 3u) {
                        __builtin_amdgcn_sched_barrier(0);
                    }
                }
            }
        }
    };

    const int32_t step = static_cast<int32_t>(kKeys);
    // pages up to a tile's end in LDS (called by all, between barriers)
    const auto reach_pages = [&](int32_t first) {
        if ((static_cast<uint32_t>(first + step - 1) >> cache.page_shift) - first_page >= kBlock) {
            fill_pages(first);
            __syncthreads();
        }
    };
    if (begin < end) {
        fill_pages(begin);
        __syncthreads();
        int32_t first = begin;
        uint32_t turn = 0;
        float score[kSub][kHeld];
        if constexpr (kBuffers == 2u) {
            // two tiles in LDS: while one is computed the next is staged, from
            // registers whose loads went out a tile before
            Held key_in, value_in;
            load(key_in, keys, begin);
            load(value_in, values, begin);
            stage_keys(key_in, begin, 0u, 0u);
            stage_values(value_in, begin, 0u);
            // (the queries are here before the loop: a wait for them within it
            // would be one for the tiles on their way)
            __builtin_amdgcn_s_waitcnt(0);
            if (begin + step < end) {
                load(key_in, keys, begin + step);
                load(value_in, values, begin + step);
            }
            do {
                const int32_t ahead = first + 2 * step;
                __syncthreads();  // the other buffer's readers are done
                if (ahead < end) {
                    reach_pages(ahead);
                }
                if (first + step < end) {
                    stage_keys(key_in, first + step, turn ^ 1u, turn ^ 1u);
                    stage_values(value_in, first + step, turn ^ 1u);
                }
                if (ahead < end) {
                    load(key_in, keys, ahead);
                    load(value_in, values, ahead);
                }
                if (sees(first)) {
                    scores(turn, score);
                    attend(first, turn, turn, score);
                }
                turn ^= 1u;
                first += step;
            } while (first < end);
        } else {
            // one: while its keys are multiplied its values are staged, and the
            // next one's keys while its values are; one set of registers holds what
            // is on its way. The waves' second half stages first and the first
            // half last: a SIMD has a wave of either, of which one then uses the
            // vector units while the other's products run.
            const bool early = wave >= Shape::kWaves / 2u;
            Held in;
            load(in, keys, begin);
            stage_keys(in, begin, 0u, 0u);
            __builtin_amdgcn_s_waitcnt(0);
            load(in, values, begin);
            do {
                const bool live = sees(first), more = first + step < end;
                const auto pass_values = [&] {
                    stage_values(in, first, 0u);
                    if (more) {
                        load(in, keys, first + step);
                    }
                };
                const auto pass_keys = [&] {
                    if (more) {
                        stage_keys(in, first + step, 0u, turn ^ 1u);
                        load(in, values, first + step);
                    }
                };
                __syncthreads();
                if (early) {
                    pass_values();
                }
                if (live) {
                    scores(0u, score);
                }
                if (!early) {
                    pass_values();
                }
                __syncthreads();
                if (early) {
                    pass_keys();
                }
                if (live) {
                    attend(first, 0u, turn, score);
                }
                if (!early) {
                    pass_keys();
                }
                turn ^= 1u;
                if (more) {
                    if (first + 2 * step < end &&
                        (static_cast<uint32_t>(first + 3 * step - 1) >> cache.page_shift) - first_page >= kBlock) {
                        __syncthreads();  // every wave has read its pages
                        fill_pages(first + 2 * step);
                    }
                }
                first += step;
            } while (first < end);
        }
    }

    if (marks[0] != ~0u) {
        // Values that are not finite, in tiles of which some rows see only a part:
        // the products left them out, the rows that see them get them.
        for (int32_t first = begin; first < end; first += step) {
            for (int32_t entry = first; edge_tile(first) && entry < min(first + step, end); ++entry) {
                const float weight = odd_weight<T, R, D>(args, table, keys, query, entry, maximum);
                const bool visible = entry <= position && entry >= oldest;
                const Page page = page_of(cache, table, entry);
                const T *const value = values + page.at;
#pragma unroll
                for (uint32_t m = 0; m < D / W; ++m) {
#pragma unroll
                    for (uint32_t r = 0; r < kRegisters; ++r) {
                        const float v = static_cast<float>(value[dimension_of(m, r)]);
                        sums[m][r] += visible && !page.bad && odd_float(v) ? v * weight : 0.0f;
                    }
                }
            }
        }
    }

    if constexpr (W == 16u) {
        denominator += lane_xor<16>(denominator);
    }
    denominator += lane_xor<32>(denominator);
    if (!wave_live || wave_row + column >= rows) {
        return;
    }
    // a row whose entries are all in this part is done
    const bool none = position < 0;
    const bool whole = none || (oldest >= base + static_cast<int32_t>(part * args.span) &&
                                position < base + static_cast<int32_t>((part + 1u) * args.span));
    if (none ? part != 0u : position < begin || oldest >= end) {
        return;  // the part holds nothing the row sees
    }
    float *const to = whole ? nullptr : partial_row<D>(args, part, token, head);
    const float scale = none ? 0.0f : whole ? 1.0f / denominator : settle_of<R>(args, maximum);
#pragma unroll
    for (uint32_t m = 0; m < D / W; ++m) {
#pragma unroll
        for (uint32_t q = 0; q < kRegisters / 4u; ++q) {
            const uint32_t at = dimension_of(m, 4u * q);
            const f32x4 v = {sums[m][4u * q], sums[m][4u * q + 1u], sums[m][4u * q + 2u], sums[m][4u * q + 3u]};
            if (whole) {
                float out[4];
#pragma unroll
                for (uint32_t k = 0; k < 4u; ++k) {
                    out[k] = none ? 0.0f : v[k] * scale;
                }
                store_output<R, 4>(args, token, head, at, out, none);
            } else {
                *reinterpret_cast<f32x4 *>(to + at) = P == 3u ? v : v * scale;
            }
        }
    }
    if (!whole && side == 0u) {
        to[D] = maximum;
        to[D + 1u] = P == 3u ? denominator : denominator * scale;
    }
}

// ---- host ---------------------------------------------------------------------

template <typename T, typename R, uint32_t D>
void launch_attention(adi_hip_context *ctx, AttendArgs args, const adi_hip_paged_workspace *workspace) {
    const PagedView &c = args.c;
    const uint64_t heads = uint64_t(c.heads) * args.group;
    // entries a sequence's parts may cover, their base rounded down with a window
    uint64_t extent = std::max(c.max_length, 1u);
    if (args.window != 0) {
        extent = std::min<uint64_t>(extent, uint64_t(args.window) + c.max_tokens + kSpanUnit);
    }
    const auto span_of = [&](uint64_t parts, uint64_t unit) {
        return static_cast<uint32_t>((ceil_div(extent, parts) + unit - 1) / unit * unit);
    };
    const size_t room = workspace->bytes - kTickets * sizeof(uint32_t);
    float *const partial = reinterpret_cast<float *>(static_cast<char *>(workspace->base) + kTickets * sizeof(uint32_t));
    using Shape = typename ChunkOf<T, R, D>::Shape;
    constexpr uint32_t kBlockRows = chunk_rows<T, R, D>();
    // A chunk's parts, those that end first, by us: 32 keys of a row tile about
    // kTurn, rounds of the blocks the chip holds (half a round more where there
    // are several, for their uneven ends), a block's own start and end as 6 turns;
    // the parts' way through memory at 5 TB/s, and a join's launch and loop. Within
    // 3% of the best number of parts for six chunks of 64 to 512 tokens behind 4000
    // and 8000 entries (64 tokens, 16 heads of 128 on 2 in bf16: 16 parts 30.2 us,
    // 8 32.8, 32 35.2).
    constexpr double kTurn = D / 64.0 * (std::is_same_v<R, float> ? 0.8 : 0.5);
    struct Parts {
        uint32_t span;
        double cost;
    };
    const uint64_t part_bytes = uint64_t(c.tokens) * heads * (D + 4u) * sizeof(float);
    const auto parts_of = [&](uint64_t row_tiles) {
        const uint64_t most = std::clamp<uint64_t>(room / part_bytes, 1u, 64u);
        const double resident = double(ctx->cu_count) * Shape::kBlocks;
        Parts best{0, 0.0};
        for (uint64_t parts = 1; parts <= most; ++parts) {
            const uint64_t span = span_of(parts, kSpanUnit), real = ceil_div(extent, span);
            const double count = double(row_tiles * c.heads * real);
            const double rounds = count <= resident ? 1.0 : count / resident + 0.5;
            const double cost = rounds * (span / 32.0 + 6.0) * kTurn +
                                (real > 1 ? 4.0 + 0.3 * real + 2.0 * part_bytes * real / 5.0e6 : 0.0);
            if (parts == 1 || cost < best.cost) {
                best = {static_cast<uint32_t>(span), cost};
            }
        }
        return best;
    };
    // Few rows of every sequence: k_paged_step. Many of every one (as many as
    // there may be): k_paged_chunk. Else both, each for its sequences: in the
    // chunk kernel a single token costs its block a tile's whole staging (31 of
    // them beside 512 tokens: 62 us of 175). But where the single tokens' blocks have
    // room beside the chunks' (4 us by the parts' estimate) it takes them too, as
    // the other's launch, start and end are 8 us: 80 tokens beside two single ones, an
    // f32 head of 256, 32.0 us, so 23.6; 200 beside 7 behind 500 entries, 32 bf16
    // heads on 8 of 128, 34.7 and 27.5; 256 beside 7 behind 2000, 16 f32 heads on 2
    // of 256 in bf16, 75.5 as two, 98.9 as one.
    const bool few = uint64_t(c.max_tokens) * args.group <= kStepRows;
    const bool many = uint64_t(c.sequences) * c.max_tokens == c.tokens || c.sequences == 1;
    // row tiles at most, about how many, and with the single tokens'
    const uint64_t row_tiles =
        std::min<uint64_t>(ceil_div(uint64_t(c.max_tokens) * args.group, kBlockRows) * uint64_t(c.sequences),
                           uint64_t(c.tokens) * args.group / kBlockRows + c.sequences);
    const uint64_t full = ceil_div(uint64_t(c.tokens) * args.group, kBlockRows);
    Parts chunk{};
    if (!few) {
        chunk = parts_of(std::min(row_tiles, full + (many ? c.sequences / 2u : 0u)));
        if (!many) {
            const Parts all = parts_of(std::min<uint64_t>(row_tiles, full + c.sequences - 1u));
            args.mixed = all.cost > chunk.cost + 4.0 ? 1u : 0u;
            chunk = args.mixed != 0 ? chunk : all;
        }
        args.span = chunk.span;
        args.parts = ceil_div(extent, args.span);
        require((uint64_t(c.heads) * args.parts + 7u) / 8u * 8u * row_tiles < (1u << 23), "paged attention: too many rows");
    }
    if (few || args.mixed != 0) {
        AttendArgs a = args;
        a.partial = partial;
        a.tickets = static_cast<uint32_t *>(workspace->base);
        const uint64_t blocks = uint64_t(c.sequences) * c.heads;
        const uint64_t region = uint64_t(kStepRows) * (D + 4u) * sizeof(float);
        // (one tile a wave at least)
        constexpr uint64_t kUnit = std::is_same_v<T, float> ? 64 : 128;
        // A part's tiles, and the parts that the last block joins, both go through
        // one CU at about its rate, so a part takes at least the entries for which
        // the two are even (a token of 16 heads on 2 behind 8000 entries: f32 of
        // 256, spans of 64, 192 and 256 entries 37.0, 27.5 and 27.8 us; bf16 of 256
        // under f32 rows, 128, 256 and 384 24.2, 19.9 and 22.2; bf16 of 128 15.0,
        // 12.5 and 13.7).
        const uint64_t rows = std::min<uint64_t>(uint64_t(c.max_tokens) * args.group, kStepRows);
        const double even = std::sqrt(double(extent) * rows * (D + 4u) * sizeof(float) / (2.0 * D * sizeof(T)));
        const uint32_t least = std::max(span_of(kStepParts, kUnit), static_cast<uint32_t>(uint64_t(even / kUnit + 0.5) * kUnit));
        const uint64_t resident = uint64_t(step_blocks<T, R, D>()) * ctx->cu_count;
        const uint64_t slots = std::min({resident / c.heads, room / (c.heads * region),
                                         uint64_t(c.sequences) * ceil_div(extent, least)});
        if (c.sequences > 1 && c.sequences <= 64 && slots > c.sequences && blocks <= kTickets) {
            // As many blocks as the chip holds, shared by the lengths on the device.
            // As many parts a sequence as if all were of max_length leave a
            // third of the chip idle with lengths that are even up to it: 32
            // sequences up to 4,096 of 16 f32 heads on 2 of 256 in bf16 43.1
            // us, so 34.8; up to 8,000 of 32 heads on 8 of 128 146 and 130; 8
            // sequences up to 4,000 of 2 f32 heads of 256 28.5 and 29.5.
            a.span = least;
            a.slots = static_cast<uint32_t>(slots);
            launch(ctx, "paged_step", k_paged_step<T, R, D>, dim3(a.slots * c.heads), dim3(kThreads), 0, a);
        } else {
            uint64_t parts = 1;
            if (blocks <= kTickets) {
                parts = std::clamp<uint64_t>(std::min(resident / blocks, room / (blocks * region)), 1u, kStepParts);
            }
            a.span = std::max(span_of(parts, kUnit), parts > 1 ? least : 0u);
            a.parts = ceil_div(extent, a.span);
            launch(ctx, "paged_step", k_paged_step<T, R, D>, dim3(a.parts * c.heads, c.sequences), dim3(kThreads), 0, a);
        }
        if (few) {
            return;
        }
    }
    args.partial = partial;
    constexpr size_t lds = chunk_lds<T, R, D>();
    // (once a device)
    static std::atomic<uint64_t> raised{0};
    const uint64_t device = uint64_t(1) << (static_cast<uint32_t>(ctx->device) & 63u);
    if ((raised.load() & device) == 0) {
        set_lds_limit(reinterpret_cast<const void *>(k_paged_chunk<T, R, D>), lds);
        raised.fetch_or(device);
    }
    const uint64_t pairs = uint64_t(c.heads) * args.parts;
    const uint64_t grid = (pairs < 8u ? pairs : (pairs + 7u) / 8u * 8u) * row_tiles;
    launch(ctx, "paged_chunk", k_paged_chunk<T, R, D>, dim3(static_cast<uint32_t>(grid)), dim3(Shape::kWaves * 64u),
           lds, args);
    if (args.parts > 1) {
        const uint64_t rows = uint64_t(c.tokens) * heads;
        launch(ctx, "paged_join", k_paged_join<R, D>,
               dim3(static_cast<uint32_t>(std::min<uint64_t>((rows + 3) / 4, 1u << 20))), dim3(kThreads), 0, args);
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

void require_attention(const adi_hip_context *ctx, const adi_hip_paged_cache *cache, const adi_hip_paged_batch *batch,
                       uint32_t query_heads, const adi_hip_paged_workspace *workspace) {
    require_paged(cache, batch);
    require(workspace != nullptr, "paged attention: null argument");
    require(workspace->device == ctx->device, "paged attention: the workspace is on another device");
    require(query_heads >= 1 && query_heads % cache->heads == 0 && query_heads / cache->heads <= 256,
            "paged attention: query heads must be 1 to 256 times the cache's");
    require(cache->heads < (1u << 16) && batch->sequences < (1u << 16),
            "paged attention: more than 65535 heads or sequences");
}

void paged_attention(adi_hip_context *ctx, const adi_hip_paged_cache *cache, const adi_hip_paged_batch *batch,
                     const adi_hip_paged_attention_arguments *a, adi_hip_paged_workspace *workspace) {
    require(a != nullptr, "paged attention: null argument");
    require_attention(ctx, cache, batch, a->query_heads, workspace);
    const uint32_t type = a->queries.type;
    require(known_type(type) && (type == cache->type || (type == ADI_HIP_F32 && cache->type == ADI_HIP_BF16)),
            "paged attention: f32 rows read an f32 or bf16 cache, others their own type");
    require(a->scale >= 0.0f && a->scale <= 1e38f, "paged attention: scale must be positive and at most 1e38, or 0");
    if (batch->tokens == 0 || batch->sequences == 0) {
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
    const double log2_scale = scale * 1.4426950408889634;
    const auto in_scores = [&](float powers) { return static_cast<float>(std::min(powers / log2_scale, 3e38)); };
    const AttendArgs args{paged_view(*cache, *batch), rows_view(a->queries), rows_view(a->outputs), rows_view(a->gate),
                          static_cast<float>(log2_scale), in_scores(kSlack), in_scores(kFar), window,
                          a->query_heads / cache->heads, 0, 0, 0, 0, nullptr, nullptr};
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
