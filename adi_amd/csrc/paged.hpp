// paged.hpp -- rotary positions and the paged cache: what the calls check on
// the host, and the views their kernels share.
#pragma once

#include "context.hpp"

#include <algorithm>

// The frequencies of an adi_hip_rope_options, in turns a position (2 pi
// radians), so that an angle's whole turns drop out by one rounding.
struct adi_hip_rope {
    int device;
    uint32_t rotary;
    uint32_t layout;
    float magnitude;
    double *turns;  // device [rotary / 2]
};

namespace adi_hip {

inline uint32_t type_bytes(uint32_t type) { return type == ADI_HIP_F32 ? 4u : 2u; }
inline bool known_type(uint32_t type) { return type <= ADI_HIP_BF16; }

// The rows of one array, as kernels read them.
struct RowsView {
    char *data;
    uint64_t token_stride, head_stride;  // elements
};
inline RowsView rows_view(const adi_hip_rows &rows) {
    return {static_cast<char *>(rows.data), rows.token_stride, rows.head_stride};
}
inline bool same_rows(const adi_hip_rows &a, const adi_hip_rows &b) {
    return a.data == b.data && a.token_stride == b.token_stride && a.head_stride == b.head_stride;
}

// Rows a kernel moves 16 bytes at a time.
inline void require_rows(const adi_hip_rows &rows, uint32_t type, const char *message) {
    const uint64_t step = 16u / type_bytes(type);
    require(rows.type == type && rows.data != nullptr && aligned_to(rows.data, 16) &&
                rows.token_stride % step == 0 && rows.head_stride % step == 0,
            message);
}

struct PagedView {
    char *keys, *values;
    uint64_t page_stride, entry_stride, head_stride;  // elements
    uint32_t page_shift, pages, heads;
    const uint32_t *offsets, *lengths, *table;
    uint32_t table_stride, sequences, tokens, max_tokens, max_length;
};

// The checks of both descriptors, which the calls and adi_hip_paged_check share.
void require_paged(const adi_hip_paged_cache *cache, const adi_hip_paged_batch *batch);
PagedView paged_view(const adi_hip_paged_cache &cache, const adi_hip_paged_batch &batch);

// ---- device side -----------------------------------------------------------

// Sequence s's rows first .. first + count - 1 and entries. The arrays are the
// caller's device memory: whatever they hold, rows stay below `tokens`.
struct SequenceRows {
    uint32_t first, count, length;
    bool over;  // past max_tokens or max_length
};
__device__ __forceinline__ SequenceRows sequence_rows(const PagedView &c, uint32_t s) {
    const uint32_t a = min(c.offsets[s], c.tokens), b = min(c.offsets[s + 1u], c.tokens);
    const uint32_t count = b > a ? b - a : 0u, length = c.lengths[s];
    return {a, count, length, count > c.max_tokens || length > c.max_length};
}

__device__ __forceinline__ float bf16_of(uint32_t bits) { return __uint_as_float(bits << 16); }

// Two floats rounded to nearest and packed.
template <typename T>
__device__ __forceinline__ uint32_t pack(float x, float y) {
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    typedef T t2 __attribute__((ext_vector_type(2)));
    const f32x2 v = {x, y};
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, t2));
}

// N floats (1, 2, 4 or 8) rounded to T and stored side by side in as few stores
// as their bytes take (as an array of T the compiler stores them in pieces), `to`
// aligned to them or to 16 bytes.
template <typename T, uint32_t N>
__device__ __forceinline__ void store_values(T *to, const float (&v)[N]) {
    constexpr uint32_t kWords = N * sizeof(T) / 4u;
    if constexpr (kWords == 0u) {
        *to = static_cast<T>(v[0]);
    } else {
        uint32_t word[kWords];
#pragma unroll
        for (uint32_t i = 0; i < kWords; ++i) {
            if constexpr (sizeof(T) == 4u) {
                word[i] = __float_as_uint(v[i]);
            } else {
                word[i] = pack<T>(v[2u * i], v[2u * i + 1u]);
            }
        }
        typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
        typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
        if constexpr (kWords == 1u) {
            *reinterpret_cast<uint32_t *>(to) = word[0];
        } else if constexpr (kWords == 2u) {
            *reinterpret_cast<u32x2 *>(to) = u32x2{word[0], word[1]};
        } else {
#pragma unroll
            for (uint32_t i = 0; i < kWords; i += 4u) {
                reinterpret_cast<u32x4 *>(to)[i / 4u] = u32x4{word[i], word[i + 1u], word[i + 2u], word[i + 3u]};
            }
        }
    }
}

// cos and sin of `position` times a frequency of `turns` a position: the
// product and its whole quarter turns in 64 bits (exact to 2^-21 of a turn at
// position 2^32, 2^-35 at 2^18), then the Taylor sums on an eighth of a turn
// either side, whose first left-out terms are 1.1e-10 and 1.8e-9.
struct Turn {
    float cosine, sine;
};
__device__ __forceinline__ Turn turn_of(uint32_t position, double turns) {
    const double quarters = 4.0 * (static_cast<double>(position) * turns);
    const double whole = rint(quarters);
    const float x = static_cast<float>((quarters - whole) * 1.5707963267948966);
    const float y = x * x;
    float s = fmaf(y, 2.75573192e-6f, -1.98412698e-4f);
    s = fmaf(y, s, 8.33333333e-3f);
    s = fmaf(y, s, -1.66666667e-1f);
    s = fmaf(x * y, s, x);
    float c = fmaf(y, -2.75573192e-7f, 2.48015873e-5f);
    c = fmaf(y, c, -1.38888889e-3f);
    c = fmaf(y, c, 4.16666667e-2f);
    c = fmaf(y, c, -0.5f);
    c = fmaf(y, c, 1.0f);
    // the quarter turn modulo 4: whole is an integer below 2^34
    const uint32_t quarter = static_cast<uint32_t>(static_cast<int64_t>(whole)) & 3u;
    const float first = quarter & 1u ? s : c, second = quarter & 1u ? c : s;
    return {quarter == 1u || quarter == 2u ? -first : first, quarter >= 2u ? -second : second};
}

}  // namespace adi_hip
