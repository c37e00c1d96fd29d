// beam.hip -- a step of a beam search: the best candidates of every request over
// its beams and the vocabulary, and per-beam states that follow their parents.
//
// Selection: a beam of score s whose logits are l has the candidates
//   s + (l_v - lse),  lse = m + log sum_v exp(l_v - m),
// and a request takes the best of its beams'. One pass over the logits: a wave
// holds a tile of a row in registers, adds up its exponentials and finds its best
// logits (a row's candidates are in the order of its logits, whatever lse is); a
// block a request then joins the sums and ranks the tiles' candidates.
#include "paged_attention.hpp"

#include <algorithm>

namespace adi_hip {
namespace {

constexpr uint32_t kThreads = 256;
constexpr uint32_t kWaves = kThreads / kWave;
constexpr uint32_t kMaxBeams = 64, kMaxChoices = 128;
constexpr uint32_t kNone = 0xFFFFFFFFu;

using u32x2 = uint32_t __attribute__((ext_vector_type(2)));
using u32x4 = uint32_t __attribute__((ext_vector_type(4)));

struct BeamArgs {
    const char *logits;
    uint64_t request_stride, beam_stride;  // elements
    uint32_t beams, vocabulary, choices;
    uint32_t span, parts, arrivals;  // logits of a part, a row's parts, a request's blocks
    const float *scores, *weights;
    const uint32_t *ended;
    uint32_t ended_token, settle;
    float *out_scores;
    uint32_t *parents, *tokens;
    // of each row's parts: largest logit, sum of exponentials (reference_of), best logits
    float *most;
    double *sum;
    uint64_t *best;
    uint32_t *tickets;  // of each request, zero between calls
};

// Ascending with the float, -0 as +0.
__device__ __forceinline__ uint32_t ascending_key(float v) {
    const uint32_t bits = v == 0.0f ? 0u : __float_as_uint(v);
    return bits ^ ((bits & 0x80000000u) != 0u ? 0xFFFFFFFFu : 0x80000000u);
}
__device__ __forceinline__ float of_ascending_key(uint32_t key) {
    return __uint_as_float((key & 0x80000000u) != 0u ? key ^ 0x80000000u : ~key);
}
constexpr uint32_t kLowestKey = 0x007FFFFFu;  // of -infinity

// 16 bytes at an address that is a multiple of the element's size.
template <typename T>
struct Piece {
    static constexpr uint32_t kCount = 16u / sizeof(T);
    u32x4 raw;

    __device__ __forceinline__ void load(const char *from) { __builtin_memcpy(&raw, from, 16); }
    __device__ __forceinline__ float get(uint32_t i) const {
        if constexpr (sizeof(T) == 4u) {
            return __uint_as_float(raw[i]);
        } else if constexpr (std::is_same_v<T, __bf16>) {
            return __uint_as_float(i & 1u ? raw[i / 2u] & 0xFFFF0000u : raw[i / 2u] << 16);
        } else {
            return half_bits_to_float(i & 1u ? raw[i / 2u] >> 16 : raw[i / 2u] & 0xFFFFu);
        }
    }
    __device__ __forceinline__ void set(uint32_t i, T v) {
        if constexpr (sizeof(T) == 4u) {
            raw[i] = __builtin_bit_cast(uint32_t, v);
        } else {
            const uint32_t bits = __builtin_bit_cast(uint16_t, v);
            raw[i / 2u] = i & 1u ? (raw[i / 2u] & 0xFFFFu) | bits << 16 : (raw[i / 2u] & 0xFFFF0000u) | bits;
        }
    }
};

// The larger, or a NaN where either is one.
__device__ __forceinline__ float larger(float a, float b) { return __builtin_elementwise_maximum(a, b); }

using adi_hip::lane_xor;

__device__ __forceinline__ float wave_most(float v) {
    v = larger(v, lane_xor<1>(v));
    v = larger(v, lane_xor<2>(v));
    v = larger(v, lane_xor<4>(v));
    v = larger(v, lane_xor<8>(v));
    v = larger(v, lane_xor<16>(v));
    return larger(v, lane_xor<32>(v));
}

template <int MASK>
__device__ __forceinline__ double lane_xor(double v) {
    u32x2 bits = __builtin_bit_cast(u32x2, v);
    bits[0] = lane_xor_bits<MASK>(bits[0]);
    bits[1] = lane_xor_bits<MASK>(bits[1]);
    return __builtin_bit_cast(double, bits);
}

__device__ __forceinline__ double wave_sum(double v) {
    v += lane_xor<1>(v);
    v += lane_xor<2>(v);
    v += lane_xor<4>(v);
    v += lane_xor<8>(v);
    v += lane_xor<16>(v);
    return v + lane_xor<32>(v);
}

// A lane's kPieces pieces of a wave's tile, `from` its first logit. Rows of 16-bit
// logits may begin in the middle of a word, where loads of 16 bytes are split by
// their bytes: such a piece is put together from the words around it, each of
// which holds a logit of the piece.
template <typename T, uint32_t PIECES>
__device__ __forceinline__ void load_tile(Piece<T> (&x)[PIECES], const char *from, uint32_t lane) {
    if (sizeof(T) == 4u || (reinterpret_cast<uintptr_t>(from) & 2u) == 0u) {
#pragma unroll
        for (uint32_t j = 0; j < PIECES; ++j) {
            x[j].load(from + (j * kWave + lane) * 16u);
        }
        return;
    }
    u32x4 head[PIECES];
    uint32_t tail[PIECES];
#pragma unroll
    for (uint32_t j = 0; j < PIECES; ++j) {
        const uint32_t *const words = reinterpret_cast<const uint32_t *>(from - 2 + (j * kWave + lane) * 16u);
        __builtin_memcpy(&head[j], words, 16);
        tail[j] = words[4];
    }
#pragma unroll
    for (uint32_t j = 0; j < PIECES; ++j) {
#pragma unroll
        for (uint32_t i = 0; i < 4u; ++i) {
            x[j].raw[i] = __builtin_amdgcn_alignbit(i < 3u ? head[j][i + 1u] : tail[j], head[j][i], 16u);
        }
    }
}

// The same of a tile of which only the first `live` logits are the row's: -infinity
// behind them. (No branches, so that all loads are on their way at once.)
template <typename T, uint32_t PIECES>
__device__ __forceinline__ void load_last(Piece<T> (&x)[PIECES], const char *from, uint32_t lane, uint32_t live) {
    constexpr uint32_t kCount = Piece<T>::kCount;
    T v[PIECES][kCount];
#pragma unroll
    for (uint32_t j = 0; j < PIECES; ++j) {
#pragma unroll
        for (uint32_t i = 0; i < kCount; ++i) {
            v[j][i] = reinterpret_cast<const T *>(from)[min((j * kWave + lane) * kCount + i, live - 1u)];
        }
    }
#pragma unroll
    for (uint32_t j = 0; j < PIECES; ++j) {
#pragma unroll
        for (uint32_t i = 0; i < kCount; ++i) {
            x[j].set(i, (j * kWave + lane) * kCount + i < live ? v[j][i] : static_cast<T>(-__builtin_huge_valf()));
        }
    }
}

// The largest key of 16 bits, 0s behind, that at least `count` of the two of each
// of the wave's lanes reach (0 where fewer are not 0).
__device__ __forceinline__ uint32_t reached_by(uint32_t a, uint32_t b, uint32_t count) {
    uint32_t reached = 0u;
#pragma unroll 4
    for (uint32_t bit = 0x80000000u; bit != 0x8000u; bit >>= 1) {
        const uint32_t more = reached | bit;
        const uint32_t reach = static_cast<uint32_t>(__popcll(__ballot(a >= more)) + __popcll(__ballot(b >= more)));
        reached = reach >= count ? more : reached;
    }
    return reached;
}

// e^v / 2^whole for floats of which the largest is about whole ln 2 (-65536 for
// those below). In 64 bits, since the sums' logarithms decide between beams: v log2 e
// = n + r with |r| <= 1/2 by two fused products, 2^r by the polynomial of degree 7
// that is nearest on that interval (2^-34.5 of it; solved for by exchange), n - whole
// added to its exponent. Values more than 1000 powers of two below count as 2^-1000.
constexpr double kLog2e = 1.4426950408889634, kLn2 = 0.6931471805599453;
constexpr float kFar = 65536.0f;

struct Exponentials {
    static constexpr double kRound = 6755399441055744.0;  // 1.5 2^52
    double rounding;
    float least;

    // From here on for `top`; returns whole before - whole now.
    __device__ __forceinline__ int32_t raise(float top) {
        const double whole = rint(static_cast<double>(fmaxf(top, -kFar)) * kLog2e), before = rounding;
        rounding = kRound - whole;
        least = static_cast<float>((whole - 1000.0) * kLn2);
        return static_cast<int32_t>(rounding - before);
    }
    __device__ __forceinline__ double of(float v) const {
        const double x = static_cast<double>(larger(v, least));
        const double moved = fma(x, kLog2e, rounding);
        const double r = fma(x, kLog2e, -(moved - rounding));
        double p = fma(r, 1.520192398382284e-05, 0.00015469291034881546);
        p = fma(r, p, 0.0013333922552474853);
        p = fma(r, p, 0.0096180272541093615);
        p = fma(r, p, 0.055504103534627078);
        p = fma(r, p, 0.24022651198153328);
        p = fma(r, p, 0.6931471807284425);
        p = fma(r, p, 0.99999999996168243);
        u32x2 bits = __builtin_bit_cast(u32x2, p);
        bits[1] += __builtin_bit_cast(u32x2, moved)[0] << 20;
        return __builtin_bit_cast(double, bits);
    }
};

// What a part's sum is to be multiplied by, as a logarithm (beam_part).
__device__ __forceinline__ double reference_of(float top) {
    return fabsf(top) < kFar ? rint(static_cast<double>(top) * kLog2e) * kLn2 : static_cast<double>(top);
}

using adi_hip::coherent_load;
using adi_hip::coherent_store;
__device__ __forceinline__ uint64_t coherent_load(const uint64_t *p) {
    return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ double coherent_load(const double *p) {
    return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ void coherent_store(uint64_t *p, uint64_t v) {
    __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ void coherent_store(double *p, double v) {
    __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// A candidate in the order of candidates: the larger rank (as a whole number), then
// the larger tie: the lower beam, then the larger logit, then the lower token.
// A rank of 0 is no candidate's (it would be a NaN's).
struct Candidate {
    uint64_t rank, tie;
};
__device__ __forceinline__ bool precedes(const Candidate &a, const Candidate &b) {
    return a.rank > b.rank || (a.rank == b.rank && a.tie > b.tie);
}
__device__ __forceinline__ Candidate choose(bool first, const Candidate &a, const Candidate &b) {
    return Candidate{first ? a.rank : b.rank, first ? a.tie : b.tie};
}
__device__ __forceinline__ uint64_t ascending_key(double v) {
    const uint64_t bits = __builtin_bit_cast(uint64_t, v + 0.0);
    return bits ^ (bits >> 63 != 0u ? ~0ull : 1ull << 63);
}
constexpr uint32_t kTokenBits = 24;
__device__ __forceinline__ uint64_t tie_of(uint32_t beam, uint64_t key) {
    return static_cast<uint64_t>(kMaxBeams - 1u - beam) << 56 | key >> 32 << kTokenBits |
           (key & ((1u << kTokenBits) - 1u));
}

constexpr uint32_t kJoinList = 512;

struct JoinShared {
    double lse[kMaxBeams], score[kMaxBeams], weight[kMaxBeams];
    uint32_t kind[kMaxBeams];  // 0: no candidates, 1: its logits', 2: ended
    uint64_t rank[kJoinList], tie[kJoinList];
    uint64_t taken[kMaxChoices];  // ties
    alignas(16) uint32_t keys[kThreads];
    uint32_t listed, bad;
};

__device__ __forceinline__ uint64_t read_lane(uint64_t v, uint32_t lane) {
    const u32x2 bits = __builtin_bit_cast(u32x2, v);
    const u32x2 of = {static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(bits[0]), static_cast<int>(lane))),
                      static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(bits[1]), static_cast<int>(lane)))};
    return __builtin_bit_cast(uint64_t, of);
}

// Joins a request's parts: the beams' logarithms, 64 / `group` beams a wave, then the
// candidates. The heads of the parts' lists (all candidates, where the lists are few)
// bound what is taken from below, and of each list what reaches that bound goes to
// a list in LDS, whose entries find their places by counting. Bound by its chain of
// loads, sums and barriers: 4 beams' 488 parts about 6 us, 64 requests of 8 beams with 16
// choices 9.4.
__device__ __forceinline__ void join_request(const BeamArgs &args, uint32_t request, JoinShared &lds) {
    const uint32_t t = threadIdx.x, lane = t & 63u, wave = t / kWave;
    const uint32_t k = args.beams, choices = args.choices, parts = args.parts;
    const uint64_t *const best = args.best + static_cast<uint64_t>(request) * k * parts * choices;
    // items: the lists, or their candidates one by one; then the ended beams
    const uint32_t depth = k * parts >= 4u * choices ? choices : 1u;
    const uint32_t of_beam = parts * (choices / depth), items = k * of_beam;
    // (on their way while the logarithms are made: two items' first two candidates)
    constexpr uint32_t kHeld = 2;
    uint64_t head[kHeld][kHeld];
#pragma unroll
    for (uint32_t q = 0; q < kHeld; ++q) {
#pragma unroll
        for (uint32_t j = 0; j < kHeld; ++j) {
            head[q][j] = coherent_load(best + static_cast<uint64_t>(min(q * kThreads + t, items - 1u)) * depth +
                                       min(j, depth - 1u));
        }
    }
    if (t == 0u) {
        lds.listed = 0u;
        lds.bad = 0u;
    }
    if (t < choices) {
        lds.taken[t] = 0u;
    }
    __syncthreads();
    // lanes of a beam: the power of two from the parts on, at most a wave
    const uint32_t group = min(1u << (32u - static_cast<uint32_t>(__builtin_clz(2u * parts - 1u)) - 1u), kWave);
    for (uint32_t base = wave * (kWave / group); base < k; base += kWaves * (kWave / group)) {
        const uint32_t b = base + lane / group, within = lane % group;
        const uint32_t row = request * k + min(b, k - 1u);
        const float *const most = args.most + static_cast<uint64_t>(row) * parts;
        const double *const sum = args.sum + static_cast<uint64_t>(row) * parts;
        // (its last part again, where a lane has none)
        const float s = args.scores[row], w = args.weights != nullptr ? args.weights[row] : 1.0f;
        const uint32_t gone = args.ended != nullptr ? args.ended[row] : 0u;
        float most_of[kHeld];
        double sum_of[kHeld];
#pragma unroll
        for (uint32_t q = 0; q < kHeld; ++q) {
            most_of[q] = coherent_load(most + min(within + q * group, parts - 1u));
            sum_of[q] = coherent_load(sum + min(within + q * group, parts - 1u));
        }
        uint32_t what = b >= k || s == -__builtin_huge_valf() ? 0u : gone != 0u ? 2u : 1u;
        bool wrong = what != 0u && !(__builtin_isfinite(s) && w > 0.0f && __builtin_isfinite(w));
        float top = larger(most_of[0], most_of[1]);
        for (uint32_t p = within + kHeld * group; p < parts; p += group) {
            top = larger(top, coherent_load(most + p));
        }
        const auto over_group = [&](auto &&join) {
            if (group > 1u) { join(std::integral_constant<int, 1>()); }
            if (group > 2u) { join(std::integral_constant<int, 2>()); }
            if (group > 4u) { join(std::integral_constant<int, 4>()); }
            if (group > 8u) { join(std::integral_constant<int, 8>()); }
            if (group > 16u) { join(std::integral_constant<int, 16>()); }
            if (group > 32u) { join(std::integral_constant<int, 32>()); }
        };
        over_group([&](auto step) { top = larger(top, lane_xor<decltype(step)::value>(top)); });
        const auto part = [&](float own, double value) {
            return own == -__builtin_huge_valf() ? 0.0 : value * exp(reference_of(own) - static_cast<double>(top));
        };
        double total = within < parts ? part(most_of[0], sum_of[0]) : 0.0;
        total += within + group < parts ? part(most_of[1], sum_of[1]) : 0.0;
        for (uint32_t p = within + kHeld * group; p < parts; p += group) {
            total += part(coherent_load(most + p), coherent_load(sum + p));
        }
        over_group([&](auto step) { total += lane_xor<decltype(step)::value>(total); });
        // a NaN or +infinity among the logits leaves a NaN in the sum
        wrong = wrong || (what == 1u && total != total);
        what = what == 1u && top == -__builtin_huge_valf() ? 0u : what;
        if (within == 0u && b < k) {
            lds.lse[b] = static_cast<double>(top) + log(total);
            lds.score[b] = s;
            lds.weight[b] = w;
            lds.kind[b] = what;
            if (wrong) {
                lds.bad = 1u;
            }
        }
    }
    __syncthreads();
    float *const out_scores = args.out_scores + static_cast<uint64_t>(request) * choices;
    uint32_t *const parents = args.parents + static_cast<uint64_t>(request) * choices;
    uint32_t *const tokens = args.tokens + static_cast<uint64_t>(request) * choices;
    if (lds.bad != 0u) {
        if (t < choices) {
            out_scores[t] = __builtin_nanf("");
            parents[t] = kNone;
            tokens[t] = kNone;
        }
        return;
    }
    const auto of_key = [&](uint32_t beam, uint64_t key) {
        Candidate c{0u, 0u};
        if (key != 0u && lds.kind[beam] == 1u) {
            const double logit = of_ascending_key(static_cast<uint32_t>(key >> 32));
            c.rank = ascending_key((lds.score[beam] + (logit - lds.lse[beam])) * lds.weight[beam]);
            c.tie = tie_of(beam, key);
        }
        return c;
    };
    const auto ended = [&](uint32_t beam) {
        Candidate c{0u, 0u};
        if (lds.kind[beam] == 2u) {
            c.rank = ascending_key(lds.score[beam] * lds.weight[beam]);
            c.tie = tie_of(beam, ~0ull);
        }
        return c;
    };
    // item i's candidate j
    const auto candidate = [&](uint32_t i, uint32_t j) {
        return i >= items ? ended(i - items)
                          : of_key(i / of_beam, coherent_load(best + static_cast<uint64_t>(i) * depth + j));
    };
    // the items held: candidates of ended beams come after them
    Candidate held[kHeld][kHeld];
    uint32_t own = 0u;
#pragma unroll
    for (uint32_t q = 0; q < kHeld; ++q) {
        const uint32_t i = q * kThreads + t;
#pragma unroll
        for (uint32_t j = 0; j < kHeld; ++j) {
            held[q][j] = of_key(min(i, items - 1u) / of_beam, i < items && j < depth ? head[q][j] : 0u);
        }
        own = max(own, static_cast<uint32_t>(held[q][0].rank >> 32));
    }
    for (uint32_t i = kHeld * kThreads + t; i < items; i += kThreads) {
        own = max(own, static_cast<uint32_t>(candidate(i, 0u).rank >> 32));
    }
    if (t < k) {
        own = max(own, static_cast<uint32_t>(ended(t).rank >> 32));
    }
    lds.keys[t] = own;
    __syncthreads();
    const u32x4 four = *reinterpret_cast<const u32x4 *>(lds.keys + 4u * lane);
    uint32_t least = 0u;
#pragma unroll 4
    for (uint32_t bit = 0x80000000u; bit != 0x80u; bit >>= 1) {
        const uint32_t more = least | bit;
        const uint32_t reach =
            static_cast<uint32_t>(__popcll(__ballot(four[0] >= more)) + __popcll(__ballot(four[1] >= more)) +
                                  __popcll(__ballot(four[2] >= more)) + __popcll(__ballot(four[3] >= more)));
        least = reach >= choices ? more : least;
    }
    least = max(least, 1u);
    const auto take = [&](const Candidate &c) {
        const bool takes = static_cast<uint32_t>(c.rank >> 32) >= least;
        if (takes) {
            const uint32_t at = atomicAdd(&lds.listed, 1u);
            if (at < kJoinList) {
                lds.rank[at] = c.rank;
                lds.tie[at] = c.tie;
            }
        }
        return takes;
    };
#pragma unroll
    for (uint32_t q = 0; q < kHeld; ++q) {
        bool takes = take(held[q][0]);
        takes = takes && take(held[q][1]);
        for (uint32_t j = kHeld; takes && j < depth; ++j) {
            takes = take(candidate(q * kThreads + t, j));
        }
    }
    for (uint32_t i = kHeld * kThreads + t; i < items; i += kThreads) {
        for (uint32_t j = 0; j < depth && take(candidate(i, j)); ++j) {
        }
    }
    if (t < k) {
        (void)take(ended(t));
    }
    __syncthreads();
    const uint32_t entries = lds.listed;
    if (entries <= kJoinList) {
        // (entries are read from lanes: read from LDS, each of them is a wait)
        for (uint32_t e = t; e < (entries + 63u) / 64u * 64u; e += kThreads) {
            const Candidate c{e < entries ? lds.rank[e] : 0u, e < entries ? lds.tie[e] : 0u};
            uint32_t before = 0u;
            for (uint32_t from = 0; from < entries; from += kWave) {
                const uint32_t held = min(entries - from, kWave);
                const uint32_t at = min(from + lane, entries - 1u);
                const Candidate h{lds.rank[at], lds.tie[at]};
                for (uint32_t o = 0; o < held; ++o) {
                    const Candidate other{read_lane(h.rank, o), read_lane(h.tie, o)};
                    before += precedes(other, c) ? 1u : 0u;
                }
            }
            if (e < entries && before < choices) {
                lds.taken[before] = c.tie;
            }
        }
    } else {
        // so many near each other: one after another
        Candidate last{~0ull, ~0ull};
        for (uint32_t n = 0; n < choices; ++n) {
            Candidate next{0u, 0u};
            for (uint32_t i = t; i < items + k; i += kThreads) {
                for (uint32_t j = 0; j < (i < items ? depth : 1u); ++j) {
                    const Candidate c = candidate(i, j);
                    if (c.rank == 0u) {
                        break;
                    }
                    next = choose(precedes(last, c) && precedes(c, next), c, next);
                }
            }
            lds.rank[t] = next.rank;
            lds.tie[t] = next.tie;
            __syncthreads();
            last = Candidate{0u, 0u};
            for (uint32_t o = 0; o < kThreads; ++o) {
                const Candidate c{lds.rank[o], lds.tie[o]};
                last = choose(precedes(c, last), c, last);
            }
            if (t == 0u) {
                lds.taken[n] = last.tie;
            }
            __syncthreads();
            if (last.rank == 0u) {
                break;
            }
        }
    }
    __syncthreads();
    if (t < choices) {
        const uint64_t tie = lds.taken[t];
        const bool some = tie != 0u;
        const uint32_t beam = kMaxBeams - 1u - static_cast<uint32_t>(tie >> 56);
        uint32_t place = t;
        if (args.settle != 0u) {
            // (choices = beams <= 64: the lanes of the first wave.) The parent's row
            // for its first child; the others' rows, and those of places without a
            // candidate, are the rows without one, in turn
            bool first = some;
            uint64_t children = 0u;
            for (uint32_t o = 0; o < choices; ++o) {
                const uint32_t parent = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(beam), static_cast<int>(o)));
                const bool lives = __builtin_amdgcn_readlane(some ? 1 : 0, static_cast<int>(o)) != 0;
                first = first && (o >= t || parent != beam);
                children |= lives ? 1ull << parent : 0u;
            }
            const uint64_t others = __ballot(!first) & ((1ull << t) - 1u);
            uint64_t rows = ~children;
            for (uint32_t nth = static_cast<uint32_t>(__popcll(others)); nth != 0u; --nth) {
                rows &= rows - 1u;
            }
            place = first ? beam : static_cast<uint32_t>(__builtin_ctzll(rows | 1ull << 63));
        }
        double value = -__builtin_huge_val();
        uint32_t token = kNone;
        if (some && lds.kind[beam] == 2u) {
            value = lds.score[beam];
            token = args.ended_token;
        } else if (some) {
            value = lds.score[beam] + (of_ascending_key(static_cast<uint32_t>(tie >> kTokenBits)) - lds.lse[beam]);
            token = ~static_cast<uint32_t>(tie) & ((1u << kTokenBits) - 1u);
        }
        out_scores[place] = static_cast<float>(value);
        parents[place] = some ? beam : kNone;
        tokens[place] = token;
    }
}

// The next float below a key's (the key below that of 0 is that of -0, which is
// not below 0).
__device__ __forceinline__ float below(uint32_t key) {
    return of_ascending_key(key - (key == 0x80000000u ? 2u : 1u));
}

// The best of a wave's part so far, in LDS: keys as Candidate's. `edge`: a logit is
// among the best only if it is larger.
constexpr uint32_t kPartList = 256;

__device__ __forceinline__ void wave_lds() { __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront"); }

// Keeps the `choices` first of the list's entries, in order: an entry's place is
// the number of entries before it. (Entries are held by lanes and read from
// there: read from LDS, each of them is a wait.)
__device__ __forceinline__ void keep_best(uint64_t *list, uint32_t &entries, uint32_t choices, uint32_t lane) {
    constexpr uint32_t kHeld = kPartList / kWave;
    wave_lds();
    uint64_t own[kHeld];
    uint32_t before[kHeld];
#pragma unroll
    for (uint32_t q = 0; q < kHeld; ++q) {
        own[q] = q * kWave + lane < entries ? list[q * kWave + lane] : 0u;
        before[q] = 0u;
    }
    if (entries <= kWave) {
        for (uint32_t o = 0; o < entries; ++o) {
            before[0] += read_lane(own[0], o) > own[0] ? 1u : 0u;
        }
    } else {
#pragma unroll
        for (uint32_t p = 0; p < kHeld; ++p) {
            const uint32_t held = entries > p * kWave ? min(entries - p * kWave, kWave) : 0u;
#pragma unroll 1
            for (uint32_t o = 0; o < held; ++o) {
                const uint64_t other = read_lane(own[p], o);
#pragma unroll
                for (uint32_t q = 0; q < kHeld; ++q) {
                    before[q] += other > own[q] ? 1u : 0u;
                }
            }
        }
    }
    wave_lds();
#pragma unroll
    for (uint32_t q = 0; q < kHeld; ++q) {
        if (q * kWave + lane < entries && before[q] < choices) {
            list[before[q]] = own[q];
        }
    }
    entries = min(entries, choices);
    wave_lds();
}

// Drops entries from a list of up to 64 that are not among its `choices` best: those
// below the key of 16 bits that `choices` of them reach, which is returned. Not all
// of them and in no order, but in a sixth of keep_best's instructions.
__device__ __forceinline__ uint32_t trim(uint64_t *list, uint32_t &entries, uint32_t choices, uint32_t lane) {
    wave_lds();
    const uint64_t own = lane < entries ? list[lane] : 0u;
    const uint32_t key = static_cast<uint32_t>(own >> 32), reached = reached_by(key, 0u, choices);
    const uint64_t stays = __ballot(key >= reached && lane < entries);
    wave_lds();
    if (key >= reached && lane < entries) {
        list[__builtin_amdgcn_mbcnt_hi(static_cast<uint32_t>(stays >> 32),
                                       __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(stays), 0u))] = own;
    }
    entries = static_cast<uint32_t>(__popcll(stays));
    wave_lds();
    return reached;
}

// A wave's part of a row: tiles of 64 x N logits, each held in registers, the next on
// its way. A lane adds up its own exponentials, in powers of two below its own
// largest logit so far. The best: in a first tile, the `choices` best of the lanes'
// own two largest (of their pieces' halves) bound what is taken from below, later the
// last of those taken so far, by any wave of the block. Bound by its instructions, 23
// for 64 logits, 15 of them the exponential (64 x 8 rows of 248,320 bf16 logits: 108 to
// 119 us with the join on four cards, 2.4 to 2.1 TB/s; f16 113 where bf16 takes 108); few
// tiles a wave by its start and end. A part of ONE tile is the same
// without the next tile and the bounds for it (16 x 4 rows of 248,320 f32 logits 22.9
// us in place of 24.2, 32 x 4 39.4 and 41.8).
template <typename T, uint32_t N, bool ONE>
__device__ __forceinline__ void beam_part(const BeamArgs &args, uint32_t part, uint32_t row, const char *from,
                                          uint64_t *list, uint32_t *shared) {
    constexpr uint32_t kCount = Piece<T>::kCount, kPieces = N / kCount, kTile = kWave * N;
    const uint32_t lane = threadIdx.x & 63u, choices = args.choices;
    const uint32_t first = part * args.span, end = min(first + args.span, args.vocabulary);
    uint32_t entries = 0u;
    uint64_t least = 0u;  // keys above it are taken
    float edge = -__builtin_huge_valf(), top = -__builtin_huge_valf();
    Exponentials e;
    e.rounding = Exponentials::kRound;
    (void)e.raise(-kFar);
    double total = 0.0;
    const auto load = [&](Piece<T> (&x)[kPieces], uint32_t at) {
        const char *const tile = from + static_cast<uint64_t>(at) * sizeof(T);
        if (end - at >= kTile) {
            load_tile(x, tile, lane);
        } else {
            load_last(x, tile, lane, end - at);
        }
    };
    // a key that `choices` logits of the row reach is the other waves' bound too
    const auto share = [&](uint32_t reached) {
        if (lane == 0u) {
            atomicMax(shared, reached);
        }
    };
    Piece<T> next[kPieces];
    load(next, first);
    // (asked for after the first tile, so as not to wait for one before the other)
    if (args.scores[row] == -__builtin_huge_valf() || (args.ended != nullptr && args.ended[row] != 0u)) {
        return;
    }
#pragma unroll 1
    for (uint32_t at = first; at < end; at += kTile) {
        Piece<T> x[kPieces];
#pragma unroll
        for (uint32_t j = 0; j < kPieces; ++j) {
            x[j] = next[j];
        }
        if (!ONE && end - at > kTile) {
            load(next, at + kTile);
        }
        float half[2] = {-__builtin_huge_valf(), -__builtin_huge_valf()};
#pragma unroll
        for (uint32_t j = 0; j < kPieces; ++j) {
#pragma unroll
            for (uint32_t i = 0; i < kCount; i += 2u) {
                float &own = half[(j * kCount + i) * 2u / N];
                own = larger(own, larger(x[j].get(i), x[j].get(i + 1u)));
            }
        }
        const float own = larger(half[0], half[1]);
        top = larger(top, own);
        total = ldexp(total, e.raise(top));
        if (entries < choices) {
            const uint32_t reached =
                max(reached_by(ascending_key(half[0]), ascending_key(half[1]), choices), kLowestKey + 1u);
            least = static_cast<uint64_t>(reached) << 32;
            edge = below(reached);
            if (!ONE) {
                share(reached);
            }
        }
        if (!ONE && at != first) {
            const uint32_t reached = *static_cast<volatile uint32_t *>(shared);
            least = max(least, static_cast<uint64_t>(reached) << 32);
            edge = fmaxf(edge, below(max(reached, kLowestKey + 1u)));
        }
        if (__ballot(own > edge) != 0u) {
            const uint32_t held = entries;
#pragma unroll
            for (uint32_t j = 0; j < kPieces; ++j) {
#pragma unroll
                for (uint32_t i = 0; i < kCount; ++i) {
                    const float v = x[j].get(i);
                    const uint64_t takes = __ballot(v > edge);
                    if (takes != 0u) {
                        const uint32_t place =
                            entries + __builtin_amdgcn_mbcnt_hi(
                                          static_cast<uint32_t>(takes >> 32),
                                          __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(takes), 0u));
                        if (v > edge && place < kPartList) {
                            list[place] = static_cast<uint64_t>(ascending_key(v)) << 32 |
                                          static_cast<uint32_t>(~(at + (j * kWave + lane) * kCount + i));
                        }
                        entries += static_cast<uint32_t>(__popcll(takes));
                    }
                }
            }
            if (entries > kPartList) {
                // more than the list holds (many equal ones, or all in few lanes): again
                // lane by lane, read from memory, with only the best kept
                entries = held;
                for (uint64_t holders = __ballot(own > edge); holders != 0u; holders &= holders - 1u) {
                    const uint32_t i = lane % N, holder = static_cast<uint32_t>(__builtin_ctzll(holders));
                    const uint32_t place = at + (i / kCount * kWave + holder) * kCount + i % kCount;
                    float v = -__builtin_huge_valf();
                    if (lane < N && place < end) {
                        v = static_cast<float>(reinterpret_cast<const T *>(from)[place]);
                    }
                    const uint64_t key = static_cast<uint64_t>(ascending_key(v)) << 32 | static_cast<uint32_t>(~place);
                    const bool takes = v > -__builtin_huge_valf() && key > least;
                    const uint64_t taken = __ballot(takes);
                    if (takes) {
                        list[entries + __builtin_amdgcn_mbcnt_hi(
                                           static_cast<uint32_t>(taken >> 32),
                                           __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(taken), 0u))] = key;
                    }
                    entries += static_cast<uint32_t>(__popcll(taken));
                    if (entries > kPartList - kWave) {
                        keep_best(list, entries, choices, lane);
                        least = entries == choices ? list[choices - 1u] : least;
                    }
                }
            }
            if (!ONE && end - at > kTile && entries >= choices + choices / 2u + 4u) {
                if (entries <= kWave) {
                    const uint32_t reached = trim(list, entries, choices, lane);
                    least = max(least, static_cast<uint64_t>(reached) << 32);
                    edge = fmaxf(edge, below(reached));
                    share(reached);
                } else {
                    keep_best(list, entries, choices, lane);
                    least = list[choices - 1u];
                    edge = of_ascending_key(static_cast<uint32_t>(least >> 32));
                    share(static_cast<uint32_t>(least >> 32));
                }
            }
        }
#pragma unroll
        for (uint32_t j = 0; j < kPieces; ++j) {
#pragma unroll
            for (uint32_t i = 0; i < kCount; ++i) {
                total += e.of(x[j].get(i));
            }
        }
        if constexpr (ONE) {
            break;
        }
    }
    const float most = wave_most(top);
    if (fabsf(most) < kFar) {
        Exponentials whole;
        whole.rounding = e.rounding;
        total = ldexp(total, whole.raise(most));
    } else {
        // too far from 0 for that, or a NaN or an infinity, which give a NaN
        total = 0.0;
        if (most != -__builtin_huge_valf()) {
#pragma unroll 1
            for (uint32_t at = first + lane; at < end; at += kWave) {
                total += exp(static_cast<double>(static_cast<float>(reinterpret_cast<const T *>(from)[at])) -
                             static_cast<double>(most));
            }
        }
    }
    total = wave_sum(total);
    keep_best(list, entries, choices, lane);
    const uint64_t place = static_cast<uint64_t>(row) * args.parts + part;
    for (uint32_t i = lane; i < choices; i += kWave) {
        coherent_store(args.best + place * choices + i, i < entries ? list[i] : uint64_t(0));
    }
    if (lane == 0u) {
        coherent_store(args.most + place, most);
        coherent_store(args.sum + place, total);
    }
}

// A wave a part; where the launch joins, the last block of a request's through its
// ticket does.
// (Waves a SIMD that the registers are held to: long parts of bf16 rows fit in five
// without spills, 512 rows of 248,320 115 us in place of 125; f32 and f16 rows spill.
// Parts of ONE tile take 69 to 75 registers either way.)
template <typename T, bool ONE>
constexpr int kResident = !ONE && std::is_same_v<T, __bf16> ? 5 : 4;

template <typename T, uint32_t N, bool ONE, bool JOINS>
__global__ __launch_bounds__(kThreads, (kResident<T, ONE>)) void k_beam_select(BeamArgs args) {
    __shared__ union Shared {
        uint64_t list[kWaves][kPartList];
        std::conditional_t<JOINS, JoinShared, uint32_t> join;
    } lds;
    __shared__ uint32_t last, reached;
    if (threadIdx.x == 0u) {
        reached = 0u;
    }
    __syncthreads();
    const uint32_t row = blockIdx.z * args.beams + blockIdx.y;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), part = blockIdx.x * kWaves + wave;
    if (part < args.parts) {
        const char *const from =
            args.logits + (blockIdx.z * args.request_stride + blockIdx.y * args.beam_stride) * sizeof(T);
        beam_part<T, N, ONE>(args, part, row, from, lds.list[wave], &reached);
    }
    if constexpr (JOINS) {
        wait_stores();
        __syncthreads();
        if (threadIdx.x == 0u) {
            uint32_t *const ticket = args.tickets + blockIdx.z;
            last = coherent_add(ticket, 1u) + 1u == args.arrivals ? 1u : 0u;
            if (last != 0u) {
                coherent_store(ticket, 0u);
            }
        }
        __syncthreads();
        if (last != 0u) {
            join_request(args, blockIdx.z, lds.join);
        }
    }
}

__global__ __launch_bounds__(kThreads) void k_beam_join(BeamArgs args) {
    __shared__ JoinShared lds;
    join_request(args, blockIdx.x, lds);
}

template <typename T, uint32_t N, bool ONE, bool JOINS>
void launch_select(adi_hip_context *ctx, const adi_hip_beam_arguments &a, const adi_hip_paged_workspace &workspace,
                   uint32_t tiles) {
    BeamArgs args{};
    args.logits = static_cast<const char *>(a.logits);
    args.request_stride = a.request_stride;
    args.beam_stride = a.beam_stride;
    args.beams = a.beams;
    args.vocabulary = a.vocabulary;
    args.choices = a.choices;
    args.span = tiles * kWave * N;
    args.parts = ceil_div(a.vocabulary, args.span);
    args.arrivals = ceil_div(args.parts, kWaves) * a.beams;
    args.scores = a.scores;
    args.weights = a.weights;
    args.ended = a.ended;
    args.ended_token = a.ended_token;
    args.settle = a.settle;
    args.out_scores = a.out_scores;
    args.parents = a.parents;
    args.tokens = a.tokens;
    args.tickets = static_cast<uint32_t *>(workspace.base);
    // as many requests at once as the workspace holds
    const uint64_t parts = uint64_t(a.beams) * args.parts;
    const uint64_t bytes = parts * (sizeof(double) + sizeof(uint64_t) * a.choices + sizeof(float));
    const uint64_t room = workspace.bytes - kTickets * sizeof(uint32_t);
    const uint64_t at_once = std::min<uint64_t>({room / bytes, a.requests, (1u << 23) / parts, kTickets - 1u});
    if (at_once == 0) {
        fail(ADI_HIP_OUT_OF_MEMORY, "beam select: a request needs a workspace of " +
                                        std::to_string(bytes + kTickets * sizeof(uint32_t)) + " bytes");
    }
    char *const base = static_cast<char *>(workspace.base) + kTickets * sizeof(uint32_t);
    args.sum = reinterpret_cast<double *>(base);
    args.best = reinterpret_cast<uint64_t *>(args.sum + at_once * parts);
    args.most = reinterpret_cast<float *>(args.best + at_once * parts * a.choices);
    for (uint64_t done = 0; done < a.requests; done += at_once) {
        const uint32_t requests = static_cast<uint32_t>(std::min<uint64_t>(at_once, a.requests - done));
        const dim3 grid(ceil_div(args.parts, kWaves), a.beams, requests), block(kThreads);
        launch(ctx, "beam_select", k_beam_select<T, N, ONE, JOINS>, grid, block, 0, args);
        if (!JOINS) {
            launch(ctx, "beam_join", k_beam_join, dim3(requests), block, 0, args);
        }
        args.logits += requests * args.request_stride * sizeof(T);
        args.scores += requests * a.beams;
        args.weights += args.weights != nullptr ? requests * a.beams : 0;
        args.ended += args.ended != nullptr ? requests * a.beams : 0;
        args.out_scores += requests * a.choices;
        args.parents += requests * a.choices;
        args.tokens += requests * a.choices;
    }
}

// Tiles of 512 logits where that makes at most a wave a CU, else of 2048 (one request
// of 4 x 248,320 f32 logits: 12.5 us, with tiles of 1024 and 512 15.0 and 20.5, as
// more parts are joined; of 4 x 512 in 512s 8.0, in 2048s 9.4), and as many a part as
// leave 32 waves a CU, about. Up to half a block a CU the last of a request's blocks
// joins within the launch (4 x 512 logits 8.0 us, by a launch of its own 9.5; 4 x
// 32,000 9.8 and 10.5); more wait for each other at the ticket, and the launch's end
// for the join (2 x 4 x 248,320: 13.9 and 12.5, 16 requests of them 36.7 and 23.2).
template <typename T>
void launch_select(adi_hip_context *ctx, const adi_hip_beam_arguments &a, const adi_hip_paged_workspace &workspace) {
    const uint64_t rows = uint64_t(a.requests) * a.beams, cus = static_cast<uint64_t>(ctx->cu_count);
    const auto single = [&](auto n) {
        constexpr uint32_t N = decltype(n)::value;
        if (rows * ceil_div(ceil_div(a.vocabulary, kWave * N), kWaves) <= cus / 2u) {
            launch_select<T, N, true, true>(ctx, a, workspace, 1u);
        } else {
            launch_select<T, N, true, false>(ctx, a, workspace, 1u);
        }
    };
    const uint64_t tiles = std::min<uint64_t>(rows * ceil_div(a.vocabulary, kWave * 32u) / (32u * cus), 16u);
    if (tiles > 1u) {
        launch_select<T, 32, false, false>(ctx, a, workspace, static_cast<uint32_t>(tiles));
    } else if (rows * ceil_div(a.vocabulary, kWave * 8u) <= cus) {
        single(std::integral_constant<uint32_t, 8>());
    } else {
        single(std::integral_constant<uint32_t, 32>());
    }
}

void require_select(const adi_hip_beam_arguments *a) {
    require(a != nullptr, "beam select: null arguments");
    require(known_type(a->type), "beam select: unknown type of logits");
    require(a->beams >= 1 && a->beams <= kMaxBeams, "beam select: beams must be 1 to 64");
    require(a->choices >= 1 && a->choices <= kMaxChoices, "beam select: choices must be 1 to 128");
    require(a->vocabulary >= 1 && a->vocabulary <= (1u << 24), "beam select: vocabulary must be 1 to 2^24");
    require(a->requests <= (1u << 20), "beam select: more than 2^20 requests");
    require(a->settle <= 1, "beam select: settle must be 0 or 1");
    require(a->settle == 0 || a->choices == a->beams, "beam select: settled choices must be as many as beams");
    if (a->requests == 0) {
        return;
    }
    require(a->logits != nullptr && a->scores != nullptr && a->out_scores != nullptr && a->parents != nullptr &&
                a->tokens != nullptr,
            "beam select: null argument");
    require(aligned_to(a->logits, type_bytes(a->type)) && aligned_to(a->scores, 4) && aligned_to(a->weights, 4) &&
                aligned_to(a->ended, 4) && aligned_to(a->out_scores, 4) && aligned_to(a->parents, 4) &&
                aligned_to(a->tokens, 4),
            "beam select: unaligned argument");
    require(a->out_scores != a->scores, "beam select: the scores out overlap the scores");
}

// ---- states that follow their parents -------------------------------------------

// arrays of a launch; few of them, so that its arguments are few bytes
constexpr uint32_t kArrays = 64, kFewArrays = 4;
constexpr uint32_t kReorderBlocks = 1u << 23;  // of a launch

struct RowArray {
    char *data;
    uint64_t request_stride, row_stride;  // bytes
    uint64_t units;        // of 16 bytes in a row
    uint64_t first_block;  // of the array's
    uint32_t blocks;       // of a request
    uint32_t tail;         // bytes behind them
};
template <uint32_t ARRAYS>
struct ReorderArgs {
    const uint32_t *parents;
    uint32_t arrays, beams;
    RowArray array[ARRAYS];
};

typedef uint32_t loose_u32x4 __attribute__((ext_vector_type(4), aligned(1)));

// 16 bytes of every row of a request, at any address, or one of the bytes behind
// them: the rows that others take are loaded, then stored where they go, so no order of
// the moves matters, and what stays is neither read nor written.
template <typename U, uint32_t K, uint32_t N>
__device__ __forceinline__ void reorder_units(char *base, uint64_t row_stride, const uint64_t (&takers)[K], uint64_t step,
                                              uint32_t count) {
    U v[K][N];
#pragma unroll
    for (uint32_t p = 0; p < K; ++p) {
        if (takers[p] != 0u) {
#pragma unroll
            for (uint32_t i = 0; i < N; ++i) {
                if (i < count) {
                    v[p][i] = *reinterpret_cast<const U *>(base + p * row_stride + i * step);
                }
            }
        }
    }
#pragma unroll
    for (uint32_t p = 0; p < K; ++p) {
        for (uint64_t left = takers[p]; left != 0u; left &= left - 1u) {
            char *const to = base + static_cast<uint32_t>(__builtin_ctzll(left)) * row_stride;
#pragma unroll
            for (uint32_t i = 0; i < N; ++i) {
                if (i < count) {
                    *reinterpret_cast<U *>(to + i * step) = v[p][i];
                }
            }
        }
    }
}

// Units of a row that a thread moves, a block's threads apart: as many as the
// registers hold, as rows lie far apart and one unit of each leaves most of the memory's
// channels idle (4 rows of 4 requests' 30 states, 1.05 GB: 254 us with one unit, 191
// with four, 5.5 TB/s; 8 rows 415 with one, 198 with two and with four; 16 213 and 205).
// More than 16 rows leave room for one (a request's 30 states, half of the rows moved:
// 16 rows 203 us, 17 463, 32 581, 64 939).
template <uint32_t K>
constexpr uint32_t kUnits = K <= 4u ? 4u : K <= 16u ? 2u : 1u;

template <uint32_t K, uint32_t ARRAYS>
__global__ __launch_bounds__(kThreads) void k_reorder_rows(ReorderArgs<ARRAYS> args) {
    uint32_t n = 0u;
    while (n + 1u < args.arrays && args.array[n + 1u].first_block <= blockIdx.x) {
        ++n;
    }
    const RowArray &array = args.array[n];
    const uint32_t at = static_cast<uint32_t>(blockIdx.x - array.first_block);
    const uint32_t request = at / array.blocks, block = at % array.blocks;
    const uint32_t lane = threadIdx.x & 63u;
    const uint32_t parent = lane < args.beams ? args.parents[static_cast<uint64_t>(request) * args.beams + lane] : kNone;
    // of each row, the other rows that take it (uniform)
    const bool moves = parent < args.beams && parent != lane;
    uint64_t takers[K];
#pragma unroll
    for (uint32_t p = 0; p < K; ++p) {
        takers[p] = __ballot(moves && parent == p);
    }
    constexpr uint32_t N = kUnits<K>;
    const uint64_t unit = static_cast<uint64_t>(block) * (N * kThreads) + threadIdx.x;
    char *const base = array.data + request * array.request_stride;
    if (unit < array.units) {
        const uint64_t more = (array.units - 1u - unit) / kThreads;
        reorder_units<loose_u32x4, K, N>(base + unit * 16u, array.row_stride, takers, 16u * kThreads,
                                         more < N ? static_cast<uint32_t>(more) + 1u : N);
    }
    if (block == 0u && threadIdx.x < array.tail) {
        reorder_units<uint8_t, K, 1>(base + array.units * 16u + threadIdx.x, array.row_stride, takers, 0u, 1u);
    }
}

// Blocks of a request's rows in an array.
uint64_t reorder_blocks(uint64_t row_bytes, uint32_t beams) {
    const uint64_t units = beams <= 4    ? kUnits<4>
                           : beams <= 8  ? kUnits<8>
                           : beams <= 16 ? kUnits<16>
                                         : kUnits<64>;
    return std::max<uint64_t>((row_bytes / 16u + kThreads * units - 1u) / (kThreads * units), 1u);
}

void require_reorder(const adi_hip_row_array *arrays, uint32_t count, uint32_t requests, uint32_t beams,
                     const uint32_t *parents) {
    require(beams >= 1 && beams <= kMaxBeams, "reorder rows: beams must be 1 to 64");
    require(requests <= (1u << 20), "reorder rows: more than 2^20 requests");
    require(count <= (1u << 16), "reorder rows: more than 65536 arrays");
    if (requests == 0 || count == 0) {
        return;
    }
    require(arrays != nullptr && parents != nullptr && aligned_to(parents, 4), "reorder rows: null or unaligned argument");
    for (uint32_t i = 0; i < count; ++i) {
        const adi_hip_row_array &a = arrays[i];
        require(a.row_bytes == 0 || a.data != nullptr, "reorder rows: null array");
        require(a.row_bytes < (1ull << 36) && a.row_stride < (1ull << 46) && a.request_stride < (1ull << 46),
                "reorder rows: rows must be below 2^36 bytes, strides below 2^46");
        require((beams == 1 || a.row_stride >= a.row_bytes) &&
                    (requests == 1 || a.request_stride >= (beams - 1) * a.row_stride + a.row_bytes ||
                     // (a product may pass 64 bits here)
                     (a.request_stride >= a.row_bytes && a.row_stride >= a.row_bytes &&
                      (a.row_stride - a.row_bytes) / (requests - 1) >= a.request_stride)),
                "reorder rows: an array's rows overlap");
        require(reorder_blocks(a.row_bytes, beams) * requests < kReorderBlocks,
                "reorder rows: too many rows of such a size");
    }
}

void reorder_rows(adi_hip_context *ctx, const adi_hip_row_array *arrays, uint32_t count, uint32_t requests,
                  uint32_t beams, const uint32_t *parents) {
    require_reorder(arrays, count, requests, beams, parents);
    if (requests == 0 || beams == 1) {
        return;
    }
    ReorderArgs<kArrays> args{parents, 0, beams, {}};
    uint64_t blocks = 0;
    const auto launch_of = [&](auto &&of) {
        constexpr uint32_t kOf = sizeof(of.array) / sizeof(RowArray);
        const dim3 grid(static_cast<uint32_t>(blocks)), block(kThreads);
        if (beams <= 4) {
            launch(ctx, "reorder_rows", k_reorder_rows<4, kOf>, grid, block, 0, of);
        } else if (beams <= 8) {
            launch(ctx, "reorder_rows", k_reorder_rows<8, kOf>, grid, block, 0, of);
        } else if (beams <= 16) {
            launch(ctx, "reorder_rows", k_reorder_rows<16, kOf>, grid, block, 0, of);
        } else {
            launch(ctx, "reorder_rows", k_reorder_rows<64, kOf>, grid, block, 0, of);
        }
    };
    const auto go = [&] {
        if (args.arrays > kFewArrays) {
            launch_of(args);
        } else if (args.arrays != 0) {
            ReorderArgs<kFewArrays> few{parents, args.arrays, beams, {}};
            std::copy_n(args.array, kFewArrays, few.array);
            launch_of(few);
        }
        args.arrays = 0;
        blocks = 0;
    };
    for (uint32_t i = 0; i < count; ++i) {
        const adi_hip_row_array &a = arrays[i];
        if (a.row_bytes == 0) {
            continue;
        }
        RowArray r{static_cast<char *>(a.data), a.request_stride, a.row_stride, a.row_bytes / 16, 0, 0,
                   static_cast<uint32_t>(a.row_bytes % 16)};
        const uint64_t per = reorder_blocks(a.row_bytes, beams);
        r.blocks = static_cast<uint32_t>(per);
        if (args.arrays == kArrays || blocks + per * requests >= kReorderBlocks) {
            go();
        }
        r.first_block = blocks;
        blocks += per * requests;
        args.array[args.arrays++] = r;
    }
    go();
}

}  // namespace
}  // namespace adi_hip

using namespace adi_hip;

extern "C" {

int adi_hip_beam_check(const adi_hip_beam_arguments *arguments) {
    return guarded_host([&] { require_select(arguments); });
}

int adi_hip_beam_select(adi_hip_context *ctx, const adi_hip_beam_arguments *arguments,
                        adi_hip_paged_workspace *workspace) {
    return guarded(ctx, [&] {
        require_select(arguments);
        require(workspace != nullptr, "beam select: null workspace");
        require(workspace->device == ctx->device, "beam select: the workspace is on another device");
        if (arguments->requests == 0) {
            return;
        }
        if (arguments->type == ADI_HIP_F32) {
            launch_select<float>(ctx, *arguments, *workspace);
        } else if (arguments->type == ADI_HIP_F16) {
            launch_select<_Float16>(ctx, *arguments, *workspace);
        } else {
            launch_select<__bf16>(ctx, *arguments, *workspace);
        }
    });
}

int adi_hip_reorder_check(const adi_hip_row_array *arrays, uint32_t count, uint32_t requests, uint32_t beams,
                          const uint32_t *parents) {
    return guarded_host([&] { require_reorder(arrays, count, requests, beams, parents); });
}

int adi_hip_reorder_rows(adi_hip_context *ctx, const adi_hip_row_array *arrays, uint32_t count, uint32_t requests,
                         uint32_t beams, const uint32_t *parents) {
    return guarded(ctx, [&] { reorder_rows(ctx, arrays, count, requests, beams, parents); });
}

}  // extern "C"
