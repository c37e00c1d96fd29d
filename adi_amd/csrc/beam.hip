// beam.hip -- a step of a beam search: the best candidates of every request over
// its beams and the vocabulary, and per-beam states that follow their parents.
//
// Selection: a beam of score s whose logits are l has the candidates
//   s + (l_v - lse),  lse = m + log sum_v exp(l_v - m),
// and a request takes the best of its beams'. One pass over the logits: a block
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

using u32x4 = uint32_t __attribute__((ext_vector_type(4)));

struct BeamArgs {
    const char *logits;
    uint64_t request_stride, beam_stride;  // elements
    uint32_t beams, vocabulary, choices, parts;
    const float *scores, *weights;
    const uint32_t *ended;
    uint32_t ended_token, settle;
    float *out_scores;
    uint32_t *parents, *tokens;
    // of each row's tiles: largest logit, sum of exp(logit - largest), best logits
    float *most;
    double *sum;
    uint64_t *best;
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

__device__ __forceinline__ float wave_most(float v) {
    v = fmaxf(v, lane_xor<1>(v));
    v = fmaxf(v, lane_xor<2>(v));
    v = fmaxf(v, lane_xor<4>(v));
    v = fmaxf(v, lane_xor<8>(v));
    v = fmaxf(v, lane_xor<16>(v));
    return fmaxf(v, lane_xor<32>(v));
}

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
    for (int offset = 1; offset < 64; offset <<= 1) {
        v += __shfl_xor(v, offset);
    }
    return v;
}

// The largest key that at least `count` (1 to 64) of the wave's lanes reach.
__device__ __forceinline__ uint32_t reached_by(uint32_t key, uint32_t count) {
    uint32_t reached = 0u;
#pragma unroll 1
    for (uint32_t bit = 0x80000000u; bit != 0u; bit >>= 1) {
        const uint32_t more = reached | bit;
        reached = static_cast<uint32_t>(__popcll(__ballot(key >= more))) >= count ? more : reached;
    }
    return reached;
}

// A tile of kThreads x N logits of a row. Its best: every wave's lanes hold their
// own largest logits, of which the choices / 4 best bound the tile's `choices` best
// from below; what reaches the least of the waves' bounds goes to a list in LDS,
// a little more than `choices` long, and each entry's place is the number of
// entries before it. Where many are equal (a masked run of ids) the list may not
// hold them, and the last taken is found bit by bit.
template <typename T, uint32_t N>
__global__ __launch_bounds__(kThreads) void k_beam_tiles(BeamArgs args) {
    constexpr uint32_t kCount = Piece<T>::kCount, kPieces = N / kCount, kTile = kThreads * N;
    constexpr uint32_t kList = 512;
    __shared__ uint64_t list[kList];
    __shared__ uint32_t listed, bound[kWaves];
    __shared__ float wave_top[kWaves];
    __shared__ double wave_total[kWaves];
    const uint32_t row = blockIdx.x / args.parts, part = blockIdx.x % args.parts;
    const float score = args.scores[row];
    if (score == -__builtin_huge_valf() || (args.ended != nullptr && args.ended[row] != 0u)) {
        return;
    }
    const uint32_t t = threadIdx.x, wave = t / kWave;
    const uint32_t first = part * kTile, live = min(args.vocabulary - first, kTile);
    const char *const from = args.logits + (row / args.beams * args.request_stride +
                                            row % args.beams * args.beam_stride + first) * sizeof(T);
    if (t == 0u) {
        listed = 0u;
    }
    Piece<T> x[kPieces];
    if (live == kTile) {
#pragma unroll
        for (uint32_t j = 0; j < kPieces; ++j) {
            x[j].load(from + (j * kThreads + t) * 16u);
        }
    } else {
#pragma unroll
        for (uint32_t j = 0; j < kPieces; ++j) {
            const uint32_t at = (j * kThreads + t) * kCount;
            if (at + kCount <= live) {
                x[j].load(from + at * sizeof(T));
            } else {
#pragma unroll
                for (uint32_t i = 0; i < kCount; ++i) {
                    T v = static_cast<T>(-__builtin_huge_valf());
                    if (at + i < live) {
                        v = reinterpret_cast<const T *>(from)[at + i];
                    }
                    x[j].set(i, v);
                }
            }
        }
    }
    float own = -__builtin_huge_valf();
#pragma unroll
    for (uint32_t j = 0; j < kPieces; ++j) {
#pragma unroll
        for (uint32_t i = 0; i < kCount; ++i) {
            own = fmaxf(own, x[j].get(i));
        }
    }
    const float top = wave_most(own);
    // (nothing but -infinity: all of its exponentials are 0)
    const double level = top == -__builtin_huge_valf() ? 0.0 : static_cast<double>(top);
    double total = 0.0;
#pragma unroll
    for (uint32_t j = 0; j < kPieces; ++j) {
#pragma unroll
        for (uint32_t i = 0; i < kCount; ++i) {
            total += exp(static_cast<double>(x[j].get(i)) - level);
        }
    }
    total = wave_sum(total);
    const uint32_t reached = reached_by(ascending_key(own), (args.choices + kWaves - 1u) / kWaves);
    if ((t & 63u) == 0u) {
        bound[wave] = reached;
        wave_top[wave] = top;
        wave_total[wave] = total;
    }
    __syncthreads();
    const uint32_t least = max(min(min(bound[0], bound[1]), min(bound[2], bound[3])), kLowestKey + 1u);
    const auto place_of = [&](uint32_t j, uint32_t i) { return (j * kThreads + t) * kCount + i; };
#pragma unroll
    for (uint32_t j = 0; j < kPieces; ++j) {
#pragma unroll
        for (uint32_t i = 0; i < kCount; ++i) {
            const uint32_t key = ascending_key(x[j].get(i));
            if (key >= least) {
                const uint32_t at = atomicAdd(&listed, 1u);
                if (at < kList) {
                    list[at] = static_cast<uint64_t>(key) << 32 | static_cast<uint32_t>(~(first + place_of(j, i)));
                }
            }
        }
    }
    __syncthreads();
    uint32_t entries = listed;
    if (entries > kList) {
        // the last taken, in the order of the keys and then of the places
        uint64_t last = 0u;
        constexpr uint32_t kPlaceBits = 13;
        static_assert(kTile <= 1u << kPlaceBits, "a tile's places fit their bits");
        const auto whole = [&](uint32_t j, uint32_t i) {
            return static_cast<uint64_t>(ascending_key(x[j].get(i))) << kPlaceBits |
                   ((1u << kPlaceBits) - 1u - place_of(j, i));
        };
#pragma unroll 1
        for (uint64_t bit = 1ull << (31u + kPlaceBits); bit != 0u; bit >>= 1) {
            const uint64_t more = last | bit;
            uint32_t reach = 0u;
#pragma unroll
            for (uint32_t j = 0; j < kPieces; ++j) {
#pragma unroll
                for (uint32_t i = 0; i < kCount; ++i) {
                    reach += static_cast<uint32_t>(__popcll(__ballot(whole(j, i) >= more)));
                }
            }
            __syncthreads();  // the last round's bounds are read
            if ((t & 63u) == 0u) {
                bound[wave] = reach;
            }
            __syncthreads();
            last = bound[0] + bound[1] + bound[2] + bound[3] >= args.choices ? more : last;
        }
        if (t == 0u) {
            listed = 0u;
        }
        __syncthreads();
#pragma unroll
        for (uint32_t j = 0; j < kPieces; ++j) {
#pragma unroll
            for (uint32_t i = 0; i < kCount; ++i) {
                const uint32_t key = ascending_key(x[j].get(i));
                if (key >= least && whole(j, i) >= last) {
                    list[atomicAdd(&listed, 1u)] =
                        static_cast<uint64_t>(key) << 32 | static_cast<uint32_t>(~(first + place_of(j, i)));
                }
            }
        }
        __syncthreads();
        entries = listed;  // `choices` of them
    }
    uint64_t *const best = args.best + static_cast<uint64_t>(blockIdx.x) * args.choices;
    for (uint32_t e = t; e < entries; e += kThreads) {
        const uint64_t key = list[e];
        uint32_t before = 0u;
        for (uint32_t o = 0; o < entries; ++o) {
            before += list[o] > key ? 1u : 0u;
        }
        if (before < args.choices) {
            best[before] = key;
        }
    }
    for (uint32_t e = entries + t; e < args.choices; e += kThreads) {
        best[e] = 0u;
    }
    if (t == 0u) {
        float most = -__builtin_huge_valf();
        for (uint32_t w = 0; w < kWaves; ++w) {
            most = fmaxf(most, wave_top[w]);
        }
        double sum = 0.0;
        for (uint32_t w = 0; w < kWaves; ++w) {
            sum += wave_top[w] == -__builtin_huge_valf()
                       ? wave_total[w]
                       : wave_total[w] * exp(static_cast<double>(wave_top[w]) - static_cast<double>(most));
        }
        args.most[blockIdx.x] = most;
        args.sum[blockIdx.x] = sum;
    }
}

struct Candidate {
    double rank;
    uint64_t key;   // its logit's key, then ~token; 0: none
    uint32_t beam;
};

// The order of candidates: rank, then the lower beam, then the larger logit, then
// the lower token.
__device__ __forceinline__ bool precedes(const Candidate &a, const Candidate &b) {
    return a.rank != b.rank ? a.rank > b.rank : a.beam != b.beam ? a.beam < b.beam : a.key > b.key;
}

// Joins a request's tiles.
__global__ __launch_bounds__(kThreads) void k_beam_join(BeamArgs args) {
    constexpr uint32_t kList = 1024;
    __shared__ double lse[kMaxBeams], score[kMaxBeams], weight[kMaxBeams];
    __shared__ uint32_t kind[kMaxBeams];  // 0: no candidates, 1: its logits', 2: ended
    __shared__ Candidate list[kList];
    __shared__ Candidate taken[kMaxChoices];
    __shared__ uint32_t listed, bad, bound[kWaves];
    const uint32_t t = threadIdx.x, lane = t & 63u, wave = t / kWave, request = blockIdx.x;
    const uint32_t k = args.beams, choices = args.choices, of_beam = args.parts * choices;
    if (t == 0u) {
        listed = 0u;
        bad = 0u;
    }
    for (uint32_t i = t; i < choices; i += kThreads) {
        taken[i].key = 0u;
        taken[i].beam = kNone;
    }
    __syncthreads();
    for (uint32_t b = wave; b < k; b += kWaves) {
        const uint32_t row = request * k + b;
        const float s = args.scores[row], w = args.weights != nullptr ? args.weights[row] : 1.0f;
        uint32_t what = s == -__builtin_huge_valf() ? 0u : args.ended != nullptr && args.ended[row] != 0u ? 2u : 1u;
        bool wrong = what != 0u && !(__builtin_isfinite(s) && w > 0.0f && __builtin_isfinite(w));
        double normal = 0.0;
        if (what == 1u) {
            const float *const most = args.most + static_cast<uint64_t>(row) * args.parts;
            const double *const sum = args.sum + static_cast<uint64_t>(row) * args.parts;
            float top = -__builtin_huge_valf();
            for (uint32_t p = lane; p < args.parts; p += kWave) {
                top = fmaxf(top, most[p]);
            }
            top = wave_most(top);
            double total = 0.0;
            for (uint32_t p = lane; p < args.parts; p += kWave) {
                total += most[p] == -__builtin_huge_valf()
                             ? sum[p]
                             : sum[p] * exp(static_cast<double>(most[p]) - static_cast<double>(top));
            }
            total = wave_sum(total);
            // a NaN or +infinity among the logits leaves a NaN in the sum
            wrong = wrong || total != total;
            what = top == -__builtin_huge_valf() ? 0u : what;
            normal = static_cast<double>(top) + log(total);
        }
        if (lane == 0u) {
            lse[b] = normal;
            score[b] = s;
            weight[b] = w;
            kind[b] = what;
            if (wrong) {
                bad = 1u;
            }
        }
    }
    __syncthreads();
    float *const out_scores = args.out_scores + static_cast<uint64_t>(request) * choices;
    uint32_t *const parents = args.parents + static_cast<uint64_t>(request) * choices;
    uint32_t *const tokens = args.tokens + static_cast<uint64_t>(request) * choices;
    if (bad != 0u) {
        for (uint32_t i = t; i < choices; i += kThreads) {
            out_scores[i] = __builtin_nanf("");
            parents[i] = kNone;
            tokens[i] = kNone;
        }
        return;
    }
    const uint64_t *const best = args.best + static_cast<uint64_t>(request) * k * of_beam;
    // candidate i: of the tiles' lists, then one of each ended beam
    const uint32_t candidates = k * of_beam + k;
    const auto candidate = [&](uint32_t i) {
        Candidate c{0.0, 0u, 0u};
        if (i < k * of_beam) {
            c.beam = i / of_beam;
            if (kind[c.beam] == 1u) {
                c.key = best[i];
                const double logit = of_ascending_key(static_cast<uint32_t>(c.key >> 32));
                c.rank = (score[c.beam] + (logit - lse[c.beam])) * weight[c.beam];
            }
        } else {
            c.beam = i - k * of_beam;
            if (kind[c.beam] == 2u) {
                c.key = ~0ull;
                c.rank = score[c.beam] * weight[c.beam];
            }
        }
        return c;
    };
    // of the rank: ascending with it, equal for ranks next to each other
    const auto coarse = [](const Candidate &c) {
        const uint64_t bits = __builtin_bit_cast(uint64_t, c.rank + 0.0);
        const uint32_t high = static_cast<uint32_t>(bits >> 32);
        return c.key == 0u ? 0u : high ^ ((high & 0x80000000u) != 0u ? 0xFFFFFFFFu : 0x80000000u);
    };
    uint32_t own = 0u;
    for (uint32_t i = t; i < candidates; i += kThreads) {
        own = max(own, coarse(candidate(i)));
    }
    const uint32_t reached = reached_by(own, (choices + kWaves - 1u) / kWaves);
    if (lane == 0u) {
        bound[wave] = reached;
    }
    __syncthreads();
    const uint32_t least = max(min(min(bound[0], bound[1]), min(bound[2], bound[3])), 1u);
    for (uint32_t i = t; i < candidates; i += kThreads) {
        const Candidate c = candidate(i);
        if (coarse(c) >= least) {
            const uint32_t at = atomicAdd(&listed, 1u);
            if (at < kList) {
                list[at] = c;
            }
        }
    }
    __syncthreads();
    const uint32_t entries = listed;
    if (entries <= kList) {
        for (uint32_t e = t; e < entries; e += kThreads) {
            const Candidate c = list[e];
            uint32_t before = 0u;
            for (uint32_t o = 0; o < entries; ++o) {
                before += precedes(list[o], c) ? 1u : 0u;
            }
            if (before < choices) {
                taken[before] = c;
            }
        }
    } else {
        // so many near each other: one after another
        for (uint32_t n = 0; n < choices; ++n) {
            Candidate next{0.0, 0u, 0u};
            for (uint32_t i = t; i < candidates; i += kThreads) {
                const Candidate c = candidate(i);
                if (c.key != 0u && (n == 0u || precedes(taken[n - 1u], c)) && (next.key == 0u || precedes(c, next))) {
                    next = c;
                }
            }
            list[t] = next;
            __syncthreads();
            if (t == 0u) {
                for (uint32_t o = 1; o < kThreads; ++o) {
                    if (list[o].key != 0u && (next.key == 0u || precedes(list[o], next))) {
                        next = list[o];
                    }
                }
                if (next.key != 0u) {
                    taken[n] = next;
                }
            }
            __syncthreads();
            if (taken[n].key == 0u) {
                break;
            }
        }
    }
    __syncthreads();
    uint64_t children = 0u;  // beams with one
    if (args.settle != 0u) {
        for (uint32_t i = 0; i < choices; ++i) {
            children |= taken[i].key != 0u ? 1ull << taken[i].beam : 0u;
        }
    }
    for (uint32_t i = t; i < choices; i += kThreads) {
        const Candidate c = taken[i];
        uint32_t place = i;
        if (args.settle != 0u) {
            // the parent's row for its first child; the others' rows, and those of
            // places without a candidate, are the rows without one, in turn
            const auto is_first = [&](uint32_t n) {
                bool first = taken[n].key != 0u;
                for (uint32_t o = 0; o < n; ++o) {
                    first = first && taken[o].beam != taken[n].beam;
                }
                return first;
            };
            if (is_first(i)) {
                place = c.beam;
            } else {
                uint32_t nth = 0u;
                for (uint32_t o = 0; o < i; ++o) {
                    nth += is_first(o) ? 0u : 1u;
                }
                uint64_t rows = ~children;
                for (; nth != 0u; --nth) {
                    rows &= rows - 1u;
                }
                place = static_cast<uint32_t>(__builtin_ctzll(rows));
            }
        }
        const bool some = c.key != 0u;
        const double logit = of_ascending_key(static_cast<uint32_t>(c.key >> 32));
        double value = -__builtin_huge_val();
        if (some) {
            value = kind[c.beam] == 2u ? score[c.beam] : score[c.beam] + (logit - lse[c.beam]);
        }
        out_scores[place] = static_cast<float>(value);
        parents[place] = some ? c.beam : kNone;
        tokens[place] = !some ? kNone : kind[c.beam] == 2u ? args.ended_token : ~static_cast<uint32_t>(c.key);
    }
}

template <typename T>
void launch_select(adi_hip_context *ctx, const adi_hip_beam_arguments &a, const adi_hip_paged_workspace &workspace) {
    constexpr uint32_t N = 32;
    BeamArgs args{static_cast<const char *>(a.logits), a.request_stride, a.beam_stride, a.beams, a.vocabulary,
                  a.choices, ceil_div(a.vocabulary, kThreads * N), a.scores, a.weights, a.ended, a.ended_token, a.settle,
                  a.out_scores, a.parents, a.tokens, nullptr, nullptr, nullptr};
    // as many requests at once as the workspace holds
    const uint64_t tiles = uint64_t(a.beams) * args.parts;
    const uint64_t bytes = tiles * (sizeof(double) + sizeof(uint64_t) * a.choices + sizeof(float));
    const uint64_t room = workspace.bytes - kTickets * sizeof(uint32_t);
    const uint64_t at_once = std::min<uint64_t>({room / bytes, a.requests, (1u << 23) / tiles});
    if (at_once == 0) {
        fail(ADI_HIP_OUT_OF_MEMORY, "beam select: a request needs a workspace of " +
                                        std::to_string(bytes + kTickets * sizeof(uint32_t)) + " bytes");
    }
    char *const base = static_cast<char *>(workspace.base) + kTickets * sizeof(uint32_t);
    args.sum = reinterpret_cast<double *>(base);
    args.best = reinterpret_cast<uint64_t *>(args.sum + at_once * tiles);
    args.most = reinterpret_cast<float *>(args.best + at_once * tiles * a.choices);
    for (uint64_t done = 0; done < a.requests; done += at_once) {
        const uint32_t requests = static_cast<uint32_t>(std::min<uint64_t>(at_once, a.requests - done));
        launch(ctx, "beam_tiles", k_beam_tiles<T, N>, dim3(static_cast<uint32_t>(requests * tiles)), dim3(kThreads), 0,
               args);
        launch(ctx, "beam_join", k_beam_join, dim3(requests), dim3(kThreads), 0, args);
        args.logits += requests * args.request_stride * sizeof(T);
        args.scores += requests * a.beams;
        args.weights += args.weights != nullptr ? requests * a.beams : 0;
        args.ended += args.ended != nullptr ? requests * a.beams : 0;
        args.out_scores += requests * a.choices;
        args.parents += requests * a.choices;
        args.tokens += requests * a.choices;
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

constexpr uint32_t kArrays = 64;  // of a launch

struct RowArray {
    char *data;
    uint64_t request_stride, row_stride;  // bytes
    uint64_t row_units;
    uint64_t first_block;  // of the array's
    uint32_t blocks;       // of a request
    uint32_t unit;         // bytes
};
struct ReorderArgs {
    RowArray array[kArrays];
    uint32_t arrays, beams;
    const uint32_t *parents;
};

// One unit of every row of a request a thread: the rows that others take are
// loaded, then stored where they go, so no order of the moves matters, and what
// stays is neither read nor written.
template <typename U, uint32_t K>
__device__ __forceinline__ void reorder_units(const RowArray &array, uint32_t request, uint32_t block, uint32_t beams,
                                              const uint32_t *parents) {
    const uint32_t lane = threadIdx.x & 63u;
    const uint32_t parent = lane < beams ? parents[static_cast<uint64_t>(request) * beams + lane] : kNone;
    // of each row, the other rows that take it (uniform)
    const bool moves = parent < beams && parent != lane;
    uint64_t takers[K];
#pragma unroll
    for (uint32_t p = 0; p < K; ++p) {
        takers[p] = __ballot(moves && parent == p);
    }
    const uint64_t unit = static_cast<uint64_t>(block) * kThreads + threadIdx.x;
    if (unit >= array.row_units) {
        return;
    }
    char *const base = array.data + request * array.request_stride + unit * sizeof(U);
    U v[K];
#pragma unroll
    for (uint32_t p = 0; p < K; ++p) {
        if (takers[p] != 0u) {
            v[p] = *reinterpret_cast<const U *>(base + p * array.row_stride);
        }
    }
#pragma unroll
    for (uint32_t p = 0; p < K; ++p) {
        for (uint64_t left = takers[p]; left != 0u; left &= left - 1u) {
            *reinterpret_cast<U *>(base + static_cast<uint32_t>(__builtin_ctzll(left)) * array.row_stride) = v[p];
        }
    }
}

template <uint32_t K>
__global__ __launch_bounds__(kThreads) void k_reorder_rows(ReorderArgs args) {
    uint32_t n = 0u;
    while (n + 1u < args.arrays && args.array[n + 1u].first_block <= blockIdx.x) {
        ++n;
    }
    const RowArray &array = args.array[n];
    const uint32_t at = static_cast<uint32_t>(blockIdx.x - array.first_block);
    const uint32_t request = at / array.blocks, block = at % array.blocks;
    if (array.unit == 16u) {
        reorder_units<u32x4, K>(array, request, block, args.beams, args.parents);
    } else if (array.unit == 4u) {
        reorder_units<uint32_t, K>(array, request, block, args.beams, args.parents);
    } else {
        reorder_units<uint8_t, K>(array, request, block, args.beams, args.parents);
    }
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
                     (a.request_stride >= a.row_bytes && a.row_stride >= (requests - 1) * a.request_stride + a.row_bytes)),
                "reorder rows: an array's rows overlap");
    }
}

void reorder_rows(adi_hip_context *ctx, const adi_hip_row_array *arrays, uint32_t count, uint32_t requests,
                  uint32_t beams, const uint32_t *parents) {
    require_reorder(arrays, count, requests, beams, parents);
    if (requests == 0 || beams == 1) {
        return;
    }
    ReorderArgs args{};
    args.beams = beams;
    args.parents = parents;
    uint64_t blocks = 0;
    const auto go = [&] {
        if (args.arrays != 0) {
            const dim3 grid(static_cast<uint32_t>(blocks)), block(kThreads);
            if (beams <= 4) {
                launch(ctx, "reorder_rows", k_reorder_rows<4>, grid, block, 0, args);
            } else if (beams <= 16) {
                launch(ctx, "reorder_rows", k_reorder_rows<16>, grid, block, 0, args);
            } else {
                launch(ctx, "reorder_rows", k_reorder_rows<64>, grid, block, 0, args);
            }
        }
        args.arrays = 0;
        blocks = 0;
    };
    for (uint32_t i = 0; i < count; ++i) {
        const adi_hip_row_array &a = arrays[i];
        if (a.row_bytes == 0) {
            continue;
        }
        const uint64_t all = reinterpret_cast<uintptr_t>(a.data) | a.row_stride | a.request_stride | a.row_bytes;
        RowArray r{static_cast<char *>(a.data), a.request_stride, a.row_stride, 0, 0, 0, 0};
        r.unit = all % 16 == 0 ? 16 : all % 4 == 0 ? 4 : 1;
        r.row_units = a.row_bytes / r.unit;
        const uint64_t per = (r.row_units + kThreads - 1) / kThreads;
        require(per * requests < (1u << 23), "reorder rows: too many rows of such a size");
        r.blocks = static_cast<uint32_t>(per);
        if (args.arrays == kArrays || blocks + per * requests >= (1u << 23)) {
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
