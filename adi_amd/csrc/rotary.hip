// rotary.hip -- rotary positions for rows of any layout: the frequencies of a
// stretched context and the rotation of prepare_rope and apply_rope
// (src/executor.cpp:43-72) as an operator of its own.
//
// Dimensions a, b of a head that turn together become
//   a' = m (a cos t - b sin t),  b' = m (b cos t + a sin t),  t = position f,
// f the pair's frequency, m the scaling's magnitude. The angle of a far position
// takes more than 24 bits (262,143 f_0 leaves a float 0.016 radians), so it is
// formed and reduced in 64 (turn_of); sines, products and sums are 32 bits.
#include "paged.hpp"

namespace adi_hip {
namespace {

struct Frequencies {
    std::vector<double> radians;
    double magnitude;
};

// The frequencies of checked options (adi_hip.h gives the formulas).
Frequencies frequencies_of(const adi_hip_rope_options *o) {
    require(o != nullptr, "rope options are null");
    require(o->rotary >= 2 && o->rotary <= 1024 && o->rotary % 2 == 0, "rope: rotary must be even, 2 to 1024");
    require(o->layout <= ADI_HIP_ROPE_PAIRS, "rope: unknown layout");
    require(o->scaling <= ADI_HIP_ROPE_BANDS, "rope: unknown scaling");
    require(std::isfinite(o->theta) && o->theta > 1.0, "rope: theta must be above 1");
    // (the kernels' is a float)
    require(o->magnitude == 0.0 || (o->magnitude >= 0x1p-100 && o->magnitude <= 0x1p100),
            "rope: magnitude must be 2^-100 to 2^100, or 0");
    const bool stretched = o->scaling != ADI_HIP_ROPE_PLAIN;
    require(!stretched || (std::isfinite(o->factor) && o->factor >= 1.0), "rope: factor must be at least 1");
    const bool bounded = o->scaling == ADI_HIP_ROPE_YARN || o->scaling == ADI_HIP_ROPE_BANDS;
    double fast = o->fast, slow = o->slow;
    if (bounded) {
        require(std::isfinite(o->original) && o->original >= 1.0, "rope: original context must be at least 1");
        if (fast == 0.0 && slow == 0.0) {
            fast = o->scaling == ADI_HIP_ROPE_YARN ? 32.0 : 4.0;
            slow = 1.0;
        }
        require(std::isfinite(fast) && slow > 0.0 && fast > slow, "rope: fast must be above slow and slow above 0");
    }
    require(o->scaling != ADI_HIP_ROPE_NTK || o->rotary > 2, "rope: NTK scaling needs rotary above 2");
    const double rotary = o->rotary;
    double theta = o->theta;
    if (o->scaling == ADI_HIP_ROPE_NTK) {
        theta *= std::pow(o->factor, rotary / (rotary - 2.0));
    }
    constexpr double kTurn = 6.283185307179586476925286766559;
    const auto pair_of = [&](double turns) {
        return rotary * std::log(o->original / (kTurn * turns)) / (2.0 * std::log(theta));
    };
    double low = 0.0, high = 0.0;
    if (o->scaling == ADI_HIP_ROPE_YARN) {
        low = std::max(std::floor(pair_of(fast)), 0.0);
        high = std::min(std::ceil(pair_of(slow)), rotary - 1.0);
    }
    Frequencies out{{}, 1.0};
    out.radians.reserve(o->rotary / 2);
    for (uint32_t i = 0; i < o->rotary / 2; ++i) {
        double f = std::pow(theta, -2.0 * i / rotary);
        if (o->scaling == ADI_HIP_ROPE_LINEAR) {
            f /= o->factor;
        } else if (o->scaling == ADI_HIP_ROPE_YARN) {
            const double ramp = std::clamp((i - low) / std::max(high - low, 0.001), 0.0, 1.0);
            f = f * (1.0 - ramp) + f / o->factor * ramp;
        } else if (o->scaling == ADI_HIP_ROPE_BANDS) {
            const double keep = std::clamp((o->original * f / kTurn - slow) / (fast - slow), 0.0, 1.0);
            f = f * keep + f / o->factor * (1.0 - keep);
        }
        out.radians.push_back(f);
    }
    out.magnitude = o->magnitude != 0.0                    ? o->magnitude
                    : o->scaling == ADI_HIP_ROPE_YARN ? 0.1 * std::log(o->factor) + 1.0
                                                           : 1.0;
    return out;
}

constexpr uint32_t kThreads = 256;
constexpr uint32_t kMaxPairs = 512;

struct RopeArgs {
    RowsView in, out;
    const uint32_t *positions;
    const double *turns;
    uint32_t tokens, heads, pairs;  // pairs: rotary / 2
    uint32_t turn_units, copy_units, parts;
    float magnitude;
};

template <typename T, uint32_t N>
struct alignas(sizeof(T) * N) Vector {
    T v[N];
};

// Parts of a token's heads, a block each: the token's sines once a block into
// LDS, then units of N pairs (two reads and writes of N elements: 16 bytes each,
// or one element where a size, a stride or an address is not a multiple of 16
// bytes), and units of N dimensions behind them copied. Bound by the rows'
// bytes where there are many: 4,099 tokens of 32 heads of 128 in bf16, 67 MB,
// 13.6 us, 4.9 TB/s (a large copy: 5.1); by the launch where there are few (16
// tokens: 3.3 us). With sines per head and pair they would be the work (60
// instructions a pair).
template <typename T, uint32_t N, bool PAIRS>
__global__ __launch_bounds__(kThreads) void k_rope_rows(RopeArgs args) {
    __shared__ float2 wave[kMaxPairs];
    const uint32_t units = args.turn_units + args.copy_units;
    const uint64_t jobs = static_cast<uint64_t>(args.tokens) * args.parts;
    for (uint64_t job = blockIdx.x; job < jobs; job += gridDim.x) {
        const uint32_t token = static_cast<uint32_t>(job / args.parts);
        const uint32_t part = static_cast<uint32_t>(job % args.parts);
        const uint32_t position = args.positions[token];
        for (uint32_t i = threadIdx.x; i < args.pairs; i += kThreads) {
            const Turn turn = turn_of(position, args.turns[i]);
            wave[i] = make_float2(turn.cosine * args.magnitude, turn.sine * args.magnitude);
        }
        __syncthreads();
        const T *const from = reinterpret_cast<const T *>(args.in.data) + token * args.in.token_stride;
        T *const to = reinterpret_cast<T *>(args.out.data) + token * args.out.token_stride;
        const uint64_t items = static_cast<uint64_t>(args.heads) * units;
        for (uint64_t item = part * kThreads + threadIdx.x; item < items; item += args.parts * kThreads) {
            const uint32_t head = static_cast<uint32_t>(item / units), unit = static_cast<uint32_t>(item % units);
            const T *const x = from + head * args.in.head_stride;
            T *const y = to + head * args.out.head_stride;
            using V = Vector<T, N>;
            if (unit >= args.turn_units) {
                const uint32_t at = 2u * args.pairs + (unit - args.turn_units) * N;
                *reinterpret_cast<V *>(y + at) = *reinterpret_cast<const V *>(x + at);
                continue;
            }
            const uint32_t first = PAIRS ? 2u * unit * N : unit * N;
            const uint32_t second = PAIRS ? first + N : first + args.pairs;
            const V u = *reinterpret_cast<const V *>(x + first), v = *reinterpret_cast<const V *>(x + second);
            float p[N], q[N];
#pragma unroll
            for (uint32_t k = 0; k < N; ++k) {
                const float2 w = wave[unit * N + k];
                const auto element = [&](const V &lo, const V &hi, uint32_t i) { return i < N ? lo.v[i] : hi.v[i - N]; };
                const float a = static_cast<float>(PAIRS ? element(u, v, 2u * k) : u.v[k]);
                const float b = static_cast<float>(PAIRS ? element(u, v, 2u * k + 1u) : v.v[k]);
                const float turned_a = a * w.x - b * w.y, turned_b = b * w.x + a * w.y;
                if constexpr (PAIRS) {
                    (2u * k < N ? p[(2u * k) % N] : q[(2u * k) % N]) = turned_a;
                    (2u * k + 1u < N ? p[(2u * k + 1u) % N] : q[(2u * k + 1u) % N]) = turned_b;
                } else {
                    p[k] = turned_a;
                    q[k] = turned_b;
                }
            }
            store_values<T, N>(y + first, p);
            store_values<T, N>(y + second, q);
        }
        __syncthreads();
    }
}

template <typename T>
void launch_rope(adi_hip_context *ctx, RopeArgs args, uint32_t head_size, bool in_place, bool pairs, bool wide) {
    constexpr uint32_t kWide = 16u / sizeof(T);
    const uint32_t n = wide ? kWide : 1u;
    args.turn_units = args.pairs / n;
    args.copy_units = in_place ? 0u : (head_size - 2u * args.pairs) / n;
    const uint64_t items = static_cast<uint64_t>(args.heads) * (args.turn_units + args.copy_units);
    // few tokens: a block for every 256 units; many: one a token
    const uint64_t most = std::min<uint64_t>((items + kThreads - 1) / kThreads, 2048u);
    args.parts = static_cast<uint32_t>(std::clamp<uint64_t>(2048u / args.tokens, 1u, most));
    const uint64_t jobs = static_cast<uint64_t>(args.tokens) * args.parts;
    const dim3 grid(static_cast<uint32_t>(std::min<uint64_t>(jobs, 1u << 18)));
    if (wide) {
        launch(ctx, "rope_rows", pairs ? k_rope_rows<T, kWide, true> : k_rope_rows<T, kWide, false>, grid,
               dim3(kThreads), 0, args);
    } else {
        launch(ctx, "rope_rows", pairs ? k_rope_rows<T, 1, true> : k_rope_rows<T, 1, false>, grid, dim3(kThreads), 0,
               args);
    }
}

}  // namespace
}  // namespace adi_hip

using namespace adi_hip;

extern "C" {

int adi_hip_rope_frequencies(const adi_hip_rope_options *options, double *frequencies, double *magnitude) {
    return guarded_host([&] {
        const Frequencies f = frequencies_of(options);
        if (frequencies != nullptr) {
            std::copy(f.radians.begin(), f.radians.end(), frequencies);
        }
        if (magnitude != nullptr) {
            *magnitude = f.magnitude;
        }
    });
}

int adi_hip_rope_create(adi_hip_context *ctx, const adi_hip_rope_options *options, adi_hip_rope **out) {
    return guarded(ctx, [&] {
        require(out != nullptr, "rope: null output");
        *out = nullptr;
        Frequencies f = frequencies_of(options);
        for (double &v : f.radians) {
            v /= 6.283185307179586476925286766559;
        }
        double *turns = nullptr;
        const size_t bytes = f.radians.size() * sizeof(double);
        check_hip(hipMalloc(reinterpret_cast<void **>(&turns), bytes), "rope frequencies");
        const hipError_t error = hipMemcpy(turns, f.radians.data(), bytes, hipMemcpyHostToDevice);
        auto *rope = error == hipSuccess
                         ? new (std::nothrow) adi_hip_rope{ctx->device, options->rotary, options->layout,
                                                           static_cast<float>(f.magnitude), turns}
                         : nullptr;
        if (rope == nullptr) {
            (void)hipFree(turns);
            check_hip(error, "rope frequencies upload");
            throw std::bad_alloc();
        }
        *out = rope;
    });
}

void adi_hip_rope_destroy(adi_hip_rope *rope) {
    if (rope == nullptr) {
        return;
    }
    int previous = 0;
    (void)hipGetDevice(&previous);
    (void)hipSetDevice(rope->device);
    (void)hipDeviceSynchronize();
    (void)hipFree(rope->turns);
    (void)hipSetDevice(previous);
    delete rope;
}

int adi_hip_rope_rows(adi_hip_context *ctx, const adi_hip_rope *rope, const adi_hip_rows *input, uint32_t tokens,
                      uint32_t heads, uint32_t head_size, const uint32_t *positions, const adi_hip_rows *output) {
    return guarded(ctx, [&] {
        require(rope != nullptr && input != nullptr && output != nullptr, "rope rows: null argument");
        require(rope->device == ctx->device, "rope rows: the frequencies are on another device");
        require(heads >= 1 && head_size >= rope->rotary && head_size <= 65536,
                "rope rows: heads and head size do not hold the rotary dimensions");
        require(known_type(input->type) && input->type == output->type, "rope rows: unknown or different types");
        if (tokens == 0) {
            return;
        }
        const uint32_t bytes = type_bytes(input->type);
        require(positions != nullptr && aligned_to(positions, 4) && input->data != nullptr && output->data != nullptr &&
                    aligned_to(input->data, bytes) && aligned_to(output->data, bytes),
                "rope rows: null or unaligned array");
        const bool in_place = same_rows(*input, *output);
        require(in_place || input->data != output->data, "rope rows: the output overlaps the input");
        const uint32_t n = 16u / bytes;
        const auto even = [&](const adi_hip_rows &rows) {
            return aligned_to(rows.data, 16) && rows.token_stride % n == 0 && rows.head_stride % n == 0;
        };
        const bool wide = even(*input) && even(*output) && head_size % n == 0 && rope->rotary / 2 % n == 0;
        const RopeArgs args{rows_view(*input), rows_view(*output), positions, rope->turns, tokens, heads,
                            rope->rotary / 2, 0, 0, 0, rope->magnitude};
        const bool pairs = rope->layout == ADI_HIP_ROPE_PAIRS;
        if (input->type == ADI_HIP_F32) {
            launch_rope<float>(ctx, args, head_size, in_place, pairs, wide);
        } else if (input->type == ADI_HIP_F16) {
            launch_rope<_Float16>(ctx, args, head_size, in_place, pairs, wide);
        } else {
            launch_rope<__bf16>(ctx, args, head_size, in_place, pairs, wide);
        }
    });
}

}  // extern "C"
