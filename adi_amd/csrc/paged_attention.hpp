// paged_attention.hpp -- the paged cache's append and attention for the
// package's own layers.
#pragma once

#include "paged.hpp"

// Tickets first, then the parts of histories.
struct adi_hip_paged_workspace {
    int device;
    void *base;
    size_t bytes;
};

namespace adi_hip {

constexpr uint32_t kTickets = 1u << 16;  // words, zero between calls

// adi_hip_paged_append; with `sines` the rotation of halves is taken from a
// table [position][sines_half cosines, sines_half sines] instead of a->rope.
void paged_append(adi_hip_context *ctx, const adi_hip_paged_cache *cache, const adi_hip_paged_batch *batch,
                  const adi_hip_paged_append_arguments *a, const float *sines, uint32_t sines_half);

// What adi_hip_paged_attention checks besides its rows, for a caller that has work
// of its own to do before it.
void require_attention(const adi_hip_context *ctx, const adi_hip_paged_cache *cache, const adi_hip_paged_batch *batch,
                       uint32_t query_heads, const adi_hip_paged_workspace *workspace);

void paged_attention(adi_hip_context *ctx, const adi_hip_paged_cache *cache, const adi_hip_paged_batch *batch,
                     const adi_hip_paged_attention_arguments *a, adi_hip_paged_workspace *workspace);

}  // namespace adi_hip
