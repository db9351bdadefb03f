// pkv_mass.cuh -- adding a decode's attention weights to the paged mass.
//
// The decode kernels see a token's weight only relative to the running
// maximum; they leave every score (log2 units) in scratch, by tile of the
// work stream, and each query head's final maximum and sum.  This pass turns
// them into weights exp2(x - m) / l, sums the query heads of a KV head and
// adds the sum to the token's cell.
#pragma once

#include <stddef.h>
#include <stdint.h>

#include "pkv_internal.h"

namespace pkv {

struct MassScratch {
    float *scores;    // [tiles][gv slots][128]
    float *final_ml;  // [batch][q_heads][m, l]
    int64_t tiles;    // tiles `scores` holds
};

struct MassShape {
    size_t batch, q_heads, kv_heads, head_dim, block_size, block_count, table_stride, max_seq_len;
    size_t gv, subs;  // slots of a segment, segments of a lane
};

// Most sequences of one decode launch (1024 over 16-bit pages, 512 over 8-bit
// ones: the schedule's prefix lives in shared memory), so also of a mass pass.
constexpr size_t kMassBatch = 1024;

inline size_t mass_lanes(size_t kv_heads, size_t head_dim) {
    return (kv_heads * head_dim + 127) / 128;
}
inline size_t mass_scratch_bytes(size_t batch, size_t q_heads, size_t segs, size_t gv,
                                 size_t max_seq_len) {
    const size_t n = batch < kMassBatch ? batch : kMassBatch;
    const size_t ml = (n * q_heads * 8 + 255) / 256 * 256;
    return ml + n * segs * ((max_seq_len + 127) / 128) * gv * 512;
}
inline MassScratch mass_scratch(void *at, size_t batch, size_t q_heads, size_t segs,
                                size_t max_seq_len) {
    const size_t n = batch < kMassBatch ? batch : kMassBatch;
    MassScratch s;
    s.final_ml = static_cast<float *>(at);
    s.scores = reinterpret_cast<float *>(static_cast<unsigned char *>(at) +
                                         (n * q_heads * 8 + 255) / 256 * 256);
    s.tiles = (int64_t)(n * segs * ((max_seq_len + 127) / 128));
    return s;
}

// Adds one launch's weights (stream order: after the decode and its merge).
bool mass_apply(const MassShape &shape, const MassScratch &scratch, const int32_t *tile_prefix,
                const uint32_t *tables, const int32_t *seq_lens, float *mass, PkvStream stream);

}  // namespace pkv
