// pkv_q8.cuh -- what the kernels over 8-bit pages share: the page layout and
// the quantisation rule.
//
// A page holds, for each lane (128 columns of a token's row, one KV head of
// head_dim 128 or two of head_dim 64), block_size rows of 128 int8 values
// back to back, so one (page, lane) is one contiguous run (2 KiB at 16
// tokens) and a head's pages stream at full lines.  value = q * scale, one
// FP32 scale per (page, KV head):  s = max|x| / 127,  q = rint(x / s).
#pragma once

#include "pkv_device.cuh"
#include "pkv_internal.h"

namespace pkv {

constexpr int kQ8Lane = 128;               // columns (and bytes) of one lane row
constexpr float kQ8MinScale = 1.17549435e-38f;  // 2^-126: below, a block stores zeros

enum : uint32_t { kFaultNotFinite = 5 };   // a NaN or infinity was stored in 8 bits

inline size_t q8_lanes(size_t kv_heads, size_t head_dim) {
    return (kv_heads * head_dim + kQ8Lane - 1) / kQ8Lane;
}

// The checks every entry point over 8-bit pages makes on its layer and batch
// (host; no device work).  Writes the reason and returns false.
inline bool q8_check(const PkvQ8Layer *layer, const PkvBatch *batch, char *error, size_t cap,
                     const char *what) {
    if (layer == nullptr || batch == nullptr || layer->key_pool == nullptr ||
        layer->value_pool == nullptr || layer->key_scales == nullptr ||
        layer->value_scales == nullptr || batch->block_tables == nullptr ||
        batch->seq_lens == nullptr) {
        pkv_internal_set_error(error, cap, "%s: null argument", what);
        return false;
    }
    if (layer->dtype != PKV_DTYPE_F16 && layer->dtype != PKV_DTYPE_BF16) {
        pkv_internal_set_error(error, cap, "%s: row dtype must be F16 or BF16", what);
        return false;
    }
    const size_t bs = layer->block_size;
    if ((bs != 16 && bs != 32 && bs != 64 && bs != 128) ||
        (layer->head_dim != 64 && layer->head_dim != 128) || layer->kv_heads == 0 ||
        layer->kv_heads > 1024) {
        pkv_internal_set_error(error, cap,
                               "%s: 8-bit pages hold 16, 32, 64 or 128 tokens of 1..1024 KV heads "
                               "of head_dim 64 or 128",
                               what);
        return false;
    }
    if (layer->block_count == 0 || layer->block_count > UINT32_MAX || batch->batch == 0 ||
        batch->batch > INT32_MAX / 4 || batch->table_stride == 0 ||
        batch->table_stride > INT32_MAX / bs) {
        pkv_internal_set_error(error, cap, "%s: invalid block count, batch or table stride", what);
        return false;
    }
    if (((uintptr_t)layer->key_pool | (uintptr_t)layer->value_pool) % 16 != 0 ||
        ((uintptr_t)layer->key_scales | (uintptr_t)layer->value_scales) % 4 != 0) {
        pkv_internal_set_error(error, cap,
                               "%s: pools must be 16-byte aligned, scales 4-byte aligned", what);
        return false;
    }
    return true;
}

// Four int8 values of a word, as floats.
__device__ __forceinline__ void q8_unpack4(uint32_t w, float (&f)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = (float)(int)(int8_t)(w >> (8 * i));
}
__device__ __forceinline__ uint32_t q8_pack4(const int (&q)[4]) {
    return (uint32_t)(q[0] & 255) | (uint32_t)(q[1] & 255) << 8 | (uint32_t)(q[2] & 255) << 16 |
           (uint32_t)q[3] << 24;
}
// rint, kept in [-127, 127]; NaN -> 0.
__device__ __forceinline__ int q8_round(float x) {
    return __float2int_rn(fminf(fmaxf(x == x ? x : 0.f, -127.f), 127.f));
}

}  // namespace pkv
