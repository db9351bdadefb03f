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

// The checks every entry point over 8-bit pages makes on its shapes (eviction
// of 16-bit pages too), and on its layer and batch (host; no device work).
// They write the reason and return false.
inline bool page_shape_check(size_t bs, size_t block_count, size_t kv_heads, size_t head_dim,
                             PkvDType dtype, const PkvBatch *batch, char *error, size_t cap,
                             const char *what) {
    if (dtype != PKV_DTYPE_F16 && dtype != PKV_DTYPE_BF16) {
        pkv_internal_set_error(error, cap, "%s: row dtype must be F16 or BF16", what);
        return false;
    }
    if ((bs != 16 && bs != 32 && bs != 64 && bs != 128) || (head_dim != 64 && head_dim != 128) ||
        kv_heads == 0 || kv_heads > 1024) {
        pkv_internal_set_error(error, cap,
                               "%s: pages hold 16, 32, 64 or 128 tokens of 1..1024 KV heads of "
                               "head_dim 64 or 128",
                               what);
        return false;
    }
    if (block_count == 0 || block_count > UINT32_MAX || batch->batch == 0 ||
        batch->batch > INT32_MAX / 4 || batch->table_stride == 0 ||
        batch->table_stride > INT32_MAX / bs) {
        pkv_internal_set_error(error, cap, "%s: invalid block count, batch or table stride", what);
        return false;
    }
    return true;
}
inline bool pool_check(const void *key_pool, const void *value_pool, const PkvBatch *batch,
                       char *error, size_t cap, const char *what) {
    if (batch == nullptr || key_pool == nullptr || value_pool == nullptr ||
        batch->block_tables == nullptr || batch->seq_lens == nullptr) {
        pkv_internal_set_error(error, cap, "%s: null argument", what);
        return false;
    }
    if (((uintptr_t)key_pool | (uintptr_t)value_pool) % 16 != 0) {
        pkv_internal_set_error(error, cap, "%s: pools must be 16-byte aligned", what);
        return false;
    }
    return true;
}
inline bool q8_check(const PkvQ8Layer *layer, const PkvBatch *batch, char *error, size_t cap,
                     const char *what) {
    if (layer == nullptr || layer->key_scales == nullptr || layer->value_scales == nullptr) {
        pkv_internal_set_error(error, cap, "%s: null argument", what);
        return false;
    }
    if (((uintptr_t)layer->key_scales | (uintptr_t)layer->value_scales) % 4 != 0) {
        pkv_internal_set_error(error, cap, "%s: scales must be 4-byte aligned", what);
        return false;
    }
    return pool_check(layer->key_pool, layer->value_pool, batch, error, cap, what) &&
           page_shape_check(layer->block_size, layer->block_count, layer->kv_heads,
                            layer->head_dim, layer->dtype, batch, error, cap, what);
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
