// pkv_q8_decode.cu -- decode attention over 8-bit pages (one query token per
// sequence).
//
//   o = sum_t softmax_t(scale q . k_t) v_t,   k_t = kq_t ks,  v_t = vq_t vs
//
// with one scale per (page, KV head): q . k_t = ks (q . kq_t), so the scales
// multiply a score and a softmax weight, never an element.  One CTA per
// (sequence, KV head); each warp takes every eighth token and keeps a running
// maximum, sum and output per query head, merged over the warps at the end.
#include <math.h>

#include "pkv_q8.cuh"
#include "pkv_trace.h"

namespace pkv {
namespace {

__device__ uint32_t g_q8_decode_fault;

constexpr float kLog2e = 1.4426950408889634f;
constexpr size_t kQ8MaxGroup = 16;

struct Q8DecodeArgs {
    const int8_t *kpool, *vpool;
    const float *kscales, *vscales;
    const uint32_t *tables;
    const int32_t *seq_lens;
    const void *query;
    void *out;
    int32_t table_stride, kv_heads, lanes, block_size, group;
    uint32_t block_count;
    float scale_log2;
};

template <int HD, int GM, typename T, typename OT>
__global__ void __launch_bounds__(256) q8_decode_kernel(const Q8DecodeArgs a) {
    constexpr int E = HD / 32;  // columns per thread
    __shared__ float ms[8][GM], ls[8][GM];
    __shared__ float os[8][HD];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int g = blockIdx.x, b = blockIdx.y;
    const int L = max(0, __ldg(a.seq_lens + b));
    const int q_heads = a.kv_heads * a.group;
    const int64_t qrow = ((int64_t)b * q_heads + (int64_t)g * a.group) * HD;
    float q[GM][E], acc[GM][E], m[GM], l[GM];
#pragma unroll
    for (int h = 0; h < GM; ++h) {
        m[h] = -INFINITY;
        l[h] = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            acc[h][e] = 0.f;
            q[h][e] = h < a.group ? (float)static_cast<const T *>(a.query)[qrow + h * HD + lane * E + e] *
                                        a.scale_log2
                                  : 0.f;
        }
    }
    const int col = g * HD;
    for (int t = warp; t < L; t += 8) {
        const int page = t / a.block_size;
        uint32_t fault = kFaultNone, pid = 0;
        if (page >= a.table_stride) fault = kFaultPositionOutOfRange;
        else if ((pid = __ldg(a.tables + (int64_t)b * a.table_stride + page)) >= a.block_count)
            fault = kFaultPageOutOfRange;
        if (fault != kFaultNone) {
            if (lane == 0) record_fault(&g_q8_decode_fault, fault);
            continue;
        }
        const int64_t at = (((int64_t)pid * a.lanes + col / 128) * a.block_size +
                            (t - page * a.block_size)) * 128 + col % 128 + lane * E;
        const float ks = __ldg(a.kscales + (int64_t)pid * a.kv_heads + g);
        const float vs = __ldg(a.vscales + (int64_t)pid * a.kv_heads + g);
        float k[E], v[E];
#pragma unroll
        for (int e = 0; e < E; ++e) {
            k[e] = (float)a.kpool[at + e] * ks;
            v[e] = (float)a.vpool[at + e] * vs;
        }
#pragma unroll
        for (int h = 0; h < GM; ++h) {
            float s = 0.f;
#pragma unroll
            for (int e = 0; e < E; ++e) s = fmaf(q[h][e], k[e], s);
            s = warp_sum(s);
            const float mn = fmaxf(m[h], s);
            const float al = exp2f(m[h] - mn), p = exp2f(s - mn);
            m[h] = mn;
            l[h] = l[h] * al + p;
#pragma unroll
            for (int e = 0; e < E; ++e) acc[h][e] = acc[h][e] * al + p * v[e];
        }
    }
    OT *out = static_cast<OT *>(a.out) + qrow;
    if (lane == 0)
        for (int h = 0; h < GM; ++h) {
            ms[warp][h] = m[h];
            ls[warp][h] = l[h];
        }
    __syncthreads();
#pragma unroll
    for (int h = 0; h < GM; ++h) {
        if (h < a.group) {
            float mx = -INFINITY, lt = 0.f;
            for (int w = 0; w < 8; ++w) mx = fmaxf(mx, ms[w][h]);
            for (int w = 0; w < 8; ++w) lt += ls[w][h] > 0.f ? ls[w][h] * exp2f(ms[w][h] - mx) : 0.f;
            const float f = l[h] > 0.f ? exp2f(m[h] - mx) / lt : 0.f;
#pragma unroll
            for (int e = 0; e < E; ++e) os[warp][lane * E + e] = acc[h][e] * f;
        }
        __syncthreads();
        if (h < a.group && threadIdx.x < HD) {
            float o = 0.f;
            for (int w = 0; w < 8; ++w) o += os[w][threadIdx.x];
            out[h * HD + threadIdx.x] = from_f32<OT>(o);
        }
        __syncthreads();
    }
}

template <int HD, typename T, typename OT>
void launch(const Q8DecodeArgs &a, int batch, cudaStream_t s) {
    const dim3 grid(a.kv_heads, batch);
    if (a.group <= 4) q8_decode_kernel<HD, 4, T, OT><<<grid, 256, 0, s>>>(a);
    else q8_decode_kernel<HD, 16, T, OT><<<grid, 256, 0, s>>>(a);
}

template <typename T>
void dispatch(const Q8DecodeArgs &a, int batch, size_t hd, PkvDType out, cudaStream_t s) {
    if (out == PKV_DTYPE_F32)
        hd == 128 ? launch<128, T, float>(a, batch, s) : launch<64, T, float>(a, batch, s);
    else
        hd == 128 ? launch<128, T, T>(a, batch, s) : launch<64, T, T>(a, batch, s);
}

}  // namespace
}  // namespace pkv

extern "C" {

size_t pkv_q8_decode_workspace_bytes(size_t batch, size_t q_heads, size_t kv_heads,
                                     size_t head_dim, size_t max_seq_len) {
    return 256;
}

int pkv_q8_decode(const PkvQ8Layer *layer, const PkvBatch *batch, size_t q_heads,
                  const void *query, float scale, void *output, PkvDType output_dtype,
                  size_t max_seq_len, void *workspace, size_t workspace_bytes, PkvStream stream,
                  char *error, size_t error_capacity) {
    PKV_RANGE("pkv_q8_decode");
    const char *what = "pkv_q8_decode";
    if (!pkv::q8_check(layer, batch, error, error_capacity, what)) return 0;
    if (query == nullptr || output == nullptr) {
        pkv_internal_set_error(error, error_capacity, "%s: null argument", what);
        return 0;
    }
    if (output_dtype != PKV_DTYPE_F32 && output_dtype != layer->dtype) {
        pkv_internal_set_error(error, error_capacity,
                               "%s: output dtype must be F32 or the row dtype", what);
        return 0;
    }
    if (q_heads == 0 || q_heads % layer->kv_heads != 0 ||
        q_heads / layer->kv_heads > pkv::kQ8MaxGroup) {
        pkv_internal_set_error(error, error_capacity,
                               "%s: q_heads must be 1..%zu times kv_heads", what,
                               pkv::kQ8MaxGroup);
        return 0;
    }
    pkv::Q8DecodeArgs a;
    a.kpool = layer->key_pool;
    a.vpool = layer->value_pool;
    a.kscales = layer->key_scales;
    a.vscales = layer->value_scales;
    a.tables = batch->block_tables;
    a.seq_lens = batch->seq_lens;
    a.query = query;
    a.out = output;
    a.table_stride = (int32_t)batch->table_stride;
    a.kv_heads = (int32_t)layer->kv_heads;
    a.lanes = (int32_t)pkv::q8_lanes(layer->kv_heads, layer->head_dim);
    a.block_size = (int32_t)layer->block_size;
    a.group = (int32_t)(q_heads / layer->kv_heads);
    a.block_count = (uint32_t)layer->block_count;
    a.scale_log2 = scale * pkv::kLog2e;
    const cudaStream_t s = (cudaStream_t)stream;
    if (layer->dtype == PKV_DTYPE_F16)
        pkv::dispatch<__half>(a, (int)batch->batch, layer->head_dim, output_dtype, s);
    else
        pkv::dispatch<__nv_bfloat16>(a, (int)batch->batch, layer->head_dim, output_dtype, s);
    const cudaError_t st = cudaGetLastError();
    if (st != cudaSuccess) {
        pkv_internal_set_error(error, error_capacity, "%s: launch failed: %s", what,
                               cudaGetErrorString(st));
        return 0;
    }
    return 1;
}

int pkv_internal_take_q8_decode_fault(uint32_t *code) {
    uint32_t zero = 0;
    if (cudaMemcpyFromSymbol(code, pkv::g_q8_decode_fault, sizeof(uint32_t)) != cudaSuccess)
        return 0;
    return cudaMemcpyToSymbol(pkv::g_q8_decode_fault, &zero, sizeof(uint32_t)) == cudaSuccess;
}

}  // extern "C"
