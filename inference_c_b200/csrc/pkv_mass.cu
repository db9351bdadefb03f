// pkv_mass.cu -- attention weights of a decode step, added to the paged mass
// (float32 [block_count][kv_heads][block_size]).
//
// One warp takes one tile of 128 tokens of one lane (one KV head of head_dim
// 128, two of 64): thread = 4 tokens, a 16-byte load per query head, eight of
// them in flight, one read and write of the tokens' cells per KV head.  Each
// cell belongs to one thread, so sums do not depend on any order of CTAs.
// Bound by HBM: 4 bytes a token and query head (mostly L2 hits, just written)
// and 8 bytes a token and KV head.  One load of 4 bytes a step took 27 us for
// 131072 tokens of 64 heads.
#include "pkv_device.cuh"
#include "pkv_mass.cuh"
#include "pkv_trace.h"

namespace pkv {
namespace {

__device__ uint32_t g_mass_fault;

constexpr int kTiles = 8;  // tiles (warps) of a CTA

struct MassArgs {
    const float *scores;
    const float *final_ml;
    const int32_t *tile_prefix;
    const uint32_t *tables;
    const int32_t *seq_lens;
    float *mass;
    int64_t tiles;
    int32_t max_len;  // longer sequences add nothing; the decode recorded the fault
    int32_t table_stride, kv_heads, q_heads, group, block_size, gv, per, subs, segs;
    uint32_t block_count;
};

template <bool PAIR>
__global__ void __launch_bounds__(kTiles * 32) mass_kernel(const MassArgs a) {
    pdl_launch_dependents();
    pdl_wait();
    const int lane = blockIdx.y, b = blockIdx.z;
    const int L = max(0, __ldg(a.seq_lens + b));
    const int k = blockIdx.x * kTiles + (threadIdx.x >> 5);
    const int t = k * 128 + (threadIdx.x & 31) * 4;  // this thread's first token
    if (t >= L || L > a.max_len) return;
    // the decode's tiles of this sequence
    const int64_t first = __ldcg(a.tile_prefix + b);
    const int nt = (__ldcg(a.tile_prefix + b + 1) - (int)first) / a.segs;
    const int page = t / a.block_size;  // its 4 tokens share a page
    uint32_t pid = 0, fault = kFaultNone;
    if (page >= a.table_stride) fault = kFaultPositionOutOfRange;
    else if ((pid = __ldg(a.tables + (int64_t)b * a.table_stride + page)) >= a.block_count)
        fault = kFaultPageOutOfRange;
    else if (nt != (L + 127) / 128 || first + (int64_t)a.segs * nt > a.tiles)
        // not the lengths of the decode
        fault = kFaultPositionOutOfRange;
    if (fault != kFaultNone) {
        record_fault(&g_mass_fault, fault);
        return;
    }
#pragma unroll
    for (int half = 0; half < (PAIR ? 2 : 1); ++half) {
        const int kvh = PAIR ? 2 * lane + half : lane;
        if (kvh >= a.kv_heads) return;
        float4 *cell = reinterpret_cast<float4 *>(
            a.mass + ((int64_t)pid * a.kv_heads + kvh) * a.block_size + (t - page * a.block_size));
        const float4 old = *cell;
        float4 w = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int h0 = 0; h0 < a.group; h0 += 8) {
            float4 x[8];
            float2 ml[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int hh = min(h0 + i, a.group - 1);
                const int sub = hh / a.per, h = hh - sub * a.per + half * a.per;
                const int64_t tile = first + (int64_t)(lane * a.subs + sub) * nt + k;
                x[i] = __ldcg(reinterpret_cast<const float4 *>(a.scores + (tile * a.gv + h) * 128) +
                              (threadIdx.x & 31));
                ml[i] = __ldcg(reinterpret_cast<const float2 *>(
                    a.final_ml + ((int64_t)b * a.q_heads + kvh * a.group + hh) * 2));
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                if (h0 + i >= a.group) break;
                const float inv = ml[i].y == 0.f ? 0.f : 1.f / ml[i].y;
                w.x += exp2f(x[i].x - ml[i].x) * inv;
                w.y += exp2f(x[i].y - ml[i].x) * inv;
                w.z += exp2f(x[i].z - ml[i].x) * inv;
                w.w += exp2f(x[i].w - ml[i].x) * inv;
            }
        }
        // the last tokens one by one: cells past the length stay as they are
        if (t + 4 <= L) {
            *cell = make_float4(old.x + w.x, old.y + w.y, old.z + w.z, old.w + w.w);
        } else {
            float *c = reinterpret_cast<float *>(cell);
            c[0] = old.x + w.x;
            if (t + 1 < L) c[1] = old.y + w.y;
            if (t + 2 < L) c[2] = old.z + w.z;
        }
    }
}

// Zeroes the cells of every sequence's last n_b positions: one warp a sequence
// and KV head, thread = position.
__global__ void __launch_bounds__(128)
mass_clear_kernel(const uint32_t *tables, const int32_t *seq_lens, const int32_t *offsets,
                  float *mass, int table_stride, int block_size, uint32_t block_count,
                  int kv_heads, int batch) {
    pdl_launch_dependents();
    pdl_wait();
    const int g = blockIdx.y * 4 + (threadIdx.x >> 5), b = blockIdx.x;
    if (g >= kv_heads) return;
    const int L = __ldg(seq_lens + b);
    const int n = offsets == nullptr ? 1 : __ldg(offsets + b + 1) - __ldg(offsets + b);
    if (n > L) {
        record_fault(&g_mass_fault, kFaultRowsMismatch);
        return;
    }
    for (int t = L - n + (int)(threadIdx.x & 31); t < L; t += 32) {
        const int page = t / block_size;
        uint32_t pid = 0, fault = kFaultNone;
        if (page >= table_stride) fault = kFaultPositionOutOfRange;
        else if ((pid = __ldg(tables + (int64_t)b * table_stride + page)) >= block_count)
            fault = kFaultPageOutOfRange;
        if (fault != kFaultNone) record_fault(&g_mass_fault, fault);
        else mass[((int64_t)pid * kv_heads + g) * block_size + (t - page * block_size)] = 0.f;
    }
}

}  // namespace

bool mass_apply(const MassShape &s, const MassScratch &scratch, const int32_t *tile_prefix,
                const uint32_t *tables, const int32_t *seq_lens, float *mass, PkvStream stream) {
    const bool pair = s.head_dim == 64;
    MassArgs a;
    a.scores = scratch.scores;
    a.final_ml = scratch.final_ml;
    a.tile_prefix = tile_prefix;
    a.tables = tables;
    a.seq_lens = seq_lens;
    a.mass = mass;
    a.max_len = (int32_t)s.max_seq_len;
    a.tiles = scratch.tiles;
    a.table_stride = (int32_t)s.table_stride;
    a.kv_heads = (int32_t)s.kv_heads;
    a.q_heads = (int32_t)s.q_heads;
    a.group = (int32_t)(s.q_heads / s.kv_heads);
    a.block_size = (int32_t)s.block_size;
    a.gv = (int32_t)s.gv;
    a.per = (int32_t)(pair ? s.gv / 2 : s.gv);
    a.subs = (int32_t)s.subs;
    const size_t lanes = mass_lanes(s.kv_heads, s.head_dim);
    a.segs = (int32_t)(lanes * s.subs);
    a.block_count = (uint32_t)s.block_count;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    const size_t tiles = (s.max_seq_len + 127) / 128;
    cfg.gridDim = dim3((unsigned)((tiles + kTiles - 1) / kTiles), (unsigned)lanes,
                       (unsigned)s.batch);
    cfg.blockDim = dim3(kTiles * 32);
    cfg.stream = (cudaStream_t)stream;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (tiles == 0) return true;
    const cudaError_t st = pair ? cudaLaunchKernelEx(&cfg, mass_kernel<true>, a)
                                : cudaLaunchKernelEx(&cfg, mass_kernel<false>, a);
    return st == cudaSuccess && cudaGetLastError() == cudaSuccess;
}

}  // namespace pkv

extern "C" int pkv_mass_clear(size_t block_size, size_t block_count, size_t kv_heads,
                              const PkvBatch *batch, const int32_t *row_offsets, float *mass,
                              PkvStream stream, char *error, size_t error_capacity) {
    PKV_RANGE("pkv_mass_clear");
    const char *what = "pkv_mass_clear";
    if (batch == nullptr || mass == nullptr || batch->block_tables == nullptr ||
        batch->seq_lens == nullptr || (uintptr_t)mass % 4 != 0) {
        pkv_internal_set_error(error, error_capacity, "%s: null argument or misaligned mass", what);
        return 0;
    }
    if (block_size == 0 || block_size > INT32_MAX || block_count == 0 ||
        block_count > UINT32_MAX || kv_heads == 0 || kv_heads > 1024 || batch->batch == 0 ||
        batch->batch > INT32_MAX / 4 || batch->table_stride == 0 ||
        batch->table_stride > INT32_MAX) {
        pkv_internal_set_error(error, error_capacity, "%s: invalid shape", what);
        return 0;
    }
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)batch->batch, (unsigned)((kv_heads + 3) / 4));
    cfg.blockDim = dim3(128);
    cfg.stream = (cudaStream_t)stream;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    cudaError_t st = cudaLaunchKernelEx(
        &cfg, pkv::mass_clear_kernel, batch->block_tables, batch->seq_lens, row_offsets, mass,
        (int)batch->table_stride, (int)block_size, (uint32_t)block_count, (int)kv_heads,
        (int)batch->batch);
    if (st == cudaSuccess) st = cudaGetLastError();
    if (st != cudaSuccess) {
        pkv_internal_set_error(error, error_capacity, "%s: launch failed: %s", what,
                               cudaGetErrorString(st));
        return 0;
    }
    return 1;
}

extern "C" int pkv_internal_take_mass_fault(uint32_t *code) {
    uint32_t zero = 0;
    if (cudaMemcpyFromSymbol(code, pkv::g_mass_fault, sizeof(uint32_t)) != cudaSuccess) return 0;
    return cudaMemcpyToSymbol(pkv::g_mass_fault, &zero, sizeof(uint32_t)) == cudaSuccess;
}
