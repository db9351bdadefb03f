// pkv_q8_copy.cu -- rows into 8-bit pages (append, prefix import) and back
// (gather).
//
// One unit is one (page of a sequence, lane, K or V); block_size / 16 warps
// share it, each holding 16 rows x 128 columns in registers (thread: 8
// columns of every second row), so every value crosses the bus once.  Append
// and import: the largest |x| of the page's new rows of each head is reduced
// over the warps, the scale follows, and the rows leave as 8-byte stores, two
// whole 128-byte rows a warp instruction.  A page that holds earlier tokens
// keeps its scale unless the new rows need a larger one; then its earlier
// tokens are rescaled, q' = rint(q * (s_old / s)), by the threads that own
// those rows.  Bound by HBM: 2 bytes read and 1 written a value (gather the
// reverse).
//
// Prefill expands the batch's pages to 16-bit rows in its workspace, once, and
// runs the paged prefill kernel on them: a chunk's pages are read by every
// 128-row query tile and head pair, so widening them inside the attention
// kernel would repeat each conversion that many times, while the expansion is
// one pass of 3 bytes a value.  The rows it writes are the whole numbers q, exact
// in either 16-bit type (bf16 V rows of very small or large scales: times a power
// of two); the scales go beside them and enter the exponent.
#include <math.h>

#include <type_traits>

#include "pkv_q8.cuh"
#include "pkv_trace.h"

namespace pkv {
namespace {

__device__ uint32_t g_q8_copy_fault;

constexpr int kQ8Warps = 8;  // per CTA

struct Q8RowArgs {
    uint2 *pools[2];          // K, V: [pages][lanes][block][16] eight-byte groups
    float *scales[2];         // [pages][kv_heads]
    uint4 *rows[2];           // [total_rows][kv_width / 8]
    const uint32_t *tables;
    const int32_t *seq_lens;
    const int32_t *offsets;   // null: one row per sequence
    int32_t table_stride, batch, kv_heads, lanes, block_size;
    uint32_t block_count;
    int32_t units;            // upper bound of pages touched
    int32_t total_rows;       // of the contiguous buffers
    int32_t row_vecs;         // uint4 per contiguous row
    int32_t tail;             // rows are the sequence's last (append) or first positions
    // > 0: every sequence's first seq_lens[b] rows go to rows b * pad_rows on as
    // whole numbers, their scales per 16 rows to `wide` (PkvRowScales);
    // table_out gets the identity table of those rows in pages of 128 and
    // lens_out the lengths, 0 for a sequence longer than max_len
    int32_t pad_rows;
    uint32_t *table_out;
    int32_t *lens_out;
    int32_t max_len;
    float *wide_k, *wide_log2, *wide_inverse;
};

// Largest |x| of 64 values, as a float; NaN if one is not a number.
template <typename T>
__device__ __forceinline__ float abs_max(const uint4 (&x)[8]);
template <>
__device__ __forceinline__ float abs_max<__half>(const uint4 (&x)[8]) {
    __half2 m = __float2half2_rn(0.f);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const __half2 *h = reinterpret_cast<const __half2 *>(&x[i]);
#pragma unroll
        for (int k = 0; k < 4; ++k) m = __hmax2_nan(m, __habs2(h[k]));
    }
    const float2 f = __half22float2(m);
    return f.x != f.x ? f.x : (f.y != f.y ? f.y : fmaxf(f.x, f.y));
}
template <>
__device__ __forceinline__ float abs_max<__nv_bfloat16>(const uint4 (&x)[8]) {
    __nv_bfloat162 m = __float2bfloat162_rn(0.f);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const __nv_bfloat162 *h = reinterpret_cast<const __nv_bfloat162 *>(&x[i]);
#pragma unroll
        for (int k = 0; k < 4; ++k) m = __hmax2_nan(m, __habs2(h[k]));
    }
    const float2 f = __bfloat1622float2(m);
    return f.x != f.x ? f.x : (f.y != f.y ? f.y : fmaxf(f.x, f.y));
}

// rint(x * inv) of four finite values within +-127 as the bytes of a word.
// Adding 1.5 * 2^23 rounds to a whole number, ties to even, and leaves it in
// two's complement in the sum's low bits: no conversion, whose unit takes a
// quarter of a warp a cycle.
__device__ __forceinline__ uint32_t q8_quantise4(float a, float b, float c, float d, float inv) {
    constexpr float kRound = 12582912.f;
    const uint32_t w = __float_as_uint(__fadd_rn(__fmul_rn(a, inv), kRound));
    const uint32_t x = __float_as_uint(__fadd_rn(__fmul_rn(b, inv), kRound));
    const uint32_t y = __float_as_uint(__fadd_rn(__fmul_rn(c, inv), kRound));
    const uint32_t z = __float_as_uint(__fadd_rn(__fmul_rn(d, inv), kRound));
    return __byte_perm(__byte_perm(w, x, 0x0040), __byte_perm(y, z, 0x0040), 0x5410);
}

// Sequence b touches at most floor((n_b - 1) / block) + 2 pages, so giving it
// the units from floor(offsets[b] / block) + 2 b on needs no scan: unit u
// belongs to the last sequence whose first unit is <= u.
__device__ __forceinline__ int32_t q8_first_unit(const Q8RowArgs &a, int b) {
    return __ldg(a.offsets + b) / a.block_size + 2 * b;
}

// WRITE: rows -> pages.  Otherwise pages -> rows.
template <typename T, int HD, bool WRITE>
__global__ void __launch_bounds__(kQ8Warps * 32)
q8_rows_kernel(const Q8RowArgs a) {
    pdl_launch_dependents();
    pdl_wait();
    __shared__ float top[kQ8Warps][2];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int per = a.block_size / 16;              // warps of one unit
    const int u = blockIdx.x * (kQ8Warps / per) + warp / per;
    const int part = warp % per;                    // this warp's 16 rows of the page
    const int kv = blockIdx.y & 1;
    constexpr int kHeads = 128 / HD;                // heads of a lane
    const int chunk = lane & 15;                    // this thread's 8 columns
    const int hl = HD == 64 ? chunk >> 3 : 0;       // its head within the lane

    // ---- which page ----
    bool live = u < a.units;
    const bool unit_live = u < a.units;
    int b = 0;
    int32_t first = 0, end = 0, row0 = 0, page = 0;
    bool held = false;
    uint32_t pid = 0;
    if (unit_live) {
        int32_t count = 1, slot = 0;
        if (!WRITE && a.pad_rows > 0) {
            const int per_seq = a.pad_rows / a.block_size;
            b = u / per_seq;
            slot = u - b * per_seq;
            row0 = b * a.pad_rows;
            count = max(0, __ldg(a.seq_lens + b));
            if (blockIdx.y == 0 && part == 0 && lane == 0 && slot * a.block_size % 128 == 0) {
                const int at = (row0 + slot * a.block_size) / 128;
                a.table_out[at] = (uint32_t)at;
            }
            if (count > a.max_len) {  // longer than the caller's bound
                if (lane == 0) record_fault(&g_q8_copy_fault, kFaultPositionOutOfRange);
                count = 0;
            }
            if (blockIdx.y == 0 && part == 0 && lane == 0 && slot == 0) a.lens_out[b] = count;
        } else if (a.offsets == nullptr) {
            b = u;
            row0 = u;
        } else {
            // the warp tries 32 sequences at a time: one round of loads up to 32
            int lo = 0, n = a.batch;  // the answer is in [lo, lo + n)
            while (n > 1) {
                const int step = (n + 31) / 32, at = lo + min(lane * step, n - 1);
                const uint32_t below = __ballot_sync(0xffffffffu, q8_first_unit(a, at) <= u);
                const int k = max(0, 31 - __clz(below));
                lo += min(k * step, n - 1);
                n = min(step, a.batch - lo);
                if (step == 1) break;
            }
            b = lo;
            row0 = __ldg(a.offsets + b);
            count = __ldg(a.offsets + b + 1) - row0;
            slot = u - q8_first_unit(a, b);  // below 0: before offsets[0], nobody's
        }
        const int32_t L = !WRITE && a.pad_rows > 0 ? count : __ldg(a.seq_lens + b);
        uint32_t fault = kFaultNone;
        first = a.tail ? L - count : 0;
        end = first + count;
        page = first / a.block_size + slot;
        // more rows than the sequence has, or offsets outside the buffers
        const bool bad = count > L || row0 < 0 || row0 > a.total_rows - count;
        if (bad && count > 0) fault = slot == 0 ? kFaultRowsMismatch : kFaultNone;
        if (bad || count <= 0 || slot < 0 || (int64_t)page * a.block_size >= end) live = false;
        if (live) {
            if (page >= a.table_stride) fault = kFaultPositionOutOfRange;
            else {
                pid = __ldg(a.tables + (int64_t)b * a.table_stride + page);
                if (pid >= a.block_count) fault = kFaultPageOutOfRange;
            }
        }
        if (fault != kFaultNone) {
            if (lane == 0) record_fault(&g_q8_copy_fault, fault);
            live = false;
        }
        held = page * a.block_size < first;
    }
    // the page's columns, a lane at a time: one lookup serves several
    for (int col_lane = blockIdx.y >> 1; col_lane < a.lanes; col_lane += gridDim.y >> 1) {
        const int head = col_lane * kHeads + hl;
        // ---- the page's rows: i-th is row part*16 + 2 i + lane/16 ----
        const bool on = live && head < a.kv_heads;
        const int64_t base = (((int64_t)pid * a.lanes + col_lane) * a.block_size + part * 16 + (lane >> 4)) * 16 + chunk;
        uint2 *cell = a.pools[kv] + base;
        float *sp = a.scales[kv] + (int64_t)pid * a.kv_heads + head;
        const int32_t pos0 = page * a.block_size + part * 16 + (lane >> 4);
        uint4 *row = a.rows[kv] + ((int64_t)row0 + (pos0 - first)) * a.row_vecs + col_lane * 16 + chunk;

        if constexpr (!WRITE) {
            float s = on ? __ldg(sp) : 1.f;
            if (a.pad_rows > 0) {
                // A block of zeros, or none.  Its weights meet zeros of V and only
                // enter the softmax sum, in FP32, but they also enter the maximum
                // that the others are relative to: 2^-31 is below every scale of
                // fp16 rows, whose weights would else run out of fp16's exponents
                // (V near 1e-3 beside one block of zeros).
                float t = s != 0.f ? s : kv == 0 ? 1.f : 4.65661287e-10f;
                s = 1.f;
                if (kv == 1 && std::is_same<T, __nv_bfloat16>::value) {
                    // bf16 rows have scales from 2^-126 to 2^121, and a weight times a
                    // scale 2^-100 of another's would leave FP32 and with it the
                    // softmax sum: beyond 2^-31 .. 2^31 a power of two goes into the
                    // rows, whose whole numbers bf16 holds exactly with it.
                    const int e = (int)(__float_as_uint(t) >> 23 & 255u) - 127;
                    const int j = e < -31 ? e + 31 : e > 31 ? e - 31 : 0;
                    s = __uint_as_float((uint32_t)(127 + j) << 23);
                    t *= __uint_as_float((uint32_t)(127 - j) << 23);
                }
                if (unit_live && head < a.kv_heads && (lane == 0 || (HD == 64 && lane == 8))) {
                    const int64_t at = ((int64_t)b * a.kv_heads + head) * (a.pad_rows / 16) +
                                       (page * a.block_size) / 16 + part;
                    if (kv == 0) a.wide_k[at] = t;
                    else {
                        a.wide_log2[at] = log2f(t);
                        a.wide_inverse[at] = __fdiv_rn(1.f, t);
                    }
                }
            }
            if (!on) continue;
            uint2 q[8];
#pragma unroll
            for (int i = 0; i < 8; ++i)
                q[i] = pos0 + 2 * i < end ? __ldg(cell + i * 32) : make_uint2(0, 0);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                if (pos0 + 2 * i >= end) continue;
                float lo[4], hi[4];
                q8_unpack4(q[i].x, lo);
                q8_unpack4(q[i].y, hi);
                T o[8];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    o[k] = from_f32<T>(lo[k] * s);
                    o[4 + k] = from_f32<T>(hi[k] * s);
                }
                row[(int64_t)i * 2 * a.row_vecs] = *reinterpret_cast<uint4 *>(o);
            }
            continue;
        }

        uint4 x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int32_t p = pos0 + 2 * i;
            x[i] = on && p >= first && p < end ? __ldg(row + (int64_t)i * 2 * a.row_vecs)
                                                 : make_uint4(0, 0, 0, 0);
        }
        float m = abs_max<T>(x);
        const bool odd = !(m < INFINITY);  // a NaN or an infinity among them
        if (odd) {
            record_fault(&g_q8_copy_fault, kFaultNotFinite);
            m = 0.f;
#pragma unroll 1
            for (int i = 0; i < 8; ++i) {
                float f[8];
                unpack8<T>(x[i], f);
                for (int k = 0; k < 8; ++k)
                    if (fabsf(f[k]) < INFINITY) m = fmaxf(m, fabsf(f[k]));
            }
        }
        // head_dim 64: lanes 0-7 and 16-23 hold one head, the others the second
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 16));
        if (HD == 128) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 8));
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 4));
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
        if (per > 1) {
            if ((lane & 15) == (HD == 64 ? hl * 8 : 0) && lane < 16) top[warp][hl] = m;
            __syncthreads();
            const int w0 = warp - part;
            for (int w = 0; w < per; ++w) m = fmaxf(m, top[w0 + w][hl]);
        }
        // every thread of the unit reads the old scale before one of them stores
        // the new one
        const float s_old = on && held ? *sp : 0.f;
        __syncthreads();
        if (!on) continue;
        float s = fmaxf(s_old, __fdiv_rn(m, 127.f));
        if (s < kQ8MinScale) s = 0.f;
        const float inv = s > 0.f ? __fdiv_rn(1.f, s) : 0.f;
        if (part == 0 && lane < 16 && (lane & (HD == 64 ? 7 : 15)) == 0) *sp = s;
        const bool rescale = held && s > s_old;
        const float ratio = s > 0.f ? __fdiv_rn(s_old, s) : 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int32_t p = pos0 + 2 * i;
            if (p >= first) {
                if (p >= end) continue;
                float f[8];
                unpack8<T>(x[i], f);
                if (odd) {  // infinities +-127, NaN (and 0 times a zero scale) 0
                    int lo[4], hi[4];
                    for (int k = 0; k < 4; ++k) {
                        lo[k] = q8_round(fabsf(f[k]) == INFINITY ? copysignf(127.f, f[k])
                                                                 : f[k] * inv);
                        hi[k] = q8_round(fabsf(f[4 + k]) == INFINITY ? copysignf(127.f, f[4 + k])
                                                                     : f[4 + k] * inv);
                    }
                    cell[i * 32] = make_uint2(q8_pack4(lo), q8_pack4(hi));
                } else {
                    cell[i * 32] = make_uint2(q8_quantise4(f[0], f[1], f[2], f[3], inv),
                                              q8_quantise4(f[4], f[5], f[6], f[7], inv));
                }
                continue;
            }
            if (!rescale) continue;
            int lo[4], hi[4];
            {
                const uint2 q = cell[i * 32];
                float g[4], h[4];
                q8_unpack4(q.x, g);
                q8_unpack4(q.y, h);
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    lo[k] = q8_round(g[k] * ratio);
                    hi[k] = q8_round(h[k] * ratio);
                }
            }
            cell[i * 32] = make_uint2(q8_pack4(lo), q8_pack4(hi));
        }
    }
}

template <typename T, int HD, bool WRITE>
cudaError_t launch_q8(const Q8RowArgs &a, cudaStream_t s) {
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    const int per_cta = kQ8Warps / (a.block_size / 16);
    // Lanes of a page in CTAs of their own while the SMs (148, 8 CTAs each) are
    // not full twice; then a warp takes several, so that finding the sequence
    // and the page (three dependent loads) is paid once for them.
    const int64_t ctas = (a.units + per_cta - 1) / per_cta;
    int lanes = a.lanes;
    while (lanes > 1 && ctas * lanes * 2 > 2 * 8 * 148) lanes = (lanes + 1) / 2;
    cfg.gridDim = dim3((unsigned)ctas, (unsigned)(lanes * 2));
    cfg.blockDim = dim3(kQ8Warps * 32);
    cfg.stream = s;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, q8_rows_kernel<T, HD, WRITE>, a);
}

template <bool WRITE>
int q8_rows(const PkvQ8Layer *layer, const PkvBatch *batch, const int32_t *offsets,
            const void *krows, const void *vrows, size_t total_rows, bool tail, size_t pad_rows,
            uint32_t *table_out, int32_t *lens_out, size_t max_len, const PkvRowScales *wide,
            PkvStream stream, char *error, size_t cap, const char *what) {
    if (!q8_check(layer, batch, error, cap, what)) return 0;
    if (krows == nullptr || vrows == nullptr) {
        pkv_internal_set_error(error, cap, "%s: null rows", what);
        return 0;
    }
    if (((uintptr_t)krows | (uintptr_t)vrows) % 16 != 0) {
        pkv_internal_set_error(error, cap, "%s: rows must be 16-byte aligned", what);
        return 0;
    }
    if (offsets == nullptr && pad_rows == 0 && total_rows != batch->batch) {
        pkv_internal_set_error(error, cap, "%s: one row per sequence needs total_rows == batch",
                               what);
        return 0;
    }
    if (total_rows > INT32_MAX / 4) {
        pkv_internal_set_error(error, cap, "%s: too many rows", what);
        return 0;
    }
    if (total_rows == 0) return 1;
    Q8RowArgs a;
    a.pools[0] = static_cast<uint2 *>(static_cast<void *>(layer->key_pool));
    a.pools[1] = static_cast<uint2 *>(static_cast<void *>(layer->value_pool));
    a.scales[0] = layer->key_scales;
    a.scales[1] = layer->value_scales;
    a.rows[0] = static_cast<uint4 *>(const_cast<void *>(krows));
    a.rows[1] = static_cast<uint4 *>(const_cast<void *>(vrows));
    a.tables = batch->block_tables;
    a.seq_lens = batch->seq_lens;
    a.offsets = offsets;
    a.table_stride = (int32_t)batch->table_stride;
    a.batch = (int32_t)batch->batch;
    a.kv_heads = (int32_t)layer->kv_heads;
    a.lanes = (int32_t)q8_lanes(layer->kv_heads, layer->head_dim);
    a.block_size = (int32_t)layer->block_size;
    a.block_count = (uint32_t)layer->block_count;
    a.units = offsets == nullptr
                  ? (int32_t)batch->batch
                  : (int32_t)(total_rows / layer->block_size + 2 * batch->batch);
    a.total_rows = (int32_t)total_rows;
    a.row_vecs = (int32_t)(layer->kv_heads * layer->head_dim / 8);
    a.tail = tail ? 1 : 0;
    a.pad_rows = (int32_t)pad_rows;
    a.table_out = table_out;
    a.lens_out = lens_out;
    a.max_len = (int32_t)max_len;
    a.wide_k = wide == nullptr ? nullptr : const_cast<float *>(wide->k);
    a.wide_log2 = wide == nullptr ? nullptr : const_cast<float *>(wide->v_log2);
    a.wide_inverse = wide == nullptr ? nullptr : const_cast<float *>(wide->v_inverse);
    if (pad_rows > 0) a.units = (int32_t)(total_rows / layer->block_size);
    const cudaStream_t s = (cudaStream_t)stream;
    cudaError_t st;
    if (layer->dtype == PKV_DTYPE_F16)
        st = layer->head_dim == 128 ? launch_q8<__half, 128, WRITE>(a, s)
                                    : launch_q8<__half, 64, WRITE>(a, s);
    else
        st = layer->head_dim == 128 ? launch_q8<__nv_bfloat16, 128, WRITE>(a, s)
                                    : launch_q8<__nv_bfloat16, 64, WRITE>(a, s);
    if (st == cudaSuccess) st = cudaGetLastError();
    if (st != cudaSuccess) {
        pkv_internal_set_error(error, cap, "%s: launch failed: %s", what, cudaGetErrorString(st));
        return 0;
    }
    return 1;
}

// A rolled-back step must leave the committed rows as they were, and an append
// that raises the open page's scale rounds that page's earlier rows again: so
// they are kept aside while a step is open, one page a sequence and layer (CTA:
// one of those), 2 bytes a value and row of K and V read and written in all.
template <bool RESTORE>
__global__ void __launch_bounds__(256) q8_undo_kernel(const PkvQ8Undo a, int b0) {
    pdl_launch_dependents();
    pdl_wait();
    const int b = b0 + blockIdx.x, tid = threadIdx.x;
    const int bs = (int)a.block_size, kvh = (int)a.kv_heads;
    const int n = __ldg(a.offsets + b + 1) - __ldg(a.offsets + b);
    const int first = __ldg(a.lens + b) - n;
    const int rows = first % bs;  // held
    if (n <= 0 || first <= 0 || rows == 0) return;
    const uint32_t pid = __ldg(a.tables + (int64_t)b * a.table_stride + first / bs);
    if (pid >= a.block_count) return;
    const PkvQ8Pages layer = a.layers[blockIdx.y];
    const int64_t half = (int64_t)a.lanes * bs * 8;  // uint4 of a page
    uint4 *saved = reinterpret_cast<uint4 *>(
        a.saved + ((int64_t)blockIdx.y * a.max_batch + b) * a.slot_bytes);
    const int per = rows * 8;  // uint4 of a lane's held rows
    for (int kv = 0; kv < 2; ++kv) {
        uint4 *page = static_cast<uint4 *>(kv == 0 ? layer.key_pool : layer.value_pool) +
                      (int64_t)pid * half;
        for (int i = tid; i < (int)a.lanes * per; i += 256) {
            const int at = i / per * bs * 8 + i % per;
            if (RESTORE) page[at] = saved[kv * half + at];
            else saved[kv * half + at] = page[at];
        }
        float *s = layer.scales + ((int64_t)kv * (int64_t)a.block_count + pid) * kvh;
        float *kept = reinterpret_cast<float *>(saved + 2 * half) + kv * kvh;
        for (int h = tid; h < kvh; h += 256) {
            if (RESTORE) s[h] = kept[h];
            else kept[h] = s[h];
        }
    }
}

// Scratch of the prefill: 16-bit rows of every sequence, padded to whole pages
// of 128, and their identity table.
struct PrefillSpace {
    size_t pad, k, v, table, lens, scales, total;  // scales: three arrays of scale_bytes
    size_t scale_bytes;
};

PrefillSpace prefill_space(size_t batch, size_t kv_heads, size_t head_dim, size_t max_seq_len) {
    PrefillSpace w;
    w.pad = (max_seq_len + 127) / 128 * 128;
    const size_t bytes = batch * w.pad * kv_heads * head_dim * 2;  // a multiple of 256
    w.k = 0;
    w.v = bytes;
    w.table = 2 * bytes;
    w.lens = w.table + (batch * (w.pad / 128) * 4 + 255) / 256 * 256;
    w.scales = w.lens + (batch * 4 + 255) / 256 * 256;
    w.scale_bytes = (batch * kv_heads * (w.pad / 16) * 4 + 255) / 256 * 256;
    w.total = w.scales + 3 * w.scale_bytes;
    return w;
}

}  // namespace
}  // namespace pkv

extern "C" {

int pkv_q8_append(const PkvQ8Layer *layer, const PkvBatch *batch, const int32_t *row_offsets,
                  const void *key_rows, const void *value_rows, size_t total_rows,
                  PkvStream stream, char *error, size_t error_capacity) {
    PKV_RANGE("pkv_q8_append");
    return pkv::q8_rows<true>(layer, batch, row_offsets, key_rows, value_rows, total_rows, true,
                              0, nullptr, nullptr, 0, nullptr, stream, error, error_capacity, "pkv_q8_append");
}

int pkv_q8_import(const PkvQ8Layer *layer, const PkvBatch *batch, const int32_t *row_offsets,
                  const void *key_rows, const void *value_rows, size_t total_rows,
                  PkvStream stream, char *error, size_t error_capacity) {
    PKV_RANGE("pkv_q8_import");
    return pkv::q8_rows<true>(layer, batch, row_offsets, key_rows, value_rows, total_rows, false,
                              0, nullptr, nullptr, 0, nullptr, stream, error, error_capacity, "pkv_q8_import");
}

int pkv_q8_gather(const PkvQ8Layer *layer, const PkvBatch *batch, const int32_t *row_offsets,
                  void *key_out, void *value_out, size_t total_rows, PkvStream stream, char *error,
                  size_t error_capacity) {
    PKV_RANGE("pkv_q8_gather");
    return pkv::q8_rows<false>(layer, batch, row_offsets, key_out, value_out, total_rows, false,
                               0, nullptr, nullptr, 0, nullptr, stream, error, error_capacity, "pkv_q8_gather");
}

size_t pkv_q8_prefill_workspace_bytes(size_t batch, size_t kv_heads, size_t head_dim,
                                      size_t max_seq_len) {
    return pkv::prefill_space(batch, kv_heads, head_dim, max_seq_len).total;
}

int pkv_q8_prefill(const PkvQ8Layer *layer, const PkvBatch *batch, size_t q_heads,
                   const int32_t *query_offsets, const void *query, size_t total_query_rows,
                   size_t max_query_len, float scale, int causal, void *output,
                   PkvDType output_dtype, size_t max_seq_len, void *workspace,
                   size_t workspace_bytes, PkvStream stream, char *error,
                   size_t error_capacity) {
    PKV_RANGE("pkv_q8_prefill");
    const char *what = "pkv_q8_prefill";
    if (!pkv::q8_check(layer, batch, error, error_capacity, what)) return 0;
    if (query_offsets == nullptr || query == nullptr || output == nullptr) {
        pkv_internal_set_error(error, error_capacity, "%s: null argument", what);
        return 0;
    }
    // what the prefill kernel would refuse, before the pages are widened
    const size_t kvh = layer->kv_heads, hd = layer->head_dim;
    if (output_dtype != PKV_DTYPE_F32 && output_dtype != layer->dtype) {
        pkv_internal_set_error(error, error_capacity,
                               "%s: output dtype must be F32 or the row dtype", what);
        return 0;
    }
    if (q_heads == 0 || q_heads % kvh != 0 || q_heads > 65535 || (uintptr_t)query % 16 != 0) {
        pkv_internal_set_error(error, error_capacity,
                               "%s: q_heads must be a multiple of kv_heads, query 16-byte aligned",
                               what);
        return 0;
    }
    if (max_seq_len == 0 || max_seq_len > INT32_MAX / 4 || max_query_len > INT32_MAX ||
        total_query_rows >= (size_t(1) << 31) || !isfinite(scale) || !(scale > 0.f) ||
        (causal != 0 && causal != 1)) {
        pkv_internal_set_error(error, error_capacity,
                               "%s: invalid max_seq_len, sizes, scale (positive) or causal", what);
        return 0;
    }
    if (total_query_rows == 0) return 1;
    const pkv::PrefillSpace one = pkv::prefill_space(1, kvh, hd, max_seq_len);
    // as many sequences at a time as the workspace holds (rows below 2^31)
    size_t most = workspace_bytes / one.total;  // (one's padding counted each time)
    if (most > batch->batch ||
        workspace_bytes >= pkv::prefill_space(batch->batch, kvh, hd, max_seq_len).total)
        most = batch->batch;
    if (most > (size_t)INT32_MAX / 4 / one.pad) most = (size_t)INT32_MAX / 4 / one.pad;
    if (workspace == nullptr || most == 0 || (uintptr_t)workspace % 256 != 0) {
        pkv_internal_set_error(error, error_capacity,
                               "%s: workspace needs %zu bytes a sequence, 256-byte aligned "
                               "(got %zu)",
                               what, one.total, workspace_bytes);
        return 0;
    }
    for (size_t b0 = 0; b0 < batch->batch; b0 += most) {
        const size_t n = batch->batch - b0 < most ? batch->batch - b0 : most;
        const pkv::PrefillSpace w = pkv::prefill_space(n, kvh, hd, max_seq_len);
        auto *base = static_cast<unsigned char *>(workspace);
        PkvBatch part = *batch;
        part.block_tables += b0 * batch->table_stride;
        part.seq_lens += b0;
        part.batch = n;
        auto *table = reinterpret_cast<uint32_t *>(base + w.table);
        PkvPagedLayer wide;
        wide.key_pool = base + w.k;
        wide.value_pool = base + w.v;
        wide.block_size = 128;
        wide.block_count = n * w.pad / 128;
        wide.kv_heads = kvh;
        wide.head_dim = hd;
        wide.dtype = layer->dtype;
        PkvBatch rows;
        rows.block_tables = table;
        rows.table_stride = w.pad / 128;
        auto *lens = reinterpret_cast<int32_t *>(base + w.lens);
        rows.seq_lens = lens;
        rows.batch = n;
        PkvRowScales scales;
        scales.k = reinterpret_cast<float *>(base + w.scales);
        scales.v_log2 = reinterpret_cast<float *>(base + w.scales + w.scale_bytes);
        scales.v_inverse = reinterpret_cast<float *>(base + w.scales + 2 * w.scale_bytes);
        scales.stride = w.pad / 16;
        if (!pkv::q8_rows<false>(layer, &part, nullptr, wide.key_pool, wide.value_pool, n * w.pad,
                                 false, w.pad, table, lens, max_seq_len, &scales, stream, error,
                                 error_capacity, what) ||
            !pkv_internal_paged_prefill_ex(&wide, &rows, q_heads, query_offsets + b0, query,
                                           total_query_rows, max_query_len, scale, causal, output,
                                           output_dtype, nullptr, 0, 0, 0, &scales, stream, error,
                                           error_capacity, what))
            return 0;
    }
    return 1;
}

size_t pkv_internal_q8_undo_slot(size_t kv_heads, size_t lanes, size_t block_size) {
    return 2 * lanes * block_size * 128 + (2 * kv_heads * sizeof(float) + 15) / 16 * 16;
}

int pkv_internal_q8_undo(const PkvQ8Undo *undo, size_t first, size_t count, int restore,
                         PkvStream stream) {
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)count, (unsigned)undo->layer_count);
    cfg.blockDim = dim3(256);
    cfg.stream = (cudaStream_t)stream;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const cudaError_t st =
        restore ? cudaLaunchKernelEx(&cfg, pkv::q8_undo_kernel<true>, *undo, (int)first)
                : cudaLaunchKernelEx(&cfg, pkv::q8_undo_kernel<false>, *undo, (int)first);
    return st == cudaSuccess && cudaGetLastError() == cudaSuccess;
}

int pkv_internal_take_q8_copy_fault(uint32_t *code) {
    uint32_t zero = 0;
    if (cudaMemcpyFromSymbol(code, pkv::g_q8_copy_fault, sizeof(uint32_t)) != cudaSuccess) return 0;
    return cudaMemcpyToSymbol(pkv::g_q8_copy_fault, &zero, sizeof(uint32_t)) == cudaSuccess;
}

}  // extern "C"
