// pkv_evict.cu -- eviction by accumulated attention weight (mass).
//
// evict_select_kernel: per (sequence, KV head) the positions to keep.  The
// newest `recent` stay; of the others those with the largest mass, ties to
// the lower position.  A radix select over the mass as ordered 32-bit keys
// (11 + 11 + 10 bits, most significant first) finds the smallest key kept,
// then one scan in position order writes the list.  A cluster of CTAs shares
// one list: each CTA keeps its run of positions in shared memory, so the
// paged mass is gathered once, and the histograms are summed over distributed
// shared memory.  Counts and ranks are whole numbers: the result does not
// depend on the order of the atomics.
//
// evict_move_kernel: rows, mass and (8-bit) scales to their new places.
// 8-bit rows that meet in one block take the largest of their scales,
// q' = rint(q * (s / s_max)), so rows of that scale move unchanged.  Moved in
// place, one CTA per (sequence, KV head) goes through the result in order: a
// row moves to its own or a lower position, so a chunk's reads are never
// behind an earlier chunk's writes, and reads and writes of one chunk are
// apart by a barrier.
#include <cooperative_groups.h>

#include "pkv_q8.cuh"
#include "pkv_trace.h"

namespace cg = cooperative_groups;

namespace pkv {
namespace {

__device__ uint32_t g_evict_fault;

constexpr int kSelThreads = 1024;
constexpr int kBins = 2048;

struct EvictArgs {
    const uint32_t *tables, *dst_tables;
    const int32_t *seq_lens;
    float *mass;
    int32_t *kept;          // [batch][kv_heads][keep]
    int32_t table_stride, dst_stride, kv_heads, lanes, block_size, block_shift;
    int32_t keep, recent;
    uint32_t block_count;
    int32_t cached;         // keys a CTA of the select kernel holds
    // pools: 16-bit rows [.][kv_heads * head_dim], or 8-bit pages
    uint4 *pools[2];
    float *scales[2];
    int32_t row_vecs;       // uint4 of a 16-bit row
};

// Mass as an ordered key; NaN is the smallest, -0 equals +0.
__device__ __forceinline__ uint32_t mass_key(float m) {
    const uint32_t u = __float_as_uint(m + 0.f);
    if (m != m) return 0u;
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

// Page of position t of a sequence, or a recorded fault (false).
__device__ __forceinline__ bool page_at(const EvictArgs &a, const uint32_t *trow, int32_t stride,
                                        int32_t t, uint32_t &pid) {
    const int32_t page = t >> a.block_shift;
    if (page >= stride) {
        record_fault(&g_evict_fault, kFaultPositionOutOfRange);
        return false;
    }
    pid = __ldg(trow + page);
    if (pid >= a.block_count) {
        record_fault(&g_evict_fault, kFaultPageOutOfRange);
        return false;
    }
    return true;
}

// Grid (cluster size * kv_heads, batch), clusters along x.
__global__ void __launch_bounds__(kSelThreads) evict_select_kernel(const EvictArgs a) {
    cg::cluster_group cluster = cg::this_cluster();
    extern __shared__ uint32_t keys[];
    __shared__ __align__(8) uint32_t hist[kBins];
    __shared__ uint32_t wsum[32];
    __shared__ uint32_t found[2];     // bin, keys above it
    __shared__ uint32_t count[2];     // this CTA's keys above / equal to the threshold
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int cs = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const int g = blockIdx.x / cs, b = blockIdx.y;
    const int32_t L = max(0, __ldg(a.seq_lens + b));
    const int32_t n = min(L, a.keep);
    int32_t *kept = a.kept + ((int64_t)b * a.kv_heads + g) * a.keep;
    for (int32_t i = n + rank * kSelThreads + tid; i < a.keep; i += cs * kSelThreads) kept[i] = -1;
    if (L <= a.keep) {
        for (int32_t i = rank * kSelThreads + tid; i < n; i += cs * kSelThreads) kept[i] = i;
        return;  // the whole cluster: L is the sequence's
    }
    const int32_t old = L - a.recent;       // candidates; need < old
    const int32_t need = a.keep - a.recent;
    for (int32_t i = rank * kSelThreads + tid; i < a.recent; i += cs * kSelThreads)
        kept[need + i] = old + i;
    if (need == 0) return;
    const uint32_t *trow = a.tables + (int64_t)b * a.table_stride;
    const int32_t span = (old + cs - 1) / cs;
    const int32_t lo = min(old, rank * span), hi = min(old, lo + span);
    auto gather = [&](int32_t t) -> uint32_t {
        uint32_t pid;
        if (!page_at(a, trow, a.table_stride, t, pid)) return 0u;
        return mass_key(__ldg(a.mass + ((int64_t)pid * a.kv_heads + g) * a.block_size +
                              (t & (a.block_size - 1))));
    };
    const bool held = hi - lo <= a.cached;
    if (held)
        for (int32_t t = lo + tid; t < hi; t += kSelThreads) keys[t - lo] = gather(t);
    auto key = [&](int32_t t) { return held ? keys[t - lo] : gather(t); };

    uint32_t prefix = 0, want = (uint32_t)need;  // the want-th largest of those with `prefix`
    uint32_t above = 0;
    for (int pass = 0; pass < 3; ++pass) {
        const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
        const int bits = pass == 2 ? 10 : 11;
        for (int i = tid; i < kBins; i += kSelThreads) hist[i] = 0;
        __syncthreads();
        for (int32_t t = lo + tid; t < hi; t += kSelThreads) {
            const uint32_t k = key(t);
            if (pass == 0 || (k >> (shift + bits)) == prefix)
                atomicAdd(&hist[(k >> shift) & ((1u << bits) - 1u)], 1u);
        }
        cluster.sync();
        // bins 2 tid and 2 tid + 1 of the whole list, then keys above each
        uint32_t c0 = 0, c1 = 0;
        for (int r = 0; r < cs; ++r) {
            const uint2 v = reinterpret_cast<const uint2 *>(cluster.map_shared_rank(hist, r))[tid];
            c0 += v.x;
            c1 += v.y;
        }
        uint32_t incl = c0 + c1;  // suffix sums: over this and higher lanes, then warps
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t v = __shfl_down_sync(0xffffffffu, incl, o);
            if (lane + o < 32) incl += v;
        }
        if (lane == 0) wsum[warp] = incl;
        __syncthreads();
        uint32_t higher = 0;
        for (int w = warp + 1; w < 32; ++w) higher += wsum[w];
        const uint32_t top1 = higher + incl - c0 - c1;  // keys in bins above 2 tid + 1
        const uint32_t top0 = top1 + c1;
        if (top1 < want && want <= top1 + c1) {
            found[0] = 2 * tid + 1;
            found[1] = top1;
        }
        if (top0 < want && want <= top0 + c0) {
            found[0] = 2 * tid;
            found[1] = top0;
        }
        cluster.sync();  // also: every CTA has read every histogram
        prefix = (prefix << bits) | found[0];
        above += found[1];
        want -= found[1];
        __syncthreads();
    }
    // keys above `prefix` are all kept, of those equal to it the first `want`
    uint32_t gt = 0, eq = 0;
    for (int32_t t = lo + tid; t < hi; t += kSelThreads) {
        const uint32_t k = key(t);
        gt += k > prefix;
        eq += k == prefix;
    }
    if (tid < 2) count[tid] = 0;
    __syncthreads();
    gt = __reduce_add_sync(0xffffffffu, gt);
    eq = __reduce_add_sync(0xffffffffu, eq);
    if (lane == 0) {
        atomicAdd(&count[0], gt);
        atomicAdd(&count[1], eq);
    }
    cluster.sync();
    uint32_t gt0 = 0, eq0 = 0;  // before this CTA's run
    for (int r = 0; r < rank; ++r) {
        const uint32_t *c = cluster.map_shared_rank(count, r);
        gt0 += c[0];
        eq0 += c[1];
    }
    cluster.sync();  // no CTA leaves while its counts are read
    for (int32_t t0 = lo; t0 < hi; t0 += kSelThreads) {
        const int32_t t = t0 + tid;
        const uint32_t k = t < hi ? key(t) : 0u;
        const bool is_gt = t < hi && k > prefix, is_eq = t < hi && k == prefix;
        const uint32_t bg = __ballot_sync(0xffffffffu, is_gt);
        const uint32_t be = __ballot_sync(0xffffffffu, is_eq);
        if (lane == 0) wsum[warp] = (uint32_t)__popc(bg) | (uint32_t)__popc(be) << 16;
        __syncthreads();
        uint32_t before = 0, all = 0;  // packed counts of at most 1024 each
        for (int w = 0; w < 32; ++w) {
            if (w < warp) before += wsum[w];
            all += wsum[w];
        }
        const uint32_t below = (1u << lane) - 1u;
        const uint32_t g_at = gt0 + (before & 0xffffu) + __popc(bg & below);
        const uint32_t e_at = eq0 + (before >> 16) + __popc(be & below);
        if (is_gt) kept[g_at + min(e_at, want)] = t;
        if (is_eq && e_at < want) kept[g_at + e_at] = t;
        gt0 += all & 0xffffu;
        eq0 += all >> 16;
        __syncthreads();
    }
}

// VEC: uint4 of one head's row (16-bit 8 or 16, 8-bit 4 or 8).
template <int VEC, bool Q8, bool IN_PLACE>
__global__ void __launch_bounds__(128) evict_move_kernel(const EvictArgs a) {
    pdl_launch_dependents();
    pdl_wait();
    __shared__ int64_t from[128];   // uint4 index of the source row, -1: none
    __shared__ float moved[128];    // its mass
    __shared__ float ratio[2][128];
    __shared__ float top[2];
    constexpr int ITEMS = 16 * VEC * 2 / 128;
    const int tid = threadIdx.x;
    const int g = blockIdx.y, b = blockIdx.z;
    const int32_t L = max(0, __ldg(a.seq_lens + b));
    const int32_t n = min(L, a.keep);
    const int32_t blocks = (n + a.block_size - 1) >> a.block_shift;
    const int32_t *kept = a.kept + ((int64_t)b * a.kv_heads + g) * a.keep;
    const uint32_t *trow = a.tables + (int64_t)b * a.table_stride;
    const uint32_t *drow = a.dst_tables + (int64_t)b * a.dst_stride;
    // uint4 index of row `in` of page pid, this head's columns
    auto row_at = [&](uint32_t pid, int32_t in) -> int64_t {
        if constexpr (Q8) {
            constexpr int PER = 8 / VEC;  // heads of a lane
            return (((int64_t)pid * a.lanes + g / PER) * a.block_size + in) * 8 + (g % PER) * VEC;
        } else {
            return ((int64_t)pid * a.block_size + in) * a.row_vecs + (int64_t)g * VEC;
        }
    };
    for (int32_t j = blockIdx.x; j < blocks; j += gridDim.x) {
        const int32_t rows = min(a.block_size, n - (j << a.block_shift));
        uint32_t dpid;
        if (!page_at(a, drow, a.dst_stride, j << a.block_shift, dpid)) return;  // whole CTA
        float s[2] = {0.f, 0.f};
        if (tid < 128) from[tid] = -1;
        if (tid < rows) {
            const int32_t t = kept[(j << a.block_shift) + tid];
            uint32_t pid;
            if (t >= 0 && page_at(a, trow, a.table_stride, t, pid)) {
                const int32_t in = t & (a.block_size - 1);
                from[tid] = row_at(pid, in);
                moved[tid] = a.mass[((int64_t)pid * a.kv_heads + g) * a.block_size + in];
                if (Q8) {
                    s[0] = a.scales[0][(int64_t)pid * a.kv_heads + g];
                    s[1] = a.scales[1][(int64_t)pid * a.kv_heads + g];
                }
            }
        }
        if (Q8) {
            ratio[0][tid] = s[0];
            ratio[1][tid] = s[1];
        }
        __syncthreads();
        if (Q8) {
            if (tid < 64) {  // warp kv: the largest scale of the block's rows
                float m = 0.f;
                for (int i = tid & 31; i < 128; i += 32) m = fmaxf(m, ratio[tid >> 5][i]);
                m = warp_max(m);
                if ((tid & 31) == 0) top[tid >> 5] = m;
            }
            __syncthreads();
            ratio[0][tid] = top[0] > 0.f ? __fdiv_rn(s[0], top[0]) : 0.f;
            ratio[1][tid] = top[1] > 0.f ? __fdiv_rn(s[1], top[1]) : 0.f;
            __syncthreads();
        }
        const int64_t to = row_at(dpid, 0);
        const int32_t step = Q8 ? 8 : a.row_vecs;  // uint4 between rows of a page
        for (int32_t r0 = 0; r0 < rows; r0 += 16) {
            uint4 x[ITEMS];
#pragma unroll
            for (int i = 0; i < ITEMS; ++i) {
                const int it = i * 128 + tid;
                const int kv = it / (16 * VEC), r = r0 + it / VEC % 16, c = it % VEC;
                x[i] = make_uint4(0, 0, 0, 0);
                if (from[r] >= 0) x[i] = (kv == 0 ? a.pools[0] : a.pools[1])[from[r] + c];
            }
            if (IN_PLACE) __syncthreads();
#pragma unroll
            for (int i = 0; i < ITEMS; ++i) {
                const int it = i * 128 + tid;
                const int kv = it / (16 * VEC), r = r0 + it / VEC % 16, c = it % VEC;
                if (from[r] < 0) continue;
                if (Q8 && ratio[kv][r] != 1.f) {
                    const float f = ratio[kv][r];
                    uint32_t w[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        float v[4];
                        int q[4];
                        q8_unpack4(w[k], v);
#pragma unroll
                        for (int e = 0; e < 4; ++e) q[e] = q8_round(v[e] * f);
                        w[k] = q8_pack4(q);
                    }
                    x[i] = make_uint4(w[0], w[1], w[2], w[3]);
                }
                (kv == 0 ? a.pools[0] : a.pools[1])[to + (int64_t)r * step + c] = x[i];
            }
        }
        if (tid < rows && from[tid] >= 0)
            a.mass[((int64_t)dpid * a.kv_heads + g) * a.block_size + tid] = moved[tid];
        if (Q8 && tid < 2)
            (tid == 0 ? a.scales[0] : a.scales[1])[(int64_t)dpid * a.kv_heads + g] = top[tid];
        if (IN_PLACE) __syncthreads();
    }
}

template <int VEC, bool Q8>
cudaError_t launch_move(const EvictArgs &a, size_t batch, bool in_place, cudaStream_t s) {
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    const int32_t blocks = (a.keep + a.block_size - 1) / a.block_size;
    cfg.gridDim = dim3(in_place ? 1u : (unsigned)blocks, (unsigned)a.kv_heads, (unsigned)batch);
    cfg.blockDim = dim3(128);
    cfg.stream = s;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return in_place ? cudaLaunchKernelEx(&cfg, evict_move_kernel<VEC, Q8, true>, a)
                    : cudaLaunchKernelEx(&cfg, evict_move_kernel<VEC, Q8, false>, a);
}

constexpr int32_t kCachedMax = 49152;  // keys of a select CTA: 192 KiB

int evict(EvictArgs &a, const PkvBatch *batch, size_t head_dim, bool q8, float *mass, size_t keep,
          size_t recent, const uint32_t *dst_tables, size_t dst_stride, int32_t *kept,
          size_t max_seq_len, PkvStream stream, char *error, size_t cap, const char *what) {
    if (keep == 0 || keep > INT32_MAX / 2 || recent > keep || max_seq_len > INT32_MAX / 2) {
        pkv_internal_set_error(error, cap,
                               "%s: needs 1 <= keep, recent <= keep and a max_seq_len below 2^30",
                               what);
        return 0;
    }
    if (mass == nullptr || kept == nullptr || ((uintptr_t)mass | (uintptr_t)kept) % 4 != 0) {
        pkv_internal_set_error(error, cap, "%s: mass or kept is null or not 4-byte aligned", what);
        return 0;
    }
    if (batch->batch > 65535) {
        pkv_internal_set_error(error, cap, "%s: at most 65535 sequences", what);
        return 0;
    }
    const bool in_place = dst_tables == nullptr || dst_tables == batch->block_tables;
    if (in_place) {
        dst_tables = batch->block_tables;
        dst_stride = batch->table_stride;
    }
    if (dst_stride == 0 || dst_stride > INT32_MAX / 128) {
        pkv_internal_set_error(error, cap, "%s: invalid table stride", what);
        return 0;
    }
    a.tables = batch->block_tables;
    a.dst_tables = dst_tables;
    a.seq_lens = batch->seq_lens;
    a.mass = mass;
    a.kept = kept;
    a.table_stride = (int32_t)batch->table_stride;
    a.dst_stride = (int32_t)dst_stride;
    a.block_shift = 0;
    while ((1 << a.block_shift) < a.block_size) ++a.block_shift;
    a.keep = (int32_t)keep;
    a.recent = (int32_t)recent;
    const cudaStream_t s = (cudaStream_t)stream;

    // A list is shared by eight CTAs where one would hold more than 4096 keys
    // (four a thread) and the lists alone do not fill the SMs.
    const size_t lists = batch->batch * (size_t)a.kv_heads;
    const unsigned cs = max_seq_len > 4096 && lists <= 148 ? 8 : 1;
    const size_t span = (max_seq_len + cs - 1) / cs;
    a.cached = (int32_t)(span < (size_t)kCachedMax ? span : 0);
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cs;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(cs * (unsigned)a.kv_heads, (unsigned)batch->batch);
    cfg.blockDim = dim3(kSelThreads);
    cfg.dynamicSmemBytes = (size_t)a.cached * 4;
    cfg.stream = s;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    static int configured[64];
    int dev = 0;
    cudaGetDevice(&dev);
    cudaError_t st = cudaSuccess;
    if (dev >= 0 && dev < 64 && !configured[dev]) {
        st = cudaFuncSetAttribute(evict_select_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                  kCachedMax * 4);
        if (st == cudaSuccess) configured[dev] = 1;
    }
    if (st == cudaSuccess) st = cudaLaunchKernelEx(&cfg, evict_select_kernel, a);
    if (st == cudaSuccess) {
        if (q8)
            st = head_dim == 128 ? launch_move<8, true>(a, batch->batch, in_place, s)
                                 : launch_move<4, true>(a, batch->batch, in_place, s);
        else
            st = head_dim == 128 ? launch_move<16, false>(a, batch->batch, in_place, s)
                                 : launch_move<8, false>(a, batch->batch, in_place, s);
    }
    if (st == cudaSuccess) st = cudaGetLastError();
    if (st != cudaSuccess) {
        pkv_internal_set_error(error, cap, "%s: launch failed: %s", what, cudaGetErrorString(st));
        return 0;
    }
    return 1;
}

}  // namespace
}  // namespace pkv

extern "C" {

int pkv_kv_evict(const PkvPagedLayer *layer, const PkvBatch *batch, float *mass, size_t keep,
                 size_t recent, const uint32_t *dst_tables, size_t dst_stride, int32_t *kept,
                 size_t max_seq_len, PkvStream stream, char *error, size_t error_capacity) {
    PKV_RANGE("pkv_kv_evict");
    const char *what = "pkv_kv_evict";
    if (layer == nullptr) {
        pkv_internal_set_error(error, error_capacity, "%s: null argument", what);
        return 0;
    }
    if (!pkv::pool_check(layer->key_pool, layer->value_pool, batch, error, error_capacity, what) ||
        !pkv::page_shape_check(layer->block_size, layer->block_count, layer->kv_heads,
                               layer->head_dim, layer->dtype, batch, error, error_capacity, what))
        return 0;
    pkv::EvictArgs a = {};
    a.pools[0] = static_cast<uint4 *>(layer->key_pool);
    a.pools[1] = static_cast<uint4 *>(layer->value_pool);
    a.kv_heads = (int32_t)layer->kv_heads;
    a.block_size = (int32_t)layer->block_size;
    a.block_count = (uint32_t)layer->block_count;
    a.row_vecs = (int32_t)(layer->kv_heads * layer->head_dim / 8);
    return pkv::evict(a, batch, layer->head_dim, false, mass, keep, recent, dst_tables, dst_stride,
                      kept, max_seq_len, stream, error, error_capacity, what);
}

int pkv_q8_evict(const PkvQ8Layer *layer, const PkvBatch *batch, float *mass, size_t keep,
                 size_t recent, const uint32_t *dst_tables, size_t dst_stride, int32_t *kept,
                 size_t max_seq_len, PkvStream stream, char *error, size_t error_capacity) {
    PKV_RANGE("pkv_q8_evict");
    const char *what = "pkv_q8_evict";
    if (!pkv::q8_check(layer, batch, error, error_capacity, what)) return 0;
    pkv::EvictArgs a = {};
    a.pools[0] = reinterpret_cast<uint4 *>(layer->key_pool);
    a.pools[1] = reinterpret_cast<uint4 *>(layer->value_pool);
    a.scales[0] = layer->key_scales;
    a.scales[1] = layer->value_scales;
    a.kv_heads = (int32_t)layer->kv_heads;
    a.lanes = (int32_t)pkv::q8_lanes(layer->kv_heads, layer->head_dim);
    a.block_size = (int32_t)layer->block_size;
    a.block_count = (uint32_t)layer->block_count;
    return pkv::evict(a, batch, layer->head_dim, true, mass, keep, recent, dst_tables, dst_stride,
                      kept, max_seq_len, stream, error, error_capacity, what);
}

int pkv_internal_take_evict_fault(uint32_t *code) {
    uint32_t zero = 0;
    if (cudaMemcpyFromSymbol(code, pkv::g_evict_fault, sizeof(uint32_t)) != cudaSuccess) return 0;
    return cudaMemcpyToSymbol(pkv::g_evict_fault, &zero, sizeof(uint32_t)) == cudaSuccess;
}

}  // extern "C"
