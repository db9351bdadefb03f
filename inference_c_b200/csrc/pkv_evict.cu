// pkv_evict.cu -- eviction by accumulated attention weight (mass).
//
// evict_select_kernel: per (sequence, KV head) the positions to keep.  The
// newest `recent` stay; of the others those with the largest mass, ties to
// the lower position.  A radix select over the mass as ordered 32-bit keys
// (11 + 11 + 10 bits, most significant first) finds the smallest key kept,
// then one scan in position order writes the list.  A cluster of CTAs shares
// one list: each CTA gathers the mass of its run of positions once (into
// registers, longer runs into shared memory, the longest each time anew), and
// the histograms are summed over distributed shared memory.  Counts and ranks are whole numbers: the result does not
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
constexpr int kMoveRows = 128;  // rows a move CTA takes at a time: its threads

struct EvictArgs {
    const uint32_t *tables, *dst_tables;
    const int32_t *seq_lens;
    float *mass;
    int32_t *kept;          // [batch][kv_heads][keep]
    int32_t table_stride, dst_stride, kv_heads, lanes, block_size, block_shift;
    int32_t keep, recent;
    int32_t max_len;        // longer sequences are left alone, with a fault
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

// Place of the i-th held key: a gap every 32 words, so that threads that read
// runs of their own (strides of a few powers of two) meet different banks.
__device__ __forceinline__ int key_slot(int i) { return i + (i >> 5); }

// Grid (CS * kv_heads, batch), clusters of CS CTAs along x.  RUN > 0: a thread
// holds its run of at most RUN positions (a multiple of 4) in registers; 0:
// runs of any length, keys in shared memory or, past that, gathered each time.
template <int CS, int RUN>
__global__ void __launch_bounds__(kSelThreads) evict_select_kernel(const EvictArgs a) {
    pdl_wait();
    pdl_launch_dependents();
    cg::cluster_group cluster = cg::this_cluster();
    auto list_sync = [&] {
        if constexpr (CS > 1) cluster.sync();
        else __syncthreads();
    };
    // the same variable in the list's r-th CTA
    auto of_rank = [&](uint32_t *p, int r) {
        if constexpr (CS > 1) return cluster.map_shared_rank(p, r);
        else return p;
    };
    extern __shared__ uint32_t keys[];
    __shared__ __align__(8) uint32_t hist[kBins];
    __shared__ uint32_t wsum[32];
    __shared__ uint32_t found[2];     // bin, keys above it
    __shared__ uint32_t count[2];     // this CTA's keys above / equal to the threshold
    __shared__ uint32_t wgt[32], weq[32];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    constexpr int cs = CS;
    const int rank = CS > 1 ? (int)cluster.block_rank() : 0;
    const int g = blockIdx.x / cs, b = blockIdx.y;
    const int32_t L = max(0, __ldg(a.seq_lens + b));
    const int32_t n = L > a.max_len ? 0 : min(L, a.keep);
    int32_t *kept = a.kept + ((int64_t)b * a.kv_heads + g) * a.keep;
    for (int32_t i = n + rank * kSelThreads + tid; i < a.keep; i += cs * kSelThreads) kept[i] = -1;
    if (L > a.max_len) {
        if (tid == 0) record_fault(&g_evict_fault, kFaultPositionOutOfRange);
        return;
    }
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
    const int32_t span = ((old + cs - 1) / cs + 3) & ~3;
    const int32_t lo = min(old, rank * span), hi = min(old, lo + span);
    auto gather = [&](int32_t t) -> uint32_t {
        uint32_t pid;
        if (!page_at(a, trow, a.table_stride, t, pid)) return 0u;
        return mass_key(__ldg(a.mass + ((int64_t)pid * a.kv_heads + g) * a.block_size +
                              (t & (a.block_size - 1))));
    };
    // This thread's run of positions [r0, r1).
    const int32_t run = RUN > 0 ? RUN : (hi - lo + kSelThreads - 1) / kSelThreads;
    const int32_t r0 = min(hi, lo + tid * run), r1 = min(hi, r0 + run);
    const bool held = RUN > 0 || hi - lo <= a.cached;
    uint32_t reg[RUN > 0 ? RUN : 1];
    if constexpr (RUN > 0) {  // all loads in flight; four tokens share a page
        float4 m[RUN / 4];
        bool good[RUN / 4];
#pragma unroll
        for (int i = 0; i < RUN / 4; ++i) {
            uint32_t pid = 0;
            m[i] = make_float4(0.f, 0.f, 0.f, 0.f);
            const int32_t t = r0 + 4 * i;
            good[i] = t < r1 && page_at(a, trow, a.table_stride, t, pid);
            if (good[i])
                m[i] = __ldg(reinterpret_cast<const float4 *>(
                    a.mass + ((int64_t)pid * a.kv_heads + g) * a.block_size +
                    (t & (a.block_size - 1))));
        }
#pragma unroll
        for (int i = 0; i < RUN / 4; ++i) {
            reg[4 * i] = good[i] ? mass_key(m[i].x) : 0u;
            reg[4 * i + 1] = good[i] ? mass_key(m[i].y) : 0u;
            reg[4 * i + 2] = good[i] ? mass_key(m[i].z) : 0u;
            reg[4 * i + 3] = good[i] ? mass_key(m[i].w) : 0u;
        }
    }
    if (RUN == 0 && held) {
        // four tokens a load (a page holds a multiple of 16, lo a multiple of
        // 4), four loads in flight
        const int quads = (hi - lo + 3) / 4;
        for (int q0 = tid; q0 < quads; q0 += 4 * kSelThreads) {
            float4 m[4];
            bool good[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int q = q0 + i * kSelThreads;
                uint32_t pid = 0;
                good[i] = q < quads && page_at(a, trow, a.table_stride, lo + 4 * q, pid);
                m[i] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (good[i])
                    m[i] = __ldg(reinterpret_cast<const float4 *>(
                        a.mass + ((int64_t)pid * a.kv_heads + g) * a.block_size +
                        ((lo + 4 * q) & (a.block_size - 1))));
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int k = 4 * (q0 + i * kSelThreads);  // (past hi: never read)
                if (k >= hi - lo) continue;
                keys[key_slot(k)] = good[i] ? mass_key(m[i].x) : 0u;
                keys[key_slot(k + 1)] = good[i] ? mass_key(m[i].y) : 0u;
                keys[key_slot(k + 2)] = good[i] ? mass_key(m[i].z) : 0u;
                keys[key_slot(k + 3)] = good[i] ? mass_key(m[i].w) : 0u;
            }
        }
    }
    auto key = [&](int32_t t) { return held ? keys[key_slot(t - lo)] : gather(t); };
    // f(position, key) over this thread's run, in order
    auto each = [&](auto f) {
        if constexpr (RUN > 0) {
#pragma unroll
            for (int i = 0; i < RUN; ++i)
                if (r0 + i < r1) f(r0 + i, reg[i]);
        } else {
            for (int32_t t = r0; t < r1; ++t) f(t, key(t));
        }
    };

    uint32_t prefix = 0, want = (uint32_t)need;  // the want-th largest of those with `prefix`
    uint32_t above = 0;
    for (int pass = 0; pass < 3; ++pass) {
        const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
        const int bits = pass == 2 ? 10 : 11;
        for (int i = tid; i < kBins; i += kSelThreads) hist[i] = 0;
        __syncthreads();
        auto tally = [&](int32_t, uint32_t k) {
            if (pass != 0 && (k >> (shift + bits)) != prefix) return;
            // Masses crowd into few bins, even so an atomic for each is fastest:
            // adding up a warp's equal bins first took 7 of 74 us at 131072
            // positions, with all masses equal 4 of 69.
            const uint32_t bin = (k >> shift) & ((1u << bits) - 1u);
            atomicAdd(&hist[bin], 1u);
        };
        each(tally);
        list_sync();
        // bins 2 tid and 2 tid + 1 of the whole list, then keys above each
        uint32_t c0 = 0, c1 = 0;
        uint2 part[CS];
#pragma unroll
        for (int r = 0; r < CS; ++r) part[r] = reinterpret_cast<const uint2 *>(of_rank(hist, r))[tid];
#pragma unroll
        for (int r = 0; r < CS; ++r) {
            c0 += part[r].x;
            c1 += part[r].y;
        }
        uint32_t incl = c0 + c1;  // suffix sums: over this and higher lanes, then warps
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t v = __shfl_down_sync(0xffffffffu, incl, o);
            if (lane + o < 32) incl += v;
        }
        if (lane == 0) wsum[warp] = incl;
        __syncthreads();
        const uint32_t higher = __reduce_add_sync(0xffffffffu, lane > warp ? wsum[lane] : 0u);
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
        list_sync();  // also: every CTA has read every histogram
        prefix = (prefix << bits) | found[0];
        above += found[1];
        want -= found[1];
        __syncthreads();
    }
    // Keys above `prefix` are all kept, of those equal to it the first `want`.
    // Each thread takes a run of positions: its counts, one scan over the CTA and
    // the CTAs before it, then its positions in order.
    uint32_t gt = 0, eq = 0;
    each([&](int32_t, uint32_t k) {
        gt += k > prefix;
        eq += k == prefix;
    });
    uint32_t gi = gt, ei = eq;  // inclusive over the warp
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t x = __shfl_up_sync(0xffffffffu, gi, o);
        const uint32_t y = __shfl_up_sync(0xffffffffu, ei, o);
        if (lane >= o) {
            gi += x;
            ei += y;
        }
    }
    if (lane == 31) {
        wgt[warp] = gi;
        weq[warp] = ei;
    }
    __syncthreads();
    if (warp == 0) {
        uint32_t x = wgt[lane], y = weq[lane];
        const uint32_t x0 = x, y0 = y;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t p = __shfl_up_sync(0xffffffffu, x, o);
            const uint32_t q = __shfl_up_sync(0xffffffffu, y, o);
            if (lane >= o) {
                x += p;
                y += q;
            }
        }
        wgt[lane] = x - x0;
        weq[lane] = y - y0;
        if (lane == 31) {
            count[0] = x;
            count[1] = y;
        }
    }
    list_sync();
    uint32_t g_at = wgt[warp] + gi - gt, e_at = weq[warp] + ei - eq;
    for (int r = 0; r < rank; ++r) {
        const uint32_t *c = of_rank(count, r);
        g_at += c[0];
        e_at += c[1];
    }
    each([&](int32_t t, uint32_t k) {
        if (k > prefix) kept[g_at++ + min(e_at, want)] = t;
        else if (k == prefix) {
            if (e_at < want) kept[g_at + e_at] = t;
            ++e_at;
        }
    });
    list_sync();  // no CTA leaves while its counts are read
}

// VEC: uint4 of one head's row (16-bit 8 or 16, 8-bit 4 or 8).
template <int VEC, bool Q8, bool IN_PLACE>
__global__ void __launch_bounds__(kMoveRows) evict_move_kernel(const EvictArgs a) {
    pdl_launch_dependents();
    pdl_wait();
    __shared__ int64_t from[kMoveRows];  // uint4 index of the source row, -1: none
    __shared__ int64_t to[kMoveRows];    // and of its place
    __shared__ float ratio[2][kMoveRows];
    __shared__ float wtop[2][kMoveRows / 32];
    // rows of a step: eight 16-byte loads a thread in flight (in place fewer, a
    // row's read must precede the writes behind it by a barrier each step)
    constexpr int ROWS = IN_PLACE ? 16 : 8 * kMoveRows / (2 * VEC);
    constexpr int ITEMS = ROWS * VEC * 2 / kMoveRows;
    const int tid = threadIdx.x;
    const int g = blockIdx.y, b = blockIdx.z;
    const int32_t L = max(0, __ldg(a.seq_lens + b));
    const int32_t n = L > a.max_len ? 0 : min(L, a.keep);
    if (IN_PLACE && L <= a.keep) return;  // every row is where it stays
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
    for (int32_t i0 = blockIdx.x * kMoveRows; i0 < n; i0 += gridDim.x * kMoveRows) {
        // thread: one row of the result, i0 + tid
        const int32_t row = i0 + tid, in = row & (a.block_size - 1);
        float s[2] = {0.f, 0.f}, mass = 0.f;
        uint32_t pid = 0, dpid = 0;
        int64_t src = -1;
        if (row < n && page_at(a, drow, a.dst_stride, row, dpid)) {
            const int32_t t = __ldcg(kept + row);
            if (t >= 0 && page_at(a, trow, a.table_stride, t, pid)) {
                const int32_t tin = t & (a.block_size - 1);
                src = row_at(pid, tin);
                mass = a.mass[((int64_t)pid * a.kv_heads + g) * a.block_size + tin];
                if (Q8) {
                    s[0] = a.scales[0][(int64_t)pid * a.kv_heads + g];
                    s[1] = a.scales[1][(int64_t)pid * a.kv_heads + g];
                }
            }
        }
        from[tid] = src;
        to[tid] = row_at(dpid, in);
        float top[2] = {s[0], s[1]};
        if (Q8) {  // the largest scale of the row's block
#pragma unroll
            for (int kv = 0; kv < 2; ++kv) {
                for (int o = 1; o < 32 && o < a.block_size; o <<= 1)
                    top[kv] = fmaxf(top[kv], __shfl_xor_sync(0xffffffffu, top[kv], o));
                if ((tid & 31) == 0) wtop[kv][tid >> 5] = top[kv];
            }
        }
        __syncthreads();
        if (Q8) {
#pragma unroll
            for (int kv = 0; kv < 2; ++kv) {
                const int w0 = (tid >> 5) & ~(a.block_size / 32 - 1);  // the block's warps
                for (int w = 0; w < a.block_size / 32; ++w) top[kv] = fmaxf(top[kv], wtop[kv][w0 + w]);
                ratio[kv][tid] = top[kv] > 0.f ? __fdiv_rn(s[kv], top[kv]) : 0.f;
            }
            __syncthreads();
        }
        const int32_t rows = min(kMoveRows, n - i0);
        for (int32_t r0 = 0; r0 < rows; r0 += ROWS) {
            uint4 x[ITEMS];
#pragma unroll
            for (int i = 0; i < ITEMS; ++i) {
                const int it = i * kMoveRows + tid;
                const int kv = it / (ROWS * VEC), r = r0 + it / VEC % ROWS, c = it % VEC;
                x[i] = make_uint4(0, 0, 0, 0);
                if (from[r] >= 0) x[i] = __ldcg((kv == 0 ? a.pools[0] : a.pools[1]) + from[r] + c);
            }
            if (IN_PLACE) __syncthreads();
#pragma unroll
            for (int i = 0; i < ITEMS; ++i) {
                const int it = i * kMoveRows + tid;
                const int kv = it / (ROWS * VEC), r = r0 + it / VEC % ROWS, c = it % VEC;
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
                (kv == 0 ? a.pools[0] : a.pools[1])[to[r] + c] = x[i];
            }
        }
        if (src >= 0) {
            a.mass[((int64_t)dpid * a.kv_heads + g) * a.block_size + in] = mass;
            if (Q8 && in == 0) {
                a.scales[0][(int64_t)dpid * a.kv_heads + g] = top[0];
                a.scales[1][(int64_t)dpid * a.kv_heads + g] = top[1];
            }
        }
        __syncthreads();
    }
}

template <int VEC, bool Q8>
cudaError_t launch_move(const EvictArgs &a, size_t batch, bool in_place, cudaStream_t s) {
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    const int32_t rows = a.keep < a.max_len ? a.keep : a.max_len;  // of the longest result
    cfg.gridDim = dim3(in_place || rows == 0 ? 1u : (unsigned)((rows + kMoveRows - 1) / kMoveRows),
                       (unsigned)a.kv_heads, (unsigned)batch);
    cfg.blockDim = dim3(kMoveRows);
    cfg.stream = s;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return in_place ? cudaLaunchKernelEx(&cfg, evict_move_kernel<VEC, Q8, true>, a)
                    : cudaLaunchKernelEx(&cfg, evict_move_kernel<VEC, Q8, false>, a);
}

constexpr int32_t kCachedMax = 49152;  // keys of a select CTA: 198 KiB with the gaps
constexpr size_t cached_bytes(int32_t keys) { return ((size_t)keys + keys / 32 + 1) * 4; }

// The most shared memory any call takes, once a device: a limit set to each
// call's own size could be lowered by another thread before its launch.
cudaError_t allow_cached_keys() {
    static int configured[64];
    int dev = 0;
    cudaError_t st = cudaGetDevice(&dev);
    if (st != cudaSuccess || (dev >= 0 && dev < 64 && configured[dev])) return st;
    const int bytes = (int)cached_bytes(kCachedMax);
    st = cudaFuncSetAttribute(evict_select_kernel<1, 0>,
                              cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (st == cudaSuccess)
        st = cudaFuncSetAttribute(evict_select_kernel<8, 0>,
                                  cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (st == cudaSuccess && dev >= 0 && dev < 64) configured[dev] = 1;
    return st;
}

int evict(EvictArgs &a, const PkvBatch *batch, size_t head_dim, bool q8, float *mass, size_t keep,
          size_t recent, const uint32_t *dst_tables, size_t dst_stride, int32_t *kept,
          size_t max_seq_len, PkvStream stream, char *error, size_t cap, const char *what) {
    if (keep == 0 || keep > INT32_MAX / 2 || recent > keep || max_seq_len > INT32_MAX / 2) {
        pkv_internal_set_error(error, cap,
                               "%s: needs 1 <= keep, recent <= keep and a max_seq_len below 2^30",
                               what);
        return 0;
    }
    if (mass == nullptr || kept == nullptr || (uintptr_t)mass % 16 != 0 ||
        (uintptr_t)kept % 4 != 0) {
        pkv_internal_set_error(error, cap,
                               "%s: mass (16-byte aligned) or kept (4-byte) is null or misaligned",
                               what);
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
    a.max_len = (int32_t)max_seq_len;
    const cudaStream_t s = (cudaStream_t)stream;

    // A list is shared by eight CTAs where one would hold more than 4096 keys
    // (four a thread) and the lists alone do not fill the SMs.
    const size_t lists = batch->batch * (size_t)a.kv_heads;
    const unsigned cs = max_seq_len > 4096 && lists <= 148 ? 8 : 1;
    const size_t span = ((max_seq_len + cs - 1) / cs + 3) / 4 * 4;
    // keys a thread: 4 or 16 in registers (one sequence of 131072: 36 us with the
    // keys in shared memory, read through a bounds check and a gap each time)
    const int held = span <= 4 * kSelThreads ? 4 : span <= 16 * kSelThreads ? 16 : 0;
    a.cached = (int32_t)(held == 0 && span <= (size_t)kCachedMax ? span : 0);
    cudaLaunchAttribute attr[2];
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cs;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(cs * (unsigned)a.kv_heads, (unsigned)batch->batch);
    cfg.blockDim = dim3(kSelThreads);
    cfg.dynamicSmemBytes = a.cached > 0 ? cached_bytes(a.cached) : 0;
    cfg.stream = s;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    auto kern = cs == 1 ? (held == 4    ? evict_select_kernel<1, 4>
                           : held == 16 ? evict_select_kernel<1, 16>
                                        : evict_select_kernel<1, 0>)
                        : (held == 4    ? evict_select_kernel<8, 4>
                           : held == 16 ? evict_select_kernel<8, 16>
                                        : evict_select_kernel<8, 0>);
    cudaError_t st = cudaSuccess;
    if (a.cached > 0) st = allow_cached_keys();
    if (st == cudaSuccess) st = cudaLaunchKernelEx(&cfg, kern, a);
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
