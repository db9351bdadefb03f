// pkv_q8_decode.cu -- decode attention over 8-bit pages (one query token per
// sequence) on the integer tensor cores.
//
//   o = sum_t softmax_t(scale q . k_t) v_t,   k_t = kq_t ks,  v_t = vq_t vs
//
// with one scale per (page, KV head).  The pages go to the tensor cores as
// they lie: q . k_t = ks (q . kq_t) and p v = (p vs) vq, so a scale multiplies
// a score and a softmax weight, never an element, and no byte of K or V is
// converted.  The other operand is cut into three signed base-256 digits:
//   q = f (d0 2^16 + d1 2^8 + d2), f a power of two per query head (22 bits),
//   p vs = F (d0 2^16 + d1 2^8 + d2), F per tile and head (23 bits),
// each digit one row of the B operand of tcgen05.mma kind::i8, whose sums are
// exact 32-bit integers.  So a tile costs
//   S^T[128 tok][3 GV] = K . Qd^T   and   O^T[128 dim][3 GV] = V^T . Pd^T
// and the only roundings are those of the digits, of exp and of FP32 sums
// over tiles.  Bytes past a sequence's length are finite whatever they are and
// meet digits of zero.
//
// Bound by HBM: 2 bytes a token, KV head and column.  One persistent 512-thread
// CTA per SM:
//   warps 0-3   producers, each every fourth tile: one TMA box per page of K and
//               of V (block x 128 bytes, contiguous in the pool) and the page's
//               scales by cp.async.  16 boxes of 2 KiB and their bookkeeping
//               take one warp some 2000 cycles, in which HBM delivers a tile
//               and a half, so one warp (or one for K and one for V) cannot
//               keep up; warp 0 also claims the units
//   warps 4-7   softmax group of even tiles, warps 8-11 of odd tiles: a 32 KiB
//               tile streams in half the time of a 16-bit one, and one group's
//               chain of TMEM load, maximum, exp and digit stores would not
//               keep up; each group carries its own running maximum, sum and
//               output, joined when a piece ends
//   warps 12, 13 one thread each issues tcgen05.mma, S and PV: a barrier wait
//               costs a thread some 90 cycles even when it is through and an
//               issue some 40, nearly a tile's time for one thread with both
//   warp 14     query warp: the digits of the next piece's query rows
// Few barriers a tile: s_full(j) (S done) also frees K's slot, o_full(j) (PV
// done) V's, and p_full(j) (weights written) also says that S(j) and O(j - 4)
// have been read, which is what S(j + 4) and PV(j) overwrite.
// Work split: stream-K with a dynamic tail (pkv_sched.cuh), as the 16-bit
// decode.  A segment is one lane (128 columns) of one sequence: one KV head of
// head_dim 128, or two of head_dim 64 whose query digits are zero in each
// other's columns.  GV is its padded number of query heads; a group above
// GV (per KV head) is served by several segments over the same lane.
#include <math.h>

#include <cudaTypedefs.h>

#include "pkv_mass.cuh"
#include "pkv_q8.cuh"
#include "pkv_sched.cuh"
#include "pkv_sm100.cuh"
#include "pkv_trace.h"

namespace pkv {
namespace {

__device__ uint32_t g_q8_decode_fault;

constexpr float kLog2e = 1.4426950408889634f;
constexpr size_t kQ8MaxGroup = 16;
constexpr int kThreads = 512;
constexpr int kProducers = 4;        // producer warps
constexpr int kRegsControl = 64, kRegsSoftmax = 192;
static_assert(256 * kRegsControl + 256 * kRegsSoftmax <= kThreads * 128, "register split");
constexpr int kMaxBatch = 8192;
constexpr int kLaunchBatch = 1024;   // sequences of one launch (their prefix lives in smem)
constexpr int kMaxGrid = 256;
constexpr int kInKernelMergeMax = 32;
constexpr int kMaxUnits = kMaxGrid * (1 + kMaxRounds);
constexpr size_t kMinUnitTiles = 8;  // smallest dynamic unit
constexpr int kRing = 4;             // unit ids in flight between the roles
constexpr int kScaleSlots = 16;      // tiles whose scales are in shared memory
constexpr int kPending = 64;         // cut pieces a CTA keeps before it takes their tickets
constexpr uint32_t kTileBytes = 16384;
constexpr float kDigitMax = 8323072.f;  // 127 * 2^16: three signed digits hold +-this

template <int GV>
struct Cfg {
    static constexpr int N = GV == 4 ? 16 : GV == 8 ? 32 : 48;  // B rows (digit-major, padded)
    static constexpr int KS = GV == 4 ? 6 : 5;  // K tiles in the ring
    static constexpr int VS = GV == 4 ? 6 : 5;  // V tiles (S, P and O have four buffers)
    static constexpr uint32_t BT = N * 128;                      // bytes of one B tile
    static constexpr uint32_t V_OFF = KS * kTileBytes;
    static constexpr uint32_t Q_OFF = V_OFF + VS * kTileBytes;
    static constexpr uint32_t P_OFF = Q_OFF + 2 * BT;
    static constexpr uint32_t X_OFF = P_OFF + 4 * BT;            // odd group's output
    static constexpr uint32_t SC_OFF = X_OFF + GV * 512;
    static constexpr uint32_t BAR_OFF = SC_OFF + kScaleSlots * 128;
    static constexpr uint32_t MISC_OFF = BAR_OFF + 512;
    // per group: [kInKernelMergeMax][GV] maxima, then sums, then slots
    static constexpr uint32_t MERGE_WORDS = kInKernelMergeMax * (2 * GV + 1);
    static constexpr uint32_t PREFIX_OFF = MISC_OFF + 2560 + 2 * MERGE_WORDS * 4;
    static constexpr uint32_t TMEM_COLS = GV == 4 ? 128 : GV == 8 ? 256 : 512;
    static_assert(8 * N <= (int)TMEM_COLS, "tensor memory");
    static size_t smem(int batch) { return PREFIX_OFF + 4u * ((size_t)batch + 1u) + 1024u; }
    static_assert(PREFIX_OFF + 4u * (kLaunchBatch + 1u) + 1024u <= 232448u, "shared memory");
};

struct Q8Args {
    const uint32_t *tables;
    const int32_t *seq_lens;
    const void *query;
    void *out;
    const float *kscales, *vscales;
    uint32_t *counters;      // [kMaxUnits] merge tickets by first unit
    uint32_t *claim;         // [2]
    float *part_ml;          // [units][2][GV][m, l]
    float *part_o;           // [units][2][GV][128]
    int32_t *tile_prefix;    // [batch + 1] for the merge kernel
    int32_t table_stride, batch;
    int32_t kv_heads;        // segments of one sequence (the schedule's name for them)
    int32_t heads;           // KV heads
    int32_t lanes, subs;     // segments = lanes * subs
    int32_t group, q_heads;
    int32_t block_size;
    uint32_t block_count;
    float scale_log2;
    int32_t merge_in_kernel, min_unit;
    int32_t bf16, out_f32;   // row type; 32-bit outputs
    // Mass (else null): every score by stream tile and slot, and every query
    // head's final maximum and sum (pkv_mass.cuh).
    float *scores, *final_ml;
    int64_t score_tiles;
};

struct Workspace {
    size_t claim, counters, prefix, ml, o, total;
};

size_t round_up(size_t v, size_t m) { return (v + m - 1) / m * m; }

Workspace workspace_of(size_t units, size_t gv) {
    Workspace w;
    w.claim = 0;
    w.counters = 256;
    w.prefix = w.counters + round_up((size_t)kMaxUnits * 4, 256);
    w.ml = w.prefix + round_up(((size_t)kLaunchBatch + 1) * 4, 256);
    w.o = w.ml + round_up(units * 2 * gv * 8, 256);
    w.total = w.o + round_up(units * 2 * gv * 512, 256);
    return w;
}

// Largest of a warp's values, in one instruction.
__device__ __forceinline__ float redux_max(float v) {
    float r;
    asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
    return r;
}

// The three signed base-256 digits of u as the bytes of a word: adding 128 to
// the two lower digits makes the carries, flipping their top bits takes it off.
__device__ __forceinline__ uint32_t digits(int u) { return (uint32_t)(u + 0x8080) ^ 0x8080u; }

// Byte offset of (row, col) in a tile of 128-byte rows, 128-byte swizzle.
__device__ __forceinline__ uint32_t sw_byte(uint32_t row, uint32_t col) {
    return (row >> 3) * 1024u + (row & 7u) * 128u + (((col >> 4) ^ (row & 7u)) << 4) + (col & 15u);
}

__device__ __forceinline__ void store_out(const Q8Args &a, int64_t at, float v) {
    if (a.out_f32) static_cast<float *>(a.out)[at] = v;
    else if (a.bf16) static_cast<__nv_bfloat16 *>(a.out)[at] = __float2bfloat16_rn(v);
    else static_cast<__half *>(a.out)[at] = __float2half_rn(v);
}

// Segment g's query head in slot h (head_dim 64: slots below GV / 2 belong to
// KV head 2 * lane, the others to the next), or -1 for a padding slot.
template <int GV, bool PAIR>
__device__ __forceinline__ int head_at(const Q8Args &a, int g, int h) {
    const int lane = g / a.subs, sub = g - lane * a.subs;
    constexpr int PER = PAIR ? GV / 2 : GV;
    const int half = PAIR && h >= PER ? 1 : 0;
    const int kvh = PAIR ? 2 * lane + half : lane;
    const int hh = sub * PER + h - half * PER;
    return hh < a.group && kvh < a.heads ? kvh * a.group + hh : -1;
}

// acc rows of slot h that are its head's columns, and the output element.
template <bool PAIR>
__device__ __forceinline__ bool owns(int gv, int h, int row) {
    return !PAIR || (h >= gv / 2) == (row >= 64);
}
__device__ __forceinline__ void store_ml(const Q8Args &a, int b, int qh, float m, float l) {
    *reinterpret_cast<float2 *>(a.final_ml + ((int64_t)b * a.q_heads + qh) * 2) =
        make_float2(m, l);
}
template <bool PAIR>
__device__ __forceinline__ int64_t out_at(const Q8Args &a, int b, int qh, int row) {
    return ((int64_t)b * a.q_heads + qh) * (PAIR ? 64 : 128) + (PAIR ? row & 63 : row);
}

template <int GV, bool PAIR>
__global__ void __launch_bounds__(kThreads, 1)
q8_decode_tc_kernel(const Q8Args a, const __grid_constant__ CUtensorMap kmap,
                    const __grid_constant__ CUtensorMap vmap) {
    using namespace sm100;
    using C = Cfg<GV>;
    constexpr int N = C::N, KS = C::KS, VS = C::VS;
    constexpr uint32_t kIdescQK = idesc_s8(128, N, false, false);
    constexpr uint32_t kIdescPV = idesc_s8(128, N, true, false);
    extern __shared__ unsigned char smem_raw[];
    unsigned char *sm = reinterpret_cast<unsigned char *>(
        (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t *bars = reinterpret_cast<uint64_t *>(sm + C::BAR_OFF);
    uint64_t *kfull = bars, *vfull = bars + 8, *s_full = bars + 16, *p_full = bars + 24;
    uint64_t *o_full = bars + 32;  // one per V slot
    uint64_t *q_full = bars + 44, *q_empty = bars + 46;
    uint64_t *x_full = bars + 48, *x_empty = bars + 49;
    uint64_t *ring_full = bars + 50, *ring_empty = bars + 54;  // .. 57
    unsigned char *misc = sm + C::MISC_OFF;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(misc);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(misc + 4);
    int *pend_n = reinterpret_cast<int *>(misc + 8);
    volatile int *group_unit = reinterpret_cast<volatile int *>(misc + 16);  // [2]
    volatile int *ring = reinterpret_cast<volatile int *>(misc + 32);        // [kRing]
    int *scan = reinterpret_cast<int *>(misc + 64);                          // [12]
    Sched *sched = reinterpret_cast<Sched *>(misc + 128);
    float *qscale = reinterpret_cast<float *>(misc + 256);                   // [2][16]
    float *red = reinterpret_cast<float *>(misc + 384);                      // [2 groups][2][4][16]
    float *lred = reinterpret_cast<float *>(misc + 1408);                    // [2][4][16]
    float *xml = reinterpret_cast<float *>(misc + 1920);                     // [16][m, l]
    int *pend = reinterpret_cast<int *>(misc + 2048);       // [kPending] b << 16 | segment
    int *last = reinterpret_cast<int *>(misc + 2304);       // [kPending] this CTA merges it
    float *scales = reinterpret_cast<float *>(sm + C::SC_OFF);  // [slot][K0, V0, K1, V1][8]
    int *prefix = reinterpret_cast<int *>(sm + C::PREFIX_OFF);

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (tid == 0) {
        for (int s = 0; s < KS; ++s) {
            mbar_init(&kfull[s], 33);  // TMA bytes, and each lane's scale copies
            mbar_init(&s_full[s], 2);  // the MMAs, and the issuer that saw the scales
        }
        for (int s = 0; s < VS; ++s) {
            mbar_init(&vfull[s], 1);
            mbar_init(&o_full[s], 1);
        }
        for (int i = 0; i < 4; ++i) {
            mbar_init(&p_full[i], 128);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&q_full[i], 32);
            mbar_init(&q_empty[i], 256);  // both groups saw their last S of the piece
        }
        mbar_init(x_full, 128);
        mbar_init(x_empty, 128);
        for (int i = 0; i < kRing; ++i) {
            mbar_init(&ring_full[i], 1);
            mbar_init(&ring_empty[i], 8);  // three producers, two MMA, query warp, two groups
        }
        *abort_flag = 0;
        fence_mbar_init();
    }
    // B rows past the digits (and, paired, the other head's columns) stay zero
    for (int i = tid; i < (int)(6 * C::BT / 16); i += kThreads)
        reinterpret_cast<uint4 *>(sm + C::Q_OFF)[i] = make_uint4(0, 0, 0, 0);
    if (warp == 12) {
        tmem_alloc(tmem_slot, C::TMEM_COLS);
        tmem_relinquish();
    }
    if (tid == 0) {
        tma_prefetch_desc(&kmap);
        tma_prefetch_desc(&vmap);
    }
    pdl_wait();
    pdl_launch_dependents();
    build_tile_prefix(a, prefix, scan);
    fence_proxy_async_smem();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    const int64_t total_tiles = prefix[a.batch];
    if (tid == 0) make_sched(*sched, total_tiles, (int)gridDim.x, a.min_unit);
    __syncthreads();
    const Sched &sc = *sched;
    const bool works = (int)blockIdx.x < sc.n && total_tiles > 0;
    const int n_units = sched_units(sc);
    uint32_t *fault = &g_q8_decode_fault;
    if (blockIdx.x == 0 && a.tile_prefix != nullptr)
        for (int b = tid; b <= a.batch; b += kThreads) a.tile_prefix[b] = prefix[b];

    const int page_shift = 31 - __clz(a.block_size);
    if (warp < 4 || warp >= 12) {
    setmaxnreg_dec<kRegsControl>();
    if (warp < kProducers) {
        // ----------------------------- producers -----------------------------
        uint32_t j = 0;
        bool ok = true;
        int u = works ? (int)blockIdx.x : -1;
        for (uint32_t ku = 0;; ++ku) {
            const int rs = (int)(ku % kRing);
            if (warp == 0) {  // publish the unit (-1: no more) to the other roles
                ok = __all_sync(0xffffffffu, mbar_wait(&ring_empty[rs], ((ku / kRing) & 1) ^ 1,
                                                       abort_flag, fault)) && ok;
                if (!ok) u = -1;
                if (lane == 0) {
                    ring[rs] = u;
                    mbar_arrive(&ring_full[rs]);
                }
                __syncwarp();
            } else {
                if (lane == 0) {
                    u = mbar_wait(&ring_full[rs], (ku / kRing) & 1, abort_flag, fault) ? ring[rs] : -1;
                    mbar_arrive(&ring_empty[rs]);
                }
                u = __shfl_sync(0xffffffffu, u, 0);
            }
            if (u < 0 || !ok) break;
            const int64_t ue = unit_start(sc, u + 1);
            for (int64_t t = unit_start(sc, u); ok && t < ue;) {
                const Piece P = piece_at(t, ue, prefix, a);
                t += P.k1 - P.k0;
                const int L = __ldg(a.seq_lens + P.b);
                const uint32_t *trow = a.tables + (int64_t)P.b * a.table_stride;
                const int kl = P.g / a.subs;
                const int page = lane & 7;
                // lane's page of tile k (an invalid id past the table row)
                auto entry_at = [&](int k) -> uint32_t {
                    const int at = (k * kTcTile >> page_shift) + page;
                    return k < P.k1 && at < a.table_stride ? __ldg(trow + at) : 0xffffffffu;
                };
                const int first = (int)((warp - j) & 3u);  // this warp's first tile of the piece
                uint32_t next = entry_at(P.k0 + first);
                for (int k = P.k0 + first; k < P.k1; k += kProducers) {
                    const uint32_t jj = j + (uint32_t)(k - P.k0);
                    const uint32_t ks = jj % KS, vs = jj % VS;
                    const uint32_t pid = next;
                    next = entry_at(k + kProducers);
                    const int rows = min(kTcTile, L - k * kTcTile);
                    const int np = (rows + a.block_size - 1) >> page_shift;  // 1..8
                    const bool good = page < np && pid < a.block_count;
                    if (page < np && !good) record_fault(fault, kFaultPageOutOfRange);
                    const uint32_t bytes =
                        (uint32_t)__popc(__ballot_sync(0xffffffffu, good) & 0xffu)
                        << (page_shift + 7);
                    // S(j - KS) done: K's slot is free; PV(j - VS): V's
                    ok = __all_sync(0xffffffffu,
                                    mbar_wait(&s_full[ks], ((jj / KS) & 1) ^ 1, abort_flag, fault) &&
                                        mbar_wait(&o_full[vs], ((jj / VS) & 1) ^ 1, abort_flag,
                                                  fault));
                    if (!ok) break;
                    if (lane == 0) mbar_arrive_expect_tx(&kfull[ks], bytes);
                    if (lane == 8) mbar_arrive_expect_tx(&vfull[vs], bytes);
                    __syncwarp();
                    // lanes 0-7 one page of K each, 8-15 of V
                    const bool is_v = (lane & 8) != 0;
                    if (good && lane < 16)
                        tma_load_2d(sm + (is_v ? C::V_OFF + vs * kTileBytes : ks * kTileBytes) +
                                        ((uint32_t)page << (page_shift + 7)),
                                    is_v ? &vmap : &kmap, is_v ? &vfull[vs] : &kfull[ks], 0,
                                    (int32_t)((pid * (uint32_t)a.lanes + (uint32_t)kl)
                                              << page_shift));
                    // scales: kind = lane / 8 (K0, V0, K1, V1 of the lane's heads)
                    const int head = (PAIR ? 2 * kl : kl) + (lane >> 4);
                    const bool want = good && head < a.heads && (PAIR || lane < 16);
                    const float *src = is_v ? a.vscales : a.kscales;
                    cp_async4_or_zero(scales + (jj % kScaleSlots) * 32 + lane,
                                      want ? src + (int64_t)pid * a.heads + head : src, want);
                    cp_async_mbar_arrive(&kfull[ks]);
                }
                j += (uint32_t)(P.k1 - P.k0);
            }
            if (warp == 0) {
                int claimed = -1;
                if (ok && sc.rounds > 0 && lane == 0) {
                    const int c = sc.n + (int)atomicAdd(a.claim, 1u);
                    claimed = c < n_units ? c : -1;
                }
                u = __shfl_sync(0xffffffffu, claimed, 0);
            }
        }
        // the last CTA done claiming zeroes the claim words for the next launch
        if (sc.rounds > 0 && works && tid == 0) {
            __threadfence();
            if (atomicAdd(a.claim + 1, 1u) == (uint32_t)sc.n - 1) {
                atomicExch(a.claim, 0u);
                atomicExch(a.claim + 1, 0u);
            }
        }
        asm volatile("cp.async.wait_all;\n" ::: "memory");
    } else if (warp == 14) {
        // ----------------------------- query warp -----------------------------
        uint32_t qi = 0;
        bool ok = true;
        for (uint32_t ku = 0; ok; ++ku) {
            const int rs = (int)(ku % kRing);
            int u = -1;
            if (lane == 0) {
                if (mbar_wait(&ring_full[rs], (ku / kRing) & 1, abort_flag, fault)) u = ring[rs];
                mbar_arrive(&ring_empty[rs]);
            }
            u = __shfl_sync(0xffffffffu, u, 0);
            if (u < 0) break;
            const int64_t ue = unit_start(sc, u + 1);
            for (int64_t t = unit_start(sc, u); ok && t < ue;) {
                const Piece P = piece_at(t, ue, prefix, a);
                t += P.k1 - P.k0;
                // Query digits: lane holds 4 columns of a row (head_dim 64: the
                // first half warp, at the head's half of the 128 columns).
                constexpr int HD = PAIR ? 64 : 128;
                ok = __all_sync(0xffffffffu, mbar_wait(&q_empty[qi & 1], ((qi >> 1) & 1) ^ 1,
                                                       abort_flag, fault));
                if (!ok) break;
                unsigned char *qb = sm + C::Q_OFF + (qi & 1) * C::BT;
                for (int h0 = 0; h0 < GV; h0 += 4) {
                    uint2 raw[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int qh = head_at<GV, PAIR>(a, P.g, h0 + i);
                        raw[i] = make_uint2(0, 0);
                        if (qh >= 0 && lane * 4 < HD)
                            raw[i] = __ldg(reinterpret_cast<const uint2 *>(
                                static_cast<const uint16_t *>(a.query) +
                                ((int64_t)P.b * a.q_heads + qh) * HD + lane * 4));
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int h = h0 + i;
                        float x[4];
                        if (a.bf16) {
                            x[0] = __uint_as_float(raw[i].x << 16);
                            x[1] = __uint_as_float(raw[i].x & 0xffff0000u);
                            x[2] = __uint_as_float(raw[i].y << 16);
                            x[3] = __uint_as_float(raw[i].y & 0xffff0000u);
                        } else {
                            const float2 lo = __half22float2(*reinterpret_cast<__half2 *>(&raw[i].x));
                            const float2 hi = __half22float2(*reinterpret_cast<__half2 *>(&raw[i].y));
                            x[0] = lo.x; x[1] = lo.y; x[2] = hi.x; x[3] = hi.y;
                        }
                        // |x| as ordered integers: infinities and NaN stay the largest
                        uint32_t top = 0;
#pragma unroll
                        for (int e = 0; e < 4; ++e) top = max(top, __float_as_uint(fabsf(x[e])));
                        top = __reduce_max_sync(0xffffffffu, top);
                        // f = 2^(21 - exponent of the largest): q f < 2^22, its bits
                        // down to 2^-21 of the largest kept exactly
                        const int ex = max((int)(top >> 23), 22);
                        const float f = top == 0 ? 0.f : __uint_as_float((uint32_t)(275 - ex) << 23);
                        const float back = __uint_as_float((uint32_t)(ex - 21) << 23);  // 1 / f
                        uint32_t d[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) d[e] = digits(__float2int_rn(x[e] * f));
                        if (lane * 4 < HD) {
                            const uint32_t col = lane * 4 + (PAIR && h >= GV / 2 ? 64 : 0);
#pragma unroll
                            for (int k = 0; k < 3; ++k) {  // digit k: most significant first
                                const int sh = 16 - 8 * k;
                                uint32_t w = 0;
#pragma unroll
                                for (int e = 0; e < 4; ++e) w |= ((d[e] >> sh) & 255u) << (8 * e);
                                *reinterpret_cast<uint32_t *>(qb + sw_byte(k * GV + h, col)) = w;
                            }
                        }
                        if (lane == 0)
                            qscale[(qi & 1) * 16 + h] =
                                top >= 0x7f800000u ? __uint_as_float(0x7fc00000u) : back * a.scale_log2;
                    }
                }
                fence_proxy_async_smem();
                mbar_arrive(&q_full[qi & 1]);
                ++qi;
            }
        }
    } else if (warp == 12 || warp == 13) {
        // ------------------- MMA issuers: S (warp 12), PV (warp 13) -------------------
        if (lane == 0) {
            const uint64_t kdesc = sw128_desc(smem_u32(sm), 16, 1024);
            const uint64_t vdesc = sw128_desc(smem_u32(sm + C::V_OFF), kTileBytes, 1024);
            const uint64_t qdesc = sw128_desc(smem_u32(sm + C::Q_OFF), 16, 1024);
            const uint64_t pdesc = sw128_desc(smem_u32(sm + C::P_OFF), 16, 1024);
            uint32_t j = 0, qi = 0;
            bool ok = true;
            for (uint32_t ku = 0; ok; ++ku) {
                const int rs = (int)(ku % kRing);
                int u = -1;
                if (mbar_wait(&ring_full[rs], (ku / kRing) & 1, abort_flag, fault)) u = ring[rs];
                mbar_arrive(&ring_empty[rs]);
                if (u < 0) break;
                int64_t t = unit_start(sc, u);
                const int64_t ue = unit_start(sc, u + 1);
                if (warp == 13) {  // the pieces' bounds do not matter to PV
                    for (; ok && t < ue; ++t, ++j) {
                        const uint32_t stage = j % VS, buf = j & 3;
                        if (!mbar_wait(&vfull[stage], (j / VS) & 1, abort_flag, fault) ||
                            !mbar_wait(&p_full[buf], (j >> 2) & 1, abort_flag, fault)) {
                            ok = false;
                            break;
                        }
                        tc_fence_after();
                        const uint64_t ad = vdesc + (uint64_t)(stage * (kTileBytes >> 4));
                        const uint64_t bd = pdesc + (uint64_t)(buf * (C::BT >> 4));
                        const uint32_t dst = tmem + (4 + buf) * N;
                        mma_i8_ss_at<0, 0>(dst, ad, bd, kIdescPV, 0);
                        mma_i8_ss_at<256, 2>(dst, ad, bd, kIdescPV, 1);
                        mma_i8_ss_at<512, 4>(dst, ad, bd, kIdescPV, 1);
                        mma_i8_ss_at<768, 6>(dst, ad, bd, kIdescPV, 1);
                        mma_commit(&o_full[stage]);
                    }
                    continue;
                }
                while (ok && t < ue) {
                    const Piece P = piece_at(t, ue, prefix, a);
                    t += P.k1 - P.k0;
                    ok = mbar_wait(&q_full[qi & 1], (qi >> 1) & 1, abort_flag, fault);
                    const uint64_t bd = qdesc + (uint64_t)((qi & 1) * (C::BT >> 4));
                    for (int k = P.k0; ok && k < P.k1; ++k, ++j) {
                        const uint32_t stage = j % KS, buf = j & 3;
                        if (!mbar_wait(&kfull[stage], (j / KS) & 1, abort_flag, fault) ||
                            !mbar_wait(&p_full[buf], ((j >> 2) & 1) ^ 1, abort_flag, fault)) {
                            ok = false;
                            break;
                        }
                        tc_fence_after();
                        const uint64_t ad = kdesc + (uint64_t)(stage * (kTileBytes >> 4));
                        const uint32_t dst = tmem + buf * N;
                        mma_i8_ss_at<0, 0>(dst, ad, bd, kIdescQK, 0);
                        mma_i8_ss_at<2, 2>(dst, ad, bd, kIdescQK, 1);
                        mma_i8_ss_at<4, 4>(dst, ad, bd, kIdescQK, 1);
                        mma_i8_ss_at<6, 6>(dst, ad, bd, kIdescQK, 1);
                        mma_commit(&s_full[stage]);
                        // this thread saw the scales land: its own arrival passes
                        // them on to the softmax group
                        mbar_arrive(&s_full[stage]);
                    }
                    ++qi;
                }
            }
        }
        __syncwarp();
    }
    } else {
        setmaxnreg_inc<kRegsSoftmax>();
        // ------------------------ softmax group `grp` ------------------------
        // On an abort the groups keep running the same loops and barriers but
        // stop reading TMEM; the fault word already records the failure.
        const int grp = warp >= 8 ? 1 : 0;
        const int q4 = warp & 3;        // TMEM lane quadrant
        const int row = q4 * 32 + lane; // token of S^T, column of O^T
        const int wt = tid - 128 - grp * 128;
        const uint32_t lane_off = (uint32_t)(q4 * 32) << 16;
        auto group_sync = [&] { named_barrier(1 + grp, 128); };
        uint32_t j = 0, qi = 0;
        bool aborted = false;
        auto await = [&](uint64_t *bar, uint32_t par) {
            aborted = aborted || !__all_sync(0xffffffffu, mbar_wait(bar, par, abort_flag, fault));
        };
        // Group 0: tickets of the pending pieces; last[i]: this CTA finished the
        // segment of piece i (its partials are all in memory).
        int pending = 0;
        auto take_tickets = [&] {
            group_sync();  // the group's partials and the list are written
            if (wt < pending) {
                const int b = pend[wt] >> 16, g = pend[wt] & 0xffff;
                const int nt = (prefix[b + 1] - prefix[b]) / a.kv_heads;
                const int64_t seg = prefix[b] + (int64_t)g * nt;
                const int u0 = unit_of_tile(sc, seg);
                const int np = unit_of_tile(sc, seg + nt - 1) - u0 + 1;
                __threadfence();  // publishes the group's partials (bar.sync is cumulative)
                last[wt] = atomicAdd(a.counters + u0, 1u) == (uint32_t)(np - 1);
            }
            group_sync();
        };
        float *mw = reinterpret_cast<float *>(misc + 2560) + grp * C::MERGE_WORDS;
        int *mslot = reinterpret_cast<int *>(mw + 2 * kInKernelMergeMax * GV);
        auto merge = [&](int i) {
            const int b = pend[i] >> 16, g = pend[i] & 0xffff;
            const int nt = (prefix[b + 1] - prefix[b]) / a.kv_heads;
            const int64_t seg = prefix[b] + (int64_t)g * nt;
            const int u0 = unit_of_tile(sc, seg);
            const int np = unit_of_tile(sc, seg + nt - 1) - u0 + 1;
            if (np > kInKernelMergeMax) {  // cannot happen with the host's choice of units
                if (wt == 0) record_fault(fault, kFaultPositionOutOfRange);
                return;
            }
            __threadfence();  // the other CTAs' partials, seen through the ticket
            for (int e = wt; e < np * GV; e += 128) {
                const int c = e / GV, h = e - c * GV;
                const int slot = (u0 + c) * 2 + unit_slot(sc, u0 + c, seg);
                const float2 ml = __ldcg(reinterpret_cast<const float2 *>(
                    a.part_ml + ((int64_t)slot * GV + h) * 2));
                mw[e] = ml.x;
                mw[kInKernelMergeMax * GV + e] = ml.y;
                if (h == 0) mslot[c] = slot;
            }
            group_sync();
            if (wt < GV) {
                float mx = -INFINITY, lt = 0.f;
                for (int c = 0; c < np; ++c) mx = fmaxf(mx, mw[c * GV + wt]);
                for (int c = 0; c < np; ++c) {
                    const float mc = mw[c * GV + wt];
                    const float f = mc == mx ? 1.f : exp2f(mc - mx);
                    lt += mw[kInKernelMergeMax * GV + c * GV + wt] * f;
                    mw[c * GV + wt] = f;
                }
                const float inv = lt == 0.f ? 0.f : 1.f / lt;
                for (int c = 0; c < np; ++c) mw[c * GV + wt] *= inv;
                const int qh = head_at<GV, PAIR>(a, g, wt);
                if (a.final_ml != nullptr && qh >= 0) store_ml(a, b, qh, mx, lt);
            }
            // 16 loads in flight, the first of them before the weights are known
            float o[GV];
#pragma unroll
            for (int h = 0; h < GV; ++h) o[h] = 0.f;
            constexpr int AT_ONCE = 16 / GV;
            for (int c0 = 0; c0 < np; c0 += AT_ONCE) {
                float v[AT_ONCE][GV];
#pragma unroll
                for (int k = 0; k < AT_ONCE; ++k) {
                    const float *src =
                        a.part_o + (int64_t)mslot[min(c0 + k, np - 1)] * GV * 128 + row;
#pragma unroll
                    for (int h = 0; h < GV; ++h) v[k][h] = __ldcg(src + h * 128);
                }
                if (c0 == 0) group_sync();
#pragma unroll
                for (int k = 0; k < AT_ONCE; ++k)
#pragma unroll
                    for (int h = 0; h < GV; ++h)
                        if (c0 + k < np) o[h] = fmaf(mw[(c0 + k) * GV + h], v[k][h], o[h]);
            }
#pragma unroll
            for (int h = 0; h < GV; ++h) {
                const int qh = head_at<GV, PAIR>(a, g, h);
                if (qh >= 0 && owns<PAIR>(GV, h, row))
                    store_out(a, out_at<PAIR>(a, b, qh, row), o[h]);
            }
            if (wt == 0) a.counters[u0] = 0u;
            group_sync();  // the scratch is free again
        };
        for (uint32_t ku = 0;; ++ku) {
            const int rs = (int)(ku % kRing);
            if (wt == 0) {
                int uu = -1;
                if (mbar_wait(&ring_full[rs], (ku / kRing) & 1, abort_flag, fault)) uu = ring[rs];
                group_unit[grp] = uu;
                mbar_arrive(&ring_empty[rs]);
            }
            group_sync();
            const int u = group_unit[grp];
            group_sync();
            if (u < 0) break;
            const int64_t us = unit_start(sc, u), ue = unit_start(sc, u + 1);
            for (int64_t t = us; t < ue;) {
                const Piece P = piece_at(t, ue, prefix, a);
                const bool first_piece = t == us;
                t += P.k1 - P.k0;
                const int L = __ldg(a.seq_lens + P.b);
                float m_run[GV], l_part[GV], acc[GV], alpha_prev[GV], qs[GV];
                float f_prev[PAIR ? 2 : 1];
                await(&q_full[qi & 1], (qi >> 1) & 1);
#pragma unroll
                for (int h = 0; h < GV; ++h) {
                    m_run[h] = -INFINITY;
                    l_part[h] = 0.f;
                    acc[h] = 0.f;
                    qs[h] = qscale[(qi & 1) * 16 + h];
                }
                // O of this group's previous tile, whose weights were relative
                // to that tile's maximum and scaled by F = f_prev
                auto fold = [&](uint32_t jp) {
                    const uint32_t buf = jp & 3;
                    await(&o_full[jp % VS], (jp / VS) & 1);
                    float o[N];
#pragma unroll
                    for (int i = 0; i < N; ++i) o[i] = 0.f;
                    if (!aborted) {
                        tc_fence_after();
                        if constexpr (N == 48) {
                            tmem_ld_32x32b<32>(tmem + (4 + buf) * N + lane_off,
                                               *reinterpret_cast<float(*)[32]>(&o[0]));
                            tmem_ld_32x32b<16>(tmem + (4 + buf) * N + 32 + lane_off,
                                               *reinterpret_cast<float(*)[16]>(&o[32]));
                        } else {
                            tmem_ld_32x32b<N>(tmem + (4 + buf) * N + lane_off, o);
                        }
                        tmem_wait_ld();
                        tc_fence_before();
                    }
#pragma unroll
                    for (int h = 0; h < GV; ++h) {
                        const int lo = __float_as_int(o[GV + h]) * 256 + __float_as_int(o[2 * GV + h]);
                        const float v = fmaf((float)__float_as_int(o[h]), 65536.f, (float)lo);
                        acc[h] = fmaf(v, f_prev[PAIR && h >= GV / 2 ? 1 : 0], acc[h] * alpha_prev[h]);
                    }
                };
                int64_t mine = -1;  // this group's previous tile of the piece
                for (int k = P.k0; k < P.k1; ++k, ++j) {
                    if ((int)(j & 1) != grp) continue;
                    const uint32_t buf = j & 3;
                    await(&s_full[j % KS], (j / KS) & 1);
                    float s[N];
#pragma unroll
                    for (int i = 0; i < N; ++i) s[i] = 0.f;
                    if (!aborted) {
                        tc_fence_after();
                        if constexpr (N == 48) {
                            tmem_ld_32x32b<32>(tmem + buf * N + lane_off,
                                               *reinterpret_cast<float(*)[32]>(&s[0]));
                            tmem_ld_32x32b<16>(tmem + buf * N + 32 + lane_off,
                                               *reinterpret_cast<float(*)[16]>(&s[32]));
                        } else {
                            tmem_ld_32x32b<N>(tmem + buf * N + lane_off, s);
                        }
                        tmem_wait_ld();
                        tc_fence_before();
                    }
                    const float *sl = scales + (j % kScaleSlots) * 32;
                    float ks[PAIR ? 2 : 1], pf[PAIR ? 2 : 1], f_cur[PAIR ? 2 : 1];
#pragma unroll
                    for (int e = 0; e < (PAIR ? 2 : 1); ++e) {
                        ks[e] = sl[e * 16 + (row >> page_shift)];
                        const float4 v0 = *reinterpret_cast<const float4 *>(sl + e * 16 + 8);
                        const float4 v1 = *reinterpret_cast<const float4 *>(sl + e * 16 + 12);
                        const float top = fmaxf(fmaxf(fmaxf(v0.x, v0.y), fmaxf(v0.z, v0.w)),
                                                fmaxf(fmaxf(v1.x, v1.y), fmaxf(v1.z, v1.w)));
                        // weight digits: p * vs / top * kDigitMax
                        pf[e] = top > 0.f ? __fdividef(sl[e * 16 + 8 + (row >> page_shift)], top) *
                                                kDigitMax
                                          : 0.f;
                        f_cur[e] = top * (1.f / kDigitMax);
                    }
                    const bool live = row < L - k * kTcTile;
                    // two buffers: a warp writes a tile's maxima only after all
                    // read those of the group's tile before the last
                    float *myred = red + grp * 128 + ((j >> 1) & 1) * 64;
                    float x[GV];
#pragma unroll
                    for (int h = 0; h < GV; ++h) {
                        const int lo = __float_as_int(s[GV + h]) * 256 + __float_as_int(s[2 * GV + h]);
                        const float v = fmaf((float)__float_as_int(s[h]), 65536.f, (float)lo);
                        x[h] = live ? v * (qs[h] * ks[PAIR && h >= GV / 2 ? 1 : 0]) : -INFINITY;
                        if (a.scores != nullptr && P.seg + k < a.score_tiles)
                            a.scores[((P.seg + k) * GV + h) * 128 + row] = x[h];
                        const float wm = redux_max(x[h]);
                        if (lane == 0) myred[q4 * 16 + h] = wm;
                    }
                    group_sync();
                    float alpha[GV];
                    unsigned char *pb = sm + C::P_OFF + buf * C::BT;
#pragma unroll
                    for (int h = 0; h < GV; ++h) {
                        const float tmax = fmaxf(fmaxf(myred[h], myred[16 + h]),
                                                 fmaxf(myred[32 + h], myred[48 + h]));
                        const float m_new = fmaxf(m_run[h], tmax);
                        alpha[h] = ex2_fast(m_run[h] - m_new);
                        m_run[h] = m_new;
                        const float p = ex2_fast(x[h] - m_new);
                        l_part[h] = fmaf(l_part[h], alpha[h], p);
                        const uint32_t d = digits(__float2int_rn(p * pf[PAIR && h >= GV / 2 ? 1 : 0]));
                        pb[sw_byte(h, row)] = (unsigned char)(d >> 16);
                        pb[sw_byte(GV + h, row)] = (unsigned char)(d >> 8);
                        pb[sw_byte(2 * GV + h, row)] = (unsigned char)d;
                    }
                    fence_proxy_async_smem();
                    mbar_arrive(&p_full[buf]);
                    if (mine >= 0) fold((uint32_t)mine);
                    mine = j;
#pragma unroll
                    for (int h = 0; h < GV; ++h) alpha_prev[h] = alpha[h];
#pragma unroll
                    for (int e = 0; e < (PAIR ? 2 : 1); ++e) f_prev[e] = f_cur[e];
                }
                mbar_arrive(&q_empty[qi & 1]);  // the piece's last S is done in both groups
                ++qi;
                if (mine >= 0) fold((uint32_t)mine);
                // ---- join the groups ----
                float l[GV];
#pragma unroll
                for (int h = 0; h < GV; ++h) {
                    const float ls = warp_sum(l_part[h]);
                    if (lane == 0) lred[grp * 64 + q4 * 16 + h] = ls;
                }
                group_sync();
#pragma unroll
                for (int h = 0; h < GV; ++h) {
                    const float *r = lred + grp * 64 + h;
                    l[h] = (r[0] + r[16]) + (r[32] + r[48]);
                }
                group_sync();
                float *xo = reinterpret_cast<float *>(sm + C::X_OFF);  // [GV][128]
                const uint32_t xpar = (qi - 1) & 1;
                if (grp == 1) {
                    await(x_empty, xpar ^ 1);
#pragma unroll
                    for (int h = 0; h < GV; ++h) {
                        xo[h * 128 + row] = acc[h];
                        if (wt == h) {
                            xml[h * 2] = m_run[h];
                            xml[h * 2 + 1] = l[h];
                        }
                    }
                    mbar_arrive(x_full);
                    continue;
                }
                await(x_full, xpar);
#pragma unroll
                for (int h = 0; h < GV; ++h) {
                    const float mb = xml[h * 2], lb = xml[h * 2 + 1];
                    const float m = fmaxf(m_run[h], mb);
                    // equal maxima keep a factor of 1, both -inf (a query that
                    // is not a number) included
                    const float fa = m_run[h] == m ? 1.f : ex2_fast(m_run[h] - m);
                    const float fb = mb == m ? 1.f : ex2_fast(mb - m);
                    acc[h] = acc[h] * fa + xo[h * 128 + row] * fb;
                    l[h] = l[h] * fa + lb * fb;
                    m_run[h] = m;
                }
                mbar_arrive(x_empty);
                // ---- the piece's output or partial ----
                if (P.k0 == 0 && P.k1 == P.nt) {
#pragma unroll
                    for (int h = 0; h < GV; ++h) {
                        const int qh = head_at<GV, PAIR>(a, P.g, h);
                        if (qh >= 0 && owns<PAIR>(GV, h, row))
                            store_out(a, out_at<PAIR>(a, P.b, qh, row),
                                      l[h] == 0.f ? 0.f : acc[h] / l[h]);
                        if (a.final_ml != nullptr && qh >= 0 && wt == h)
                            store_ml(a, P.b, qh, m_run[h], l[h]);
                    }
                    continue;
                }
                const int64_t slot = ((int64_t)u * 2 + (first_piece ? 0 : 1)) * GV;
#pragma unroll
                for (int h = 0; h < GV; ++h) {
                    a.part_o[(slot + h) * 128 + row] = acc[h];
                    if (wt == h)
                        *reinterpret_cast<float2 *>(a.part_ml + (slot + h) * 2) =
                            make_float2(m_run[h], l[h]);
                }
                if (!a.merge_in_kernel) continue;
                if (wt == 0) pend[pending] = P.b << 16 | P.g;
                if (++pending == kPending) {
                    take_tickets();
                    for (int i = 0; i < pending; ++i)
                        if (last[i]) merge(i);
                    pending = 0;
                }
            }
        }
        // The tickets of the cut pieces wait until the CTA's work is done: a
        // fence, a ticket and a merge in mid-stream held both groups, and so
        // the stream, for about 4 us a unit.
        if (grp == 0) {
            take_tickets();
            if (wt == 0) *pend_n = pending;
        }
        named_barrier(3, 256);
        {
            int nth = 0;
            for (int i = 0; i < *pend_n; ++i)
                if (last[i] && (nth++ & 1) == grp) merge(i);
        }
        // empty sequences: zeros
        if (grp == 0)
            for (int b = blockIdx.x; b < a.batch; b += gridDim.x) {
                if (__ldg(a.seq_lens + b) > 0) continue;
                const int n = a.q_heads * (PAIR ? 64 : 128);
                for (int i = wt; i < n; i += 128) store_out(a, (int64_t)b * n + i, 0.f);
            }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 12) tmem_dealloc(tmem, C::TMEM_COLS);
}

// Merges segments cut into more pieces than the decode kernel joins itself
// (few segments: one long sequence).  Grid (segments * GV, batch), one slot's
// query head per CTA: four threads a column, each every fourth piece.
constexpr int kMergeThreads = 512;
template <int GV, bool PAIR>
__global__ void __launch_bounds__(kMergeThreads) q8_merge_kernel(const Q8Args a, int grid) {
    pdl_wait();
    pdl_launch_dependents();
    __shared__ float w[kMaxGrid], lsum[kMaxGrid];
    __shared__ int slot[kMaxGrid];
    __shared__ float part[4][128];
    __shared__ Sched sc;
    const int b = blockIdx.y, g = blockIdx.x / GV, h = blockIdx.x - g * GV;
    const int qh = head_at<GV, PAIR>(a, g, h);
    const int64_t T = a.tile_prefix[a.batch];
    if (threadIdx.x == 0) make_sched(sc, T, grid, a.min_unit);
    __syncthreads();
    const int nt = (a.tile_prefix[b + 1] - a.tile_prefix[b]) / a.kv_heads;
    if (qh < 0 || nt == 0 || T == 0) return;
    const int64_t seg = a.tile_prefix[b] + (int64_t)g * nt;
    const int u0 = unit_of_tile(sc, seg);
    const int np = unit_of_tile(sc, seg + nt - 1) - u0 + 1;
    if (np == 1 || np > kMaxGrid) return;  // one piece: the decode kernel wrote it
    for (int c = threadIdx.x; c < np; c += kMergeThreads) {
        slot[c] = (int)(((int64_t)(u0 + c) * 2 + unit_slot(sc, u0 + c, seg)) * GV + h);
        const float2 ml = __ldcg(reinterpret_cast<const float2 *>(a.part_ml + (int64_t)slot[c] * 2));
        w[c] = ml.x;
        lsum[c] = ml.y;
    }
    __syncthreads();
    if (threadIdx.x < 32) {
        float mx = -INFINITY, lt = 0.f;
        for (int c = threadIdx.x; c < np; c += 32) mx = fmaxf(mx, w[c]);
        mx = warp_max(mx);
        for (int c = threadIdx.x; c < np; c += 32) {
            const float f = w[c] == mx ? 1.f : exp2f(w[c] - mx);
            lt += lsum[c] * f;
            w[c] = f;
        }
        lt = warp_sum(lt);
        const float inv = lt == 0.f ? 0.f : 1.f / lt;
        for (int c = threadIdx.x; c < np; c += 32) w[c] *= inv;
        if (a.final_ml != nullptr && threadIdx.x == 0) store_ml(a, b, qh, mx, lt);
    }
    __syncthreads();
    const int row = threadIdx.x & 127, share = threadIdx.x >> 7;
    float o = 0.f;
#pragma unroll 8
    for (int c = share; c < np; c += 4) o += w[c] * __ldcg(a.part_o + (int64_t)slot[c] * 128 + row);
    part[share][row] = o;
    __syncthreads();
    if (share == 0 && owns<PAIR>(GV, h, row))
        store_out(a, out_at<PAIR>(a, b, qh, row),
                  (part[0][row] + part[1][row]) + (part[2][row] + part[3][row]));
}

int sm_count() {
    static int counts[64];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
    if (counts[dev] == 0) {
        int n = 0;
        cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
        counts[dev] = n > 0 ? n : 148;
    }
    return counts[dev];
}
int decode_grid() { return sm_count() < kMaxGrid ? sm_count() : kMaxGrid; }

// One pool as [rows][128] bytes; a box is one page of one lane.
bool encode_q8_map(CUtensorMap *map, const void *pool, uint64_t rows, uint32_t box_rows) {
    static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
    if (fn == nullptr) {
        void *p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) !=
                cudaSuccess ||
            q != cudaDriverEntryPointSuccess)
            return false;
        fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
    }
    cuuint64_t dims[2] = {128, rows};
    cuuint64_t strides[1] = {128};
    cuuint32_t box[2] = {128, box_rows};
    cuuint32_t estr[2] = {1, 1};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void *>(pool), dims, strides, box,
              estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int GV, bool PAIR>
int launch(const Q8Args &a, const CUtensorMap &k, const CUtensorMap &v, int ncta,
           cudaStream_t stream) {
    auto kern = q8_decode_tc_kernel<GV, PAIR>;
    static int configured[64];
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev >= 0 && dev < 64 && !configured[dev]) {
        if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 (int)Cfg<GV>::smem(kLaunchBatch)) != cudaSuccess)
            return 0;
        configured[dev] = 1;
    }
    cudaLaunchAttribute pdl[1];
    pdl[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    pdl[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(ncta);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = Cfg<GV>::smem(a.batch);
    cfg.stream = stream;
    cfg.attrs = pdl;
    cfg.numAttrs = 1;
    if (cudaLaunchKernelEx(&cfg, kern, a, k, v) != cudaSuccess) return 0;
    if (!a.merge_in_kernel) {
        cfg.gridDim = dim3(a.kv_heads * GV, a.batch);
        cfg.blockDim = dim3(kMergeThreads);
        cfg.dynamicSmemBytes = 0;
        if (cudaLaunchKernelEx(&cfg, q8_merge_kernel<GV, PAIR>, a, ncta) != cudaSuccess) return 0;
    }
    return cudaGetLastError() == cudaSuccess;
}

// Slots of one segment: the smallest that holds the group (both groups of a
// head_dim 64 pair), else 16 and several segments a lane.
size_t slots_of(size_t group, size_t head_dim) {
    const size_t want = head_dim == 64 ? 2 * group : group;
    return want <= 4 ? 4 : want <= 8 ? 8 : 16;
}

// pkv_q8_decode, and with `mass` pkv_q8_decode_mass.
int q8_decode(const char *what, const PkvQ8Layer *layer, const PkvBatch *batch, size_t q_heads,
              const void *query, float scale, void *output, PkvDType output_dtype,
              size_t max_seq_len, float *mass, void *workspace, size_t workspace_bytes,
              PkvStream stream, char *error, size_t error_capacity) {
    if (!q8_check(layer, batch, error, error_capacity, what)) return 0;
    if (query == nullptr || output == nullptr) {
        pkv_internal_set_error(error, error_capacity, "%s: null argument", what);
        return 0;
    }
    if (output_dtype != PKV_DTYPE_F32 && output_dtype != layer->dtype) {
        pkv_internal_set_error(error, error_capacity,
                               "%s: output dtype must be F32 or the row dtype", what);
        return 0;
    }
    const size_t kvh = layer->kv_heads, hd = layer->head_dim;
    if (q_heads == 0 || q_heads % kvh != 0 || q_heads / kvh > kQ8MaxGroup) {
        pkv_internal_set_error(error, error_capacity,
                               "%s: q_heads must be 1..%zu times kv_heads", what,
                               kQ8MaxGroup);
        return 0;
    }
    const size_t lanes = q8_lanes(kvh, hd);
    const size_t rows = layer->block_count * lanes * layer->block_size;
    if (batch->batch > (size_t)kMaxBatch || !isfinite(scale) ||
        max_seq_len > INT32_MAX / 2 || layer->block_count > INT32_MAX || rows > INT32_MAX) {
        pkv_internal_set_error(error, error_capacity,
                               "%s: invalid batch (1..%d), scale, length or pool (block_count * "
                               "lanes * block_size must be below 2^31)",
                               what, kMaxBatch);
        return 0;
    }
    if ((uintptr_t)query % 16 != 0 || (uintptr_t)output % 4 != 0) {
        pkv_internal_set_error(error, error_capacity,
                               "%s: query must be 16-byte, output 4-byte aligned", what);
        return 0;
    }
    const size_t group = q_heads / kvh, gv = slots_of(group, hd);
    const size_t per = hd == 64 ? gv / 2 : gv;         // slots per KV head
    const size_t subs = (group + per - 1) / per;
    const size_t segs = lanes * subs;
    const int ncta = decode_grid();
    const Workspace ws = workspace_of((size_t)ncta * (1 + kMaxRounds), gv);
    const size_t need =
        ws.total + (mass == nullptr ? 0
                                    : mass_scratch_bytes(batch->batch, q_heads, segs, gv,
                                                         max_seq_len));
    if (workspace == nullptr || workspace_bytes < need || (uintptr_t)workspace % 256 != 0) {
        pkv_internal_set_error(error, error_capacity,
                               "%s: workspace needs %zu bytes, 256-byte aligned (got %zu)", what,
                               need, workspace_bytes);
        return 0;
    }
    CUtensorMap kmap, vmap;
    if (!encode_q8_map(&kmap, layer->key_pool, rows, (uint32_t)layer->block_size) ||
        !encode_q8_map(&vmap, layer->value_pool, rows, (uint32_t)layer->block_size)) {
        pkv_internal_set_error(error, error_capacity, "%s: tensor map encoding failed", what);
        return 0;
    }
    auto *base = static_cast<unsigned char *>(workspace);
    Q8Args a;
    a.query = query;
    a.out = output;
    a.kscales = layer->key_scales;
    a.vscales = layer->value_scales;
    a.claim = reinterpret_cast<uint32_t *>(base + ws.claim);
    a.counters = reinterpret_cast<uint32_t *>(base + ws.counters);
    a.part_ml = reinterpret_cast<float *>(base + ws.ml);
    a.part_o = reinterpret_cast<float *>(base + ws.o);
    a.tile_prefix = reinterpret_cast<int32_t *>(base + ws.prefix);
    a.table_stride = (int32_t)batch->table_stride;
    a.kv_heads = (int32_t)segs;
    a.heads = (int32_t)kvh;
    a.lanes = (int32_t)lanes;
    a.subs = (int32_t)subs;
    a.group = (int32_t)group;
    a.q_heads = (int32_t)q_heads;
    a.block_size = (int32_t)layer->block_size;
    a.block_count = (uint32_t)layer->block_count;
    a.scale_log2 = scale * kLog2e;
    a.bf16 = layer->dtype == PKV_DTYPE_BF16;
    a.out_f32 = output_dtype == PKV_DTYPE_F32;
    MassScratch ms = {};
    if (mass != nullptr) ms = mass_scratch(base + ws.total, batch->batch, q_heads, segs, max_seq_len);
    a.scores = ms.scores;
    a.final_ml = ms.final_ml;
    a.score_tiles = ms.tiles;
    // The 16-bit decode's rules: join in the kernel when a segment meets few
    // CTAs and there are many segments; dynamic units only then, none so small
    // that a segment of max_seq_len meets more than kInKernelMergeMax of them.
    const bool fits = ncta / (int)segs + 2 <= kInKernelMergeMax;
    a.merge_in_kernel = fits && batch->batch * segs * 2 >= (size_t)ncta;
    const size_t by_pieces = ((max_seq_len + kTcTile - 1) / kTcTile + 23) / 24;
    a.min_unit = a.merge_in_kernel ? (int32_t)(by_pieces > kMinUnitTiles ? by_pieces
                                                                              : kMinUnitTiles)
                                   : 0;
    const size_t osz = a.out_f32 ? 4 : 2;
    int ok = 1;
    for (size_t b0 = 0; ok && b0 < batch->batch; b0 += kLaunchBatch) {
        const size_t n = batch->batch - b0 < (size_t)kLaunchBatch ? batch->batch - b0
                                                                       : (size_t)kLaunchBatch;
        Q8Args s = a;
        s.batch = (int32_t)n;
        s.tables = batch->block_tables + b0 * batch->table_stride;
        s.seq_lens = batch->seq_lens + b0;
        s.query = static_cast<const char *>(query) + b0 * q_heads * hd * 2;
        s.out = static_cast<char *>(output) + b0 * q_heads * hd * osz;
        const cudaStream_t st = (cudaStream_t)stream;
        if (hd == 128)
            ok = gv == 4   ? launch<4, false>(s, kmap, vmap, ncta, st)
                 : gv == 8 ? launch<8, false>(s, kmap, vmap, ncta, st)
                           : launch<16, false>(s, kmap, vmap, ncta, st);
        else
            ok = gv == 4   ? launch<4, true>(s, kmap, vmap, ncta, st)
                 : gv == 8 ? launch<8, true>(s, kmap, vmap, ncta, st)
                           : launch<16, true>(s, kmap, vmap, ncta, st);
        if (ok && mass != nullptr) {
            const MassShape shape = {n, q_heads, kvh, hd, layer->block_size, layer->block_count,
                                     batch->table_stride, max_seq_len, gv, subs};
            ok = mass_apply(shape, ms, s.tile_prefix, s.tables, s.seq_lens, mass, stream);
        }
    }
    if (!ok) {
        pkv_internal_set_error(error, error_capacity, "%s: launch failed: %s", what,
                               cudaGetErrorString(cudaGetLastError()));
        return 0;
    }
    return 1;
}

}  // namespace
}  // namespace pkv

extern "C" {

size_t pkv_q8_decode_workspace_bytes(size_t batch, size_t q_heads, size_t kv_heads,
                                     size_t head_dim, size_t max_seq_len) {
    if (kv_heads == 0 || q_heads == 0 || q_heads % kv_heads != 0) return 0;
    return pkv::workspace_of((size_t)pkv::decode_grid() * (1 + pkv::kMaxRounds),
                             pkv::slots_of(q_heads / kv_heads, head_dim))
        .total;
}

int pkv_q8_decode(const PkvQ8Layer *layer, const PkvBatch *batch, size_t q_heads,
                  const void *query, float scale, void *output, PkvDType output_dtype,
                  size_t max_seq_len, void *workspace, size_t workspace_bytes, PkvStream stream,
                  char *error, size_t error_capacity) {
    PKV_RANGE("pkv_q8_decode");
    return pkv::q8_decode("pkv_q8_decode", layer, batch, q_heads, query, scale, output,
                          output_dtype, max_seq_len, nullptr, workspace, workspace_bytes, stream,
                          error, error_capacity);
}

int pkv_q8_decode_mass(const PkvQ8Layer *layer, const PkvBatch *batch, size_t q_heads,
                       const void *query, float scale, void *output, PkvDType output_dtype,
                       size_t max_seq_len, float *mass, void *workspace, size_t workspace_bytes,
                       PkvStream stream, char *error, size_t error_capacity) {
    PKV_RANGE("pkv_q8_decode_mass");
    const char *what = "pkv_q8_decode_mass";
    if (mass == nullptr || (uintptr_t)mass % 4 != 0) {
        pkv_internal_set_error(error, error_capacity, "%s: mass is null or not 4-byte aligned",
                               what);
        return 0;
    }
    return pkv::q8_decode(what, layer, batch, q_heads, query, scale, output, output_dtype,
                          max_seq_len, mass, workspace, workspace_bytes, stream, error,
                          error_capacity);
}

// Scratch of the larger of the two kernels behind the mass calls.
size_t pkv_decode_mass_workspace_bytes(size_t batch, size_t q_heads, size_t kv_heads,
                                       size_t head_dim, size_t max_seq_len) {
    if (kv_heads == 0 || q_heads == 0 || q_heads % kv_heads != 0) return 0;
    const size_t group = q_heads / kv_heads, lanes = pkv::mass_lanes(kv_heads, head_dim);
    const size_t gv8 = pkv::slots_of(group, head_dim), per = head_dim == 64 ? gv8 / 2 : gv8;
    const size_t q8 =
        pkv_q8_decode_workspace_bytes(batch, q_heads, kv_heads, head_dim, max_seq_len) +
        pkv::mass_scratch_bytes(batch, q_heads, lanes * ((group + per - 1) / per), gv8,
                                max_seq_len);
    const size_t half =
        (pkv_decode_workspace_bytes(batch, q_heads, head_dim, max_seq_len, 0) + 255) / 256 * 256 +
        pkv::mass_scratch_bytes(batch, q_heads, lanes, head_dim == 64 ? 2 * group : group,
                                max_seq_len);
    return q8 > half ? q8 : half;
}

int pkv_internal_take_q8_decode_fault(uint32_t *code) {
    uint32_t zero = 0;
    if (cudaMemcpyFromSymbol(code, pkv::g_q8_decode_fault, sizeof(uint32_t)) != cudaSuccess)
        return 0;
    return cudaMemcpyToSymbol(pkv::g_q8_decode_fault, &zero, sizeof(uint32_t)) == cudaSuccess;
}

}  // extern "C"
