// pkv_q8_decode.cu -- decode attention over 8-bit pages (one query token per
// sequence) on the integer tensor cores.
//
//   o = sum_t softmax_t(scale q . k_t) v_t,   k_t = kq_t ks,  v_t = vq_t vs
//
// with one scale per (page, KV head).  The pages go to the tensor cores as
// they lie: q . k_t = ks (q . kq_t) and p v = (p vs) vq, so a scale multiplies
// a score and a softmax weight, never an element, and no byte of K or V is
// converted.  The other operand is cut into signed base-256 digits:
//   q = f (d0 2^16 + d1 2^8 + d2), f a power of two per query head (22 bits),
//   p vs = F (d0 2^24 + d1 2^16 + d2 2^8 + d3), F the largest V scale of a pair
//   of tiles and a KV head over 127 * 2^24 (31 bits),
// each digit one row of the B operand of tcgen05.mma kind::i8, whose sums are
// exact 32-bit integers.  So a tile costs
//   S^T[128 tok][3 GV] = K . Qd^T   and   O^T[128 dim][4 GV] = V^T . Pd^T
// and the only roundings are those of the digits, of exp and of FP32 sums
// over tiles.  p is relative to the pair's own maximum (the step to the running
// one goes into the FP32 factor of the pair's O), so what the digits round off
// is 2^-32 of the pair's largest weight and not of the largest of all: with one
// dominant token (an attention sink) the other 10^5 together carry an output
// that digits relative to it would lose, 1% of it with the sink 16 nats up.
// Three digits would lose the sink's own pair: 255 weights of 2^-24.
// Bytes past a sequence's length are finite whatever they are and meet digits
// of zero.
//
// Bound by HBM: 2 bytes a token, KV head and column.  One persistent 512-thread
// CTA per SM:
//   warps 0-3   producers, each every fourth tile: one TMA box per page of K and
//               of V (block x 128 bytes, contiguous in the pool) and the page's
//               scales by cp.async.  16 boxes of 2 KiB and their bookkeeping
//               take one warp some 2000 cycles, in which HBM delivers a tile
//               and a half, so one warp (or one for K and one for V) cannot
//               keep up; warp 0 also claims the units
//   warps 4-7   softmax group of even pairs of tiles, warps 8-11 of odd pairs.
//               A 32 KiB tile streams in half the time of a 16-bit one, and a
//               group's chain (TMEM load, maximum over its warps, exp, digit
//               stores, O of the pair before) is latency: two groups overlap
//               theirs, and a pair of tiles shares one chain and one O.  Each
//               group carries its own running maximum, sum and output, a
//               partial of its own that the merge kernel joins: joining them
//               when a piece ends made each group wait for the other
//   warps 12, 13 one thread each issues tcgen05.mma, S and PV: a barrier wait
//               costs a thread some 90 cycles even when it is through and an
//               issue some 40, nearly a tile's time for one thread with both
//   warp 14     query warp: the digits of the next piece's query rows
// p_full of a pair (weights written) also says that its S and the O of the pair
// NB before have been read, which is what the next S and this PV overwrite.
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
constexpr int kRegsControl = 72, kRegsSoftmax = 184;
static_assert(256 * kRegsControl + 256 * kRegsSoftmax <= kThreads * 128, "register split");
constexpr int kMaxBatch = 8192;
constexpr int kLaunchBatch = 512;    // sequences of one launch: one a thread of the prologue
static_assert(kLaunchBatch == kThreads && kLaunchBatch <= (int)kMassBatch, "launch");
constexpr int kMaxGrid = 152;
constexpr int kMaxPieces = 256;      // of one segment
constexpr size_t kMinUnitTiles = 8;  // smallest dynamic unit
constexpr int kRing = 4;             // unit ids in flight between the roles
constexpr int kScaleSlots = 16;      // tiles whose scales are in shared memory
constexpr uint32_t kTileBytes = 16384;
constexpr float kDigitMax = 2130706432.f;  // 127 * 2^24: four signed digits hold +-this
constexpr float kLowest = -3.40282347e38f;  // FP32's lowest finite number

template <int GV>
struct Cfg {
    // B rows, digit-major, padded to 16: three digits a query, four a weight
    static constexpr int NQ = GV == 4 ? 16 : GV == 8 ? 32 : 48, NP = 4 * GV;
    static constexpr int KS = GV == 4 ? 6 : 5;  // K tiles in the ring
    static constexpr int VS = GV == 4 ? 6 : 5;  // V tiles
    static constexpr int NB = GV == 16 ? 2 : 4; // S, P and O buffers, one per pair of tiles
    static constexpr uint32_t QT = NQ * 128, PT = NP * 128;      // bytes of one B tile
    static constexpr uint32_t V_OFF = KS * kTileBytes;
    static constexpr uint32_t Q_OFF = V_OFF + VS * kTileBytes;
    static constexpr int QB = GV == 16 ? 2 : 4;                  // query tiles ahead
    static constexpr uint32_t P_OFF = Q_OFF + QB * QT;
    static constexpr uint32_t SC_OFF = P_OFF + 2 * NB * PT;
    static constexpr uint32_t BAR_OFF = SC_OFF + kScaleSlots * 128;
    static constexpr uint32_t MISC_OFF = BAR_OFF + 512;
    static constexpr uint32_t PREFIX_OFF = MISC_OFF + 2624;
    static constexpr uint32_t O_COL = 2 * NB * NQ;               // S of two tiles, then O
    static constexpr uint32_t TMEM_COLS = GV == 4 ? 256 : 512;
    static_assert(NB * (2 * NQ + NP) <= (int)TMEM_COLS, "tensor memory");
    // tile prefix and lengths of the sequences
    static size_t smem(int batch) { return PREFIX_OFF + 4u * (2u * (size_t)batch + 1u) + 1024u; }
    static_assert(PREFIX_OFF + 4u * (2u * kLaunchBatch + 1u) + 1024u <= 232448u, "shared memory");
};

struct Q8Args {
    const uint32_t *tables;
    const int32_t *seq_lens;
    const void *query;
    void *out;
    const float *kscales, *vscales;
    uint32_t *claim;         // [2]
    // Partials: [slot][pairs 0, 2, .. and 1, 3, .. of the piece][GV] of (m, l) and
    // of 128 columns; slots 2 u and
    // 2 u + 1 are unit u's first and last piece, whole_slot + i segment i whole.
    float *part_ml, *part_o;
    int32_t whole_slot;
    int32_t *tile_prefix;    // [batch + 1] for the merge and the mass kernels
    Sched *sched;            // for the merge kernel
    int32_t table_stride, batch;
    int32_t kv_heads;        // segments of one sequence (the schedule's name for them)
    int32_t heads;           // KV heads
    int32_t lanes, subs;     // segments = lanes * subs
    int32_t group, q_heads;
    int32_t block_size;
    uint32_t block_count;
    float scale_log2;
    int32_t min_unit;
    int32_t max_len;         // longer sequences are cut there, with a fault
    int32_t bf16, out_f32;   // row type; 32-bit outputs
    // Mass (else null): every score by stream tile and slot, and every query
    // head's final maximum and sum (pkv_mass.cuh).
    float *scores, *final_ml;
    int64_t score_tiles;
};

struct Workspace {
    size_t claim, sched, prefix, ml, o, total;
};

size_t round_up(size_t v, size_t m) { return (v + m - 1) / m * m; }

// `segments` of the launch's largest batch; a partial is two groups' GV heads.
Workspace workspace_of(size_t units, size_t segments, size_t gv) {
    const size_t partials = (2 * units + segments) * 2 * gv;
    Workspace w;
    w.claim = 0;
    w.sched = kZeroBytes;
    w.prefix = w.sched + 256;
    w.ml = w.prefix + round_up(((size_t)kLaunchBatch + 1) * 4, 256);
    w.o = w.ml + round_up(partials * 8, 256);
    w.total = w.o + round_up(partials * 512, 256);
    return w;
}

// Largest of a warp's values, in one instruction.
__device__ __forceinline__ float redux_max(float v) {
    float r;
    asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
    return r;
}

// The signed base-256 digits of u as the bytes of a word: adding 128 to the
// lower digits makes the carries, flipping their top bits takes it off.
__device__ __forceinline__ uint32_t digits3(int u) { return (uint32_t)(u + 0x8080) ^ 0x8080u; }
__device__ __forceinline__ uint32_t digits4(int u) { return ((uint32_t)u + 0x808080u) ^ 0x808080u; }

// Byte offset of (row, col) in a tile of 128-byte rows, 128-byte swizzle.
__device__ __forceinline__ uint32_t sw_byte(uint32_t row, uint32_t col) {
    return (row >> 3) * 1024u + (row & 7u) * 128u + (((col >> 4) ^ (row & 7u)) << 4) + (col & 15u);
}

// The lowest byte of v to shared memory.
__device__ __forceinline__ void store_byte(uint32_t at, uint32_t v) {
    asm volatile("st.shared.b8 [%0], %1;\n" ::"r"(at), "r"(v) : "memory");
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
    constexpr int NQ = C::NQ, NP = C::NP, KS = C::KS, VS = C::VS, NB = C::NB, QB = C::QB;
    constexpr uint32_t kIdescQK = idesc_s8(128, NQ, false, false);
    constexpr uint32_t kIdescPV = idesc_s8(128, NP, true, false);
    extern __shared__ unsigned char smem_raw[];
    unsigned char *sm = reinterpret_cast<unsigned char *>(
        (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t *bars = reinterpret_cast<uint64_t *>(sm + C::BAR_OFF);
    uint64_t *kfull = bars, *kempty = bars + 6, *vfull = bars + 12, *vempty = bars + 18;
    uint64_t *s_full = bars + 24, *p_full = bars + 28, *o_full = bars + 32;
    uint64_t *q_full = bars + 36, *q_empty = bars + 40;  // a piece's digits and descriptor
    uint64_t *ring_full = bars + 44, *ring_empty = bars + 48;
    unsigned char *misc = sm + C::MISC_OFF;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(misc);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(misc + 4);
    volatile int *ring = reinterpret_cast<volatile int *>(misc + 32);        // [kRing]
    int *scan = reinterpret_cast<int *>(misc + 64);                          // [12]
    Sched *sched = reinterpret_cast<Sched *>(misc + 128);
    float *qscale = reinterpret_cast<float *>(misc + 256);                   // [QB][16]
    volatile int4 *desc = reinterpret_cast<volatile int4 *>(misc + 512);     // [QB], see below
    float *red = reinterpret_cast<float *>(misc + 576);                      // [2 groups][2][16][4]
    float *lred = reinterpret_cast<float *>(misc + 1600);                    // [2 groups][2][4][16]
    float *scales = reinterpret_cast<float *>(sm + C::SC_OFF);  // [slot][K0, V0, K1, V1][8]
    int *prefix = reinterpret_cast<int *>(sm + C::PREFIX_OFF);
    int *lens = prefix + a.batch + 1;

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (tid == 0) {
        for (int s = 0; s < KS; ++s) {
            mbar_init(&kfull[s], 33);  // TMA bytes, and each lane's scale copies
            mbar_init(&kempty[s], 1);
        }
        for (int s = 0; s < VS; ++s) {
            mbar_init(&vfull[s], 1);
            mbar_init(&vempty[s], 1);
        }
        for (int i = 0; i < NB; ++i) {
            mbar_init(&s_full[i], 2);  // the MMAs, and the issuer that saw the scales
            mbar_init(&o_full[i], 1);
            mbar_init(&p_full[i], 128);
        }
        for (int i = 0; i < QB; ++i) {
            mbar_init(&q_full[i], 32);
            mbar_init(&q_empty[i], 258);  // both groups saw their last S, both issuers started
        }
        for (int i = 0; i < kRing; ++i) {
            mbar_init(&ring_full[i], 1);
            mbar_init(&ring_empty[i], 4);  // three producers, query warp
        }
        *abort_flag = 0;
        fence_mbar_init();
    }
    // B rows past the digits (and, paired, the other head's columns) stay zero
    for (int i = tid; i < (int)((QB * C::QT + 2 * NB * C::PT) / 16); i += kThreads)
        reinterpret_cast<uint4 *>(sm + C::Q_OFF)[i] = make_uint4(0, 0, 0, 0);
    if (warp == 12) {
        tmem_alloc(tmem_slot, C::TMEM_COLS);
        tmem_relinquish();
    }
    if (tid == 0) {
        tma_prefetch_desc(&kmap);
        tma_prefetch_desc(&vmap);
    }
    // Lengths and block tables (the first 2 MiB) into L2 while the kernel before
    // this one finishes (a hint: nothing is read before the wait).
    {
        const size_t all = (size_t)a.batch * (size_t)a.table_stride * 4u;
        const size_t bytes = all < (size_t(2) << 20) ? all : (size_t(2) << 20);
        const char *tb = reinterpret_cast<const char *>(a.tables);
        for (size_t off = ((size_t)blockIdx.x * kThreads + tid) * 128u; off < bytes;
             off += (size_t)gridDim.x * kThreads * 128u)
            prefetch_l2(tb + off);
        if (tid < a.batch && tid % 32 == 0) prefetch_l2(a.seq_lens + tid);
    }
    pdl_wait();
    pdl_launch_dependents();
    // Exclusive prefix of tiles (one sequence a thread), lengths and schedule.
    {
        int len = tid < a.batch ? max(0, __ldg(a.seq_lens + tid)) : 0;
        if (len > a.max_len) {
            if (blockIdx.x == 0) record_fault(&g_q8_decode_fault, kFaultPositionOutOfRange);
            len = a.max_len;
        }
        const int tiles = (len + kTcTile - 1) / kTcTile * a.kv_heads;
        int incl = tiles;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += v;
        }
        if (lane == 31) scan[warp] = incl;
        __syncthreads();
        int before = 0, total = 0;
#pragma unroll
        for (int w = 0; w < kThreads / 32; ++w) {
            const int v = scan[w];
            if (w < warp) before += v;
            total += v;
        }
        if (tid < a.batch) {
            prefix[tid] = before + incl - tiles;
            lens[tid] = len;
        }
        if (tid == 0) {
            prefix[a.batch] = total;
            make_sched(*sched, total, (int)gridDim.x, a.min_unit);
        }
    }
    fence_proxy_async_smem();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    const int64_t total_tiles = prefix[a.batch];
    const Sched &sc = *sched;
    const bool works = (int)blockIdx.x < sc.n && total_tiles > 0;
    const int n_units = sched_units(sc);
    uint32_t *fault = &g_q8_decode_fault;
    if (blockIdx.x == 0) {
        for (int b = tid; b <= a.batch; b += kThreads) a.tile_prefix[b] = prefix[b];
        if (tid == 0) *a.sched = sc;
    }

    const int page_shift = 31 - __clz(a.block_size);
    if (warp < 4 || warp >= 12) {
    setmaxnreg_dec<kRegsControl>();
    if (warp < kProducers) {
        // ----------------------------- producers -----------------------------
        // pages leave L2 first: the partials and the scores stay for the kernels
        // behind this one
        const uint64_t once = policy_evict_first();
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
                const int L = lens[P.b];
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
                    // lanes 0-7 one page each
                    const uint32_t off = (uint32_t)page << (page_shift + 7);
                    const int32_t y =
                        (int32_t)((pid * (uint32_t)a.lanes + (uint32_t)kl) << page_shift);
                    ok = __all_sync(0xffffffffu, mbar_wait(&kempty[ks], ((jj / KS) & 1) ^ 1,
                                                           abort_flag, fault));
                    if (!ok) break;
                    if (lane == 0) mbar_arrive_expect_tx(&kfull[ks], bytes);
                    __syncwarp();
                    if (good && lane < 8)
                        tma_load_2d_policy(sm + ks * kTileBytes + off, &kmap, &kfull[ks], 0, y,
                                           once);
                    // scales: kind = lane / 8 (K0, V0, K1, V1 of the lane's heads)
                    const int head = (PAIR ? 2 * kl : kl) + (lane >> 4);
                    const bool want = good && head < a.heads && (PAIR || lane < 16);
                    const float *src = (lane & 8) != 0 ? a.vscales : a.kscales;
                    cp_async4_or_zero(scales + (jj % kScaleSlots) * 32 + lane,
                                      want ? src + (int64_t)pid * a.heads + head : src, want);
                    cp_async_mbar_arrive(&kfull[ks]);
                    ok = __all_sync(0xffffffffu, mbar_wait(&vempty[vs], ((jj / VS) & 1) ^ 1,
                                                           abort_flag, fault));
                    if (!ok) break;
                    if (lane == 0) mbar_arrive_expect_tx(&vfull[vs], bytes);
                    __syncwarp();
                    if (good && lane < 8)
                        tma_load_2d_policy(sm + C::V_OFF + vs * kTileBytes + off, &vmap, &vfull[vs],
                                           0, y, once);
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
        // Walks the pieces ahead of the issuers and the groups and hands each of
        // them on as query digits, their scales and a descriptor: tiles (0: no
        // more), positions left from its first tile, partial slot, stream tile.
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
            const int64_t us = u < 0 ? 0 : unit_start(sc, u), ue = u < 0 ? 1 : unit_start(sc, u + 1);
            for (int64_t t = us; ok && t < ue;) {
                const uint32_t qb_i = qi % QB;
                ok = __all_sync(0xffffffffu, mbar_wait(&q_empty[qb_i], ((qi / QB) & 1) ^ 1,
                                                       abort_flag, fault));
                if (!ok) break;
                if (u < 0) {
                    if (lane == 0) desc[qb_i].x = 0;
                    mbar_arrive(&q_full[qb_i]);
                    ok = false;
                    break;
                }
                const Piece P = piece_at(t, ue, prefix, a);
                if (lane == 0) {
                    desc[qb_i].x = P.k1 - P.k0;
                    desc[qb_i].y = lens[P.b] - P.k0 * kTcTile;
                    // a cut piece is its unit's first or last; a whole segment has
                    // its own place behind those
                    desc[qb_i].z = P.k0 == 0 && P.k1 == P.nt
                                       ? a.whole_slot + P.b * a.kv_heads + P.g
                                       : u * 2 + (t == us ? 0 : 1);
                    desc[qb_i].w = (int)t;
                }
                t += P.k1 - P.k0;
                // Query digits: lane holds 4 columns of a row (head_dim 64: the
                // first half warp, at the head's half of the 128 columns).
                constexpr int HD = PAIR ? 64 : 128;
                unsigned char *qb = sm + C::Q_OFF + qb_i * C::QT;
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
                        for (int e = 0; e < 4; ++e) d[e] = digits3(__float2int_rn(x[e] * f));
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
                            qscale[qb_i * 16 + h] =
                                top >= 0x7f800000u ? __uint_as_float(0x7fc00000u) : back * a.scale_log2;
                    }
                }
                fence_proxy_async_smem();
                mbar_arrive(&q_full[qb_i]);
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
            uint32_t j = 0, pc = 0;  // tiles, pairs
            bool ok = true;
            for (uint32_t qi = 0; ok; ++qi) {
                const uint32_t qb_i = qi % QB;
                if (!mbar_wait(&q_full[qb_i], (qi / QB) & 1, abort_flag, fault)) break;
                const int n = desc[qb_i].x;
                mbar_arrive(&q_empty[qb_i]);
                if (n == 0) break;
                const uint64_t qd = qdesc + (uint64_t)(qb_i * (C::QT >> 4));
                for (int k = 0; ok && k < n; k += 2, ++pc) {
                    const uint32_t buf = pc % NB;
                    const int n2 = min(2, n - k);
                    if (warp == 12) {
                        ok = mbar_wait(&p_full[buf], ((pc / NB) & 1) ^ 1, abort_flag, fault);
                        for (int i = 0; ok && i < n2; ++i, ++j) {
                            const uint32_t stage = j % KS;
                            ok = mbar_wait(&kfull[stage], (j / KS) & 1, abort_flag, fault);
                            if (!ok) break;
                            tc_fence_after();
                            const uint64_t ad = kdesc + (uint64_t)(stage * (kTileBytes >> 4));
                            const uint32_t dst = tmem + (2 * buf + i) * NQ;
                            mma_i8_ss_at<0, 0>(dst, ad, qd, kIdescQK, 0);
                            mma_i8_ss_at<2, 2>(dst, ad, qd, kIdescQK, 1);
                            mma_i8_ss_at<4, 4>(dst, ad, qd, kIdescQK, 1);
                            mma_i8_ss_at<6, 6>(dst, ad, qd, kIdescQK, 1);
                            mma_commit(&kempty[stage]);
                        }
                        mma_commit(&s_full[buf]);
                        // this thread saw the scales land: its own arrival passes
                        // them on to the softmax group
                        mbar_arrive(&s_full[buf]);
                    } else {
                        ok = mbar_wait(&p_full[buf], (pc / NB) & 1, abort_flag, fault);
                        const uint32_t dst = tmem + C::O_COL + buf * NP;
                        for (int i = 0; ok && i < n2; ++i, ++j) {
                            const uint32_t stage = j % VS;
                            ok = mbar_wait(&vfull[stage], (j / VS) & 1, abort_flag, fault);
                            if (!ok) break;
                            tc_fence_after();
                            const uint64_t ad = vdesc + (uint64_t)(stage * (kTileBytes >> 4));
                            const uint64_t bd = pdesc + (uint64_t)((2 * buf + i) * (C::PT >> 4));
                            mma_i8_ss_at<0, 0>(dst, ad, bd, kIdescPV, i);
                            mma_i8_ss_at<256, 2>(dst, ad, bd, kIdescPV, 1);
                            mma_i8_ss_at<512, 4>(dst, ad, bd, kIdescPV, 1);
                            mma_i8_ss_at<768, 6>(dst, ad, bd, kIdescPV, 1);
                            mma_commit(&vempty[stage]);
                        }
                        mma_commit(&o_full[buf]);
                    }
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
        uint32_t j = 0, pc = 0;  // tiles, pairs
        bool aborted = false;
        auto await = [&](uint64_t *bar, uint32_t par) {
            aborted = aborted || !__all_sync(0xffffffffu, mbar_wait(bar, par, abort_flag, fault));
        };
        for (uint32_t qi = 0;; ++qi) {
                const uint32_t qb_i = qi % QB;
                await(&q_full[qb_i], (qi / QB) & 1);
                // all warps of the group leave together, also where only some
                // of them saw a wait give up
                aborted = named_barrier_or(1 + grp, 128, aborted);
                const int n = desc[qb_i].x;
                if (aborted || n == 0) break;
                const int len = desc[qb_i].y, slot = desc[qb_i].z, tile0 = desc[qb_i].w;
                float m_run[GV], l_part[GV], acc[GV], alpha_prev[GV], f_prev[GV];
#pragma unroll
                for (int h = 0; h < GV; ++h) {
                    m_run[h] = -INFINITY;
                    l_part[h] = 0.f;
                    acc[h] = 0.f;
                }
                // COLS columns of TMEM at `col`, this thread's row
                auto load_cols = [&](uint32_t col, auto &v) {
                    constexpr int COLS = sizeof(v) / sizeof(v[0]);
#pragma unroll
                    for (int i = 0; i < COLS; ++i) v[i] = 0.f;
                    if (aborted) return;
                    if constexpr (COLS > 32) {
                        tmem_ld_32x32b<32>(tmem + col + lane_off,
                                           *reinterpret_cast<float(*)[32]>(&v[0]));
                        tmem_ld_32x32b<COLS - 32>(tmem + col + 32 + lane_off,
                                                  *reinterpret_cast<float(*)[COLS - 32]>(&v[32]));
                    } else {
                        tmem_ld_32x32b<COLS>(tmem + col + lane_off, v);
                    }
                };
                // two digit sums as one whole number (a sum is 2^22 at most)
                auto two = [](float hi, float lo) {
                    return __float_as_int(hi) * 256 + __float_as_int(lo);
                };
                // slot h's score from its three digit sums
                auto number = [&](const float (&v)[NQ], int h) -> float {
                    return fmaf((float)__float_as_int(v[h]), 65536.f,
                                (float)two(v[GV + h], v[2 * GV + h]));
                };
                // O of this group's previous pair from its four digit sums; its
                // weights were cut by a factor that f_prev takes back
                auto fold = [&](uint32_t pair) {
                    const uint32_t buf = pair % NB;
                    await(&o_full[buf], (pair / NB) & 1);
                    tc_fence_after();
                    // (1 / kDigitMax here and not in f_prev, which would leave FP32
                    // with V scales below 2^-95)
                    auto add = [&](const float (&o)[2 * GV], float unit) {
#pragma unroll
                        for (int h = 0; h < GV; ++h)
                            acc[h] = fmaf((float)two(o[h], o[GV + h]) * unit, f_prev[h], acc[h]);
                    };
#pragma unroll
                    for (int h = 0; h < GV; ++h) acc[h] *= alpha_prev[h];
                    if constexpr (GV == 16) {  // two digits at a time: registers
                        float o[2 * GV];
                        load_cols(C::O_COL + buf * NP, o);
                        tmem_wait_ld();
                        add(o, 65536.f / kDigitMax);
                        load_cols(C::O_COL + buf * NP + 2 * GV, o);
                        tmem_wait_ld();
                        add(o, 1.f / kDigitMax);
                    } else {
                        float o[2][2 * GV];
                        load_cols(C::O_COL + buf * NP, reinterpret_cast<float (&)[NP]>(o));
                        tmem_wait_ld();
                        add(o[0], 65536.f / kDigitMax);
                        add(o[1], 1.f / kDigitMax);
                    }
                    tc_fence_before();
                };
                int64_t mine = -1;  // this group's previous pair of the piece
                // The group with the piece's first pair fills its first partial:
                // which of the two that is depends on the units this CTA claimed
                // before, and with it the order of the merge's sums would.
                const int part = grp ^ (int)(pc & 1);
                for (int k = 0; k < n; k += 2, ++pc) {
                    const int n2 = min(2, n - k);
                    const uint32_t j0 = j;
                    j += (uint32_t)n2;
                    if ((int)(pc & 1) != grp) continue;
                    const uint32_t buf = pc % NB;
                    await(&s_full[buf], (pc / NB) & 1);
                    // Both tiles' sums at once, or with 16 heads one tile at a time
                    // (registers); past an odd end: not used
                    constexpr int AT_ONCE = GV == 16 ? 1 : 2;
                    float s[AT_ONCE][NQ];
                    tc_fence_after();
#pragma unroll
                    for (int i = 0; i < AT_ONCE; ++i) load_cols((2 * buf + i) * NQ, s[i]);
                    // scales: a token's own, and the largest V scale of the pair
                    float ks[2][PAIR ? 2 : 1], pf[2][PAIR ? 2 : 1], top[PAIR ? 2 : 1];
                    const float *sl0 = scales + (j0 % kScaleSlots) * 32;
                    const float *sl1 = n2 > 1 ? scales + ((j0 + 1) % kScaleSlots) * 32 : sl0;
#pragma unroll
                    for (int e = 0; e < (PAIR ? 2 : 1); ++e) {
                        const float4 v0 = *reinterpret_cast<const float4 *>(sl0 + e * 16 + 8);
                        const float4 v1 = *reinterpret_cast<const float4 *>(sl0 + e * 16 + 12);
                        const float4 v2 = *reinterpret_cast<const float4 *>(sl1 + e * 16 + 8);
                        const float4 v3 = *reinterpret_cast<const float4 *>(sl1 + e * 16 + 12);
                        top[e] = fmaxf(
                            kQ8MinScale,
                            fmaxf(fmaxf(fmaxf(fmaxf(v0.x, v0.y), fmaxf(v0.z, v0.w)),
                                        fmaxf(fmaxf(v1.x, v1.y), fmaxf(v1.z, v1.w))),
                                  fmaxf(fmaxf(fmaxf(v2.x, v2.y), fmaxf(v2.z, v2.w)),
                                        fmaxf(fmaxf(v3.x, v3.y), fmaxf(v3.z, v3.w)))));
                        // weight digits: p * (vs / top) * kDigitMax
                        const float inv = __fdividef(1.f, top[e]);
                        const int at = e * 16 + (row >> page_shift);
                        ks[0][e] = sl0[at];
                        ks[1][e] = sl1[at];
                        pf[0][e] = sl0[at + 8] * inv * kDigitMax;
                        pf[1][e] = sl1[at + 8] * inv * kDigitMax;
                    }
                    const int left = len - k * kTcTile;
                    const bool live[2] = {row < left, row + kTcTile < left && n2 > 1};
                    // two buffers: a warp writes a pair's maxima only after all
                    // read those of the group's pair before the last
                    float *myred = red + grp * 128 + ((pc >> 1) & 1) * 64;  // [slot][warp]
                    float x[2][GV];
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        if (AT_ONCE == 1 && i == 1) load_cols((2 * buf + 1) * NQ, s[0]);
                        if (AT_ONCE == 1 || i == 0) tmem_wait_ld();
#pragma unroll
                        for (int h = 0; h < GV; ++h) {
                            const int e = PAIR && h >= GV / 2 ? 1 : 0;
                            x[i][h] = live[i] ? number(s[i % AT_ONCE], h) *
                                                    (qscale[qb_i * 16 + h] * ks[i][e])
                                              : -INFINITY;
                        }
                    }
                    tc_fence_before();
#pragma unroll
                    for (int h = 0; h < GV; ++h) {
                        const float wm = redux_max(fmaxf(x[0][h], x[1][h]));
                        if (lane == 0) myred[h * 4 + q4] = wm;
                    }
                    if constexpr (NB == 2)  // the weights below overwrite the previous pair's
                        if (mine >= 0) fold((uint32_t)mine);
                    group_sync();
                    float alpha[GV], f_cur[GV];
                    // this token's column of the swizzled B tiles: row r's byte is at
                    // ((r & 7) << 4 ^ column) + 128 r, one operation a store (with 16
                    // heads the generic form took 448 us of what is now 416, 64
                    // sequences of 512-32k)
                    const uint32_t pcol = smem_u32(sm + C::P_OFF + 2 * buf * C::PT) + (uint32_t)row;
#pragma unroll
                    for (int h = 0; h < GV; ++h) {
                        const int e = PAIR && h >= GV / 2 ? 1 : 0;
                        const float4 r = *reinterpret_cast<const float4 *>(myred + h * 4);
                        // the pair's maximum (finite, should every score be -inf)
                        const float m_pair =
                            fmaxf(kLowest, fmaxf(fmaxf(r.x, r.y), fmaxf(r.z, r.w)));
                        // steps to the new running maximum: one of them is 1
                        const float up = m_run[h] - m_pair;
                        const float less = ex2_fast(-fabsf(up));
                        const float step = up >= 0.f ? less : 1.f;
                        alpha[h] = up >= 0.f ? 1.f : less;
                        m_run[h] = fmaxf(m_run[h], m_pair);
                        const float p0 = ex2_fast(x[0][h] - m_pair);
                        const float p1 = ex2_fast(x[1][h] - m_pair);
                        l_part[h] = fmaf(l_part[h], alpha[h], (p0 + p1) * step);
                        f_cur[h] = top[e] * step;
                        const uint32_t d0 = digits4(__float2int_rn(p0 * pf[0][e]));
                        const uint32_t d1 = digits4(__float2int_rn(p1 * pf[1][e]));
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const uint32_t r = (uint32_t)(i * GV + h);
                            const uint32_t at = (pcol ^ (r & 7u) << 4) + r * 128u;
                            store_byte(at, d0 >> (24 - 8 * i));
                            store_byte(at + C::PT, d1 >> (24 - 8 * i));
                        }
                    }
                    fence_proxy_async_smem();
                    mbar_arrive(&p_full[buf]);
                    // scores for the mass: behind the fence, which would wait for
                    // these stores (one sequence of 131072, 64 heads: 84 us so)
                    if (a.scores != nullptr && tile0 + k + n2 <= a.score_tiles) {
                        float *sp = a.scores + (int64_t)(tile0 + k) * GV * 128 + row;
#pragma unroll
                        for (int h = 0; h < GV; ++h) {
                            sp[h * 128] = x[0][h];
                            if (n2 > 1) sp[(GV + h) * 128] = x[1][h];
                        }
                    }
                    if constexpr (NB != 2)
                        if (mine >= 0) fold((uint32_t)mine);
                    mine = pc;
#pragma unroll
                    for (int h = 0; h < GV; ++h) {
                        alpha_prev[h] = alpha[h];
                        f_prev[h] = f_cur[h];
                    }
                }
                mbar_arrive(&q_empty[qb_i]);  // the piece's last S is done in both groups
                // ---- this group's partial: the merge kernel joins the groups' ----
                // (a group without a pair in the piece leaves m = -inf, and no O)
                float *my_l = lred + grp * 128 + (qi & 1) * 64;
#pragma unroll
                for (int h = 0; h < GV; ++h) {
                    const float ls = warp_sum(l_part[h]);
                    if (lane == 0) my_l[q4 * 16 + h] = ls;
                }
                const int64_t at = ((int64_t)slot * 2 + part) * GV;
                if (mine >= 0) {
                    fold((uint32_t)mine);
#pragma unroll
                    for (int h = 0; h < GV; ++h) a.part_o[(at + h) * 128 + row] = acc[h];
                }
                group_sync();
#pragma unroll
                for (int h = 0; h < GV; ++h)
                    if (wt == h)
                        *reinterpret_cast<float2 *>(a.part_ml + (at + h) * 2) = make_float2(
                            m_run[h], (my_l[h] + my_l[16 + h]) + (my_l[32 + h] + my_l[48 + h]));
        }
        // empty sequences: zeros
        if (grp == 0)
            for (int b = blockIdx.x; b < a.batch; b += gridDim.x) {
                if (lens[b] > 0) continue;
                const int n = a.q_heads * (PAIR ? 64 : 128);
                for (int i = wt; i < n; i += 128) store_out(a, (int64_t)b * n + i, 0.f);
            }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 12) tmem_dealloc(tmem, C::TMEM_COLS);
}

// Joins a segment's partials (two groups' for each of its pieces) into its
// output; a CTA takes HPC of a segment's query heads: all of them where there
// are segments enough, one where few long segments have many pieces each.  A merge inside the decode kernel (a fence, a
// ticket, two rounds of dependent loads: about 5 us) falls to the CTA that ends
// last, after its own work and once for each of its pieces: 27 us of 200 at 64
// sequences of 512-32k.  Here all run at once, their CTAs wait on the SMs as the
// decode's leave them, and the partials' loads go out with those of the weights.
constexpr int kMergeThreads = 256;
template <int GV, bool PAIR, int HPC>
__global__ void __launch_bounds__(kMergeThreads) q8_merge_kernel(const Q8Args a) {
    pdl_launch_dependents();
    pdl_wait();
    __shared__ float w[2 * kMaxPieces * HPC];
    __shared__ int slot[2 * kMaxPieces];
    __shared__ float4 part[kMergeThreads];
    __shared__ Sched sc;
    const int tid = threadIdx.x, lane = tid & 31, b = blockIdx.y;
    const int g = blockIdx.x / (GV / HPC), h0 = blockIdx.x % (GV / HPC) * HPC;
    if (HPC == 1 && head_at<GV, PAIR>(a, g, h0) < 0) return;
    const int first = __ldcg(a.tile_prefix + b), next = __ldcg(a.tile_prefix + b + 1);
    if (tid < (int)(sizeof(Sched) / 4))
        reinterpret_cast<int *>(&sc)[tid] = __ldcg(reinterpret_cast<const int *>(a.sched) + tid);
    if (next == first) return;
    __syncthreads();
    const int nt = (next - first) / a.kv_heads;
    const int64_t seg = first + (int64_t)g * nt;
    const int u0 = unit_of_tile(sc, seg);
    const int np = (unit_of_tile(sc, seg + nt - 1) - u0 + 1) * 2;  // partials
    if (np > 2 * kMaxPieces) {  // cannot happen with the host's choice of units
        if (tid == 0) record_fault(&g_q8_decode_fault, kFaultPositionOutOfRange);
        return;
    }
    for (int c = tid; c < np; c += kMergeThreads)
        slot[c] = (np == 2 ? a.whole_slot + b * a.kv_heads + g
                           : (u0 + c / 2) * 2 + unit_slot(sc, u0 + c / 2, seg)) *
                      2 +
                  (c & 1);
    __syncthreads();
    // thread: one float4 of the HPC x 128 columns, every SHARES-th partial
    constexpr int COLS = HPC * 32;
    constexpr int SHARES = COLS < kMergeThreads ? kMergeThreads / COLS : 1;
    constexpr int AHEAD = 4;  // partials loaded before the weights are known
    for (int f0 = 0; f0 < COLS; f0 += kMergeThreads) {
        const int f = f0 + tid % COLS, share = tid / COLS;
        auto load = [&](int i) {
            const int c = share + i * SHARES;
            return c < np ? __ldcg(reinterpret_cast<const float4 *>(
                                       a.part_o + ((int64_t)slot[c] * GV + h0) * 128) + f)
                          : make_float4(0.f, 0.f, 0.f, 0.f);
        };
        float4 v[AHEAD];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) v[i] = load(i);
        if (f0 == 0) {
            for (int h = tid >> 5; h < HPC; h += kMergeThreads / 32) {  // a warp a head
                auto ml_at = [&](int c) {
                    return __ldcg(reinterpret_cast<const float2 *>(
                        a.part_ml + ((int64_t)slot[c] * GV + h0 + h) * 2));
                };
                float mx = -INFINITY, lt = 0.f;
                for (int c = lane; c < np; c += 32) mx = fmaxf(mx, ml_at(c).x);
                mx = warp_max(mx);
                for (int c = lane; c < np; c += 32) {
                    const float2 ml = ml_at(c);
                    // a query that is not a number: every m is -inf, l is not 0
                    const float k = ml.x == mx ? 1.f : exp2f(ml.x - mx);
                    lt += ml.y == 0.f ? 0.f : ml.y * k;
                    w[c * HPC + h] = ml.y == 0.f ? 0.f : k;  // nothing there: O was not written
                }
                lt = warp_sum(lt);
                const float inv = lt == 0.f ? 0.f : 1.f / lt;
                for (int c = lane; c < np; c += 32) w[c * HPC + h] *= inv;
                const int qh = head_at<GV, PAIR>(a, g, h0 + h);
                if (a.final_ml != nullptr && qh >= 0 && lane == 0) store_ml(a, b, qh, mx, lt);
            }
            __syncthreads();
        }
        const int h = f >> 5;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int i0 = 0; share + i0 * SHARES < np; i0 += AHEAD) {
            if (i0 > 0) {
#pragma unroll
                for (int i = 0; i < AHEAD; ++i) v[i] = load(i0 + i);
            }
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) {
                const int c = share + (i0 + i) * SHARES;
                const float k = c < np ? w[c * HPC + h] : 0.f;
                if (k == 0.f) continue;
                o.x = fmaf(k, v[i].x, o.x);
                o.y = fmaf(k, v[i].y, o.y);
                o.z = fmaf(k, v[i].z, o.z);
                o.w = fmaf(k, v[i].w, o.w);
            }
        }
        if constexpr (SHARES > 1) {
            part[tid] = o;
            __syncthreads();
            if (share > 0) return;
#pragma unroll
            for (int k = 1; k < SHARES; ++k) {
                const float4 r = part[k * COLS + tid];
                o.x += r.x;
                o.y += r.y;
                o.z += r.z;
                o.w += r.w;
            }
        }
        const int qh = head_at<GV, PAIR>(a, g, h0 + h), d = (f & 31) * 4;
        if (qh >= 0 && owns<PAIR>(GV, h0 + h, d)) {
            const int64_t at = out_at<PAIR>(a, b, qh, d);
            store_out(a, at, o.x);
            store_out(a, at + 1, o.y);
            store_out(a, at + 2, o.z);
            store_out(a, at + 3, o.w);
        }
    }
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
    // One head a CTA where that makes two CTAs an SM or fewer (one sequence of
    // 131072, 64 heads: 56 us against 67), else the start of more CTAs costs
    // more than their parallelism gives (32 sequences, 256 segments: 42 us
    // against 38 with all heads in one).
    const bool all_heads = (int64_t)a.kv_heads * GV * a.batch > 2 * ncta;
    cfg.gridDim = dim3(all_heads ? a.kv_heads : a.kv_heads * GV, a.batch);
    cfg.blockDim = dim3(kMergeThreads);
    cfg.dynamicSmemBytes = 0;
    if ((all_heads ? cudaLaunchKernelEx(&cfg, q8_merge_kernel<GV, PAIR, GV>, a)
                   : cudaLaunchKernelEx(&cfg, q8_merge_kernel<GV, PAIR, 1>, a)) != cudaSuccess)
        return 0;
    return cudaGetLastError() == cudaSuccess;
}

// Slots of one segment: the smallest that holds the group (both groups of a
// head_dim 64 pair), else 16 and several segments a lane.
size_t slots_of(size_t group, size_t head_dim) {
    const size_t want = head_dim == 64 ? 2 * group : group;
    return want <= 4 ? 4 : want <= 8 ? 8 : 16;
}

// Segments of one lane: groups above a segment's slots take several.
size_t subs_of(size_t group, size_t head_dim) {
    const size_t gv = slots_of(group, head_dim), per = head_dim == 64 ? gv / 2 : gv;
    return (group + per - 1) / per;
}

Workspace decode_space(size_t batch, size_t group, size_t kv_heads, size_t head_dim) {
    const size_t n = batch < (size_t)kLaunchBatch ? batch : (size_t)kLaunchBatch;
    return workspace_of((size_t)decode_grid() * (1 + kMaxRounds),
                        n * q8_lanes(kv_heads, head_dim) * subs_of(group, head_dim),
                        slots_of(group, head_dim));
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
    // the stream's tiles are counted in 32 bits
    if (lanes * subs_of(q_heads / kvh, hd) * ((max_seq_len + 127) / 128) >
        (size_t)INT32_MAX / kLaunchBatch) {
        pkv_internal_set_error(error, error_capacity,
                               "%s: max_seq_len times KV heads is too large", what);
        return 0;
    }
    if ((uintptr_t)query % 16 != 0 || (uintptr_t)output % 4 != 0) {
        pkv_internal_set_error(error, error_capacity,
                               "%s: query must be 16-byte, output 4-byte aligned", what);
        return 0;
    }
    const size_t group = q_heads / kvh, gv = slots_of(group, hd);
    const size_t subs = subs_of(group, hd);
    const size_t segs = lanes * subs;
    const int ncta = decode_grid();
    const Workspace ws = decode_space(batch->batch, group, kvh, hd);
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
    a.part_ml = reinterpret_cast<float *>(base + ws.ml);
    a.part_o = reinterpret_cast<float *>(base + ws.o);
    a.whole_slot = 2 * ncta * (1 + kMaxRounds);
    a.tile_prefix = reinterpret_cast<int32_t *>(base + ws.prefix);
    a.sched = reinterpret_cast<Sched *>(base + ws.sched);
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
    a.max_len = (int32_t)max_seq_len;
    a.bf16 = layer->dtype == PKV_DTYPE_BF16;
    a.out_f32 = output_dtype == PKV_DTYPE_F32;
    MassScratch ms = {};
    if (mass != nullptr) ms = mass_scratch(base + ws.total, batch->batch, q_heads, segs, max_seq_len);
    a.scores = ms.scores;
    a.final_ml = ms.final_ml;
    a.score_tiles = ms.tiles;
    // Pieces of one segment: the dynamic tail is at most a quarter of the
    // stream, so static units hold 3/4 of T / ncta tiles or more and a segment
    // meets at most 4/3 ncta + 2 <= 205 of them; min_unit is chosen so that a
    // segment of max_seq_len meets at most 42 dynamic ones: kMaxPieces holds.
    const size_t by_pieces = (max_seq_len + kTcTile - 1) / kTcTile / 40 + 1;
    a.min_unit = (int32_t)(by_pieces > kMinUnitTiles ? by_pieces : kMinUnitTiles);
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
    return pkv::decode_space(batch, q_heads / kv_heads, kv_heads, head_dim).total;
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
    if (mass == nullptr || (uintptr_t)mass % 16 != 0) {
        pkv_internal_set_error(error, error_capacity, "%s: mass is null or not 16-byte aligned",
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
    const size_t q8 =
        pkv_q8_decode_workspace_bytes(batch, q_heads, kv_heads, head_dim, max_seq_len) +
        pkv::mass_scratch_bytes(batch, q_heads, lanes * pkv::subs_of(group, head_dim),
                                pkv::slots_of(group, head_dim), max_seq_len);
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
