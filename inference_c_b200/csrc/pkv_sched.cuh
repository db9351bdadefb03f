// pkv_sched.cuh -- the stream-K work split of the tensor-core decode kernels.
//
// The 128-token tiles of all (sequence, segment) pairs form one stream.  Most
// of it is cut evenly over the CTAs (static units); on long launches the last
// part is cut into smaller units that CTAs claim as they finish.  Args is a
// kernel's argument struct: batch, seq_lens, kv_heads (the segments of one
// sequence) and max_len (longer sequences are cut there) are read.
#pragma once

#include <stddef.h>

#include "pkv_device.cuh"

namespace pkv {

constexpr int kTcTile = 128;    // tokens of one tile
constexpr int kMaxRounds = 5;   // dynamic rounds
constexpr int kTcMaxGrid = 256;
constexpr int kTcMaxUnits = kTcMaxGrid * (1 + kMaxRounds);  // work units of one launch

// Both decode kernels keep what must be zero between launches in the first
// kZeroBytes of their workspace (two claim words, then the 16-bit decode's
// merge tickets, by unit), so one workspace serves either in turn.
constexpr size_t kTicketsAt = 256;
constexpr size_t kZeroBytes = kTicketsAt + (kTcMaxUnits * 4 + 255) / 256 * 256;

// Work units of one launch; every CTA (and the merge kernel) derives the same
// schedule from T, the grid and the smallest unit.
struct Sched {
    int64_t T, S;  // tiles; static region [0, S)
    int n;         // working CTAs = static units
    int rounds;    // dynamic rounds of n units each
    int size[kMaxRounds];
};

// Written in place (shared memory in the decode kernel: no local copy).
__host__ __device__ inline void make_sched(Sched &s, int64_t T, int grid, int min_unit) {
    s.T = T;
    s.n = (int)(T < (int64_t)grid ? (T > 1 ? T : 1) : grid);
    s.rounds = 0;
    int64_t dyn = 0;
    // an eighth of a CTA's share first, halving down to min_unit: the
    // dynamic tiles stay under a quarter of T, every unit >= min_unit
    int64_t sz = T / ((int64_t)s.n * 8);
    if (min_unit > 0 && sz >= min_unit) {
        while (s.rounds < kMaxRounds) {
            const int64_t cur = sz > min_unit ? sz : min_unit;
            s.size[s.rounds++] = (int)cur;
            dyn += cur * s.n;
            if (cur == min_unit) break;
            sz >>= 1;
        }
    }
    s.S = T - dyn;
}

__host__ __device__ inline int sched_units(const Sched &s) { return s.n * (1 + s.rounds); }

// First tile of unit u (T for u == sched_units).
__device__ __forceinline__ int64_t unit_start(const Sched &s, int u) {
    if (u < s.n) return s.S * u / s.n;
    int64_t off = s.S;
    int k = u - s.n;
    for (int r = 0; r < s.rounds; ++r) {
        if (k < s.n) return off + (int64_t)k * s.size[r];
        off += (int64_t)s.n * s.size[r];
        k -= s.n;
    }
    return s.T;
}

// The unit that holds tile t.
__device__ __forceinline__ int unit_of_tile(const Sched &s, int64_t t) {
    if (t < s.S) return (int)(((t + 1) * s.n - 1) / s.S);
    int64_t off = t - s.S;
    int u = s.n;
    for (int r = 0; r < s.rounds; ++r) {
        const int64_t span = (int64_t)s.n * s.size[r];
        if (off < span) return u + (int)(off / s.size[r]);
        off -= span;
        u += s.n;
    }
    return u;
}

// Partial slot a unit used for the piece of the segment starting at tile `seg`.
__device__ __forceinline__ int unit_slot(const Sched &s, int u, int64_t seg) {
    return unit_start(s, u) < seg ? 1 : 0;
}

// Sequence b's length as the launch sees it.
template <typename Args>
__device__ __forceinline__ int length_of(const Args &a, int b) {
    return min(max(0, __ldg(a.seq_lens + b)), a.max_len);
}

// Exclusive prefix of tiles per sequence times kv_heads (0 for empty ones).
template <typename Args>
__device__ void build_tile_prefix(const Args &a, int *prefix, int *scratch) {
    const int tid = threadIdx.x, nthr = blockDim.x;
    const int lane = tid & 31, warp = tid >> 5;
    const int per = (a.batch + nthr - 1) / nthr;
    int local = 0;
    for (int k = 0; k < per; ++k) {
        const int b = tid * per + k;
        if (b < a.batch)
            local += (length_of(a, b) + kTcTile - 1) / kTcTile * a.kv_heads;
    }
    int incl = local;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += v;
    }
    if (lane == 31) scratch[warp] = incl;
    __syncthreads();
    int before = 0;
    for (int w = 0; w < warp; ++w) before += scratch[w];
    int run = before + incl - local;
    for (int k = 0; k < per; ++k) {
        const int b = tid * per + k;
        if (b < a.batch) {
            prefix[b] = run;
            run += (length_of(a, b) + kTcTile - 1) / kTcTile * a.kv_heads;
        }
    }
    if (tid == nthr - 1) prefix[a.batch] = before + incl;
}

// One contiguous run of tiles of one (sequence, KV head) segment.
struct Piece {
    int b, g, k0, k1, nt;
    int64_t seg;  // stream index of the segment's first tile
};

template <typename Args>
__device__ __forceinline__ Piece piece_at(int64_t t, int64_t end, const int *prefix,
                                          const Args &a) {
    Piece P;
    int lo = 0, hi = a.batch - 1;  // last sequence whose first tile is <= t
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (prefix[mid] <= t) lo = mid; else hi = mid - 1;
    }
    P.b = lo;
    P.nt = (prefix[lo + 1] - prefix[lo]) / a.kv_heads;
    const int64_t within = t - prefix[lo];
    P.g = (int)(within / P.nt);
    P.k0 = (int)(within - (int64_t)P.g * P.nt);
    P.seg = prefix[lo] + (int64_t)P.g * P.nt;
    P.k1 = (int)min((int64_t)P.nt, (int64_t)P.k0 + (end - t));
    return P;
}

}  // namespace pkv
