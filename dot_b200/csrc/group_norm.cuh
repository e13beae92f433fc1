// Group normalisation with an activation on channels-last features, forward
// and backward (dot_group_norm_fwd / _bwd in include/dot_b200.h): kernels and
// their dispatch for one element type (group_norm_<type>.cu instantiate it).
//
//   z = (x - mean) rstd w + b,  y = act(z)
//   dz = dy act'(z),  db_c = sum dz,  dw_c = sum dz xh,  xh = (x - mean) rstd
//   dx = rstd (w dz - S1/m - xh S2/m),  S1 = sum_g w dz,  S2 = sum_g w dz xh
//
// Bound: memory.  A position's channels are consecutive, so a thread owns one
// vector of VEC channels (its parameters stay in registers) and walks the
// positions.  ONEG: a vector never crosses a group (VEC divides C/G), so its
// statistics are one value each.
//
// Three forms, chosen by size and layout (run): a cluster of blocks that holds
// its share of a sample in registers and reads it once; beyond that, for rows
// one after another in memory, one cooperative launch that walks them twice;
// else the same two walks as two launches.  No atomics on values; every merge
// has a fixed order, so results are bitwise reproducible.
//
// Measured (device time, 6.55 TB/s copy rate): 8 x 4800 x 256 bfloat16 with silu
// 16.6 us forward; 16 x 76800 x 64 with relu 82.2 us; 2 x 76800 x 256 with silu
// 45.9 us forward and 72.6 backward; 16 x 1024 x 256 padded sets 7.9 and 14.0.
//
// Moments are kept as (mean, sum M of squared deviations) of x - pivot, the
// pivot one of the group's values: a mean far from zero then costs its own
// rounding and no more.  A thread takes two passes over the positions in its
// registers and merges a batch into its running pair, n = n1 + n2,
// d = mean2 - mean1:  mean = mean1 + d n2/n,  M = M1 + M2 + d^2 n1 n2/n
// (Chan, Golub and LeVeque, 1979); threads' and blocks' pairs are joined by Merge.
#pragma once

#include <atomic>
#include <cooperative_groups.h>

#include "cluster.cuh"
#include "feature.cuh"
#include "feature_ops.h"
#include "internal.h"
#include "tma.cuh"

namespace dotb {
namespace {

constexpr int kSMs = 148;
// One block of 512 threads per SM: up to 128 registers a thread, so that enough
// loads are in flight (8 of 16 bytes a thread, 64 KB per SM).  1024 threads of
// 64 registers measured 90 us where these take 84 (clip backward in two
// launches); two blocks per SM are packed onto half the SMs.
constexpr int kGnThreads = 512;
constexpr int kGnWarps = kGnThreads / 32;
constexpr int kMaxCluster = 8;

// Shared memory: what a block may have, what it has without asking, and what the
// merges over a sample's chunks (sample_stats, sample_sums) hold beside the
// dynamic part.  The sweeps' groups are bounded by it: 8 bytes each next to those
// merges in the second sweep, next to the threads' pairs in the first (fits()).
constexpr size_t kSmemMost = 227 * 1024, kSmemDefault = 48 * 1024;
constexpr size_t kSmemMerges = size_t(kGnWarps) * 32 * sizeof(float2);
constexpr int64_t kMaxGroups = int64_t((kSmemMost - kSmemMerges) / sizeof(float2));
static_assert((size_t(kMaxGroups) + kGnThreads) * sizeof(float2) <= kSmemMost, "vectors of one element take any G");

// Resident path: vectors that a thread keeps of x (forward), or of x and of dy.
constexpr int res_vecs(int bytes, bool backward) {
    const int n = bytes >= 16 ? 8 : bytes >= 8 ? 16 : 32;
    return backward || n == 32 ? n : 2 * n;
}

struct GnPlan {
    GroupNormArgs a;
    int chunks;          // blocks that share a sample's positions
    int rows;            // positions per chunk
    int slab_groups;     // resident: groups of a block's channel slab
    int slabs;           // resident: slabs per sample
    int share;           // resident, bwd: the blocks meet at the end and sum the parameters' gradients
    float2* moments;     // sweeps, fwd: [N][chunks][G] (mean, M) of a chunk
    float2* gsums;       // sweeps, bwd: [N][chunks][G] (sum w dz, sum w dz xh)
    float2* csums;       // bwd: [N][chunks][C] (sum dz, sum dz xh)
};

// Merging partial moments (mean_i, M_i) of n_i values each about one of the
// means:  d_i = mean_i - about,
//   mean = about + sum n_i d_i / n,   M = sum (M_i + n_i d_i^2) - (sum n_i d_i)^2 / n.
// What cancels in M is at most n / n_i of it, from that mean's own distance.
struct Merge {
    float nd = 0.0f, m2 = 0.0f;
    __device__ __forceinline__ void add(float about, float ni, float mean, float m) {
        const float d = mean - about, w = ni * d;
        if (ni > 0.0f) {   // the moments of nothing are not looked at
            nd += w;
            m2 += m + w * d;
        }
    }
    // over 2^log lanes of a warp
    __device__ __forceinline__ void lanes(int log) {
        for (int off = (1 << log) >> 1; off > 0; off >>= 1) {
            nd += __shfl_xor_sync(0xffffffffu, nd, off);
            m2 += __shfl_xor_sync(0xffffffffu, m2, off);
        }
    }
    // (mean, M) of n values
    __device__ __forceinline__ float2 pair(float about, float n) const {
        const float d = n > 0.0f ? nd / n : 0.0f;
        return n > 0.0f ? make_float2(about + d, m2 - nd * d) : make_float2(0.0f, 0.0f);
    }
};

__device__ __forceinline__ float2 lanes_sum(float2 s, int log) {
    for (int off = (1 << log) >> 1; off > 0; off >>= 1) {
        s.x += __shfl_xor_sync(0xffffffffu, s.x, off);
        s.y += __shfl_xor_sync(0xffffffffu, s.y, off);
    }
    return s;
}

// How many lanes a block gives each of `count` groups: the largest power of two
// (as its logarithm) that leaves none waiting, at most a warp.
__device__ __forceinline__ int lanes_log(int count, int threads) {
    int log = 5;
    while (log > 0 && (count << log) > threads) --log;
    return log;
}

// The group of each of a thread's channels c, c + 1, ...: one division.
struct GroupOf {
    int g, left, Cg;
    __device__ GroupOf(int c, int Cg_) : g(c / Cg_), left(Cg_ - (c - g * Cg_)), Cg(Cg_) {}
    __device__ __forceinline__ int next() {   // the current channel's group, then on to the next channel
        const int now = g;
        if (--left == 0) {
            left = Cg;
            ++g;
        }
        return now;
    }
};

__device__ __forceinline__ float2 mean_rstd(float pivot, float2 mean_m, int len, int Cg, float eps) {
    float var = len > 0 ? mean_m.y / (float(len) * float(Cg)) : 0.0f;
    if (var < 0.0f) var = 0.0f;   // the merges' rounding of a variance next to nothing; a NaN stays one
    return make_float2(pivot + mean_m.x, 1.0f / sqrtf(var + eps));
}

// The value that a group's moments are taken about: its sample's first
// position in the group's first channel c.
template <typename T>
__device__ __forceinline__ float group_pivot(const T* x, int len, int c) {
    return len > 0 ? to_f32(x[c]) : 0.0f;
}

__device__ __forceinline__ int valid_len(const GroupNormArgs& a, int n) {
    if (a.lengths == nullptr) return int(a.S);
    return int(min(max(int64_t(__ldg(a.lengths + n)), int64_t(0)), a.S));
}

// A thread's channels: per-channel parameters in pairs, a group's values once
// where the vector lies in one group.
template <int VEC, bool ONEG>
struct PerGroup {
    static constexpr int NP = pairs_of(VEC);
    float2 v[ONEG ? 1 : NP];
    __device__ __forceinline__ float2 operator[](int j) const { return v[ONEG ? 0 : j]; }
    // f(g): the value of group g; c: the first channel
    template <typename F>
    __device__ __forceinline__ void fill(int c, int Cg, F f) {
        GroupOf of(c, Cg);
        if constexpr (ONEG) {
            v[0] = splat2(f(of.g));
        } else {
#pragma unroll
            for (int j = 0; j < NP; ++j) {
                v[j].x = f(of.next());
                v[j].y = VEC == 1 ? 0.0f : f(of.next());
            }
        }
    }
};

// y of a vector.  The mean is subtracted first rather than taken into the shift:
// a group of equal values then gives its bias exactly.
template <typename T, int VEC, int ACT, bool ONEG>
struct Forward {
    static constexpr int NP = pairs_of(VEC);
    PerGroup<VEC, ONEG> mean;
    float2 scale[NP], shift[NP];
    // st: (mean, rstd) by group; c: the first channel, c_st: counted from st's first group
    __device__ __forceinline__ void load(const GroupNormArgs& a, int c, int c_st, int Cg, const float2* st) {
        params(a, c);
        stats(c_st, Cg, st);
    }
    __device__ __forceinline__ void params(const GroupNormArgs& a, int c) {
        load_params<VEC>(a.weight, a.param_dtype, c, 1.0f, scale);
        load_params<VEC>(a.bias, a.param_dtype, c, 0.0f, shift);
    }
    __device__ __forceinline__ void stats(int c_st, int Cg, const float2* st) {
        mean.fill(c_st, Cg, [&](int g) { return st[g].x; });
        PerGroup<VEC, ONEG> r;
        r.fill(c_st, Cg, [&](int g) { return st[g].y; });
#pragma unroll
        for (int j = 0; j < NP; ++j) scale[j] = mul2(scale[j], r[j]);
    }
    __device__ __forceinline__ Pack<T, VEC> operator()(const Pack<T, VEC>& raw, int act) const {
        float2 f[NP];
        unpack(raw, f);
#pragma unroll
        for (int j = 0; j < NP; ++j)
            f[j] = act_fwd<ACT>(fma2(sub2(f[j], mean[j]), scale[j], shift[j]), act);
        return pack<T, VEC>(f);
    }
};

// The backward's chain for a vector: xh, dz; the sums of dz and dz xh; dx.
template <typename T, int VEC, int ACT, bool ONEG>
struct Backward {
    static constexpr int NP = pairs_of(VEC);
    PerGroup<VEC, ONEG> mean, rstd;
    float2 w[NP], b[NP];
    // st: a pair or more by group, mean and rstd first; c_st: c counted from st's first group
    template <typename S>
    __device__ __forceinline__ void load(const GroupNormArgs& a, int c, int c_st, int Cg, const S* st) {
        load_params<VEC>(a.weight, a.param_dtype, c, 1.0f, w);
        load_params<VEC>(a.bias, a.param_dtype, c, 0.0f, b);
        mean.fill(c_st, Cg, [&](int g) { return st[g].x; });
        rstd.fill(c_st, Cg, [&](int g) { return st[g].y; });
    }
    __device__ __forceinline__ void chain(float2 x, float2 dy, int j, int act, float2& xh, float2& dz) const {
        xh = mul2(sub2(x, mean[j]), rstd[j]);
        dz = mul2(dy, act_slope<ACT>(fma2(xh, w[j], b[j]), act));
    }
    __device__ __forceinline__ void sums(const Pack<T, VEC>& rx, const Pack<T, VEC>& rg, int act, float2 (&sa)[NP],
                                         float2 (&sb)[NP]) const {
        float2 x[NP], g[NP];
        unpack(rx, x);
        unpack(rg, g);
#pragma unroll
        for (int j = 0; j < NP; ++j) {
            float2 xh, dz;
            chain(x[j], g[j], j, act, xh, dz);
            sa[j] = add2(sa[j], dz);
            sb[j] = fma2(dz, xh, sb[j]);
        }
    }
};

// dx = (rstd w) dz - rstd S1/m - xh (rstd S2/m)
template <typename T, int VEC, int ACT, bool ONEG>
struct BackwardDx : Backward<T, VEC, ACT, ONEG> {
    using Base = Backward<T, VEC, ACT, ONEG>;
    static constexpr int NP = Base::NP;
    PerGroup<VEC, ONEG> s1, s2;   // -rstd S1/m, -rstd S2/m
    float2 rw[NP];
    // sum(g): group g's (S1/m, S2/m).  A group of one value has no gradient.
    template <typename F>
    __device__ __forceinline__ void finish(int c_st, int Cg, int len, F sum) {
        const float on = int64_t(len) * Cg > 1 ? 1.0f : 0.0f;
        s1.fill(c_st, Cg, [&](int g) { return -on * sum(g).x; });
        s2.fill(c_st, Cg, [&](int g) { return -on * sum(g).y; });
#pragma unroll
        for (int j = 0; j < NP; ++j) {
            rw[j] = mul2(mul2(this->rstd[j], splat2(on)), this->w[j]);
            if (!ONEG || j == 0) {
                s1.v[j] = mul2(s1.v[j], this->rstd[j]);
                s2.v[j] = mul2(s2.v[j], this->rstd[j]);
            }
        }
    }
    __device__ __forceinline__ Pack<T, VEC> dx(const Pack<T, VEC>& rx, const Pack<T, VEC>& rg, int act) const {
        float2 x[NP], g[NP];
        unpack(rx, x);
        unpack(rg, g);
#pragma unroll
        for (int j = 0; j < NP; ++j) {
            float2 xh, dz;
            this->chain(x[j], g[j], j, act, xh, dz);
            x[j] = fma2(xh, s2[j], fma2(rw[j], dz, s1[j]));
        }
        return pack<T, VEC>(x);
    }
};

// ---- backward: the parameters' gradients from the blocks' channel sums ---------

// Channels c = first + warp, + the block's warps, ... < end: a warp sums a channel's
// pairs over all samples' chunks, in an order that depends on nothing else.
__device__ __forceinline__ void param_grads(const GnPlan& pl, int first, int end) {
    const GroupNormArgs& a = pl.a;
    const int C = int(a.C), lane = threadIdx.x & 31;
    const int64_t rows = a.N * pl.chunks;
    for (int c = first + int(threadIdx.x >> 5); c < end; c += int(blockDim.x) / 32) {
        float2 s = make_float2(0.0f, 0.0f);
#pragma unroll 4
        for (int64_t r = lane; r < rows; r += 32) {
            const float2 v = __ldcg(pl.csums + r * C + c);
            s.x += v.x;
            s.y += v.y;
        }
        s = lanes_sum(s, 5);
        if (lane == 0) {
            if (a.dbias) store_param(a.dbias, a.param_dtype, c, s.x);
            if (a.dweight) store_param(a.dweight, a.param_dtype, c, s.y);
        }
    }
}

// The blocks of a launch share out the channels.
__device__ __forceinline__ void share_param_grads(const GnPlan& pl) {
    const int C = int(pl.a.C), per = (C + int(gridDim.x) - 1) / int(gridDim.x);
    if (pl.a.dweight || pl.a.dbias) param_grads(pl, int(blockIdx.x) * per, min(C, int(blockIdx.x + 1) * per));
}

// A launch of its own where no other one follows the sums.
__global__ void __launch_bounds__(kGnThreads) gn_params_kernel(GnPlan pl) {
    pdl_wait();
    param_grads(pl, int(blockIdx.x) * kGnWarps, min(int(pl.a.C), int(blockIdx.x + 1) * kGnWarps));
}

// ---- two sweeps per direction --------------------------------------------------
//
// For strided rows, vectors under 16 bytes and what the other forms do not
// take.  A block reads whole rows of one chunk (a range of one sample's
// positions).  The first sweep leaves the chunk's partial sums in the
// workspace, the second merges its sample's partials at its start and writes
// the result, walking its rows backwards: it begins with those that the first
// sweep read last.

// Valid positions of chunk k of `rows`.
__device__ __forceinline__ int rows_of(int len, int k, int rows) { return min(max(len - k * rows, 0), rows); }

// Where a block's threads stand in a tile of at most kGnThreads channel
// vectors: vector v of `nv`, first of the rows r, r + rp, ...
struct Place {
    int nv, rp, r, v;
    bool on;
    __device__ Place(int cv, int tile) {
        nv = min(kGnThreads, cv - tile * kGnThreads);
        rp = kGnThreads / nv;
        r = int(threadIdx.x) / nv;
        v = int(threadIdx.x) - r * nv;
        on = r < rp;
    }
};

// A ring of bulk copies for rows that lie one after another in memory, walked
// forwards and then backwards: up to 160 KB in flight per SM without a
// register, and the way back begins with the stages that are still there.  A
// stage holds U rows for each row position of the block, of x and for NT = 2 of
// dy; the last of the 16 warps to leave a stage refills it.  Waits are bounded.
// A thread whose wait expired goes on without waiting and writes NaN, into every
// channel of its partial sums on the way in and of its rows on the way out; its
// warp leaves no stage any more, so that the block starts no further copy (the
// barrier of the lost one is still in its phase), and before it ends it waits
// (again with a limit) for those in flight.
constexpr int kRingStages = 5;
constexpr int kRingStageBytes = 32 * 1024;

// Whether the c-th copy into stage i's slot is left out: never, but for the test of
// the expired wait, which defines it before including this file.
#ifndef DOTB_RING_LOSES
#define DOTB_RING_LOSES(i, c) false
#endif

template <int NT>
struct Ring {
    static constexpr int kPart = kRingStageBytes / NT;   // bytes of one tensor in a stage
    unsigned char* buf;
    uint64_t* full;                     // [kRingStages]
    int* left;                          // [kRingStages] warps that have left the stage
    int* copies;                        // [kRingStages] copies started into the slot
    const unsigned char* src[NT];       // row 0 of the block's range
    int row_bytes, rows, stage_rows, n; // rows in all, per stage; stages
    bool dead = false;

    static constexpr size_t bytes() {   // what follows is 16-byte aligned
        return (size_t(kRingStages) * (kRingStageBytes + sizeof(uint64_t) + 2 * sizeof(int)) + 15) / 16 * 16;
    }
    // By all threads, before a block barrier.
    __device__ __forceinline__ void init(unsigned char* smem, int rows_, int stage_rows_, int row_bytes_) {
        buf = smem;
        full = reinterpret_cast<uint64_t*>(smem + kRingStages * kRingStageBytes);
        left = reinterpret_cast<int*>(full + kRingStages);
        copies = left + kRingStages;
        rows = rows_;
        stage_rows = stage_rows_;
        row_bytes = row_bytes_;
        n = (rows + stage_rows - 1) / stage_rows;
        if (threadIdx.x == 0) {
#pragma unroll
            for (int k = 0; k < kRingStages; ++k) {
                mbar_init(full + k, 1);
                left[k] = copies[k] = 0;
            }
            mbar_fence_init();
        }
    }
    // Stage i holds rows [i stage_rows, + count(i)).
    __device__ __forceinline__ int count(int i) const { return min(stage_rows, rows - i * stage_rows); }
    // Stage i as the c-th copy into its slot.
    __device__ __forceinline__ void issue(int i, int c) {
        const int slot = i % kRingStages;
        const uint32_t bytes = uint32_t(count(i)) * uint32_t(row_bytes);
        if (DOTB_RING_LOSES(i, c)) return;
        copies[slot] = c + 1;
        mbar_arrive_expect_tx(full + slot, NT * bytes);
#pragma unroll
        for (int t = 0; t < NT; ++t)
            bulk_g2s(buf + slot * kRingStageBytes + t * kPart, src[t] + int64_t(i) * stage_rows * row_bytes, bytes,
                     full + slot);
    }
    // After that barrier.
    __device__ __forceinline__ void fill() {
        if (threadIdx.x == 0)
            for (int i = 0; i < min(n, kRingStages); ++i) issue(i, 0);
    }
    // A warp leaves stage i; the last one brings stage `next` into its place, its c-th copy.
    __device__ __forceinline__ void leave(int i, int next, int c) {
        const int slot = i % kRingStages;
        if (!__any_sync(0xffffffffu, dead) && (threadIdx.x & 31) == 0) {
            __threadfence_block();
            if (atomicAdd(left + slot, 1) == kGnWarps - 1) {
                left[slot] = 0;
                __threadfence_block();
                fence_proxy_async_smem();
                issue(next, c);
            }
        }
    }
    __device__ __forceinline__ void wait(int i) {
        if (!dead) dead = !mbar_wait_sleep(full + i % kRingStages, uint32_t(i / kRingStages) & 1u, nullptr);
    }
    // use(stage's bytes, its first row, its rows), first stage to last.  The
    // c-th copy into a slot completes its barrier's phase c: stage i is copy
    // i / kRingStages of its slot on the way forwards ...
    template <typename F>
    __device__ __forceinline__ void forwards(F use) {
        for (int i = 0; i < n; ++i) {
            wait(i);
            use(buf + (i % kRingStages) * kRingStageBytes, i * stage_rows, count(i));
            if (i + kRingStages < n) leave(i, i + kRingStages, i / kRingStages + 1);
        }
    }
    // ... and, m = (slot's last stage) / kRingStages, copy 2 m - i / kRingStages
    // on the way back, which has the same parity (the stage below it in the slot is
    // one copy more).  The last stages are still there.
    template <typename F>
    __device__ __forceinline__ void backwards(F use) {
        for (int i = n - 1; i >= 0; --i) {
            if (i < n - kRingStages) wait(i);
            use(buf + (i % kRingStages) * kRingStageBytes, i * stage_rows, count(i));
            if (i >= kRingStages)
                leave(i, i - kRingStages, (n - 1 - i % kRingStages) / kRingStages * 2 - i / kRingStages + 1);
        }
    }
    // At the end: copies still in flight must not outlive the block.  Whichever thread
    // started one has either seen it arrive or waits for it here.
    __device__ __forceinline__ void drain() {
        if (dead)
            for (int k = 0; k < min(n, kRingStages); ++k)
                if (copies[k] > 0) mbar_wait_sleep(full + k, uint32_t(copies[k] - 1) & 1u, nullptr);
    }
};

// NaN for what an expired wait left without its data.
template <int N>
__device__ __forceinline__ void poison(float (&v)[N]) {
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = __int_as_float(0x7fffffff);
}
template <int N>
__device__ __forceinline__ void poison(float2 (&v)[N]) {
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = splat2(__int_as_float(0x7fffffff));
}

// Mean (about the pivot) and M of the first `k` of U vectors of a thread, per
// channel, or one for all channels of a vector that lies in one group: two
// passes over the registers.  The sum of a batch of 16-bit values is taken as
// it is (their few bits leave its rounding far below the pivot's), float32
// subtracts the pivot first.
template <typename T, int VEC, bool ONEG>
struct Batch {
    static constexpr int NP = pairs_of(VEC), NG = ONEG ? 1 : VEC;
    float mean[NG], m2[NG];
    template <int U, bool FULL>
    __device__ __forceinline__ void take(Pack<T, VEC> (&raw)[U], const PerGroup<VEC, ONEG>& pivot, int k) {
        constexpr bool RAW = sizeof(T) == 2;
        const float inv = (FULL ? 1.0f / float(U) : 1.0f / float(k > 0 ? k : 1)) * (ONEG ? 1.0f / float(VEC) : 1.0f);
        float2 s[NP], q[NP], about[NP];
#pragma unroll
        for (int j = 0; j < NP; ++j) s[j] = q[j] = splat2(0.0f);
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (FULL || u < k) {
                float2 f[NP];
                unpack(raw[u], f);
#pragma unroll
                for (int j = 0; j < NP; ++j) s[j] = add2(s[j], RAW ? f[j] : sub2(f[j], pivot[j]));
            }
        if constexpr (ONEG) {
            const float2 t = tree_sum2(s);
            const float all = VEC == 1 ? t.x : t.x + t.y;
            const float p = pivot[0].x;
            mean[0] = RAW ? fmaf(all, inv, -p) : all * inv;
#pragma unroll
            for (int j = 0; j < NP; ++j) about[j] = splat2(p + mean[0]);
        } else {
#pragma unroll
            for (int j = 0; j < NP; ++j) {
                const float2 p = pivot[j];
                const float2 m = RAW ? fma2(s[j], splat2(inv), make_float2(-p.x, -p.y)) : mul2(s[j], splat2(inv));
                about[j] = add2(p, m);
                mean[2 * j] = m.x;
                if constexpr (VEC > 1) mean[2 * j + 1] = m.y;
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (U > 4) reload(raw[u]);
            if (FULL || u < k) {
                float2 f[NP];
                unpack(raw[u], f);
#pragma unroll
                for (int j = 0; j < NP; ++j) {
                    const float2 d = sub2(f[j], about[j]);
                    q[j] = fma2(d, d, q[j]);
                }
            }
            if (U > 4) reload(raw[u]);
        }
        if constexpr (ONEG) {
            const float2 t = tree_sum2(q);
            m2[0] = VEC == 1 ? t.x : t.x + t.y;
        } else {
#pragma unroll
            for (int j = 0; j < NP; ++j) {
                m2[2 * j] = q[j].x;
                if constexpr (VEC > 1) m2[2 * j + 1] = q[j].y;
            }
        }
    }
};

// Joins a batch's pairs to a thread's running ones.
template <typename T, int VEC, bool ONEG>
struct Running {
    static constexpr int W = ONEG ? 1 : VEC;
    float n = 0.0f, mean[W], m2[W];
    __device__ __forceinline__ Running() {
#pragma unroll
        for (int j = 0; j < W; ++j) mean[j] = m2[j] = 0.0f;
    }
    __device__ __forceinline__ void join(const Batch<T, VEC, ONEG>& b, float k) {
        const float tot = n + k, f = __fdividef(k, tot), w = n * f * float(VEC / W);
#pragma unroll
        for (int j = 0; j < W; ++j) {
            const float d = b.mean[j] - mean[j];
            mean[j] += d * f;
            m2[j] += b.m2[j] + d * d * w;
        }
        n = tot;
    }
};

// A tile's groups from its threads' pairs `part` [rp][nv * W] over `rows`
// positions, joined to what earlier tiles left of them in acc [G].
template <int VEC, int W>
__device__ __forceinline__ void tile_moments(const Place& pc, int tile, int Cg, int rows, const float2* part, float2* acc) {
    const int c0 = tile * kGnThreads * VEC, c1 = c0 + pc.nv * VEC;
    const int g0 = c0 / Cg, gn = (c1 - 1) / Cg - g0 + 1, log = lanes_log(gn, kGnThreads);
    const int lane = int(threadIdx.x) & ((1 << log) - 1), full = rows / pc.rp;
    for (int i0 = 0; i0 < gn; i0 += kGnThreads >> log) {
        const int gi = i0 + (int(threadIdx.x) >> log), g = g0 + gi;
        const bool mine = gi < gn;
        const int ca = max(c0, g * Cg), before = ca - g * Cg;   // channels of the group in earlier tiles
        const int wd = (min(c1, (g + 1) * Cg) - ca) / (VEC / W), at = (ca - c0) / (VEC / W);
        const float2 old = mine ? acc[g] : make_float2(0.0f, 0.0f);
        const float about = mine ? part[at].x : 0.0f;   // row 0 is there if any is
        Merge m;
        if (mine) {
            for (int i = lane; i < pc.rp * wd; i += 1 << log) {
                const int r = wd == 1 ? i : i / wd;
                const float2 v = part[r * pc.nv * W + at + i - r * wd];
                const int cnt = full + (r < rows - full * pc.rp ? 1 : 0);
                m.add(about, float(cnt * (VEC / W)), v.x, v.y);
            }
            if (before > 0 && lane == 0) m.add(about, float(rows) * float(before), old.x, old.y);
        }
        m.lanes(log);
        __syncwarp();
        if (mine && lane == 0) acc[g] = m.pair(about, float(rows) * float(min(c1, (g + 1) * Cg) - g * Cg));
    }
}

// Statistics [G] of sample n from its chunks' moments, by the whole block;
// pivot(g): the value that group g's moments are about.
template <typename F>
__device__ __forceinline__ void sample_stats(const GnPlan& pl, int n, bool write, int len, F pivot, float2* st) {
    __shared__ Merge merged[kGnWarps][32];
    static_assert(sizeof(merged) == kSmemMerges, "as launch() is told");
    const GroupNormArgs& a = pl.a;
    const int G = int(a.G), Cg = int(a.C) / G, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (int g = lane; g < (G + 31) / 32 * 32; g += 32) {   // a lane a group, the warps share the chunks
        Merge m;
        const float2* from = pl.moments + int64_t(n) * pl.chunks * G + g;
        const float about = g < G ? __ldcg(from).x : 0.0f;
        if (g < G)
#pragma unroll 8
            for (int k = warp; k < pl.chunks; k += kGnWarps) {
                const float2 v = __ldcg(from + int64_t(k) * G);
                m.add(about, float(rows_of(len, k, pl.rows)) * float(Cg), v.x, v.y);
            }
        merged[warp][lane] = m;
        __syncthreads();
        if (warp == 0 && g < G) {
#pragma unroll
            for (int k = 1; k < kGnWarps; ++k) {
                m.nd += merged[k][lane].nd;
                m.m2 += merged[k][lane].m2;
            }
            st[g] = mean_rstd(pivot(g), m.pair(about, float(len) * float(Cg)), len, Cg, a.eps);
            if (write) reinterpret_cast<float2*>(a.stats)[int64_t(n) * G + g] = st[g];
        }
        __syncthreads();
    }
}

// A tile's channel sums (into the workspace's row `slot`) and, weighted, its
// groups' (added to acc [G]) from its threads' pairs `part` [rp][nv * VEC].
template <int VEC>
__device__ __forceinline__ void tile_sums(const GnPlan& pl, const Place& pc, int tile, int64_t slot, float2* part, float2* acc) {
    const GroupNormArgs& a = pl.a;
    const int C = int(a.C), Cg = C / int(a.G), c0 = tile * kGnThreads * VEC, c1 = c0 + pc.nv * VEC;
    for (int i = threadIdx.x; i < pc.nv * VEC; i += kGnThreads) {   // rows of a channel, in order
        float2 s = part[i];
        for (int r = 1; r < pc.rp; ++r) {
            const float2 v = part[r * pc.nv * VEC + i];
            s.x += v.x;
            s.y += v.y;
        }
        part[i] = s;
        pl.csums[slot * C + c0 + i] = s;
    }
    __syncthreads();
    const int g0 = c0 / Cg, gn = (c1 - 1) / Cg - g0 + 1, log = lanes_log(gn, kGnThreads);
    const int lane = int(threadIdx.x) & ((1 << log) - 1);
    for (int i0 = 0; i0 < gn; i0 += kGnThreads >> log) {
        const int gi = i0 + (int(threadIdx.x) >> log), g = g0 + gi;
        float2 s = make_float2(0.0f, 0.0f);
        if (gi < gn)
            for (int c = max(c0, g * Cg) + lane; c < min(c1, (g + 1) * Cg); c += 1 << log) {
                const float w = a.weight ? load_param(a.weight, a.param_dtype, c) : 1.0f;
                s.x += w * part[c - c0].x;
                s.y += w * part[c - c0].y;
            }
        s = lanes_sum(s, log);
        if (gi < gn && lane == 0) {
            acc[g].x += s.x;
            acc[g].y += s.y;
        }
    }
}

// S1/m and S2/m of sample n's groups from its chunks' sums, by the whole block;
// put(g, pair) takes group g's.
template <typename F>
__device__ __forceinline__ void sample_sums(const GnPlan& pl, int n, int len, F put) {
    __shared__ float2 merged[kGnWarps][32];
    static_assert(sizeof(merged) == kSmemMerges, "as launch() is told");
    const GroupNormArgs& a = pl.a;
    const int C = int(a.C), G = int(a.G), warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const float inv = len > 0 ? 1.0f / (float(len) * float(C / G)) : 0.0f;
    for (int g = lane; g < (G + 31) / 32 * 32; g += 32) {   // a lane a group, the warps share the chunks
        float2 s = make_float2(0.0f, 0.0f);
        if (g < G)
#pragma unroll 8
            for (int k = warp; k < pl.chunks; k += kGnWarps) {
                const float2 v = __ldcg(pl.gsums + (int64_t(n) * pl.chunks + k) * G + g);
                s.x += v.x;
                s.y += v.y;
            }
        merged[warp][lane] = s;
        __syncthreads();
        if (warp == 0 && g < G) {
#pragma unroll
            for (int k = 1; k < kGnWarps; ++k) {
                s.x += merged[k][lane].x;
                s.y += merged[k][lane].y;
            }
            put(g, make_float2(s.x * inv, s.y * inv));
        }
        __syncthreads();
    }
}

// Zeros at a chunk's positions from pv on.
template <typename T, int VEC>
__device__ __forceinline__ void pad_rows(const Place& pc, T* out, int C, int c, int pv, int pe) {
    for (int p = pv + pc.r; pc.on && p < pe; p += pc.rp) store_pack<T, VEC>(out + int64_t(p) * C + c, pack_zero<T, VEC>());
}

template <int VEC>
__device__ __forceinline__ void put_pairs(float2* part, const float2* sa, const float2* sb) {
#pragma unroll
    for (int j = 0; j < VEC; ++j)
        part[j] = j % 2 ? make_float2(sa[j / 2].y, sb[j / 2].y) : make_float2(sa[j / 2].x, sb[j / 2].x);
}

// Forward, sweep 1: moments of every group over a chunk.
template <typename T, int VEC, bool ONEG>
__global__ void __launch_bounds__(kGnThreads, 1) gn_moments_kernel(GnPlan pl) {
    const GroupNormArgs& a = pl.a;
    extern __shared__ float gn_smem[];
    constexpr int W = ONEG ? 1 : VEC, U = 8;
    const int C = int(a.C), G = int(a.G), Cg = C / G, cv = C / VEC;
    float2* acc = reinterpret_cast<float2*>(gn_smem);   // [G] mean, M of the tiles so far
    float2* part = acc + G;                             // [rp][nv * W]
    const int n = int(blockIdx.x) / pl.chunks, chunk = int(blockIdx.x) % pl.chunks;
    const int len = valid_len(a, n);
    const int p0 = min(len, chunk * pl.rows), p1 = min(len, p0 + pl.rows);
    const T* x = static_cast<const T*>(a.x) + int64_t(n) * a.xb;
    pdl_launch_dependents();
    for (int tile = 0; tile * kGnThreads < cv; ++tile) {
        const Place pc(cv, tile);
        const int c = (tile * kGnThreads + pc.v) * VEC;
        if (pc.on) {
            PerGroup<VEC, ONEG> pivot;
            pivot.fill(c, Cg, [&](int g) { return group_pivot(x, len, g * Cg); });
            const T* xc = x + int64_t(p0 + pc.r) * a.xp + c;
            const int64_t step = int64_t(pc.rp) * a.xp;
            Running<T, VEC, ONEG> run;
            Batch<T, VEC, ONEG> bt;
            int left = max(0, p1 - p0 - pc.r + pc.rp - 1) / pc.rp;
            for (; left >= U; left -= U) {
                Pack<T, VEC> raw[U];
#pragma unroll
                for (int u = 0; u < U; ++u, xc += step) raw[u] = load_pack<T, VEC>(xc);
                bt.template take<U, true>(raw, pivot, U);
                run.join(bt, float(U));
            }
            if (left > 0) {
                Pack<T, VEC> raw[U];
#pragma unroll
                for (int u = 0; u < U; ++u, xc += step)
                    if (u < left) raw[u] = load_pack<T, VEC>(xc);
                bt.template take<U, false>(raw, pivot, left);
                run.join(bt, float(left));
            }
#pragma unroll
            for (int j = 0; j < W; ++j) part[(pc.r * pc.nv + pc.v) * W + j] = make_float2(run.mean[j], run.m2[j]);
        }
        __syncthreads();
        tile_moments<VEC, W>(pc, tile, Cg, p1 - p0, part, acc);
        __syncthreads();
    }
    for (int g = threadIdx.x; g < G; g += kGnThreads)
        pl.moments[(int64_t(n) * pl.chunks + chunk) * G + g] = acc[g];
}

// Forward, sweep 2: merges the sample's chunks, writes y.
template <typename T, int VEC, int ACT, bool ONEG>
__global__ void __launch_bounds__(kGnThreads, 1) gn_apply_kernel(GnPlan pl) {
    const GroupNormArgs& a = pl.a;
    extern __shared__ float gn_smem[];
    float2* st = reinterpret_cast<float2*>(gn_smem);   // [G] mean, rstd
    constexpr int U = 8;
    const int C = int(a.C), Cg = C / int(a.G), cv = C / VEC;
    const int n = int(blockIdx.x) / pl.chunks, chunk = int(blockIdx.x) % pl.chunks;
    const int len = valid_len(a, n);
    const T* x = static_cast<const T*>(a.x) + int64_t(n) * a.xb;
    pdl_launch_dependents();
    pdl_wait();
    sample_stats(pl, n, chunk == 0, len, [&](int g) { return group_pivot(x, len, g * Cg); }, st);
    const int p0 = chunk * pl.rows, pe = min(int(a.S), p0 + pl.rows), pv = min(max(len, p0), pe);
    T* y = static_cast<T*>(a.y) + int64_t(n) * a.S * C;
    for (int tile = 0; tile * kGnThreads < cv; ++tile) {
        const Place pc(cv, tile);
        if (!pc.on) continue;
        const int c = (tile * kGnThreads + pc.v) * VEC;
        Forward<T, VEC, ACT, ONEG> fw;
        fw.load(a, c, c, Cg, st);
        pad_rows<T, VEC>(pc, y, C, c, pv, pe);
        int left = max(0, pv - p0 - pc.r + pc.rp - 1) / pc.rp;
        const T* xc = x + int64_t(pv - 1 - pc.r) * a.xp + c;
        T* yc = y + int64_t(pv - 1 - pc.r) * C + c;
        const int64_t xs = int64_t(pc.rp) * a.xp, ys = int64_t(pc.rp) * C;
        for (; left >= U; left -= U) {
            Pack<T, VEC> raw[U];
#pragma unroll
            for (int u = 0; u < U; ++u, xc -= xs) raw[u] = load_pack<T, VEC>(xc);
#pragma unroll
            for (int u = 0; u < U; ++u, yc -= ys) store_pack<T, VEC>(yc, fw(raw[u], a.act));
        }
        for (; left > 0; --left, xc -= xs, yc -= ys) store_pack<T, VEC>(yc, fw(load_pack<T, VEC>(xc), a.act));
    }
}

// Backward, sweep 1: per-channel and per-group sums over a chunk.
template <typename T, int VEC, int ACT, bool ONEG>
__global__ void __launch_bounds__(kGnThreads, 1) gn_sums_kernel(GnPlan pl) {
    const GroupNormArgs& a = pl.a;
    extern __shared__ float gn_smem[];
    constexpr int U = 4, NP = pairs_of(VEC);
    const int C = int(a.C), G = int(a.G), Cg = C / G, cv = C / VEC;
    float2* acc = reinterpret_cast<float2*>(gn_smem);   // [G]
    float2* part = acc + G;                             // [rp][nv * VEC]
    const int n = int(blockIdx.x) / pl.chunks, chunk = int(blockIdx.x) % pl.chunks;
    const int64_t slot = int64_t(n) * pl.chunks + chunk;
    const int len = valid_len(a, n);
    const int p0 = min(len, chunk * pl.rows), p1 = min(len, p0 + pl.rows);
    const T* x = static_cast<const T*>(a.x) + int64_t(n) * a.xb;
    const T* dy = static_cast<const T*>(a.dy) + int64_t(n) * a.gb;
    pdl_launch_dependents();
    for (int g = threadIdx.x; g < G; g += kGnThreads) acc[g] = make_float2(0.0f, 0.0f);
    __syncthreads();
    for (int tile = 0; tile * kGnThreads < cv; ++tile) {
        const Place pc(cv, tile);
        if (pc.on) {
            const int c = (tile * kGnThreads + pc.v) * VEC;
            Backward<T, VEC, ACT, ONEG> bw;
            bw.load(a, c, c, Cg, reinterpret_cast<const float2*>(a.stats) + int64_t(n) * G);
            float2 sa[NP], sb[NP];
#pragma unroll
            for (int j = 0; j < NP; ++j) sa[j] = sb[j] = splat2(0.0f);
            int left = max(0, p1 - p0 - pc.r + pc.rp - 1) / pc.rp;
            const T* xc = x + int64_t(p0 + pc.r) * a.xp + c;
            const T* gc = dy + int64_t(p0 + pc.r) * a.gp + c;
            const int64_t xs = int64_t(pc.rp) * a.xp, gs = int64_t(pc.rp) * a.gp;
            for (; left >= U; left -= U) {
                Pack<T, VEC> rx[U], rg[U];
#pragma unroll
                for (int u = 0; u < U; ++u, xc += xs, gc += gs) {
                    rx[u] = load_pack<T, VEC>(xc);
                    rg[u] = load_pack<T, VEC>(gc);
                }
#pragma unroll
                for (int u = 0; u < U; ++u) bw.sums(rx[u], rg[u], a.act, sa, sb);
            }
            for (; left > 0; --left, xc += xs, gc += gs)
                bw.sums(load_pack<T, VEC>(xc), load_pack<T, VEC>(gc), a.act, sa, sb);
            put_pairs<VEC>(part + (pc.r * pc.nv + pc.v) * VEC, sa, sb);
        }
        __syncthreads();
        tile_sums<VEC>(pl, pc, tile, slot, part, acc);
        __syncthreads();
    }
    for (int g = threadIdx.x; g < G; g += kGnThreads) pl.gsums[slot * G + g] = acc[g];
}

// Backward, sweep 2: merges the sample's group sums, writes dx.
template <typename T, int VEC, int ACT, bool ONEG>
__global__ void __launch_bounds__(kGnThreads, 1) gn_dx_kernel(GnPlan pl) {
    const GroupNormArgs& a = pl.a;
    extern __shared__ float gn_smem[];
    float2* sums = reinterpret_cast<float2*>(gn_smem);   // [G] S1/m, S2/m
    constexpr int U = 4;
    const int C = int(a.C), Cg = C / int(a.G), cv = C / VEC;
    const int n = int(blockIdx.x) / pl.chunks, chunk = int(blockIdx.x) % pl.chunks;
    const int len = valid_len(a, n);
    pdl_launch_dependents();
    pdl_wait();
    sample_sums(pl, n, len, [&](int g, float2 s) { sums[g] = s; });
    const int p0 = chunk * pl.rows, pe = min(int(a.S), p0 + pl.rows), pv = min(max(len, p0), pe);
    const T* x = static_cast<const T*>(a.x) + int64_t(n) * a.xb;
    const T* dy = static_cast<const T*>(a.dy) + int64_t(n) * a.gb;
    T* dx = static_cast<T*>(a.dx) + int64_t(n) * a.S * C;
    for (int tile = 0; tile * kGnThreads < cv; ++tile) {
        const Place pc(cv, tile);
        if (!pc.on) continue;
        const int c = (tile * kGnThreads + pc.v) * VEC;
        BackwardDx<T, VEC, ACT, ONEG> bw;
        bw.load(a, c, c, Cg, reinterpret_cast<const float2*>(a.stats) + int64_t(n) * a.G);
        bw.finish(c, Cg, len, [&](int g) { return sums[g]; });
        pad_rows<T, VEC>(pc, dx, C, c, pv, pe);
        int left = max(0, pv - p0 - pc.r + pc.rp - 1) / pc.rp;
        const T* xc = x + int64_t(pv - 1 - pc.r) * a.xp + c;
        const T* gc = dy + int64_t(pv - 1 - pc.r) * a.gp + c;
        T* dc = dx + int64_t(pv - 1 - pc.r) * C + c;
        const int64_t xs = int64_t(pc.rp) * a.xp, gs = int64_t(pc.rp) * a.gp, ds = int64_t(pc.rp) * C;
        for (; left >= U; left -= U) {
            Pack<T, VEC> rx[U], rg[U];
#pragma unroll
            for (int u = 0; u < U; ++u, xc -= xs, gc -= gs) {
                rx[u] = load_pack<T, VEC>(xc);
                rg[u] = load_pack<T, VEC>(gc);
            }
#pragma unroll
            for (int u = 0; u < U; ++u, dc -= ds) store_pack<T, VEC>(dc, bw.dx(rx[u], rg[u], a.act));
        }
        for (; left > 0; --left, xc -= xs, gc -= gs, dc -= ds)
            store_pack<T, VEC>(dc, bw.dx(load_pack<T, VEC>(xc), load_pack<T, VEC>(gc), a.act));
    }
    share_param_grads(pl);
}

// ---- both sweeps in one launch --------------------------------------------------
//
// For rows one after another in memory: the same two sweeps on the ring, with a
// grid barrier between them where a sample's chunks lie in several blocks (a
// cooperative launch, one block per SM), so the second one finds the last 160 KB
// of every block's rows on chip and no launch lies between them.  Against two
// launches with plain loads: 8 x 4800 x 256 18.9 -> 16.6 us, clip backward 90 ->
// 73.  HBM bounds the way forwards (6.3 TB/s with the write-backs of earlier
// results).  The way back of 79 MB takes 20 us: 16 without silu, 16 without the
// stores, 16 us of HBM and L2 traffic in either case; where x exceeds L2 HBM
// bounds it too (157 MB read and written: 6.2 TB/s).

template <typename T, int VEC, int ACT, bool ONEG>
__global__ void __launch_bounds__(kGnThreads, 1) gn_fused_fwd_kernel(GnPlan pl) {
    const GroupNormArgs& a = pl.a;
    extern __shared__ __align__(16) unsigned char gn_ring[];
    constexpr int W = ONEG ? 1 : VEC, U = 4;
    const int C = int(a.C), G = int(a.G), Cg = C / G;
    float2* acc = reinterpret_cast<float2*>(gn_ring + Ring<1>::bytes());   // [G] mean, M; then mean, rstd
    float* piv = reinterpret_cast<float*>(acc + G);                        // [G]
    float2* part = acc + (G + 1) / 2 * 3;                                  // [rp][nv * W]
    const int n = int(blockIdx.x) / pl.chunks, chunk = int(blockIdx.x) % pl.chunks;
    const int len = valid_len(a, n);
    const int p0 = chunk * pl.rows, pe = min(int(a.S), p0 + pl.rows), pv = min(max(len, p0), pe);
    const T* x = static_cast<const T*>(a.x) + int64_t(n) * a.xb;
    const Place pc(C / VEC, 0);
    const int c = pc.v * VEC, step = pc.rp * C;   // elements from a thread's row to its next
    Ring<1> ring;
    ring.init(gn_ring, max(pv - p0, 0), pc.rp * U, C * int(sizeof(T)));
    ring.src[0] = reinterpret_cast<const unsigned char*>(x + int64_t(p0) * C);
    __syncthreads();
    ring.fill();
    for (int g = threadIdx.x; g < G; g += kGnThreads) piv[g] = group_pivot(x, len, g * Cg);
    __syncthreads();
    {
        PerGroup<VEC, ONEG> pivot;
        if (pc.on) pivot.fill(c, Cg, [&](int g) { return piv[g]; });
        Running<T, VEC, ONEG> run;
        Batch<T, VEC, ONEG> bt;
        ring.forwards([&](const unsigned char* sx, int, int rows) {
            const T* at = reinterpret_cast<const T*>(sx) + pc.r * C + c;
            const int k = pc.on ? (rows - pc.r + pc.rp - 1) / pc.rp : 0;
            Pack<T, VEC> raw[U];
            if (k == U) {
#pragma unroll
                for (int u = 0; u < U; ++u) raw[u] = load_pack<T, VEC>(at + u * step);
                bt.template take<U, true>(raw, pivot, U);
                run.join(bt, float(U));
            } else if (k > 0) {
#pragma unroll
                for (int u = 0; u < U; ++u)
                    if (u < k) raw[u] = load_pack<T, VEC>(at + u * step);
                bt.template take<U, false>(raw, pivot, k);
                run.join(bt, float(k));
            }
        });
        if (ring.dead) poison(run.mean);
        if (pc.on)
#pragma unroll
            for (int j = 0; j < W; ++j) part[(pc.r * pc.nv + pc.v) * W + j] = make_float2(run.mean[j], run.m2[j]);
    }
    __syncthreads();
    tile_moments<VEC, W>(pc, 0, Cg, max(pv - p0, 0), part, acc);
    __syncthreads();
    for (int g = threadIdx.x; g < G; g += kGnThreads)
        pl.moments[(int64_t(n) * pl.chunks + chunk) * G + g] = acc[g];
    Forward<T, VEC, ACT, ONEG> fw;
    if (pc.on) fw.params(a, c);   // on their way over the barrier
    if (pl.chunks > 1)
        cooperative_groups::this_grid().sync();
    else
        __syncthreads();
    sample_stats(pl, n, chunk == 0, len, [&](int g) { return piv[g]; }, acc);
    T* y = static_cast<T*>(a.y) + int64_t(n) * a.S * C;
    if (pc.on) fw.stats(c, Cg, acc);
    ring.backwards([&](const unsigned char* sx, int first, int rows) {
        if (ring.dead) poison(fw.scale);
        const T* at = reinterpret_cast<const T*>(sx) + pc.r * C + c;
        T* to = y + int64_t(p0 + first + pc.r) * C + c;
        if (!pc.on) return;
        if (rows == ring.stage_rows) {   // a whole stage: its vectors side by side
            Pack<T, VEC> raw[U];
#pragma unroll
            for (int u = 0; u < U; ++u) raw[u] = load_pack<T, VEC>(at + u * step);
#pragma unroll
            for (int u = 0; u < U; ++u) raw[u] = fw(raw[u], a.act);
#pragma unroll
            for (int u = 0; u < U; ++u) store_pack<T, VEC>(to + u * step, raw[u]);
        } else {
            for (int r = pc.r; r < rows; r += pc.rp, at += step, to += step)
                store_pack<T, VEC>(to, fw(load_pack<T, VEC>(at), a.act));
        }
    });
    pad_rows<T, VEC>(pc, y, C, c, pv, pe);
    ring.drain();
}

template <typename T, int VEC, int ACT, bool ONEG>
__global__ void __launch_bounds__(kGnThreads, 1) gn_fused_bwd_kernel(GnPlan pl) {
    const GroupNormArgs& a = pl.a;
    extern __shared__ __align__(16) unsigned char gn_ring[];
    constexpr int U = 2, NP = pairs_of(VEC);
    const int C = int(a.C), G = int(a.G), Cg = C / G;
    float4* gv = reinterpret_cast<float4*>(gn_ring + Ring<2>::bytes());   // [G] mean, rstd, S1/m, S2/m
    float2* acc = reinterpret_cast<float2*>(gv + G);                      // [G]
    float2* part = acc + (G + 1) / 2 * 2;                                 // [rp][nv * VEC]
    const int n = int(blockIdx.x) / pl.chunks, chunk = int(blockIdx.x) % pl.chunks;
    const int64_t slot = int64_t(n) * pl.chunks + chunk;
    const int len = valid_len(a, n);
    const int p0 = chunk * pl.rows, pe = min(int(a.S), p0 + pl.rows), pv = min(max(len, p0), pe);
    const T* x = static_cast<const T*>(a.x) + int64_t(n) * a.xb;
    const T* dy = static_cast<const T*>(a.dy) + int64_t(n) * a.gb;
    const Place pc(C / VEC, 0);
    const int c = pc.v * VEC, step = pc.rp * C;   // elements from a thread's row to its next
    Ring<2> ring;
    ring.init(gn_ring, max(pv - p0, 0), pc.rp * U, C * int(sizeof(T)));
    ring.src[0] = reinterpret_cast<const unsigned char*>(x + int64_t(p0) * C);
    ring.src[1] = reinterpret_cast<const unsigned char*>(dy + int64_t(p0) * C);
    __syncthreads();
    ring.fill();
    for (int g = threadIdx.x; g < G; g += kGnThreads) {
        const float2 v = reinterpret_cast<const float2*>(a.stats)[int64_t(n) * G + g];
        gv[g] = make_float4(v.x, v.y, 0.0f, 0.0f);
        acc[g] = make_float2(0.0f, 0.0f);
    }
    __syncthreads();
    BackwardDx<T, VEC, ACT, ONEG> bw;
    if (pc.on) bw.load(a, c, c, Cg, gv);
    {
        float2 sa[NP], sb[NP];
#pragma unroll
        for (int j = 0; j < NP; ++j) sa[j] = sb[j] = splat2(0.0f);
        ring.forwards([&](const unsigned char* s0, int, int rows) {
            const T* sx = reinterpret_cast<const T*>(s0) + pc.r * C + c;
            const T* sg = reinterpret_cast<const T*>(s0 + Ring<2>::kPart) + pc.r * C + c;
            if (!pc.on) return;
            if (rows == ring.stage_rows) {   // a whole stage: its vectors side by side
                Pack<T, VEC> rx[U], rg[U];
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    rx[u] = load_pack<T, VEC>(sx + u * step);
                    rg[u] = load_pack<T, VEC>(sg + u * step);
                }
#pragma unroll
                for (int u = 0; u < U; ++u) bw.sums(rx[u], rg[u], a.act, sa, sb);
            } else {
                for (int r = pc.r; r < rows; r += pc.rp, sx += step, sg += step)
                    bw.sums(load_pack<T, VEC>(sx), load_pack<T, VEC>(sg), a.act, sa, sb);
            }
        });
        if (ring.dead) {
            poison(sa);
            poison(sb);
        }
        if (pc.on) put_pairs<VEC>(part + (pc.r * pc.nv + pc.v) * VEC, sa, sb);
    }
    __syncthreads();
    tile_sums<VEC>(pl, pc, 0, slot, part, acc);
    __syncthreads();
    for (int g = threadIdx.x; g < G; g += kGnThreads) pl.gsums[slot * G + g] = acc[g];
    cooperative_groups::this_grid().sync();   // the parameters' gradients need every block's sums
    sample_sums(pl, n, len, [&](int g, float2 s) { gv[g] = make_float4(gv[g].x, gv[g].y, s.x, s.y); });
    T* dx = static_cast<T*>(a.dx) + int64_t(n) * a.S * C;
    if (pc.on) bw.finish(c, Cg, len, [&](int g) { return make_float2(gv[g].z, gv[g].w); });
    ring.backwards([&](const unsigned char* s0, int first, int rows) {
        if (ring.dead) poison(bw.rw);
        const T* sx = reinterpret_cast<const T*>(s0) + pc.r * C + c;
        const T* sg = reinterpret_cast<const T*>(s0 + Ring<2>::kPart) + pc.r * C + c;
        T* to = dx + int64_t(p0 + first + pc.r) * C + c;
        if (!pc.on) return;
        if (rows == ring.stage_rows) {   // a whole stage: its vectors side by side
            Pack<T, VEC> rx[U], rg[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                rx[u] = load_pack<T, VEC>(sx + u * step);
                rg[u] = load_pack<T, VEC>(sg + u * step);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) rx[u] = bw.dx(rx[u], rg[u], a.act);
#pragma unroll
            for (int u = 0; u < U; ++u) store_pack<T, VEC>(to + u * step, rx[u]);
        } else {
            for (int r = pc.r; r < rows; r += pc.rp, sx += step, sg += step, to += step)
                store_pack<T, VEC>(to, bw.dx(load_pack<T, VEC>(sx), load_pack<T, VEC>(sg), a.act));
        }
    });
    pad_rows<T, VEC>(pc, dx, C, c, pv, pe);
    share_param_grads(pl);
    ring.drain();
}

// ---- resident path ------------------------------------------------------------
//
// A cluster of `chunks` blocks holds one sample's positions of one channel slab
// (whole groups) in registers: x (and dy) are read once, the blocks exchange
// their groups' partial sums through distributed shared memory, and the result
// is written from the registers.  One launch per direction: the parameters'
// gradients, which cross clusters, follow a grid barrier at the end where all
// clusters run at once (a launch of their own costs a training call 7 us of 73
// on the host and saves 1 us of 14 on the device), else they are a second
// launch.  Bound by latency: 3.5 us for one 64 x 64 sample, 7.9 us forward and
// 14.0 us backward for 8.4 MB.

// Where a block stands: chunk (its rank in the cluster), slab, sample.
struct ResPlace {
    int n, chunk, g0, gs, c0, nv, rp, r, v;
    bool on;
    __device__ ResPlace(const GnPlan& pl, int Cg, int vec) {
        chunk = int(blockIdx.x) % pl.chunks;
        const int u = int(blockIdx.x) / pl.chunks;
        const int slab = u % pl.slabs;
        n = u / pl.slabs;
        g0 = slab * pl.slab_groups;
        gs = min(int(pl.a.G) - g0, pl.slab_groups);
        c0 = g0 * Cg;
        nv = gs * Cg / vec;
        rp = int(blockDim.x) / nv;
        r = int(threadIdx.x) / nv;
        v = int(threadIdx.x) - r * nv;
        on = r < rp;
    }
};

template <typename T, int VEC, int ACT, bool ONEG, int KV>
__global__ void __launch_bounds__(kGnThreads, 1) gn_resident_fwd_kernel(GnPlan pl) {
    const GroupNormArgs& a = pl.a;
    extern __shared__ float gn_smem[];
    const int C = int(a.C), G = int(a.G), Cg = C / G;
    const ResPlace pc(pl, Cg, VEC);
    float2* st = reinterpret_cast<float2*>(gn_smem);    // [slab_groups] mean, rstd
    float2* mine = st + pl.slab_groups;                 // [slab_groups] this block's mean, M
    float2* part = mine + pl.slab_groups;               // [rp][nv * (ONEG ? 1 : VEC)]
    const int len = valid_len(a, pc.n);
    const int p0 = pc.chunk * pl.rows, pv = min(len, p0 + pl.rows), pe = min(int(a.S), p0 + pl.rows);
    const int c = pc.c0 + pc.v * VEC;
    const T* x = static_cast<const T*>(a.x) + int64_t(pc.n) * a.xb + c;
    Pack<T, VEC> raw[KV];
    int cnt = 0;
#pragma unroll
    for (int k = 0; k < KV; ++k) {
        const int p = p0 + pc.r + k * pc.rp;
        if (pc.on && p < pv) {
            raw[k] = load_pack<T, VEC>(x + int64_t(p) * a.xp);
            ++cnt;
        }
    }
    if (pc.on) {
        PerGroup<VEC, ONEG> pivot;
        pivot.fill(c, Cg, [&](int g) { return group_pivot(x - c, len, g * Cg); });
        Batch<T, VEC, ONEG> bt;
        bt.template take<KV, false>(raw, pivot, cnt);
        constexpr int W = ONEG ? 1 : VEC;
#pragma unroll
        for (int j = 0; j < W; ++j) part[(pc.r * pc.nv + pc.v) * W + j] = make_float2(bt.mean[j], bt.m2[j]);
    }
    __syncthreads();
    {
        constexpr int J = ONEG ? VEC : 1;
        const int wd = Cg / J, width = pc.nv * (VEC / J), rows = max(pv - p0, 0), full = rows / pc.rp;
        const int log = lanes_log(pc.gs, int(blockDim.x)), lane = int(threadIdx.x) & ((1 << log) - 1);
        for (int i0 = 0; i0 < pc.gs; i0 += int(blockDim.x) >> log) {
            const int g = i0 + (int(threadIdx.x) >> log);
            const float about = g < pc.gs ? part[g * wd].x : 0.0f;   // row 0 is there if any is
            Merge m;
            if (g < pc.gs)
                for (int i = lane; i < pc.rp * wd; i += 1 << log) {
                    const int r = wd == 1 ? i : i / wd;
                    const float2 v = part[r * width + g * wd + i - r * wd];
                    m.add(about, float((full + (r < rows - full * pc.rp ? 1 : 0)) * J), v.x, v.y);
                }
            m.lanes(log);
            if (g < pc.gs && lane == 0) mine[g] = m.pair(about, float(rows) * float(Cg));
        }
    }
    if (pl.chunks > 1) cl_sync();
    else __syncthreads();
    for (int g = threadIdx.x; g < pc.gs; g += blockDim.x) {
        float2 m = mine[g];
        if (pl.chunks > 1) {
            float2 v[kMaxCluster];
#pragma unroll
            for (int k = 0; k < kMaxCluster; ++k)
                if (k < pl.chunks) v[k] = ld_cluster_f2(cluster_map(mine + g, uint32_t(k)));
            Merge all;
#pragma unroll
            for (int k = 0; k < kMaxCluster; ++k)
                if (k < pl.chunks) all.add(v[0].x, float(rows_of(len, k, pl.rows)) * float(Cg), v[k].x, v[k].y);
            m = all.pair(v[0].x, float(len) * float(Cg));
        }
        st[g] = mean_rstd(group_pivot(x - c, len, (pc.g0 + g) * Cg), m, len, Cg, a.eps);
        if (pc.chunk == 0) reinterpret_cast<float2*>(a.stats)[int64_t(pc.n) * G + pc.g0 + g] = st[g];
    }
    if (pl.chunks > 1) cl_arrive();   // this block has read its peers' sums
    __syncthreads();
    if (pc.on) {
        Forward<T, VEC, ACT, ONEG> fw;
        fw.load(a, c, pc.v * VEC, Cg, st);
        T* y = static_cast<T*>(a.y) + int64_t(pc.n) * a.S * C + c;
#pragma unroll
        for (int k = 0; k < KV; ++k) {
            const int p = p0 + pc.r + k * pc.rp;
            if (p >= pe) break;
            store_pack<T, VEC>(y + int64_t(p) * C, k < cnt ? fw(raw[k], a.act) : pack_zero<T, VEC>());
        }
    }
    if (pl.chunks > 1) cl_wait();     // no block leaves while a peer may read its sums
}

template <typename T, int VEC, int ACT, bool ONEG, int KV>
__global__ void __launch_bounds__(kGnThreads, 1) gn_resident_bwd_kernel(GnPlan pl) {
    const GroupNormArgs& a = pl.a;
    extern __shared__ float gn_smem[];
    const int C = int(a.C), G = int(a.G), Cg = C / G;
    pdl_launch_dependents();
    const ResPlace pc(pl, Cg, VEC);
    float2* sums = reinterpret_cast<float2*>(gn_smem);   // [slab_groups] S1/m, S2/m
    float2* mine = sums + pl.slab_groups;                // [slab_groups] this block's S1, S2
    float2* part = mine + pl.slab_groups;                // [rp][nv * VEC]
    const int len = valid_len(a, pc.n);
    const int p0 = pc.chunk * pl.rows, pv = min(len, p0 + pl.rows), pe = min(int(a.S), p0 + pl.rows);
    const int c = pc.c0 + pc.v * VEC;
    const T* x = static_cast<const T*>(a.x) + int64_t(pc.n) * a.xb + c;
    const T* dy = static_cast<const T*>(a.dy) + int64_t(pc.n) * a.gb + c;
    Pack<T, VEC> rx[KV], rg[KV];
    int cnt = 0;
#pragma unroll
    for (int k = 0; k < KV; ++k) {
        const int p = p0 + pc.r + k * pc.rp;
        if (pc.on && p < pv) {
            rx[k] = load_pack<T, VEC>(x + int64_t(p) * a.xp);
            rg[k] = load_pack<T, VEC>(dy + int64_t(p) * a.gp);
            ++cnt;
        }
    }
    const float2* stats = reinterpret_cast<const float2*>(a.stats) + int64_t(pc.n) * G + pc.g0;
    BackwardDx<T, VEC, ACT, ONEG> bw;
    if (pc.on) {
        bw.load(a, c, pc.v * VEC, Cg, stats);
        constexpr int NP = pairs_of(VEC);
        float2 sa[NP], sb[NP];
#pragma unroll
        for (int j = 0; j < NP; ++j) sa[j] = sb[j] = splat2(0.0f);
#pragma unroll
        for (int k = 0; k < KV; ++k) {
            if (k < cnt) bw.sums(rx[k], rg[k], a.act, sa, sb);
            reload(rx[k]);
            reload(rg[k]);
        }
#pragma unroll
        for (int j = 0; j < VEC; ++j)
            part[(pc.r * pc.nv + pc.v) * VEC + j] =
                j % 2 ? make_float2(sa[j / 2].y, sb[j / 2].y) : make_float2(sa[j / 2].x, sb[j / 2].x);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < pc.nv * VEC; i += blockDim.x) {   // rows of a channel, in order
        float2 s = part[i];
        for (int r = 1; r < pc.rp; ++r) {
            const float2 v = part[r * pc.nv * VEC + i];
            s.x += v.x;
            s.y += v.y;
        }
        part[i] = s;
        pl.csums[(int64_t(pc.n) * pl.chunks + pc.chunk) * C + pc.c0 + i] = s;
    }
    __syncthreads();
    {
        const int log = lanes_log(pc.gs, int(blockDim.x)), lane = int(threadIdx.x) & ((1 << log) - 1);
        for (int i0 = 0; i0 < pc.gs; i0 += int(blockDim.x) >> log) {
            const int g = i0 + (int(threadIdx.x) >> log);
            float2 s = make_float2(0.0f, 0.0f);
            if (g < pc.gs)
                for (int i = g * Cg + lane; i < (g + 1) * Cg; i += 1 << log) {
                    const float w = a.weight ? load_param(a.weight, a.param_dtype, pc.c0 + i) : 1.0f;
                    s.x += w * part[i].x;
                    s.y += w * part[i].y;
                }
            s = lanes_sum(s, log);
            if (g < pc.gs && lane == 0) mine[g] = s;
        }
    }
    if (pl.chunks > 1) cl_sync();
    else __syncthreads();
    const float inv = len > 0 ? 1.0f / (float(len) * float(Cg)) : 0.0f;
    for (int g = threadIdx.x; g < pc.gs; g += blockDim.x) {
        float2 s = mine[g];
        if (pl.chunks > 1) {
            s = make_float2(0.0f, 0.0f);
#pragma unroll
            for (int k = 0; k < kMaxCluster; ++k)
                if (k < pl.chunks) {
                    const float2 v = ld_cluster_f2(cluster_map(mine + g, uint32_t(k)));
                    s.x += v.x;
                    s.y += v.y;
                }
        }
        sums[g] = make_float2(s.x * inv, s.y * inv);
    }
    if (pl.chunks > 1) cl_arrive();   // this block has read its peers' sums
    __syncthreads();
    if (pc.on && a.dx != nullptr) {
        T* dx = static_cast<T*>(a.dx) + int64_t(pc.n) * a.S * C + c;
        bw.finish(pc.v * VEC, Cg, len, [&](int g) { return sums[g]; });
#pragma unroll
        for (int k = 0; k < KV; ++k) {
            const int p = p0 + pc.r + k * pc.rp;
            if (p >= pe) break;
            store_pack<T, VEC>(dx + int64_t(p) * C,
                               k < cnt ? bw.dx(rx[k], rg[k], a.act) : pack_zero<T, VEC>());
        }
    }
    if (pl.chunks > 1) cl_wait();     // no block leaves while a peer may read its sums
    if (pl.share) {
        cooperative_groups::this_grid().sync();
        share_param_grads(pl);
    }
}

// ---- host ---------------------------------------------------------------------

// Sweeps: one block per SM over all samples, at least 32 positions each.
void sweep_plan(GnPlan& pl) {
    const GroupNormArgs& a = pl.a;
    int64_t want = kSMs / a.N < 1 ? 1 : kSMs / a.N;
    if (want > ceil_div(a.S, 32)) want = ceil_div(a.S, 32);
    pl.rows = int(ceil_div(a.S, want));
    pl.chunks = int(ceil_div(a.S, pl.rows));
}

size_t carve(void* ws, GnPlan& pl, bool backward) {
    const GroupNormArgs& a = pl.a;
    Carve cv(ws);
    const size_t blocks = size_t(a.N) * size_t(pl.chunks);
    if (!backward) {
        pl.moments = cv.take<float2>(blocks * size_t(a.G));
    } else {
        pl.gsums = cv.take<float2>(blocks * size_t(a.G));
        pl.csums = cv.take<float2>(blocks * size_t(a.C));
    }
    return cv.size();
}

// Workspace of either path and any element type.  The resident path needs none
// forward; backward its chunks are at most a cluster's, a sample's positions, and
// the SMs there are for each sample.
size_t workspace_bytes(int64_t N, int64_t S, int64_t C, int64_t G, bool backward) {
    GnPlan pl{};
    pl.a.N = N;
    pl.a.S = S;
    pl.a.C = C;
    pl.a.G = G;
    sweep_plan(pl);
    const size_t sweeps = carve(nullptr, pl, backward);
    int64_t chunks = kSMs / N < S ? kSMs / N : S;
    if (chunks > kMaxCluster) chunks = kMaxCluster;
    pl.chunks = int(chunks);
    const size_t resident = backward ? carve(nullptr, pl, true) : 0;
    return sweeps > resident ? sweeps : resident;
}

// How a launch stands to the one before it, or to its own blocks.
enum LaunchKind { kPlain, kDependent, kCooperative };

// What has been asked of a device is kept, for each of them; calls come from any thread.
constexpr int kMaxDevices = 64;

// The current device if it takes a cooperative launch of one block for each of kSMs SMs, else -1.
int cooperative_device() {
    static std::atomic<int> known[kMaxDevices];   // 0: not asked yet, 1: yes, -1: no
    int dev = 0, sms = 0, coop = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return -1;
    int answer = known[dev].load(std::memory_order_relaxed);
    if (answer == 0) {
        cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
        cudaDeviceGetAttribute(&coop, cudaDevAttrCooperativeLaunch, dev);
        answer = sms >= kSMs && coop ? 1 : -1;
        known[dev].store(answer, std::memory_order_relaxed);
    }
    return answer > 0 ? dev : -1;
}

// Whether a launch's clusters can all run at the same time, so that its blocks
// may wait for one another (asked once for each device, kernel and cluster size).
template <void (*kernel)(GnPlan)>
bool all_at_once(int64_t blocks, int threads, size_t smem, int cluster) {
    const int dev = cooperative_device();
    if (dev < 0) return false;
    if (cluster == 1) return blocks <= kSMs;
    static std::atomic<int> known[kMaxDevices][kMaxCluster + 1];   // this kernel's clusters; 0: not asked yet
    int most = known[dev][cluster].load(std::memory_order_relaxed);
    if (most == 0) {
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(unsigned(cluster * kSMs));
        cfg.blockDim = dim3(unsigned(kGnThreads));
        cfg.dynamicSmemBytes = 48 * 1024;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = unsigned(cluster);
        attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        if (cudaOccupancyMaxActiveClusters(&most, kernel, &cfg) != cudaSuccess || most <= 0) {
            cudaGetLastError();
            most = -1;
        }
        known[dev][cluster].store(most, std::memory_order_relaxed);
    }
    return threads <= kGnThreads && smem <= 48 * 1024 && blocks / cluster <= most;
}

// What launch() answers where the blocks of a cooperative launch cannot all run at
// once although the device could hold them: the stream's context has fewer SMs (a
// partition of the device).  Nothing was launched.
constexpr int kTooLarge = 1;

// smem: dynamic, beside `merges` static bytes.  The opt-in is the kernel's and not the
// launch's: all calls, from any thread, set it to the same most.
template <typename K>
int launch(K kernel, const GnPlan& pl, int64_t blocks, int threads, size_t smem, size_t merges, int cluster,
           LaunchKind kind, cudaStream_t st) {
    if (blocks > 0x7fffffff) return fail(DOT_ERR_UNSUPPORTED, "group norm: too many blocks");
    if (smem + merges > kSmemDefault &&
        cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(kSmemMost - merges)) !=
            cudaSuccess)
        return check_launch("group norm");
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(unsigned(blocks));
    cfg.blockDim = dim3(unsigned(threads));
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    int n = 0;
    if (cluster > 1) {
        attr[n].id = cudaLaunchAttributeClusterDimension;
        attr[n].val.clusterDim.x = unsigned(cluster);
        attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
        ++n;
    }
    if (kind == kDependent) {
        attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[n].val.programmaticStreamSerializationAllowed = 1;
        ++n;
    }
    if (kind == kCooperative) {
        attr[n].id = cudaLaunchAttributeCooperative;
        attr[n].val.cooperative = 1;
        ++n;
    }
    cfg.attrs = attr;
    cfg.numAttrs = unsigned(n);
    if (cudaLaunchKernelEx(&cfg, kernel, pl) == cudaErrorCooperativeLaunchTooLarge) {
        cudaGetLastError();
        return kTooLarge;
    }
    return check_launch("group norm");
}

int launch_params(const GnPlan& pl, cudaStream_t st) {
    if (!pl.a.dweight && !pl.a.dbias) return DOT_OK;
    ProfScope ps(DOT_K_NORM_BWD, st);
    return launch(gn_params_kernel, pl, ceil_div(pl.a.C, kGnWarps), kGnThreads, 0, 0, 1, kDependent, st);
}

// The resident plan of a problem, if its blocks hold it in registers all at
// once, one block per SM.
//
// The slab is the narrowest run of whole groups of at least 64 bytes (two DRAM
// sectors, so neighbouring slabs share no sector pair) whose width is a whole
// number of vectors; blocks are added to a cluster until its registers hold
// the sample's positions, and beyond that (up to 8) while every block has an
// SM of its own, since a smaller share per block is a shorter call.
bool resident_plan(GnPlan& pl, int vec, int esz, bool backward, int& threads, int& vecs) {
    const GroupNormArgs& a = pl.a;
    const int64_t Cg = a.C / a.G;
    int64_t gs = 1;
    while (gs < a.G && (gs * Cg * esz < 64 || (gs * Cg) % vec != 0)) ++gs;
    const int64_t nv = gs * Cg / vec;
    if ((gs * Cg) % vec != 0 || nv > kGnThreads) return false;
    const int64_t rp = kGnThreads / nv, slabs = ceil_div(a.G, gs);
    int64_t K = ceil_div(a.S, rp * res_vecs(vec * esz, backward));
    if (K > kMaxCluster || a.N * slabs * K > kSMs) return false;
    while (2 * K <= kMaxCluster && a.N * slabs * 2 * K <= kSMs && ceil_div(a.S, 2 * K) >= rp) K *= 2;
    const int64_t rows = ceil_div(a.S, K);
    K = ceil_div(a.S, rows);
    pl.chunks = int(K);
    pl.rows = int(rows);
    pl.slab_groups = int(gs);
    pl.slabs = int(slabs);
    threads = kGnThreads;
    while (threads > 128 && (threads / 2) / nv >= rows) threads /= 2;   // one vector a thread is enough
    vecs = int(ceil_div(rows, threads / nv));
    return true;
}

template <typename T, int VEC, int ACT, bool ONEG, int KV>
int resident_run(GnPlan& pl, void* ws, int threads, bool backward, cudaStream_t st) {
    const size_t per = backward || !ONEG ? VEC : 1;
    const size_t smem = (2 * size_t(pl.slab_groups) + size_t(threads) * per) * sizeof(float2);
    const int64_t blocks = pl.a.N * pl.slabs * pl.chunks;
    if (!backward) {
        ProfScope ps(DOT_K_NORM_FWD, st);
        return launch(gn_resident_fwd_kernel<T, VEC, ACT, ONEG, KV>, pl, blocks, threads, smem, 0, pl.chunks, kPlain,
                      st);
    }
    int rc = DOT_OK;
    if constexpr (KV <= res_vecs(VEC * sizeof(T), true)) {
        carve(ws, pl, true);
        constexpr auto kernel = gn_resident_bwd_kernel<T, VEC, ACT, ONEG, KV>;
        pl.share = (pl.a.dweight || pl.a.dbias) && all_at_once<kernel>(blocks, threads, smem, pl.chunks);
        ProfScope ps(DOT_K_NORM_BWD, st);
        rc = launch(kernel, pl, blocks, threads, smem, 0, pl.chunks, pl.share ? kCooperative : kPlain, st);
        if (rc == kTooLarge) {
            pl.share = 0;
            rc = launch(kernel, pl, blocks, threads, smem, 0, pl.chunks, kPlain, st);
        }
    }
    if (rc || pl.share) return rc;
    return launch_params(pl, st);
}

template <typename T, int VEC, int ACT, bool ONEG>
int sweep_run(GnPlan& pl, void* ws, bool backward, cudaStream_t st) {
    const GroupNormArgs& a = pl.a;
    sweep_plan(pl);
    carve(ws, pl, backward);
    const size_t part = size_t(kGnThreads) * (backward || !ONEG ? VEC : 1);
    const size_t s1 = (size_t(a.G) + part) * sizeof(float2);
    const size_t s2 = size_t(a.G) * sizeof(float2);
    const int64_t blocks = a.N * pl.chunks;
    const bool second = !backward || a.dx != nullptr;
    int rc;
    {
        ProfScope ps(backward ? DOT_K_NORM_BWD : DOT_K_NORM_FWD, st, second ? 2 : 1);
        rc = backward ? launch(gn_sums_kernel<T, VEC, ACT, ONEG>, pl, blocks, kGnThreads, s1, 0, 1, kPlain, st)
                      : launch(gn_moments_kernel<T, VEC, ONEG>, pl, blocks, kGnThreads, s1, 0, 1, kPlain, st);
        if (!rc && second)
            rc = backward ? launch(gn_dx_kernel<T, VEC, ACT, ONEG>, pl, blocks, kGnThreads, s2, kSmemMerges, 1,
                                   kDependent, st)
                          : launch(gn_apply_kernel<T, VEC, ACT, ONEG>, pl, blocks, kGnThreads, s2, kSmemMerges, 1,
                                   kDependent, st);
    }
    if (rc) return rc;
    return backward && !second ? launch_params(pl, st) : DOT_OK;
}

// Both sweeps in one launch, where the rows lie one after another in memory, a
// row's vectors are at most one per thread, the groups leave the ring its shared
// memory, and every block that waits for others has an SM of its own; false where
// that does not hold.
template <typename T, int VEC, int ACT, bool ONEG>
bool fused_run(GnPlan& pl, void* ws, bool backward, cudaStream_t st, int& rc) {
    const GroupNormArgs& a = pl.a;
    if (a.C / VEC > kGnThreads || a.G > 1024 || a.xp != a.C || (backward && (a.gp != a.C || a.dx == nullptr)))
        return false;
    sweep_plan(pl);
    const int64_t blocks = a.N * pl.chunks;
    const bool waits = backward || pl.chunks > 1;
    if (waits && (blocks > kSMs || cooperative_device() < 0)) return false;
    carve(ws, pl, backward);
    const size_t part = size_t(kGnThreads) * (backward || !ONEG ? VEC : 1) * sizeof(float2);
    const size_t groups = size_t(a.G + 1) * (backward ? sizeof(float4) + sizeof(float2) : sizeof(float2) + sizeof(float));
    ProfScope ps(backward ? DOT_K_NORM_BWD : DOT_K_NORM_FWD, st);
    rc = backward ? launch(gn_fused_bwd_kernel<T, VEC, ACT, ONEG>, pl, blocks, kGnThreads,
                           Ring<2>::bytes() + groups + part, kSmemMerges, 1, kCooperative, st)
                  : launch(gn_fused_fwd_kernel<T, VEC, ACT, ONEG>, pl, blocks, kGnThreads,
                           Ring<1>::bytes() + groups + part, kSmemMerges, 1, waits ? kCooperative : kPlain, st);
    return rc != kTooLarge;
}

template <typename T, int VEC, int ACT, bool ONEG>
int run(const GroupNormArgs& a, void* ws, bool backward, cudaStream_t st) {
    GnPlan pl{};
    pl.a = a;
    int threads, vecs;
    if (!resident_plan(pl, VEC, sizeof(T), backward, threads, vecs)) {
        if constexpr (VEC * sizeof(T) == 16) {
            int rc = DOT_OK;
            if (fused_run<T, VEC, ACT, ONEG>(pl, ws, backward, st, rc)) return rc;
        }
        return sweep_run<T, VEC, ACT, ONEG>(pl, ws, backward, st);
    }
    constexpr int most = res_vecs(VEC * sizeof(T), true);
    if (vecs <= most / 4) return resident_run<T, VEC, ACT, ONEG, most / 4>(pl, ws, threads, backward, st);
    if (vecs <= most) return resident_run<T, VEC, ACT, ONEG, most>(pl, ws, threads, backward, st);
    return resident_run<T, VEC, ACT, ONEG, res_vecs(VEC * sizeof(T), false)>(pl, ws, threads, false, st);
}

template <typename T, int VEC, int ACT>
int by_group(const GroupNormArgs& a, void* ws, bool backward, cudaStream_t st) {
    if constexpr (VEC > 1)
        if ((a.C / a.G) % VEC != 0) return run<T, VEC, ACT, false>(a, ws, backward, st);
    return run<T, VEC, ACT, true>(a, ws, backward, st);
}

template <typename T, int VEC>
int by_act(const GroupNormArgs& a, void* ws, bool backward, cudaStream_t st) {
    // full-width vectors take the activation at compile time, narrower ones at run time
    if constexpr (VEC * sizeof(T) == 16) {
        switch (a.act) {
            case DOT_ACT_NONE: return by_group<T, VEC, kActNone>(a, ws, backward, st);
            case DOT_ACT_SILU: return by_group<T, VEC, kActSilu>(a, ws, backward, st);
            case DOT_ACT_GELU: return by_group<T, VEC, kActGelu>(a, ws, backward, st);
            default: return by_group<T, VEC, kActRelu>(a, ws, backward, st);
        }
    } else {
        return by_group<T, VEC, -1>(a, ws, backward, st);
    }
}

// Whether vectors of `vec` elements of `esz` bytes are aligned in every tensor, and
// a block's pairs of them leave the groups' their shared memory.
bool fits(const GroupNormArgs& a, int vec, int esz) {
    if (size_t(a.G + int64_t(kGnThreads) * vec) * sizeof(float2) > kSmemMost) return false;
    const int64_t bytes = int64_t(vec) * esz;
    auto ok = [&](const void* p) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; };
    if (a.C % vec || a.xb % vec || a.xp % vec || a.gb % vec || a.gp % vec) return false;
    return ok(a.x) && ok(a.dy) && ok(a.y) && ok(a.dx);
}

template <typename T>
int by_width(const GroupNormArgs& a, void* ws, bool backward, cudaStream_t st) {
    if (a.G > kMaxGroups) return fail(DOT_ERR_UNSUPPORTED, "more than " + std::to_string(kMaxGroups) + " groups");
    if constexpr (sizeof(T) == 2)
        if (fits(a, 8, 2)) return by_act<T, 8>(a, ws, backward, st);
    if (fits(a, 4, sizeof(T))) return by_act<T, 4>(a, ws, backward, st);
    if (fits(a, 2, sizeof(T))) return by_act<T, 2>(a, ws, backward, st);
    return by_act<T, 1>(a, ws, backward, st);
}

}  // namespace
}  // namespace dotb
