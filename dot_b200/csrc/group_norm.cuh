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
// Two paths, chosen by size (resident_plan): a cluster of blocks that holds its
// share of a sample in registers and reads it once, and two sweeps for samples
// beyond that.  No atomics; every merge has a fixed order, so results are
// bitwise reproducible.
//
// Moments are kept as (mean, sum M of squared deviations) of x - pivot, the
// pivot one of the group's values: a mean far from zero then costs its own
// rounding and no more.  A thread takes two passes over the positions in its
// registers and merges a batch into its running pair, n = n1 + n2,
// d = mean2 - mean1:  mean = mean1 + d n2/n,  M = M1 + M2 + d^2 n1 n2/n
// (Chan, Golub and LeVeque, 1979); threads' and blocks' pairs are joined by Merge.
#pragma once

#include "cluster.cuh"
#include "feature.cuh"
#include "features.h"
#include "internal.h"
#include "tma.cuh"

namespace dotb {
namespace {

constexpr int kGnThreads = 256;
constexpr int kGnWarps = kGnThreads / 32;

// Resident path: threads of a block, and the registers of a thread that hold
// x (and as many dy): vectors of 16 bytes or fewer.
constexpr int kResThreads = 512;
constexpr int kMaxCluster = 8;
constexpr int res_vecs(int bytes) { return bytes >= 16 ? 8 : bytes >= 8 ? 16 : 32; }

struct GnPlan {
    GroupNormArgs a;
    int n0;              // sweeps: first sample of this launch
    int chunks;          // blocks that share a sample's positions
    int rows;            // positions per chunk
    int parts;           // partial sums per sample in the workspace
    int slab_groups;     // resident: groups of a block's channel slab
    int slabs;           // resident: slabs per sample
    float2* moments;     // sweeps, fwd: [N][parts][G] (mean, M) of a cluster
    float2* gsums;       // sweeps, bwd: [N][parts][G] (sum w dz, sum w dz xh)
    float2* csums;       // bwd: [N][parts][C] (sum dz, sum dz xh)
};

// Merging partial moments (mean_i, M_i) of n_i values each about one of the
// means:  d_i = mean_i - about,
//   mean = about + sum n_i d_i / n,   M = sum (M_i + n_i d_i^2) - (sum n_i d_i)^2 / n.
// What cancels in M is at most n / n_i of it, from that mean's own distance.
struct Merge {
    float n = 0.0f, nd = 0.0f, m2 = 0.0f;
    __device__ __forceinline__ void add(float about, float ni, float mean, float m) {
        const float d = mean - about, w = ni * d;
        if (ni > 0.0f) {   // the moments of nothing are not looked at
            n += ni;
            nd += w;
            m2 += m + w * d;
        }
    }
    __device__ __forceinline__ void warp() {
        n = warp_sum<32>(n);
        nd = warp_sum<32>(nd);
        m2 = warp_sum<32>(m2);
    }
    // (mean, M)
    __device__ __forceinline__ float2 pair(float about) const {
        const float d = n > 0.0f ? nd / n : 0.0f;
        return n > 0.0f ? make_float2(about + d, m2 - nd * d) : make_float2(0.0f, 0.0f);
    }
};

__device__ __forceinline__ float2 mean_rstd(float pivot, float2 mean_m, int len, int Cg, float eps) {
    const float var = len > 0 ? mean_m.y / (float(len) * float(Cg)) : 0.0f;
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

// dx of one element from its group's statistics and sums (S1/m, S2/m).  w dz is
// rounded as in its sum: the gradient of a group of one value is 0.
template <int ACT>
__device__ __forceinline__ float dx_of(float x, float dy, float mean, float rstd, float w, float b, float2 s, int act) {
    const float xh = (x - mean) * rstd;
    const float dz = dy * act_slope<ACT>(xh * w + b, act);
    return rstd * (__fsub_rn(__fmul_rn(w, dz), s.x) - xh * s.y);
}

// ---- backward: the parameters' gradients from the blocks' channel sums ---------
__global__ void __launch_bounds__(kGnThreads) gn_params_kernel(GnPlan pl) {
    const GroupNormArgs& a = pl.a;
    __shared__ float2 part[kGnWarps][32];
    const int C = int(a.C), lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int c = blockIdx.x * 32 + lane;
    const int64_t rows = a.N * pl.parts;
    float2 s = make_float2(0.0f, 0.0f);
    if (c < C)
        for (int64_t r = warp; r < rows; r += kGnWarps) {
            const float2 v = pl.csums[r * C + c];
            s.x += v.x;
            s.y += v.y;
        }
    part[warp][lane] = s;
    __syncthreads();
    if (warp == 0 && c < C) {
        for (int k = 1; k < kGnWarps; ++k) {
            s.x += part[k][lane].x;
            s.y += part[k][lane].y;
        }
        if (a.dbias) store_param(a.dbias, a.param_dtype, c, s.x);
        if (a.dweight) store_param(a.dweight, a.param_dtype, c, s.y);
    }
}

// ---- two sweeps per direction --------------------------------------------------
//
// A block reads whole rows of one chunk (a range of one sample's positions).
// The first sweep leaves the chunk's partial sums in the workspace, the second
// merges its sample's partials at its start and writes the result, walking its
// rows backwards: it begins with those that the first sweep read last.

// Clusters of kSweepCluster blocks join their partials through distributed
// shared memory first, so a sample's chunks leave an eighth as many.
constexpr int kSweepCluster = 8;

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

// A running (count of positions, mean, M) per channel, or one for a vector
// that lies in one group.
template <int VEC, bool ONEG>
struct Running {
    static constexpr int NG = ONEG ? 1 : VEC;
    float n = 0.0f, mean[NG], m2[NG];
    __device__ Running() {
#pragma unroll
        for (int j = 0; j < NG; ++j) mean[j] = m2[j] = 0.0f;
    }
    // Merges the first k of U positions, by two passes over registers.
    template <typename T, int U, bool FULL>
    __device__ __forceinline__ void add(const Pack<T, VEC> (&raw)[U], const float (&pivot)[NG], int k) {
        constexpr int J = ONEG ? VEC : 1;   // values of a position in a pair
        const float fk = FULL ? float(U) : float(k), tot = n + fk, f = fk / tot, w = n * f;
        const float inv = (FULL ? 1.0f / float(U) : 1.0f / fk) * (1.0f / float(J));
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            float s = 0.0f, q = 0.0f;
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (FULL || u < k)
#pragma unroll
                    for (int j = 0; j < J; ++j) s += to_f32(raw[u].v[g + j]) - pivot[g];
            s *= inv;
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (FULL || u < k)
#pragma unroll
                    for (int j = 0; j < J; ++j) {
                        const float d = (to_f32(raw[u].v[g + j]) - pivot[g]) - s;
                        q += d * d;
                    }
            const float d = s - mean[g];
            mean[g] += d * f;
            m2[g] += q + d * d * (w * float(J));
        }
        n = tot;
    }
};

// Forward, sweep 1: moments of every group over a chunk.
template <typename T, int VEC, bool ONEG>
__global__ void __launch_bounds__(kGnThreads) gn_moments_kernel(GnPlan pl) {
    const GroupNormArgs& a = pl.a;
    extern __shared__ float gn_smem[];
    constexpr int W = ONEG ? 1 : VEC, U = 8;
    const int C = int(a.C), G = int(a.G), Cg = C / G, cv = C / VEC;
    float2* acc = reinterpret_cast<float2*>(gn_smem);   // [G] mean, M of the tiles so far
    float2* part = acc + G;                             // [rp][nv * W]
    const int n = pl.n0 + int(blockIdx.x) / pl.chunks, chunk = int(blockIdx.x) % pl.chunks;
    const int len = valid_len(a, n);
    const int p0 = min(len, chunk * pl.rows), p1 = min(len, p0 + pl.rows);
    const T* x = static_cast<const T*>(a.x) + int64_t(n) * a.xb;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    pdl_launch_dependents();
    for (int tile = 0; tile * kGnThreads < cv; ++tile) {
        const Place pc(cv, tile);
        const int c0 = tile * kGnThreads * VEC, c1 = c0 + pc.nv * VEC;
        if (pc.on) {
            Running<VEC, ONEG> run;
            const T* xc = x + c0 + pc.v * VEC;
            float pivot[W];
#pragma unroll
            for (int j = 0; j < W; ++j) pivot[j] = group_pivot(x, len, (c0 + pc.v * VEC + j) / Cg * Cg);
            const int64_t step = int64_t(pc.rp) * a.xp;
            int p = p0 + pc.r;
            for (; p + (U - 1) * pc.rp < p1; p += U * pc.rp) {
                Pack<T, VEC> raw[U];
                const T* at = xc + int64_t(p) * a.xp;
#pragma unroll
                for (int u = 0; u < U; ++u) raw[u] = load_pack<T, VEC>(at + u * step);
                run.template add<T, U, true>(raw, pivot, U);
            }
            if (p < p1) {
                Pack<T, VEC> raw[U];
                const T* at = xc + int64_t(p) * a.xp;
                const int k = (p1 - p + pc.rp - 1) / pc.rp;
#pragma unroll
                for (int u = 0; u < U; ++u)
                    if (u < k) raw[u] = load_pack<T, VEC>(at + u * step);
                run.template add<T, U, false>(raw, pivot, k);
            }
#pragma unroll
            for (int j = 0; j < W; ++j) part[(pc.r * pc.nv + pc.v) * W + j] = make_float2(run.mean[j], run.m2[j]);
        }
        __syncthreads();
        for (int g = c0 / Cg + warp; g <= (c1 - 1) / Cg; g += kGnWarps) {
            const int ca = max(c0, g * Cg), before = ca - g * Cg;   // channels of the group in earlier tiles
            const int wd = (min(c1, (g + 1) * Cg) - ca) / (VEC / W), at = (ca - c0) / (VEC / W);
            const float2 old = acc[g];
            const float about = part[at].x;   // row 0 is there if any is
            Merge m;
            for (int i = lane; i < pc.rp * wd; i += 32) {
                const int r = i / wd;
                const float2 v = part[r * pc.nv * W + at + i - r * wd];
                m.add(about, float((max(p1 - p0 - r, 0) + pc.rp - 1) / pc.rp) * float(VEC / W), v.x, v.y);
            }
            if (before > 0 && lane == 0) m.add(about, float(p1 - p0) * float(before), old.x, old.y);
            m.warp();
            if (lane == 0) acc[g] = m.pair(about);
        }
        __syncthreads();
    }
    // one partial per cluster: its blocks share out the groups
    cl_sync();
    const int rank = chunk % kSweepCluster, first = chunk - rank;
    pdl_wait();   // the launches before this one are done when it is
    for (int g = rank * kGnThreads + int(threadIdx.x); g < G; g += kSweepCluster * kGnThreads) {
        float2 v[kSweepCluster];
#pragma unroll
        for (int k = 0; k < kSweepCluster; ++k) v[k] = ld_cluster_f2(cluster_map(acc + g, uint32_t(k)));
        Merge m;
#pragma unroll
        for (int k = 0; k < kSweepCluster; ++k)
            m.add(v[0].x, float(rows_of(len, first + k, pl.rows)) * float(Cg), v[k].x, v[k].y);
        pl.moments[(int64_t(n) * (pl.parts) + first / kSweepCluster) * G + g] = m.pair(v[0].x);
    }
    cl_sync();    // no block leaves while a peer may read its moments
}

// Forward, sweep 2: merges the sample's chunks, writes y.
template <typename T, int VEC, int ACT, bool ONEG>
__global__ void __launch_bounds__(kGnThreads) gn_apply_kernel(GnPlan pl) {
    const GroupNormArgs& a = pl.a;
    extern __shared__ float gn_smem[];
    float2* st = reinterpret_cast<float2*>(gn_smem);   // [G] mean, rstd
    constexpr int NG = ONEG ? 1 : VEC, U = 4;
    const int C = int(a.C), G = int(a.G), Cg = C / G, cv = C / VEC;
    const int n = pl.n0 + int(blockIdx.x) / pl.chunks, chunk = int(blockIdx.x) % pl.chunks;
    const int len = valid_len(a, n);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const T* x = static_cast<const T*>(a.x) + int64_t(n) * a.xb;
    pdl_launch_dependents();
    pdl_wait();
    {
        __shared__ Merge merged[kGnWarps][32];
        const int parts = pl.parts, span = kSweepCluster * pl.rows;
        for (int g = lane; g < (G + 31) / 32 * 32; g += 32) {   // a lane a group, the warps share the partials
            Merge m;
            const float2* from = pl.moments + int64_t(n) * parts * G + g;
            const float about = g < G ? from[0].x : 0.0f;
            if (g < G)
#pragma unroll 8
                for (int k = warp; k < parts; k += kGnWarps) {
                    const float2 v = from[int64_t(k) * G];
                    m.add(about, float(rows_of(len, k, span)) * float(Cg), v.x, v.y);
                }
            merged[warp][lane] = m;
            __syncthreads();
            if (warp == 0 && g < G) {
#pragma unroll
                for (int k = 1; k < kGnWarps; ++k) {
                    m.n += merged[k][lane].n;
                    m.nd += merged[k][lane].nd;
                    m.m2 += merged[k][lane].m2;
                }
                st[g] = mean_rstd(group_pivot(x, len, g * Cg), m.pair(about), len, Cg, a.eps);
                if (chunk == 0) reinterpret_cast<float2*>(a.stats)[int64_t(n) * G + g] = st[g];
            }
            __syncthreads();
        }
    }
    const int p0 = chunk * pl.rows, pe = min(int(a.S), p0 + pl.rows), pv = min(max(len, p0), pe);
    T* y = static_cast<T*>(a.y) + int64_t(n) * a.S * C;
    for (int tile = 0; tile * kGnThreads < cv; ++tile) {
        const Place pc(cv, tile);
        if (!pc.on) continue;
        const int c = (tile * kGnThreads + pc.v) * VEC;
        float mean[NG], sc[VEC], sh[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            const float2 v = st[(c + j) / Cg];
            if (j < NG) mean[j] = v.x;
            sc[j] = v.y * (a.weight ? load_param(a.weight, a.param_dtype, c + j) : 1.0f);
            sh[j] = a.bias ? load_param(a.bias, a.param_dtype, c + j) : 0.0f;
        }
        auto write = [&](int p, const Pack<T, VEC>& raw) {
            float o[VEC];
#pragma unroll
            for (int j = 0; j < VEC; ++j)
                o[j] = act_fwd<ACT>((to_f32(raw.v[j]) - mean[ONEG ? 0 : j]) * sc[j] + sh[j], a.act);
            store_pack<T, VEC>(y + int64_t(p) * C + c, pack<T, VEC>(o));
        };
        for (int p = pv + pc.r; p < pe; p += pc.rp) {   // padding
            float o[VEC];
#pragma unroll
            for (int j = 0; j < VEC; ++j) o[j] = 0.0f;
            store_pack<T, VEC>(y + int64_t(p) * C + c, pack<T, VEC>(o));
        }
        int p = pv - 1 - pc.r;
        for (; p - (U - 1) * pc.rp >= p0; p -= U * pc.rp) {
            Pack<T, VEC> raw[U];
#pragma unroll
            for (int u = 0; u < U; ++u) raw[u] = load_pack<T, VEC>(x + int64_t(p - u * pc.rp) * a.xp + c);
#pragma unroll
            for (int u = 0; u < U; ++u) write(p - u * pc.rp, raw[u]);
        }
        for (; p >= p0; p -= pc.rp) write(p, load_pack<T, VEC>(x + int64_t(p) * a.xp + c));
    }
}

// Backward, sweep 1: per-channel and per-group sums over a chunk.
template <typename T, int VEC, int ACT, bool ONEG>
__global__ void __launch_bounds__(kGnThreads) gn_sums_kernel(GnPlan pl) {
    const GroupNormArgs& a = pl.a;
    extern __shared__ float gn_smem[];
    constexpr int NG = ONEG ? 1 : VEC, U = 4;
    const int C = int(a.C), G = int(a.G), Cg = C / G, cv = C / VEC;
    float2* acc = reinterpret_cast<float2*>(gn_smem);   // [G]
    float2* part = acc + G;                             // [rp][nv * VEC]
    const int n = pl.n0 + int(blockIdx.x) / pl.chunks, chunk = int(blockIdx.x) % pl.chunks;
    const int rank = chunk % kSweepCluster;
    const int64_t slot = int64_t(n) * (pl.parts) + chunk / kSweepCluster;
    const int len = valid_len(a, n);
    const int p0 = min(len, chunk * pl.rows), p1 = min(len, p0 + pl.rows);
    const T* x = static_cast<const T*>(a.x) + int64_t(n) * a.xb;
    const T* dy = static_cast<const T*>(a.dy) + int64_t(n) * a.gb;
    const float2* st = reinterpret_cast<const float2*>(a.stats) + int64_t(n) * G;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    pdl_launch_dependents();
    for (int g = threadIdx.x; g < G; g += kGnThreads) acc[g] = make_float2(0.0f, 0.0f);
    __syncthreads();
    for (int tile = 0; tile * kGnThreads < cv; ++tile) {
        const Place pc(cv, tile);
        const int c0 = tile * kGnThreads * VEC, c1 = c0 + pc.nv * VEC;
        if (pc.on) {
            const int c = c0 + pc.v * VEC;
            float mean[NG], rstd[NG], w[VEC], b[VEC], sa[VEC], sb[VEC];
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                if (j < NG) {
                    const float2 v = st[(c + j) / Cg];
                    mean[j] = v.x;
                    rstd[j] = v.y;
                }
                w[j] = a.weight ? load_param(a.weight, a.param_dtype, c + j) : 1.0f;
                b[j] = a.bias ? load_param(a.bias, a.param_dtype, c + j) : 0.0f;
                sa[j] = sb[j] = 0.0f;
            }
            auto take = [&](const Pack<T, VEC>& rx, const Pack<T, VEC>& rg) {
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    const float xh = (to_f32(rx.v[j]) - mean[ONEG ? 0 : j]) * rstd[ONEG ? 0 : j];
                    const float dz = to_f32(rg.v[j]) * act_slope<ACT>(xh * w[j] + b[j], a.act);
                    sa[j] += dz;
                    sb[j] += dz * xh;
                }
            };
            int p = p0 + pc.r;
            for (; p + (U - 1) * pc.rp < p1; p += U * pc.rp) {
                Pack<T, VEC> rx[U], rg[U];
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    rx[u] = load_pack<T, VEC>(x + int64_t(p + u * pc.rp) * a.xp + c);
                    rg[u] = load_pack<T, VEC>(dy + int64_t(p + u * pc.rp) * a.gp + c);
                }
#pragma unroll
                for (int u = 0; u < U; ++u) take(rx[u], rg[u]);
            }
            for (; p < p1; p += pc.rp)
                take(load_pack<T, VEC>(x + int64_t(p) * a.xp + c), load_pack<T, VEC>(dy + int64_t(p) * a.gp + c));
#pragma unroll
            for (int j = 0; j < VEC; ++j) part[(pc.r * pc.nv + pc.v) * VEC + j] = make_float2(sa[j], sb[j]);
        }
        __syncthreads();
        for (int i = threadIdx.x; i < pc.nv * VEC; i += kGnThreads) {   // rows of a channel, in order
            float2 s = part[i];
            for (int r = 1; r < pc.rp; ++r) {
                const float2 v = part[r * pc.nv * VEC + i];
                s.x += v.x;
                s.y += v.y;
            }
            part[i] = s;
        }
        cl_sync();
        // one partial per cluster: its blocks share out the channels
        for (int i = rank * kGnThreads + int(threadIdx.x); i < pc.nv * VEC; i += kSweepCluster * kGnThreads) {
            float2 s = make_float2(0.0f, 0.0f);
#pragma unroll
            for (int k = 0; k < kSweepCluster; ++k) {
                const float2 v = ld_cluster_f2(cluster_map(part + i, uint32_t(k)));
                s.x += v.x;
                s.y += v.y;
            }
            pl.csums[slot * C + c0 + i] = s;
        }
        for (int g = c0 / Cg + warp; g <= (c1 - 1) / Cg; g += kGnWarps) {
            const int ca = max(c0, g * Cg), cb = min(c1, (g + 1) * Cg);
            float2 s = make_float2(0.0f, 0.0f);
            for (int c = ca + lane; c < cb; c += 32) {
                const float w = a.weight ? load_param(a.weight, a.param_dtype, c) : 1.0f;
                s.x += w * part[c - c0].x;
                s.y += w * part[c - c0].y;
            }
            s.x = warp_sum<32>(s.x);
            s.y = warp_sum<32>(s.y);
            if (lane == 0) {
                acc[g].x += s.x;
                acc[g].y += s.y;
            }
        }
        cl_sync();    // the peers have read this tile's sums
    }
    pdl_wait();   // the launches before this one are done when it is
    for (int g = rank * kGnThreads + int(threadIdx.x); g < G; g += kSweepCluster * kGnThreads) {
        float2 s = make_float2(0.0f, 0.0f);
#pragma unroll
        for (int k = 0; k < kSweepCluster; ++k) {
            const float2 v = ld_cluster_f2(cluster_map(acc + g, uint32_t(k)));
            s.x += v.x;
            s.y += v.y;
        }
        pl.gsums[slot * G + g] = s;
    }
    cl_sync();        // no block leaves while a peer may read its sums
}

// Backward, sweep 2: merges the sample's group sums, writes dx.
template <typename T, int VEC, int ACT, bool ONEG>
__global__ void __launch_bounds__(kGnThreads) gn_dx_kernel(GnPlan pl) {
    const GroupNormArgs& a = pl.a;
    extern __shared__ float gn_smem[];
    float4* gv = reinterpret_cast<float4*>(gn_smem);   // [G] mean, rstd, S1/m, S2/m
    constexpr int NG = ONEG ? 1 : VEC, U = 4;
    const int C = int(a.C), G = int(a.G), Cg = C / G, cv = C / VEC;
    const int n = pl.n0 + int(blockIdx.x) / pl.chunks, chunk = int(blockIdx.x) % pl.chunks;
    const int len = valid_len(a, n);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const float inv = len > 0 ? 1.0f / (float(len) * float(Cg)) : 0.0f;
    pdl_launch_dependents();
    pdl_wait();
    {
        __shared__ float2 merged[kGnWarps][32];
        const int parts = pl.parts;
        for (int g = lane; g < (G + 31) / 32 * 32; g += 32) {   // a lane a group, the warps share the partials
            float2 s = make_float2(0.0f, 0.0f);
            if (g < G)
#pragma unroll 8
                for (int k = warp; k < parts; k += kGnWarps) {
                    const float2 v = pl.gsums[(int64_t(n) * parts + k) * G + g];
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
                const float2 v = reinterpret_cast<const float2*>(a.stats)[int64_t(n) * G + g];
                gv[g] = make_float4(v.x, v.y, s.x * inv, s.y * inv);
            }
            __syncthreads();
        }
    }
    const int p0 = chunk * pl.rows, pe = min(int(a.S), p0 + pl.rows), pv = min(max(len, p0), pe);
    const T* x = static_cast<const T*>(a.x) + int64_t(n) * a.xb;
    const T* dy = static_cast<const T*>(a.dy) + int64_t(n) * a.gb;
    T* dx = static_cast<T*>(a.dx) + int64_t(n) * a.S * C;
    for (int tile = 0; tile * kGnThreads < cv; ++tile) {
        const Place pc(cv, tile);
        if (!pc.on) continue;
        const int c = (tile * kGnThreads + pc.v) * VEC;
        float w[VEC], b[VEC];
        float4 gr[NG];
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            if (j < NG) gr[j] = gv[(c + j) / Cg];
            w[j] = a.weight ? load_param(a.weight, a.param_dtype, c + j) : 1.0f;
            b[j] = a.bias ? load_param(a.bias, a.param_dtype, c + j) : 0.0f;
        }
        auto write = [&](int p, const Pack<T, VEC>& rx, const Pack<T, VEC>& rg) {
            float o[VEC];
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                const float4 v = gr[ONEG ? 0 : j];
                o[j] = dx_of<ACT>(to_f32(rx.v[j]), to_f32(rg.v[j]), v.x, v.y, w[j], b[j], make_float2(v.z, v.w), a.act);
            }
            store_pack<T, VEC>(dx + int64_t(p) * C + c, pack<T, VEC>(o));
        };
        for (int p = pv + pc.r; p < pe; p += pc.rp) {   // padding
            float o[VEC];
#pragma unroll
            for (int j = 0; j < VEC; ++j) o[j] = 0.0f;
            store_pack<T, VEC>(dx + int64_t(p) * C + c, pack<T, VEC>(o));
        }
        int p = pv - 1 - pc.r;
        for (; p - (U - 1) * pc.rp >= p0; p -= U * pc.rp) {
            Pack<T, VEC> rx[U], rg[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                rx[u] = load_pack<T, VEC>(x + int64_t(p - u * pc.rp) * a.xp + c);
                rg[u] = load_pack<T, VEC>(dy + int64_t(p - u * pc.rp) * a.gp + c);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) write(p - u * pc.rp, rx[u], rg[u]);
        }
        for (; p >= p0; p -= pc.rp)
            write(p, load_pack<T, VEC>(x + int64_t(p) * a.xp + c), load_pack<T, VEC>(dy + int64_t(p) * a.gp + c));
    }
}

// ---- resident path ------------------------------------------------------------
//
// A cluster of `chunks` blocks holds one sample's positions of one channel slab
// (whole groups) in registers: x (and dy) are read once, the blocks exchange
// their groups' partial sums through distributed shared memory, and the result
// is written from the registers.  One launch per direction.

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
__global__ void __launch_bounds__(kResThreads, 2) gn_resident_fwd_kernel(GnPlan pl) {
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
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = int(blockDim.x) >> 5;
    if (pc.on) {
        // two passes over the registers
        constexpr int W = ONEG ? 1 : VEC, J = VEC / W;
        const float inv = cnt > 0 ? 1.0f / float(cnt * J) : 0.0f;
        float s[W], q[W], pivot[W];
#pragma unroll
        for (int j = 0; j < W; ++j) {
            s[j] = q[j] = 0.0f;
            pivot[j] = group_pivot(x - c, len, (c + j) / Cg * Cg);
        }
#pragma unroll
        for (int k = 0; k < KV; ++k)
            if (k < cnt)
#pragma unroll
                for (int j = 0; j < VEC; ++j) s[j / J] += to_f32(raw[k].v[j]) - pivot[j / J];
#pragma unroll
        for (int j = 0; j < W; ++j) s[j] *= inv;
#pragma unroll
        for (int k = 0; k < KV; ++k) {
            reload(raw[k]);
            if (k < cnt)
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    const float d = (to_f32(raw[k].v[j]) - pivot[j / J]) - s[j / J];
                    q[j / J] += d * d;
                }
            reload(raw[k]);
        }
#pragma unroll
        for (int j = 0; j < W; ++j) part[(pc.r * pc.nv + pc.v) * W + j] = make_float2(s[j], q[j]);
    }
    __syncthreads();
    {
        const int wd = ONEG ? Cg / VEC : Cg, width = pc.nv * (ONEG ? 1 : VEC), rows = max(pv - p0, 0);
        for (int g = warp; g < pc.gs; g += warps) {
            const float about = part[g * wd].x;   // row 0 is there if any is
            Merge m;
            for (int i = lane; i < pc.rp * wd; i += 32) {
                const int r = i / wd;
                const float2 v = part[r * width + g * wd + i - r * wd];
                m.add(about, float((max(rows - r, 0) + pc.rp - 1) / pc.rp) * float(ONEG ? VEC : 1), v.x, v.y);
            }
            m.warp();
            if (lane == 0) mine[g] = m.pair(about);
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
            m = all.pair(v[0].x);
        }
        st[g] = mean_rstd(group_pivot(x - c, len, (pc.g0 + g) * Cg), m, len, Cg, a.eps);
        if (pc.chunk == 0) reinterpret_cast<float2*>(a.stats)[int64_t(pc.n) * G + pc.g0 + g] = st[g];
    }
    if (pl.chunks > 1) cl_arrive();   // this block has read its peers' sums
    __syncthreads();
    if (pc.on) {
        float mean[ONEG ? 1 : VEC], sc[VEC], sh[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            const float2 v = st[(pc.v * VEC + j) / Cg];
            mean[ONEG ? 0 : j] = v.x;
            sc[j] = v.y * (a.weight ? load_param(a.weight, a.param_dtype, c + j) : 1.0f);
            sh[j] = a.bias ? load_param(a.bias, a.param_dtype, c + j) : 0.0f;
        }
        T* y = static_cast<T*>(a.y) + int64_t(pc.n) * a.S * C + c;
#pragma unroll
        for (int k = 0; k < KV; ++k) {
            const int p = p0 + pc.r + k * pc.rp;
            if (p >= pe) break;
            float o[VEC];
#pragma unroll
            for (int j = 0; j < VEC; ++j) o[j] = 0.0f;
            if (k < cnt)
#pragma unroll
                for (int j = 0; j < VEC; ++j)
                    o[j] = act_fwd<ACT>((to_f32(raw[k].v[j]) - mean[ONEG ? 0 : j]) * sc[j] + sh[j], a.act);
            store_pack<T, VEC>(y + int64_t(p) * C, pack<T, VEC>(o));
        }
    }
    if (pl.chunks > 1) cl_wait();     // no block leaves while a peer may read its sums
}

template <typename T, int VEC, int ACT, bool ONEG, int KV>
__global__ void __launch_bounds__(kResThreads, 1) gn_resident_bwd_kernel(GnPlan pl) {
    const GroupNormArgs& a = pl.a;
    extern __shared__ float gn_smem[];
    const int C = int(a.C), G = int(a.G), Cg = C / G;
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
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = int(blockDim.x) >> 5;
    const float2* stats = reinterpret_cast<const float2*>(a.stats) + int64_t(pc.n) * G + pc.g0;
    constexpr int NG = ONEG ? 1 : VEC;
    float mean[NG], rstd[NG], w[VEC], b[VEC];
    if (pc.on) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            if (j < NG) {
                const float2 v = stats[(pc.v * VEC + j) / Cg];
                mean[j] = v.x;
                rstd[j] = v.y;
            }
            w[j] = a.weight ? load_param(a.weight, a.param_dtype, c + j) : 1.0f;
            b[j] = a.bias ? load_param(a.bias, a.param_dtype, c + j) : 0.0f;
        }
        float sa[VEC], sb[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) sa[j] = sb[j] = 0.0f;
#pragma unroll
        for (int k = 0; k < KV; ++k) {
            if (k < cnt)
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    const float xh = (to_f32(rx[k].v[j]) - mean[ONEG ? 0 : j]) * rstd[ONEG ? 0 : j];
                    const float dz = to_f32(rg[k].v[j]) * act_slope<ACT>(xh * w[j] + b[j], a.act);
                    sa[j] += dz;
                    sb[j] += dz * xh;
                }
            reload(rx[k]);
            reload(rg[k]);
        }
#pragma unroll
        for (int j = 0; j < VEC; ++j) part[(pc.r * pc.nv + pc.v) * VEC + j] = make_float2(sa[j], sb[j]);
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
        pl.csums[(int64_t(pc.n) * pl.parts + pc.chunk) * C + pc.c0 + i] = s;
    }
    __syncthreads();
    for (int g = warp; g < pc.gs; g += warps) {
        float2 s = make_float2(0.0f, 0.0f);
        for (int i = g * Cg + lane; i < (g + 1) * Cg; i += 32) {
            const float wi = a.weight ? load_param(a.weight, a.param_dtype, pc.c0 + i) : 1.0f;
            s.x += wi * part[i].x;
            s.y += wi * part[i].y;
        }
        s.x = warp_sum<32>(s.x);
        s.y = warp_sum<32>(s.y);
        if (lane == 0) mine[g] = s;
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
        float2 sg[NG];
#pragma unroll
        for (int j = 0; j < NG; ++j) sg[j] = sums[(pc.v * VEC + j) / Cg];
#pragma unroll
        for (int k = 0; k < KV; ++k) {
            const int p = p0 + pc.r + k * pc.rp;
            if (p >= pe) break;
            float o[VEC];
#pragma unroll
            for (int j = 0; j < VEC; ++j) o[j] = 0.0f;
            if (k < cnt)
#pragma unroll
                for (int j = 0; j < VEC; ++j)
                    o[j] = dx_of<ACT>(to_f32(rx[k].v[j]), to_f32(rg[k].v[j]), mean[ONEG ? 0 : j], rstd[ONEG ? 0 : j],
                                      w[j], b[j], sg[ONEG ? 0 : j], a.act);
            store_pack<T, VEC>(dx + int64_t(p) * C, pack<T, VEC>(o));
        }
    }
    if (pl.chunks > 1) cl_wait();     // no block leaves while a peer may read its sums
}

// ---- host ---------------------------------------------------------------------

// Sweeps: samples are taken in batches whose x (and dy) the L2 cache still
// holds when the second sweep reads them again.
constexpr int64_t kBatchBytes = int64_t(48) << 20;

void sweep_plan(GnPlan& pl, int esz, bool backward, int& batch) {
    const GroupNormArgs& a = pl.a;
    const int64_t bytes = a.S * a.C * esz * (backward ? 2 : 1);
    int64_t nb = kBatchBytes / (bytes > 0 ? bytes : 1);
    nb = nb < 1 ? 1 : nb > a.N ? a.N : nb;
    nb = ceil_div(a.N, ceil_div(a.N, nb));   // batches of one size
    // about four blocks per SM over a batch, at least 32 positions each
    int64_t want = ceil_div(int64_t(148) * 4, nb);
    if (want > ceil_div(a.S, 32)) want = ceil_div(a.S, 32);
    batch = int(nb);
    pl.parts = int(ceil_div(want, kSweepCluster));
    pl.chunks = pl.parts * kSweepCluster;
    pl.rows = int(ceil_div(a.S, pl.chunks));   // the last chunks may be empty
}

size_t carve(void* ws, GnPlan& pl, bool backward) {
    const GroupNormArgs& a = pl.a;
    Carve cv(ws);
    const size_t blocks = size_t(a.N) * size_t(pl.parts);
    if (!backward) {
        pl.moments = cv.take<float2>(blocks * size_t(a.G));
    } else {
        pl.gsums = cv.take<float2>(blocks * size_t(a.G));
        pl.csums = cv.take<float2>(blocks * size_t(a.C));
    }
    return cv.size();
}

// Workspace of either path and any element type.
size_t workspace_bytes(int64_t N, int64_t S, int64_t C, int64_t G, bool backward) {
    GnPlan pl{};
    pl.a.N = N;
    pl.a.S = S;
    pl.a.C = C;
    pl.a.G = G;
    size_t most = 0;
    for (int esz = 2; esz <= 4; esz += 2) {
        int batch;
        sweep_plan(pl, esz, backward, batch);
        const size_t b = carve(nullptr, pl, backward);
        if (b > most) most = b;
    }
    pl.parts = kMaxCluster;   // resident: one of each block
    const size_t b = backward ? carve(nullptr, pl, true) : 0;
    return b > most ? b : most;
}

template <typename K>
int launch(K kernel, const GnPlan& pl, int64_t blocks, int threads, size_t smem, int cluster, bool dependent,
           cudaStream_t st) {
    if (blocks > 0x7fffffff) return fail(DOT_ERR_UNSUPPORTED, "group norm: too many blocks");
    if (smem > 48 * 1024) {
        if (smem > 227 * 1024) return fail(DOT_ERR_UNSUPPORTED, "group norm: too many groups");
        if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem)) != cudaSuccess)
            return check_launch("group norm");
    }
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
    if (dependent) {
        attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[n].val.programmaticStreamSerializationAllowed = 1;
        ++n;
    }
    cfg.attrs = attr;
    cfg.numAttrs = unsigned(n);
    cudaLaunchKernelEx(&cfg, kernel, pl);
    return check_launch("group norm");
}

int launch_params(const GnPlan& pl, cudaStream_t st) {
    if (!pl.a.dweight && !pl.a.dbias) return DOT_OK;
    ProfScope ps(DOT_K_NORM_BWD, st);
    return launch(gn_params_kernel, pl, ceil_div(pl.a.C, 32), kGnThreads, 0, 1, false, st);
}

// The resident plan of a problem, if a cluster holds a slab of it.
//
// The slab is the narrowest run of whole groups of at least 64 bytes (two DRAM
// sectors, so neighbouring slabs share no sector pair) whose width is a whole
// number of vectors; blocks are added to a cluster until its registers hold
// the sample's positions, and beyond that (up to 8) while all blocks together
// stay within two per SM, since a smaller share per block is a shorter call.
bool resident_plan(GnPlan& pl, int vec, int esz, int& threads, int& vecs) {
    const GroupNormArgs& a = pl.a;
    const int64_t Cg = a.C / a.G;
    int64_t gs = 1;
    while (gs < a.G && (gs * Cg * esz < 64 || (gs * Cg) % vec != 0)) ++gs;
    const int64_t nv = gs * Cg / vec;
    if ((gs * Cg) % vec != 0 || nv > kResThreads) return false;
    const int64_t rp = kResThreads / nv, slabs = ceil_div(a.G, gs);
    int64_t K = ceil_div(a.S, rp * res_vecs(vec * esz));
    if (K > kMaxCluster) return false;
    while (2 * K <= kMaxCluster && a.N * slabs * 2 * K <= 2 * 148 && ceil_div(a.S, 2 * K) >= rp) K *= 2;
    const int64_t rows = ceil_div(a.S, K);
    K = ceil_div(a.S, rows);
    pl.chunks = pl.parts = int(K);
    pl.rows = int(rows);
    pl.slab_groups = int(gs);
    pl.slabs = int(slabs);
    threads = kResThreads;
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
        return launch(gn_resident_fwd_kernel<T, VEC, ACT, ONEG, KV>, pl, blocks, threads, smem, pl.chunks, false, st);
    }
    carve(ws, pl, true);
    int rc;
    {
        ProfScope ps(DOT_K_NORM_BWD, st);
        rc = launch(gn_resident_bwd_kernel<T, VEC, ACT, ONEG, KV>, pl, blocks, threads, smem, pl.chunks, false, st);
    }
    return rc ? rc : launch_params(pl, st);
}

template <typename T, int VEC, int ACT, bool ONEG>
int sweep_run(GnPlan& pl, void* ws, bool backward, cudaStream_t st) {
    const GroupNormArgs& a = pl.a;
    int batch;
    sweep_plan(pl, sizeof(T), backward, batch);
    carve(ws, pl, backward);
    const size_t part = size_t(kGnThreads) * (backward || !ONEG ? VEC : 1);
    const size_t s1 = (size_t(a.G) + part) * sizeof(float2);
    const size_t s2 = size_t(a.G) * (backward ? sizeof(float4) : sizeof(float2));
    for (int64_t n = 0; n < a.N; n += batch) {
        pl.n0 = int(n);
        const int64_t blocks = (a.N - n < batch ? a.N - n : batch) * pl.chunks;
        const bool second = !backward || a.dx != nullptr;
        ProfScope ps(backward ? DOT_K_NORM_BWD : DOT_K_NORM_FWD, st, second ? 2 : 1);
        int rc = backward
            ? launch(gn_sums_kernel<T, VEC, ACT, ONEG>, pl, blocks, kGnThreads, s1, kSweepCluster, n > 0, st)
            : launch(gn_moments_kernel<T, VEC, ONEG>, pl, blocks, kGnThreads, s1, kSweepCluster, n > 0, st);
        if (!rc && second)
            rc = backward ? launch(gn_dx_kernel<T, VEC, ACT, ONEG>, pl, blocks, kGnThreads, s2, 1, true, st)
                          : launch(gn_apply_kernel<T, VEC, ACT, ONEG>, pl, blocks, kGnThreads, s2, 1, true, st);
        if (rc) return rc;
    }
    return backward ? launch_params(pl, st) : DOT_OK;
}

template <typename T, int VEC, int ACT, bool ONEG>
int run(const GroupNormArgs& a, void* ws, bool backward, cudaStream_t st) {
    GnPlan pl{};
    pl.a = a;
    int threads, vecs;
    if (!resident_plan(pl, VEC, sizeof(T), threads, vecs)) return sweep_run<T, VEC, ACT, ONEG>(pl, ws, backward, st);
    constexpr int most = res_vecs(VEC * sizeof(T)), some = most / 2;
    if (vecs == 1 && VEC * sizeof(T) == 16) return resident_run<T, VEC, ACT, ONEG, 1>(pl, ws, threads, backward, st);
    if (vecs <= some) return resident_run<T, VEC, ACT, ONEG, some>(pl, ws, threads, backward, st);
    return resident_run<T, VEC, ACT, ONEG, most>(pl, ws, threads, backward, st);
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

// Whether vectors of `vec` elements of `esz` bytes are aligned in every tensor.
bool fits(const GroupNormArgs& a, int vec, int esz) {
    const int64_t bytes = int64_t(vec) * esz;
    auto ok = [&](const void* p) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; };
    if (a.C % vec || a.xb % vec || a.xp % vec || a.gb % vec || a.gp % vec) return false;
    return ok(a.x) && ok(a.dy) && ok(a.y) && ok(a.dx);
}

template <typename T>
int by_width(const GroupNormArgs& a, void* ws, bool backward, cudaStream_t st) {
    if constexpr (sizeof(T) == 2)
        if (fits(a, 8, 2)) return by_act<T, 8>(a, ws, backward, st);
    if (fits(a, 4, sizeof(T))) return by_act<T, 4>(a, ws, backward, st);
    if (fits(a, 2, sizeof(T))) return by_act<T, 2>(a, ws, backward, st);
    return by_act<T, 1>(a, ws, backward, st);
}

}  // namespace
}  // namespace dotb
