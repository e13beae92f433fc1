// Group normalisation with an activation on channels-last features, forward
// and backward (dot_group_norm_fwd / _bwd in include/dot_b200.h).
//
//   z = (x - mean) rstd w + b,  y = act(z)
//   dz = dy act'(z),  db_c = sum dz,  dw_c = sum dz xh,  xh = (x - mean) rstd
//   dx = rstd (w dz - S1/m - xh S2/m),  S1 = sum_g w dz,  S2 = sum_g w dz xh
//
// Bound: memory.  A position's channels are consecutive, so a thread owns one
// vector of VEC channels (its parameters stay in registers) and walks the
// positions; a block reads whole rows.
//
// Two sweeps per direction: the first leaves per-chunk partial sums in the
// workspace (a chunk: a range of one sample's positions), the second merges
// its sample's partials at its start and writes the result.  No atomics;
// every merge has a fixed order, so results are bitwise reproducible.
//
// Moments are kept as (mean, sum M of squared deviations): a thread merges a
// few positions at a time into its running pair, n = n1 + n2, d = mean2 - mean1,
//   mean = mean1 + d n2/n,  M = M1 + M2 + d^2 n1 n2/n
// (Chan, Golub and LeVeque, 1979), and warps merge the threads' and chunks'
// pairs against their common mean, so a mean far from zero cancels nothing.
#include "feature.cuh"
#include "features.h"
#include "internal.h"

namespace dotb {
namespace {

constexpr int kGnThreads = 256;
constexpr int kGnWarps = kGnThreads / 32;

struct GnPlan {
    GroupNormArgs a;
    int chunks;          // per sample
    int rows;            // positions per chunk
    float2* moments;     // fwd: [N][chunks][G] (mean, M) of a chunk
    float2* gsums;       // bwd: [N][chunks][G] (sum w dz, sum w dz xh)
    float2* csums;       // bwd: [N][chunks][C] (sum dz, sum dz xh)
};

__device__ __forceinline__ double warp_sum_f64(double v) {
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
    return v;
}

// A warp's merge of partial moments (mean_i, M_i) of n_i values each:
//   mean = sum n_i mean_i / n   (in fp64: the rounding of a mean far from zero
//                                is the stored value's only one),
//   M = sum M_i + n_i (mean_i - mean)^2.
// part(i) returns {n_i, mean_i, M_i} for i < count (n_i = 0: nothing there).
template <typename F>
__device__ __forceinline__ float2 warp_moments(int count, F part) {
    const int lane = threadIdx.x & 31;
    double n = 0.0, s = 0.0;
    for (int i = lane; i < count; i += 32) {
        const float3 v = part(i);
        n += double(v.x);
        s += double(v.x) * double(v.y);
    }
    n = warp_sum_f64(n);
    s = warp_sum_f64(s);
    const double mean = n > 0.0 ? s / n : 0.0;
    float m2 = 0.0f;
    for (int i = lane; i < count; i += 32) {
        const float3 v = part(i);
        const float d = float(double(v.y) - mean);
        if (v.x > 0.0f) m2 += v.z + v.x * d * d;
    }
    return make_float2(float(mean), warp_sum<32>(m2));
}

__device__ __forceinline__ int valid_len(const GroupNormArgs& a, int n) {
    if (a.lengths == nullptr) return int(a.S);
    return int(min(max(int64_t(__ldg(a.lengths + n)), int64_t(0)), a.S));
}

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

// ---- forward, sweep 1: moments of every group over a chunk --------------------
template <typename T, int VEC>
__global__ void __launch_bounds__(kGnThreads) gn_moments_kernel(GnPlan pl) {
    const GroupNormArgs& a = pl.a;
    extern __shared__ float gn_smem[];
    const int C = int(a.C), G = int(a.G), Cg = C / G, cv = C / VEC;
    float2* acc = reinterpret_cast<float2*>(gn_smem);   // [G] mean, M of the tiles so far
    float2* part = acc + G;                             // [rp][nv * VEC]
    const int n = blockIdx.x / pl.chunks, chunk = blockIdx.x - n * pl.chunks;
    const int len = valid_len(a, n);
    const int p0 = min(len, chunk * pl.rows), p1 = min(len, p0 + pl.rows);
    const T* x = static_cast<const T*>(a.x) + int64_t(n) * a.xb;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (int tile = 0; tile * kGnThreads < cv; ++tile) {
        const Place pc(cv, tile);
        const int c0 = tile * kGnThreads * VEC, c1 = c0 + pc.nv * VEC;
        if (pc.on) {
            constexpr int U = 4;
            float cnt = 0.0f, mean[VEC], m2[VEC];
#pragma unroll
            for (int j = 0; j < VEC; ++j) mean[j] = m2[j] = 0.0f;
            const T* xc = x + c0 + pc.v * VEC;
            for (int p = p0 + pc.r; p < p1; p += U * pc.rp) {
                Pack<T, VEC> raw[U];
                int k = 0;
#pragma unroll
                for (int u = 0; u < U; ++u)
                    if (p + u * pc.rp < p1) {
                        raw[u] = load_pack<T, VEC>(xc + int64_t(p + u * pc.rp) * a.xp);
                        ++k;
                    }
                // the batch's own moments (two passes over registers), merged into the running ones
                const float inv = 1.0f / float(k), tot = cnt + float(k), f = float(k) / tot, w = cnt * f;
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    float s = 0.0f, q = 0.0f;
#pragma unroll
                    for (int u = 0; u < U; ++u)
                        if (u < k) s += to_f32(raw[u].v[j]);
                    s *= inv;
#pragma unroll
                    for (int u = 0; u < U; ++u)
                        if (u < k) {
                            const float d = to_f32(raw[u].v[j]) - s;
                            q += d * d;
                        }
                    const float d = s - mean[j];
                    mean[j] += d * f;
                    m2[j] += q + d * d * w;
                }
                cnt = tot;
            }
#pragma unroll
            for (int j = 0; j < VEC; ++j) part[(pc.r * pc.nv + pc.v) * VEC + j] = make_float2(mean[j], m2[j]);
        }
        __syncthreads();
        for (int g = c0 / Cg + warp; g <= (c1 - 1) / Cg; g += kGnWarps) {
            const int ca = max(c0, g * Cg) - c0, wd = min(c1, (g + 1) * Cg) - c0 - ca;
            const int before = c0 + ca - g * Cg;   // channels of the group in earlier tiles
            const float2 old = acc[g];
            const float2 m = warp_moments(pc.rp * wd + (before > 0 ? 1 : 0), [&](int i) {
                if (i == pc.rp * wd) return make_float3(float(p1 - p0) * float(before), old.x, old.y);
                const int r = i / wd;
                const float2 v = part[r * pc.nv * VEC + ca + i - r * wd];
                return make_float3(float((max(p1 - p0 - r, 0) + pc.rp - 1) / pc.rp), v.x, v.y);
            });
            if (lane == 0) acc[g] = m;
        }
        __syncthreads();
    }
    for (int g = threadIdx.x; g < G; g += kGnThreads)
        pl.moments[int64_t(blockIdx.x) * G + g] = acc[g];
}

// ---- forward, sweep 2: merge the sample's chunks, write y ---------------------
template <typename T, int VEC, int ACT>
__global__ void __launch_bounds__(kGnThreads) gn_apply_kernel(GnPlan pl) {
    const GroupNormArgs& a = pl.a;
    extern __shared__ float gn_smem[];
    float2* st = reinterpret_cast<float2*>(gn_smem);   // [G] mean, rstd
    const int C = int(a.C), G = int(a.G), Cg = C / G, cv = C / VEC;
    const int n = blockIdx.x / pl.chunks, chunk = blockIdx.x - n * pl.chunks;
    const int len = valid_len(a, n);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (int g = warp; g < G; g += kGnWarps) {
        const float2 m = warp_moments(pl.chunks, [&](int k) {
            const float2 v = pl.moments[(int64_t(n) * pl.chunks + k) * G + g];
            return make_float3(float(min(max(len - k * pl.rows, 0), pl.rows)) * float(Cg), v.x, v.y);
        });
        if (lane == 0) {
            const float rstd = 1.0f / sqrtf((len > 0 ? m.y / (float(len) * float(Cg)) : 0.0f) + a.eps);
            st[g] = make_float2(m.x, rstd);
            if (chunk == 0) reinterpret_cast<float2*>(a.stats)[int64_t(n) * G + g] = st[g];
        }
    }
    __syncthreads();
    const int p0 = chunk * pl.rows, p1 = min(int(a.S), p0 + pl.rows);
    const T* x = static_cast<const T*>(a.x) + int64_t(n) * a.xb;
    T* y = static_cast<T*>(a.y) + int64_t(n) * a.S * C;
    for (int tile = 0; tile * kGnThreads < cv; ++tile) {
        const Place pc(cv, tile);
        if (!pc.on) continue;
        const int c = (tile * kGnThreads + pc.v) * VEC;
        float mean[VEC], sc[VEC], sh[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            const float2 v = st[(c + j) / Cg];
            mean[j] = v.x;
            sc[j] = v.y * (a.weight ? load_param(a.weight, a.param_dtype, c + j) : 1.0f);
            sh[j] = a.bias ? load_param(a.bias, a.param_dtype, c + j) : 0.0f;
        }
        for (int p = p0 + pc.r; p < p1; p += pc.rp) {
            float o[VEC];
            if (p < len) {
                const Pack<T, VEC> raw = load_pack<T, VEC>(x + int64_t(p) * a.xp + c);
#pragma unroll
                for (int j = 0; j < VEC; ++j)
                    o[j] = act_fwd<ACT>((to_f32(raw.v[j]) - mean[j]) * sc[j] + sh[j], a.act);
            } else {
#pragma unroll
                for (int j = 0; j < VEC; ++j) o[j] = 0.0f;
            }
            store_pack<T, VEC>(y + int64_t(p) * C + c, pack<T, VEC>(o));
        }
    }
}

// ---- backward, sweep 1: per-channel and per-group sums over a chunk -----------
template <typename T, int VEC, int ACT>
__global__ void __launch_bounds__(kGnThreads) gn_sums_kernel(GnPlan pl) {
    const GroupNormArgs& a = pl.a;
    extern __shared__ float gn_smem[];
    const int C = int(a.C), G = int(a.G), Cg = C / G, cv = C / VEC;
    float2* acc = reinterpret_cast<float2*>(gn_smem);   // [G]
    float2* part = acc + G;                             // [rp][nv * VEC]
    const int n = blockIdx.x / pl.chunks, chunk = blockIdx.x - n * pl.chunks;
    const int len = valid_len(a, n);
    const int p0 = min(len, chunk * pl.rows), p1 = min(len, p0 + pl.rows);
    const T* x = static_cast<const T*>(a.x) + int64_t(n) * a.xb;
    const T* dy = static_cast<const T*>(a.dy) + int64_t(n) * a.gb;
    const float2* st = reinterpret_cast<const float2*>(a.stats) + int64_t(n) * G;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (int g = threadIdx.x; g < G; g += kGnThreads) acc[g] = make_float2(0.0f, 0.0f);
    __syncthreads();
    for (int tile = 0; tile * kGnThreads < cv; ++tile) {
        const Place pc(cv, tile);
        const int c0 = tile * kGnThreads * VEC, c1 = c0 + pc.nv * VEC;
        if (pc.on) {
            const int c = c0 + pc.v * VEC;
            float mean[VEC], rstd[VEC], w[VEC], b[VEC], sa[VEC], sb[VEC];
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                const float2 v = st[(c + j) / Cg];
                mean[j] = v.x;
                rstd[j] = v.y;
                w[j] = a.weight ? load_param(a.weight, a.param_dtype, c + j) : 1.0f;
                b[j] = a.bias ? load_param(a.bias, a.param_dtype, c + j) : 0.0f;
                sa[j] = sb[j] = 0.0f;
            }
            for (int p = p0 + pc.r; p < p1; p += pc.rp) {
                const Pack<T, VEC> rx = load_pack<T, VEC>(x + int64_t(p) * a.xp + c);
                const Pack<T, VEC> rg = load_pack<T, VEC>(dy + int64_t(p) * a.gp + c);
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    const float xh = (to_f32(rx.v[j]) - mean[j]) * rstd[j];
                    const float dz = to_f32(rg.v[j]) * act_slope<ACT>(xh * w[j] + b[j], a.act);
                    sa[j] += dz;
                    sb[j] += dz * xh;
                }
            }
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
            pl.csums[int64_t(blockIdx.x) * C + c0 + i] = s;
        }
        __syncthreads();
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
        __syncthreads();
    }
    for (int g = threadIdx.x; g < G; g += kGnThreads) pl.gsums[int64_t(blockIdx.x) * G + g] = acc[g];
}

// ---- backward, sweep 2: merge the sample's group sums, write dx ---------------
template <typename T, int VEC, int ACT>
__global__ void __launch_bounds__(kGnThreads) gn_dx_kernel(GnPlan pl) {
    const GroupNormArgs& a = pl.a;
    extern __shared__ float gn_smem[];
    float4* gv = reinterpret_cast<float4*>(gn_smem);   // [G] mean, rstd, S1/m, S2/m
    const int C = int(a.C), G = int(a.G), Cg = C / G, cv = C / VEC;
    const int n = blockIdx.x / pl.chunks, chunk = blockIdx.x - n * pl.chunks;
    const int len = valid_len(a, n);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const float inv = len > 0 ? 1.0f / (float(len) * float(Cg)) : 0.0f;
    for (int g = warp; g < G; g += kGnWarps) {
        float2 s = make_float2(0.0f, 0.0f);
        for (int k = lane; k < pl.chunks; k += 32) {
            const float2 v = pl.gsums[(int64_t(n) * pl.chunks + k) * G + g];
            s.x += v.x;
            s.y += v.y;
        }
        s.x = warp_sum<32>(s.x);
        s.y = warp_sum<32>(s.y);
        if (lane == 0) {
            const float2 v = reinterpret_cast<const float2*>(a.stats)[int64_t(n) * G + g];
            gv[g] = make_float4(v.x, v.y, s.x * inv, s.y * inv);
        }
    }
    __syncthreads();
    const int p0 = chunk * pl.rows, p1 = min(int(a.S), p0 + pl.rows);
    const T* x = static_cast<const T*>(a.x) + int64_t(n) * a.xb;
    const T* dy = static_cast<const T*>(a.dy) + int64_t(n) * a.gb;
    T* dx = static_cast<T*>(a.dx) + int64_t(n) * a.S * C;
    for (int tile = 0; tile * kGnThreads < cv; ++tile) {
        const Place pc(cv, tile);
        if (!pc.on) continue;
        const int c = (tile * kGnThreads + pc.v) * VEC;
        float w[VEC], b[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            w[j] = a.weight ? load_param(a.weight, a.param_dtype, c + j) : 1.0f;
            b[j] = a.bias ? load_param(a.bias, a.param_dtype, c + j) : 0.0f;
        }
        for (int p = p0 + pc.r; p < p1; p += pc.rp) {
            float o[VEC];
            if (p < len) {
                const Pack<T, VEC> rx = load_pack<T, VEC>(x + int64_t(p) * a.xp + c);
                const Pack<T, VEC> rg = load_pack<T, VEC>(dy + int64_t(p) * a.gp + c);
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    const float4 v = gv[(c + j) / Cg];
                    const float xh = (to_f32(rx.v[j]) - v.x) * v.y;
                    const float dz = to_f32(rg.v[j]) * act_slope<ACT>(xh * w[j] + b[j], a.act);
                    // w dz rounded as in its sum: the gradient of a group of one value is 0
                    o[j] = v.y * (__fsub_rn(__fmul_rn(w[j], dz), v.z) - xh * v.w);
                }
            } else {
#pragma unroll
                for (int j = 0; j < VEC; ++j) o[j] = 0.0f;
            }
            store_pack<T, VEC>(dx + int64_t(p) * C + c, pack<T, VEC>(o));
        }
    }
}

// ---- backward: the parameters' gradients from the chunks' channel sums --------
__global__ void __launch_bounds__(kGnThreads) gn_params_kernel(GnPlan pl) {
    const GroupNormArgs& a = pl.a;
    __shared__ float2 part[kGnWarps][32];
    const int C = int(a.C), lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int c = blockIdx.x * 32 + lane;
    const int64_t rows = a.N * pl.chunks;
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

// ---- host ---------------------------------------------------------------------

void plan_chunks(int64_t N, int64_t S, int& chunks, int& rows) {
    // about four blocks per SM over all samples, at least 32 positions each
    int64_t want = ceil_div(int64_t(148) * 4, N);
    if (want > ceil_div(S, 32)) want = ceil_div(S, 32);
    rows = int(ceil_div(S, want));
    chunks = int(ceil_div(S, rows));
}

void carve(Carve& cv, GnPlan& pl, bool backward) {
    const GroupNormArgs& a = pl.a;
    const size_t blocks = size_t(a.N) * size_t(pl.chunks);
    if (!backward) {
        pl.moments = cv.take<float2>(blocks * size_t(a.G));
    } else {
        pl.gsums = cv.take<float2>(blocks * size_t(a.G));
        pl.csums = cv.take<float2>(blocks * size_t(a.C));
    }
}

GnPlan make_plan(const GroupNormArgs& a) {
    GnPlan pl{};
    pl.a = a;
    plan_chunks(a.N, a.S, pl.chunks, pl.rows);
    return pl;
}

template <typename K>
int allow_smem(K kernel, size_t bytes) {
    if (bytes <= 48 * 1024) return DOT_OK;
    if (bytes > 227 * 1024) return fail(DOT_ERR_UNSUPPORTED, "group norm: too many groups");
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(bytes)) != cudaSuccess)
        return check_launch("group norm");
    return DOT_OK;
}

template <typename T, int VEC, int ACT>
int fwd_launch(const GnPlan& pl, cudaStream_t st) {
    const unsigned blocks = unsigned(pl.a.N * pl.chunks);
    const size_t s1 = (size_t(pl.a.G) + size_t(kGnThreads) * VEC) * sizeof(float2);
    const size_t s2 = size_t(pl.a.G) * sizeof(float2);
    int rc = allow_smem(gn_moments_kernel<T, VEC>, s1);
    if (!rc) rc = allow_smem(gn_apply_kernel<T, VEC, ACT>, s2);
    if (rc) return rc;
    ProfScope ps(DOT_K_NORM_FWD, st, 2);
    gn_moments_kernel<T, VEC><<<blocks, kGnThreads, s1, st>>>(pl);
    gn_apply_kernel<T, VEC, ACT><<<blocks, kGnThreads, s2, st>>>(pl);
    return check_launch("group norm forward");
}

template <typename T, int VEC, int ACT>
int bwd_launch(const GnPlan& pl, cudaStream_t st) {
    const unsigned blocks = unsigned(pl.a.N * pl.chunks);
    const size_t s1 = (size_t(pl.a.G) + size_t(kGnThreads) * VEC) * sizeof(float2);
    const size_t s2 = size_t(pl.a.G) * sizeof(float4);
    int rc = allow_smem(gn_sums_kernel<T, VEC, ACT>, s1);
    if (!rc) rc = allow_smem(gn_dx_kernel<T, VEC, ACT>, s2);
    if (rc) return rc;
    const bool params = pl.a.dweight || pl.a.dbias;
    ProfScope ps(DOT_K_NORM_BWD, st, 1 + (pl.a.dx ? 1 : 0) + (params ? 1 : 0));
    gn_sums_kernel<T, VEC, ACT><<<blocks, kGnThreads, s1, st>>>(pl);
    if (pl.a.dx) gn_dx_kernel<T, VEC, ACT><<<blocks, kGnThreads, s2, st>>>(pl);
    if (params) gn_params_kernel<<<unsigned(ceil_div(pl.a.C, 32)), kGnThreads, 0, st>>>(pl);
    return check_launch("group norm backward");
}

template <typename T, int VEC, bool BWD>
int by_act(const GnPlan& pl, cudaStream_t st) {
    // full-width vectors take the activation at compile time, narrower ones at run time
    if constexpr (VEC * sizeof(T) == 16) {
        switch (pl.a.act) {
            case DOT_ACT_NONE: return BWD ? bwd_launch<T, VEC, kActNone>(pl, st) : fwd_launch<T, VEC, kActNone>(pl, st);
            case DOT_ACT_SILU: return BWD ? bwd_launch<T, VEC, kActSilu>(pl, st) : fwd_launch<T, VEC, kActSilu>(pl, st);
            case DOT_ACT_GELU: return BWD ? bwd_launch<T, VEC, kActGelu>(pl, st) : fwd_launch<T, VEC, kActGelu>(pl, st);
            default: return BWD ? bwd_launch<T, VEC, kActRelu>(pl, st) : fwd_launch<T, VEC, kActRelu>(pl, st);
        }
    } else {
        return BWD ? bwd_launch<T, VEC, -1>(pl, st) : fwd_launch<T, VEC, -1>(pl, st);
    }
}

// Whether vectors of `vec` elements of `esz` bytes are aligned in every tensor.
bool fits(const GroupNormArgs& a, int vec, int esz) {
    const int64_t bytes = int64_t(vec) * esz;
    auto ok = [&](const void* p) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; };
    if (a.C % vec || a.xb % vec || a.xp % vec || a.gb % vec || a.gp % vec) return false;
    return ok(a.x) && ok(a.dy) && ok(a.y) && ok(a.dx);
}

template <typename T, bool BWD>
int by_width(const GnPlan& pl, cudaStream_t st) {
    if constexpr (sizeof(T) == 2)
        if (fits(pl.a, 8, 2)) return by_act<T, 8, BWD>(pl, st);
    if (fits(pl.a, 4, sizeof(T))) return by_act<T, 4, BWD>(pl, st);
    if (fits(pl.a, 2, sizeof(T))) return by_act<T, 2, BWD>(pl, st);
    return by_act<T, 1, BWD>(pl, st);
}

template <bool BWD>
int by_dtype(const GnPlan& pl, cudaStream_t st) {
    switch (pl.a.dtype) {
        case DOT_F32: return by_width<float, BWD>(pl, st);
        case DOT_BF16: return by_width<__nv_bfloat16, BWD>(pl, st);
        default: return by_width<__half, BWD>(pl, st);
    }
}

size_t ws_bytes(int64_t N, int64_t S, int64_t C, int64_t G, bool backward) {
    GroupNormArgs a{};
    a.N = N;
    a.S = S;
    a.C = C;
    a.G = G;
    GnPlan pl = make_plan(a);
    Carve cv(nullptr);
    carve(cv, pl, backward);
    return cv.size();
}

}  // namespace

size_t gn_fwd_ws(int64_t N, int64_t S, int64_t C, int64_t G) { return ws_bytes(N, S, C, G, false); }
size_t gn_bwd_ws(int64_t N, int64_t S, int64_t C, int64_t G) { return ws_bytes(N, S, C, G, true); }

int gn_fwd(const GroupNormArgs& a, void* ws, cudaStream_t st) {
    GnPlan pl = make_plan(a);
    Carve cv(ws);
    carve(cv, pl, false);
    return by_dtype<false>(pl, st);
}

int gn_bwd(const GroupNormArgs& a, void* ws, cudaStream_t st) {
    GnPlan pl = make_plan(a);
    Carve cv(ws);
    carve(cv, pl, true);
    return by_dtype<true>(pl, st);
}

}  // namespace dotb
