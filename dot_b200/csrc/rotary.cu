// Rotary positions with several axes (dot_rotary in include/dot_b200.h).
//
//   angle[t, p] = sum_a positions[t, a] * freqs[p, a]
//   (x, y) -> (x cos - y sin, y cos + x sin)   for pair p of every head of token t
//
// The backward is the same kernel with the sine negated: the turn is
// orthogonal.  Bound: memory (each element is read and written once, with
// about five operations); a token's P sines and cosines serve all its heads.
//
// A block takes kRotThreads threads' worth of whole tokens: it forms their
// sines and cosines once into shared memory, then every thread owns one
// vector of VP pairs of a token (kept in registers) and walks the heads.
#include "feature.cuh"
#include "features.h"
#include "internal.h"

namespace dotb {
namespace {

constexpr int kRotThreads = 256;

struct RotPlan {
    int slots;          // threads per head: P / VP pair vectors, then the copied tail's vectors (two per slot)
    int pair_slots;
    int hgroups;        // heads of a token handled side by side
    int tokens;         // tokens per block
    int64_t ntok;       // B * L
};

template <typename I>
__device__ __forceinline__ double position(const void* p, int64_t i) {
    return double(static_cast<const I*>(p)[i]);
}

// Sine and cosine of a token's angle.  The angle in turns is formed in fp64
// and reduced to [-1/2, 1/2] before it is rounded to fp32: a position of 2^30
// keeps an absolute error below 2^-20 turns where an fp32 angle has lost it.
template <typename PT>
__device__ __forceinline__ float2 sincos_of(const RotaryArgs& a, int64_t pos_off, int p) {
    double angle = 0.0;
    for (int ax = 0; ax < a.A; ++ax)
        angle = fma(position<PT>(a.positions, pos_off + ax * a.ps[2]), double(a.freqs[p * a.A + ax]), angle);
    const double turns = angle * 0.15915494309189533577;   // 1 / (2 pi)
    const float r = float(turns - rint(turns));
    float s, c;
    sincospif(2.0f * r, &s, &c);
    return make_float2(c, a.inverse ? -s : s);
}

template <typename T, int VP, bool IL, typename PT>
__global__ void __launch_bounds__(kRotThreads) rotary_kernel(RotaryArgs a, RotPlan pl) {
    extern __shared__ float2 cs[];   // [tokens][P] cos, sin
    const int P = int(a.P);
    const int64_t t0 = int64_t(blockIdx.x) * pl.tokens;
    const int nt = int(min(int64_t(pl.tokens), pl.ntok - t0));
    for (int i = threadIdx.x; i < nt * P; i += kRotThreads) {
        const int tl = i / P, p = i - tl * P;
        const int64_t t = t0 + tl, b = t / a.L, l = t - b * a.L;
        cs[i] = sincos_of<PT>(a, b * a.ps[0] + l * a.ps[1], p);
    }
    __syncthreads();

    const int per_token = pl.slots * pl.hgroups;
    const int H = int(a.Hq + a.Hk);
    for (int i = threadIdx.x; i < nt * per_token; i += kRotThreads) {
        const int tl = i / per_token, w = i - tl * per_token;
        const int hg = w / pl.slots, slot = w - hg * pl.slots;
        const int64_t t = t0 + tl, b = t / a.L, l = t - b * a.L;
        const bool turn = slot < pl.pair_slots;
        float c[VP], s[VP];
        int o0, o1;          // offsets of the slot's two vectors within a head
        bool second = true;
        if (turn) {
#pragma unroll
            for (int j = 0; j < VP; ++j) {
                const float2 v = cs[tl * P + slot * VP + j];
                c[j] = v.x;
                s[j] = v.y;
            }
            o0 = IL ? slot * 2 * VP : slot * VP;
            o1 = IL ? o0 + VP : P + o0;
        } else {
            o0 = 2 * P + (slot - pl.pair_slots) * 2 * VP;
            o1 = o0 + VP;
            second = o1 < int(a.D);
        }
        for (int h = hg; h < H; h += pl.hgroups) {
            const bool is_q = h < int(a.Hq);
            const int hh = is_q ? h : h - int(a.Hq);
            const T* src = is_q ? static_cast<const T*>(a.q) + b * a.qs[0] + l * a.qs[1] + hh * a.qs[2]
                                : static_cast<const T*>(a.k) + b * a.ks[0] + l * a.ks[1] + hh * a.ks[2];
            T* dst = is_q ? static_cast<T*>(a.q_out) + (t * a.Hq + hh) * a.D
                          : static_cast<T*>(a.k_out) + (t * a.Hk + hh) * a.D;
            const Pack<T, VP> p0 = load_pack<T, VP>(src + o0);
            if (!turn) {
                store_pack<T, VP>(dst + o0, p0);
                if (second) store_pack<T, VP>(dst + o1, load_pack<T, VP>(src + o1));
                continue;
            }
            const Pack<T, VP> p1 = load_pack<T, VP>(src + o1);
            float e[2 * VP];
#pragma unroll
            for (int j = 0; j < VP; ++j) {
                e[j] = to_f32(p0.v[j]);
                e[VP + j] = to_f32(p1.v[j]);
            }
            Pack<T, VP> r0, r1;
#pragma unroll
            for (int j = 0; j < VP; ++j) {
                const float x = IL ? e[2 * j] : e[j], y = IL ? e[2 * j + 1] : e[VP + j];
                // the products' roundings are spelled out: every width gives the same bits
                const T u = from_f32<T>(__fmaf_rn(x, c[j], -__fmul_rn(y, s[j])));
                const T v = from_f32<T>(__fmaf_rn(y, c[j], __fmul_rn(x, s[j])));
                const int iu = IL ? 2 * j : j, iv = IL ? 2 * j + 1 : VP + j;
                (iu < VP ? r0.v[iu % VP] : r1.v[iu % VP]) = u;
                (iv < VP ? r0.v[iv % VP] : r1.v[iv % VP]) = v;
            }
            store_pack<T, VP>(dst + o0, r0);
            store_pack<T, VP>(dst + o1, r1);
        }
    }
}

template <typename T, int VP, bool IL, typename PT>
int launch(const RotaryArgs& a, cudaStream_t st) {
    RotPlan pl;
    pl.ntok = a.B * a.L;
    pl.pair_slots = int(a.P / VP);
    pl.slots = pl.pair_slots + int(ceil_div(ceil_div(a.D - 2 * a.P, VP), 2));
    const int64_t H = a.Hq + a.Hk;
    // Heads side by side: all of them for a few tokens (one access each, so a
    // small call is one round trip), fewer as the tokens alone fill the GPU.
    int64_t hg = H;
    while (hg > 1 && pl.ntok * pl.slots * hg > int64_t(148) * 2048 * 4) hg = (hg + 1) / 2;
    pl.hgroups = int(hg);
    const int64_t per_token = int64_t(pl.slots) * pl.hgroups;
    int64_t tokens = per_token >= kRotThreads ? 1 : kRotThreads / per_token;
    const int64_t fit = a.P > 0 ? kMaxPairs / a.P : tokens;
    if (tokens > fit) tokens = fit;
    pl.tokens = int(tokens);
    const int64_t blocks = ceil_div(pl.ntok, tokens);
    if (blocks > 0x7fffffff) return fail(DOT_ERR_UNSUPPORTED, "too many tokens");
    ProfScope ps(DOT_K_ROTARY, st);
    rotary_kernel<T, VP, IL, PT>
        <<<unsigned(blocks), kRotThreads, size_t(tokens) * size_t(a.P) * sizeof(float2), st>>>(a, pl);
    return check_launch("rotary");
}

template <typename T, int VP, bool IL>
int by_position(const RotaryArgs& a, cudaStream_t st) {
    switch (a.pos_dtype) {
        case DOT_F32: return launch<T, VP, IL, float>(a, st);
        case DOT_I32: return launch<T, VP, IL, int32_t>(a, st);
        default: return launch<T, VP, IL, long long>(a, st);
    }
}

// Whether vectors of `vp` elements of `esz` bytes are aligned in every tensor.
bool fits(const RotaryArgs& a, int vp, int esz) {
    const int64_t bytes = int64_t(vp) * esz;
    if (a.P % vp != 0 || a.D % vp != 0) return false;
    auto ok = [&](const void* in, const void* out, const int64_t* s, int64_t H) {
        if (H == 0) return true;
        if (reinterpret_cast<uintptr_t>(in) % bytes || reinterpret_cast<uintptr_t>(out) % bytes) return false;
        return s[0] % vp == 0 && s[1] % vp == 0 && s[2] % vp == 0;
    };
    return ok(a.q, a.q_out, a.qs, a.Hq) && ok(a.k, a.k_out, a.ks, a.Hk);
}

template <typename T, bool IL>
int by_width(const RotaryArgs& a, cudaStream_t st) {
    if constexpr (sizeof(T) == 2)
        if (fits(a, 8, 2)) return by_position<T, 8, IL>(a, st);
    if (fits(a, 4, sizeof(T))) return by_position<T, 4, IL>(a, st);
    if (fits(a, 2, sizeof(T))) return by_position<T, 2, IL>(a, st);
    return by_position<T, 1, IL>(a, st);
}

template <typename T>
int by_layout(const RotaryArgs& a, cudaStream_t st) {
    return a.interleaved ? by_width<T, true>(a, st) : by_width<T, false>(a, st);
}

}  // namespace

int rotary(const RotaryArgs& a, cudaStream_t st) {
    switch (a.dtype) {
        case DOT_F32: return by_layout<float>(a, st);
        case DOT_BF16: return by_layout<__nv_bfloat16>(a, st);
        default: return by_layout<__half>(a, st);
    }
}

}  // namespace dotb
