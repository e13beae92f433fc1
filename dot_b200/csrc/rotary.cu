// Rotary positions with several axes (dot_rotary in include/dot_b200.h).
//
//   angle[t, p] = sum_a positions[t, a] * freqs[p, a]
//   (x, y) -> (x cos - y sin, y cos + x sin)   for pair p of every head of token t
//
// The backward is the same kernel with the sine negated: the turn is
// orthogonal.  Bound: memory (each element is read and written once, with
// about five operations); a token's P sines and cosines serve all its heads.
//
// A block takes a few whole tokens.  Each thread owns one vector of VP pairs of
// a token over a run of heads and issues its first loads; while they are on
// their way the block forms the tokens' sines and cosines, once, in shared
// memory; then the thread keeps its own in registers and turns its heads.
#include "feature.cuh"
#include "feature_ops.h"
#include "internal.h"

namespace dotb {
namespace {

constexpr int kRotThreads = 128;
constexpr int kRotRun = 4;      // consecutive heads of a thread in a large call

// Heads that a thread loads together, and blocks per SM.  Small blocks, so that
// one block's angles overlap another's copies.  Measured on 98 MB of bfloat16
// and 32 MB of float32 (both read and written): 4 heads and 5 blocks 35.9 and
// 15.3 us, 2 and 8 38.2 and 13.9, 4 and 4 38.3 and 15.4; blocks of 256 threads
// 40.1 and 16.2.
template <typename T>
constexpr int rot_heads() { return sizeof(T) == 2 ? 4 : 2; }
template <typename T>
constexpr int rot_blocks() { return sizeof(T) == 2 ? 5 : 8; }

struct RotPlan {
    int slots;          // threads per head: P / VP pair vectors, then the copied tail's vectors (two per slot)
    int pair_slots;
    int run;            // consecutive heads of a thread
    int q_runs, runs;   // runs of q, and of q and k, that a token is split into
    int tokens;         // tokens per block
    int64_t ntok;       // B * L
    FastDiv by_slots, by_token, by_pairs, by_axes, by_len;   // slots, slots * runs, P, A, L
};

template <typename I>
__device__ __forceinline__ double position(const void* p, int64_t i) {
    return double(static_cast<const I*>(p)[i]);
}

// Cosine and sine of an angle given in turns, in fp64: reduced to [-1/2, 1/2]
// before it is rounded to fp32, so a position of 2^30 keeps an absolute error
// below 2^-20 turns where an fp32 angle has lost it.  16-bit results take the
// SFU's sine and cosine (absolute error 2^-21 within half a turn, a thousandth
// of their rounding), float32 the accurate ones.
template <typename T>
__device__ __forceinline__ float2 cos_sin(double turns) {
    const float r = float(turns - rint(turns));
    float s, c;
    if constexpr (sizeof(T) == 2) {
        const float x = r * 6.2831853f;
        s = __sinf(x);
        c = __cosf(x);
    } else {
        sincospif(2.0f * r, &s, &c);
    }
    return make_float2(c, s);
}

// A vector of VP pairs of one head, turned: (x, y) -> (x c - y s, y c + x s).
// The roundings are the same at every width: a product, then an fma.
template <typename T, int VP, bool IL>
struct Turn {
    static constexpr int NP = pairs_of(VP);
    float2 c[IL ? VP : NP], s[IL ? VP : NP], ns[IL ? 1 : NP];
    __device__ __forceinline__ void load(const float2* cs) {
        if constexpr (IL) {
#pragma unroll
            for (int j = 0; j < VP; ++j) {
                c[j] = splat2(cs[j].x);
                s[j] = make_float2(-cs[j].y, cs[j].y);
            }
        } else {
#pragma unroll
            for (int j = 0; j < NP; ++j) {
                const float2 u = cs[2 * j], v = VP == 1 ? u : cs[2 * j + 1];
                c[j] = make_float2(u.x, v.x);
                s[j] = make_float2(u.y, v.y);
                ns[j] = make_float2(-u.y, -v.y);
            }
        }
    }
    // p0, p1: the pairs' first and second elements, or with IL the 2 VP elements in order
    __device__ __forceinline__ void operator()(Pack<T, VP>& p0, Pack<T, VP>& p1) const {
        if constexpr (IL && VP == 1) {
            const float2 e = make_float2(to_f32(p0.v[0]), to_f32(p1.v[0]));
            const float2 r = fma2(e, c[0], mul2(make_float2(e.y, e.x), s[0]));
            p0.v[0] = from_f32<T>(r.x);
            p1.v[0] = from_f32<T>(r.y);
        } else {
            float2 x[NP], y[NP];
            unpack(p0, x);
            unpack(p1, y);
#pragma unroll
            for (int j = 0; j < NP; ++j) {
                if constexpr (IL) {
                    x[j] = fma2(x[j], c[j], mul2(make_float2(x[j].y, x[j].x), s[j]));
                    y[j] = fma2(y[j], c[NP + j], mul2(make_float2(y[j].y, y[j].x), s[NP + j]));
                } else {
                    const float2 u = fma2(x[j], c[j], mul2(y[j], ns[j]));
                    y[j] = fma2(y[j], c[j], mul2(x[j], s[j]));
                    x[j] = u;
                }
            }
            p0 = pack<T, VP>(x);
            p1 = pack<T, VP>(y);
        }
    }
};

template <typename T, int VP, bool IL, typename PT>
__global__ void __launch_bounds__(kRotThreads, rot_blocks<T>()) rotary_kernel(RotaryArgs a, RotPlan pl) {
    extern __shared__ double rot_smem[];
    const int P = int(a.P), A = a.A;
    double* pos = rot_smem;                                            // [tokens][A] positions in turns
    float2* cs = reinterpret_cast<float2*>(pos + pl.tokens * A);       // [tokens][P] cos, sin
    const int64_t t0 = int64_t(blockIdx.x) * pl.tokens;
    const int nt = int(min(int64_t(pl.tokens), pl.ntok - t0));
    const int64_t b0 = pl.ntok <= 0x7fffffff ? int64_t(pl.by_len.div(int(t0))) : t0 / a.L;
    const int l0 = int(t0 - b0 * a.L);   // and at most 128 tokens on: below 2^31

    // A thread's work: token tl, `heads` consecutive heads of q or of k, and the
    // offsets o0, o1 of its two vectors within a head.
    constexpr int U = rot_heads<T>();
    const int work = nt * pl.slots * pl.runs;
    int tl, slot, heads;
    int64_t o1, stride;        // o1 counted from o0
    bool turn, second;
    const T* src;
    T* dst;
    auto place = [&](int i) {
        tl = pl.by_token.div(i);
        const int w = i - tl * (pl.slots * pl.runs);
        const int run = pl.by_slots.div(w);
        slot = w - run * pl.slots;
        turn = slot < pl.pair_slots;
        const int o0 = turn ? (IL ? slot * 2 * VP : slot * VP) : 2 * P + (slot - pl.pair_slots) * 2 * VP;
        o1 = turn && !IL ? P : VP;
        second = turn || o0 + VP < int(a.D);
        const int db = pl.by_len.div(l0 + tl);
        const int64_t b = b0 + db, l = l0 + tl - db * int(a.L), t = t0 + tl;
        const bool is_q = run < pl.q_runs;
        const int h0 = (is_q ? run : run - pl.q_runs) * pl.run;
        const int64_t H = is_q ? a.Hq : a.Hk;
        heads = min(pl.run, int(H) - h0);
        stride = is_q ? a.qs[2] : a.ks[2];
        src = is_q ? static_cast<const T*>(a.q) + b * a.qs[0] + l * a.qs[1]
                   : static_cast<const T*>(a.k) + b * a.ks[0] + l * a.ks[1];
        src += h0 * stride + o0;
        dst = static_cast<T*>(is_q ? a.q_out : a.k_out) + (t * H + h0) * a.D + o0;
    };
    Pack<T, VP> p0[U], p1[U];
    auto fetch = [&]() {
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (u < heads) {
                p0[u] = load_pack<T, VP>(src + u * stride);
                if (second) p1[u] = load_pack<T, VP>(src + u * stride + o1);
            }
    };
    int i = threadIdx.x;
    if (i < work) {
        place(i);
        fetch();   // on their way while the angles are formed
    }

    for (int j = threadIdx.x; j < nt * A; j += kRotThreads) {
        const int tk = pl.by_axes.div(j), ax = j - tk * A;
        const int db = pl.by_len.div(l0 + tk), l = l0 + tk - db * int(a.L);
        pos[j] = position<PT>(a.positions, (b0 + db) * a.ps[0] + l * a.ps[1] + ax * a.ps[2]) *
                 0.15915494309189533577;   // 1 / (2 pi)
    }
    __syncthreads();
    for (int j = threadIdx.x; j < nt * P; j += kRotThreads) {
        const int tk = pl.by_pairs.div(j), p = j - tk * P;
        double turns = 0.0;
        for (int ax = 0; ax < A; ++ax) turns = fma(pos[tk * A + ax], double(a.freqs[p * A + ax]), turns);
        const float2 v = cos_sin<T>(turns);
        cs[j] = make_float2(v.x, a.inverse ? -v.y : v.y);
    }
    __syncthreads();

    for (; i < work; i += kRotThreads) {
        if (i >= kRotThreads) {
            place(i);
            fetch();
        }
        Turn<T, VP, IL> tn;
        if (turn) tn.load(cs + tl * P + slot * VP);
        for (;;) {
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (u < heads) {
                    if (turn) tn(p0[u], p1[u]);
                    store_pack<T, VP>(dst + u * a.D, p0[u]);
                    if (second) store_pack<T, VP>(dst + u * a.D + o1, p1[u]);
                }
            heads -= U;
            if (heads <= 0) break;
            src += U * stride;
            dst += U * a.D;
            fetch();
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
    // A head a thread for a few tokens (one access each, so a small call is one
    // round trip), runs of heads where those alone fill the GPU.
    pl.run = pl.ntok * pl.slots * H <= int64_t(148) * 2048 ? 1 : kRotRun;
    pl.q_runs = int(ceil_div(a.Hq, pl.run));
    pl.runs = pl.q_runs + int(ceil_div(a.Hk, pl.run));
    const int64_t per_token = int64_t(pl.slots) * pl.runs;
    if (per_token > 0x3fffffff) return fail(DOT_ERR_UNSUPPORTED, "too many heads in a token");
    int64_t tokens = per_token >= kRotThreads ? 1 : kRotThreads / per_token;
    const int64_t fit = a.P > 0 ? kMaxPairs / a.P : tokens;
    if (tokens > fit) tokens = fit;
    pl.tokens = int(tokens);
    pl.by_slots = FastDiv(uint32_t(pl.slots));
    pl.by_token = FastDiv(uint32_t(per_token));
    pl.by_pairs = FastDiv(uint32_t(a.P > 0 ? a.P : 1));
    pl.by_axes = FastDiv(uint32_t(a.A));
    pl.by_len = FastDiv(uint32_t(a.L));
    const int64_t blocks = ceil_div(pl.ntok, tokens);
    if (blocks > 0x7fffffff) return fail(DOT_ERR_UNSUPPORTED, "too many tokens");
    ProfScope ps(DOT_K_ROTARY, st);
    rotary_kernel<T, VP, IL, PT>
        <<<unsigned(blocks), kRotThreads, size_t(tokens) * size_t(a.P + a.A) * 8, st>>>(a, pl);
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
