// extern "C" boundary of the feature operators (declared in
// include/dot_b200.h): argument checks, then the launchers of feature_ops.h.
#include <cmath>
#include <string>

#include "feature_ops.h"
#include "internal.h"

using namespace dotb;

namespace {

bool float_dtype(int d) { return d == DOT_F32 || d == DOT_BF16 || d == DOT_F16; }

// Whether every address (NULL among them) is a multiple of `bytes`: the kernels read
// pairs and single elements whatever the vectors' width.
template <typename... Ps>
bool aligned(size_t bytes, Ps... p) {
    return ((reinterpret_cast<uintptr_t>(p) % bytes == 0) && ...);
}
size_t size_of(int dtype) { return dtype == DOT_I64 ? 8 : dtype == DOT_F32 || dtype == DOT_I32 ? 4 : 2; }

int check_norm_addresses(const GroupNormArgs& a, const void* ws) {
    if (!aligned(8, a.stats, ws)) return fail(DOT_ERR_INVALID, "stats and workspace must be 8-byte aligned");
    if (!aligned(size_of(a.dtype), a.x, a.dy, a.y, a.dx) || !aligned(4, a.lengths) ||
        !aligned(size_of(a.param_dtype), a.weight, a.bias, a.dweight, a.dbias))
        return fail(DOT_ERR_INVALID, "tensor address not aligned to its elements");
    return DOT_OK;
}

// Sizes, group count and types common to the forward and the backward.
int check_norm(int dtype, int param_dtype, int64_t N, int64_t S, int64_t C, int64_t G, int activation) {
    if (N < 0 || S < 0 || C < 0) return fail(DOT_ERR_INVALID, "negative dimension");
    if (G < 1 || C % G != 0) return fail(DOT_ERR_INVALID, "num_groups must be >= 1 and divide the channels");
    if (!float_dtype(dtype) || !float_dtype(param_dtype))
        return fail(DOT_ERR_UNSUPPORTED, "dtype must be float32, bfloat16 or float16");
    if (activation < DOT_ACT_NONE || activation > DOT_ACT_RELU) return fail(DOT_ERR_INVALID, "unknown activation");
    // positions and channels are 32-bit indices in the kernels (a thread's walk ends up
    // to a block's rows past S), addresses 64-bit
    if (S > 0x7fff0000 || C > 0x7fffff || N > 0x7fffff) return fail(DOT_ERR_UNSUPPORTED, "dimension too large");
    return DOT_OK;
}

}  // namespace

extern "C" {

size_t dot_group_norm_fwd_workspace_bytes(int64_t N, int64_t S, int64_t C, int64_t G) {
    if (N <= 0 || S <= 0 || C <= 0 || G <= 0) return 0;
    return gn_fwd_ws(N, S, C, G);
}

size_t dot_group_norm_bwd_workspace_bytes(int64_t N, int64_t S, int64_t C, int64_t G) {
    if (N <= 0 || S <= 0 || C <= 0 || G <= 0) return 0;
    return gn_bwd_ws(N, S, C, G);
}

int dot_group_norm_fwd(const void* x, int dtype, int64_t x_batch_stride, int64_t x_pos_stride, const void* weight,
                       const void* bias, int param_dtype, const int32_t* lengths, int64_t N, int64_t S, int64_t C,
                       int64_t G, float eps, int activation, void* y, float* stats, void* workspace,
                       size_t workspace_bytes, void* stream) {
    clear_error();
    const int rc = check_norm(dtype, param_dtype, N, S, C, G, activation);
    if (rc) return rc;
    if (!std::isfinite(eps) || !(eps >= 0.0f)) return fail(DOT_ERR_INVALID, "eps must be finite and >= 0");
    if (N == 0 || S == 0 || C == 0) return DOT_OK;
    if (!x || !y || !stats) return fail(DOT_ERR_INVALID, "null tensor pointer");
    const size_t need = gn_fwd_ws(N, S, C, G);
    if (need > 0 && (workspace == nullptr || workspace_bytes < need))
        return fail(DOT_ERR_WORKSPACE, "workspace too small: need " + std::to_string(need) + " bytes");
    GroupNormArgs a{};
    a.x = x;
    a.xb = N > 1 ? x_batch_stride : 0;   // the stride of a single sample or position says nothing
    a.xp = S > 1 ? x_pos_stride : 0;
    a.weight = weight;
    a.bias = bias;
    a.lengths = lengths;
    a.y = y;
    a.stats = stats;
    a.N = N;
    a.S = S;
    a.C = C;
    a.G = G;
    a.dtype = dtype;
    a.param_dtype = param_dtype;
    a.act = activation;
    a.eps = eps;
    const int at = check_norm_addresses(a, workspace);
    if (at) return at;
    return gn_run(a, workspace, false, static_cast<cudaStream_t>(stream));
}

int dot_group_norm_bwd(const void* x, int dtype, int64_t x_batch_stride, int64_t x_pos_stride, const void* dy,
                       int64_t dy_batch_stride, int64_t dy_pos_stride, const void* weight, const void* bias,
                       int param_dtype, const int32_t* lengths, int64_t N, int64_t S, int64_t C, int64_t G,
                       int activation, const float* stats, void* dx, void* dweight, void* dbias, void* workspace,
                       size_t workspace_bytes, void* stream) {
    clear_error();
    const int rc = check_norm(dtype, param_dtype, N, S, C, G, activation);
    if (rc) return rc;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (N == 0 || S == 0 || C == 0) {   // nothing contributes to the parameters' gradients
        const size_t bytes = size_t(C) * (param_dtype == DOT_F32 ? 4 : 2);
        if (dweight && bytes) cudaMemsetAsync(dweight, 0, bytes, st);
        if (dbias && bytes) cudaMemsetAsync(dbias, 0, bytes, st);
        return check_launch("group norm backward");
    }
    if (!x || !dy || !stats) return fail(DOT_ERR_INVALID, "null tensor pointer");
    if (!dx && !dweight && !dbias) return DOT_OK;
    const size_t need = gn_bwd_ws(N, S, C, G);
    if (need > 0 && (workspace == nullptr || workspace_bytes < need))
        return fail(DOT_ERR_WORKSPACE, "workspace too small: need " + std::to_string(need) + " bytes");
    GroupNormArgs a{};
    a.x = x;
    a.xb = N > 1 ? x_batch_stride : 0;   // the stride of a single sample or position says nothing
    a.xp = S > 1 ? x_pos_stride : 0;
    a.dy = dy;
    a.gb = N > 1 ? dy_batch_stride : 0;
    a.gp = S > 1 ? dy_pos_stride : 0;
    a.weight = weight;
    a.bias = bias;
    a.lengths = lengths;
    a.dx = dx;
    a.dweight = dweight;
    a.dbias = dbias;
    a.stats = const_cast<float*>(stats);
    a.N = N;
    a.S = S;
    a.C = C;
    a.G = G;
    a.dtype = dtype;
    a.param_dtype = param_dtype;
    a.act = activation;
    const int at = check_norm_addresses(a, workspace);
    if (at) return at;
    return gn_run(a, workspace, true, st);
}

int dot_rotary(const void* q, const int64_t* q_strides, int64_t Hq, const void* k, const int64_t* k_strides,
               int64_t Hk, int dtype, const void* positions, int pos_dtype, const int64_t* pos_strides,
               const float* freqs, int64_t B, int64_t L, int64_t D, int64_t P, int A, int interleaved, int inverse,
               void* q_out, void* k_out, void* stream) {
    clear_error();
    if (B < 0 || L < 0 || D < 0 || Hq < 0 || Hk < 0 || P < 0) return fail(DOT_ERR_INVALID, "negative dimension");
    if (D > 0x7fffff || 2 * P > D) return fail(DOT_ERR_INVALID, "freqs must hold at most D/2 pairs");
    if (A < 1 || A > kMaxAxes) return fail(DOT_ERR_INVALID, "positions must have 1 to 4 axes");
    if (!float_dtype(dtype)) return fail(DOT_ERR_UNSUPPORTED, "dtype must be float32, bfloat16 or float16");
    if (pos_dtype != DOT_F32 && pos_dtype != DOT_I32 && pos_dtype != DOT_I64)
        return fail(DOT_ERR_UNSUPPORTED, "positions must be int32, int64 or float32");
    if (P > kMaxPairs) return fail(DOT_ERR_UNSUPPORTED, "more than 4096 pairs in a head");
    // a block's tokens are counted past the end of a sample in 31 bits
    if (B > 0x7fffffff || L > 0x7fffff00 || Hq + Hk > 0x7fffff) return fail(DOT_ERR_UNSUPPORTED, "dimension too large");
    if (B == 0 || L == 0 || D == 0 || Hq + Hk == 0) return DOT_OK;
    if ((Hq > 0 && (!q || !q_out || !q_strides)) || (Hk > 0 && (!k || !k_out || !k_strides)) || !positions ||
        !pos_strides || (P > 0 && !freqs))
        return fail(DOT_ERR_INVALID, "null tensor pointer");
    if ((Hq > 0 && !aligned(size_of(dtype), q, q_out)) || (Hk > 0 && !aligned(size_of(dtype), k, k_out)) ||
        !aligned(size_of(pos_dtype), positions) || !aligned(4, freqs))
        return fail(DOT_ERR_INVALID, "tensor address not aligned to its elements");
    RotaryArgs a{};
    a.q = q;
    a.k = k;
    a.q_out = q_out;
    a.k_out = k_out;
    a.positions = positions;
    a.freqs = freqs;
    const int64_t q_sizes[3] = {B, L, Hq}, k_sizes[3] = {B, L, Hk};
    for (int i = 0; i < 3; ++i) {   // the stride of a single entry says nothing
        a.qs[i] = q_sizes[i] > 1 && Hq > 0 ? q_strides[i] : 0;
        a.ks[i] = k_sizes[i] > 1 && Hk > 0 ? k_strides[i] : 0;
        a.ps[i] = pos_strides[i];
    }
    a.B = B;
    a.L = L;
    a.D = D;
    a.P = P;
    a.Hq = Hq;
    a.Hk = Hk;
    a.A = A;
    a.dtype = dtype;
    a.pos_dtype = pos_dtype;
    a.interleaved = interleaved != 0;
    a.inverse = inverse != 0;
    return rotary(a, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
