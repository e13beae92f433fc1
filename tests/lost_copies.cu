// The fused group norm kernels with one stage's copies left out, for the test of
// expired waits: the wait for that stage runs into its limit.  Compiled by
// test_norm_lost_copies_gpu.py; test_norm_partition_gpu.py uses launch() from it.
__device__ int lost_stage = -1;   // a stage of every block's ring
__device__ int lost_back = 0;     // its copy on the way back, not the one on the way in
#define DOTB_RING_LOSES(i, c) ((i) == lost_stage && ((c) > (i) / kRingStages) == (lost_back != 0))

#include "../dot_b200/csrc/group_norm.cuh"

namespace dotb {
int fail(int code, const std::string&) { return code; }
int check_launch(const char*) { return cudaGetLastError() == cudaSuccess ? DOT_OK : DOT_ERR_CUDA; }
void prof_pre(int, cudaStream_t, int) {}
void prof_post(int, cudaStream_t) {}
}  // namespace dotb

// x, dy, y, dx [N,S,C] float16 (dense), weight and bias float32, silu.  `backward` takes stats,
// else it writes them.  stage < 0 leaves nothing out.
extern "C" DOT_API int norm_losing(int stage, int back, int backward, const void* x, const void* dy, const void* weight,
                                   const void* bias, void* y, void* dx, void* dweight, void* dbias, float* stats,
                                   void* ws, int64_t N, int64_t S, int64_t C, int64_t G) {
    using namespace dotb;
    if (cudaMemcpyToSymbol(lost_stage, &stage, sizeof(int)) != cudaSuccess) return -100;
    if (cudaMemcpyToSymbol(lost_back, &back, sizeof(int)) != cudaSuccess) return -100;
    GnPlan pl{};
    GroupNormArgs& a = pl.a;
    a.x = x;
    a.dy = dy;
    a.weight = weight;
    a.bias = bias;
    a.y = y;
    a.dx = dx;
    a.dweight = dweight;
    a.dbias = dbias;
    a.stats = stats;
    a.xb = a.gb = S * C;
    a.xp = a.gp = C;
    a.N = N;
    a.S = S;
    a.C = C;
    a.G = G;
    a.dtype = DOT_F16;
    a.param_dtype = DOT_F32;
    a.act = DOT_ACT_SILU;
    a.eps = 1e-5f;
    int rc = DOT_OK;
    const bool taken = (C / G) % 8 == 0 ? fused_run<__half, 8, kActSilu, true>(pl, ws, backward != 0, nullptr, rc)
                                        : fused_run<__half, 8, kActSilu, false>(pl, ws, backward != 0, nullptr, rc);
    if (!taken) return -101;
    if (rc != DOT_OK) return rc;
    return cudaDeviceSynchronize() == cudaSuccess ? DOT_OK : -102;
}
// The fused forward as a cooperative launch of `blocks` blocks of [blocks, 1, C] float16: what
// launch() answers, with 1000 added if it leaves an error behind.
extern "C" DOT_API int launch_together(int blocks, const void* x, void* y, float* stats, void* ws, int64_t C,
                                       int64_t G) {
    using namespace dotb;
    GnPlan pl{};
    pl.a.x = x;
    pl.a.y = y;
    pl.a.stats = stats;
    pl.a.xb = pl.a.xp = C;
    pl.a.N = blocks;
    pl.a.S = 1;
    pl.a.C = C;
    pl.a.G = G;
    pl.a.dtype = DOT_F16;
    pl.a.act = DOT_ACT_SILU;
    pl.a.eps = 1e-5f;
    pl.chunks = pl.rows = 1;
    carve(ws, pl, false);
    const size_t groups = size_t(G + 1) * (sizeof(float2) + sizeof(float));
    const size_t smem = Ring<1>::bytes() + groups + kGnThreads * sizeof(float2);
    const int rc = launch(gn_fused_fwd_kernel<__half, 8, kActSilu, true>, pl, blocks, kGnThreads, smem, kSmemMerges, 1,
                          kCooperative, nullptr);
    return cudaDeviceSynchronize() == cudaSuccess && cudaGetLastError() == cudaSuccess ? rc : 1000 + rc;
}
extern "C" DOT_API size_t norm_workspace(int64_t N, int64_t S, int64_t C, int64_t G) {
    const size_t f = dotb::workspace_bytes(N, S, C, G, false), b = dotb::workspace_bytes(N, S, C, G, true);
    return f > b ? f : b;
}
