// Kernel launchers of the feature operators, called by their C-ABI boundary
// (capi_features.cu) after it has checked the arguments.
#pragma once

#include <cstddef>
#include <cstdint>
#include <cuda_runtime.h>

namespace dotb {

struct GroupNormArgs {
    const void* x;
    const void* dy;        // backward
    const void* weight;
    const void* bias;
    const int32_t* lengths;
    void* y;               // forward
    void* dx;              // backward
    void* dweight;         // backward
    void* dbias;           // backward
    float* stats;          // [N,G,2] mean, rstd: written by the forward, read by the backward
    int64_t xb, xp;        // x: elements between samples / positions
    int64_t gb, gp;        // dy
    int64_t N, S, C, G;
    int dtype, param_dtype, act;
    float eps;
};

size_t gn_fwd_ws(int64_t N, int64_t S, int64_t C, int64_t G);
size_t gn_bwd_ws(int64_t N, int64_t S, int64_t C, int64_t G);
int gn_run(const GroupNormArgs& a, void* ws, bool backward, cudaStream_t st);
// one unit per element type
int gn_f32(const GroupNormArgs& a, void* ws, bool backward, cudaStream_t st);
int gn_bf16(const GroupNormArgs& a, void* ws, bool backward, cudaStream_t st);
int gn_f16(const GroupNormArgs& a, void* ws, bool backward, cudaStream_t st);

constexpr int kMaxAxes = 4;

struct RotaryArgs {
    const void* q;
    const void* k;
    void* q_out;
    void* k_out;
    const void* positions;
    const float* freqs;    // [P, A]
    int64_t qs[3], ks[3];  // elements between samples, tokens, heads
    int64_t ps[3];         // positions: elements between samples, tokens, axes
    int64_t B, L, D, P;
    int64_t Hq, Hk;
    int A, dtype, pos_dtype, interleaved, inverse;
};

// Largest P whose angles a block holds in shared memory.
constexpr int64_t kMaxPairs = 4096;

int rotary(const RotaryArgs& a, cudaStream_t st);

}  // namespace dotb
