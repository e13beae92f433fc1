// Group norm kernels for float elements (group_norm.cuh).
#include "group_norm.cuh"

namespace dotb {

int gn_f32(const GroupNormArgs& a, void* ws, bool backward, cudaStream_t st) {
    return by_width<float>(a, ws, backward, st);
}

// float32's unit also holds what does not depend on the type.
size_t gn_fwd_ws(int64_t N, int64_t S, int64_t C, int64_t G) { return workspace_bytes(N, S, C, G, false); }
size_t gn_bwd_ws(int64_t N, int64_t S, int64_t C, int64_t G) { return workspace_bytes(N, S, C, G, true); }

int gn_run(const GroupNormArgs& a, void* ws, bool backward, cudaStream_t st) {
    switch (a.dtype) {
        case DOT_F32: return gn_f32(a, ws, backward, st);
        case DOT_BF16: return gn_bf16(a, ws, backward, st);
        default: return gn_f16(a, ws, backward, st);
    }
}

}  // namespace dotb
