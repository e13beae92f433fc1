// Group norm kernels for __nv_bfloat16 elements (group_norm.cuh).
#include "group_norm.cuh"

namespace dotb {

int gn_bf16(const GroupNormArgs& a, void* ws, bool backward, cudaStream_t st) {
    return by_width<__nv_bfloat16>(a, ws, backward, st);
}

}  // namespace dotb
