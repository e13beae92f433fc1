// Group norm kernels for __half elements (group_norm.cuh).
#include "group_norm.cuh"

namespace dotb {

int gn_f16(const GroupNormArgs& a, void* ws, bool backward, cudaStream_t st) {
    return by_width<__half>(a, ws, backward, st);
}

}  // namespace dotb
