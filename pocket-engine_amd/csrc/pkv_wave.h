// Reductions and prefix sums over a wave's 64 lanes by row moves and lane swaps.
#pragma once
#include "pkv_common.h"

namespace pkv {

// Reductions and the inclusive prefix sum over the wave's lanes by row moves.
template <class Op>
__device__ __forceinline__ int wave_all(int v, Op op) {
    v = op(v, __builtin_amdgcn_update_dpp(0, v, DPP_QUAD_XOR1, 0xf, 0xf, false));
    v = op(v, __builtin_amdgcn_update_dpp(0, v, DPP_QUAD_XOR2, 0xf, 0xf, false));
    v = op(v, __builtin_amdgcn_update_dpp(0, v, DPP_ROW_HALF_MIRROR, 0xf, 0xf, false));
    v = op(v, __builtin_amdgcn_update_dpp(0, v, DPP_ROW_MIRROR, 0xf, 0xf, false));
    auto r = __builtin_amdgcn_permlane16_swap((unsigned)v, (unsigned)v, true, false);
    v = op((int)r[0], (int)r[1]);
    r = __builtin_amdgcn_permlane32_swap((unsigned)v, (unsigned)v, true, false);
    return __builtin_amdgcn_readfirstlane(op((int)r[0], (int)r[1]));
}
__device__ __forceinline__ int wave_sum(int v) {
    return wave_all(v, [](int a, int b) { return a + b; });
}
__device__ __forceinline__ int wave_max(int v) {
    return wave_all(v, [](int a, int b) { return a > b ? a : b; });
}
// (op has 0 as its neutral value: lanes without a partner get 0)
template <class Op>
__device__ __forceinline__ int wave_prefix(int v, Op op) {
    v = op(v, __builtin_amdgcn_update_dpp(0, v, 0x111 /* row_shr:1 */, 0xf, 0xf, false));
    v = op(v, __builtin_amdgcn_update_dpp(0, v, 0x112 /* row_shr:2 */, 0xf, 0xf, false));
    v = op(v, __builtin_amdgcn_update_dpp(0, v, 0x114 /* row_shr:4 */, 0xf, 0xf, false));
    v = op(v, __builtin_amdgcn_update_dpp(0, v, 0x118 /* row_shr:8 */, 0xf, 0xf, false));
    v = op(v, __builtin_amdgcn_update_dpp(0, v, 0x142 /* row_bcast:15 */, 0xa, 0xf, false));
    return op(v, __builtin_amdgcn_update_dpp(0, v, 0x143 /* row_bcast:31 */, 0xc, 0xf, false));
}
__device__ __forceinline__ int wave_prefix(int v) {
    return wave_prefix(v, [](int a, int b) { return a + b; });
}

}  // namespace pkv
