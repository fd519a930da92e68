// The 8-bit K/V cache's quantizer, shared by the kernels that write rows.
#pragma once
#include "tf_common.hpp"

// Four values a lane, eight lanes a 32-value group (aligned): the lane's four int8 and,
// in every lane, the group's scale; as tf_quantize_q8.
__device__ __forceinline__ uint32_t tf_q8_quad(const float* x, float& d) {
    float amax = fmaxf(fmaxf(fabsf(x[0]), fabsf(x[1])), fmaxf(fabsf(x[2]), fabsf(x[3])));
    amax = fmaxf(amax, tf_dpp<TF_DPP_QUAD_1032>(amax));
    amax = fmaxf(amax, tf_dpp<TF_DPP_QUAD_2301>(amax));
    amax = fmaxf(amax, tf_dpp<TF_DPP_ROW_HALF_MIRROR>(amax));
    d = amax * (1.0f / 127.0f);
    const float r = __builtin_amdgcn_rcpf(d);
    uint32_t b = 0;
#pragma unroll
    for (int i = 0; i < 4; i++)
        b |= (uint32_t)(uint8_t)(int8_t)tf_q8_value_r(x[i], amax, d, r) << (8 * i);
    return b;
}
