// The 8-bit K/V cache's quantizer, shared by the kernels that write rows, and the
// decode step's append.
#pragma once
#include "tf_common.hpp"

// tf_rope_neox of q and k (the reference's f32 angle, which prompts have too, so that one
// cache has one rotation) with k and v appended to the 8-bit cache, for one token.
// head_dim 64, 128 or 256; 16-byte aligned.
int tf_rope_append_kv8(float* q, const float* k, const float* v, int8_t* k8, float* kd, int8_t* v8,
                       float* vd, int n_head, int n_kv, int head_dim, int pos, const int* pos_dev,
                       float theta, tf_stream_t stream);

// N values of a 32-value group with the largest magnitude amax: their int8, four a word,
// and the group's scale; as tf_quantize_q8.
//
// x * rcp(d) is within 2^-15 of x / d, so only a quotient within 2^-14 of halfway
// between integers (one in 10^4), or a scale below f32's normal range, needs the
// division; one test serves all N (a test and branch a value cost a quarter of the time
// of quantizing 32768 f16 rows).
template <int N>
__device__ __forceinline__ float tf_q8_words(const float (&x)[N], float amax, uint32_t (&out)[N / 4]) {
    const float d = amax * (1.0f / 127.0f), r = __builtin_amdgcn_rcpf(d);
    float q[N];
    bool near = !(d >= 1.17549435e-38f);
#pragma unroll
    for (int i = 0; i < N; i++) {
        const float y = x[i] * r;
        q[i] = __builtin_rintf(y);
        near |= fabsf(y - q[i]) > 0.5f - 6.103515625e-05f;
    }
    if (near)
#pragma unroll
        for (int i = 0; i < N; i++) q[i] = (float)tf_q8_value_r(x[i], amax, d, r);
#pragma unroll
    for (int w = 0; w < N / 4; w++) {
        out[w] = 0;
#pragma unroll
        for (int i = 0; i < 4; i++) out[w] |= ((uint32_t)(int)q[4 * w + i] & 255u) << (8 * i);
    }
    return d;
}

// Four values a lane, eight lanes a group (aligned): the lane's four int8 and, in every
// lane, the group's scale.
__device__ __forceinline__ uint32_t tf_q8_quad(const float (&x)[4], float& d) {
    float amax = fmaxf(fmaxf(fabsf(x[0]), fabsf(x[1])), fmaxf(fabsf(x[2]), fabsf(x[3])));
    amax = fmaxf(amax, tf_dpp<TF_DPP_QUAD_1032>(amax));
    amax = fmaxf(amax, tf_dpp<TF_DPP_QUAD_2301>(amax));
    amax = fmaxf(amax, tf_dpp<TF_DPP_ROW_HALF_MIRROR>(amax));
    uint32_t b[1];
    d = tf_q8_words(x, amax, b);
    return b[0];
}
