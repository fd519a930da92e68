// Per-head RMS norms of q and k with the NeoX rotation in the same pass; the
// rows go to f32 rows, or K and V are appended to the f16 or the 8-bit cache
// as they are formed.
//
//   y = x * (1 / sqrt(mean(x^2) + eps)) * w        over the head_dim values
//   (y_i, y_{i + h/2}) turned by pos * theta^(-2i / head_dim)
//
// The angle is formed in 64 bits, in turns: a position of 10^6 times a
// frequency of 1 leaves f32 no bits below 2^-4 rad, while the reference's f32
// angle (tf_rope_neox) is what the model files were not trained with.  Its
// fraction of a turn is exact to 2^-32 there, and sine and cosine of that
// fraction are f32.
#include "kv8.hpp"
#include "tf_common.hpp"
#include "tf_host.hpp"

#define TF_QK_MAX_HEAD_DIM 256

namespace {

enum Dest { kRows, kF16, kKv8 };

struct QkArgs {
    const float *q, *k, *v;
    long long q_stride, k_stride, v_stride;
    const float *q_norm, *k_norm;
    float eps;
    float *q_out, *k_out;
    uint16_t *kc, *vc;
    int8_t *k8, *v8;
    float *kd, *vd;
    int n_head, n_kv, head_dim;
    int pos0;
    const int* pos0_dev;
    double log2_theta;
    float theta;
};

// Turns of pair i at position pos, less their whole part.
__device__ __forceinline__ float turns(long long pos, int i, int head_dim, double log2_theta) {
    constexpr double kInv2Pi = 0.15915494309189533577;
    const double f = exp2(-2.0 * i / head_dim * log2_theta) * kInv2Pi;
    const double a = (double)pos * f;
    return (float)(a - rint(a));
}

// head_dim 64, 128 and 256 on 16-byte aligned rows: a lane holds four values of a
// head's first half and the four that they turn with, HD / 8 lanes a head, so every
// access is 16 bytes a lane and the sum of squares a few DPP steps.  A workgroup takes
// TOK tokens; their angles' sines and cosines, the same for all heads, are formed once,
// a thread a pair, into LDS.  One token a workgroup (of few tokens, `share` heads of
// one), four where they fill the CUs.
// Bound by its bytes: 4096 tokens of 28 + 8 heads of 128 into the 8-bit cache move 139
// MB in 31.2 us (4.5 TB/s); 777 tokens of 16 + 2 heads of 128 to f32 rows 8.8 us (heads in
// passes of 16 a token, so the second has 2); one token of 14 + 2 heads of 64 3.8, where a
// row that is stored without angles takes 1.7: f64 exponentials, sines and a barrier.
// F32: the angle as tf_rope_neox and the prompts' kernels form it.
template <int HD, Dest D, int TOK, bool F32 = false>
__global__ __launch_bounds__(256) void tf_qk_norm_rope_vec_kernel(QkArgs a, int n_tok, int share) {
    constexpr int HALF = HD / 2, LPH = HD / 8, HEADS = 256 / LPH;
    __shared__ __align__(16) float cs[2][TOK][HALF];
    const int tid = threadIdx.x;
    const int tok0 = blockIdx.x * TOK;
    const int pos0 = a.pos0_dev ? a.pos0_dev[0] : a.pos0;
    const int heads = a.n_head + (D == kRows ? 1 : 2) * a.n_kv;
    const int item0 = TOK == 1 ? (int)blockIdx.y * share : 0;
    const int items = TOK == 1 ? min(heads, item0 + share) : heads * min(TOK, n_tok - tok0);
    const int m = tid % LPH;
    // the lane's eight values of an item (a head of a token)
    auto where = [&](int item, int& t, int& h, int& kind) {
        t = TOK == 1 ? 0 : item / heads;
        h = TOK == 1 ? item : item - t * heads;
        kind = h < a.n_head ? 0 : h < a.n_head + a.n_kv ? 1 : 2;  // q, k, v
        h -= kind == 0 ? 0 : kind == 1 ? a.n_head : a.n_head + a.n_kv;
        t += tok0;
    };
    auto row = [&](int t, int h, int kind) {
        const float* x = kind == 0   ? a.q + t * a.q_stride
                         : kind == 1 ? a.k + t * a.k_stride
                                     : a.v + t * a.v_stride;
        return x + (size_t)h * HD + 4 * m;
    };
    int item = item0 + tid / LPH, t = 0, h = 0, kind = 2;
    float4 x0 = make_float4(0.f, 0.f, 0.f, 0.f), x1 = x0;
    if (item < items) {  // the first item's loads go out under the angles
        where(item, t, h, kind);
        const float* x = row(t, h, kind);
        x0 = *reinterpret_cast<const float4*>(x);
        x1 = *reinterpret_cast<const float4*>(x + HALF);
    }
    float4 wq[2], wk[2];
    const float4 one = make_float4(1.f, 1.f, 1.f, 1.f);
#pragma unroll
    for (int i = 0; i < 2; i++) {
        wq[i] = a.q_norm ? *reinterpret_cast<const float4*>(a.q_norm + 4 * m + HALF * i) : one;
        wk[i] = a.k_norm ? *reinterpret_cast<const float4*>(a.k_norm + 4 * m + HALF * i) : one;
    }
    for (int i = tid; i < TOK * HALF; i += 256) {
        const int tt = i / HALF, pair = i % HALF;
        float s, c;
        if constexpr (F32) {
            const float freq = powf(a.theta, -2.f * (float)pair / (float)HD);
            sincosf((float)(pos0 + tok0 + tt) * freq, &s, &c);
        } else {
            sincospif(2.f * turns((long long)pos0 + tok0 + tt, pair, HD, a.log2_theta), &s, &c);
        }
        cs[0][tt][pair] = c;
        cs[1][tt][pair] = s;
    }
    __syncthreads();
    for (; item < items; item += HEADS) {
        float v[8] = {x0.x, x0.y, x0.z, x0.w, x1.x, x1.y, x1.z, x1.w};
        const int t_now = t, h_now = h, kind_now = kind;
        if (item + HEADS < items) {  // the next item's loads
            where(item + HEADS, t, h, kind);
            const float* x = row(t, h, kind);
            x0 = *reinterpret_cast<const float4*>(x);
            x1 = *reinterpret_cast<const float4*>(x + HALF);
        }
        if (kind_now != 2) {
            const bool is_q = kind_now == 0;
            if (is_q ? a.q_norm : a.k_norm) {
                float ss = 0.f;
#pragma unroll
                for (int i = 0; i < 8; i++) ss = fmaf(v[i], v[i], ss);
                if (LPH == 8) {
                    ss += tf_dpp<TF_DPP_QUAD_1032>(ss);
                    ss += tf_dpp<TF_DPP_QUAD_2301>(ss);
                    ss += tf_dpp<TF_DPP_ROW_HALF_MIRROR>(ss);
                } else {
                    ss = tf_group_sum<LPH == 8 ? 16 : LPH>(ss);
                }
                const float rs = 1.0f / sqrtf(ss / (float)HD + a.eps);
                const float4 w0 = is_q ? wq[0] : wk[0], w1 = is_q ? wq[1] : wk[1];
                v[0] = v[0] * rs * w0.x, v[1] = v[1] * rs * w0.y;
                v[2] = v[2] * rs * w0.z, v[3] = v[3] * rs * w0.w;
                v[4] = v[4] * rs * w1.x, v[5] = v[5] * rs * w1.y;
                v[6] = v[6] * rs * w1.z, v[7] = v[7] * rs * w1.w;
            }
            const float4 c4 = *reinterpret_cast<const float4*>(&cs[0][t_now - tok0][4 * m]);
            const float4 s4 = *reinterpret_cast<const float4*>(&cs[1][t_now - tok0][4 * m]);
            const float c[4] = {c4.x, c4.y, c4.z, c4.w}, s[4] = {s4.x, s4.y, s4.z, s4.w};
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float y0 = v[i], y1 = v[i + 4];
                v[i] = y0 * c[i] - y1 * s[i];
                v[i + 4] = y0 * s[i] + y1 * c[i];
            }
        }
        if (kind_now == 0 || D == kRows) {
            float* out = kind_now == 0 ? a.q_out + ((size_t)t_now * a.n_head + h_now) * HD
                                       : a.k_out + ((size_t)t_now * a.n_kv + h_now) * HD;
            *reinterpret_cast<float4*>(out + 4 * m) = make_float4(v[0], v[1], v[2], v[3]);
            *reinterpret_cast<float4*>(out + 4 * m + HALF) = make_float4(v[4], v[5], v[6], v[7]);
            continue;
        }
        const long long pos = (long long)pos0 + t_now;
        if (pos < 0) continue;  // no place in the cache
        const size_t at = ((size_t)pos * a.n_kv + h_now) * HD + 4 * m;
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const float y[4] = {v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]};
            const size_t o = at + HALF * i;
            if (D == kF16) {
                uint16_t* dst = (kind_now == 1 ? a.kc : a.vc) + o;
                const tf_u32x2 b = {(uint32_t)tf_f2h_halfup(y[0]) | (uint32_t)tf_f2h_halfup(y[1]) << 16,
                                    (uint32_t)tf_f2h_halfup(y[2]) | (uint32_t)tf_f2h_halfup(y[3]) << 16};
                *reinterpret_cast<tf_u32x2*>(dst) = b;
            } else {  // eight lanes hold a group
                float d;
                const uint32_t b = tf_q8_quad(y, d);
                *reinterpret_cast<uint32_t*>((kind_now == 1 ? a.k8 : a.v8) + o) = b;
                if ((m & 7) == 0) (kind_now == 1 ? a.kd : a.vd)[o >> 5] = d;
            }
        }
    }
}

// What a wave's lanes wrote to LDS is there for each other.
__device__ __forceinline__ void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// Any other even head_dim, any alignment: a head a wave, a workgroup a token and four
// heads.  y: the head in LDS.
template <Dest D>
__global__ __launch_bounds__(256) void tf_qk_norm_rope_kernel(QkArgs a) {
    __shared__ float lds[4][TF_QK_MAX_HEAD_DIM];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    float* y = lds[wave];
    const int heads = a.n_head + (D == kRows ? 1 : 2) * a.n_kv;
    int h = blockIdx.y * 4 + wave;
    if (h >= heads) return;
    const long long t = blockIdx.x;
    const long long pos = (long long)(a.pos0_dev ? a.pos0_dev[0] : a.pos0) + t;
    const int hd = a.head_dim, half = hd / 2;
    const int kind = h < a.n_head ? 0 : h < a.n_head + a.n_kv ? 1 : 2;  // q, k, v
    h -= kind == 0 ? 0 : kind == 1 ? a.n_head : a.n_head + a.n_kv;
    const float* x = kind == 0   ? a.q + t * a.q_stride
                     : kind == 1 ? a.k + t * a.k_stride
                                 : a.v + t * a.v_stride;
    x += (size_t)h * hd;
    const float* w = kind == 0 ? a.q_norm : kind == 1 ? a.k_norm : nullptr;
    float ss = 0.f;
    for (int i = lane; i < hd; i += 64) {
        y[i] = x[i];
        ss = fmaf(y[i], y[i], ss);
    }
    ss = tf_group_sum<64>(ss);
    const float rs = 1.0f / sqrtf(ss / (float)hd + a.eps);
    wave_sync();
    if (kind != 2)
        for (int i = lane; i < half; i += 64) {
            float y0 = y[i], y1 = y[i + half];
            if (w) {
                y0 = y0 * rs * w[i];
                y1 = y1 * rs * w[i + half];
            }
            float s, c;
            sincospif(2.f * turns(pos, i, hd, a.log2_theta), &s, &c);
            y[i] = y0 * c - y1 * s;
            y[i + half] = y0 * s + y1 * c;
        }
    wave_sync();
    if (kind == 0 || D == kRows) {
        float* out = kind == 0 ? a.q_out + ((size_t)t * a.n_head + h) * hd
                               : a.k_out + ((size_t)t * a.n_kv + h) * hd;
        for (int i = lane; i < hd; i += 64) out[i] = y[i];
        return;
    }
    if (pos < 0) return;  // no place in the cache
    const size_t at = ((size_t)pos * a.n_kv + h) * hd;
    if (D == kF16) {
        uint16_t* c = (kind == 1 ? a.kc : a.vc) + at;
        for (int i = lane; i < hd; i += 64) c[i] = tf_f2h_halfup(y[i]);
    } else {
        int8_t* c = (kind == 1 ? a.k8 : a.v8) + at;
        float* d8 = (kind == 1 ? a.kd : a.vd) + at / 32;
        for (int i = lane; i < hd; i += 64) {
            const float amax = tf_group32_max(fabsf(y[i]));
            const float d = amax * (1.0f / 127.0f);
            c[i] = (int8_t)tf_q8_value(y[i], amax, d);
            if ((lane & 31) == 0) d8[i >> 5] = d;
        }
    }
}

template <Dest D>
int launch(const QkArgs& a, int n_tok, float theta, tf_stream_t stream) {
    TF_CHECK_ARG(a.q && a.k && a.q_out && a.n_head > 0 && a.n_kv > 0 && n_tok > 0);
    TF_CHECK_ARG(a.head_dim > 0 && a.head_dim <= TF_QK_MAX_HEAD_DIM && a.head_dim % 2 == 0);
    TF_CHECK_ARG(theta > 0.f && theta < INFINITY && a.eps >= 0.f);
    TF_CHECK_ARG(a.pos0_dev || (a.pos0 >= 0 && a.pos0 <= INT32_MAX - n_tok));
    const long long qw = (long long)a.n_head * a.head_dim, kw = (long long)a.n_kv * a.head_dim;
    TF_CHECK_ARG(a.q_stride >= qw && a.k_stride >= kw && qw + 2 * kw <= INT32_MAX);
    TF_CHECK_ARG(a.q != a.q_out || a.q_stride == qw);
    TF_CHECK_ARG(n_tok <= (int)(UINT32_MAX / 256) && a.n_head + 2LL * a.n_kv <= 65535);
    QkArgs b = a;
    b.log2_theta = log2((double)theta);
    const int heads = a.n_head + (D == kRows ? 1 : 2) * a.n_kv;
    uintptr_t rows = (uintptr_t)a.q | (uintptr_t)a.k | (uintptr_t)a.v | (uintptr_t)a.q_norm |
                     (uintptr_t)a.k_norm | (uintptr_t)a.q_out | (uintptr_t)a.k_out;
    const long long strides = a.q_stride | a.k_stride | a.v_stride;
    const uintptr_t f16 = (uintptr_t)a.kc | (uintptr_t)a.vc, i8 = (uintptr_t)a.k8 | (uintptr_t)a.v8;
    if ((rows & 15) == 0 && strides % 4 == 0 && (f16 & 7) == 0 && (i8 & 3) == 0) {
        auto go = [&](auto few, auto many, int hd) {
            // heads that a workgroup takes at once; all of them where the tokens are enough
            const int share = n_tok < 128 ? 2048 / hd : heads;
            if (n_tok < 1024)
                hipLaunchKernelGGL(few, dim3(n_tok, (heads + share - 1) / share), dim3(256), 0,
                                   tf_stream(stream), b, n_tok, share);
            else
                hipLaunchKernelGGL(many, dim3((n_tok + 3) / 4), dim3(256), 0, tf_stream(stream), b,
                                   n_tok, share);
            return TF_LAUNCH_RESULT();
        };
        switch (a.head_dim) {
        case 64:
            return go(tf_qk_norm_rope_vec_kernel<64, D, 1>, tf_qk_norm_rope_vec_kernel<64, D, 4>, 64);
        case 128:
            return go(tf_qk_norm_rope_vec_kernel<128, D, 1>, tf_qk_norm_rope_vec_kernel<128, D, 4>, 128);
        case 256:
            return go(tf_qk_norm_rope_vec_kernel<256, D, 1>, tf_qk_norm_rope_vec_kernel<256, D, 4>, 256);
        }
    }
    hipLaunchKernelGGL(tf_qk_norm_rope_kernel<D>, dim3(n_tok, (heads + 3) / 4), dim3(256), 0,
                       tf_stream(stream), b);
    return TF_LAUNCH_RESULT();
}

}  // namespace

int tf_rope_append_kv8(float* q, const float* k, const float* v, int8_t* k8, float* kd, int8_t* v8,
                       float* vd, int n_head, int n_kv, int head_dim, int pos, const int* pos_dev,
                       float theta, tf_stream_t stream) {
    TF_CHECK_ARG(n_head > 0 && n_kv > 0 && n_head + 2LL * n_kv <= 65535 && head_dim > 0 &&
                 (pos_dev || pos >= 0));
    TF_CHECK_ARG((((uintptr_t)q | (uintptr_t)k | (uintptr_t)v) & 15) == 0 &&
                 (((uintptr_t)k8 | (uintptr_t)v8) & 3) == 0);
    QkArgs a{};
    a.q = q, a.k = k, a.v = v;  // one token: no strides
    a.q_out = q, a.k8 = k8, a.kd = kd, a.v8 = v8, a.vd = vd;
    a.n_head = n_head, a.n_kv = n_kv, a.head_dim = head_dim;
    a.pos0 = pos, a.pos0_dev = pos_dev, a.theta = theta;
    const int heads = n_head + 2 * n_kv, share = 2048 / head_dim;
    auto go = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3(1, (heads + share - 1) / share), dim3(256), 0,
                           tf_stream(stream), a, 1, share);
        return TF_LAUNCH_RESULT();
    };
    switch (head_dim) {
    case 64: return go(tf_qk_norm_rope_vec_kernel<64, kKv8, 1, true>);
    case 128: return go(tf_qk_norm_rope_vec_kernel<128, kKv8, 1, true>);
    case 256: return go(tf_qk_norm_rope_vec_kernel<256, kKv8, 1, true>);
    }
    return (int)hipErrorInvalidValue;
}

extern "C" int tf_qk_norm_rope(const float* q, int q_stride, const float* k, int k_stride,
                               const float* q_norm, const float* k_norm, float eps, float* q_out,
                               float* k_out, int n_head, int n_kv, int head_dim, int n_tok,
                               int pos0, const int* pos0_dev, float theta, tf_stream_t stream) {
    QkArgs a{};
    a.q = q, a.k = k, a.q_stride = q_stride, a.k_stride = k_stride;
    a.q_norm = q_norm, a.k_norm = k_norm, a.eps = eps;
    a.q_out = q_out, a.k_out = k_out;
    a.n_head = n_head, a.n_kv = n_kv, a.head_dim = head_dim;
    a.pos0 = pos0, a.pos0_dev = pos0_dev;
    TF_CHECK_ARG(k_out && (k != k_out || k_stride == (long long)n_kv * head_dim));
    return launch<kRows>(a, n_tok, theta, stream);
}

extern "C" int tf_qk_norm_rope_append(const float* q, int q_stride, const float* k, int k_stride,
                                      const float* v, int v_stride, const float* q_norm,
                                      const float* k_norm, float eps, float* q_out,
                                      uint16_t* k_cache, uint16_t* v_cache, int n_head, int n_kv,
                                      int head_dim, int n_tok, int pos0, const int* pos0_dev,
                                      float theta, tf_stream_t stream) {
    QkArgs a{};
    a.q = q, a.k = k, a.v = v, a.q_stride = q_stride, a.k_stride = k_stride, a.v_stride = v_stride;
    a.q_norm = q_norm, a.k_norm = k_norm, a.eps = eps;
    a.q_out = q_out, a.kc = k_cache, a.vc = v_cache;
    a.n_head = n_head, a.n_kv = n_kv, a.head_dim = head_dim;
    a.pos0 = pos0, a.pos0_dev = pos0_dev;
    TF_CHECK_ARG(v && k_cache && v_cache && v_stride >= (long long)n_kv * head_dim);
    return launch<kF16>(a, n_tok, theta, stream);
}

extern "C" int tf_qk_norm_rope_append_kv8(const float* q, int q_stride, const float* k,
                                          int k_stride, const float* v, int v_stride,
                                          const float* q_norm, const float* k_norm, float eps,
                                          float* q_out, int8_t* k8, float* kd, int8_t* v8,
                                          float* vd, int n_head, int n_kv, int head_dim, int n_tok,
                                          int pos0, const int* pos0_dev, float theta,
                                          tf_stream_t stream) {
    QkArgs a{};
    a.q = q, a.k = k, a.v = v, a.q_stride = q_stride, a.k_stride = k_stride, a.v_stride = v_stride;
    a.q_norm = q_norm, a.k_norm = k_norm, a.eps = eps;
    a.q_out = q_out, a.k8 = k8, a.kd = kd, a.v8 = v8, a.vd = vd;
    a.n_head = n_head, a.n_kv = n_kv, a.head_dim = head_dim;
    a.pos0 = pos0, a.pos0_dev = pos0_dev;
    TF_CHECK_ARG(v && k8 && kd && v8 && vd && head_dim > 0 && head_dim % 32 == 0);
    TF_CHECK_ARG(v_stride >= (long long)n_kv * head_dim);
    return launch<kKv8>(a, n_tok, theta, stream);
}
