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
};

// Turns of pair i at position pos, less their whole part.
__device__ __forceinline__ float turns(long long pos, int i, int head_dim, double log2_theta) {
    constexpr double kInv2Pi = 0.15915494309189533577;
    const double f = exp2(-2.0 * i / head_dim * log2_theta) * kInv2Pi;
    const double a = (double)pos * f;
    return (float)(a - rint(a));
}

// A head a wave, a workgroup a token and four heads.  y: the head in LDS.
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
    __builtin_amdgcn_wave_barrier();
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
    __builtin_amdgcn_wave_barrier();
    if (kind == 0 || D == kRows) {
        float* out = kind == 0 ? a.q_out + ((size_t)t * a.n_head + h) * hd
                               : a.k_out + ((size_t)t * a.n_kv + h) * hd;
        for (int i = lane; i < hd; i += 64) out[i] = y[i];
        return;
    }
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
    hipLaunchKernelGGL(tf_qk_norm_rope_kernel<D>, dim3(n_tok, (heads + 3) / 4), dim3(256), 0,
                       tf_stream(stream), b);
    return TF_LAUNCH_RESULT();
}

}  // namespace

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
