// K/V cache rows in 8 bits: written, read back, and one token's attention
// over them.
//
// A row is the Q8 of tf_quantize_q8: int8 q[n] and one f32 scale per 32
// values, d = amax * fl(1/127), q = rint_even(x / d); value = q * d.  36 bytes
// per 32 values where f16 takes 64.  The scale is f32, as in that format, so
// that rows of any magnitude keep their 7 bits.
#include "tf_common.hpp"
#include "tf_host.hpp"

#define TF_NEG_BIG (-1e30f)

template <class T>
__device__ __forceinline__ float tf_kv8_src(T v);
template <>
__device__ __forceinline__ float tf_kv8_src<float>(float v) { return v; }
template <>
__device__ __forceinline__ float tf_kv8_src<uint16_t>(uint16_t v) { return tf_h2f(v); }

// One value a lane, a 32-lane half a group; blockIdx.y: K or V.
template <class T>
__global__ __launch_bounds__(256) void tf_kv8_write_kernel(const T* __restrict__ k,
                                                           const T* __restrict__ v,
                                                           long long src_stride,
                                                           int8_t* __restrict__ k8,
                                                           float* __restrict__ kd,
                                                           int8_t* __restrict__ v8,
                                                           float* __restrict__ vd, int n, int pos0,
                                                           const int* __restrict__ pos0_dev,
                                                           size_t count) {
    const size_t e = (size_t)blockIdx.x * 256 + threadIdx.x;
    if (e >= count) return;  // whole 32-lane halves: count % 32 == 0
    const long long t = e / n;
    const int i = (int)(e - t * n);
    const bool is_v = blockIdx.y == 1;
    const long long pos = (long long)(pos0_dev ? pos0_dev[0] : pos0) + t;
    const float x = tf_kv8_src<T>((is_v ? v : k)[t * src_stride + i]);
    const float amax = tf_group32_max(fabsf(x));
    const float d = amax * (1.0f / 127.0f);
    const size_t at = (size_t)pos * n + i;
    (is_v ? v8 : k8)[at] = (int8_t)tf_q8_value(x, amax, d);
    if ((threadIdx.x & 31) == 0) (is_v ? vd : kd)[at >> 5] = d;
}

template <class T>
__global__ __launch_bounds__(256) void tf_kv8_read_kernel(const int8_t* __restrict__ k8,
                                                          const float* __restrict__ kd,
                                                          const int8_t* __restrict__ v8,
                                                          const float* __restrict__ vd,
                                                          T* __restrict__ k, T* __restrict__ v,
                                                          size_t first, size_t count) {
    const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= count) return;
    const bool is_v = blockIdx.y == 1;
    const size_t at = first + i;
    float x = (float)(is_v ? v8 : k8)[at] * (is_v ? vd : kd)[at >> 5];
    asm("" : "+v"(x));  // the f32 product is rounded: not fused with the conversion
    T* out = is_v ? v : k;
    if constexpr (sizeof(T) == 4) out[i] = x;
    else out[i] = __builtin_bit_cast(uint16_t, (_Float16)x);
}

// One head a wave, the split walked in tiles of 64 tokens.
template <int HD>
__global__ __launch_bounds__(256) void tf_flash_kv8_kernel(
    const float* __restrict__ q, const int8_t* __restrict__ k8, const float* __restrict__ kd,
    const int8_t* __restrict__ v8, const float* __restrict__ vd, float* __restrict__ partial,
    int n_head, int n_kv, int pos0, const int* __restrict__ pos0_dev, int n_split, float scale) {
    constexpr int DPL = HD / 64;
    __shared__ float p_lds[4][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int h = blockIdx.x * 4 + wave, s = blockIdx.y;
    if (h >= n_head) return;
    const int kv_h = h / (n_head / n_kv);
    if (pos0_dev) pos0 = pos0_dev[0];
    const int seq = pos0 + 1;
    const int chunk = (seq + n_split - 1) / n_split;
    const int t_begin = (int)min((long long)s * chunk, (long long)seq);
    const int t_end = min(t_begin + chunk, seq);
    const float* qh = q + (size_t)h * HD;
    float m = TF_NEG_BIG, l = 0.f, o[DPL];
    for (int i = 0; i < DPL; i++) o[i] = 0.f;
    for (int t0 = t_begin; t0 < t_end; t0 += 64) {
        const int t = t0 + lane;
        float sc = TF_NEG_BIG;
        if (t < t_end) {
            const size_t row = ((size_t)t * n_kv + kv_h) * HD;
            float acc = 0.f;
            for (int g = 0; g < HD / 32; g++) {
                float a = 0.f;
                for (int i = 0; i < 32; i++) a = fmaf(qh[32 * g + i], (float)k8[row + 32 * g + i], a);
                acc = fmaf(a, kd[row / 32 + g], acc);
            }
            sc = acc * scale;
        }
        const float m_new = fmaxf(m, tf_wave_max(sc));
        const float alpha = __expf(m - m_new);
        const float e = t < t_end ? __expf(sc - m_new) : 0.f;
        p_lds[wave][lane] = e;
        l = l * alpha + tf_group_sum<64>(e);
        m = m_new;
        for (int i = 0; i < DPL; i++) o[i] *= alpha;
        __builtin_amdgcn_wave_barrier();
        for (int tt = 0; tt < min(64, t_end - t0); tt++) {
            const size_t row = ((size_t)(t0 + tt) * n_kv + kv_h) * HD;
            for (int i = 0; i < DPL; i++) {
                const int dim = lane + 64 * i;
                o[i] = fmaf(p_lds[wave][tt] * vd[(row + dim) / 32], (float)v8[row + dim], o[i]);
            }
        }
        __builtin_amdgcn_wave_barrier();
    }
    float* base = partial + ((size_t)h * n_split + s) * (2 + HD);
    if (lane == 0) {
        base[0] = m;
        base[1] = l;
    }
    for (int i = 0; i < DPL; i++) base[2 + lane + 64 * i] = o[i];
}

// ---------------------------------------------------------------- C ABI

extern "C" int tf_kv8_write(const void* k, const void* v, int src_type, int src_stride, int8_t* k8,
                            float* kd, int8_t* v8, float* vd, int n, int pos0, const int* pos0_dev,
                            int n_tok, tf_stream_t stream) {
    TF_CHECK_ARG(k && v && k8 && kd && v8 && vd && n > 0 && n % 32 == 0 && n_tok > 0);
    TF_CHECK_ARG((src_type == TF_KV_F32 || src_type == TF_KV_F16) && src_stride >= n);
    TF_CHECK_ARG(pos0_dev || (pos0 >= 0 && pos0 <= INT32_MAX - n_tok));
    const size_t count = (size_t)n_tok * n;
    TF_CHECK_ARG((count + 255) / 256 <= UINT32_MAX / 256);
    const dim3 grid((unsigned)((count + 255) / 256), 2);
    if (src_type == TF_KV_F32)
        hipLaunchKernelGGL(tf_kv8_write_kernel<float>, grid, dim3(256), 0, tf_stream(stream),
                           (const float*)k, (const float*)v, src_stride, k8, kd, v8, vd, n, pos0,
                           pos0_dev, count);
    else
        hipLaunchKernelGGL(tf_kv8_write_kernel<uint16_t>, grid, dim3(256), 0, tf_stream(stream),
                           (const uint16_t*)k, (const uint16_t*)v, src_stride, k8, kd, v8, vd, n,
                           pos0, pos0_dev, count);
    return TF_LAUNCH_RESULT();
}

extern "C" int tf_kv8_read(const int8_t* k8, const float* kd, const int8_t* v8, const float* vd,
                           void* k, void* v, int dst_type, int n, int row0, int n_rows,
                           tf_stream_t stream) {
    TF_CHECK_ARG(k && v && k8 && kd && v8 && vd && n > 0 && n % 32 == 0 && n_rows > 0 && row0 >= 0);
    TF_CHECK_ARG(dst_type == TF_KV_F32 || dst_type == TF_KV_F16);
    const size_t first = (size_t)row0 * n, count = (size_t)n_rows * n;
    TF_CHECK_ARG((count + 255) / 256 <= UINT32_MAX / 256);
    const dim3 grid((unsigned)((count + 255) / 256), 2);
    if (dst_type == TF_KV_F32)
        hipLaunchKernelGGL(tf_kv8_read_kernel<float>, grid, dim3(256), 0, tf_stream(stream), k8, kd,
                           v8, vd, (float*)k, (float*)v, first, count);
    else
        hipLaunchKernelGGL(tf_kv8_read_kernel<uint16_t>, grid, dim3(256), 0, tf_stream(stream), k8,
                           kd, v8, vd, (uint16_t*)k, (uint16_t*)v, first, count);
    return TF_LAUNCH_RESULT();
}

extern "C" int tf_flash_decode_kv8_n_split(int n_kv, int head_dim, int max_seq) {
    (void)head_dim;
    return tf_flash_decode_n_split(n_kv, max_seq);
}

extern "C" int tf_flash_decode_kv8(const float* q, const int8_t* k8, const float* kd,
                                   const int8_t* v8, const float* vd, float* partial, float* out,
                                   int8_t* q8, float* d8, int n_head, int n_kv, int head_dim,
                                   int pos0, const int* pos0_dev, int n_split, float scale,
                                   tf_stream_t stream) {
    TF_CHECK_ARG(q && k8 && kd && v8 && vd && partial && out && ((q8 == nullptr) == (d8 == nullptr)));
    TF_CHECK_ARG(n_head > 0 && n_kv > 0 && n_head % n_kv == 0 && n_head / n_kv <= 16);
    TF_CHECK_ARG(n_split >= 1 && n_split <= 1024 && (pos0_dev || (pos0 >= 0 && pos0 < INT32_MAX - 1024)));
    auto go = [&](auto kern) {
        hipLaunchKernelGGL(kern, dim3((n_head + 3) / 4, n_split), dim3(256), 0, tf_stream(stream), q,
                           k8, kd, v8, vd, partial, n_head, n_kv, pos0, pos0_dev, n_split, scale);
        return TF_LAUNCH_RESULT();
    };
    int rc;
    switch (head_dim) {
    case 64: rc = go(tf_flash_kv8_kernel<64>); break;
    case 128: rc = go(tf_flash_kv8_kernel<128>); break;
    case 256: rc = go(tf_flash_kv8_kernel<256>); break;
    default: return (int)hipErrorInvalidValue;
    }
    if (rc) return rc;
    return q8 ? tf_flash_decode_reduce_q8(partial, out, q8, d8, n_head, head_dim, n_split, stream)
              : tf_flash_decode_reduce(partial, out, n_head, head_dim, n_split, 1, stream);
}
