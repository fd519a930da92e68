// K/V cache rows in 8 bits: written, read back, and one token's attention
// over them.
//
// A row is the Q8 of tf_quantize_q8: int8 q[n] and one f32 scale per 32
// values, d = amax * fl(1/127), q = rint_even(x / d); value = q * d.  36 bytes
// per 32 values where f16 takes 64.  The scale is f32, as in that format, so
// that rows of any magnitude keep their 7 bits.
#include <math.h>

#include "kv8.hpp"
#include "lds_dma.hpp"
#include "tf_common.hpp"
#include "tf_host.hpp"

#define TF_NEG_BIG (-1e30f)

// Rows of n values (n % 32 == 0), blockIdx.y K or V.  What bounds both is their bytes,
// so a lane moves 16 of the wider side at once; VEC false: a value a lane, for rows
// that are not so aligned.  32768 f16 rows of 512, K and V (67 MB in, 38 out): 21.8 us,
// 4.8 TB/s, with the VALU busy for 11 of them;
// read back as f32 (38 in, 134 out) 25.2 us, 6.8 TB/s with what the last-level cache holds.
typedef _Float16 tf_h2x __attribute__((ext_vector_type(2)));

struct TfKv8Rows {
    const void *k, *v;
    long long stride;
    int8_t *k8, *v8;
    float *kd, *vd;
    int n, pos0;
    const int* pos0_dev;
    size_t count;  // values
};

template <bool F16, bool VEC>
__global__ __launch_bounds__(256) void tf_kv8_write_kernel(TfKv8Rows a) {
    constexpr int PER = !VEC ? 1 : F16 ? 8 : 4;  // values a lane
    const size_t e = ((size_t)blockIdx.x * 256 + threadIdx.x) * PER;
    if (e >= a.count) return;  // whole groups: count % 32 == 0
    const bool is_v = blockIdx.y == 1;
    const long long to = (long long)(a.pos0_dev ? a.pos0_dev[0] : a.pos0) * a.n + (long long)e;
    if (to < 0) return;  // a row before the cache
    const size_t at = (size_t)to;
    size_t from = e;  // tight rows
    if (a.stride != a.n) {
        const size_t t = e >> 32 == 0 ? (uint32_t)e / (uint32_t)a.n : e / a.n;
        from += t * (a.stride - a.n);
    }
    const void* src = is_v ? a.v : a.k;
    int8_t* q = (is_v ? a.v8 : a.k8) + at;
    float* ds = (is_v ? a.vd : a.kd) + (at >> 5);
    if constexpr (!VEC) {
        const float x = F16 ? tf_h2f(static_cast<const uint16_t*>(src)[from])
                            : static_cast<const float*>(src)[from];
        const float amax = tf_group32_max(fabsf(x));
        const float d = amax * (1.0f / 127.0f);
        *q = (int8_t)tf_q8_value(x, amax, d);
        if ((threadIdx.x & 31) == 0) *ds = d;
    } else if constexpr (F16) {
        const tf_u32x4 b = tf_ld16(static_cast<const uint16_t*>(src) + from);
        float x[8], amax = 0.f;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            x[j] = tf_h2f(b[j >> 1] >> (16 * (j & 1)));
            amax = fmaxf(amax, fabsf(x[j]));
        }
        amax = fmaxf(amax, tf_dpp<TF_DPP_QUAD_1032>(amax));
        amax = fmaxf(amax, tf_dpp<TF_DPP_QUAD_2301>(amax));
        uint32_t o[2];
        const float d = tf_q8_words(x, amax, o);
        *reinterpret_cast<tf_u32x2*>(q) = tf_u32x2{o[0], o[1]};
        if ((threadIdx.x & 3) == 0) *ds = d;
    } else {
        const tf_u32x4 b = tf_ld16(static_cast<const float*>(src) + from);
        const float x[4] = {__uint_as_float(b.x), __uint_as_float(b.y), __uint_as_float(b.z),
                            __uint_as_float(b.w)};
        float d;
        *reinterpret_cast<uint32_t*>(q) = tf_q8_quad(x, d);
        if ((threadIdx.x & 7) == 0) *ds = d;
    }
}

template <bool F16, bool VEC>
__global__ __launch_bounds__(256) void tf_kv8_read_kernel(const int8_t* __restrict__ k8,
                                                          const float* __restrict__ kd,
                                                          const int8_t* __restrict__ v8,
                                                          const float* __restrict__ vd,
                                                          void* __restrict__ k, void* __restrict__ v,
                                                          size_t first, size_t count) {
    constexpr int PER = !VEC ? 1 : F16 ? 8 : 4;
    const size_t i = ((size_t)blockIdx.x * 256 + threadIdx.x) * PER;
    if (i >= count) return;
    const bool is_v = blockIdx.y == 1;
    const size_t at = first + i;
    const int8_t* q = (is_v ? v8 : k8) + at;
    const float d = (is_v ? vd : kd)[at >> 5];
    uint32_t b[PER > 4 ? 2 : 1];
    if constexpr (!VEC) {
        b[0] = (uint8_t)*q;
    } else {
#pragma unroll
        for (int j = 0; j < PER / 4; j++) b[j] = reinterpret_cast<const uint32_t*>(q)[j];
    }
    float x[PER];
#pragma unroll
    for (int j = 0; j < PER; j++) {
        x[j] = (float)(int8_t)(b[j >> 2] >> (8 * (j & 3))) * d;
        asm("" : "+v"(x[j]));  // the f32 product is rounded: not fused with the conversion
    }
    if constexpr (F16) {
        uint16_t* out = static_cast<uint16_t*>(is_v ? v : k) + i;
        if constexpr (VEC) {
            tf_u32x4 o;
#pragma unroll
            for (int j = 0; j < 4; j++)
                o[j] = __builtin_bit_cast(uint32_t, tf_h2x{(_Float16)x[2 * j], (_Float16)x[2 * j + 1]});
            *reinterpret_cast<tf_u32x4*>(out) = o;
        } else {
            *out = __builtin_bit_cast(uint16_t, (_Float16)x[0]);
        }
    } else {
        float* out = static_cast<float*>(is_v ? v : k) + i;
        if constexpr (VEC) *reinterpret_cast<float4*>(out) = make_float4(x[0], x[1], x[2], x[3]);
        else *out = x[0];
    }
}

// ------------------------------------------- one token's attention
//
// out_h = sum_t softmax_t(scale q_h . K_t) V_t with K_t = kd[t][g] k8[t], V_t =
// vd[t][g] v8[t] (g: 32 dims).  Grid (kv head, split); a workgroup reads each
// byte of its split once, for the G query heads of the kv head.
//
// A wave owns the 32-token tiles j = wave, wave + W, ... of the split and moves
// them HBM -> LDS itself (global_load_lds, no register staging) into a two-slot
// ring of its own, one tile ahead; the waves meet only to share the query and
// to merge their (m, l, O).  Per tile, on v_mfma_f32_16x16x32_f16 (lane l, n = l
// % 16, g = l / 16: A[n][8g ..], B[8g ..][n], C[4g + r][n]):
//   K Q^T  one k step is one scale group: A = 8 bytes of token n (or 16 + n), as
//          f16 (exact), B = 8 dims of head n in two f16 parts after a power of
//          two of the head's own (2^-22 of its largest); the sums of a group are f32
//          and take the token's scale there.
//   softmax of head n over the lane's tokens 4g + r and 16 + 4g + r, in f32.
//          The maximum and the factor f below are renewed, and O rescaled, only
//          where a lane found a larger one.
//   V^T P^T with the tokens in the order in which the lane has them: A = 8 tokens
//          of dim n (ds_read_b64_tr_b8), as f16 (exact); B = p vd[t][g] f, for each
//          group of dims, in two f16 parts.  f is a power of two of the head's that
//          keeps every p vd f below 2^15 and the largest met so far (in the weights of
//          the maximum so far) within 2^12 of that, so the parts end at 2^-28 of the
//          largest product or below, whatever the scales of rows without weight.
// 131072 tokens of 28/4 heads of 128 (151 MB): 35.8 us and 4.7 for the merge, 4.2 TB/s of
// the 5.8 that a plain read reaches; the copies alone take 30, and conversions, splits
// and exponentials keep the VALU busy for 18 beside them.  5001 tokens of
// 14/2 heads of 64: 5.5 + 3.7 us; 512 of 16/2 of 128: 6.9 + 2.7; there a launch's chain
// of query, first tile and merge is what there is.
//
// LDS rows keep their 16-byte chunks xor-ed with the row (the copies' sources
// are permuted), so that the 16 rows that half a wave reads lie in distinct banks.
template <int HD>
struct TfKv8 {
    static constexpr int T = 32;                       // tokens per tile
    static constexpr int W = HD == 256 ? 4 : 8;        // waves
    static constexpr int NG = HD / 32, DB = HD / 16;
    static constexpr int NC = HD / 16;                 // 16-byte chunks of a row
    static constexpr int TILE = T * HD;                // bytes of K (or V)
    static constexpr int SC = T * NG * 4;              // bytes of its scales
    static constexpr int KOFF = 0, KDOFF = TILE, VDOFF = TILE + SC, VOFF = TILE + 2 * SC;
    static constexpr int SLOT = 2 * (TILE + SC);
    static constexpr int COPIES = TILE / 1024;         // 16 bytes a lane
    static constexpr int K_COPIES = COPIES + (HD == 128 ? 1 : 2);  // K and both scales
    static constexpr int PER = K_COPIES + COPIES;
    static constexpr int LDS = W * 2 * SLOT;
    static constexpr int CR = HD + 4;                  // merge row: m, l, pad, O
    static_assert(16 * HD * 4 <= SLOT, "the query fits a slot");
    static_assert(W * 16 * CR * 4 <= LDS, "the merge rows fit the ring");
    // the chunk permutation of a K row (16 consecutive rows are read together) and
    // of a V row (8a .. 8a + 7 and 16 + 8a .. are)
    static __device__ __forceinline__ int kswz(int r) {
        return HD == 64 ? (r >> 2) & 3 : HD == 128 ? (r >> 1) & 7 : r & 15;
    }
    static __device__ __forceinline__ int vswz(int r) {
        return HD == 64    ? ((r >> 2) & 1) | ((r >> 4) << 1)
               : HD == 128 ? ((r >> 1) & 3) | ((r >> 4) << 2)
                           : (r & 7) | ((r >> 4) << 3);
    }
};

// Eight int8 values as f16: with the sign bit flipped a byte is q + 128, behind
// 0x64 the f16 number 1024 + q + 128, less 1152 exactly q.
__device__ __forceinline__ tf_h16x8 tf_i8_f16(tf_u32x2 b) {
    union {
        uint32_t u[4];
        tf_h2x h[4];
        tf_h16x8 v;
    } r;
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const uint32_t x = b[i] ^ 0x80808080u;
        r.u[2 * i] = __builtin_amdgcn_perm(0x64646464u, x, 0x04010400u);
        r.u[2 * i + 1] = __builtin_amdgcn_perm(0x64646464u, x, 0x04030402u);
    }
#pragma unroll
    for (int i = 0; i < 4; i++) r.h[i] -= tf_h2x{(_Float16)1152.f, (_Float16)1152.f};
    return r.v;
}

// a, b = hi + lo in f16 parts.  hi is opaque to the compiler, which would otherwise
// round the product behind a value a second time, and not always alike, for lo's
// difference (2^-11 of a value in one of 2^13: 4e-6 of an output of 5000 tokens).
__device__ __forceinline__ void tf_kv8_split(float a, float b, tf_h2x& hi, tf_h2x& lo) {
    uint32_t h = __builtin_bit_cast(uint32_t, tf_h2x{(_Float16)a, (_Float16)b});
    asm("" : "+v"(h));
    hi = __builtin_bit_cast(tf_h2x, h);
    lo = tf_h2x{(_Float16)(a - (float)hi.x), (_Float16)(b - (float)hi.y)};
}

template <int N>
__device__ __forceinline__ void tf_kv8_wait() {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

// With out (n_split == 1 only) the workgroup writes the output itself, and its
// Q8 with q8, as tf_flash_decode does.
template <int HD>
__global__ __launch_bounds__(64 * TfKv8<HD>::W) void tf_flash_kv8_kernel(
    const float* __restrict__ q, const int8_t* __restrict__ k8, const float* __restrict__ kd,
    const int8_t* __restrict__ v8, const float* __restrict__ vd, float* __restrict__ partial,
    int G, int n_kv, int pos0, const int* __restrict__ pos0_dev, int n_split, float scale,
    float* __restrict__ out, int8_t* __restrict__ q8, float* __restrict__ d8) {
    using L = TfKv8<HD>;
    constexpr int NG = L::NG, DB = L::DB, W = L::W;
    extern __shared__ __align__(16) uint8_t lds[];
    const int kv_h = blockIdx.y, s = blockIdx.x + 8 * blockIdx.z;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = lane & 15, g = lane >> 4;
    if (pos0_dev) pos0 = pos0_dev[0];
    const int seq = pos0 + 1;
    // whole tiles a split
    const uint32_t tiles = seq > 0 ? ((uint32_t)seq + L::T - 1) / L::T : 0;
    const uint32_t share = (tiles + n_split - 1) / (uint32_t)n_split;
    const uint32_t first = min(s * share, tiles);
    const int n_tiles = (int)min(share, tiles - first);
    const int t_begin = (int)first * L::T;
    const int t_end = n_tiles ? min(t_begin + n_tiles * L::T, seq) : t_begin;
    const uint32_t row8 = (uint32_t)n_kv * HD, rowd = (uint32_t)n_kv * NG * 4;  // bytes
    uint8_t* ring = lds + wave * 2 * L::SLOT;

    // the query's rows (heads past G repeat the last) into wave 0's second slot
    constexpr int HPC = 1024 / (HD * 4);  // heads of a copy
    const float* qk = q + (size_t)kv_h * G * HD;
#pragma unroll
    for (int i = 0; i < 16 / HPC; i++)
        if (i % W == wave) {
            const int h = min(i * HPC + lane / (HD / 4), G - 1);
            tf_lds_dma16(qk + (size_t)h * HD + 4 * (lane % (HD / 4)),
                         tf_lds_off(lds) + L::SLOT + 1024 * i);
        }
    // tile j -> slot: K and the scales of K and V (issue_k), then V (issue_v); rows
    // past the split repeat its last (their weights are zero).  Offsets inside a tile
    // are 24-bit products: row8 < 2^24.
    constexpr int RPC = 64 / L::NC;  // rows of a copy
    const int lr = lane / L::NC, lc = lane % L::NC;
    auto k_off = [&](int i, int last) {
        const int r = RPC * i + lr;
        return __umul24(min(r, last), row8) + 16 * (lc ^ L::kswz(r));
    };
    auto v_off = [&](int i, int last) {
        const int r = RPC * i + lr;
        return __umul24(min(r, last), row8) + 16 * (lc ^ L::vswz(r));
    };
    auto s_off = [&](int last) {
        const int l = HD == 128 ? lane & 31 : lane >> 1;
        return __umul24(min(l, last), rowd) +
               (HD == 128 ? 0 : (HD == 256 ? 16 : 4) * (lane & 1));
    };
    const uint8_t* k_head = reinterpret_cast<const uint8_t*>(k8) + kv_h * HD;
    const uint8_t* v_head = reinterpret_cast<const uint8_t*>(v8) + kv_h * HD;
    const uint8_t* kd_head = reinterpret_cast<const uint8_t*>(kd) + kv_h * NG * 4;
    const uint8_t* vd_head = reinterpret_cast<const uint8_t*>(vd) + kv_h * NG * 4;
    auto issue_k = [&](int j, int slot) {
        const int t0 = t_begin + L::T * j, last = t_end - 1 - t0;
        const uint32_t base = tf_lds_off(ring) + slot * L::SLOT;
        const uint8_t* kb = k_head + (size_t)t0 * row8;
        const uint8_t* kdb = kd_head + (size_t)t0 * rowd;
        const uint8_t* vdb = vd_head + (size_t)t0 * rowd;
#pragma unroll
        for (int i = 0; i < L::COPIES; i++)
            tf_lds_dma_s<16>(kb, k_off(i, last), base + L::KOFF + 1024 * i);
        const uint32_t so = s_off(last);
        if constexpr (HD == 128) {
            tf_lds_dma16((lane < 32 ? kdb : vdb) + so, base + L::KDOFF);
        } else {
            constexpr int DW = HD == 256 ? 16 : 4;
            tf_lds_dma_s<DW>(kdb, so, base + L::KDOFF);
            tf_lds_dma_s<DW>(vdb, so, base + L::VDOFF);
        }
    };
    auto issue_v = [&](int j, int slot) {
        const int t0 = t_begin + L::T * j, last = t_end - 1 - t0;
        const uint32_t base = tf_lds_off(ring) + slot * L::SLOT;
        const uint8_t* vb = v_head + (size_t)t0 * row8;
#pragma unroll
        for (int i = 0; i < L::COPIES; i++)
            tf_lds_dma_s<16>(vb, v_off(i, last), base + L::VOFF + 1024 * i);
    };
    auto issue = [&](int j, int slot) {
        issue_k(j, slot);
        issue_v(j, slot);
    };
    const bool any = wave < n_tiles;
    if (any) {
        issue(wave, 0);
        tf_kv8_wait<L::PER>();  // the query's copies are older
    } else {
        tf_kv8_wait<0>();
    }
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");

    // the query of head n: dims 32 j + 8 g .. + 7 as two f16 parts of q 2^-e, the
    // head's largest in [2^14, 2^15) (an infinite one stays in its head)
    tf_h16x8 qa[NG][2];
    {
        const float* ql = reinterpret_cast<const float*>(lds + L::SLOT) + n * HD + 8 * g;
        float qv[NG][8], qmax = 0.f;
#pragma unroll
        for (int j = 0; j < NG; j++)
#pragma unroll
            for (int i = 0; i < 8; i += 4) {
                const float4 v = *reinterpret_cast<const float4*>(ql + 32 * j + i);
                const float f = n < G ? 1.f : 0.f;
                qv[j][i] = v.x * f, qv[j][i + 1] = v.y * f;
                qv[j][i + 2] = v.z * f, qv[j][i + 3] = v.w * f;
            }
#pragma unroll
        for (int j = 0; j < NG; j++)
#pragma unroll
            for (int i = 0; i < 8; i++) qmax = fmaxf(qmax, fabsf(qv[j][i]));
        qmax = fmaxf(qmax, __shfl_xor(qmax, 16));
        qmax = fmaxf(qmax, __shfl_xor(qmax, 32));
        int fe = 141 - (int)(__float_as_uint(qmax) >> 23);
        fe = fe > 126 ? 126 : fe < -113 ? -113 : fe;
        const float f = __uint_as_float((uint32_t)(fe + 127) << 23);
#pragma unroll
        for (int j = 0; j < NG; j++)
#pragma unroll
            for (int i = 0; i < 8; i += 2) {
                tf_h2x h2, l2;
                tf_kv8_split(qv[j][i] * f, qv[j][i + 1] * f, h2, l2);
                qa[j][0][i] = h2.x, qa[j][0][i + 1] = h2.y;
                qa[j][1][i] = l2.x, qa[j][1][i + 1] = l2.y;
            }
        scale *= __uint_as_float((uint32_t)(127 - fe) << 23);
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();  // the query has been read: its slot is free
    asm volatile("" ::: "memory");
    if (wave + W < n_tiles) issue(wave + W, 1);

    float m = TF_NEG_BIG, l = 0.f;  // head n: the maximum, this lane's share of the sum
    // of head n: the largest weighted scale met, as of m; those below vtop fit under vf
    float vmost = 0.f, vtop = 0.f, vf = 0x1p26f;
    tf_f32x4v o[DB];                // O^T of dims 16 b + 4 g + r, head n, times vf
#pragma unroll
    for (int b = 0; b < DB; b++) o[b] = tf_f32x4v{0.f, 0.f, 0.f, 0.f};
    const int tr = ((lane & 15) >> 1);                             // the lane's row of a transposing read
    const int vrow = (tr < 4 ? tr : 12 + tr) + 4 * g;              // its token
    const uint32_t vbase = L::VOFF + vrow * HD + 8 * (lane & 1);
    const int vx = L::vswz(vrow);

    int slot = 0;
    for (int j = wave; j < n_tiles; j += W, slot ^= 1) {
        const uint8_t* sl = ring + slot * L::SLOT;
        const int t0 = t_begin + L::T * j;
        const bool next = j + W < n_tiles;
        if (next) tf_kv8_wait<L::PER + L::COPIES>();
        else tf_kv8_wait<L::COPIES>();
        // everything that the scores take, at once: the reads overlap, and the next tile's
        // K can be on its way under all of the arithmetic
        const bool refill = j + 2 * W < n_tiles;
        tf_u32x2 kraw[2][NG];
        float ksc[2][4][NG], vsc[2][4][NG];
#pragma unroll
        for (int u = 0; u < 2; u++)
#pragma unroll
            for (int i = 0; i < NG; i++) {
                const int row = 16 * u + n;
                kraw[u][i] = *reinterpret_cast<const tf_u32x2*>(
                    sl + L::KOFF + row * HD + 16 * ((2 * i + (g >> 1)) ^ L::kswz(row)) + 8 * (g & 1));
            }
#pragma unroll
        for (int u = 0; u < 2; u++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const int row = 16 * u + 4 * g + r;
                const float* kp = reinterpret_cast<const float*>(sl + L::KDOFF) + row * NG;
                const float* vp = reinterpret_cast<const float*>(sl + L::VDOFF) + row * NG;
#pragma unroll
                for (int i = 0; i < NG; i++) ksc[u][r][i] = kp[i], vsc[u][r][i] = vp[i];
            }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        if (refill) issue_k(j + 2 * W, slot);
        // ---- scores of tokens 16 u + 4 g + r
        float sv[2][4];
#pragma unroll
        for (int u = 0; u < 2; u++) {
            float acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < NG; i++) {
                const tf_h16x8 kf = tf_i8_f16(kraw[u][i]);
                tf_f32x4v c = tf_f32x4v{0.f, 0.f, 0.f, 0.f};
                c = tf_mfma_f16_k32(kf, qa[i][1], c);
                c = tf_mfma_f16_k32(kf, qa[i][0], c);
#pragma unroll
                for (int r = 0; r < 4; r++) acc[r] = fmaf(c[r], ksc[u][r][i], acc[r]);
            }
#pragma unroll
            for (int r = 0; r < 4; r++) {
                float x = acc[r] * scale;
                asm("" : "+v"(x));  // rounded before the maximum is subtracted
                sv[u][r] = t0 + 16 * u + 4 * g + r < t_end ? x : -INFINITY;
            }
        }
        float tt[2][4], top = 0.f, tm = sv[0][0];  // tt: a token's largest scale
#pragma unroll
        for (int u = 0; u < 2; u++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
                tt[u][r] = vsc[u][r][0];
#pragma unroll
                for (int i = 1; i < NG; i++) tt[u][r] = fmaxf(tt[u][r], vsc[u][r][i]);
                top = fmaxf(top, tt[u][r]);
                tm = fmaxf(tm, sv[u][r]);
            }
        if (__ballot(tm > m) | __ballot(top >= vtop)) {
            tm = fmaxf(tm, __shfl_xor(tm, 16));
            tm = fmaxf(tm, __shfl_xor(tm, 32));
            top = tf_wave_max(top);
            const float m_new = fmaxf(m, tm);
            const float alpha = __expf(m - m_new);
            float re = alpha;
            vmost *= alpha;
            if (__ballot(top >= vtop) | __ballot(vmost < vtop * 0x1p-5f)) {
                // Where the tile's scales are within 8 of each other and one of its tokens
                // has a weight of e^-2 or more, the largest weighted one is within 2^6 of
                // the largest; else it is formed.
                float low = INFINITY;
#pragma unroll
                for (int u = 0; u < 2; u++)
#pragma unroll
                    for (int r = 0; r < 4; r++) low = fminf(low, tt[u][r]);
                low = -tf_wave_max(-low);
                if (__ballot(low * 8.f < top || tm < m_new - 2.f)) {
                    float most = 0.f;
#pragma unroll
                    for (int u = 0; u < 2; u++)
#pragma unroll
                        for (int r = 0; r < 4; r++)
                            most = fmaxf(most, tt[u][r] * __builtin_amdgcn_exp2f(
                                                   (sv[u][r] - m_new) * 1.44269504088896340736f));
                    most = fmaxf(most, __shfl_xor(most, 16));
                    most = fmaxf(most, __shfl_xor(most, 32));
                    top = fminf(top, most * 64.f);
                }
                vmost = fmaxf(vmost, top);
                // the power of two that takes products up to vmost below 2^15
                int fe = 141 - (int)(__float_as_uint(vmost) >> 23);
                fe = fe > 126 ? 126 : fe < -113 ? -113 : fe;
                // (by no more than 2^100 at once: the quotient is finite)
                const float f = fminf(__uint_as_float((uint32_t)(fe + 127) << 23), vf * 0x1p100f);
                re *= f / vf;
                vf = f;
                vtop = __uint_as_float((269u << 23) - __float_as_uint(f));  // 2^15 / f
            }
            m = m_new;
            l *= alpha;
#pragma unroll
            for (int b = 0; b < DB; b++) o[b] *= re;
        }
        float p[2][4];
#pragma unroll
        for (int u = 0; u < 2; u++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
                p[u][r] = __builtin_amdgcn_exp2f((sv[u][r] - m) * 1.44269504088896340736f);
                l += p[u][r];
                p[u][r] *= vf;
            }
        tf_h16x8 ph[NG], pl[NG];  // p vd[t][i], by group of dims
#pragma unroll
        for (int i = 0; i < NG; i++)
#pragma unroll
            for (int u = 0; u < 2; u++)
#pragma unroll
                for (int r = 0; r < 4; r += 2) {
                    tf_h2x h2, l2;
                    tf_kv8_split(p[u][r] * vsc[u][r][i], p[u][r + 1] * vsc[u][r + 1][i], h2, l2);
                    ph[i][4 * u + r] = h2.x, ph[i][4 * u + r + 1] = h2.y;
                    pl[i][4 * u + r] = l2.x, pl[i][4 * u + r + 1] = l2.y;
                }
        if (refill) tf_kv8_wait<L::PER + L::K_COPIES>();
        else if (next) tf_kv8_wait<L::PER>();
        else tf_kv8_wait<0>();
        // ---- V^T P^T
        typedef int i32x2 __attribute__((ext_vector_type(2)));
        i32x2 vraw[DB];
#pragma unroll
        for (int b = 0; b < DB; b++)
            vraw[b] = __builtin_amdgcn_ds_read_tr8_b64_v2i32(
                (__attribute__((address_space(3))) i32x2*)(sl + vbase + 16 * (b ^ vx)));
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        if (refill) issue_v(j + 2 * W, slot);
#pragma unroll
        for (int b = 0; b < DB; b++) {
            const tf_h16x8 va = tf_i8_f16(__builtin_bit_cast(tf_u32x2, vraw[b]));
            o[b] = tf_mfma_f16_k32(va, pl[b / 2], o[b]);
            o[b] = tf_mfma_f16_k32(va, ph[b / 2], o[b]);
        }
    }

    // ---- merge the waves' (m, l, O)
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    __syncthreads();  // every wave is done with its ring
    float* cmb = reinterpret_cast<float*>(lds);
    const int nw = n_tiles < W ? n_tiles : W;
    if (wave < nw) {
        float* row = cmb + (wave * 16 + n) * L::CR;
        if (g == 0) {
            row[0] = m;
            row[1] = l;
        }
        const float inv = 1.f / vf;  // a power of two
#pragma unroll
        for (int b = 0; b < DB; b++) *reinterpret_cast<tf_f32x4v*>(row + 4 + 16 * b + 4 * g) = o[b] * inv;
    }
    __syncthreads();
    for (int i = tid; i < G * HD; i += 64 * W) {
        const int h = i / HD, d = i % HD;
        float M = TF_NEG_BIG;
        for (int w = 0; w < nw; w++) M = fmaxf(M, cmb[(w * 16 + h) * L::CR]);
        float O = 0.f, S = 0.f;
        for (int w = 0; w < nw; w++) {
            const float* row = cmb + (w * 16 + h) * L::CR;
            const float a = __expf(row[0] - M);
            O += a * row[4 + d];
            S += a * row[1];
        }
        if (out) {  // workgroup-uniform; G * HD is a multiple of 64
            const float v = O / fmaxf(S, 1e-20f);
            const size_t oi = (size_t)kv_h * G * HD + i;
            out[oi] = v;
            if (q8) {  // this 32-lane half holds one 32-value group
                const float amax = tf_group32_max(fabsf(v));
                const float dq = amax * (1.0f / 127.0f);
                q8[oi] = (int8_t)tf_q8_value(v, amax, dq);
                if ((lane & 31) == 0) d8[oi >> 5] = dq;
            }
            continue;
        }
        float* base = partial + ((size_t)(kv_h * G + h) * n_split + s) * (2 + HD);
        if (d == 0) {
            base[0] = M;
            base[1] = S;
        }
        base[2 + d] = O;
    }
}

template <int HD>
static int tf_flash_kv8_launch(const float* q, const int8_t* k8, const float* kd, const int8_t* v8,
                               const float* vd, float* partial, int n_head, int n_kv, int pos0,
                               const int* pos0_dev, int n_split, float scale, float* out,
                               int8_t* q8, float* d8, tf_stream_t stream) {
    using L = TfKv8<HD>;
    // 4 bytes a copy for the scales of head_dim 64, else 16
    const uintptr_t sc = (uintptr_t)kd | (uintptr_t)vd;
    TF_CHECK_ARG((((uintptr_t)q | (uintptr_t)k8 | (uintptr_t)v8) & 15) == 0 &&
                 (sc & (HD == 64 ? 3 : 15)) == 0);
    const int rc = tf_set_lds_limit((const void*)tf_flash_kv8_kernel<HD>, L::LDS);
    if (rc) return rc;
    // Workgroup b runs on XCD b mod 8: where the splits divide by 8, the kv heads of
    // one split, whose rows lie side by side, share an XCD and its L2 (8 kv heads, 302
    // MB: 83 -> 71 us).
    const bool eights = n_split % 8 == 0;
    const dim3 grid(eights ? 8 : n_split, n_kv, eights ? n_split / 8 : 1);
    hipLaunchKernelGGL(tf_flash_kv8_kernel<HD>, grid, dim3(64 * L::W), L::LDS, tf_stream(stream), q,
                       k8, kd, v8, vd, partial, n_head / n_kv, n_kv, pos0, pos0_dev, n_split, scale,
                       n_split == 1 ? out : nullptr, q8, d8);
    return TF_LAUNCH_RESULT();
}

// ---------------------------------------------------------------- C ABI

extern "C" int tf_kv8_write(const void* k, const void* v, int src_type, int src_stride, int8_t* k8,
                            float* kd, int8_t* v8, float* vd, int n, int pos0, const int* pos0_dev,
                            int n_tok, tf_stream_t stream) {
    TF_CHECK_ARG(k && v && k8 && kd && v8 && vd && n > 0 && n % 32 == 0 && n_tok > 0);
    TF_CHECK_ARG((src_type == TF_KV_F32 || src_type == TF_KV_F16) && src_stride >= n);
    TF_CHECK_ARG(pos0_dev || (pos0 >= 0 && pos0 <= INT32_MAX - n_tok));
    const size_t count = (size_t)n_tok * n;
    const bool f16 = src_type == TF_KV_F16;
    const int el = f16 ? 2 : 4;
    const bool vec = (((uintptr_t)k | (uintptr_t)v) & 15) == 0 && (long long)src_stride * el % 16 == 0 &&
                     (((uintptr_t)k8 | (uintptr_t)v8) & 7) == 0;
    const int per = 256 * (vec ? 16 / el : 1);
    TF_CHECK_ARG((count + per - 1) / per <= UINT32_MAX / 256);
    const dim3 grid((unsigned)((count + per - 1) / per), 2);
    const TfKv8Rows a{k, v, src_stride, k8, v8, kd, vd, n, pos0, pos0_dev, count};
    auto go = [&](auto kern) {
        hipLaunchKernelGGL(kern, grid, dim3(256), 0, tf_stream(stream), a);
        return TF_LAUNCH_RESULT();
    };
    if (f16) return vec ? go(tf_kv8_write_kernel<true, true>) : go(tf_kv8_write_kernel<true, false>);
    return vec ? go(tf_kv8_write_kernel<false, true>) : go(tf_kv8_write_kernel<false, false>);
}

extern "C" int tf_kv8_read(const int8_t* k8, const float* kd, const int8_t* v8, const float* vd,
                           void* k, void* v, int dst_type, int n, int row0, int n_rows,
                           tf_stream_t stream) {
    TF_CHECK_ARG(k && v && k8 && kd && v8 && vd && n > 0 && n % 32 == 0 && n_rows > 0 && row0 >= 0);
    TF_CHECK_ARG(dst_type == TF_KV_F32 || dst_type == TF_KV_F16);
    const size_t first = (size_t)row0 * n, count = (size_t)n_rows * n;
    const bool f16 = dst_type == TF_KV_F16;
    const bool vec = (((uintptr_t)k | (uintptr_t)v) & 15) == 0 &&
                     (((uintptr_t)k8 | (uintptr_t)v8) & 7) == 0;
    const int per = 256 * (vec ? (f16 ? 8 : 4) : 1);
    TF_CHECK_ARG((count + per - 1) / per <= UINT32_MAX / 256);
    const dim3 grid((unsigned)((count + per - 1) / per), 2);
    auto go = [&](auto kern) {
        hipLaunchKernelGGL(kern, grid, dim3(256), 0, tf_stream(stream), k8, kd, v8, vd, k, v, first,
                           count);
        return TF_LAUNCH_RESULT();
    };
    if (f16) return vec ? go(tf_kv8_read_kernel<true, true>) : go(tf_kv8_read_kernel<true, false>);
    return vec ? go(tf_kv8_read_kernel<false, true>) : go(tf_kv8_read_kernel<false, false>);
}

// One split (and one launch) where it gives each wave at most one tile: 256 tokens
// of 14/2 heads of 64 take 6.0 us against 7.1 in 8 splits, of 16/2 heads of 128 8.7
// against 8.5.  Past that one for every 64 tokens, in eights for the XCDs, while the
// workgroups fit the CUs at once (a second one has no LDS beside the first): 5001
// tokens of 14/2 heads of 64 8.3 us in 64, 11 in 8; 131072 of 28/4 heads of 128 54 us
// in 32, 40 in 64, 50 in 128.
extern "C" int tf_flash_decode_kv8_n_split(int n_kv, int head_dim, int max_seq) {
    if (n_kv <= 0 || max_seq <= (head_dim == 256 ? TfKv8<256>::W : TfKv8<128>::W) * TfKv8<128>::T)
        return 1;
    const int fit = tf_device_cus() / n_kv;
    if (fit < 8) return fit > 0 ? fit : 1;
    const int want = ((max_seq - 1) / 512 + 1) * 8;
    return want < fit ? want : fit / 8 * 8;
}

extern "C" int tf_flash_decode_kv8(const float* q, const int8_t* k8, const float* kd,
                                   const int8_t* v8, const float* vd, float* partial, float* out,
                                   int8_t* q8, float* d8, int n_head, int n_kv, int head_dim,
                                   int pos0, const int* pos0_dev, int n_split, float scale,
                                   tf_stream_t stream) {
    TF_CHECK_ARG(q && k8 && kd && v8 && vd && partial && out && ((q8 == nullptr) == (d8 == nullptr)));
    TF_CHECK_ARG(n_head > 0 && n_kv > 0 && n_head % n_kv == 0 && n_head / n_kv <= 16);
    TF_CHECK_ARG(n_kv <= 65535 && n_split >= 1 && n_split <= 1024 && (pos0_dev || (pos0 >= 0 && pos0 < INT32_MAX - 1024)));
    auto go = [&](auto fn) {
        return fn(q, k8, kd, v8, vd, partial, n_head, n_kv, pos0, pos0_dev, n_split, scale, out, q8,
                  d8, stream);
    };
    int rc;
    switch (head_dim) {
    case 64: rc = go(tf_flash_kv8_launch<64>); break;
    case 128: rc = go(tf_flash_kv8_launch<128>); break;
    case 256: rc = go(tf_flash_kv8_launch<256>); break;
    default: return (int)hipErrorInvalidValue;
    }
    if (rc || n_split == 1) return rc;
    return q8 ? tf_flash_decode_reduce_q8(partial, out, q8, d8, n_head, head_dim, n_split, stream)
              : tf_flash_decode_reduce(partial, out, n_head, head_dim, n_split, 1, stream);
}
