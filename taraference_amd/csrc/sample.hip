// A token a row drawn from its logits: temperature, top-k, top-p and min-p,
// then the inverse of the kept distribution's running sum at a given u.
//
//   z_i = l_i / T, w_i = exp(z_i - max z)                       (64 bits)
//   in the order of falling l, ties by rising index:
//     top-k   the first k;
//     top-p   of these the shortest run whose sum reaches p of theirs;
//     min-p   of these the ones with w >= min_p (the largest has w = 1);
//   token = the first kept index, in vocabulary order, at which the running
//   sum of kept w exceeds u times their sum.
// NaN and -inf are never drawn, +inf takes all the weight there is; T <= 0
// takes the largest (lowest index); a row with nothing to draw gives 0.
//
// Every filter keeps a run from the front of one order, so what is kept is
// named by its last element: a cut (key, number of elements kept that tie with
// it, by index).  The cut is found by radix selection over the 32 bits of the
// ordered logit, 8 bits a pass, by count for top-k and by weight for top-p;
// no sort.  Weights are added as integers of 2^-44 of the largest, so that a
// sum has one value whatever the order in which its atomics land.
#include <math.h>

#include "tf_common.hpp"
#include "tf_host.hpp"

namespace {

typedef unsigned long long u64;

// Ordered bits of a logit: NaN lowest, -0 as +0.
__device__ __forceinline__ uint32_t order_key(float l) {
    if (l != l) return 0;
    if (l == 0.f) l = 0.f;
    const uint32_t u = __float_as_uint(l);
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

struct SampleArgs {
    const float* logits;
    long long stride;
    int n;
    const float* temperature;
    const int* top_k;
    const float* top_p;
    const float* min_p;
    const float* u;
    int* out;
};

// What turns a logit of a row into its weight.
struct RowWeight {
    double t, z_max;
    bool inf;
    __device__ double operator()(float l) const {
        if (inf) return l == INFINITY ? 1.0 : 0.0;
        return l > -INFINITY ? exp((double)l / t - z_max) : 0.0;  // NaN: 0
    }
};

constexpr int kThreads = 1024, kWaves = kThreads / 64;
constexpr double kUnit = 0x1p44;  // integer weights; n < 2^19 keeps their sum below 2^63

struct Cut {
    uint32_t key;  // the last element's
    int ties;      // elements with this key that are kept, lowest indices first
};

__device__ __forceinline__ double wave_sum(double v) {
    for (int off = 32; off; off >>= 1) v += __shfl_xor(v, off, 64);
    return v;
}

// The cut of the element at which the running total, in falling order, reaches
// `target` (1 <= target <= the total): of counts, or of integer weights.
// Elements outside `within` are not there.
template <bool WEIGHTS>
__device__ Cut radix_cut(const float* x, int n, const RowWeight& w, Cut within, u64 target,
                         u64* hist /* 256, LDS */, u64* share /* 2, LDS */) {
    const int tid = threadIdx.x;
    uint32_t prefix = 0;
    u64 each = 1, tied = 0;
    for (int shift = 24; shift >= 0; shift -= 8) {
        if (tid < 256) hist[tid] = 0;
        __syncthreads();
        const uint32_t mask = shift == 24 ? 0u : ~0u << (shift + 8);
        for (int i = tid; i < n; i += kThreads) {
            const uint32_t key = order_key(x[i]);
            if ((key & mask) != prefix || key < within.key) continue;
            // the elements that tie with `within` count for what is kept of them: below
            if (key == within.key) continue;
            atomicAdd(&hist[(key >> shift) & 255],
                      WEIGHTS ? (u64)(w(x[i]) * kUnit + 0.5) : (u64)1);
        }
        __syncthreads();
        if (tid == 0) {
            if (within.ties > 0 && (within.key & mask) == prefix) {
                const float l = __uint_as_float((within.key & 0x80000000u) ? within.key ^ 0x80000000u
                                                                            : ~within.key);
                hist[(within.key >> shift) & 255] +=
                    (u64)within.ties * (WEIGHTS ? (u64)(w(l) * kUnit + 0.5) : (u64)1);
            }
            int b = 255;
            while (b > 0 && hist[b] < target) target -= hist[b--];
            share[0] = target;
            share[1] = (u64)b;
        }
        __syncthreads();
        target = share[0];
        prefix |= (uint32_t)share[1] << shift;
        tied = hist[share[1]];
        __syncthreads();
    }
    if (WEIGHTS) {
        const float l = __uint_as_float((prefix & 0x80000000u) ? prefix ^ 0x80000000u : ~prefix);
        each = (u64)(w(l) * kUnit + 0.5);
    }
    // the first tie that reaches the target; a weight that rounds to nothing keeps them all
    u64 need = each ? (target + each - 1) / each : (u64)n;
    if (need < 1) need = 1;
    if (need > (u64)n) need = (u64)n;
    (void)tied;
    return {prefix, (int)need};
}

__global__ __launch_bounds__(kThreads) void tf_sample_row_kernel(SampleArgs a) {
    __shared__ u64 hist[256], share[2];
    __shared__ double wave_w[kWaves], found_w;
    __shared__ int wave_n[kWaves], first_max, answer;
    const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const float* x = a.logits + (size_t)row * a.stride;
    const int n = a.n;

    // the largest logit, and the lowest index that has it
    uint32_t top = 0;
    for (int i = tid; i < n; i += kThreads) top = max(top, order_key(x[i]));
    for (int off = 32; off; off >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, off, 64));
    if (lane == 0) wave_n[wave] = (int)top;
    if (tid == 0) first_max = n, answer = -1;
    __syncthreads();
    for (int i = 0; i < kWaves; i++) top = max(top, (uint32_t)wave_n[i]);
    for (int i = tid; i < n; i += kThreads)
        if (order_key(x[i]) == top) {
            atomicMin(&first_max, i);
            break;
        }
    __syncthreads();
    const float l_max = __uint_as_float((top & 0x80000000u) ? top ^ 0x80000000u : ~top);
    const float temp = a.temperature ? a.temperature[row] : 1.f;
    if (top <= 0x007fffffu) {  // all NaN or -inf
        if (tid == 0) a.out[row] = 0;
        return;
    }
    if (!(temp > 0.f)) {
        if (tid == 0) a.out[row] = first_max;
        return;
    }
    RowWeight w;
    w.t = (double)temp;
    w.inf = l_max == INFINITY;
    w.z_max = (double)l_max / w.t;

    Cut cut{0u, n};  // everything
    const int k = a.top_k ? a.top_k[row] : 0;
    if (k > 0 && k < n) cut = radix_cut<false>(x, n, w, cut, (u64)k, hist, share);
    const float p = a.top_p ? a.top_p[row] : 1.f;
    if (p < 1.f) {
        // the sum of what top-k keeps
        if (tid == 0) share[0] = 0;
        __syncthreads();
        u64 mine = 0;
        for (int i = tid; i < n; i += kThreads)
            if (order_key(x[i]) > cut.key) mine += (u64)(w(x[i]) * kUnit + 0.5);
        atomicAdd(&share[0], mine);
        __syncthreads();
        u64 total = share[0];
        if (cut.key > 0) {
            const float l =
                __uint_as_float((cut.key & 0x80000000u) ? cut.key ^ 0x80000000u : ~cut.key);
            total += (u64)cut.ties * (u64)(w(l) * kUnit + 0.5);
        }
        __syncthreads();
        u64 target = p > 0.f ? (u64)ceil((double)p * (double)total) : 1;
        target = target < 1 ? 1 : target > total ? total : target;
        cut = radix_cut<true>(x, n, w, cut, target, hist, share);
    }
    const float mp = a.min_p ? a.min_p[row] : 0.f;
    const double min_w = mp > 0.f ? fmin((double)mp, 1.0) : 0.0;  // NaN: off

    // A wave takes a run of indices; its kept ties, then its kept sum.
    const int run = ((n + kWaves - 1) / kWaves + 63) / 64 * 64;
    const int i0 = min(wave * run, n), i1 = min(i0 + run, n);
    int ties = 0;
    for (int i = i0 + lane; i < i1; i += 64) ties += order_key(x[i]) == cut.key;
    for (int off = 32; off; off >>= 1) ties += __shfl_xor(ties, off, 64);
    __syncthreads();
    if (lane == 0) wave_n[wave] = ties;
    __syncthreads();
    int before = 0;
    for (int i = 0; i < wave; i++) before += wave_n[i];
    // walks the run 64 indices at a time: f(i, kept weight of the lane)
    auto walk = [&](auto f) {
        int seen = before;
        for (int b = i0; b < i1; b += 64) {
            const int i = b + lane;
            const float l = i < i1 ? x[i] : -INFINITY;
            const uint32_t key = order_key(l);
            const u64 tie = __ballot(i < i1 && key == cut.key);
            const int rank = seen + __popcll(tie & ((1ull << lane) - 1));
            seen += __popcll(tie);
            double v = 0.0;
            if (i < i1 && (key > cut.key || (key == cut.key && rank < cut.ties))) {
                v = w(l);
                if (!(v >= min_w)) v = 0.0;
            }
            if (f(i, v)) return;
        }
    };
    double sum = 0.0;
    walk([&](int, double v) {
        sum += v;
        return false;
    });
    sum = wave_sum(sum);
    if (lane == 0) wave_w[wave] = sum;
    __syncthreads();
    double total = 0.0, ahead = 0.0;
    int last = 0;
    for (int i = 0; i < kWaves; i++) {
        if (i < wave) ahead += wave_w[i];
        total += wave_w[i];
        if (wave_w[i] > 0.0) last = i;
    }
    double u = a.u ? (double)a.u[row] : 0.0;
    u = u > 0.0 ? u : 0.0;  // NaN: 0
    const double target = u * total;
    // the wave in whose run the sum passes the target, or the last one that has any
    const bool here = (ahead <= target && ahead + sum > target) || (wave == last && target >= total);
    if (here) {
        double at = ahead;
        int best = -1;
        walk([&](int i, double v) {
            double c = v;
            for (int off = 1; off < 64; off <<= 1) {
                const double o = __shfl_up(c, off, 64);
                if (lane >= off) c += o;
            }
            c += at;
            const u64 over = __ballot(v > 0.0 && c > target);
            const u64 any = __ballot(v > 0.0);
            if (over) {
                best = i - lane + __builtin_ctzll(over);
                return true;
            }
            if (any) best = i - lane + 63 - __builtin_clzll(any);
            at = __shfl(c, 63, 64);
            return false;
        });
        if (lane == 0 && best >= 0) atomicMax(&answer, best);
    }
    __syncthreads();
    if (tid == 0) a.out[row] = answer >= 0 ? answer : first_max;
}

}  // namespace

extern "C" long long tf_sample_ws_bytes(int n_rows, int n_vocab) {
    return n_rows > 0 && n_vocab > 0 && n_vocab < (1 << 19) ? 256LL * n_rows : -1;
}

extern "C" int tf_sample(const float* logits, int n_rows, int n_vocab, int row_stride,
                         const float* temperature, const int* top_k, const float* top_p,
                         const float* min_p, const float* u, int* out_idx, void* ws,
                         long long ws_bytes, tf_stream_t stream) {
    TF_CHECK_ARG(logits && u && out_idx && ws && n_rows > 0 && n_vocab > 0);
    TF_CHECK_ARG(n_vocab < (1 << 19) && row_stride >= n_vocab);
    TF_CHECK_ARG(ws_bytes >= tf_sample_ws_bytes(n_rows, n_vocab) && ((uintptr_t)ws & 15) == 0);
    const SampleArgs a{logits, row_stride, n_vocab, temperature, top_k, top_p, min_p, u, out_idx};
    hipLaunchKernelGGL(tf_sample_row_kernel, dim3(n_rows), dim3(kThreads), 0, tf_stream(stream), a);
    return TF_LAUNCH_RESULT();
}
