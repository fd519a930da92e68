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
// Weights and their sums are f64: with f32 sums of 10^5 weights the token
// would depend on the order of addition for one u in a few thousand.  Where
// sums are formed by atomics, weights are integers of 2^-46 of the largest (or
// 2^-44, for a whole row), so that a sum has one value whatever the order.
//
// Every filter keeps a run from the front of one order, so what is kept is
// named by its last element, and no row is sorted.  Three launches, rows cut
// into chunks so that one row has the loads of many CUs:
//   1. stats: a chunk's largest logit, and a histogram of counts (top-k) and
//      weights (top-p) over bins of 1/8 of z or less below it (no filter: its sum of
//      weights);
//   2. gather: each chunk's workgroup adds the row's histograms, finds the bins
//      in which the cuts of top-k, top-p and min-p lie, and lists its elements of
//      those bins; the weights of the bins before them are kept for sure, and
//      their sums come from the histograms, or without top-p, where few are kept,
//      from the elements;
//   3. draw: a workgroup a row takes the cuts from the list, finds the segments in
//      which the running sum passes u, and walks those.
// Without top-k, top-p and min-p the second launch is left out.  A row whose cut lies
// among more elements than the list holds (equal logits by the thousand), whose logits
// the bins cannot hold (an infinite one, T below 1e-37), or whose u is below 2^-20, is
// selected by radix passes over the row itself in the third launch: the same cut, found by
// one workgroup (151936 equal logits with top-p 317 us, u = 0 with no filter 65).  Bins of
// the row's own size keep others from there: logits within 0.1 of each other, or T = 3,
// take the time of any row.
//
// One row of 151936 with all filters: 8 + 8 + 4.7 us, without filters 5.5 + 4.7; bound by
// chains of loads and barriers (19 workgroups, then one).  64 rows with top-p: 23.2 + 20.0
// + 14.7 us.  There the first launch has its VALU busy for 16 us (64 instructions for an
// element's bin and weight); without exponentials it took 6.5 less, without the atomics 1.
// 1216 workgroups run in two rounds of three a CU: more a CU would spill registers, and
// cost 2 us.
#include <math.h>

#include "tf_common.hpp"
#include "tf_host.hpp"

namespace {

typedef unsigned long long u64;

// 512 bins of 1/16: one row's first launch 11 us instead of 7, by LDS atomics and scans.
constexpr int kBins = 256;          // of 1/8 of z: 32 below a chunk's largest, the last open
constexpr int kMaxFine = 16;        // finer ones, by powers of two, where a chunk's spread is less,
constexpr int kMinFine = -240;      // and wider where their numbers would pass 2^21
constexpr float kNoWeight = 5560.f; // bins below the largest from which exp2_neg() gives 0
constexpr float kPerZ = 8.f;
constexpr int kList = 8192;         // elements of a row's list, and
constexpr int kChunkList = 2048;    // of a chunk's part of it, three quarters of its workspace
constexpr int kChunkThreads = 512, kChunkWaves = kChunkThreads / 64;
constexpr int kBlock = 16 * kChunkThreads;  // elements of a chunk: its workgroup's registers
constexpr int kMaxVocab = 1 << 19;
constexpr int kMaxChunks = kMaxVocab / kBlock;  // 64
constexpr int kSegment = 1024;                  // elements of a wave: what the draw walks
constexpr int kMaxSegments = kMaxVocab / kSegment;
constexpr int kRowThreads = 1024, kRowWaves = kRowThreads / 64;
// Integer weights: a chunk has 2^13 elements, a row fewer than 2^19, so that their sums
// stay below 2^63.
constexpr double kChunkUnit = 0x1p46, kRowUnit = 0x1p44;

// Ordered bits of a logit: NaN lowest, -0 as +0.
__device__ __forceinline__ uint32_t order_key(float l) {
    if (l != l) return 0;
    if (l == 0.f) l = 0.f;
    const uint32_t u = __float_as_uint(l);
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float key_logit(uint32_t k) {
    return __uint_as_float((k & 0x80000000u) ? k ^ 0x80000000u : ~k);
}
constexpr uint32_t kKeyMinusInf = 0x007fffffu;

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
    int chunks;  // of a row
    uint8_t* ws;
    long long row_bytes;  // of the workspace
};

// A row's workspace.
struct RowInfo {
    int lo, hi, k_bin;          // listed bins: lo .. hi, and k_bin
    int k_before;               // elements in bins before k_bin
    u64 w_before_k, w_before_lo, w_all;  // weights in bins before k_bin, before lo, in all
    int cut;                    // 0: no cut, kept is what min-p keeps; 1: the list; 2: the row itself
    int use_k;                  // top-k cuts something
    int fine;                   // the row's bins are 2^-fine of the widest
    int wide;                   // segments' sums are of kWide, in the first one's place
};
struct ChunkStat {
    float top;    // the largest logit
    int index;    // its lowest index (T <= 0 only)
    int listed;   // elements of its list
    int fine;     // its bins are 2^-fine of the widest
};
__device__ __forceinline__ RowInfo* row_info(const SampleArgs& a, int row) {
    return reinterpret_cast<RowInfo*>(a.ws + row * a.row_bytes);
}
__device__ __forceinline__ ChunkStat* row_stats(const SampleArgs& a, int row) {
    return reinterpret_cast<ChunkStat*>(a.ws + row * a.row_bytes + 128);
}
// Of each segment (or kWide): the sum of its weights, of its chunk's largest (no filter;
// f64), or of the row's, of what is kept for sure (kRowUnit).
__device__ __forceinline__ u64* segment_sums(const SampleArgs& a, int row) {
    return reinterpret_cast<u64*>(row_stats(a, row) + kMaxChunks);
}
// Parts of a chunk whose weights are told apart.  Of four the draw would walk half as
// much (1.3 us less at 64 rows), but the first launch form and store more (2.0 us).
constexpr int kParts = 2;
constexpr int kWide = kBlock / kSegment / kParts;  // segments of a part
constexpr int kChunkWords = kChunkList + (1 + kParts) * kBins;
__device__ __forceinline__ u64* chunk_list(const SampleArgs& a, int row, int c) {
    return segment_sums(a, row) + kMaxSegments + (size_t)c * kChunkWords;
}
// Its histogram as totals up to each bin: counts, then the weights (kChunkUnit) of its
// first part and of all.
__device__ __forceinline__ double* chunk_totals(const SampleArgs& a, int row, int c) {
    return reinterpret_cast<double*>(chunk_list(a, row, c) + kChunkList);
}
static_assert(sizeof(RowInfo) <= 128 && sizeof(ChunkStat) == 16, "the workspace's layout");

struct Settings {
    float temp;
    bool greedy, use_k, use_p, bad;
    int k;
    float p;
    double min_w;
    float per_l;  // bins a unit of logit
    __device__ bool filtered() const { return use_k || use_p; }
    __device__ bool plain() const { return !use_k && !use_p && !(min_w > 0.0); }
};
// A row's value of a setting, or `off`: one value a workgroup, read by a scalar load, which
// waits for no vector load, and branches on it are scalar too.
template <class T>
__device__ __forceinline__ T scalar_at(const T* p, int row, T off) {
    typedef const __attribute__((address_space(4))) T Const;
    return p ? ((Const*)(uintptr_t)p)[row] : off;
}
__device__ __forceinline__ Settings settings(const SampleArgs& a, int row) {
    auto uni = [](float v) { return tf_readlane(v, 0); };
    Settings s;
    s.temp = uni(scalar_at(a.temperature, row, 1.f));
    s.greedy = !(s.temp > 0.f);
    s.k = __builtin_amdgcn_readfirstlane(scalar_at(a.top_k, row, 0));
    s.use_k = s.k > 0 && s.k < a.n;
    s.p = uni(scalar_at(a.top_p, row, 1.f));
    s.use_p = s.p < 1.f;
    const float m = uni(scalar_at(a.min_p, row, 0.f));
    s.min_w = m > 0.f ? fmin((double)m, 1.0) : 0.0;
    s.per_l = uni(kPerZ / s.temp);
    s.bad = !(s.temp >= 1e-37f);
    return s;
}
// Whether the bins can hold a row with this largest logit: their numbers are to be exact
// floats.
__device__ __forceinline__ bool no_bins(const Settings& s, float l_max) {
    return s.bad || !(fabsf(l_max) * s.per_l < 0x1p22f);
}
// The bin of a logit, counted from that of `base`; both by the same monotone product.
__device__ __forceinline__ float bin_of(float l, float per_l) { return floorf(l * per_l); }
__device__ __forceinline__ int bin_below(float base, float b) {
    return (int)fminf(fmaxf(base - b, 0.f), (float)(kBins - 1));
}

// 2^y for y <= 0, to 2^-51: y is a multiple of 1/32 (read off the low bits of y plus
// 1.5 * 2^47) and a rest below 1/64, whose series ends at the 6th power (the next term
// is 2^-58), times 2^(j/32) from a table and the exponent.  NaN and what lies below
// 2^-1000 give 0.  In place of exp(), which a row would call for every token, it took 64
// rows' first launch from 41 to 25 us.
__constant__ double kExp2Table[32] = {
    1, 1.0218971486541166, 1.0442737824274138, 1.0671404006768237,
    1.0905077326652577, 1.1143867425958924, 1.1387886347566916, 1.1637248587775775,
    1.189207115002721, 1.215247359980469, 1.241857812073484, 1.2690509571917332,
    1.2968395546510096, 1.3252366431597413, 1.3542555469368927, 1.383909881963832,
    1.4142135623730951, 1.4451808069770467, 1.4768261459394993, 1.5091644275934228,
    1.5422108254079407, 1.5759808451078865, 1.6104903319492543, 1.6457554781539649,
    1.681792830507429, 1.7186192981224779, 1.7562521603732995, 1.7947090750031072,
    1.8340080864093424, 1.8741676341103, 1.9152065613971474, 1.9571441241754002};
__device__ __forceinline__ void fill_exp2(double* table) {
    if (threadIdx.x < 32) table[threadIdx.x] = kExp2Table[threadIdx.x];
}
__device__ __forceinline__ double exp2_neg(double y, const double* table) {
    constexpr double kShift = 0x1.8p47, ln2 = 0.69314718055994530942;
    constexpr double c2 = ln2 * ln2 / 2, c3 = c2 * ln2 / 3, c4 = c3 * ln2 / 4, c5 = c4 * ln2 / 5,
                     c6 = c5 * ln2 / 6;
    const double t = y + kShift;
    const int k = (int)(uint32_t)__builtin_bit_cast(u64, t);
    const double f = y - (t - kShift);
    double r = c6;
    r = fma(r, f, c5);
    r = fma(r, f, c4);
    r = fma(r, f, c3);
    r = fma(r, f, c2);
    r = fma(r, f, ln2);
    r = fma(r, f, 1.0);
    r *= table[k & 31];
    const u64 bits = __builtin_bit_cast(u64, r) + ((u64)(uint32_t)(k >> 5 << 20) << 32);
    return y >= -1000.0 ? __builtin_bit_cast(double, bits) : 0.0;
}

// The running sum at which top-p is reached: p of a sum of weights, at least the first.
__device__ __forceinline__ u64 p_goal(const Settings& s, u64 all) {
    const double goal = s.p > 0.f ? ceil((double)s.p * (double)all) : 0.0;
    return goal >= 1.0 ? (u64)goal : 1;
}

// What turns a logit of a row into its weight: exp((l - l_max) / T).
struct RowWeight {
    const double* table;
    double per_t, l_max;  // per_t: powers of two a unit of logit
    bool inf;
    __device__ RowWeight(const double* table_, float temp, float l_max_) {
        table = table_;
        per_t = 1.44269504088896340736 / (double)temp;
        inf = l_max_ == INFINITY;
        l_max = (double)l_max_;
    }
    __device__ double operator()(float l) const {
        if (inf) return l == INFINITY ? 1.0 : 0.0;
        // T = inf: -inf times 0 is NaN and gives 0
        return exp2_neg(((double)l - l_max) * per_t, table);
    }
};
// The nearest integer to w / 2^-46 (2^-44) for w in [0, 1]: the low bits of w plus the
// power of two with that last bit.
__device__ __forceinline__ u64 chunk_units(double w) {
    return __builtin_bit_cast(u64, w + 64.0) - __builtin_bit_cast(u64, 64.0);
}
__device__ __forceinline__ u64 row_units(double w) {
    return __builtin_bit_cast(u64, w + 256.0) - __builtin_bit_cast(u64, 256.0);
}

// Inclusive sum over the wave's lanes, in DPP row shifts and broadcasts: a tenth of
// the latency of six exchanges through LDS.
template <int CTRL, int ROWS, class T>
__device__ __forceinline__ T dpp_or_0(T v) {
    if constexpr (sizeof(T) == 4) {
        return __builtin_bit_cast(T, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL,
                                                                 ROWS, 0xF, false));
    } else {
        const u64 b = __builtin_bit_cast(u64, v);
        const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)b, CTRL, ROWS, 0xF, false);
        const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(b >> 32), CTRL, ROWS, 0xF, false);
        return __builtin_bit_cast(T, (u64)hi << 32 | lo);
    }
}
template <class T>
__device__ __forceinline__ T wave_scan(T v) {
    v += dpp_or_0<0x111, 0xF>(v);  // row_shr 1, 2, 4, 8
    v += dpp_or_0<0x112, 0xF>(v);
    v += dpp_or_0<0x114, 0xF>(v);
    v += dpp_or_0<0x118, 0xF>(v);
    v += dpp_or_0<0x142, 0xA>(v);  // lane 15 of a row to the next row, of rows 1 and 3
    v += dpp_or_0<0x143, 0xC>(v);  // lane 31 to rows 2 and 3
    return v;
}
template <class T>
__device__ __forceinline__ T lane_value(T v, int lane) {
    if constexpr (sizeof(T) == 4) {
        return __builtin_bit_cast(T, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), lane));
    } else {
        const u64 b = __builtin_bit_cast(u64, v);
        const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)b, lane);
        const uint32_t hi = __builtin_amdgcn_readlane((int)(b >> 32), lane);
        return __builtin_bit_cast(T, (u64)hi << 32 | lo);
    }
}
template <class T>
__device__ __forceinline__ T wave_sum(T v) {
    return lane_value(wave_scan(v), 63);
}
__device__ __forceinline__ uint32_t wave_max_u32(uint32_t v) {
    v = max(v, dpp_or_0<0x111, 0xF>(v));
    v = max(v, dpp_or_0<0x112, 0xF>(v));
    v = max(v, dpp_or_0<0x114, 0xF>(v));
    v = max(v, dpp_or_0<0x118, 0xF>(v));
    v = max(v, dpp_or_0<0x142, 0xA>(v));
    v = max(v, dpp_or_0<0x143, 0xC>(v));
    return lane_value(v, 63);
}

// A block's elements: a wave holds a segment, a lane index(e) = i0 + 1024 wave + 256 (e
// / 4) + 4 lane + e % 4; past `end`: -inf.
__device__ __forceinline__ int block_index(int i0, int e) {
    return i0 + kSegment * (int)(threadIdx.x >> 6) + 256 * (e >> 2) + 4 * (int)(threadIdx.x & 63) +
           (e & 3);
}
__device__ __forceinline__ void load_block(const float* x, int i0, int end, float (&v)[16]) {
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const int i = block_index(i0, 4 * j);
        if (i + 3 < end) {
            const tf_u32x4 b = tf_ld16_a4(x + i);
#pragma unroll
            for (int e = 0; e < 4; e++) v[4 * j + e] = __uint_as_float(b[e]);
        } else {
#pragma unroll
            for (int e = 0; e < 4; e++) v[4 * j + e] = i + e < end ? x[i + e] : -INFINITY;
        }
    }
}

// Four elements at a time, the others moved down behind them: f(j, v[0 .. 3]) for
// elements 4 j ..  A quarter of the code of sixteen in a row, for little launches that
// find the instruction cache cold; where the body is short the moves would cost more.
template <class F>
__device__ __forceinline__ void each_four(float (&v)[16], F f) {
#pragma unroll 1
    for (int j = 0; j < 4; j++) {
        f(j);
        const float a[4] = {v[0], v[1], v[2], v[3]};
#pragma unroll
        for (int i = 0; i < 12; i++) v[i] = v[i + 4];
#pragma unroll
        for (int i = 0; i < 4; i++) v[12 + i] = a[i];
    }
}

__global__ __launch_bounds__(kChunkThreads, 6) void tf_sample_stats_kernel(SampleArgs a) {
    // several histograms, by lane (weights: and by part): half of a wave's elements may
    // share a bin.  A wave's neighbouring bins lie in neighbouring banks, those of its other
    // copies half of the banks further.
    __shared__ u64 weight[2 * kParts][kBins + 16];
    __shared__ uint32_t count[4][kBins + 16];
    __shared__ double table[32];
    __shared__ u64 totals[kParts][kChunkWaves];
    __shared__ float part[kChunkWaves], part_low[kChunkWaves];
    __shared__ int first;
    const int row = blockIdx.x / a.chunks, c = blockIdx.x - row * a.chunks;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const float* x = a.logits + (size_t)row * a.stride;
    const int i0 = c * kBlock, end = min(i0 + kBlock, a.n);
    float v[16];
    load_block(x, i0, end, v);
    const Settings s = settings(a, row);
    fill_exp2(table);
    for (int i = tid; i < 4 * (kBins + 16); i += kChunkThreads) count[0][i] = 0;
    for (int i = tid; i < 2 * kParts * (kBins + 16); i += kChunkThreads) weight[0][i] = 0;
    if (tid == 0) first = a.n;
    float top = -INFINITY;  // fmaxf passes NaN by
#pragma unroll
    for (int e = 0; e < 16; e++) top = fmaxf(top, v[e]);
    top = tf_wave_max(top);
    if (lane == 0) part[wave] = top;
    __syncthreads();
    for (int i = 0; i < kChunkWaves; i++) top = fmaxf(top, part[i]);
    ChunkStat* stat = row_stats(a, row) + c;
    if (tid == 0) stat->top = top;
    const bool empty = !(top > -INFINITY);
    if (s.greedy) {
        for (int i = i0 + tid; i < end; i += kChunkThreads)
            if (x[i] == top) {
                atomicMin(&first, i);
                break;
            }
        __syncthreads();
        if (tid == 0) stat->index = first;
        return;
    }
    if (!s.filtered() && !s.plain()) return;
    const RowWeight w(table, s.temp, top);
    int fine = 0;
    if (s.filtered() && !empty && !s.bad) {
        // the finest bins that hold all elements within 32 of the largest
        float low = top;
        const float far = top - 254.f / kPerZ * s.temp;
#pragma unroll
        for (int e = 0; e < 16; e++) low = fminf(low, v[e] > far ? v[e] : top);
        low = -tf_wave_max(-low);
        if (lane == 0) part_low[wave] = low;
        __syncthreads();
        for (int i = 0; i < kChunkWaves; i++) low = fminf(low, part_low[i]);
        const float spread = fmaxf((top - low) * s.per_l, 1e-6f);
        const float at = 21.f - __log2f(fabsf(top)) - __log2f(s.per_l);
        fine = (int)floorf(fminf(__log2f(252.f / spread), fmaxf(at, (float)kMinFine)));
        fine = max(kMinFine, min(fine, kMaxFine));
        if (tid == 0) stat->fine = fine;
    }
    if (s.plain()) {
        double sum = 0.0;
        if (!empty)
            each_four(v, [&](int) {
#pragma unroll
                for (int e = 0; e < 4; e++) sum += w(v[e]);
            });
        sum = wave_sum(sum);
        const int seg = (i0 >> 10) + wave;
        if (lane == 0 && seg * kSegment < a.n)
            segment_sums(a, row)[seg] = __builtin_bit_cast(u64, sum);
        return;
    }
    if (!empty && !s.bad) {
        const float per_l = ldexpf(s.per_l, fine), base = bin_of(top, per_l);
        const float far = 1.f + ldexpf(kNoWeight, fine);
        const int copy = 2 * (wave / (kChunkWaves / kParts)) + (lane & 1);
        each_four(v, [&](int) {
#pragma unroll
            for (int e = 0; e < 4; e++) {  // -inf, NaN and what has no weight add nothing
                const float b = bin_of(v[e], per_l);
                const int bin = bin_below(base, b);
                if (s.use_k) atomicAdd(&count[lane & 3][bin], base - b <= far ? 1u : 0u);
                if (s.use_p) atomicAdd(&weight[copy][bin], chunk_units(w(v[e])));
            }
        });
    }
    __syncthreads();
    // the first half of the workgroup adds up counts, the second weights
    const int half = wave / (kChunkWaves / 2), bin = tid % kBins;
    u64 sum[kParts];
#pragma unroll
    for (int q = 0; q < kParts; q++) {
        sum[q] = q ? sum[q - 1] : 0;
        sum[q] += half ? weight[2 * q][bin] + weight[2 * q + 1][bin]
                       : count[2 * q][bin] + count[2 * q + 1][bin];
    }
#pragma unroll
    for (int q = 0; q < kParts; q++) {
        sum[q] = wave_scan(sum[q]);
        if (lane == 63) totals[q][wave] = sum[q];
    }
    __syncthreads();
    double* to = chunk_totals(a, row, c) + bin;
#pragma unroll
    for (int q = 0; q < kParts; q++) {
        for (int i = half * (kChunkWaves / 2); i < wave; i++) sum[q] += totals[q][i];
        if (half && s.use_p) to[(1 + q) * kBins] = (double)sum[q];
    }
    if (!half && s.use_k) to[0] = (double)sum[kParts - 1];
}

static_assert(kChunkThreads == 2 * kBins, "a half for counts, a half for weights");
__global__ __launch_bounds__(kChunkThreads, 6) void tf_sample_gather_kernel(SampleArgs a) {
    __shared__ u64 n_upto[kBins], w_upto[kBins];  // the row's totals up to a bin
    __shared__ double table[32];
    __shared__ float kept[kChunkWaves][kSegment];
    __shared__ int first[3], place;
    const int row = blockIdx.x / a.chunks, c = blockIdx.x - row * a.chunks;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const float* x = a.logits + (size_t)row * a.stride;
    const int i0 = c * kBlock, end = min(i0 + kBlock, a.n);
    float v[16];
    load_block(x, i0, end, v);
    Settings s = settings(a, row);
    float mine_top = -INFINITY;
    int mine_fine = kMaxFine;
    if (lane < a.chunks) mine_top = row_stats(a, row)[lane].top, mine_fine = row_stats(a, row)[lane].fine;
    // the workgroup's first half adds up the histograms' counts, the second their weights
    const int half = wave / (kChunkWaves / 2), bin = tid % kBins;
    fill_exp2(table);
    if (s.greedy || s.plain()) return;
    const float l_max = tf_wave_max(mine_top);
    if (!(l_max > -INFINITY)) return;
    RowInfo info{};
    __syncthreads();  // the table
    const RowWeight w(table, s.temp, l_max);
    // of chunk `lane`: its weights' scale, its bins' size and its largest's
    const double lane_f = mine_top > -INFINITY ? w(mine_top) * (kRowUnit / kChunkUnit) : 0.0;
    const bool any = lane_f > 0.0;
    info.fine = s.filtered() ? kMaxFine - (int)wave_max_u32(any ? kMaxFine - mine_fine : 0) : 0;
    const float lane_base = bin_of(mine_top, ldexpf(s.per_l, mine_fine));
    const float lane_step = ldexpf(1.f, mine_fine - info.fine);
    s.per_l = ldexpf(s.per_l, info.fine);
    if (s.filtered() && no_bins(s, l_max)) {
        info.cut = 2;
        if (c == 0 && tid == 0) *row_info(a, row) = info;
        return;
    }
    const float base = bin_of(l_max, s.per_l);
    // min-p's bound on the product that places an element: one above m_keep is past it and
    // one below m_drop is not, whatever the rounding of products, logarithm and sums
    float m_keep = -INFINITY, m_drop = -INFINITY;
    {
        const float m_top = l_max * s.per_l;
        const float depth = s.min_w > 0.0 ? -__log2f((float)s.min_w) * ldexpf(0.69314718f * kPerZ, info.fine)
                                          : INFINITY;
        const float margin = 0.02f + (fabsf(m_top) + depth) * 0x1p-21f;
        if (margin < INFINITY) m_keep = m_top - depth + margin, m_drop = m_top - depth - margin;
    }
    if (tid < 3) first[tid] = kBins - 1;
    if (tid == 0) place = 0;
    __syncthreads();
    int lo = kBins, hi = -1, k_bin = -1;  // min-p alone: no cut by bins
    int list_from = kBins;
    // a chunk's bin with which those up to a row's bin end (< 0: none)
    auto chunk_bin = [&](int cc, int bin) {
        if (bin == kBins - 1) return bin;
        const float at = lane_value(lane_base, cc) - (base - (float)bin) * lane_value(lane_step, cc);
        return (int)fminf(fmaxf(at, -1.f), (float)(kBins - 2));
    };
    if (s.filtered()) {
        // the row's total up to a bin: each chunk's up to the bin that lies as far below its
        // own largest, weights scaled alike; the last bin has all there is.  Sums of rising
        // terms in one order: they rise with the bin.
        double total = 0.0;
        if (half ? s.use_p : s.use_k) {
            constexpr int kAtOnce = 10;  // 20: registers spill, twice the launch's time
            const double* of = chunk_totals(a, row, 0) + kParts * kBins * half;
            for (int c0 = 0; c0 < a.chunks; c0 += kAtOnce) {
                double got[kAtOnce];
#pragma unroll
                for (int i = 0; i < kAtOnce; i++) {  // all loads at once
                    const int cc = min(c0 + i, a.chunks - 1);
                    const int from = chunk_bin(cc, bin);
                    got[i] = (of + (size_t)cc * kChunkWords)[(uint32_t)max(from, 0)];
                    if (from < 0) got[i] = 0.0;
                }
#pragma unroll
                for (int i = 0; i < kAtOnce; i++)
                    if (c0 + i < a.chunks)
                        total += got[i] * lane_value(half ? lane_f : any ? 1.0 : 0.0, c0 + i);
            }
        }
        u64* upto_of = half ? w_upto : n_upto;
        const u64 upto = (u64)(total + 0.5);
        upto_of[bin] = upto;
        __syncthreads();
        // the bin in which a running total reaches a goal; one thread's
        auto reach = [&](u64 goal, int slot) {
            if (upto >= goal && (bin == 0 || upto_of[bin - 1] < goal)) first[slot] = bin;
        };
        const bool use_k = s.use_k && n_upto[kBins - 1] > (u64)s.k;
        if (use_k && !half) reach((u64)s.k, 0);
        __syncthreads();
        info.use_k = use_k;
        if (use_k) {
            k_bin = first[0];
            info.k_before = k_bin ? (int)n_upto[k_bin - 1] : 0;
            info.w_before_k = k_bin ? w_upto[k_bin - 1] : 0;
            lo = hi = k_bin;
        }
        info.w_all = w_upto[kBins - 1];
        if (s.use_p) {
            // the goal is p of what top-k keeps: between these two until k_bin is resolved
            if (half) {
                reach(p_goal(s, use_k ? info.w_before_k : info.w_all), 1);
                reach(p_goal(s, use_k ? w_upto[k_bin] : info.w_all), 2);
            }
            __syncthreads();
            lo = first[1];
            hi = first[2];
            if (use_k) lo = min(lo, k_bin), hi = min(hi, k_bin);
        }
        if (!use_k && !s.use_p) {
            lo = kBins, hi = -1;
        } else {
            info.cut = 1;
            info.w_before_lo = lo ? w_upto[lo - 1] : 0;
            auto in_bins = [&](int b0, int b1) { return n_upto[b1] - (b0 ? n_upto[b0 - 1] : 0); };
            // the bins that min-p's bound cuts
            const int first_m = (int)fminf(fmaxf(base - floorf(m_keep), 0.f), (float)kBins);
            const bool m_first = base - floorf(m_drop) < (float)lo;
            list_from = min(lo, first_m);
            // with top-k the list's length is known here; else the draw finds it too long
            const u64 listed = in_bins(list_from, hi) + (k_bin > hi ? in_bins(k_bin, k_bin) : 0);
            if (m_first) {  // the other cuts are past it
                info.cut = 0;
                lo = kBins, hi = -1, k_bin = -1;
            } else if (listed > kList) {
                info.cut = 2;
            }
        }
    }
    // the weights of bins that are kept for sure are in the histograms, if top-p took them
    info.wide = info.cut == 1 && s.use_p;
    info.lo = lo, info.hi = hi, info.k_bin = k_bin;
    if (c == 0 && tid == 0) *row_info(a, row) = info;
    if (info.cut == 2) return;
    // the chunk's part of the list, and its weight before it
    // bins as bounds on the product that bin_of() rounds down: bin b holds base - b <= l
    // per_l < base - b + 1, the last one all below
    const float sure = lo < kBins ? base - (float)(list_from - 1) : m_drop;
    const float no_weight = base - 1.f - ldexpf(kNoWeight, info.fine);
    const float listed = hi < kBins - 1 ? base - (float)hi : no_weight;
    const float k_from = k_bin < 0 ? INFINITY : k_bin < kBins - 1 ? base - (float)k_bin : no_weight;
    const float k_to = base - (float)(k_bin - 1);
    const float low = hi >= 0 ? fminf(listed, k_from) : sure;
    const bool all = sure == -INFINITY;  // products may be NaN
    auto in_list = [&](float m) {
        return m < sure && ((hi >= 0 && m >= listed) || (m >= k_from && m < k_to));
    };
    auto put = [&](float l, int e) {  // the list has no order: places by an LDS counter
        const int to = atomicAdd(&place, 1);
        if (to < kChunkList)
            chunk_list(a, row, c)[to] = (u64)order_key(l) << 32 | (uint32_t)block_index(i0, e);
    };
    if (info.wide) {
        uint32_t which = 0;
#pragma unroll
        for (int e = 0; e < 16; e++)
            which |= v[e] > -INFINITY && in_list(v[e] * s.per_l) ? 1u << e : 0;
        for (; which; which &= which - 1) {  // few: read again
            const int e = __builtin_ctz(which);
            put(x[block_index(i0, e)], e);
        }
        if (tid < kParts) {  // a part's total is what it adds to those before it
            const double* of = chunk_totals(a, row, c) + kBins;
            const int from = list_from > 0 ? chunk_bin(c, list_from - 1) : -1;
            double w_q = 0.0;
            if (from >= 0)
                w_q = (of[tid * kBins + from] - (tid ? of[(tid - 1) * kBins + from] : 0.0)) *
                      lane_value(lane_f, c);
            u64* to = segment_sums(a, row) + c * (kBlock / kSegment) + kWide * tid;
            to[0] = (u64)(w_q + 0.5);
#pragma unroll
            for (int i = 1; i < kWide; i++) to[i] = 0;
        }
        __syncthreads();
        if (tid == 0) row_stats(a, row)[c].listed = place;
        return;
    }
    // the segment's elements that are kept for sure, side by side in LDS: few of a
    // lane's are, and a branch for each would form weights in every wave
    int n_kept = 0;
    each_four(v, [&](int j) {
        // most have nothing of the kept or listed
        const float most = fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3]));
        if (!all && !__ballot(most * s.per_l >= low)) return;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const float m = v[e] * s.per_l;
            const bool is = v[e] > -INFINITY, in = is && (all || m >= sure);
            const u64 who = __ballot(in);
            const int at = n_kept + (int)__builtin_amdgcn_mbcnt_hi(
                                        (uint32_t)(who >> 32),
                                        __builtin_amdgcn_mbcnt_lo((uint32_t)who, 0));
            if (in) kept[wave][at] = v[e];
            n_kept += __popcll(who);
            if (is && in_list(m)) put(v[e], 4 * j + e);
        }
    });
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    u64 sum = 0;
    for (int i = lane; i < n_kept; i += 64) {
        const double we = w(kept[wave][i]);
        sum += we >= s.min_w ? row_units(we) : 0;
    }
    sum = wave_sum(sum);
    const int seg = (i0 >> 10) + wave;
    if (lane == 0 && seg * kSegment < a.n) segment_sums(a, row)[seg] = sum;
    __builtin_amdgcn_wave_barrier();
    __syncthreads();
    if (tid == 0) row_stats(a, row)[c].listed = place;
}

// ------------------------------------------------------------------ the cut

struct Cut {
    uint32_t key;  // the last kept element's: kept are larger ones,
    int index;     // and equal ones up to this index
    __device__ bool keeps(uint32_t k, int i) const { return k > key || (k == key && i <= index); }
    // a cut found among what `outer` keeps: all of its equals are those that outer keeps
    __device__ void within(const Cut& outer) {
        if (key == outer.key) index = min(index, outer.index);
    }
};

// LDS of a selection.
struct Select {
    u64 hist[256];
    u64 left;
    u64 few[64];  // elements that are ranked directly
    uint32_t many[256];  // elements of each digit
    int digit, count, place;
    uint32_t least, most;
};

// The largest digit d such that the total of digits >= d reaches s.left, which
// is reduced by the total of those above it (0 if none reaches it); wave 0.
__device__ __forceinline__ void pick_digit(Select& s) {
    const int lane = threadIdx.x;
    u64 h[4], sum = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) sum += h[i] = s.hist[255 - (4 * lane + i)];
    const u64 upto = wave_scan(sum);
    const u64 left = s.left, over = __ballot(upto >= left);
    const int who = over ? __builtin_ctzll(over) : 63;
    if (lane == who) {
        u64 run = upto - sum;
        int i = 0;
        while (i < 3 && run + h[i] < left) run += h[i++];
        s.digit = 255 - (4 * lane + i);
        s.left = left - run;
    }
}

// The cut of the element at which the running total of `value`, in falling order
// of key and rising order of index, reaches `goal` (of the elements that `each`
// visits: each(f) calls f(key, index) for the thread's share).  `value(key)` is
// an element's part of the total.
template <class Each, class Value>
__device__ Cut select_cut(Select& s, u64 goal, Each each, Value value) {
    const int tid = threadIdx.x;
    auto pass = [&](auto digit_of) {  // digit_of(key, index) < 0: not among them
        __syncthreads();
        if (tid < 256) s.hist[tid] = 0;
        __syncthreads();
        each([&](uint32_t key, int index) {
            const int d = digit_of(key, index);
            if (d >= 0) atomicAdd(&s.hist[d], value(key));
        });
        __syncthreads();
        if (tid < 64) pick_digit(s);
        __syncthreads();
        return s.digit;
    };
    // all alike (a row of zeros): no passes over the key
    __syncthreads();
    if (tid == 0) s.left = goal > 0 ? goal : 1, s.least = ~0u, s.most = 0;
    __syncthreads();
    uint32_t least = ~0u, most = 0;
    each([&](uint32_t key, int) { least = min(least, key), most = max(most, key); });
    least = ~wave_max_u32(~least);
    most = wave_max_u32(most);
    if ((tid & 63) == 0) {
        atomicMin(&s.least, least);
        atomicMax(&s.most, most);
    }
    __syncthreads();
    uint32_t prefix = s.least;
    if (s.least != s.most) {
        prefix = 0;
        for (int shift = 24; shift >= 0; shift -= 8) {
            const uint32_t mask = shift == 24 ? 0u : ~0u << (shift + 8);
            prefix |= (uint32_t)pass([&](uint32_t key, int) {
                          return (key & mask) == prefix ? (int)(key >> shift & 255) : -1;
                      })
                      << shift;
        }
    }
    // equal elements share the total: how many of them, and which index is the last
    const u64 each_value = value(prefix), left = s.left;
    const u64 need = each_value ? (left + each_value - 1) / each_value : ~0ull;
    __syncthreads();
    if (tid == 0) s.hist[0] = 0;
    __syncthreads();
    u64 mine = 0;
    each([&](uint32_t key, int) { mine += key == prefix; });
    mine = wave_sum(mine);
    if (mine && (tid & 63) == 0) atomicAdd(&s.hist[0], mine);
    __syncthreads();
    if (need >= s.hist[0]) return {prefix, kMaxVocab};
    __syncthreads();
    // the need-th lowest index: digits of its complement, so that falling order is rising
    if (tid == 0) s.left = need;
    uint32_t at = 0;
    for (int shift = 16; shift >= 0; shift -= 8) {
        const uint32_t mask = ~0u << (shift + 8) & 0xffffffu;
        __syncthreads();
        if (tid < 256) s.hist[tid] = 0;
        __syncthreads();
        each([&](uint32_t key, int index) {
            const uint32_t r = ~(uint32_t)index & 0xffffffu;
            if (key != prefix || (r & mask) != at) return;
            // neighbours share their digits: one of them adds for all
            const int d = r >> shift & 255;
            const u64 here = __ballot(true);
            const bool alike = __ballot(d == __builtin_amdgcn_readfirstlane(d)) == here;
            if (!alike || (tid & 63) == __builtin_ctzll(here))
                atomicAdd(&s.hist[d], alike ? (u64)__popcll(here) : 1);
        });
        __syncthreads();
        if (tid < 64) pick_digit(s);
        __syncthreads();
        at |= (uint32_t)s.digit << shift;
    }
    return {prefix, (int)(~at & 0xffffffu)};
}

// The same for elements in LDS, of a few bins: step(key) of 0 .. 255, which rises as keys
// fall.  One pass over the steps leaves a handful, and a wave ranks up to 64 by comparing
// each with all.
template <class Each, class Value, class Step>
__device__ Cut select_near(Select& s, u64 goal, Each each, Value value, Step step) {
    const int tid = threadIdx.x, lane = tid & 63;
    if (goal < 1) goal = 1;
    if (tid < 256) s.hist[tid] = 0, s.many[tid] = 0;
    __syncthreads();
    each([&](uint32_t key, int) {
        const int d = step(key);
        atomicAdd(&s.hist[d], value(key));
        atomicAdd(&s.many[d], 1u);
    });
    __syncthreads();
    if (tid < 64) {  // the first step at which the total reaches the goal
        u64 h[4], sum = 0;
        uint32_t m[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            sum += h[i] = s.hist[4 * lane + i];
            m[i] = s.many[4 * lane + i];
        }
        const u64 upto = wave_scan(sum), over = __ballot(upto >= goal);
        // none: the goal is past them all, to which rounding may have led: the last
        const u64 has = __ballot(m[0] | m[1] | m[2] | m[3]);
        const int who = over ? __builtin_ctzll(over) : has ? 63 - __builtin_clzll(has) : 0;
        if (lane == who) {
            u64 run = upto - sum;
            int i = 0;
            if (over)
                while (i < 3 && run + h[i] < goal) run += h[i++];
            else
                for (i = 3; i > 0 && !m[i];) i--;
            s.digit = 4 * lane + i;
            s.left = over ? goal - run : ~0ull;
            s.count = m[i];
            s.place = 0;
        }
    }
    __syncthreads();
    const int digit = s.digit, count = s.count;
    if (count > 64) return select_cut(s, goal, each, value);
    each([&](uint32_t key, int index) {
        if (step(key) == digit) s.few[atomicAdd(&s.place, 1)] = (u64)key << 32 | (uint32_t)~index;
    });
    __syncthreads();
    if (tid < 64) {
        const u64 me = lane < count ? s.few[lane] : 0;
        const u64 part = lane < count ? value((uint32_t)(me >> 32)) : 0;
        u64 before = 0;
        for (int j = 0; j < count; j++) before += lane_value(me, j) > me ? lane_value(part, j) : 0;
        const u64 left = s.left;
        const u64 hit = __ballot(lane < count && before < left && before + part >= left);
        u64 last = ~0ull;
        if (!hit)
            for (int j = 0; j < count; j++) last = min(last, lane_value(me, j));
        if (lane == 0) s.few[0] = hit ? lane_value(me, __builtin_ctzll(hit)) : last;
    }
    __syncthreads();
    const u64 at = s.few[0];
    return {(uint32_t)(at >> 32), (int)~(uint32_t)at};
}

__global__ __launch_bounds__(kRowThreads) void tf_sample_draw_kernel(SampleArgs a) {
    extern __shared__ __align__(16) uint8_t lds[];
    u64* list = reinterpret_cast<u64*>(lds);                        // kList
    u64* seg_sum = list + kList;                                    // kMaxSegments
    Select& sel = *reinterpret_cast<Select*>(seg_sum + kMaxSegments);
    __shared__ double wave_w[2][kRowWaves], table[32], seg_before;
    __shared__ u64 total_w;
    __shared__ int first_at[2], last_at[2], chunk_upto[kMaxChunks];
    const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const float* x = a.logits + (size_t)row * a.stride;
    const int n = a.n;
    // everything that the workspace may hold of the row, at once
    Settings s = settings(a, row);
    ChunkStat mine_c{-INFINITY, 0, 0, 0};
    if (lane < a.chunks) mine_c = row_stats(a, row)[lane];
    RowInfo info = *row_info(a, row);
    if (s.plain()) info.cut = 0, info.wide = 0;
    // the list's length and each chunk's place in it; too long for LDS, or a chunk's for
    // its room: the row itself
    // A u below 2^-20 may fall among weights that the sums' unit of 2^-44 rounds away, or into
    // a part whose weights are all below 2^-1000: such a row takes its sums, and its cut,
    // from its logits.  Past it the rounding, 2^-26 for a whole row, is below 2^-6 of u.
    float u = tf_readlane(scalar_at(a.u, row, 0.f), 0);
    u = u > 0.f ? u : 0.f;  // NaN: 0
    const bool small = u < 0x1p-20f;
    if (small) info.cut = s.filtered() ? 2 : 0, info.wide = 0;
    int list_upto = 0, count = 0;
    if (info.cut == 1) {
        list_upto = wave_scan(mine_c.listed);
        count = lane_value(list_upto, 63);
        if (count > kList || __ballot(mine_c.listed > kChunkList)) info.cut = 2, info.wide = 0;
    }
    const int segments = (n + kSegment - 1) / kSegment;
    u64 my_seg = 0;
    if (tid < segments) my_seg = segment_sums(a, row)[tid];
    fill_exp2(table);
    const float l_max = tf_wave_max(mine_c.top);
    if (!(l_max > -INFINITY) || s.greedy) {  // nothing to draw, or nothing to choose
        const u64 has = __ballot(lane < a.chunks && mine_c.top == l_max);
        const int index = __shfl(mine_c.index, has ? __builtin_ctzll(has) : 0, 64);
        if (tid == 0) a.out[row] = l_max > -INFINITY ? index : 0;
        return;
    }
    const RowWeight w(table, s.temp, l_max);
    auto units = [&](uint32_t key) { return row_units(w(key_logit(key))); };
    auto one = [](uint32_t) { return (u64)1; };
    if (tid == 0) total_w = 0;
    if (tid < 2) first_at[tid] = INT32_MAX, last_at[tid] = -1;
    if (tid < segments) seg_sum[tid] = my_seg;
    if (tid < kMaxChunks) chunk_upto[tid] = list_upto;
    __syncthreads();

    Cut cut{0u, kMaxVocab};
    if (info.cut == 1) {
        for (int i = tid; i < count; i += kRowThreads) {
            int c = 0;  // its chunk: as many end at or before i
#pragma unroll
            for (int b = kMaxChunks / 2; b; b >>= 1)
                if (chunk_upto[c + b - 1] <= i) c += b;
            list[i] = chunk_list(a, row, c)[i - (c ? chunk_upto[c - 1] : 0)];
        }
        s.per_l = ldexpf(s.per_l, info.fine);
        const float base = bin_of(l_max, s.per_l);
        auto each = [&](auto f) {
            for (int i = tid; i < count; i += kRowThreads)
                f((uint32_t)(list[i] >> 32), (int)(uint32_t)list[i]);
        };
        auto bin = [&](uint32_t key) { return bin_below(base, bin_of(key_logit(key), s.per_l)); };
        // 256 steps over bins b0 .. b1
        auto steps = [&](int b0, int b1) {
            const float top = base - (float)(b0 - 1), per = 256.f / (float)(b1 - b0 + 1);
            return [=](uint32_t key) {
                return (int)fminf(fmaxf((top - key_logit(key) * s.per_l) * per, 0.f), 255.f);
            };
        };
        u64 kept_w = info.w_all;
        if (info.use_k) {
            auto in_k = [&](auto f) {
                each([&](uint32_t key, int i) {
                    if (bin(key) == info.k_bin) f(key, i);
                });
            };
            cut = select_near(sel, (u64)(s.k - info.k_before), in_k, one,
                              steps(info.k_bin, info.k_bin));
            if (s.use_p) {
                u64 add = 0;
                in_k([&](uint32_t key, int i) { add += cut.keeps(key, i) ? units(key) : 0; });
                add = wave_sum(add);
                if (add && lane == 0) atomicAdd(&total_w, add);
                __syncthreads();
                kept_w = info.w_before_k + total_w;
            }
        }
        if (s.use_p) {
            const u64 goal = p_goal(s, kept_w);
            const Cut k_cut = cut;
            cut = select_near(
                sel, goal > info.w_before_lo ? goal - info.w_before_lo : 1,
                [&](auto f) {
                    each([&](uint32_t key, int i) {
                        const int b = bin(key);
                        if (b >= info.lo && b <= info.hi && k_cut.keeps(key, i)) f(key, i);
                    });
                },
                units, steps(info.lo, info.hi));
            cut.within(k_cut);
        }
        // what the list adds to each segment
        each([&](uint32_t key, int i) {
            if (!cut.keeps(key, i)) return;
            const double we = w(key_logit(key));
            if (we >= s.min_w)
                atomicAdd(&seg_sum[(i / kSegment) & (info.wide ? -kWide : ~0)], row_units(we));
        });
        __syncthreads();
    } else if (info.cut == 2) {
        auto each = [&](auto f) {
            for (int i = tid; i < n; i += kRowThreads) {
                const uint32_t key = order_key(x[i]);
                if (key > kKeyMinusInf) f(key, i);
            }
        };
        if (s.use_k) cut = select_cut(sel, (u64)s.k, each, one);
        if (s.use_p) {
            u64 add = 0;
            const Cut k_cut = cut;
            auto kept = [&](auto f) {
                each([&](uint32_t key, int i) {
                    if (k_cut.keeps(key, i)) f(key, i);
                });
            };
            kept([&](uint32_t key, int) { add += units(key); });
            add = wave_sum(add);
            if (add && lane == 0) atomicAdd(&total_w, add);
            __syncthreads();
            cut = select_cut(sel, p_goal(s, total_w), kept, units);
            cut.within(k_cut);
        }
    }

    // ---- the running sum over segments, then inside the one that passes u times the sum
    const float cut_l = cut.key ? key_logit(cut.key) : -INFINITY;
    auto weight_of = [&](float l, int i) {
        if (!(l > cut_l || (l == cut_l && i <= cut.index))) return 0.0;
        const double v = w(l);
        return v >= s.min_w ? v : 0.0;
    };
    // inclusive running sum over the workgroup, and the sum; each once, with its own LDS
    auto scan = [&](int which, double v, double& all) {
        const double upto = wave_scan(v);
        if (lane == 63) wave_w[which][wave] = upto;
        __syncthreads();
        double ahead = 0.0;
        all = 0.0;
        for (int i = 0; i < kRowWaves; i++) {
            if (i < wave) ahead += wave_w[which][i];
            all += wave_w[which][i];
        }
        return ahead + upto;
    };
    const bool formed = w.inf || info.cut == 2 || small;
    if (formed) {  // the segments' sums are not there: form them
        __syncthreads();
        for (int g = wave; g < segments; g += kRowWaves) {
            double v = 0.0;
            for (int i = g * kSegment + lane; i < min((g + 1) * kSegment, n); i += 64)
                v += weight_of(x[i], i);
            v = wave_sum(v);
            if (lane == 0) seg_sum[g] = __builtin_bit_cast(u64, v);
        }
        __syncthreads();
    }
    double seg_w = 0.0;
    if (tid < segments) {
        const u64 b = seg_sum[tid];
        if (formed) {
            seg_w = __builtin_bit_cast(double, b);
        } else if (s.plain()) {  // its chunk's largest -> the row's
            const float top = row_stats(a, row)[tid * kSegment / kBlock].top;
            seg_w = __builtin_bit_cast(double, b) * w(top);
        } else {
            seg_w = (double)b * (1.0 / kRowUnit);
        }
    }
    double total;
    const double upto = scan(0, seg_w, total);
    const double target = (double)u * total;
    // the first that passes the target (rounding may leave none: the last with a weight)
    auto choose = [&](int which, bool passes, int at, bool any, int last) {
        const u64 hits = __ballot(passes), has = __ballot(any);
        if (hits && lane == __builtin_ctzll(hits)) atomicMin(&first_at[which], at);
        if (has && lane == 63 - __builtin_clzll(has)) atomicMax(&last_at[which], last);
        __syncthreads();
        return first_at[which] != INT32_MAX ? first_at[which] : max(last_at[which], 0);
    };
    const int seg = choose(0, seg_w > 0.0 && upto > target, tid, seg_w > 0.0, tid);
    if (seg == tid) seg_before = upto - seg_w;
    const int per = info.wide ? kWide : 1, i = seg * kSegment + per * tid;
    double v[kWide], sum = 0.0, all;
    float l[kWide];
#pragma unroll
    for (int e = 0; e < kWide; e++) l[e] = e < per && i + e < n ? x[i + e] : -INFINITY;
#pragma unroll
    for (int e = 0; e < kWide; e++) {
        v[e] = e < per && i + e < n ? weight_of(l[e], i + e) : 0.0;
        sum += v[e];
    }
    const double upto_i = scan(1, sum, all);
    // falling from the lane's last: the first that passes, and the last with a weight
    double run = seg_before + upto_i;
    int pass = -1, last = -1;
#pragma unroll
    for (int e = kWide - 1; e >= 0; e--) {
        if (v[e] > 0.0 && run > target) pass = i + e;
        if (v[e] > 0.0) last = max(last, i + e);
        run -= v[e];
    }
    const int at = choose(1, pass >= 0, pass, last >= 0, last);
    if (tid == 0) a.out[row] = at;
}

long long row_bytes_of(int chunks) {
    return 128 + sizeof(ChunkStat) * kMaxChunks + 8LL * (kMaxSegments + (long long)chunks * kChunkWords);
}

int chunks_of(int n_vocab) { return (n_vocab + kBlock - 1) / kBlock; }

// Sizes whose grids have fewer than 2^32 threads.
bool sizes_ok(int n_rows, int n_vocab) {
    return n_rows > 0 && n_vocab > 0 && n_vocab < kMaxVocab &&
           (long long)n_rows * chunks_of(n_vocab) <= (long long)(UINT32_MAX / kRowThreads);
}

}  // namespace

extern "C" long long tf_sample_ws_bytes(int n_rows, int n_vocab) {
    return sizes_ok(n_rows, n_vocab) ? n_rows * row_bytes_of(chunks_of(n_vocab)) : -1;
}

extern "C" int tf_sample(const float* logits, int n_rows, int n_vocab, int row_stride,
                         const float* temperature, const int* top_k, const float* top_p,
                         const float* min_p, const float* u, int* out_idx, void* ws,
                         long long ws_bytes, tf_stream_t stream) {
    TF_CHECK_ARG(logits && u && out_idx && ws && sizes_ok(n_rows, n_vocab));
    TF_CHECK_ARG(row_stride >= n_vocab && ((uintptr_t)ws & 15) == 0);
    TF_CHECK_ARG(ws_bytes >= tf_sample_ws_bytes(n_rows, n_vocab));
    SampleArgs a{};
    a.logits = logits, a.stride = row_stride, a.n = n_vocab;
    a.temperature = temperature, a.top_k = top_k, a.top_p = top_p, a.min_p = min_p;
    a.u = u, a.out = out_idx;
    a.chunks = chunks_of(n_vocab);
    a.ws = static_cast<uint8_t*>(ws);
    a.row_bytes = row_bytes_of(a.chunks);
    const unsigned grid = (unsigned)n_rows * (unsigned)a.chunks;
    hipLaunchKernelGGL(tf_sample_stats_kernel, dim3(grid), dim3(kChunkThreads), 0,
                       tf_stream(stream), a);
    if (top_k || top_p || min_p)
        hipLaunchKernelGGL(tf_sample_gather_kernel, dim3(grid), dim3(kChunkThreads), 0,
                           tf_stream(stream), a);
    constexpr int bytes = 8 * (kList + kMaxSegments) + (int)sizeof(Select);
    const int rc = tf_set_lds_limit((const void*)tf_sample_draw_kernel, bytes);
    if (rc) return rc;
    hipLaunchKernelGGL(tf_sample_draw_kernel, dim3(n_rows), dim3(kRowThreads), bytes,
                       tf_stream(stream), a);
    return TF_LAUNCH_RESULT();
}
