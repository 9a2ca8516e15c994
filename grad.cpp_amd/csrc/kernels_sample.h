// Picks from rows of logits with a temperature, top-k, top-p and min-p of each row's own (gh_sample).
//
// With x the logits of a row and M the largest, w_i = exp((x_i - M) / T).  The tokens are ordered by x, equal ones by index.
// top-k keeps the first k of that order, top-p the shortest leading stretch of those whose w reach p of their sum, min-p what has
// w >= min_p; the pick is the lowest kept index up to which the kept w reach u of their sum.
//
// Whether a draw falls on this or the other side of a border is decided in 64 bits: with 32-bit exponentials equal logits (a
// 16-bit row has thousands) share one error, and one draw in a hundred from 128 k tokens of a flat row would be
// another token than the definition's.  The card's 64-bit instructions have the rate of plain 32-bit ones.
//
// No order is ever sorted out over the whole row: a cut is found by histograms, of counts or of w, over buckets of x.  w are whole
// numbers there (multiples of 2^-scale of the largest), so that the atomics' order does not matter.
#pragma once

#include "kernels_cache_attn.h"

namespace gh {

constexpr int kSampleThreads = 1024;
constexpr int kSampleWaves = kSampleThreads / 64;
constexpr int kMaxSampleVocab = 1 << 20;
constexpr int kBuckets = 2048;
constexpr double kLeastPower = 44.0;  // w below 2^-44 of the largest are nothing: all of a million tokens together are below 2^-24

struct SampleParams {
    const void* logits;
    long long row_stride;
    int vocab;
    int scale_bits;  // of the histograms' whole numbers: vocab * 2^scale_bits < 2^63
    const float* temperature;
    const int* top_k;
    const float* top_p;
    const float* min_p;
    const float* uniforms;
    int* ids;
    float* probs;
};

// Order-preserving whole numbers of floats.
__device__ __forceinline__ unsigned order_key(float x) {
    const unsigned b = __float_as_uint(x);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d);
    return v;
}
template <typename T>
__device__ __forceinline__ T wave_scan(T v) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const T o = __shfl_up(v, d);
        if (lane >= d) v += o;
    }
    return v;
}
// Total of the lanes before this one.
template <typename T>
__device__ __forceinline__ T wave_scan_before(T inclusive) {
    const T o = __shfl_up(inclusive, 1);
    return (threadIdx.x & 63) == 0 ? T(0) : o;
}
// Totals over the workgroup's threads: of those before this one (exactly zero where they hold nothing), and of all.  `waves` is
// scratch; every thread calls.
template <typename T>
__device__ __forceinline__ T block_scan(T v, T* waves, T& all) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const T upto = wave_scan(v);
    __syncthreads();
    if (lane == 63) waves[wave] = upto;
    __syncthreads();
    T before = 0, sum = 0;
#pragma unroll
    for (int w = 0; w < kSampleWaves; w++) {
        if (w == wave) before = sum;
        sum += waves[w];
    }
    all = sum;
    return before + wave_scan_before(upto);
}

template <int TYPE>
struct SampleRow {
    using T = typename CacheType<TYPE>::T;
    static constexpr int kVec = 16 / CacheType<TYPE>::kBytes;
    const T* at;
    int vocab;
    int vectors;
    __device__ __forceinline__ SampleRow(const SampleParams& p, int row)
        : at(static_cast<const T*>(p.logits) + row * p.row_stride), vocab(p.vocab), vectors((p.vocab + kVec - 1) / kVec) {}
    // Vector j's logits; NaN and what is behind the row are minus infinity.  (Rows begin anywhere: loads of 16 bytes need no alignment.)
    __device__ __forceinline__ void load(int j, float (&x)[kVec]) const {
        T e[kVec];
        if ((j + 1) * kVec <= vocab) {
            __builtin_memcpy(e, at + j * kVec, 16);
#pragma unroll
            for (int i = 0; i < kVec; i++) x[i] = static_cast<float>(e[i]);
        } else {
#pragma unroll
            for (int i = 0; i < kVec; i++) x[i] = j * kVec + i < vocab ? static_cast<float>(at[j * kVec + i]) : -INFINITY;
        }
#pragma unroll
        for (int i = 0; i < kVec; i++) x[i] = x[i] == x[i] ? x[i] + 0.0f : -INFINITY;  // (zeros of either sign are equal)
    }
    template <typename F>
    __device__ __forceinline__ void each(F&& f) const {
        for (int j = threadIdx.x; j < vectors; j += kSampleThreads) {
            float x[kVec];
            load(j, x);
#pragma unroll
            for (int i = 0; i < kVec; i++) f(x[i], j * kVec + i);
        }
    }
};

// What is kept: keys above `key`, and of those equal to it the indices up to `index`; of these, w of at least `least`.
struct Cut {
    unsigned key = 0;
    int index = 0x7FFFFFFF;
    __device__ __forceinline__ bool keeps(unsigned k, int i) const { return k > key || (k == key && i <= index); }
};

struct SampleShared {
    unsigned long long bins[kBuckets];
    unsigned long long scan[kSampleWaves];
    double sums[kSampleWaves];
    float tops[kSampleWaves];
    int indices[kSampleWaves];
    unsigned low, high;
    unsigned long long above;  // of the histogram, before the bucket that was found
    int bucket;
    int found;
};

struct SampleWeights {
    float top;
    double turn;  // log2(e) / temperature
    double scale;
    __device__ __forceinline__ double power(float x) const { return x == top ? 0.0 : (static_cast<double>(x) - top) * turn; }
    __device__ __forceinline__ double weight(float x) const {
        const double y = power(x);
        return y > -kLeastPower ? exp2(y) : 0.0;
    }
    __device__ __forceinline__ unsigned long long whole(double w) const { return static_cast<unsigned long long>(__double_as_longlong(fma(w, scale, 0x1p52))) & 0xFFFFFFFFFFFFFull; }
};

// The bucket in which the running total of sh.bins, from bucket 0 on, reaches `target`, or all there is if that is less; for targets of zero
// and less the first that holds anything.  The totals before it and of all are left in sh.above and `all`.
__device__ __forceinline__ int find_bucket(SampleShared& sh, double target, unsigned long long& all) {
    __syncthreads();
    const unsigned long long a = sh.bins[2 * threadIdx.x], b = sh.bins[2 * threadIdx.x + 1];
    const unsigned long long before = block_scan(a + b, sh.scan, all);
    target = fmin(target, static_cast<double>(all));
    const auto first = [&](unsigned long long sum_before, unsigned long long own) {
        return own > 0 && (sum_before == 0 || static_cast<double>(sum_before) < target) && static_cast<double>(sum_before + own) >= target;
    };
    if (first(before, a)) {
        sh.bucket = 2 * threadIdx.x;
        sh.above = before;
    } else if (first(before + a, b)) {
        sh.bucket = 2 * threadIdx.x + 1;
        sh.above = before + a;
    }
    __syncthreads();
    return sh.bucket;
}

// The cut behind which the running total, in the order of the tokens, of 1 (MASS: of w as whole numbers) per token that `kept` keeps reaches
// `target`.  Buckets of x relative to the largest first, then of the keys of one bucket, finer and finer, then equal keys by
// their index.  Tokens whose w are nothing are left out.
template <int TYPE, bool MASS>
__device__ __forceinline__ Cut find_cut(const SampleRow<TYPE>& row, const SampleWeights& w, const Cut& kept, double target, SampleShared& sh) {
    const double fine = kBuckets / kLeastPower;
    const auto bucket_of = [&](float x) { return min(static_cast<int>(-w.power(x) * fine), kBuckets - 1); };
    const auto clear = [&] {
        __syncthreads();
        sh.bins[2 * threadIdx.x] = 0;
        sh.bins[2 * threadIdx.x + 1] = 0;
        __syncthreads();
    };
    const auto amount = [&](float x) { return MASS ? w.whole(w.weight(x)) : 1ull; };
    clear();
    row.each([&](float x, int i) {
        if (w.power(x) > -kLeastPower && kept.keeps(order_key(x), i)) atomicAdd(&sh.bins[bucket_of(x)], amount(x));
    });
    unsigned long long all;
    const int bucket = find_bucket(sh, target, all);
    if (!MASS && static_cast<double>(all) < target) return kept;  // (there are fewer)
    unsigned long long above = sh.above;
    if (threadIdx.x == 0) {
        sh.low = 0xFFFFFFFFu;
        sh.high = 0;
    }
    __syncthreads();
    row.each([&](float x, int i) {
        if (w.power(x) > -kLeastPower && bucket_of(x) == bucket && kept.keeps(order_key(x), i)) {
            atomicMin(&sh.low, order_key(x));
            atomicMax(&sh.high, order_key(x));
        }
    });
    __syncthreads();
    unsigned low = sh.low, high = sh.high;
    while (low < high) {
        const int shift = max(0, 32 - __clz(high - low) - 11);
        clear();
        row.each([&](float x, int i) {
            const unsigned k = order_key(x);
            if (k >= low && k <= high && kept.keeps(k, i)) atomicAdd(&sh.bins[(high - k) >> shift], amount(x));
        });
        const int b = find_bucket(sh, target - static_cast<double>(above), all);
        above += sh.above;
        high -= static_cast<unsigned>(b) << shift;
        if (high - low > (1u << shift) - 1) low = high - ((1u << shift) - 1);
    }
    // equal keys: so many of them, the lowest indices
    const float x0 = __uint_as_float(low & 0x80000000u ? low ^ 0x80000000u : ~low);
    const double each = static_cast<double>(amount(x0));
    const double wanted = ceil((target - static_cast<double>(above)) / each);
    const int take = wanted < 1.0 ? 1 : wanted > 1e9 ? 1000000000 : static_cast<int>(wanted);
    Cut cut;
    cut.key = low;
    if (threadIdx.x == 0) sh.found = 0x7FFFFFFF;
    int counted = 0;
    for (int j0 = 0; j0 < row.vectors && counted < take; j0 += kSampleThreads) {
        const int j = j0 + threadIdx.x;
        float x[SampleRow<TYPE>::kVec];
        unsigned equal = 0;
        if (j < row.vectors) {
            row.load(j, x);
#pragma unroll
            for (int i = 0; i < SampleRow<TYPE>::kVec; i++) {
                const int index = j * SampleRow<TYPE>::kVec + i;
                if (index < row.vocab && order_key(x[i]) == low && kept.keeps(low, index)) equal |= 1u << i;
            }
        }
        const int before = counted + static_cast<int>(block_scan(static_cast<unsigned long long>(__popc(equal)), sh.scan, all));
        if (before < take && before + __popc(equal) >= take) {
            for (int n = take - before; n > 1; n--) equal &= equal - 1;
            sh.found = j * SampleRow<TYPE>::kVec + __ffs(equal) - 1;
        }
        counted += static_cast<int>(all);
    }
    __syncthreads();
    cut.index = sh.found;
    return cut;
}

// One workgroup per row.
template <int TYPE>
__global__ __launch_bounds__(kSampleThreads) void sample_row_kernel(const SampleParams p) {
    using Row = SampleRow<TYPE>;
    constexpr int kVec = Row::kVec;
    constexpr int kSegments = kMaxSampleVocab / (64 * 4);
    __shared__ SampleShared sh;
    __shared__ double segments[kSegments];
    const int r = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const Row row(p, r);

    // the largest logit and the lowest index that has it
    float top = -INFINITY;
    int first = 0x7FFFFFFF;
    row.each([&](float x, int i) {
        if (x > top) {
            top = x;
            first = i;
        }
    });
    wave_first_max(top, first);
    if (lane == 0) {
        sh.tops[wave] = top;
        sh.indices[wave] = first;
    }
    __syncthreads();
    for (int w = 0; w < kSampleWaves; w++)
        if (sh.tops[w] > top || (sh.tops[w] == top && sh.indices[w] < first)) {
            top = sh.tops[w];
            first = sh.indices[w];
        }
    const float temperature = p.temperature ? p.temperature[r] : 1.0f;
    if (top == -INFINITY || !(temperature > 0.0f)) {
        if (threadIdx.x == 0) {
            p.ids[r] = top == -INFINITY ? -1 : first;
            if (p.probs) p.probs[r] = top == -INFINITY ? 0.0f : 1.0f;
        }
        return;
    }
    SampleWeights w{top, 1.44269504088896340736 / temperature, __longlong_as_double(static_cast<long long>(1023 + p.scale_bits) << 52)};

    Cut cut;
    const int top_k = p.top_k ? p.top_k[r] : 0;
    if (top_k > 0 && top_k < p.vocab) cut = find_cut<TYPE, false>(row, w, cut, top_k, sh);
    const float top_p = p.top_p ? p.top_p[r] : 1.0f;
    if (top_p < 1.0f) {
        unsigned long long mine = 0;
        row.each([&](float x, int i) {
            if (cut.keeps(order_key(x), i)) mine += w.whole(w.weight(x));
        });
        unsigned long long all;
        (void)block_scan(mine, sh.scan, all);
        cut = find_cut<TYPE, true>(row, w, cut, static_cast<double>(top_p) * static_cast<double>(all), sh);
    }
    const float min_p = p.min_p ? p.min_p[r] : 0.0f;
    const double least = min_p > 0.0f ? fminf(min_p, 1.0f) : 0.0f;
    const auto kept = [&](float x, int i) {
        const double v = cut.keeps(order_key(x), i) ? w.weight(x) : 0.0;
        return v >= least ? v : 0.0;
    };

    // sums of what a wavefront reads at a time, in the order of the indices; the one in which the draw falls
    const int count = (row.vectors + 63) / 64;
    for (int s = wave; s < count; s += kSampleWaves) {
        double sum = 0.0;
        const int j = s * 64 + lane;
        if (j < row.vectors) {
            float x[kVec];
            row.load(j, x);
#pragma unroll
            for (int i = 0; i < kVec; i++) sum += kept(x[i], j * kVec + i);
        }
        sum = wave_sum(sum);
        if (lane == 0) segments[s] = sum;
    }
    __syncthreads();
    const int each = (count + kSampleThreads - 1) / kSampleThreads, from = min(count, static_cast<int>(threadIdx.x) * each), to = min(count, from + each);
    double mine = 0.0;
    for (int s = from; s < to; s++) mine += segments[s];
    if (threadIdx.x == 0) sh.found = -1;
    double total;
    const double before = block_scan(mine, sh.sums, total);
    const float u = p.uniforms[r];
    const double target = (u > 0.0f ? static_cast<double>(u) : 0.0) * total;  // (NaN: 0)
    // the last segment whose running total before it is below the target, among those that hold anything
    double below = before;
    for (int s = from; s < to; s++) {
        if (segments[s] > 0.0 && (below < target || below == 0.0)) atomicMax(&sh.found, s);
        below += segments[s];
    }
    __syncthreads();
    const int segment = sh.found;
    if (segment >= from && segment < to) {
        below = before;
        for (int s = from; s < segment; s++) below += segments[s];
        sh.sums[0] = below;
    }
    __syncthreads();
    if (wave != 0) return;
    const int j = segment * 64 + lane;
    double v[kVec], sum = 0.0;
    float x[kVec];
#pragma unroll
    for (int i = 0; i < kVec; i++) v[i] = 0.0;
    if (j < row.vectors) {
        row.load(j, x);
#pragma unroll
        for (int i = 0; i < kVec; i++) sum += v[i] = kept(x[i], j * kVec + i);
    }
    double running = sh.sums[0] + wave_scan_before(wave_scan(sum));
    int mine_hit = 0x7FFFFFFF, mine_last = -1;
    double hit_weight = 0.0, last_weight = 0.0;
#pragma unroll
    for (int i = 0; i < kVec; i++) {
        running += v[i];
        if (v[i] > 0.0) {
            mine_last = i;
            last_weight = v[i];
            if (running >= target && mine_hit == 0x7FFFFFFF) {
                mine_hit = i;
                hit_weight = v[i];
            }
        }
    }
    const unsigned long long hits = __ballot(mine_hit != 0x7FFFFFFF), lasts = __ballot(mine_last >= 0);
    const int chosen = hits ? __ffsll(hits) - 1 : 63 - __clzll(lasts);
    if (lane == chosen) {
        p.ids[r] = j * kVec + (hits ? mine_hit : mine_last);
        if (p.probs) p.probs[r] = static_cast<float>((hits ? hit_weight : last_weight) / total);
    }
}

}  // namespace gh
