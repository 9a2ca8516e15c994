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
// A row is read once, in chunks, all of it in registers: what stays of it are the largest logits of groups of 64, and where the sum of all w
// matters (no top-k), sums relative to the chunk's largest: with top-p w by buckets of x, without it those of segments of 512.  From these
// follows a bound below which nothing is kept:
//   top-k: k groups have a logit of at least the k-th largest of the groups' largest (so buckets of these will do; where groups are few, of all logits);
//   top-p: the bucket in which the running sum of w reaches p of the whole;   min-p: the logarithm.
// Only groups that reach the bound are looked at again; the tokens above it become a list, which is put in order, cut and drawn from.  What does
// not fit a list (a nucleus of thousands of tokens) is cut among the bucket's own tokens, and only the chunk that the draw falls into is read again;
// where a bucket's tokens do not fit a list either (thousands of equal logits, k of thousands), histograms over the row find the cut.
// Bucket sums are whole numbers, so the order in which atomics arrive changes nothing.  A bucket's are of a unit of its own, 2^-48 and less of its
// w: with one unit for a row a tail of a million equal w of 2^-26 would be rounded alike, and its cut be off by tokens.
#pragma once

#include "kernels_cache_attn.h"

#include <type_traits>

namespace gh {

constexpr int kSampleThreads = 256;  // that pick: most of it is steps one behind the other, which four wavefronts take in less time than sixteen
constexpr int kSampleWaves = kSampleThreads / 64;
constexpr int kWideThreads = 512;   // that read large chunks
constexpr int kMaxSampleVocab = 1 << 20;
constexpr int kVec = 8;               // logits of a lane
constexpr int kGroup = 64;            // of eight lanes
constexpr int kSegment = 64 * kVec;   // of a wavefront
constexpr int kRounds = 4;            // vectors of a thread, in registers: a chunk
constexpr int kChunk = kSampleThreads * kVec * kRounds, kWideChunk = kWideThreads * kVec * kRounds;
constexpr int kMaxSegments = kMaxSampleVocab / kSegment;
constexpr int kListed = 2048;                 // tokens that are sorted
constexpr int kPowers = 256;                  // a table of 2^(j / 256), j < 256
static_assert(kPowers == 1 << 8, "");
constexpr int kBuckets = 2048;                // of the histograms over the row
constexpr double kLeastPower = 44.0;          // w below 2^-44 of the largest are nothing: all of a million tokens together are below 2^-24
// w by buckets of x: so many to a power of two, on a grid that all chunks share
constexpr int kMassBuckets = 1024;
constexpr double kMassFine = 40.0;
constexpr int kMassBits = 47;  // of a w in its bucket's unit: a chunk's 2^14 tokens sum to less than 2^63
static_assert(kWideChunk <= 1 << 14, "");

struct SampleParams {
    const void* logits;
    long long row_stride;
    int vocab;
    int scale_bits;  // of a w in the unit of its bucket, for the histograms over the row: vocab * 2^scale_bits < 2^63
    const float* temperature;
    const int* top_k;
    const float* top_p;
    const float* min_p;
    const float* uniforms;
    int* ids;
    float* probs;
    int first_row;
    double powers[kPowers];
    // what the chunks leave, of every row: [groups], [chunks], [segments], [chunks][kMassBuckets]
    int chunks;
    float* group_tops;
    float* chunk_tops;
    double* segment_sums;
    unsigned long long* masses;
    // where several workgroups look through a row of many groups: [2] (listed, arrived), [kListed]
    int shares;
    unsigned* counters;
    unsigned long long* lists;
};

constexpr int groups_of(int vocab) { return (vocab + kGroup - 1) / kGroup; }
constexpr int segments_of(int vocab) { return (vocab + kSegment - 1) / kSegment; }

// Order-preserving whole numbers of floats.
__device__ __forceinline__ unsigned order_key(float x) {
    const unsigned b = __float_as_uint(x);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float key_value(unsigned k) { return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k); }

template <int CTRL, int ROW_MASK>
__device__ __forceinline__ double dpp_move(double v) {
    const long long b = __double_as_longlong(v);
    const int lo = dpp_move_int<CTRL, ROW_MASK>(static_cast<int>(b)), hi = dpp_move_int<CTRL, ROW_MASK>(static_cast<int>(b >> 32));
    return __longlong_as_double(static_cast<long long>(hi) << 32 | static_cast<unsigned>(lo));
}
// Running total over the lanes, this lane's included.
__device__ __forceinline__ double wave_scan(double v) {
    v += dpp_move<0x111, 0xF>(v);  // row_shr:1
    v += dpp_move<0x112, 0xF>(v);
    v += dpp_move<0x114, 0xF>(v);
    v += dpp_move<0x118, 0xF>(v);
    v += dpp_move<0x142, 0xA>(v);  // row_bcast:15 into rows 1 and 3
    v += dpp_move<0x143, 0xC>(v);  // row_bcast:31 into rows 2 and 3
    return v;
}
__device__ __forceinline__ unsigned long long wave_scan(unsigned long long v) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const unsigned long long o = __shfl_up(v, d);
        if (lane >= d) v += o;
    }
    return v;
}
__device__ __forceinline__ int wave_scan(int v) { return wave_inclusive_scan(v); }

// Totals over the workgroup's threads: of those before this one (exactly zero where they hold nothing), and of all.  `waves` is
// scratch; every thread calls.  (Of the threads that pick.)
template <typename T>
__device__ __forceinline__ T block_scan(T v, T* waves, T& all) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const T upto = wave_scan(v), shifted = __shfl_up(upto, 1);
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
    return before + (lane == 0 ? T(0) : shifted);
}

// A row's logits, eight neighbours to a lane; NaN and what is behind the row are minus infinity, zeros of either sign are equal.
// (Rows begin anywhere: loads of 16 bytes need no alignment.)
template <int TYPE>
struct SampleRow {
    using T = typename CacheType<TYPE>::T;
    const T* at;
    int vocab;
    __device__ __forceinline__ SampleRow(const SampleParams& p, int row) : at(static_cast<const T*>(p.logits) + row * p.row_stride), vocab(p.vocab) {}
    static __device__ __forceinline__ float clean(T e) {
        const float x = static_cast<float>(e);
        return x == x ? x + 0.0f : -INFINITY;
    }
    // (Without a condition but for the row's end, so that many loads can be under way at once.)
    __device__ __forceinline__ void load_raw(int i0, T (&e)[kVec]) const {
        if (vocab >= kVec) __builtin_memcpy(e, at + min(i0, vocab - kVec), sizeof(e));
        if (i0 + kVec > vocab) {
#pragma unroll
            for (int i = 0; i < kVec; i++) e[i] = i0 + i < vocab ? at[i0 + i] : static_cast<T>(-INFINITY);
        }
    }
    __device__ __forceinline__ void load(int i0, float (&x)[kVec]) const {
        T e[kVec];
        load_raw(i0, e);
#pragma unroll
        for (int i = 0; i < kVec; i++) x[i] = clean(e[i]);
    }
    __device__ __forceinline__ float one(int i) const {
        const float x = clean(at[min(i, vocab - 1)]);
        return i < vocab ? x : -INFINITY;
    }
    // Every logit, in any order, f called by all threads alike; many loads at a time, or each would be a trip to memory of its own.
    template <typename F>
    __device__ __forceinline__ void each(F&& f) const {
        constexpr int kDeep = 4;
        for (int from = 0; from < vocab; from += kDeep * kSampleThreads * kVec) {
            T e[kDeep][kVec];
#pragma unroll
            for (int k = 0; k < kDeep; k++) load_raw(from + (k * kSampleThreads + static_cast<int>(threadIdx.x)) * kVec, e[k]);
#pragma unroll
            for (int k = 0; k < kDeep; k++) {
                if (from + k * kSampleThreads * kVec >= vocab) break;
#pragma unroll
                for (int i = 0; i < kVec; i++) f(clean(e[k][i]), from + (k * kSampleThreads + static_cast<int>(threadIdx.x)) * kVec + i);
            }
        }
    }
};

// What is kept: keys above `key`, and of those equal to it the indices up to `index`.
struct Cut {
    unsigned key = 0;
    int index = 0x7FFFFFFF;
    __device__ __forceinline__ bool keeps(unsigned k, int i) const { return (k > key) | ((k == key) & (i <= index)); }
};

// What a chunk leaves.
template <int THREADS>
struct ChunkShared {
    unsigned long long masses[kMassBuckets];
    double segments[THREADS * kVec * kRounds / kSegment];
    float group_tops[THREADS * kVec * kRounds / kGroup];
    float tops[THREADS / 64];
};

struct PickShared {
    union {
        unsigned long long bins[kBuckets];
        unsigned counts[kBuckets];
    };
    unsigned long long list[kListed];
    union {
        double segments[kMaxSegments];
        int hot[kListed];  // groups
        double weights[kListed];
    };
    double chunk_sums[kMaxSampleVocab / kChunk];
    double chunk_shares[kMaxSampleVocab / kChunk];  // of a w relative to its chunk's largest, relative to the row's
    int chunk_shifts[kMaxSampleVocab / kChunk];     // how far its buckets lie behind the row's; all of them where it has none
    double chunk_scales[kMaxSampleVocab / kChunk];  // of its buckets' units, relative to the row's
    unsigned long long scan[kSampleWaves];
    double sums[kSampleWaves];
    int ints[kSampleWaves];
    float tops[kSampleWaves], lows[kSampleWaves];
    unsigned long long chunk_wholes[kMaxSampleVocab / kChunk];
    unsigned low, high;
    unsigned long long above;  // of the histogram, before the bucket that was found
    double mass_above, mass_upto;
    int bucket, found, listed;
};

// w = exp((x - top) / T) = 2^(n / 256 + r / 256), |r| <= 1/2: 2^(n / 256) from a table, the series of the rest cut off behind the third power (relative
// error below 2e-13).  Exactly 1 at the top, 0 below 2^-44.
constexpr double kLeastTurns = -kPowers * kLeastPower;
constexpr double kMagic = 0x1.8p52;  // added to a number below 2^51 leaves it rounded in the last bits

// 256 log2 of a w of `z`, or what is not a number.
__device__ __forceinline__ double weight_of(double z, const double* powers) {
    constexpr double l = 0.69314718055994530942 / kPowers, c2 = l * l / 2, c3 = l * l * l / 6;
    z = z > kLeastTurns ? z : -1e9;  // (at 0 then)
    const double t = z + kMagic, r = z - (t - kMagic);
    const int n = static_cast<int>(__double_as_longlong(t));
    const double head = powers[n & (kPowers - 1)];
    return ldexp(fma(head, r * fma(r, fma(r, c3, c2), l), head), n >> 8);
}

struct SampleWeights {
    float top;
    double turn;  // 256 log2(e) / T
    const double* powers;
    __device__ __forceinline__ double turns(float x) const { return x == top ? 0.0 : (static_cast<double>(x) - top) * turn; }
    __device__ __forceinline__ double weight(float x) const { return weight_of(turns(x), powers); }
};

__device__ __forceinline__ unsigned long long whole_number(double w, double scale) {
    return static_cast<unsigned long long>(__double_as_longlong(fma(w, scale, 0x1p52))) & 0xFFFFFFFFFFFFFull;
}

__device__ __forceinline__ double power_of_two(int n) { return __longlong_as_double(static_cast<long long>(1023 + n) << 52); }

// The unit of a bucket is 2^-kMassBits of the power of two that its place on the grid falls into: kMassFine places to each.  Seen from a larger logit's place
// these are `octaves_to(b, rest)` powers of two down, for the bucket b places down (not beyond kMassBuckets); all chunks cut the grid alike.
constexpr int kOctave = static_cast<int>(kMassFine);
__device__ __forceinline__ int octave_rest(int place) { return kOctave - 1 - ((place % kOctave + kOctave) % kOctave); }
__device__ __forceinline__ int octaves_to(int b, int rest) {
    static_assert(kOctave == 40 && kMassBuckets == 1024, "1639 / 2^16: (b + rest) / 40 up to 2600");
    return (b + rest) * 1639 >> 16;
}

// What a row's settings come to.
struct SampleSettings {
    float temperature;
    int top_k;      // 0: off
    double top_p;   // 1: off
    double min_p;   // 0: off
    __device__ __forceinline__ SampleSettings(const SampleParams& p, int r) {
        temperature = p.temperature ? p.temperature[r] : 1.0f;
        top_k = p.top_k ? p.top_k[r] : 0;
        if (top_k < 0 || top_k >= p.vocab) top_k = 0;
        const float tp = p.top_p ? p.top_p[r] : 1.0f, mp = p.min_p ? p.min_p[r] : 0.0f;
        top_p = tp < 1.0f ? tp : 1.0f;
        min_p = mp > 0.0f ? fminf(mp, 1.0f) : 0.0f;
    }
    __device__ __forceinline__ bool greedy() const { return !(temperature > 0.0f); }
    __device__ __forceinline__ double turn() const { return fmax(kPowers * 1.44269504088896340736 / temperature, 1e-290); }
    // the whole row's sum: by segments; by buckets as well
    __device__ __forceinline__ bool sums() const { return !greedy() && top_k == 0 && (top_p < 1.0 || min_p == 0.0); }
    __device__ __forceinline__ bool masses() const { return !greedy() && top_k == 0 && top_p < 1.0; }
    // places are whole numbers below 2^31, a chunk's where the row's largest is below 2^29
    __device__ __forceinline__ bool on_grid(float top, double limit = 0x1p30) const { return fabs(top * grid()) < limit; }
    __device__ __forceinline__ double grid() const { return kMassFine * 1.44269504088896340736 / temperature; }
};

// The place on the grid: larger logits have larger ones.  Chunks leave a bucket at its place modulo kMassBuckets, which does not depend on what is largest.
__device__ __forceinline__ int grid_place(float x, double grid) { return static_cast<int>(__double_as_longlong(fma(static_cast<double>(x), grid, kMagic))); }

__device__ __forceinline__ void fill_powers(const SampleParams& p, double* powers) {
    if (threadIdx.x < kPowers) powers[threadIdx.x] = p.powers[threadIdx.x];
}

template <int THREADS>
__device__ __forceinline__ float block_top(float v, float* tops) {
    v = wave_max(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) tops[threadIdx.x >> 6] = v;
    __syncthreads();
    v = tops[0];
#pragma unroll
    for (int w = 1; w < THREADS / 64; w++) v = fmaxf(v, tops[w]);
    return v;
}

// The largest and the least of the workgroup's. (Of the threads that pick.)
__device__ __forceinline__ void block_ends(float& high, float& low, PickShared& sh) {
    high = wave_max(high);
    low = -wave_max(-low);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) {
        sh.tops[threadIdx.x >> 6] = high;
        sh.lows[threadIdx.x >> 6] = low;
    }
    __syncthreads();
    high = sh.tops[0];
    low = sh.lows[0];
#pragma unroll
    for (int w = 1; w < kSampleWaves; w++) {
        high = fmaxf(high, sh.tops[w]);
        low = fminf(low, sh.lows[w]);
    }
}

// One chunk of a row, from `first` on.  Leaves the groups' largest logits, and where they are wanted the segments' sums (with buckets, the wavefronts'), relative
// to the largest of the chunk, and w by buckets of x, from the chunk's largest down.  Returns the largest.
//
// The logits are loaded in one go, kept as they are, and gone through twice, because the exponentials need the chunk's largest first.  Without w it is bound
// by reading; with w and buckets (some 44 vector instructions a logit, a look-up and an atomic in shared memory) by neither alone: what is resident
// loads, then computes.
template <int TYPE, int THREADS>
__device__ __forceinline__ float scan_chunk(const SampleParams& p, const SampleRow<TYPE>& row, const SampleSettings& set, int first, const double* powers,
                                            ChunkShared<THREADS>& sh) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    using T = typename SampleRow<TYPE>::T;
    T raw[kRounds][kVec];
#pragma unroll
    for (int r = 0; r < kRounds; r++) row.load_raw(first + (r * THREADS + static_cast<int>(threadIdx.x)) * kVec, raw[r]);
    float top = -INFINITY;
#pragma unroll
    for (int r = 0; r < kRounds; r++) {
        float high = -INFINITY;
#pragma unroll
        for (int i = 0; i < kVec; i++) high = fmaxf(high, static_cast<float>(raw[r][i]));  // (not a NaN)
        high = fmaxf(high, dpp_move<0xB1, 0xF>(high, high));   // over the eight lanes of a group
        high = fmaxf(high, dpp_move<0x4E, 0xF>(high, high));
        high = fmaxf(high, dpp_move<0x141, 0xF>(high, high));  // row_half_mirror
        if ((lane & 7) == 0) sh.group_tops[r * (THREADS * kVec / kGroup) + (threadIdx.x >> 3)] = high;
        top = fmaxf(top, high);
    }
    const bool masses = set.masses();
    if (masses)
        for (int b = threadIdx.x; b < kMassBuckets; b += THREADS) sh.masses[b] = 0;
    top = block_top<THREADS>(top, sh.tops);
    if (!set.sums() || top == -INFINITY) return top;
    float base = top;
    if (top == INFINITY) {  // infinity less infinity is none
        base = 0.0f;
#pragma unroll
        for (int r = 0; r < kRounds; r++)
#pragma unroll
            for (int i = 0; i < kVec; i++) raw[r][i] = static_cast<T>(static_cast<float>(raw[r][i]) == INFINITY ? 0.0f : -INFINITY);
    }
    const double turn = set.turn(), grid = set.grid();
    const int place = grid_place(top, grid), rest = octave_rest(place);
    const auto sum_up = [&](auto counted) {
        double all = 0.0;
#pragma unroll
        for (int r = 0; r < kRounds; r++) {
            double sum = 0.0;
#pragma unroll
            for (int i = 0; i < kVec; i++) {
                const float x = static_cast<float>(raw[r][i]);  // (NaN: nothing)
                const double z = (static_cast<double>(x) - base) * turn, v = weight_of(z, powers);
                sum += v;
                if constexpr (decltype(counted)::value) {
                    // (what has no place on the grid has a w of nothing)
                    const unsigned b = static_cast<unsigned>(place - grid_place(x, grid));
                    if (z > kLeastTurns && b < kMassBuckets) atomicAdd(&sh.masses[b], whole_number(v, power_of_two(kMassBits + octaves_to(static_cast<int>(b), rest))));
                }
            }
            if constexpr (decltype(counted)::value) {
                all += sum;
            } else {
                sum = wave_scan(sum);
                if (lane == 63) sh.segments[r * (THREADS / 64) + wave] = sum;
            }
        }
        if constexpr (decltype(counted)::value) {
            all = wave_scan(all);
            if (lane == 63) sh.segments[wave] = all;
        }
    };
    // (with buckets the first THREADS / 64 sums are those of the wavefronts over the whole chunk)
    if (masses && set.on_grid(top)) {
        sum_up(std::true_type{});
    } else {
        sum_up(std::false_type{});
    }
    return top;
}

// ---------------------------------------------------------- histograms over the row

// The bucket in which the running total of sh.bins, from bucket 0 on, reaches `target`, or all there is if that is less; for targets of zero
// and less the first that holds anything.  The totals before it and of all are left in sh.above and `all`.
__device__ __forceinline__ int find_bucket(PickShared& sh, double target, unsigned long long& all) {
    constexpr int kOwn = kBuckets / kSampleThreads;
    __syncthreads();
    unsigned long long own[kOwn], sum = 0;
#pragma unroll
    for (int k = 0; k < kOwn; k++) sum += own[k] = sh.bins[kOwn * threadIdx.x + k];
    unsigned long long before = block_scan(sum, sh.scan, all);
    target = fmin(target, static_cast<double>(all));
#pragma unroll
    for (int k = 0; k < kOwn; k++) {
        if (own[k] > 0 && (before == 0 || static_cast<double>(before) < target) && static_cast<double>(before + own[k]) >= target) {
            sh.bucket = kOwn * static_cast<int>(threadIdx.x) + k;
            sh.above = before;
        }
        before += own[k];
    }
    __syncthreads();
    return sh.bucket;
}

// The same for w of `buckets` buckets, value(b) of each, of which one is above zero: the last in front of which the running total is below the
// target (a total that rounding leaves between two threads' takes the same one in every thread).  Leaves the total before it in sh.mass_above, with it in
// sh.mass_upto.
template <int BUCKETS, typename F>
__device__ __forceinline__ int find_mass(PickShared& sh, double target, F&& value) {
    constexpr int kOwn = BUCKETS / kSampleThreads;
    const int first = kOwn * static_cast<int>(threadIdx.x);
    __syncthreads();
    double own[kOwn], sum = 0.0, all;
#pragma unroll
    for (int k = 0; k < kOwn; k++) sum += own[k] = value(first + k);
    if (threadIdx.x == 0) sh.bucket = 0;
    const double before = block_scan(sum, sh.sums, all);
    double running = before;
    int last = -1;
#pragma unroll
    for (int k = 0; k < kOwn; k++) {
        if (own[k] > 0.0 && (running == 0.0 || running < target)) last = first + k;
        running += own[k];
    }
    // (one atomic a wavefront: one for each bucket before the target took 7 us of a flat row of 201001)
    const unsigned long long any = __ballot(last >= 0);
    if (any && static_cast<int>(threadIdx.x & 63) == 63 - __clzll(any)) atomicMax(&sh.bucket, last);
    __syncthreads();
    const int bucket = sh.bucket;
    running = before;
#pragma unroll
    for (int k = 0; k < kOwn; k++) {
        if (first + k == bucket) {
            sh.mass_above = running;
            sh.mass_upto = running + own[k];
        }
        running += own[k];
    }
    __syncthreads();
    return bucket;
}

// The cut behind which the running total, in the order of the tokens, of 1 (MASS: of w) per token that `kept` keeps reaches
// `target`.  Buckets of x relative to the largest first, then of the keys of one bucket, finer and finer, then equal keys by
// their index.  Tokens whose w are nothing are left out.
template <int TYPE, bool MASS>
__device__ __noinline__ Cut find_cut(const SampleRow<TYPE>& row, const SampleWeights& w, int scale_bits, const Cut& kept, double target, PickShared& sh) {
    const double fine = kBuckets / -kLeastTurns;
    // w of bucket b are 2^(-44 b / kBuckets) and less; the whole powers of two in it
    static_assert(kLeastPower * 512 == 22528.0 && kBuckets == 2048, "");
    const auto octaves = [](int b) { return b * 11 >> 9; };
    const auto counts = [&](float x) { return w.turns(x) > kLeastTurns; };
    const auto bucket_of = [&](float x) { return min(static_cast<int>(-w.turns(x) * fine), kBuckets - 1); };
    const auto clear = [&] {
        __syncthreads();
        for (int b = threadIdx.x; b < kBuckets; b += kSampleThreads) sh.bins[b] = 0;
        __syncthreads();
    };
    clear();
    row.each([&](float x, int i) {
        if (!counts(x) || !kept.keeps(order_key(x), i)) return;
        const int b = bucket_of(x);
        atomicAdd(&sh.bins[b], MASS ? whole_number(w.weight(x), power_of_two(scale_bits + octaves(b))) : 1ull);
    });
    int bucket;
    unsigned long long above = 0, all;
    double scale = 1.0;  // of the bucket
    if constexpr (MASS) {
        bucket = find_mass<kBuckets>(sh, target, [&](int b) { return static_cast<double>(sh.bins[b]) * power_of_two(-scale_bits - octaves(b)); });
        scale = power_of_two(scale_bits + octaves(bucket));
        target = (target - sh.mass_above) * scale;
    } else {
        bucket = find_bucket(sh, target, all);
        if (static_cast<double>(all) < target) return kept;  // (there are fewer)
        above = sh.above;
    }
    const auto amount = [&](float x) { return MASS ? whole_number(w.weight(x), scale) : 1ull; };
    if (threadIdx.x == 0) {
        sh.low = 0xFFFFFFFFu;
        sh.high = 0;
    }
    __syncthreads();
    row.each([&](float x, int i) {
        if (counts(x) && bucket_of(x) == bucket && kept.keeps(order_key(x), i)) {
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
    const double each = MASS ? w.weight(key_value(low)) * scale : 1.0;
    const double wanted = ceil((target - static_cast<double>(above)) / each);
    const int take = wanted < 1.0 ? 1 : wanted > 1e9 ? 1000000000 : static_cast<int>(wanted);
    Cut cut;
    cut.key = low;
    if (threadIdx.x == 0) sh.found = 0x7FFFFFFF;
    int counted = 0;
    for (int from = 0; from < row.vocab && counted < take; from += kSampleThreads * kVec) {
        const int i0 = from + static_cast<int>(threadIdx.x) * kVec;
        float x[kVec];
        unsigned equal = 0;
        if (i0 < row.vocab) {
            row.load(i0, x);
#pragma unroll
            for (int i = 0; i < kVec; i++)
                if (i0 + i < row.vocab && order_key(x[i]) == low && kept.keeps(low, i0 + i)) equal |= 1u << i;
        }
        int here;
        const int before = counted + block_scan(static_cast<int>(__popc(equal)), sh.ints, here);
        if (before < take && before + __popc(equal) >= take) {
            for (int n = take - before; n > 1; n--) equal &= equal - 1;
            sh.found = i0 + __ffs(equal) - 1;
        }
        counted += here;
    }
    __syncthreads();
    cut.index = sh.found;
    return cut;
}

// ------------------------------------------------------------------------ lists

__device__ __forceinline__ unsigned long long read_lane(unsigned long long v, int lane) {
    return static_cast<unsigned long long>(static_cast<unsigned>(__builtin_amdgcn_readlane(static_cast<int>(v >> 32), lane))) << 32
           | static_cast<unsigned>(__builtin_amdgcn_readlane(static_cast<int>(v), lane));
}
__device__ __forceinline__ unsigned long long to_lane(unsigned long long v, int lane) {
    return static_cast<unsigned long long>(static_cast<unsigned>(__builtin_amdgcn_ds_permute(lane * 4, static_cast<int>(v >> 32)))) << 32
           | static_cast<unsigned>(__builtin_amdgcn_ds_permute(lane * 4, static_cast<int>(v)));
}

// A number of each lane's, all different: how many are smaller among the first n lanes'.
__device__ __forceinline__ int rank_in_wave(unsigned long long mine, int n) {
    int rank = 0;
    for (int j = 0; j < n; j++) rank += read_lane(mine, j) < mine;
    return rank;
}
__device__ __forceinline__ int rank_in_wave(unsigned mine, int n) {
    int rank = 0;
    for (int j = 0; j < n; j++) rank += static_cast<unsigned>(__builtin_amdgcn_readlane(static_cast<int>(mine), j)) < mine;
    return rank;
}

// n different numbers of sh.list in ascending order; what lies behind them, up to the next power of two, is overwritten.  Up to a number for each thread:
// every wavefront orders its own, and each finds its place among the others' by halves.  More are sorted by pairs, each of whose steps is a meeting of all.
__device__ __forceinline__ void sort_list(PickShared& sh, int n) {
    if (n <= kSampleThreads) {
        const int wave = static_cast<int>(threadIdx.x) >> 6, runs = (n + 63) / 64;
        __syncthreads();
        const unsigned long long mine = static_cast<int>(threadIdx.x) < n ? sh.list[threadIdx.x] : ~0ull << 11 | threadIdx.x;  // (behind all others)
        const int rank = wave < runs ? rank_in_wave(mine, 64) : 0;
        sh.list[wave * 64 + rank] = mine;  // (a wavefront's own places)
        __syncthreads();
        int place = rank;
        for (int run = 0; run < runs; run++) {
            if (run == wave) continue;
            int before = 0;
#pragma unroll
            for (int step = 32; step > 0; step /= 2) before += sh.list[run * 64 + before + step - 1] < mine ? step : 0;
            place += before + (sh.list[run * 64 + before] < mine);
        }
        __syncthreads();
        if (static_cast<int>(threadIdx.x) < n) sh.list[place] = mine;
        __syncthreads();
        return;
    }
    int size = 64;
    while (size < n) size *= 2;
    for (int i = n + static_cast<int>(threadIdx.x); i < size; i += kSampleThreads) sh.list[i] = ~0ull;
    __syncthreads();
    for (int k = 2; k <= size; k *= 2)
        for (int j = k / 2; j > 0; j /= 2) {
            for (int i = threadIdx.x; i < size / 2; i += kSampleThreads) {
                const int a = 2 * i - (i & (j - 1)), b = a + j;
                const unsigned long long u = sh.list[a], v = sh.list[b];
                if ((u > v) == ((a & k) == 0)) {
                    sh.list[a] = v;
                    sh.list[b] = u;
                }
            }
            __syncthreads();
        }
}

// The sorted list's first n tokens' w into sh.weights, and of each thread's share of them, [from, to), the sum before it, and of all.
__device__ __forceinline__ double weigh_list(const SampleWeights& w, int n, int& from, int& to, double& all, PickShared& sh) {
    for (int i = threadIdx.x; i < n; i += kSampleThreads) sh.weights[i] = w.weight(key_value(~static_cast<unsigned>(sh.list[i] >> 32)));
    __syncthreads();
    const int each = (n + kSampleThreads - 1) / kSampleThreads;
    from = min(n, static_cast<int>(threadIdx.x) * each);
    to = min(n, from + each);
    double mine = 0.0;
    for (int i = from; i < to; i++) mine += sh.weights[i];
    return block_scan(mine, sh.sums, all);
}

// How many of them are kept: of w above zero and at least min_p, with less than `target` before them.  All cuts leave the first of what there is: w falls
// and the sum before it grows.
__device__ __forceinline__ int count_kept(double before, int from, int to, double target, double min_p, bool first, PickShared& sh) {
    int kept = 0;
    for (int i = from; i < to; i++) {
        const double v = sh.weights[i];
        kept += v > 0.0 && ((first && i == 0) || (before < target && v >= min_p));
        before += v;
    }
    int all;
    (void)block_scan(kept, sh.ints, all);
    return all;
}

// A place for each lane that `wants` one, counted in *count; one atomic for all of them.
__device__ __forceinline__ int take_places(bool wants, int* count) {
    const unsigned long long all = __ballot(wants);
    if (all == 0) return 0;
    int first = 0;
    if ((threadIdx.x & 63) == 0) first = atomicAdd(count, __popcll(all));
    first = __builtin_amdgcn_readfirstlane(first);
    return first + __popcll(all & ((1ull << (threadIdx.x & 63)) - 1));
}

// The groups' largest logits: the first ones in registers, the others read again each time.
template <typename TOPS>
struct GroupTops {
    static constexpr int kOwn = 8;
    const TOPS& at;
    int groups;
    float own[kOwn];
    __device__ __forceinline__ GroupTops(const TOPS& tops, int n) : at(tops), groups(n) { read(0, own); }
    __device__ __forceinline__ void read(int from, float (&v)[kOwn]) const {
#pragma unroll
        for (int k = 0; k < kOwn; k++) {
            const int g = from + k * kSampleThreads + static_cast<int>(threadIdx.x);
            const float t = at(min(g, groups - 1));
            v[k] = g < groups ? t : -INFINITY;
        }
    }
    // f called by all threads alike
    template <typename F>
    __device__ __forceinline__ void each(F&& f) const {
        float v[kOwn];
#pragma unroll
        for (int k = 0; k < kOwn; k++) v[k] = own[k];
        for (int from = 0; from < groups; from += kOwn * kSampleThreads) {
            if (from > 0) read(from, v);
#pragma unroll
            for (int k = 0; k < kOwn; k++) {
                if (from + k * kSampleThreads >= groups) break;
                f(v[k], from + k * kSampleThreads + static_cast<int>(threadIdx.x));
            }
        }
    }
};

// The least logit, up to `top`, that `may`, where all larger ones may: a wavefront tries 64 at a time.
template <typename F>
__device__ __forceinline__ float least_that(float top, F&& may) {
    unsigned low = order_key(-3.402823466e38f), high = order_key(top);
    while (low < high) {
        const unsigned step = (high - low) / 64 + 1;
        const unsigned mine = min(static_cast<unsigned long long>(high), low + static_cast<unsigned long long>(threadIdx.x & 63) * step);
        const unsigned long long yes = __ballot(may(key_value(mine)));
        const int first = yes ? __ffsll(yes) - 1 : 64;
        const unsigned long long end = low + static_cast<unsigned long long>(first) * step;
        if (first > 0) low += (first - 1) * step + 1;
        if (end < high) high = static_cast<unsigned>(end);
    }
    return key_value(high);
}

// A float a little below x.
__device__ __forceinline__ float below(double x) {
    constexpr float kMost = 3.402823466e38f;
    const unsigned key = order_key(static_cast<float>(fmin(fmax(x, -kMost), kMost)));
    return key_value(max(key - 2, order_key(-kMost)));
}

// Which of the row's logits are from `least` to `most`: f(set bits' count) gives a thread's first place, put(place, index) takes each.  `share` of `shares`.
template <int TYPE, typename F, typename G>
__device__ __forceinline__ void look_through(const SampleRow<TYPE>& row, float least, float most, int share, int shares, F&& places, G&& put) {
    using T = typename SampleRow<TYPE>::T;
    constexpr int kDeep = 8, kStep = kSampleThreads * kVec, kMasks = kDeep * kVec / 32;
    for (int from = share * kDeep * kStep; from < row.vocab; from += shares * kDeep * kStep) {
        const int i0 = from + static_cast<int>(threadIdx.x) * kVec;
        T e[kDeep][kVec];
        unsigned mask[kMasks];
#pragma unroll
        for (int k = 0; k < kDeep; k++) row.load_raw(i0 + k * kStep, e[k]);
        int wants = 0;
#pragma unroll
        for (int m = 0; m < kMasks; m++) {
            mask[m] = 0;
#pragma unroll
            for (int b = 0; b < 32; b++) {
                const float x = static_cast<float>(e[m * 32 / kVec + b / kVec][b % kVec]);
                mask[m] |= x >= least && x <= most ? 1u << b : 0u;
            }
            wants += __popc(mask[m]);
        }
        int at = places(wants);
#pragma unroll
        for (int m = 0; m < kMasks; m++)
            for (; mask[m]; mask[m] &= mask[m] - 1, at++) {
                const int b = m * 32 + __ffs(mask[m]) - 1;
                put(at, i0 + b / kVec * kStep + b % kVec);
            }
    }
}
// Places for all that a wavefront's lanes want, from a counter that `add` adds to.
template <typename F>
__device__ __forceinline__ int wave_places(int wants, F&& add) {
    const int upto = wave_scan(wants);
    int first = 0;
    if ((threadIdx.x & 63) == 63 && upto > 0) first = add(upto);
    return __builtin_amdgcn_readlane(first, 63) + upto - wants;
}
template <int TYPE>
__device__ __forceinline__ unsigned long long list_entry(const SampleRow<TYPE>& row, int index) {
    return static_cast<unsigned long long>(~order_key(row.one(index))) << 32 | static_cast<unsigned>(index);
}

// The tokens of logits from `least` to `most` into sh.list, by (key descending, index).  Returns how many; more than kListed: the list is not
// whole.  Only groups whose largest reaches `least` are looked at.  `fresh`: sh.listed and sh.found are zero already.
template <int TYPE, typename TOPS>
__device__ __forceinline__ int make_list(const SampleRow<TYPE>& row, const TOPS& tops, PickShared& sh, float least, float most, bool fresh) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    if (!fresh) {
        __syncthreads();
        if (threadIdx.x == 0) sh.listed = sh.found = 0;
        __syncthreads();
    }
    tops.each([&](float t, int g) {
        const bool hot = t >= least;
        const int at = take_places(hot, &sh.found);
        if (hot && at < kListed) sh.hot[at] = g;
    });
    __syncthreads();
    const int hot = sh.found;
    const auto add = [&](int n) { return atomicAdd(&sh.listed, n); };
    if (hot <= kListed) {
        constexpr int kDeep = 32;
        for (int h = wave; h < hot; h += kDeep * kSampleWaves) {
            float x[kDeep];
            int index[kDeep];
            unsigned wants = 0;
#pragma unroll
            for (int k = 0; k < kDeep; k++) {
                const int g = h + k * kSampleWaves;
                index[k] = g < hot ? sh.hot[g] * kGroup + lane : row.vocab;
                x[k] = row.one(index[k]);
            }
#pragma unroll
            for (int k = 0; k < kDeep; k++) wants |= x[k] >= least && x[k] <= most ? 1u << k : 0u;
            int at = wave_places(__popc(wants), add);
#pragma unroll
            for (int k = 0; k < kDeep; k++)
                if (wants >> k & 1) {
                    if (at < kListed) sh.list[at] = static_cast<unsigned long long>(~order_key(x[k])) << 32 | static_cast<unsigned>(index[k]);
                    at++;
                }
        }
    } else if (most == INFINITY) {
        return hot;  // (each holds one at least)
    } else {
        look_through(row, least, most, 0, 1, [&](int wants) { return wave_places(wants, add); },
                     [&](int at, int index) {
                         if (at < kListed) sh.list[at] = list_entry(row, index);
                     });
    }
    __syncthreads();
    return sh.listed;
}

// The same for rows that p.shares workgroups look through: -1 to all but the last of them to end.
template <int TYPE>
__device__ __forceinline__ int make_list_together(const SampleParams& p, int r, const SampleRow<TYPE>& row, int share, PickShared& sh, float least, float most) {
    unsigned* const counters = p.counters + 2 * static_cast<size_t>(r);
    unsigned long long* const list = p.lists + static_cast<size_t>(r) * kListed;
    look_through(row, least, most, share, p.shares,
                 [&](int wants) {
                     return wave_places(wants, [&](int n) {
                         return static_cast<int>(__hip_atomic_fetch_add(counters, static_cast<unsigned>(n), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
                     });
                 },
                 [&](int at, int index) {
                     if (at < kListed) __hip_atomic_store(list + at, list_entry(row, index), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                 });
    // the stores have to be out before the workgroup counts as arrived
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    if (threadIdx.x == 0)
        sh.found = __hip_atomic_fetch_add(counters + 1, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == static_cast<unsigned>(p.shares - 1);
    __syncthreads();
    if (!sh.found) return -1;
    const int listed = static_cast<int>(__hip_atomic_load(counters, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
    for (int i = threadIdx.x; i < min(listed, kListed); i += kSampleThreads) sh.list[i] = __hip_atomic_load(list + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    return listed;
}

// The cut among the list's n tokens behind which the running sum of w, `above` before the first of them, reaches `target`; one is kept at least.  The
// tokens are left, in any order, in sh.bins.  Many are first told apart by buckets of their keys, in whole numbers of w times `scale`.
__device__ __forceinline__ Cut cut_list(const SampleWeights& w, int n, double above, double target, double scale, PickShared& sh) {
    constexpr int kOwn = kListed / kSampleThreads;
    unsigned long long own[kOwn];
#pragma unroll
    for (int k = 0; k < kOwn; k++) {
        const int i = static_cast<int>(threadIdx.x) + k * kSampleThreads;
        own[k] = i < n ? sh.list[i] : 0;
    }
    const auto key_of = [&](int k) { return ~static_cast<unsigned>(own[k] >> 32); };
    const auto there = [&](int k) { return static_cast<int>(threadIdx.x) + k * kSampleThreads < n; };
    int bucket = 0, shift = 31;
    unsigned high = 0;
    if (n > kSampleThreads) {
        float most = -INFINITY, least = INFINITY;
#pragma unroll
        for (int k = 0; k < kOwn; k++)
            if (there(k)) {
                most = fmaxf(most, key_value(key_of(k)));
                least = fminf(least, key_value(key_of(k)));
            }
        for (int b = threadIdx.x; b < kBuckets; b += kSampleThreads) sh.bins[b] = 0;
        block_ends(most, least, sh);
        high = order_key(most);
        shift = max(0, 32 - __clz(high - order_key(least)) - 11);
#pragma unroll
        for (int k = 0; k < kOwn; k++)
            if (there(k)) atomicAdd(&sh.bins[(high - key_of(k)) >> shift], whole_number(w.weight(key_value(key_of(k))), scale));
        unsigned long long all;
        bucket = find_bucket(sh, (target - above) * scale, all);
        above += static_cast<double>(sh.above) / scale;
        if (threadIdx.x == 0) sh.listed = 0;
        __syncthreads();
    }
#pragma unroll
    for (int k = 0; k < kOwn; k++) {
        const int i = static_cast<int>(threadIdx.x) + k * kSampleThreads;
        if (i < n) sh.bins[i] = own[k];
        if (n > kSampleThreads) {
            const bool wants = there(k) && static_cast<int>((high - key_of(k)) >> shift) == bucket;
            const int at = take_places(wants, &sh.listed);
            if (wants) sh.list[at] = own[k];
        }
    }
    __syncthreads();
    if (n > kSampleThreads) n = sh.listed;
    sort_list(sh, n);
    int from, to;
    double all;
    const double before = above + weigh_list(w, n, from, to, all, sh);
    const int kept = count_kept(before, from, to, target, 0.0, true, sh);
    Cut cut;
    cut.key = ~static_cast<unsigned>(sh.list[kept - 1] >> 32);
    cut.index = static_cast<int>(static_cast<unsigned>(sh.list[kept - 1]));
    return cut;
}

__device__ __forceinline__ double target_of(const SampleParams& p, int r, double total) {
    const float u = p.uniforms[r];
    return (u > 0.0f ? static_cast<double>(u) : 0.0) * total;  // (NaN: 0)
}

// Draws from the tokens of a wavefront's first `kept` lanes, of indices `index` and w `v`.
__device__ __forceinline__ void draw_few(const SampleParams& p, int r, int index, double v, int kept) {
    const int lane = threadIdx.x & 63;
    const int rank = lane < kept ? rank_in_wave(static_cast<unsigned>(index), kept) : lane;
    index = __builtin_amdgcn_ds_permute(rank * 4, index);
    v = __longlong_as_double(static_cast<long long>(to_lane(static_cast<unsigned long long>(__double_as_longlong(lane < kept ? v : 0.0)), rank)));
    const double upto = wave_scan(v), all = __shfl(upto, 63);
    const unsigned long long hits = __ballot(lane < kept && upto >= target_of(p, r, all));
    if (lane == (hits ? __ffsll(hits) - 1 : kept - 1)) {
        p.ids[r] = index;
        if (p.probs) p.probs[r] = static_cast<float>(v / all);
    }
}

// Draws from the sorted list's first `kept` tokens, whose w are in sh.weights: by their indices.
__device__ __forceinline__ void draw_listed(const SampleParams& p, int r, int kept, PickShared& sh) {
    if (kept <= 64) {
        if (threadIdx.x < 64) draw_few(p, r, static_cast<int>(static_cast<unsigned>(sh.list[threadIdx.x])), sh.weights[threadIdx.x], kept);
        return;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < kept; i += kSampleThreads) sh.list[i] = sh.list[i] << 32 | static_cast<unsigned>(i);  // (the key goes)
    if (threadIdx.x == 0) {
        sh.low = 0xFFFFFFFFu;
        sh.found = 0;
    }
    __syncthreads();
    sort_list(sh, kept);
    const auto weight = [&](int i) { return sh.weights[static_cast<unsigned>(sh.list[i])]; };
    const int each = (kept + kSampleThreads - 1) / kSampleThreads, from = min(kept, static_cast<int>(threadIdx.x) * each), to = min(kept, from + each);
    double mine = 0.0, total;
    for (int i = from; i < to; i++) mine += weight(i);
    double upto = block_scan(mine, sh.sums, total);
    const double target = target_of(p, r, total);
    for (int i = from; i < to; i++) {
        upto += weight(i);
        if (upto >= target) {
            atomicMin(&sh.low, static_cast<unsigned>(i));
            break;
        }
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        const int at = min(static_cast<int>(min(sh.low, 0x7FFFFFFFu)), kept - 1);
        p.ids[r] = static_cast<int>(sh.list[at] >> 32);
        if (p.probs) p.probs[r] = static_cast<float>(weight(at) / total);
    }
}

// A list of at most 64 tokens from its order to the pick, by one wavefront, a token to a lane.
__device__ __forceinline__ void pick_few(const SampleParams& p, int r, const SampleWeights& w, const SampleSettings& set, int n, double total, const PickShared& sh) {
    const int lane = threadIdx.x;
    unsigned long long item = lane < n ? sh.list[lane] : ~0ull << 32 | static_cast<unsigned>(lane);
    item = to_lane(item, lane < n ? rank_in_wave(item, n) : lane);
    if (set.top_k > 0) n = min(n, set.top_k);
    double v = lane < n ? w.weight(key_value(~static_cast<unsigned>(item >> 32))) : 0.0;
    double upto = wave_scan(v), before = __shfl_up(upto, 1);
    if (lane == 0) before = 0.0;
    const double target = set.top_p < 1.0 ? set.top_p * (set.top_k > 0 ? __shfl(upto, 63) : total) : INFINITY;
    const int kept = __popcll(__ballot(v > 0.0 && (lane == 0 || (before < target && v >= set.min_p))));
    draw_few(p, r, static_cast<int>(static_cast<unsigned>(item)), v, kept);
}

// ------------------------------------------------------------- segments of the row

// Sums of what `weight` keeps of segments [first, first + count) into sh.segments.
template <int TYPE, typename F>
__device__ __forceinline__ void sum_segments(const SampleRow<TYPE>& row, int first, int count, PickShared& sh, F&& weight) {
    constexpr int kDeep = 8;
    __syncthreads();
    for (int s0 = threadIdx.x >> 6; s0 < count; s0 += kDeep * kSampleWaves) {
        typename SampleRow<TYPE>::T e[kDeep][kVec];
#pragma unroll
        for (int k = 0; k < kDeep; k++) row.load_raw((first + s0 + k * kSampleWaves) * kSegment + static_cast<int>(threadIdx.x & 63) * kVec, e[k]);
#pragma unroll
        for (int k = 0; k < kDeep; k++) {
            const int s = s0 + k * kSampleWaves;
            if (s >= count) break;
            const int i0 = (first + s) * kSegment + static_cast<int>(threadIdx.x & 63) * kVec;
            double sum = 0.0;
#pragma unroll
            for (int i = 0; i < kVec; i++) sum += weight(SampleRow<TYPE>::clean(e[k][i]), i0 + i);
            sum = wave_scan(sum);
            if ((threadIdx.x & 63) == 63) sh.segments[s] = sum;
        }
    }
}

// Draws from what `weight` keeps of `count` segments from `first` on, whose sums are in sh.segments: `ahead` is kept before them and `total` of the
// whole row (negative: what they hold).
template <int TYPE, typename F>
__device__ __forceinline__ void draw_segments(const SampleParams& p, int r, const SampleRow<TYPE>& row, int first, int count, double ahead, double total,
                                              PickShared& sh, F&& weight) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    __syncthreads();
    const int each = (count + kSampleThreads - 1) / kSampleThreads, from = min(count, static_cast<int>(threadIdx.x) * each), to = min(count, from + each);
    double mine = 0.0, all;
    for (int s = from; s < to; s++) mine += sh.segments[s];
    if (threadIdx.x == 0) sh.found = -1;
    const double before = block_scan(mine, sh.sums, all);
    if (total < 0.0) total = all;
    const double target = target_of(p, r, total) - ahead;
    // the last segment whose running total before it is below the target, among those that hold anything
    double below = before;
    for (int s = from; s < to; s++) {
        if (sh.segments[s] > 0.0 && (below < target || below == 0.0)) atomicMax(&sh.found, s);
        below += sh.segments[s];
    }
    __syncthreads();
    const int segment = sh.found;
    if (segment >= from && segment < to) {
        below = before;
        for (int s = from; s < segment; s++) below += sh.segments[s];
        sh.sums[0] = below;
    }
    __syncthreads();
    if (wave != 0) return;
    // A chunk's sums hold what is nothing beside the row's largest: a segment that has nothing else gives way to the next that has a kept token, or
    // to the last one before it.
    int here = segment, step = 1, i0;
    double v[kVec], sum;
    for (;;) {
        i0 = (first + here) * kSegment + lane * kVec;
        float x[kVec];
        row.load(i0, x);
        sum = 0.0;
#pragma unroll
        for (int i = 0; i < kVec; i++) sum += v[i] = weight(x[i], i0 + i);
        if (__ballot(sum > 0.0)) break;
        do {
            here += step;
            if (here == count) {
                step = -1;
                here = segment - 1;
            }
        } while (here >= 0 && !(sh.segments[here] > 0.0));
        if (here < 0) return;  // (not reached: the row's largest has a w of 1)
    }
    const double upto = wave_scan(sum), shifted = __shfl_up(upto, 1);
    double running = (here == segment ? sh.sums[0] : here > segment ? target : -INFINITY) + (lane == 0 ? 0.0 : shifted);
    int hit = -1, last = -1;
    double hit_weight = 0.0, last_weight = 0.0;
#pragma unroll
    for (int i = 0; i < kVec; i++) {
        running += v[i];
        if (v[i] > 0.0) {
            last = i;
            last_weight = v[i];
            if (running >= target && hit < 0) {
                hit = i;
                hit_weight = v[i];
            }
        }
    }
    const unsigned long long hits = __ballot(hit >= 0), lasts = __ballot(last >= 0);
    const int chosen = hits ? __ffsll(hits) - 1 : 63 - __clzll(lasts);
    if (lane == chosen) {
        p.ids[r] = i0 + (hits ? hit : last);
        if (p.probs) p.probs[r] = static_cast<float>((hits ? hit_weight : last_weight) / total);
    }
}

// ----------------------------------------------------------------------- a row

// From what the chunks left to the pick.  group_top(g), chunk_top(c), segment_sum(s) and mass(c, place on the grid), the last two relative to their chunk's
// largest and only there where that is not minus infinity.  `share`: this workgroup's of the row's (p.shares).
template <int TYPE, typename GROUP, typename CHUNK, typename SEGMENT, typename MASS>
__device__ __forceinline__ void pick_row(const SampleParams& p, int r, const SampleRow<TYPE>& row, const SampleSettings& set, int chunk, int chunks, int share,
                                         const GROUP& group_top, const CHUNK& chunk_top, const SEGMENT& segment_sum, const MASS& mass, const double* powers, PickShared& sh) {
    const int lane = threadIdx.x & 63;
    if (share > 0 && !set.masses()) return;  // (the first alone has work)
    // what the chunks left is requested in the order in which it is wanted, all of it before the first is there
    static_assert(kMaxSampleVocab / kChunk <= 128, "");
    const float tops_here = fmaxf(chunk_top(min(lane, chunks - 1)), chunk_top(min(lane + 64, chunks - 1)));
    const float own_top = chunk_top(min(static_cast<int>(threadIdx.x), chunks - 1));
    constexpr int kOwnMasses = kMassBuckets / kSampleThreads, kFirst = 8;
    unsigned long long masses_here[kFirst][kOwnMasses];
    const auto read_masses = [&](int c0, unsigned long long (&v)[kFirst][kOwnMasses]) {
#pragma unroll
        for (int d = 0; d < kFirst; d++)
#pragma unroll
            for (int k = 0; k < kOwnMasses; k++) v[d][k] = mass(min(c0 + d, chunks - 1), static_cast<int>(threadIdx.x) + k * kSampleThreads);
    };
    if (set.masses()) read_masses(0, masses_here);
    const GroupTops<GROUP> tops(group_top, groups_of(p.vocab));
    const float top = wave_max(tops_here);
    if (threadIdx.x == 0) sh.listed = sh.found = 0;
    if (top == -INFINITY) {
        if (threadIdx.x == 0) {
            p.ids[r] = -1;
            if (p.probs) p.probs[r] = 0.0f;
        }
        return;
    }
    if (set.greedy()) {
        if (threadIdx.x == 0) sh.low = 0xFFFFFFFFu;
        __syncthreads();
        tops.each([&](float t, int g) {
            if (t == top) atomicMin(&sh.low, static_cast<unsigned>(g));
        });
        __syncthreads();
        if (threadIdx.x < 64) {
            const int g = static_cast<int>(sh.low);
            const unsigned long long here = __ballot(row.one(g * kGroup + static_cast<int>(threadIdx.x)) == top);
            if (threadIdx.x == 0) {
                p.ids[r] = g * kGroup + __ffsll(here) - 1;
                if (p.probs) p.probs[r] = 1.0f;
            }
        }
        return;
    }
    const SampleWeights w{top, set.turn(), powers};
    const int segments = segments_of(p.vocab);
    const double grid = set.grid();
    const int place = grid_place(top, grid), rest = octave_rest(place);
    __syncthreads();  // (the table of powers, which every wavefront filled a part of, is whole; loads go on)
    if (set.sums() && static_cast<int>(threadIdx.x) < chunks) {
        const double chunk_share = w.weight(own_top);
        sh.chunk_shares[threadIdx.x] = chunk_share;
        const int shift = chunk_share > 0.0 ? min(place - grid_place(own_top, grid), kMassBuckets) : kMassBuckets;
        sh.chunk_shifts[threadIdx.x] = shift;
        sh.chunk_scales[threadIdx.x] = chunk_share * power_of_two(octaves_to(shift, rest));
    }
    __syncthreads();
    const auto sum_of = [&](int s) {
        const double chunk_share = sh.chunk_shares[s * kSegment / chunk];
        return chunk_share > 0.0 ? segment_sum(s) * chunk_share : 0.0;
    };

    if (set.sums() && set.top_p == 1.0) {  // nothing is cut
        constexpr int kOwn = kMaxSegments / kSampleThreads;
        double own[kOwn];
#pragma unroll
        for (int k = 0; k < kOwn; k++) {
            const int s = static_cast<int>(threadIdx.x) + k * kSampleThreads;
            own[k] = s < segments ? sum_of(s) : 0.0;
        }
#pragma unroll
        for (int k = 0; k < kOwn; k++) sh.segments[threadIdx.x + k * kSampleThreads] = own[k];
        draw_segments(p, r, row, 0, segments, 0.0, -1.0, sh, [&](float x, int) { return w.weight(x); });
        return;
    }

    // The logit of w = min_p, or one a little below it, by more than the error of a w: of a hot row (T of 1e38) many logits have the same
    const auto min_p_reach = [&] { return top + (kPowers * log2(set.min_p) - 1e-9) / w.turn; };
    Cut cut;
    double total = 0.0;  // of what top-p is a share of
    int listed = kListed + 1;
    if (set.top_k > 0) {
        // Buckets of the logits, from the largest down, and the one that holds the k-th largest of the groups' largest, or of all where groups are few.
        // Groups without a w are left out: one of nothing but forbidden tokens, at the type's lowest value, would stretch the first bucket over all the others
        // (32 x 50257, fp32, k = 40: 17 us, with them 198)
        if (set.top_k <= kListed) {
            const float nothing = below(static_cast<double>(top) + kLeastTurns / w.turn);
            float high = top, low = INFINITY;
            tops.each([&](float t, int) { low = t >= nothing ? fminf(low, t) : low; });
            block_ends(high, low, sh);
            double fine = 0.0;
            const auto bucket_of = [&](float x) { return x == top ? 0 : static_cast<int>(fmin((static_cast<double>(top) - x) * fine, 1e9)); };
            int bound = kBuckets;
            for (int by_group = 4 * set.top_k <= 3 * tops.groups; by_group >= 0 && bound == kBuckets; by_group--) {
                fine = by_group ? (kBuckets - 1) / fmax(static_cast<double>(top) - low, 1e-300) : kBuckets / -kLeastTurns * w.turn;
                for (int b = threadIdx.x; b < kBuckets; b += kSampleThreads) sh.counts[b] = 0;
                if (threadIdx.x == 0) sh.bucket = kBuckets;
                __syncthreads();
                const auto count = [&](float x, int) {
                    if (!(x >= nothing)) return;
                    if (const int b = bucket_of(x); b < kBuckets) atomicAdd(&sh.counts[b], 1u);
                };
                if (by_group) {
                    tops.each(count);
                } else {
                    row.each(count);
                }
                __syncthreads();
                constexpr int kOwn = kBuckets / kSampleThreads;
                int own[kOwn], sum = 0, all;
#pragma unroll
                for (int k = 0; k < kOwn; k++) sum += own[k] = static_cast<int>(sh.counts[kOwn * threadIdx.x + k]);
                int before = block_scan(sum, sh.ints, all);
#pragma unroll
                for (int k = 0; k < kOwn; k++) {
                    if (before < set.top_k && before + own[k] >= set.top_k) sh.bucket = kOwn * static_cast<int>(threadIdx.x) + k;
                    before += own[k];
                }
                __syncthreads();
                bound = sh.bucket;
            }
            // (none: fewer than k tokens have a w)
            listed = make_list(row, tops, sh, below(static_cast<double>(top) - (bound + 1) / fine), INFINITY, true);
        }
        if (listed > kListed) {
            cut = find_cut<TYPE, false>(row, w, p.scale_bits, cut, set.top_k, sh);
            if (set.top_p < 1.0) {
                double mine = 0.0, all;
                row.each([&](float x, int i) { mine += w.weight(cut.keeps(order_key(x), i) ? x : -INFINITY); });
                (void)block_scan(mine, sh.sums, all);
                cut = find_cut<TYPE, true>(row, w, p.scale_bits, cut, set.top_p * all, sh);
            }
        }
    } else if (set.top_p < 1.0) {
        double mine = 0.0;
        const int waves = chunk / (kVec * kRounds * 64);
        for (int i = threadIdx.x; i < chunks * waves; i += kSampleThreads)
            if (const int s = i / waves * (chunk / kSegment) + i % waves; s < segments) mine += sum_of(s);
        (void)block_scan(mine, sh.sums, total);
        const double target = set.top_p * total;
        int bound = kMassBuckets;
        // a thread's places on the grid, and how far they lie behind the row's largest
        const auto bucket_at = [&](int k) { return (place - static_cast<int>(threadIdx.x) - k * kSampleThreads) & (kMassBuckets - 1); };
        const auto unit_at = [&](int k) { return power_of_two(-kMassBits - octaves_to(bucket_at(k), rest)); };
        if (set.on_grid(top, 0x1p29)) {
            // w by buckets, of all chunks, and the one in which their running sum reaches the target
            constexpr int kOwn = kOwnMasses;
            double own[kOwn];
#pragma unroll
            for (int k = 0; k < kOwn; k++) own[k] = 0.0;
            for (int c0 = 0; c0 < chunks; c0 += kFirst) {
                if (c0 > 0) read_masses(c0, masses_here);
#pragma unroll
                for (int d = 0; d < kFirst; d++) {
                    const int shift = c0 + d < chunks ? sh.chunk_shifts[c0 + d] : kMassBuckets;
                    const double chunk_scale = c0 + d < chunks ? sh.chunk_scales[c0 + d] : 0.0;
#pragma unroll
                    for (int k = 0; k < kOwn; k++) own[k] += static_cast<double>(bucket_at(k) >= shift ? masses_here[d][k] : 0) * chunk_scale;
                }
            }
#pragma unroll
            for (int k = 0; k < kOwn; k++) sh.weights[bucket_at(k)] = own[k] * unit_at(k);
            const int bucket = find_mass<kMassBuckets>(sh, target, [&](int b) { return sh.weights[b]; });
            if (sh.mass_upto >= target) bound = bucket;
        }
        if (bound < kMassBuckets) {  // (buckets end there)
            const double above = sh.mass_above;
            const auto bucket_of = [&](float x) { return w.turns(x) > kLeastTurns ? place - grid_place(x, grid) : kMassBuckets; };
            const double reach = (place - bound - 0.5) / grid;
            listed = make_list(row, tops, sh, below(fmax(reach, set.min_p > 0.0 ? min_p_reach() : reach)), INFINITY, true);
            if (listed > kListed) {  // the bucket's own tokens say where the cut is
                const float least = least_that(top, [&](float x) { return bucket_of(x) <= bound; });
                const float next = bound > 0 ? least_that(top, [&](float x) { return bucket_of(x) < bound; }) : INFINITY;
                const float most = bound > 0 ? key_value(order_key(next) - 1) : 3.402823466e38f;
                const bool together = p.shares > 1 && sh.found > kListed;  // (found: the groups that reach so far)
                if (share > 0 && !together) return;
                const int own = together ? make_list_together(p, r, row, share, sh, least, most) : make_list(row, tops, sh, least, most, false);
                if (own < 0) return;
                share = 0;  // (the last of them goes on)
                if (own <= kListed) {
                    const double scale = power_of_two(kMassBits + octaves_to(bound, rest));
                    cut = cut_list(w, own, above, target, scale, sh);
                    if (set.min_p == 0.0 || -log2(set.min_p) * kMassFine > bound + 2) {
                        // what the chunks keep: all above the bucket, and of its own what is kept.  Only the chunk that the draw falls into is read again
                        for (int c = threadIdx.x; c < chunks; c += kSampleThreads) sh.chunk_wholes[c] = 0;
                        __syncthreads();
                        for (int i = threadIdx.x; i < own; i += kSampleThreads) {
                            const unsigned key = ~static_cast<unsigned>(sh.bins[i] >> 32);
                            const int index = static_cast<int>(static_cast<unsigned>(sh.bins[i]));
                            if (cut.keeps(key, index)) atomicAdd(&sh.chunk_wholes[index / chunk], whole_number(w.weight(key_value(key)), scale));
                        }
                        for (int c0 = 0; c0 < chunks; c0 += kFirst) {
                            read_masses(c0, masses_here);
#pragma unroll
                            for (int d = 0; d < kFirst; d++) {
                                const int shift = c0 + d < chunks ? sh.chunk_shifts[c0 + d] : kMassBuckets;
                                double sum = 0.0;
#pragma unroll
                                for (int k = 0; k < kOwnMasses; k++)
                                    if (const int b = bucket_at(k); (b >= shift) & (b < bound)) sum += static_cast<double>(masses_here[d][k]) * unit_at(k);
                                sum = wave_scan(sum);
                                if (c0 + d < chunks && lane == 63) sh.segments[(c0 + d) * kSampleWaves + (threadIdx.x >> 6)] = sum;
                            }
                        }
                        __syncthreads();
                        for (int c = threadIdx.x; c < chunks; c += kSampleThreads) {
                            double sum = 0.0;
                            for (int k = 0; k < kSampleWaves; k++) sum += sh.segments[c * kSampleWaves + k];
                            sh.chunk_sums[c] = sum * sh.chunk_scales[c] + static_cast<double>(sh.chunk_wholes[c]) / scale;
                        }
                        __syncthreads();
                        double held = 0.0;
                        for (int c = 0; c < chunks; c++) held += sh.chunk_sums[c];
                        const double wanted = target_of(p, r, held);
                        int here = -1;
                        double ahead = 0.0, running = 0.0;
                        for (int c = 0; c < chunks; c++) {
                            if (sh.chunk_sums[c] > 0.0 && (running < wanted || running == 0.0)) {
                                here = c;
                                ahead = running;
                            }
                            running += sh.chunk_sums[c];
                        }
                        // (a logit that is left out has a w of nothing: a branch around each exponential would make them follow each other)
                        const auto weight = [&](float x, int i) { return w.weight(cut.keeps(order_key(x), i) ? x : -INFINITY); };
                        const int first = here * (chunk / kSegment), count = min(chunk / kSegment, segments - first);
                        sum_segments(row, first, count, sh, weight);
                        draw_segments(p, r, row, first, count, ahead, held, sh, weight);
                        return;
                    }
                    bound = -1;
                }
            }
        }
        if (share > 0) return;
        if (listed > kListed && bound >= 0) {
            double mine = 0.0, all;
            row.each([&](float x, int) { mine += w.weight(x); });
            (void)block_scan(mine, sh.sums, all);
            cut = find_cut<TYPE, true>(row, w, p.scale_bits, cut, set.top_p * all, sh);
        }
    } else {
        listed = make_list(row, tops, sh, below(min_p_reach()), INFINITY, true);
    }

    if (listed <= 64) {
        if (threadIdx.x < 64) pick_few(p, r, w, set, listed, total, sh);
        return;
    }
    if (listed <= kListed) {
        sort_list(sh, listed);
        if (set.top_k > 0) listed = min(listed, set.top_k);
        int from, to;
        double all;
        const double before = weigh_list(w, listed, from, to, all, sh);
        const double target = set.top_p < 1.0 ? set.top_p * (set.top_k > 0 ? all : total) : INFINITY;
        draw_listed(p, r, count_kept(before, from, to, target, set.min_p, true, sh), sh);
        return;
    }
    const auto weight = [&](float x, int i) {
        const double v = w.weight(cut.keeps(order_key(x), i) ? x : -INFINITY);
        return v >= set.min_p ? v : 0.0;
    };
    sum_segments(row, 0, segments, sh, weight);
    draw_segments(p, r, row, 0, segments, 0.0, -1.0, sh, weight);
}

// A row of one chunk, from its logits to the pick: up to 8192 tokens, one launch.  Nothing in it is bound by memory or arithmetic: it is some 20 steps
// one behind the other (loads, meetings of the workgroup, look-ups in shared memory), which is why few threads do it (5000 tokens in fp32, top-k 40 and
// top-p 0.95: 12 us, of which a launch that does nothing is 4.5).
template <int TYPE>
__global__ __launch_bounds__(kSampleThreads) void sample_row_kernel(const SampleParams p) {
    __shared__ ChunkShared<kSampleThreads> left;
    __shared__ PickShared sh;
    __shared__ double powers[kPowers];
    fill_powers(p, powers);
    const int r = p.first_row + static_cast<int>(blockIdx.x);
    const SampleRow<TYPE> row(p, r);
    const SampleSettings set(p, r);
    const float top = scan_chunk<TYPE, kSampleThreads>(p, row, set, 0, powers, left);
    __syncthreads();
    const int place = grid_place(top, set.grid());
    pick_row(p, r, row, set, kChunk, 1, 0, [&](int g) { return left.group_tops[g]; }, [&](int) { return top; }, [&](int s) { return left.segments[s]; },
             [&](int, int at) { return left.masses[(place - at) & (kMassBuckets - 1)]; }, powers, sh);
}

// One chunk of a row, for sample_pick_kernel.  Several workgroups to a compute unit, so that one reads while the others compute: registers for
// five wavefronts on a SIMD (six cost min-p alone no spills, 27 us for 30, but w and buckets some: 106 for 99; eight 128).
//   256 x 128000 bf16, min-p: 17 us, 3.8 TB/s; 100 x 201001 fp32, top-p: 36 us, 2.2 TB/s, of which the buckets' own units are 2 to 3 (without
//   them 33, and as long with 25 instructions a logit instead of 39, turns and rest by one rounding each); 64 x 50257 bf16, top-p: 9.9.
template <int TYPE, int THREADS>
__global__ __launch_bounds__(THREADS, 5) void sample_scan_kernel(const SampleParams p) {
    __shared__ ChunkShared<THREADS> left;
    __shared__ double powers[kPowers];
    fill_powers(p, powers);
    constexpr int kLength = THREADS * kVec * kRounds, kGroups = kLength / kGroup, kSegments = kLength / kSegment;
    const int c = static_cast<int>(blockIdx.x) % p.chunks, r = p.first_row + static_cast<int>(blockIdx.x) / p.chunks, t = threadIdx.x;
    const SampleRow<TYPE> row(p, r);
    const SampleSettings set(p, r);
    const float top = scan_chunk<TYPE, THREADS>(p, row, set, c * kLength, powers, left);
    __syncthreads();
    for (int g = t; g < kGroups && c * kGroups + g < groups_of(p.vocab); g += THREADS)
        p.group_tops[static_cast<size_t>(r) * groups_of(p.vocab) + c * kGroups + g] = left.group_tops[g];
    if (p.shares > 1 && c == 0 && t < 2) p.counters[2 * static_cast<size_t>(r) + t] = 0;
    if (t == 0) p.chunk_tops[static_cast<size_t>(r) * p.chunks + c] = top;
    if (top == -INFINITY) return;
    if (set.sums() && t < kSegments && c * kSegments + t < segments_of(p.vocab))
        p.segment_sums[static_cast<size_t>(r) * segments_of(p.vocab) + c * kSegments + t] = left.segments[t];
    const int place = grid_place(top, set.grid());
    if (set.masses() && set.on_grid(top))
        for (int b = t; b < kMassBuckets; b += THREADS)
            p.masses[(static_cast<size_t>(r) * p.chunks + c) * kMassBuckets + ((place - b) & (kMassBuckets - 1))] = left.masses[b];
}

// What follows: a workgroup to a row, or several where rows have more groups than a list holds and a nucleus may have to be looked for in all of
// them (launch rules in sample.hip).  Short lists are steps one behind the other, 12.0 to 12.8 us (256 rows of 128000, min-p; 64 of 50257, top-p 0.9); 13 rows of
// 32000 with settings of every kind 22, the time of the row with the longest list; 100 flat rows of 201001, top-p 0.98, 65: 13 for what the chunks
// left (50 MB, read by every workgroup of a row), 16 to look the rows through (80 MB), then 28 of the last workgroup of each: the cut 7, sums of the
// chunks 6, those of the draw's chunk 8, the draw.
template <int TYPE>
__global__ __launch_bounds__(kSampleThreads) void sample_pick_kernel(const SampleParams p, int chunk) {
    __shared__ PickShared sh;
    __shared__ double powers[kPowers];
    const int r = p.first_row + static_cast<int>(blockIdx.x) / p.shares, share = static_cast<int>(blockIdx.x) % p.shares;
    const SampleRow<TYPE> row(p, r);
    const SampleSettings set(p, r);
    fill_powers(p, powers);
    const float* const group_tops = p.group_tops + static_cast<size_t>(r) * groups_of(p.vocab);
    const float* const chunk_tops = p.chunk_tops + static_cast<size_t>(r) * p.chunks;
    const double* const segment_sums = p.segment_sums + static_cast<size_t>(r) * segments_of(p.vocab);
    const unsigned long long* const masses = p.masses + static_cast<size_t>(r) * p.chunks * kMassBuckets;
    pick_row(p, r, row, set, chunk, p.chunks, share, [&](int g) { return group_tops[g]; }, [&](int c) { return chunk_tops[c]; },
             [&](int s) { return segment_sums[s]; }, [&](int c, int at) { return masses[c * kMassBuckets + at]; }, powers, sh);
}

}  // namespace gh
