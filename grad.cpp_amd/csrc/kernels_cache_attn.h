// Attention of a pass's rows over a paged cache.
//
// For row r of a sequence (a token at position t and one of the query heads of a kv head):
//   z_u = scale q.K_u for the visible positions u,   o = sum_u exp(z_u - m) V_u / sum_u exp(z_u - m),   m = max_u z_u,
// in one pass over K and V: a wavefront keeps the running maximum m, its share of the sum and the unnormalised output of its
// rows and corrects the last two when the maximum grows.
//
// Everything runs on the matrix cores with the rows in the COLUMNS of the products: Z^T = K Q^T and O^T = V^T P^T.  A lane
// then holds scores of ONE row (lane & 15) in both products: the maximum, the sum and the correction are values of its own,
// and the probabilities it made are, in the order it made them, the operand that the second product wants from it, because
// which position goes to which of the product's k slots is free as long as K and V agree.  Nothing passes through shared
// memory between the products.  A lane's k slots are positions 4 (lane / 16) .. + 3 of each block of 16.
//
//   Z^T operand K:   lane l holds position l & 15, eight (four) consecutive dims of its quarter l >> 4: one 16-byte load
//   O^T operand V^T: lane l holds c = DH / 16 consecutive dims (l & 15) c .. of its positions: 16 lanes read one whole row of a
//                    head; which of the c products a dim goes to is free too, so products are numbered by the place in
//                    the run.  16-bit elements are paired up over positions in registers (v_perm).
#pragma once

#include "cache_plan.h"
#include "kernels_common.h"

namespace gh {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));

enum { kCacheF32 = 0, kCacheBf16 = 1, kCacheF16 = 2 };

template <int TYPE>
struct CacheType;
template <>
struct CacheType<kCacheF32> {
    using T = float;
    static constexpr int kBytes = 4;
    static constexpr float kLift = 0.0f;
};
template <>
struct CacheType<kCacheBf16> {
    using T = __bf16;
    using V8 = __bf16 __attribute__((ext_vector_type(8)));
    using V2 = __bf16 __attribute__((ext_vector_type(2)));
    static constexpr int kBytes = 2;
    static constexpr float kLift = 0.0f;
    static constexpr unsigned kInf = 0x7F80u, kOne = 0x3F80u;  // infinity's and one's bits
    static __device__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(V8, a), __builtin_bit_cast(V8, b), c, 0, 0, 0);
    }
};
template <>
struct CacheType<kCacheF16> {
    using T = _Float16;
    using V8 = _Float16 __attribute__((ext_vector_type(8)));
    using V2 = _Float16 __attribute__((ext_vector_type(2)));
    static constexpr int kBytes = 2;
    // Probabilities are kept 2^14 times as large (the sum too): one of 2^-28 of the largest is still a normal number.
    static constexpr float kLift = 14.0f;
    static constexpr unsigned kInf = 0x7C00u, kOne = 0x3C00u;
    static __device__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(V8, a), __builtin_bit_cast(V8, b), c, 0, 0, 0);
    }
};

// Where things are in the pool: [page][layer][K, V][kv head][place in the page][dim].
struct CacheLayout {
    char* pool;
    size_t page_bytes;
    size_t run_bytes;  // of one (layer, K or V, head): page_tokens * dim elements
    int kv_heads;
    int dim;
    int page_shift;
    int layers;
};

__device__ __forceinline__ char* cache_run(const CacheLayout& l, int page, int layer, int which, int head) {
    return l.pool + static_cast<size_t>(page) * l.page_bytes + (static_cast<size_t>(layer * 2 + which) * l.kv_heads + head) * l.run_bytes;
}

// Rows of heads of the caller's: element strides.
struct CacheRows {
    char* at;
    long long row, head;
};

struct AttendParams {
    CacheLayout cache;
    CacheRows q, out;
    const int* table;
    const AttendItem* items;
    const AttendJoin* joins;
    const int* maps;
    int layer;
    int group;
    float scale;  // of the scores, times log2(e)
    int causal;
    int window;
    int sinks, lead;    // first positions that rows see beside their window, and those rounded up to 16 (AttendItem)
    int vector_rows;    // q's and out's rows can be read and written 16 bytes at a time
    float* parts;       // [part][kv head][tile height][DH + 4]: output, maximum, sum, two of padding
    unsigned* arrived;  // [join][kv head], zero between launches
};

constexpr int kBeyond = 0x40000000;  // past the end of any run (a run is a megabyte at most)

// Largest value and sum over the four lanes that hold a row (lanes l, l ^ 16, l ^ 32, l ^ 48).
__device__ __forceinline__ float row_max(float v) {
    v = fmaxf(v, __shfl_xor(v, 16));
    return fmaxf(v, __shfl_xor(v, 32));
}
__device__ __forceinline__ float row_sum(float v) {
    v += __shfl_xor(v, 16);
    return v + __shfl_xor(v, 32);
}

// The position that an item's place v is.  Places of one block of 16 are neighbours.
template <bool SINKS>
__device__ __forceinline__ int position_of(const AttendParams& p, const AttendItem& it, int v) {
    return SINKS && v >= p.lead ? v + it.gap : v;
}
// Its page.
template <bool SINKS>
__device__ __forceinline__ int page_of(const AttendParams& p, const AttendItem& it, const int* table, int v) {
    return table[(position_of<SINKS>(p, it, v) >> p.cache.page_shift) - (SINKS && v >= p.lead ? it.hole() : 0)];
}
// What a row at `pos` sees of an item's positions, as bounds: two comparisons an element, where the conditions themselves are some ten.
template <bool SINKS>
struct Visible {
    int low, high, sinks;
    __device__ __forceinline__ Visible(const AttendParams& p, const AttendItem& it, int pos)
        : low(p.window > 0 ? pos - p.window + 1 : 0), high(position_of<SINKS>(p, it, it.k1 - 1)), sinks(p.sinks) {
        if (p.causal) high = min(high, pos);
    }
    __device__ __forceinline__ bool at(int t) const { return (t <= high) & ((t >= low) | (SINKS && t < sinks)); }
};
// Whether a mask cuts `tokens` places from `at` on, for rows at positions first to final; whether none of the rows sees any of them.
// Without conditional evaluation: where a branch of its own stands between a matrix product and what reads the result, the compiler puts
// the product's wait states on one of the two paths only.
template <bool SINKS>
__device__ __forceinline__ bool cuts(const AttendParams& p, const AttendItem& it, int at, int tokens, int first, int final) {
    const int u0 = position_of<SINKS>(p, it, at), u1 = position_of<SINKS>(p, it, at + tokens - 1);
    return ((p.causal != 0) & (u1 > first)) | ((p.window > 0) & (u0 <= final - p.window) & (!SINKS || u1 >= p.sinks));
}
template <bool SINKS>
__device__ __forceinline__ bool hides(const AttendParams& p, const AttendItem& it, int at, int tokens, int first, int final) {
    const int u0 = position_of<SINKS>(p, it, at), u1 = position_of<SINKS>(p, it, at + tokens - 1);
    return ((p.causal != 0) & (u0 > final)) | ((p.window > 0) & (u1 <= first - p.window) & (!SINKS || u0 >= p.sinks));
}

// What a wavefront reads at a time: a granule of 32 (16-bit) or 16 (fp32) positions of one head.
template <int TYPE, int DH>
struct Granule {
    static constexpr bool kWide = TYPE == kCacheF32;
    static constexpr int kTokens = kWide ? 16 : 32;
    static constexpr int kBlocks = kTokens / 16;
    static constexpr int kDims = DH / 16;                      // dims of a lane in V
    static constexpr int kKeyWords = kWide ? DH / 4 : DH / 8;  // of one block
    static constexpr int kValueWords = kWide ? kDims : kDims / 2;  // of one position
    static constexpr int kQuarter = kWide ? 4 : 8;             // dims of 16 bytes
    unsigned k[kBlocks][kKeyWords];
    unsigned v[kBlocks * 4][kValueWords];
};

// The pages of a granule; a block behind the last position may have none: it reads the last one's, and counts for nothing.
template <bool SINKS, int BLOCKS>
__device__ __forceinline__ void look_up(const AttendParams& p, const AttendItem& it, const int* table, int at, int (&pages)[BLOCKS]) {
#pragma unroll
    for (int b = 0; b < BLOCKS; b++) pages[b] = page_of<SINKS>(p, it, table, min(at + 16 * b, it.k1 - 1));
}

// FULL: the head has DH dims.  Otherwise lanes whose dims do not exist read past the end of the run: zeros.
// `pages`: of the granule's blocks of 16 positions, looked up ahead (look_up), or the loads would wait for them one by one.
template <int TYPE, int DH, bool FULL, bool SINKS>
__device__ __forceinline__ void load_granule(const AttendParams& p, const AttendItem& it, const int (&pages)[Granule<TYPE, DH>::kBlocks], int head,
                                             int at, Granule<TYPE, DH>& g) {
    using G = Granule<TYPE, DH>;
    const CacheLayout& cache = p.cache;
    constexpr int kBytes = CacheType<TYPE>::kBytes;
    const int lane = threadIdx.x & 63, row = cache.dim * kBytes;
    const int key_lane = (lane & 15) * row + (lane >> 4) * 16;
    const int value_dim = (lane & 15) * G::kDims;
    const int value_lane = (lane >> 4) * 4 * row + value_dim * kBytes;
#pragma unroll
    for (int b = 0; b < G::kBlocks; b++) {
        const int offset = (position_of<SINKS>(p, it, at + 16 * b) & ((1 << cache.page_shift) - 1)) * row, page = pages[b];
        const char* run = cache_run(cache, page, p.layer, 0, head);
        const __amdgpu_buffer_rsrc_t ks = make_buffer(run, static_cast<unsigned>(cache.run_bytes));
        const __amdgpu_buffer_rsrc_t vs = make_buffer(run + cache.kv_heads * cache.run_bytes, static_cast<unsigned>(cache.run_bytes));
#pragma unroll
        for (int c = 0; c < G::kKeyWords / 4; c++) {
            const bool there = FULL || 4 * G::kQuarter * c + G::kQuarter * (lane >> 4) < cache.dim;
            const u32x4 w = __builtin_bit_cast(
                u32x4, __builtin_amdgcn_raw_buffer_load_b128(ks, there ? key_lane + 64 * c : kBeyond, offset, 0));
            g.k[b][4 * c] = w.x;
            g.k[b][4 * c + 1] = w.y;
            g.k[b][4 * c + 2] = w.z;
            g.k[b][4 * c + 3] = w.w;
        }
#pragma unroll
        for (int i = 0; i < 4; i++) {
            unsigned* to = g.v[4 * b + i];
            if constexpr (G::kValueWords == 1) {
                to[0] = __builtin_amdgcn_raw_buffer_load_b32(vs, FULL || value_dim < cache.dim ? value_lane : kBeyond, offset + i * row, 0);
            } else if constexpr (G::kValueWords == 2) {
                const u32x2 w = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(
                                                              vs, FULL || value_dim < cache.dim ? value_lane : kBeyond, offset + i * row, 0));
                to[0] = w.x;
                to[1] = w.y;
            } else {
#pragma unroll
                for (int c = 0; c < G::kValueWords / 4; c++) {
                    const bool there = FULL || value_dim + G::kQuarter * c < cache.dim;
                    const u32x4 w = __builtin_bit_cast(
                        u32x4, __builtin_amdgcn_raw_buffer_load_b128(vs, there ? value_lane + 16 * c : kBeyond, offset + i * row, 0));
                    to[4 * c] = w.x;
                    to[4 * c + 1] = w.y;
                    to[4 * c + 2] = w.z;
                    to[4 * c + 3] = w.w;
                }
            }
        }
    }
}

// The second product's operand for dims `word`'s low or high halves: a lane's eight positions, two to a register.
template <int WORDS>
__device__ __forceinline__ u32x4 value_operand(const unsigned (&v)[8][WORDS], int word, bool high) {
    const unsigned sel = high ? 0x07060302u : 0x05040100u;
    u32x4 r;
    r.x = __builtin_amdgcn_perm(v[1][word], v[0][word], sel);
    r.y = __builtin_amdgcn_perm(v[3][word], v[2][word], sel);
    r.z = __builtin_amdgcn_perm(v[5][word], v[4][word], sel);
    r.w = __builtin_amdgcn_perm(v[7][word], v[6][word], sel);
    return r;
}

// Infinities and NaN among the values of a granule that some rows may not see: 0 * infinity would reach those rows
// through the product.  Such elements leave the granule (they become zeros) and are added to the rows that do see
// them: a product with visibility in the place of the probabilities counts them, infinity as 1, minus infinity as 64 and
// NaN as 4096 (at most 32 positions, sums below 2^24).  Rare, and only in granules that a mask cuts.
__device__ __forceinline__ float unbounded_sum(float n) {
    const unsigned c = static_cast<unsigned>(n);
    float v = c & 63u ? INFINITY : 0.0f;
    if (c & 4032u) v -= INFINITY;
    return c > 4095u ? NAN : v;
}

// Two 16-bit values: what they count for, and themselves if they are bounded and zero if not.
template <int TYPE>
__device__ __forceinline__ unsigned unbounded_kind(unsigned word) {
    using C = CacheType<TYPE>;
    const typename C::V2 e = __builtin_bit_cast(typename C::V2, word);
    typename C::V2 to;
#pragma unroll
    for (int half = 0; half < 2; half++) {
        const float f = static_cast<float>(e[half]);
        to[half] = static_cast<typename C::T>(f - f == 0.0f ? 0.0f : f > 0.0f ? 1.0f : f < 0.0f ? 64.0f : 4096.0f);
    }
    return __builtin_bit_cast(unsigned, to);
}
template <int TYPE>
__device__ __forceinline__ unsigned bounded(unsigned e) {
    using C = CacheType<TYPE>;
    e = (e & C::kInf) == C::kInf ? e & 0xFFFF0000u : e;
    return (e & (C::kInf << 16)) == (C::kInf << 16) ? e & 0x0000FFFFu : e;
}

template <int TYPE, int DH>
__device__ __forceinline__ void add_unbounded(Granule<TYPE, DH>& g, unsigned seen, f32x4 (&o)[DH / 16]) {
    using G = Granule<TYPE, DH>;
    using C = CacheType<TYPE>;
#pragma unroll
    for (int cc = 0; cc < G::kDims; cc++) {
        f32x4 n{0, 0, 0, 0};
        if constexpr (G::kWide) {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float e = __uint_as_float(g.v[i][cc]);
                const float w = e - e == 0.0f ? 0.0f : e > 0.0f ? 1.0f : e < 0.0f ? 64.0f : 4096.0f;
                n = __builtin_amdgcn_mfma_f32_16x16x4f32(w, static_cast<float>((seen >> i) & 1u), n, 0, 0, 0);
            }
        } else {
            u32x4 a = value_operand(g.v, cc / 2, cc & 1);
#pragma unroll
            for (int w = 0; w < 4; w++) a[w] = unbounded_kind<TYPE>(a[w]);
            u32x4 b;
#pragma unroll
            for (int w = 0; w < 4; w++) b[w] = ((seen >> (2 * w)) & 1u) * C::kOne | ((seen >> (2 * w + 1)) & 1u) * (C::kOne << 16);
            n = C::mfma(a, b, n);
        }
#pragma unroll
        for (int i = 0; i < 4; i++) o[cc][i] += unbounded_sum(n[i]);
    }
#pragma unroll
    for (int i = 0; i < 4 * G::kBlocks; i++)
#pragma unroll
        for (int w = 0; w < G::kValueWords; w++) {
            unsigned& e = g.v[i][w];
            if constexpr (G::kWide) {
                e = (e & 0x7F800000u) == 0x7F800000u ? 0u : e;
            } else {
                e = bounded<TYPE>(e);
            }
        }
}

// Whether a word of the cache's type holds an infinity or NaN: the exponent's bits are all ones.
template <int TYPE>
__device__ __forceinline__ bool unbounded(unsigned w) {
    using C = CacheType<TYPE>;
    if constexpr (TYPE == kCacheF32) {
        return (w & 0x7F800000u) == 0x7F800000u;
    } else {
        return (w & C::kInf) == C::kInf || (w & (C::kInf << 16)) == (C::kInf << 16);
    }
}

template <int TYPE>
__device__ __forceinline__ void store_four(const CacheRows& rows, long long at, bool vector, const f32x4& o) {
    using T = typename CacheType<TYPE>::T;
    typedef T T4 __attribute__((ext_vector_type(4)));
    const T4 v = __builtin_convertvector(o, T4);
    T* to = reinterpret_cast<T*>(rows.at) + at;
    if (vector) {
        *reinterpret_cast<T4*>(to) = v;
    } else {
#pragma unroll
        for (int e = 0; e < 4; e++) to[e] = v[e];
    }
}

// Scores go into the exponent unscaled, scale and maximum in one multiply-add, whose unrounded product may be above the rounded
// maximum: by less than half for maxima up to this, and by the same for all.  Beyond, they are scaled, and rounded, first.
constexpr float kFusedTop = 4194304.0f;

// What a thread has folded of the parts of four output elements: their weighted sum, the maximum it is relative to, the sum.
struct Folded {
    f32x4 out;
    float top, total;
    __device__ __forceinline__ void fold(const f32x4& o, float high, float sum) {
        const float up = fmaxf(top, high);
        const float keep = top == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(top - up);
        const float take = high == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(high - up);
        total = fmaf(total, keep, sum * take);
#pragma unroll
        for (int i = 0; i < 4; i++) out[i] = fmaf(out[i], keep, o[i] * take);
        top = up;
    }
};

constexpr int kMostJoins = 16;  // that wait for one item: it has a row of each at least

struct Meeting {
    int shared_row[kMostJoins + 1];  // where a join's rows begin among the item's
    int last[kMostJoins];            // whether this workgroup is the last for it
};

// Puts together the joins that this workgroup is the last for.  Every trip to memory is a microsecond, so a thread has several
// elements and parts in flight, threads that have no element of their own share the parts, and all joins are made at once; the
// order of the folding is that of the positions, whoever arrived when.  MANY: the item's rows are of several joins.
// stash: 32 bytes of shared memory for each thread.
template <int TYPE, int DH, bool FULL, int HEIGHT, int THREADS, bool MANY>
__device__ __forceinline__ void join_parts(const AttendParams& p, const AttendItem& it, const AttendJoin& mine, int head, const Meeting& meeting,
                                           char* stash) {
    constexpr int kPad = DH + 4, kChunks = DH / 4, kBlock = HEIGHT * kPad;
    constexpr int kSide = HEIGHT > 64 ? 4 : 1, kDeep = HEIGHT > 64 ? 4 : MANY ? 8 : 16;  // elements of a thread and parts, in flight
    const __amdgpu_buffer_rsrc_t rs = make_buffer(p.parts, 0xFFFFFFFFu);  // (the host keeps all parts below 4 GB)
    const int elements = it.rows * kChunks;
    const auto join_of = [&](int e) {
        int j = 0;
        if constexpr (MANY)
            while (j + 1 < it.joins && meeting.shared_row[j + 1] <= e / kChunks) j++;
        return it.join + j;
    };
    const int most = mine.shared_parts + mine.parts;  // (members' own parts of a prefix's rest: one or a few)
    // shares of the parts.  (One where a prefix is among them: its items and the members' own end in any order, have different rows,
    // and have to fold alike.)
    const int shares = MANY || mine.shared_parts > 0 ? 1 : max(1, min(THREADS / elements, (most + kDeep - 1) / kDeep));
    const int share = static_cast<int>(threadIdx.x) / elements;                      // (0 where there is one)
    const auto write = [&](int e, const f32x4& out, float total) {
        const int dim = e % kChunks * 4, j = join_of(e);
        if ((MANY && !meeting.last[j - it.join]) || (!FULL && dim >= p.cache.dim)) return;
        const int r = (MANY ? p.joins[j].r0 - p.joins[j].shared_row : mine.r0) + e / kChunks, row0 = MANY ? p.joins[j].row0 : mine.row0;
        store_four<TYPE>(p.out, (row0 + r / p.group) * p.out.row + (head * p.group + r % p.group) * p.out.head + dim, p.vector_rows,
                         out / total);
    };
    for (int e0 = shares > 1 ? static_cast<int>(threadIdx.x) % elements : threadIdx.x; e0 < elements; e0 += kSide * THREADS) {
        Folded f[kSide];
#pragma unroll
        for (int k = 0; k < kSide; k++) f[k] = {f32x4{0, 0, 0, 0}, -INFINITY, 0.0f};
        const int which = join_of(e0);
        const AttendJoin* const join = MANY ? p.joins + which : &mine;
        const int shared_parts = join->shared_parts, shared_part = join->shared_part, own_part = join->part, shared_row = join->shared_row;
        int all = shared_parts + join->parts;
        if (MANY && !meeting.last[which - it.join]) all = 0;
        const int each = (all + shares - 1) / shares;
        const int skip = MANY ? shared_row : 0;  // rows of the item before the join's
        const int from = shares > 1 ? min(share * each, all) : 0, to = shares > 1 ? min(from + each, all) : all;
        for (int j0 = from; j0 < to; j0 += kDeep) {
            v4i a[kDeep][kSide], st[kDeep][kSide];
#pragma unroll
            for (int j = 0; j < kDeep; j++) {
                const int part = min(j0 + j, all - 1), own = part - shared_parts;
                const int place = own < 0 ? shared_part + part : own_part + own, up = (own < 0 ? shared_row : 0) - skip;
                const unsigned block = static_cast<unsigned>(place * p.cache.kv_heads + head) * (kBlock * 4u);
#pragma unroll
                for (int k = 0; k < kSide; k++) {
                    const int e = min(e0 + k * THREADS, elements - 1);
                    const unsigned row = block + (up + e / kChunks) * (kPad * 4);
                    a[j][k] = coherent_load16(rs, row + e % kChunks * 16);
                    st[j][k] = coherent_load16(rs, row + DH * 4);
                }
            }
#pragma unroll
            for (int j = 0; j < kDeep; j++)
                if (j0 + j < to)
#pragma unroll
                    for (int k = 0; k < kSide; k++)
                        f[k].fold(__builtin_bit_cast(f32x4, a[j][k]), __int_as_float(st[j][k].x), __int_as_float(st[j][k].y));
        }
        if (shares == 1) {
#pragma unroll
            for (int k = 0; k < kSide; k++)
                if (e0 + k * THREADS < elements) write(e0 + k * THREADS, f[k].out, f[k].total);
        } else if (share < shares) {
            *reinterpret_cast<f32x4*>(stash + threadIdx.x * 32) = f[0].out;
            *reinterpret_cast<f32x4*>(stash + threadIdx.x * 32 + 16) = f32x4{f[0].top, f[0].total, 0.0f, 0.0f};
        }
    }
    if (shares == 1) return;
    __syncthreads();
    if (static_cast<int>(threadIdx.x) < elements) {
        Folded f{f32x4{0, 0, 0, 0}, -INFINITY, 0.0f};
        for (int k = 0; k < shares; k++) {
            const char* at = stash + (k * elements + threadIdx.x) * 32;
            const f32x4 st = *reinterpret_cast<const f32x4*>(at + 16);
            f.fold(*reinterpret_cast<const f32x4*>(at), st.x, st.y);
        }
        write(threadIdx.x, f.out, f.total);
    }
}

// The workgroup's part is in memory: it arrives at the joins that wait for it and makes those it is the last for.
template <int TYPE, int DH, bool FULL, int HEIGHT, int THREADS>
__device__ __forceinline__ void finish_parts(const AttendParams& p, const AttendItem& it, const AttendJoin& mine, int head, Meeting& meeting,
                                             char* stash) {
    // the stores have to be out before the workgroup counts as arrived
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    if (static_cast<int>(threadIdx.x) < it.joins) {
        const AttendJoin join = it.joins == 1 ? mine : p.joins[it.join + threadIdx.x];
        unsigned* const arrived = p.arrived + static_cast<size_t>(it.join + threadIdx.x) * p.cache.kv_heads + head;
        const bool last = __hip_atomic_fetch_add(arrived, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT)
                          == static_cast<unsigned>(join.shared_parts + join.parts - 1);
        if (last) __hip_atomic_store(arrived, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        meeting.shared_row[threadIdx.x] = join.shared_row;
        meeting.last[threadIdx.x] = last;
    }
    __syncthreads();
    int any = 0;
    for (int i = 0; i < it.joins; i++) any |= meeting.last[i];
    if (__builtin_amdgcn_readfirstlane(any) == 0) return;
    if constexpr (HEIGHT == 16) {
        if (it.map >= 0) {
            join_parts<TYPE, DH, FULL, HEIGHT, THREADS, true>(p, it, mine, head, meeting, stash);
            return;
        }
    }
    join_parts<TYPE, DH, FULL, HEIGHT, THREADS, false>(p, it, mine, head, meeting, stash);
}

// The join of an item that has one, requested early: at the end it would be one more trip to memory.
__device__ __forceinline__ AttendJoin first_join(const AttendParams& p, const AttendItem& it) {
    return it.joins > 0 ? p.joins[it.join] : AttendJoin{};
}

// Wavefronts of a workgroup: as many as take 128 positions at a time (fp32, one token: 64 sequences of up to 2 k positions
// 88 us, with four 91; bf16 and fp16: 32 sequences at a window of 1024, heads of 80, 15.6 us, with eight 19.2; one of
// 128 k positions 61 and 59), where 256 registers hold what one needs.
constexpr int attend_waves(int type, int dh) { return type == kCacheF32 && dh <= 128 ? 8 : 4; }

// Tiles of 16 rows; the wavefronts of a workgroup share the positions, granule by granule, and meet at the end.
// A tile whose positions were dealt to several workgroups is finished by the last of them to arrive.
//
// Bound by memory: a position is read once for all 16 rows, straight into the registers that the products take, one granule ahead (16
// sequences of 4 k to 32 k positions, 32/8 heads of 128 in bf16, 1.41 GB: 258 us, 5.5 TB/s of the 5.8 that a plain read reaches; 64 of up
// to 2 k, 12 heads of 64 in fp32, 457 MB: 85 us, 5.4 TB/s).  A short pass is bound by its trips one behind the other, items, pages, keys
// and values, joins (one token over 96 positions 5.8 us, of which a launch that does nothing is 4.5).
// With windows and sinks the same: 16 sequences with windows of 4 k and 4 sinks, heads as above, 269 MB: 47 us, 5.8 TB/s; 64 with windows of 512,
// 12 heads of 64 in fp32, 195 MB: 35 us, 5.5 TB/s; one token with a window of 256: 9.0 us, the trips, one part.
template <int TYPE, int DH, bool FULL, bool SINKS>
__global__ __launch_bounds__(64 * attend_waves(TYPE, DH), DH <= 64 ? 4 : 1) void attend_rows_kernel(const AttendParams p) {
    constexpr int kAttendWaves = attend_waves(TYPE, DH);
    using C = CacheType<TYPE>;
    using T = typename C::T;
    using G = Granule<TYPE, DH>;
    constexpr int kDims = G::kDims, kPad = DH + 4;
    __shared__ __align__(16) float meet[kAttendWaves][16][kPad];
    __shared__ float tops[kAttendWaves][16], sums[kAttendWaves][16];
    __shared__ Meeting meeting;

    const AttendItem it = p.items[blockIdx.x / p.cache.kv_heads];
    const int head = blockIdx.x % p.cache.kv_heads;
    const AttendJoin mine = first_join(p, it);
    const int* table = p.table + it.table;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int quarter = lane >> 4;

    // the rows' queries, as the first product's second operand
    unsigned q[G::kKeyWords];
    const bool row = (lane & 15) < it.rows;
    // (a map's rows are of several sequences, all of them behind all of the positions)
    const int r = !row ? 0 : it.map >= 0 ? p.maps[it.map + (lane & 15)] : it.r0 + (lane & 15);
    const int token = r / p.group, h = r % p.group;
    const int pos = !row ? -1 : it.map >= 0 ? it.first : it.first + token;
    const T* from = reinterpret_cast<const T*>(p.q.at) + (it.row0 + token) * p.q.row + (head * p.group + h) * p.q.head;
#pragma unroll
    for (int c = 0; c < G::kKeyWords / 4; c++) {
        const int dim = 4 * G::kQuarter * c + G::kQuarter * quarter;
        u32x4 w{0, 0, 0, 0};
        if (row && (FULL || dim < p.cache.dim)) {
            if (p.vector_rows) {
                w = *reinterpret_cast<const u32x4*>(from + dim);
            } else if constexpr (G::kWide) {
#pragma unroll
                for (int e = 0; e < 4; e++) w[e] = __float_as_uint(from[dim + e]);
            } else {
#pragma unroll
                for (int e = 0; e < 8; e++)
                    w[e / 2] |= static_cast<unsigned>(__builtin_bit_cast(unsigned short, from[dim + e])) << (16 * (e & 1));
            }
        }
#pragma unroll
        for (int e = 0; e < 4; e++) q[4 * c + e] = w[e];
    }
    const int first = it.first + it.r0 / p.group, final = it.first + (it.r0 + it.rows - 1) / p.group;

    f32x4 o[kDims];
    float m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int cc = 0; cc < kDims; cc++) o[cc] = f32x4{0, 0, 0, 0};

    Granule<TYPE, DH> now, next;
    int pages[G::kBlocks];
    int at = it.k0 + wave * G::kTokens;
    if (at < it.k1) {
        look_up<SINKS>(p, it, table, at, pages);
        load_granule<TYPE, DH, FULL, SINKS>(p, it, pages, head, at, now);
        look_up<SINKS>(p, it, table, at + kAttendWaves * G::kTokens, pages);
    }
    while (at < it.k1) {
        const int then = at + kAttendWaves * G::kTokens;
        if (then < it.k1) {
            load_granule<TYPE, DH, FULL, SINKS>(p, it, pages, head, then, next);
            look_up<SINKS>(p, it, table, then + kAttendWaves * G::kTokens, pages);
        }

        // does a mask cut this granule?
        const bool cut = (at + G::kTokens > it.k1) | cuts<SINKS>(p, it, at, G::kTokens, first, final);
        float z[4 * G::kBlocks];
#pragma unroll
        for (int b = 0; b < G::kBlocks; b++) {
            f32x4 acc{0, 0, 0, 0};
            if constexpr (G::kWide) {
                // 64 dims to a chain of products, chains added in fp32: one chain of 256 dims is off by three times a sum in pairs
#pragma unroll
                for (int from = 0; from < G::kKeyWords; from += 16) {
                    f32x4 chain{0, 0, 0, 0};
#pragma unroll
                    for (int w = from; w < from + 16; w++)
                        chain = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(now.k[b][w]), __uint_as_float(q[w]), chain, 0, 0, 0);
                    acc = from == 0 ? chain : acc + chain;
                }
            } else {
#pragma unroll
                for (int w = 0; w < G::kKeyWords; w += 4)
                    acc = C::mfma(u32x4{now.k[b][w], now.k[b][w + 1], now.k[b][w + 2], now.k[b][w + 3]},
                                  u32x4{q[w], q[w + 1], q[w + 2], q[w + 3]}, acc);
            }
#pragma unroll
            for (int i = 0; i < 4; i++) z[4 * b + i] = acc[i];
        }
        unsigned seen = 0;
        bool hidden = false;
        if (cut) {
            const Visible<SINKS> visible(p, it, pos);
#pragma unroll
            for (int i = 0; i < 4 * G::kBlocks; i++) {
                const bool see = visible.at(position_of<SINKS>(p, it, at + 16 * (i / 4)) + 4 * quarter + (i & 3));
                z[i] = see ? z[i] : -INFINITY;
                seen |= see ? 1u << i : 0u;
            }
            // places behind the last position hold anything; a position that some rows may not see is looked at
#pragma unroll
            for (int i = 0; i < 4 * G::kBlocks; i++) {
                const bool there = at + 16 * (i / 4) + 4 * quarter + (i & 3) < it.k1;
#pragma unroll
                for (int w = 0; w < G::kValueWords; w++) {
                    now.v[i][w] = there ? now.v[i][w] : 0u;
                    hidden = hidden || unbounded<TYPE>(now.v[i][w]);
                }
            }
        }
        float top = z[0];
#pragma unroll
        for (int i = 1; i < 4 * G::kBlocks; i++) top = fmaxf(top, z[i]);
        top = __fmul_rn(row_max(top), p.scale);
        if (__any(top > m)) {
            const float keep = top > m ? __builtin_amdgcn_exp2f(m - top) : 1.0f;
            m = fmaxf(m, top);
            l *= keep;
#pragma unroll
            for (int cc = 0; cc < kDims; cc++) o[cc] *= keep;
        }
        const float base = m == -INFINITY ? 0.0f : m - C::kLift;
        float scale = p.scale;
        if (__any(fabsf(base) > kFusedTop)) {
            scale = 1.0f;
#pragma unroll
            for (int i = 0; i < 4 * G::kBlocks; i++) z[i] = __fmul_rn(z[i], p.scale);
        }
#pragma unroll
        for (int i = 0; i < 4 * G::kBlocks; i++) {
            z[i] = __builtin_amdgcn_exp2f(fmaf(z[i], scale, -base));
            l += z[i];
        }
        if (cut && __any(hidden)) add_unbounded<TYPE, DH>(now, seen, o);  // (behind the correction: infinity * 0 is none)
        if constexpr (G::kWide) {
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int cc = 0; cc < kDims; cc++)
                    o[cc] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(now.v[i][cc]), z[i], o[cc], 0, 0, 0);
        } else {
            // probabilities in the cache's type: off by half a step of theirs each, at random, which is what the outputs'
            // own rounding is
            u32x4 prob;
#pragma unroll
            for (int w = 0; w < 4; w++)
                prob[w] = __builtin_bit_cast(unsigned, typename C::V2{static_cast<T>(z[2 * w]), static_cast<T>(z[2 * w + 1])});
#pragma unroll
            for (int cc = 0; cc < kDims; cc++) {
                const u32x4 a = value_operand(now.v, cc / 2, cc & 1);
                o[cc] = C::mfma(a, prob, o[cc]);
            }
        }
        now = next;
        at = then;
    }

    const bool only = it.joins == 0;
    constexpr int kBlock = 16 * kPad;  // floats of a part
    float* const part = p.parts + (static_cast<size_t>(only ? 0 : it.part) * p.cache.kv_heads + head) * kBlock;
    constexpr int kChunks = DH / 4;  // of a row
    const float sum = row_sum(l);
    if (quarter == 0) {
        tops[wave][lane] = m;
        sums[wave][lane] = sum;
    }
    __syncthreads();
    const int own = lane & 15;
    float top = tops[0][own];
#pragma unroll
    for (int w = 1; w < kAttendWaves; w++) top = fmaxf(top, tops[w][own]);
    const float keep = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - top);
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
        for (int cc = 0; cc < kDims; cc++) meet[wave][own][(4 * quarter + i) * kDims + cc] = o[cc][i] * keep;
    __syncthreads();
    for (int e = threadIdx.x; e < 16 * kChunks; e += 64 * kAttendWaves) {
        const int row = e / kChunks, dim = e % kChunks * 4;
        if (row >= it.rows) break;
        float high = tops[0][row], total = 0.0f;
#pragma unroll
        for (int w = 1; w < kAttendWaves; w++) high = fmaxf(high, tops[w][row]);
        f32x4 out{0, 0, 0, 0};
#pragma unroll
        for (int w = 0; w < kAttendWaves; w++) {
            total += sums[w][row] * (tops[w][row] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(tops[w][row] - high));
            out += *reinterpret_cast<const f32x4*>(&meet[w][row][dim]);
        }
        if (only) {
            const int r = it.r0 + row;
            if (FULL || dim < p.cache.dim)
                store_four<TYPE>(p.out, (it.row0 + r / p.group) * p.out.row + (head * p.group + r % p.group) * p.out.head + dim,
                                 p.vector_rows, out / total);
        } else {
            const __amdgpu_buffer_rsrc_t rs = make_buffer(part, kBlock * 4);
            const int base = row * kPad * 4;
            __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(v4i, out), rs, base + dim * 4, 0, kAuxDeviceScope);
            if (dim == 0)
                __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(v4i, f32x4{high, total, 0.0f, 0.0f}), rs, base + DH * 4, 0, kAuxDeviceScope);
        }
    }
    __syncthreads();
    if (only) return;

    finish_parts<TYPE, DH, FULL, 16, 64 * kAttendWaves>(p, it, mine, head, meeting, reinterpret_cast<char*>(meet));
}

}  // namespace gh
