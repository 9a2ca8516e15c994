// Attention of many rows over a paged cache: tiles of 128 rows, 32 to a wavefront, whose positions pass through shared memory
// once for all four.  The mathematics, the transposed products and the order of the k slots are those of
// kernels_cache_attn.h, on 32 x 32 x 16 products: a lane holds scores of row (lane & 31), of the positions
// 8 b + 4 (lane / 32) + j of every 32.
//
// Shared memory holds K and V as they are in the pages, position by position, with a stride that spreads what a product's
// lanes read over all banks: K rows are read 16 bytes to a lane (eight lanes to a cycle: rows 16 bytes apart modulo 128), V through
// the transposing read, which hands a lane four positions of one dim (16 lanes to a cycle: four rows 32 bytes apart modulo 128).
//
// Bound by the products and the softmax between them, which a wavefront does in turn: four sequences of 2048 rows onto 6 k positions,
// 32/8 heads of 128 in bf16, 962 GFLOP: 1.07 to 1.16 ms, 830 to 900 TFLOP/s where a large plain product reaches 1124; of
// a SIMD's cycles 36 % have a product under way and 38 % a vector instruction.  A position that a wavefront fetches itself would be fetched four
// times: 3.6 ms with the 16-row tiles' kernel.
#pragma once

#include "kernels_attn.h"
#include "kernels_cache_attn.h"

namespace gh {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

constexpr int kTileWaves = 4;
constexpr int kTileRows = 32 * kTileWaves;

template <int TYPE>
__device__ __forceinline__ f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c) {
    using C = CacheType<TYPE>;
    using V8 = typename C::V8;
    if constexpr (TYPE == kCacheBf16) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(V8, a), __builtin_bit_cast(V8, b), c, 0, 0, 0);
    } else {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(V8, a), __builtin_bit_cast(V8, b), c, 0, 0, 0);
    }
}

// Largest of a value's two halves of the wavefront, in both.
__device__ __forceinline__ float both_max(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float both_sum(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

__device__ __forceinline__ u32x2 read_transposed(const char* at) {
    const auto r = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        reinterpret_cast<__attribute__((address_space(3))) s16x4*>(reinterpret_cast<uintptr_t>(at)));
    return __builtin_bit_cast(u32x2, r);
}

// Asks the scheduler for PRODUCTS products that have READS reads from shared memory each, with DEEP products' reads under way
// ahead of the first: on its own it reads for one product, waits, multiplies.
template <int PRODUCTS, int READS, int DEEP>
__device__ __forceinline__ void ahead_of_products() {
    constexpr int kRead = 0x100, kProduct = 0x8;
    __builtin_amdgcn_sched_group_barrier(kRead, READS * DEEP, 0);
#pragma unroll
    for (int i = 0; i < PRODUCTS; i++) {
        __builtin_amdgcn_sched_group_barrier(kProduct, 1, 0);
        if (i + DEEP < PRODUCTS) __builtin_amdgcn_sched_group_barrier(kRead, READS, 0);
    }
}

// A wavefront's rows [from, from + rows) of a tile, one after the other and term by term: 64 positions at a time, the scores with a
// position to a lane, the output with a dim to a lane.  What a row may not see takes no part at all, infinities and NaN are what
// they are.  For the tiles that hold such values (a matrix product would carry them to rows that do not see them, and make
// NaN of an infinity's parts): 40 to 100 times as slow as the products (397 rows at 1.6 k with one infinity among the chunk's values:
// fp32, 12 heads of 64, 1.9 ms where 48 us do without; bf16, 32/8 heads of 128, 5.6 ms and 58 us).
template <int TYPE, int DH>
__device__ void rows_one_by_one(const AttendParams& p, const AttendItem& it, const int* table, int head, int from, int rows, float* part) {
    using C = CacheType<TYPE>;
    using T = typename C::T;
    constexpr int kPad = DH + 4, kOwn = DH / 64;
    const int lane = threadIdx.x & 63, dims = p.cache.dim, mask = (1 << p.cache.page_shift) - 1;
    const auto at = [&](int which, int t) {
        return reinterpret_cast<const T*>(cache_run(p.cache, table[t >> p.cache.page_shift], p.layer, which, head)) + static_cast<size_t>(t & mask) * dims;
    };
#pragma unroll 1
    for (int i = from; i < from + rows; i++) {
        const int r = it.r0 + i, token = r / p.group, h = head * p.group + r % p.group, pos = it.first + token;
        const T* query = reinterpret_cast<const T*>(p.q.at) + (it.row0 + token) * p.q.row + h * p.q.head;
        const int begin = p.window > 0 ? max(it.k0, pos - p.window + 1) : it.k0, end = p.causal ? min(it.k1, pos + 1) : it.k1;
        float m = -INFINITY, l = 0.0f, o[kOwn];
#pragma unroll
        for (int k = 0; k < kOwn; k++) o[k] = 0.0f;
#pragma unroll 1
        for (int t0 = begin; t0 < end; t0 += 64) {
            const int n = min(64, end - t0);
            float z = -INFINITY;
            if (lane < n) {
                const T* key = at(0, t0 + lane);
                z = 0.0f;
#pragma unroll 1
                for (int d = 0; d < dims; d++) z = fmaf(static_cast<float>(query[d]), static_cast<float>(key[d]), z);
                z = __fmul_rn(z, p.scale);  // (rounded as the maximum is)
            }
            const float top = fmaxf(m, wave_max(z));
            const float keep = m == top ? 1.0f : __builtin_amdgcn_exp2f(m - top);
            const float prob = lane < n ? __builtin_amdgcn_exp2f(z - (top == -INFINITY ? 0.0f : top - C::kLift)) : 0.0f;
            m = top;
            l = l * keep + wave_sum(prob);
#pragma unroll
            for (int k = 0; k < kOwn; k++) o[k] *= keep;
#pragma unroll 1
            for (int j = 0; j < n; j++) {
                const float w = __shfl(prob, j);
                const T* value = at(1, t0 + j);
#pragma unroll
                for (int k = 0; k < kOwn; k++)
                    if (lane + 64 * k < dims) o[k] = fmaf(w, static_cast<float>(value[lane + 64 * k]), o[k]);
            }
        }
        if (it.joins == 0) {
            T* to = reinterpret_cast<T*>(p.out.at) + (it.row0 + token) * p.out.row + h * p.out.head;
#pragma unroll
            for (int k = 0; k < kOwn; k++)
                if (lane + 64 * k < dims) to[lane + 64 * k] = static_cast<T>(o[k] / l);
        } else {
            float* to = part + i * kPad;
#pragma unroll
            for (int k = 0; k < kOwn; k++) partial_store(to + lane + 64 * k, o[k]);
            if (lane < 2) partial_store(to + DH + lane, lane == 0 ? m : l);
        }
    }
}

// A wavefront's rows, whole and to the caller, or a part of them and to the place of the part.  A lane has every other run of
// four dims of its row.
template <int TYPE, int DH, bool FULL>
__device__ __forceinline__ void leave_rows(const AttendParams& p, const AttendItem& it, const f32x16 (&o)[DH / 32], float m, float l, bool row,
                                           int token, int h, int r, int half, float* part) {
    constexpr int kPad = DH + 4, kBlock = kTileRows * kPad;
    if (!row) return;
    const __amdgpu_buffer_rsrc_t rs = make_buffer(part, kBlock * 4);
    const int base = r * kPad * 4;
    const long long to = (it.row0 + token) * p.out.row + h * p.out.head;
#pragma unroll
    for (int d = 0; d < DH / 32; d++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int dim = 32 * d + 8 * i + 4 * half;
            const f32x4 four{o[d][4 * i], o[d][4 * i + 1], o[d][4 * i + 2], o[d][4 * i + 3]};
            if (it.joins == 0) {
                if (FULL || dim < p.cache.dim) store_four<TYPE>(p.out, to + dim, p.vector_rows, four / l);
            } else {
                __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(v4i, four), rs, base + dim * 4, 0, kAuxDeviceScope);
            }
        }
    if (it.joins > 0 && half == 0)
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(v4i, f32x4{m, l, 0.0f, 0.0f}), rs, base + DH * 4, 0, kAuxDeviceScope);
}

// Sixteen-bit types.  TOKENS positions at a time.
template <int TYPE, int DH, bool FULL, int TOKENS>
__global__ __launch_bounds__(64 * kTileWaves, DH > 128 ? 1 : 2) void attend_tile_kernel(const AttendParams p) {
    using C = CacheType<TYPE>;
    using T = typename C::T;
    constexpr int kKeyRow = DH * 2 + 16, kValueRow = DH * 2 + 32;  // bytes
    constexpr int kUnits = DH / 8;                                  // of 16 bytes in a row
    constexpr int kLoads = TOKENS * kUnits / (64 * kTileWaves);     // of a thread, for K and for V
    constexpr int kBlocks = TOKENS / 32, kSteps = DH / 16, kWide = DH / 32;
    __shared__ __align__(16) char keys[TOKENS * kKeyRow];
    __shared__ __align__(16) char values[TOKENS * kValueRow];
    __shared__ Meeting meeting;
    __shared__ unsigned odd;

    const AttendItem it = p.items[blockIdx.x / p.cache.kv_heads];
    const int head = blockIdx.x % p.cache.kv_heads;
    const AttendJoin mine = first_join(p, it);
    const int* table = p.table + it.table;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int half = lane >> 5;

    // this lane's row and its query
    const int r = it.r0 + 32 * wave + (lane & 31);
    const bool row = 32 * wave + (lane & 31) < it.rows;
    const int token = row ? r / p.group : 0, h = row ? r % p.group : 0;
    const int pos = row ? it.first + token : -1;
    u32x4 q[kSteps];
    {
        const T* from = reinterpret_cast<const T*>(p.q.at) + (it.row0 + token) * p.q.row + (head * p.group + h) * p.q.head;
#pragma unroll
        for (int c = 0; c < kSteps; c++) {
            const int dim = 16 * c + 8 * half;
            q[c] = u32x4{0, 0, 0, 0};
            if (row && (FULL || dim < p.cache.dim)) {
                if (p.vector_rows) {
                    q[c] = *reinterpret_cast<const u32x4*>(from + dim);
                } else {
#pragma unroll
                    for (int e = 0; e < 8; e++)
                        q[c][e / 2] |= static_cast<unsigned>(__builtin_bit_cast(unsigned short, from[dim + e])) << (16 * (e & 1));
                }
            }
        }
    }
    // positions of the tile's and of this wavefront's first and last rows
    const int rows_here = min(32, it.rows - 32 * wave);
    const int first_all = it.first + it.r0 / p.group, final_all = it.first + (it.r0 + it.rows - 1) / p.group;
    const int first = it.first + (it.r0 + 32 * wave) / p.group;
    const int final = it.first + (it.r0 + 32 * wave + max(rows_here, 1) - 1) / p.group;

    f32x16 o[kWide];
#pragma unroll
    for (int d = 0; d < kWide; d++)
#pragma unroll
        for (int i = 0; i < 16; i++) o[d][i] = 0.0f;
    float m = -INFINITY, l = 0.0f;

    // A wavefront's loads are whole rows of one block of 16 positions, so of one page; the pages of the tile behind the next are
    // looked up while the next one is fetched, or every load would wait for its own look at the list.
    u32x4 kr[kLoads], vr[kLoads];
    int pages[kLoads];
    const int bytes = p.cache.dim * 2, own_row = lane / kUnits;
    static_assert(64 % kUnits == 0, "whole rows");
    const int own = FULL || lane % kUnits * 8 < p.cache.dim ? own_row * bytes + lane % kUnits * 16 : kBeyond;
    const auto row_of = [&](int i) { return 64 * (kTileWaves * i + wave) / kUnits; };
    const auto look = [&](int at) {
#pragma unroll
        for (int i = 0; i < kLoads; i++) pages[i] = table[min(at + row_of(i), it.k1 - 1) >> p.cache.page_shift];
    };
    const auto fetch = [&](int at) {
#pragma unroll
        for (int i = 0; i < kLoads; i++) {
            const char* run = cache_run(p.cache, pages[i], p.layer, 0, head);
            const __amdgpu_buffer_rsrc_t ks = make_buffer(run, static_cast<unsigned>(p.cache.run_bytes));
            const __amdgpu_buffer_rsrc_t vs = make_buffer(run + p.cache.kv_heads * p.cache.run_bytes, static_cast<unsigned>(p.cache.run_bytes));
            const int t = at + row_of(i);
            const int offset = t + own_row < it.k1 ? own : kBeyond;  // (places behind the last position: zeros)
            const int base = (t & ((1 << p.cache.page_shift) - 1)) * bytes;
            kr[i] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(ks, offset, base, 0));
            vr[i] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(vs, offset, base, 0));
        }
    };
    // how a lane reads them back
    const char* const key_at = keys + (lane & 31) * kKeyRow + half * 16;
    const char* const value_at = values + (4 * half + ((lane & 15) >> 2)) * kValueRow + 32 * ((lane >> 4) & 1) + 8 * (lane & 3);

    if (threadIdx.x == 0) odd = 0;
    look(it.k0);
    fetch(it.k0);
    look(it.k0 + TOKENS);
    for (int at = it.k0; at < it.k1; at += TOKENS) {
        const bool cut_all = (p.causal && at + TOKENS - 1 > first_all) || (p.window > 0 && at <= final_all - p.window);
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kLoads; i++) {
            const int unit = 64 * (kTileWaves * i + wave) + lane;
            const int to = unit / kUnits, c = unit % kUnits * 16;
            *reinterpret_cast<u32x4*>(keys + to * kKeyRow + c) = kr[i];
            *reinterpret_cast<u32x4*>(values + to * kValueRow + c) = vr[i];
        }
        if (cut_all) {
            bool bad = false;
#pragma unroll
            for (int i = 0; i < kLoads; i++)
#pragma unroll
                for (int w = 0; w < 4; w++) bad = bad || unbounded<TYPE>(vr[i][w]);
            if (bad) odd = 1;
        }
        __syncthreads();
        // Infinities and NaN among values that some rows may not see.  (Nobody writes `odd` before everybody has read it: the next
        // tile is put in place behind the next meeting.)
        if (cut_all && __builtin_amdgcn_readfirstlane(odd)) break;
        if (at + TOKENS < it.k1) {
            fetch(at + TOKENS);
            look(at + 2 * TOKENS);
        }
        if (rows_here <= 0 || (p.causal && at > final) || (p.window > 0 && at + TOKENS - 1 <= first - p.window)) continue;

        f32x16 z[kBlocks];
#pragma unroll
        for (int b = 0; b < kBlocks; b++)
#pragma unroll
            for (int i = 0; i < 16; i++) z[b][i] = 0.0f;
#pragma unroll
        for (int c = 0; c < kSteps; c++)
#pragma unroll
            for (int b = 0; b < kBlocks; b++)
                z[b] = mfma32<TYPE>(*reinterpret_cast<const u32x4*>(key_at + b * 32 * kKeyRow + c * 32), q[c], z[b]);
        ahead_of_products<kBlocks * kSteps, 1, 6>();
        const bool cut = at + TOKENS > it.k1 || (p.causal && at + TOKENS - 1 > first) || (p.window > 0 && at <= final - p.window);
        if (cut) {
#pragma unroll
            for (int b = 0; b < kBlocks; b++)
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    const int t = at + 32 * b + 8 * (i / 4) + 4 * half + (i & 3);
                    const bool see = t < it.k1 && (!p.causal || t <= pos) && (p.window <= 0 || t > pos - p.window);
                    z[b][i] = see ? z[b][i] : -INFINITY;
                }
        }
        float top = z[0][0];
#pragma unroll
        for (int b = 0; b < kBlocks; b++)
#pragma unroll
            for (int i = 0; i < 16; i++) top = fmaxf(top, z[b][i]);
        top = __fmul_rn(both_max(top), p.scale);
        if (__any(top > m)) {
            const float keep = top > m ? __builtin_amdgcn_exp2f(m - top) : 1.0f;
            m = fmaxf(m, top);
            l *= keep;
#pragma unroll
            for (int d = 0; d < kWide; d++)
#pragma unroll
                for (int i = 0; i < 16; i++) o[d][i] *= keep;
        }
        const float base = m == -INFINITY ? 0.0f : m - C::kLift;
        float scale = p.scale;
        if (__any(fabsf(base) > kFusedTop)) {
            scale = 1.0f;
#pragma unroll
            for (int b = 0; b < kBlocks; b++)
#pragma unroll
                for (int i = 0; i < 16; i++) z[b][i] = __fmul_rn(z[b][i], p.scale);
        }
#pragma unroll
        for (int b = 0; b < kBlocks; b++)
#pragma unroll
            for (int i = 0; i < 16; i++) {
                z[b][i] = __builtin_amdgcn_exp2f(fmaf(z[b][i], scale, -base));
                l += z[b][i];
            }
        u32x4 prob[kBlocks][2];
#pragma unroll
        for (int b = 0; b < kBlocks; b++)
#pragma unroll
            for (int u = 0; u < 2; u++)
#pragma unroll
                for (int w = 0; w < 4; w++)
                    prob[b][u][w] = __builtin_bit_cast(
                        unsigned, typename C::V2{static_cast<T>(z[b][8 * u + 2 * w]), static_cast<T>(z[b][8 * u + 2 * w + 1])});
#pragma unroll
        for (int b = 0; b < kBlocks; b++)
#pragma unroll
            for (int u = 0; u < 2; u++)
#pragma unroll
                for (int d = 0; d < kWide; d++) {
                    const char* v = value_at + (32 * b + 16 * u) * kValueRow + d * 64;
                    const u32x2 low = read_transposed(v), high = read_transposed(v + 8 * kValueRow);
                    o[d] = mfma32<TYPE>(u32x4{low.x, low.y, high.x, high.y}, prob[b][u], o[d]);
                }
        ahead_of_products<kBlocks * 2 * kWide, 2, 4>();
    }

    const bool only = it.joins == 0;
    constexpr int kPad = DH + 4, kBlock = kTileRows * kPad;
    float* const part = p.parts + (static_cast<size_t>(only ? 0 : it.part) * p.cache.kv_heads + head) * kBlock;
    if (__builtin_amdgcn_readfirstlane(odd)) {
        rows_one_by_one<TYPE, DH>(p, it, table, head, 32 * wave, rows_here, part);
    } else {
        leave_rows<TYPE, DH, FULL>(p, it, o, m, both_sum(l), row, token, head * p.group + h, 32 * wave + (lane & 31), half, part);
    }
    if (only) return;
    finish_parts<TYPE, DH, FULL, kTileRows, 64 * kTileWaves>(p, it, mine, head, meeting, keys);
}

// ---------------------------------------------------------------------- fp32
//
// The fp32 matrix instructions have a sixteenth of the 16-bit ones' rate, so fp32 operands, probabilities among them, are taken as
// sums of three bf16 parts, x = high + middle + low, each the rest rounded to bf16: the last one is exact.  The parts of an element are
// its own: nothing is lost whatever its neighbours are, and nothing overflows (below 2^-103 low parts are subnormal: at
// most 2^-125 times the other factor is lost).  Six of the nine products of parts are formed; the three left out are below
// 2^-26 of the whole.  The matrix core cuts sums off where fp32 rounds, so the small products are summed before
// the large ones, whose cut-off bits they would share, a tile of positions from zero, and added to the running output in fp32.
// Infinities and NaN have no parts: their items go row by row.  16 x 1024 rows of 12 heads of 64: 187 us, 138 TFLOP/s where plain fp32
// products reach 153.  (Pairs of fp16 parts, three products, take 150, but need a power of two that neighbours share: an element
// 2^24 below the largest of its row or tile has lost digits, one 2^40 below it all of them.)

struct Parts {
    u32x2 high, middle, low;  // of four values, bf16
};

// `taint` becomes NaN if any value is infinite, NaN or rounded up to infinity: its rest is.
__device__ __forceinline__ Parts three_parts(const f32x4& x, float& taint) {
    Parts p;
#pragma unroll
    for (int w = 0; w < 2; w++) {
        float a = x[2 * w], b = x[2 * w + 1];
        const auto part = [&] {  // of both, which keep their rests
            const unsigned two = __builtin_bit_cast(unsigned, CacheType<kCacheBf16>::V2{static_cast<__bf16>(a), static_cast<__bf16>(b)});
            a -= __uint_as_float(two << 16);
            b -= __uint_as_float(two & 0xFFFF0000u);
            return two;
        };
        p.high[w] = part();
        p.middle[w] = part();
        taint = fmaf(a, 0.0f, fmaf(b, 0.0f, taint));
        p.low[w] = __builtin_bit_cast(unsigned, CacheType<kCacheBf16>::V2{static_cast<__bf16>(a), static_cast<__bf16>(b)});
    }
    return p;
}

template <int DH, bool FULL, int TOKENS>
__global__ __launch_bounds__(64 * kTileWaves, DH > 128 ? 1 : 2) void attend_wide_kernel(const AttendParams p) {
    constexpr int kKeyRow = DH * 2 + 16, kValueRow = DH * 2 + 32;  // bytes of a part's row
    constexpr int kKeys = TOKENS * kKeyRow, kValues = TOKENS * kValueRow;
    constexpr int kUnits = DH / 4;                               // of four values in a row
    constexpr int kLoads = TOKENS * kUnits / (64 * kTileWaves);  // of a thread, for K and for V
    constexpr int kBlocks = TOKENS / 32, kSteps = DH / 16, kWide = DH / 32;
    __shared__ __align__(16) char keys[3 * kKeys];
    __shared__ __align__(16) char values[3 * kValues];
    __shared__ Meeting meeting;
    __shared__ unsigned odd;

    const AttendItem it = p.items[blockIdx.x / p.cache.kv_heads];
    const int head = blockIdx.x % p.cache.kv_heads;
    const AttendJoin mine = first_join(p, it);
    const int* table = p.table + it.table;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int half = lane >> 5;

    const int r = it.r0 + 32 * wave + (lane & 31);
    const bool row = 32 * wave + (lane & 31) < it.rows;
    const int token = row ? r / p.group : 0, h = row ? r % p.group : 0;
    const int pos = row ? it.first + token : -1;
    const float* const query = reinterpret_cast<const float*>(p.q.at) + (it.row0 + token) * p.q.row + (head * p.group + h) * p.q.head;
    u32x4 q[3][kSteps];
    float taint = 0.0f;
#pragma unroll
    for (int c = 0; c < kSteps; c++) {
        const int dim = 16 * c + 8 * half;
#pragma unroll
        for (int side = 0; side < 2; side++) {
            f32x4 x{0, 0, 0, 0};
            if (row && (FULL || dim < p.cache.dim)) {
                if (p.vector_rows) {
                    x = *reinterpret_cast<const f32x4*>(query + dim + 4 * side);
                } else {
#pragma unroll
                    for (int e = 0; e < 4; e++) x[e] = query[dim + 4 * side + e];
                }
            }
            const Parts parts = three_parts(x, taint);
#pragma unroll
            for (int w = 0; w < 2; w++) {
                q[0][c][2 * side + w] = parts.high[w];
                q[1][c][2 * side + w] = parts.middle[w];
                q[2][c][2 * side + w] = parts.low[w];
            }
        }
    }
    const int rows_here = min(32, it.rows - 32 * wave);
    const int first = it.first + (it.r0 + 32 * wave) / p.group;
    const int final = it.first + (it.r0 + 32 * wave + max(rows_here, 1) - 1) / p.group;

    f32x16 o[kWide];
#pragma unroll
    for (int d = 0; d < kWide; d++)
#pragma unroll
        for (int i = 0; i < 16; i++) o[d][i] = 0.0f;
    float m = -INFINITY, l = 0.0f;

    f32x4 kr[kLoads], vr[kLoads];
    int pages[kLoads];
    const int bytes = p.cache.dim * 4, own_row = lane / kUnits;
    static_assert(64 % kUnits == 0, "whole rows");
    const int own = FULL || lane % kUnits * 4 < p.cache.dim ? own_row * bytes + lane % kUnits * 16 : kBeyond;
    const auto row_of = [&](int i) { return 64 * (kTileWaves * i + wave) / kUnits; };
    const auto look = [&](int at) {
#pragma unroll
        for (int i = 0; i < kLoads; i++) pages[i] = table[min(at + row_of(i), it.k1 - 1) >> p.cache.page_shift];
    };
    const auto fetch = [&](int at) {
#pragma unroll
        for (int i = 0; i < kLoads; i++) {
            const char* run = cache_run(p.cache, pages[i], p.layer, 0, head);
            const __amdgpu_buffer_rsrc_t ks = make_buffer(run, static_cast<unsigned>(p.cache.run_bytes));
            const __amdgpu_buffer_rsrc_t vs = make_buffer(run + p.cache.kv_heads * p.cache.run_bytes, static_cast<unsigned>(p.cache.run_bytes));
            const int t = at + row_of(i);
            const int offset = t + own_row < it.k1 ? own : kBeyond;  // (places behind the last position: zeros)
            const int base = (t & ((1 << p.cache.page_shift) - 1)) * bytes;
            kr[i] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(ks, offset, base, 0));
            vr[i] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(vs, offset, base, 0));
        }
    };
    const char* const key_at = keys + (lane & 31) * kKeyRow + half * 16;
    const char* const value_at = values + (4 * half + ((lane & 15) >> 2)) * kValueRow + 32 * ((lane >> 4) & 1) + 8 * (lane & 3);

    if (threadIdx.x == 0) odd = 0;
    look(it.k0);
    fetch(it.k0);
    look(it.k0 + TOKENS);
    for (int at = it.k0; at < it.k1; at += TOKENS) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kLoads; i++) {
            const Parts k = three_parts(kr[i], taint), v = three_parts(vr[i], taint);
            const int unit = 64 * (kTileWaves * i + wave) + lane;
            char* const to_k = keys + unit / kUnits * kKeyRow + unit % kUnits * 8;
            char* const to_v = values + unit / kUnits * kValueRow + unit % kUnits * 8;
            *reinterpret_cast<u32x2*>(to_k) = k.high;
            *reinterpret_cast<u32x2*>(to_k + kKeys) = k.middle;
            *reinterpret_cast<u32x2*>(to_k + 2 * kKeys) = k.low;
            *reinterpret_cast<u32x2*>(to_v) = v.high;
            *reinterpret_cast<u32x2*>(to_v + kValues) = v.middle;
            *reinterpret_cast<u32x2*>(to_v + 2 * kValues) = v.low;
        }
        if (taint != 0.0f) odd = 1;
        __syncthreads();
        if (__builtin_amdgcn_readfirstlane(odd)) break;  // (written again behind the next meeting only)
        if (at + TOKENS < it.k1) {
            fetch(at + TOKENS);
            look(at + 2 * TOKENS);
        }
        if (rows_here <= 0 || (p.causal && at > final) || (p.window > 0 && at + TOKENS - 1 <= first - p.window)) continue;

        f32x16 z[kBlocks];
#pragma unroll
        for (int b = 0; b < kBlocks; b++) {
            f32x16 acc;
#pragma unroll
            for (int i = 0; i < 16; i++) acc[i] = 0.0f;
            if constexpr (kSteps <= 4) {  // registers hold the parts of all dims: small products first, then the large ones
                u32x4 k[3][kSteps];
#pragma unroll
                for (int c = 0; c < kSteps; c++)
#pragma unroll
                    for (int part = 0; part < 3; part++)
                        k[part][c] = *reinterpret_cast<const u32x4*>(key_at + part * kKeys + b * 32 * kKeyRow + c * 32);
#pragma unroll
                for (int c = 0; c < kSteps; c++) {
                    acc = mfma32<kCacheBf16>(k[2][c], q[0][c], acc);
                    acc = mfma32<kCacheBf16>(k[1][c], q[1][c], acc);
                    acc = mfma32<kCacheBf16>(k[0][c], q[2][c], acc);
                }
#pragma unroll
                for (int c = 0; c < kSteps; c++) {
                    acc = mfma32<kCacheBf16>(k[1][c], q[0][c], acc);
                    acc = mfma32<kCacheBf16>(k[0][c], q[1][c], acc);
                }
#pragma unroll
                for (int c = 0; c < kSteps; c++) acc = mfma32<kCacheBf16>(k[0][c], q[0][c], acc);
            } else {  // ... or the two have sums of their own
                f32x16 small;
#pragma unroll
                for (int i = 0; i < 16; i++) small[i] = 0.0f;
#pragma unroll
                for (int c = 0; c < kSteps; c++) {
                    const char* k = key_at + b * 32 * kKeyRow + c * 32;
                    const u32x4 k0 = *reinterpret_cast<const u32x4*>(k), k1 = *reinterpret_cast<const u32x4*>(k + kKeys),
                                k2 = *reinterpret_cast<const u32x4*>(k + 2 * kKeys);
                    small = mfma32<kCacheBf16>(k2, q[0][c], small);
                    small = mfma32<kCacheBf16>(k1, q[1][c], small);
                    small = mfma32<kCacheBf16>(k0, q[2][c], small);
                    small = mfma32<kCacheBf16>(k1, q[0][c], small);
                    small = mfma32<kCacheBf16>(k0, q[1][c], small);
                    acc = mfma32<kCacheBf16>(k0, q[0][c], acc);
                }
#pragma unroll
                for (int i = 0; i < 16; i++) acc[i] += small[i];
            }
            z[b] = acc;
        }
        const bool cut = at + TOKENS > it.k1 || (p.causal && at + TOKENS - 1 > first) || (p.window > 0 && at <= final - p.window);
        if (cut) {
#pragma unroll
            for (int b = 0; b < kBlocks; b++)
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    const int t = at + 32 * b + 8 * (i / 4) + 4 * half + (i & 3);
                    const bool see = t < it.k1 && (!p.causal || t <= pos) && (p.window <= 0 || t > pos - p.window);
                    z[b][i] = see ? z[b][i] : -INFINITY;
                }
        }
        float scale = p.scale;
        float top = z[0][0];
#pragma unroll
        for (int b = 0; b < kBlocks; b++)
#pragma unroll
            for (int i = 0; i < 16; i++) top = fmaxf(top, z[b][i]);
        top = __fmul_rn(both_max(top), scale);
        if (__any(top > m)) {
            const float keep = top > m ? __builtin_amdgcn_exp2f(m - top) : 1.0f;
            m = fmaxf(m, top);
            l *= keep;
#pragma unroll
            for (int d = 0; d < kWide; d++)
#pragma unroll
                for (int i = 0; i < 16; i++) o[d][i] *= keep;
        }
        const float base = m == -INFINITY ? 0.0f : m;
        if (__any(fabsf(base) > kFusedTop)) {
#pragma unroll
            for (int b = 0; b < kBlocks; b++)
#pragma unroll
                for (int i = 0; i < 16; i++) z[b][i] = __fmul_rn(z[b][i], scale);
            scale = 1.0f;
        }
        u32x4 prob[3][kBlocks][2];
#pragma unroll
        for (int b = 0; b < kBlocks; b++)
#pragma unroll
            for (int g = 0; g < 4; g++) {
                f32x4 e;
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    e[i] = __builtin_amdgcn_exp2f(fmaf(z[b][4 * g + i], scale, -base));
                    l += e[i];
                }
                float none = 0.0f;
                const Parts parts = three_parts(e, none);
#pragma unroll
                for (int w = 0; w < 2; w++) {
                    prob[0][b][g / 2][2 * (g & 1) + w] = parts.high[w];
                    prob[1][b][g / 2][2 * (g & 1) + w] = parts.middle[w];
                    prob[2][b][g / 2][2 * (g & 1) + w] = parts.low[w];
                }
            }
#pragma unroll
        for (int d = 0; d < kWide; d++) {
            u32x4 v[3][kBlocks][2];
#pragma unroll
            for (int b = 0; b < kBlocks; b++)
#pragma unroll
                for (int u = 0; u < 2; u++)
#pragma unroll
                    for (int part = 0; part < 3; part++) {
                        const char* from = value_at + part * kValues + (32 * b + 16 * u) * kValueRow + d * 64;
                        const u32x2 low = read_transposed(from), high = read_transposed(from + 8 * kValueRow);
                        v[part][b][u] = u32x4{low.x, low.y, high.x, high.y};
                    }
            f32x16 acc;
#pragma unroll
            for (int i = 0; i < 16; i++) acc[i] = 0.0f;
#pragma unroll
            for (int b = 0; b < kBlocks; b++)
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    acc = mfma32<kCacheBf16>(v[2][b][u], prob[0][b][u], acc);
                    acc = mfma32<kCacheBf16>(v[1][b][u], prob[1][b][u], acc);
                    acc = mfma32<kCacheBf16>(v[0][b][u], prob[2][b][u], acc);
                }
#pragma unroll
            for (int b = 0; b < kBlocks; b++)
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    acc = mfma32<kCacheBf16>(v[1][b][u], prob[0][b][u], acc);
                    acc = mfma32<kCacheBf16>(v[0][b][u], prob[1][b][u], acc);
                }
#pragma unroll
            for (int b = 0; b < kBlocks; b++)
#pragma unroll
                for (int u = 0; u < 2; u++) acc = mfma32<kCacheBf16>(v[0][b][u], prob[0][b][u], acc);
#pragma unroll
            for (int i = 0; i < 16; i++) o[d][i] += acc[i];
        }
    }

    const bool only = it.joins == 0;
    constexpr int kPad = DH + 4, kBlock = kTileRows * kPad;
    float* const part = p.parts + (static_cast<size_t>(only ? 0 : it.part) * p.cache.kv_heads + head) * kBlock;
    if (__builtin_amdgcn_readfirstlane(odd)) {
        rows_one_by_one<kCacheF32, DH>(p, it, table, head, 32 * wave, rows_here, part);
    } else {
        leave_rows<kCacheF32, DH, FULL>(p, it, o, m, both_sum(l), row, token, head * p.group + h, 32 * wave + (lane & 31), half, part);
    }
    if (only) return;
    finish_parts<kCacheF32, DH, FULL, kTileRows, 64 * kTileWaves>(p, it, mine, head, meeting, keys);
}

}  // namespace gh
