// Attention of many rows over a paged cache: tiles of 128 rows, 32 to a wavefront, whose positions pass through shared memory
// once for all four.  The mathematics, the transposed products and the order of the k slots are those of
// kernels_cache_attn.h, on 32 x 32 x 16 products: a lane holds scores of row (lane & 31), of the positions
// 8 b + 4 (lane / 32) + j of every 32.
//
// Shared memory holds K and V as they are in the pages, position by position, with a stride that spreads what a product's
// lanes read over all banks: K rows are read 16 bytes to a lane (eight lanes to a cycle: rows 16 bytes apart modulo 128), V through
// the transposing read, which hands a lane four positions of one dim (16 lanes to a cycle: four rows 32 bytes apart modulo 128).
#pragma once

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
    __shared__ unsigned last, odd;

    const AttendItem it = p.items[blockIdx.x / p.cache.kv_heads];
    const int head = blockIdx.x % p.cache.kv_heads;
    const PassSeq s = p.seqs[it.seq];
    const int* table = p.table + s.table;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int half = lane >> 5;

    // this lane's row and its query
    const int r = it.r0 + 32 * wave + (lane & 31);
    const bool row = 32 * wave + (lane & 31) < it.rows;
    const int token = row ? r / p.group : 0, h = row ? r % p.group : 0;
    const int pos = row ? s.first + token : -1;
    u32x4 q[kSteps];
    {
        const T* from = reinterpret_cast<const T*>(p.q.at) + (s.row0 + token) * p.q.row + (head * p.group + h) * p.q.head;
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
    const int first_all = s.first + it.r0 / p.group, final_all = s.first + (it.r0 + it.rows - 1) / p.group;
    const int first = s.first + (it.r0 + 32 * wave) / p.group;
    const int final = s.first + (it.r0 + 32 * wave + max(rows_here, 1) - 1) / p.group;

    f32x16 o[kWide];
#pragma unroll
    for (int d = 0; d < kWide; d++)
#pragma unroll
        for (int i = 0; i < 16; i++) o[d][i] = 0.0f;
    float m = -INFINITY, l = 0.0f;

    // a thread's units of 16 bytes: rows of one block of 16 positions for a wavefront, so one page
    u32x4 kr[kLoads], vr[kLoads];
    const int bytes = p.cache.dim * 2;
    const auto fetch = [&](int at) {
#pragma unroll
        for (int i = 0; i < kLoads; i++) {
            constexpr int kRows = 64 / kUnits > 0 ? 64 / kUnits : 1;  // of a wavefront's load (DH 512 and more: none)
            const int unit = 64 * (kTileWaves * i + wave);
            const int row0 = unit / kUnits;  // first row of the load
            const int t0 = at + row0 < it.k1 ? at + row0 : at;
            const int page = table[t0 >> p.cache.page_shift];
            const char* run = cache_run(p.cache, page, p.layer, 0, head);
            const __amdgpu_buffer_rsrc_t ks = make_buffer(run, static_cast<unsigned>(p.cache.run_bytes));
            const __amdgpu_buffer_rsrc_t vs = make_buffer(run + p.cache.kv_heads * p.cache.run_bytes, static_cast<unsigned>(p.cache.run_bytes));
            const int mine = lane / kUnits, dim = lane % kUnits * 8;
            static_assert(kRows * kUnits == 64, "whole rows");
            const bool there = (FULL || dim < p.cache.dim) && at + row0 + mine < it.k1;
            const int offset = there ? mine * bytes + dim * 2 : kBeyond;  // (places behind the last position: zeros)
            const int base = (t0 & ((1 << p.cache.page_shift) - 1)) * bytes;
            kr[i] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(ks, offset, base, 0));
            vr[i] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(vs, offset, base, 0));
        }
    };
    // how a lane reads them back
    const char* const key_at = keys + (lane & 31) * kKeyRow + half * 16;
    const char* const value_at = values + (4 * half + ((lane & 15) >> 2)) * kValueRow + 32 * ((lane >> 4) & 1) + 8 * (lane & 3);

    if (threadIdx.x == 0) odd = 0;
    fetch(it.k0);
    for (int at = it.k0; at < it.k1; at += TOKENS) {
        const bool cut_all = (p.causal && at + TOKENS - 1 > first_all) || (p.window > 0 && at <= final_all - p.window);
        __syncthreads();
        bool bad = false;
#pragma unroll
        for (int i = 0; i < kLoads; i++) {
            const int unit = 64 * (kTileWaves * i + wave) + lane;
            const int to = unit / kUnits, c = unit % kUnits * 16;
            *reinterpret_cast<u32x4*>(keys + to * kKeyRow + c) = kr[i];
            *reinterpret_cast<u32x4*>(values + to * kValueRow + c) = vr[i];
            if (cut_all)
#pragma unroll
                for (int w = 0; w < 4; w++) bad = bad || unbounded<TYPE>(vr[i][w]);
        }
        // infinities and NaN among values that some rows may not see: the positions from `at` on are marked
        if (bad) odd = static_cast<unsigned>(at) + 1;
        __syncthreads();
        if (at + TOKENS < it.k1) fetch(at + TOKENS);
        if (rows_here <= 0 || (p.causal && at > final) || (p.window > 0 && at + TOKENS - 1 <= first - p.window)) continue;

        float z[kBlocks][16];
#pragma unroll
        for (int b = 0; b < kBlocks; b++) {
            f32x16 acc;
#pragma unroll
            for (int i = 0; i < 16; i++) acc[i] = 0.0f;
#pragma unroll
            for (int c = 0; c < kSteps; c++)
                acc = mfma32<TYPE>(*reinterpret_cast<const u32x4*>(key_at + b * 32 * kKeyRow + c * 32), q[c], acc);
#pragma unroll
            for (int i = 0; i < 16; i++) z[b][i] = acc[i];
        }
        const bool cut = at + TOKENS > it.k1 || (p.causal && at + TOKENS - 1 > first) || (p.window > 0 && at <= final - p.window);
        unsigned seen[kBlocks];
        if (cut) {
#pragma unroll
            for (int b = 0; b < kBlocks; b++) {
                seen[b] = 0;
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    const int t = at + 32 * b + 8 * (i / 4) + 4 * half + (i & 3);
                    const bool see = t < it.k1 && (!p.causal || t <= pos) && (p.window <= 0 || t > pos - p.window);
                    z[b][i] = see ? z[b][i] : -INFINITY;
                    seen[b] |= see ? 1u << i : 0u;
                }
            }
        }
        float top = z[0][0];
#pragma unroll
        for (int b = 0; b < kBlocks; b++)
#pragma unroll
            for (int i = 0; i < 16; i++) top = fmaxf(top, z[b][i]);
        top = both_max(top) * p.scale;
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
#pragma unroll
        for (int b = 0; b < kBlocks; b++)
#pragma unroll
            for (int i = 0; i < 16; i++) {
                z[b][i] = __builtin_amdgcn_exp2f(z[b][i] * p.scale - base);
                l += z[b][i];
            }
        const bool careful = cut && __builtin_amdgcn_readfirstlane(odd) == static_cast<unsigned>(at) + 1;
#pragma unroll
        for (int b = 0; b < kBlocks; b++)
#pragma unroll
            for (int u = 0; u < 2; u++) {
                u32x4 prob;
#pragma unroll
                for (int w = 0; w < 4; w++)
                    prob[w] = __builtin_bit_cast(
                        unsigned, typename C::V2{static_cast<T>(z[b][8 * u + 2 * w]), static_cast<T>(z[b][8 * u + 2 * w + 1])});
#pragma unroll
                for (int d = 0; d < kWide; d++) {
                    const char* v = value_at + (32 * b + 16 * u) * kValueRow + d * 64;
                    const u32x2 low = read_transposed(v), high = read_transposed(v + 8 * kValueRow);
                    u32x4 a{low.x, low.y, high.x, high.y};
                    if (careful) {
                        u32x4 kind, see;
#pragma unroll
                        for (int w = 0; w < 4; w++) {
                            kind[w] = unbounded_kind<TYPE>(a[w]);
                            a[w] = bounded<TYPE>(a[w]);
                            const unsigned bits = seen[b] >> (8 * u + 2 * w);
                            see[w] = (bits & 1u) * C::kOne | ((bits >> 1) & 1u) * (C::kOne << 16);
                        }
                        f32x16 n;
#pragma unroll
                        for (int i = 0; i < 16; i++) n[i] = 0.0f;
                        n = mfma32<TYPE>(kind, see, n);
#pragma unroll
                        for (int i = 0; i < 16; i++) o[d][i] += unbounded_sum(n[i]);
                    }
                    o[d] = mfma32<TYPE>(a, prob, o[d]);
                }
            }
    }

    const bool only = it.parts == 1;
    constexpr int kPad = DH + 4, kBlock = kTileRows * kPad;
    float* const parts = p.parts + (static_cast<size_t>(only ? 0 : it.part) * p.cache.kv_heads + head) * kBlock;
    const size_t part_stride = static_cast<size_t>(p.cache.kv_heads) * kBlock;
    l = both_sum(l);
    if (row) {
        const __amdgpu_buffer_rsrc_t rs = make_buffer(parts + (only ? 0 : it.index) * part_stride, kBlock * 4);
        const int base = (32 * wave + (lane & 31)) * kPad * 4;
        const long long to = (s.row0 + token) * p.out.row + (head * p.group + h) * p.out.head;
#pragma unroll
        for (int d = 0; d < kWide; d++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int dim = 32 * d + 8 * i + 4 * half;
                const f32x4 four{o[d][4 * i], o[d][4 * i + 1], o[d][4 * i + 2], o[d][4 * i + 3]};
                if (only) {
                    if (FULL || dim < p.cache.dim) store_four<TYPE>(p.out, to + dim, p.vector_rows, four / l);
                } else {
                    __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(v4i, four), rs, base + dim * 4, 0, kAuxDeviceScope);
                }
            }
        if (!only && half == 0)
            __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(v4i, f32x4{m, l, 0.0f, 0.0f}), rs, base + DH * 4, 0, kAuxDeviceScope);
    }
    if (only) return;
    finish_parts<TYPE, DH, FULL, kTileRows, 64 * kTileWaves>(p, it, s, head, parts, part_stride, last);
}

}  // namespace gh
