// The paged cache's kernels that move data: plans to the device, new rows into the pages (rotated to their positions), pages
// to pages, and positions back out.  All are bound by memory; none keeps anything in shared memory but the angles of a row.
#pragma once

#include "kernels_cache_attn.h"
#include "page_book.h"

namespace gh {

// Words of 16 bytes out of pinned host memory.
__global__ __launch_bounds__(256) void cache_load_kernel(const u32x4* __restrict__ host, u32x4* __restrict__ to, size_t n) {
    for (size_t i = blockIdx.x * 256ull + threadIdx.x; i < n; i += gridDim.x * 256ull) to[i] = host[i];
}

// ... or a few that come with the launch.
constexpr size_t kWordsListed = 224;
struct WordList {
    u32x4 words[kWordsListed];
};
__global__ __launch_bounds__(256) void cache_hand_kernel(const WordList list, u32x4* __restrict__ to, int n) {
    if (static_cast<int>(threadIdx.x) < n) to[threadIdx.x] = list.words[threadIdx.x];
}

struct AppendParams {
    CacheLayout cache;
    CacheRows k, v, q, q_out;  // q.at null: no queries
    const RowAt* rows;
    const double* speed;  // turns per position of every pair of dims; null: keys and queries go as they are
    int layer;
    int heads;  // of q
    int vector_rows;
};

template <int TYPE>
struct Eight {
    using T = typename CacheType<TYPE>::T;
    T e[8];
    __device__ __forceinline__ void load(const char* at, bool vector) {
        if (vector) {
            *reinterpret_cast<u32x4*>(e) = *reinterpret_cast<const u32x4*>(at);
            if constexpr (sizeof(T) == 4) *reinterpret_cast<u32x4*>(e + 4) = *reinterpret_cast<const u32x4*>(at + 16);
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++) e[i] = reinterpret_cast<const T*>(at)[i];
        }
    }
    __device__ __forceinline__ void store(char* at, bool vector) const {
        if (vector) {
            *reinterpret_cast<u32x4*>(at) = *reinterpret_cast<const u32x4*>(e);
            if constexpr (sizeof(T) == 4) *reinterpret_cast<u32x4*>(at + 16) = *reinterpret_cast<const u32x4*>(e + 4);
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++) reinterpret_cast<T*>(at)[i] = e[i];
        }
    }
    // Pairs (2j, 2j + 1) by the angles of their row, in 64 bits, rounded to 32 and then to the type: a caller that rotates in
    // 32 bits or converts from there finds the same value (one rounding instead of two would differ near ties).
    __device__ __forceinline__ void turn(const double2* angle) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const double a = e[2 * i], b = e[2 * i + 1];
            const double2 t = angle[i];  // cosine and sine
            float x = static_cast<float>(a * t.x - b * t.y), y = static_cast<float>(a * t.y + b * t.x);
            asm volatile("" : "+v"(x), "+v"(y));  // (the compiler would make one conversion of the two)
            e[2 * i] = static_cast<T>(x);
            e[2 * i + 1] = static_cast<T>(y);
        }
    }
};

// One workgroup per row: its keys, values and queries, eight dims to a thread, requested before anything is computed.  Angles
// and rotations are 64-bit (a position of a million keeps all its digits, and a result is rounded as the exact one is but
// for ties): the sines of a row are formed once for all its heads (13 rows
// of 12 heads of 64: 4.6 us, 5.0 with 32-bit sines and a correction).
template <int TYPE>
__global__ __launch_bounds__(256) void cache_append_kernel(const AppendParams p) {
    constexpr int kBytes = CacheType<TYPE>::kBytes;
    __shared__ double2 angle[128];
    const long long row = blockIdx.x;
    const int eights = p.cache.dim / 8, cached = p.cache.kv_heads * eights;
    const int all = 2 * cached + (p.q.at ? p.heads * eights : 0);
    const auto place_of = [&](int i, int& which, int& head, int& dim) {
        which = i < cached ? 0 : i < 2 * cached ? 1 : 2;
        const int j = i - which * cached;
        head = j / eights;
        dim = j % eights * 8;
    };
    const auto load = [&](int i, Eight<TYPE>& x) {
        int which, head, dim;
        place_of(i, which, head, dim);
        const CacheRows& from = which == 0 ? p.k : which == 1 ? p.v : p.q;
        x.load(from.at + (row * from.row + head * from.head + dim) * kBytes, p.vector_rows);
    };
    Eight<TYPE> first;
    if (static_cast<int>(threadIdx.x) < all) load(threadIdx.x, first);
    const RowAt at = p.rows[row];
    if (p.speed) {
        if (threadIdx.x < static_cast<unsigned>(p.cache.dim / 2)) {
            const double turns = at.pos * p.speed[threadIdx.x];
            double sine, cosine;
            sincospi(2.0 * (turns - rint(turns)), &sine, &cosine);
            angle[threadIdx.x] = double2{cosine, sine};
        }
        __syncthreads();
    }
    const int page = at.slot >> p.cache.page_shift, place = at.slot & ((1 << p.cache.page_shift) - 1);
    for (int i = threadIdx.x; i < all; i += 256) {
        Eight<TYPE> x;
        if (i == static_cast<int>(threadIdx.x)) {
            x = first;
        } else {
            load(i, x);
        }
        int which, head, dim;
        place_of(i, which, head, dim);
        if (p.speed && which != 1) x.turn(angle + dim / 2);
        if (which < 2) {
            x.store(cache_run(p.cache, page, p.layer, which, head) + (static_cast<size_t>(place) * p.cache.dim + dim) * kBytes, true);
        } else {
            x.store(p.q_out.at + (row * p.q_out.row + head * p.q_out.head + dim) * kBytes, p.vector_rows);
        }
    }
}

// Lists of up to so many entries travel with the launch itself.
constexpr int kListed = 256;
struct CopyList {
    PageCopy copies[kListed];
};
struct PageList {
    int pages[2 * kListed];
};

// The first positions of pages into other pages (of this pool or of one of the same shape), 4 KB of a run at a time: whole runs, one
// to a workgroup, are four trips to memory one behind the other (16 KB runs; six sequences of up to 1.5 k positions, 8 layers, 12 heads
// of 64 in fp32, copied, half dropped, made dense, the rest read, 1.3 GB in all: 265 us, with whole runs 273).
__global__ __launch_bounds__(256) void cache_copy_kernel(const char* __restrict__ from, char* __restrict__ to, size_t page_bytes, int runs,
                                                         int run_words, int token_bytes, const CopyList list) {
    const PageCopy copy = list.copies[blockIdx.y];
    const int words = copy.tokens * token_bytes / 16, pieces = (words + 255) / 256;
    const u32x4* a = reinterpret_cast<const u32x4*>(from + static_cast<size_t>(copy.from) * page_bytes);
    u32x4* b = reinterpret_cast<u32x4*>(to + static_cast<size_t>(copy.to) * page_bytes);
    for (long long i = blockIdx.x; i < static_cast<long long>(runs) * pieces; i += gridDim.x) {
        const int run = static_cast<int>(i / pieces), w = static_cast<int>(i % pieces) * 256 + static_cast<int>(threadIdx.x);
        if (w < words) b[static_cast<size_t>(run) * run_words + w] = a[static_cast<size_t>(run) * run_words + w];
    }
}

struct ReadParams {
    CacheLayout cache;
    CacheRows k, v;  // position start goes to row 0
    long long k_layer, v_layer;
    int layer, start, count;
    int vector_rows;
};

constexpr int kReadPositions = 16;

// 16 positions of a layer, K or V, to a workgroup.
template <int TYPE>
__global__ __launch_bounds__(256) void cache_read_kernel(const ReadParams p, const PageList list) {  // pages from start's on
    constexpr int kBytes = CacheType<TYPE>::kBytes;
    const int which = blockIdx.z, layer = blockIdx.y, n0 = blockIdx.x * kReadPositions;
    const int eights = p.cache.dim / 8, tokens = min(kReadPositions, p.count - n0);
    const CacheRows& to = which ? p.v : p.k;
    const long long base = layer * (which ? p.v_layer : p.k_layer);
    const int first_page = p.start >> p.cache.page_shift;
    for (int i = threadIdx.x; i < tokens * eights * p.cache.kv_heads; i += 256) {
        const int dim = i % eights * 8, token = i / eights % tokens, head = i / eights / tokens;
        const int t = p.start + n0 + token;
        const int page = list.pages[(t >> p.cache.page_shift) - first_page], place = t & ((1 << p.cache.page_shift) - 1);
        Eight<TYPE> x;
        x.load(cache_run(p.cache, page, p.layer + layer, which, head) + (static_cast<size_t>(place) * p.cache.dim + dim) * kBytes, true);
        x.store(to.at + (base + (n0 + token) * to.row + head * to.head + dim) * kBytes, p.vector_rows);
    }
}

struct SessionCopyParams {
    CacheLayout cache;
    KvLayout kv;
    int seq;           // of the session
    int start, count;  // positions; the list of pages begins with start's
    int to_session;
};

// 16 positions of a layer, K or V, between a session's pages and a cache's, both fp32, 16 bytes to a thread.
__global__ __launch_bounds__(256) void cache_session_kernel(const SessionCopyParams p, const PageList list) {
    const int which = blockIdx.z, layer = blockIdx.y, n0 = blockIdx.x * kReadPositions;
    const int fours = p.cache.dim / 4, tokens = min(kReadPositions, p.count - n0);
    const int first_page = p.start >> p.cache.page_shift;
    for (int i = threadIdx.x; i < tokens * fours * p.cache.kv_heads; i += 256) {
        const int dim = i % fours * 4, token = i / fours % tokens, head = i / fours / tokens;
        const int t = p.start + n0 + token;
        const int page = list.pages[(t >> p.cache.page_shift) - first_page], place = t & ((1 << p.cache.page_shift) - 1);
        float4* const cached = reinterpret_cast<float4*>(reinterpret_cast<float*>(cache_run(p.cache, page, layer, which, head))
                                                         + static_cast<size_t>(place) * p.cache.dim + dim);
        float4* const session = reinterpret_cast<float4*>(p.kv.pool + kv_offset(p.kv, layer, p.seq, which, head, t) + dim);
        if (p.to_session) {
            *session = *cached;
        } else {
            *cached = *session;
        }
    }
}

}  // namespace gh
