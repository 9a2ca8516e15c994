// Picks from rows of logits with settings of each row's own (gh_sample).
#include "device_scope.h"
#include "kernels_sample.h"

#include <array>
#include <cmath>

namespace gh {

[[noreturn]] static void refuse(const std::string& why) { throw ApiError{GH_ERR_INVALID_ARGUMENT, "gh_sample: " + why}; }

static void check_sizes(int type, int rows, int vocab) {
    if (type != GH_F32 && type != GH_BF16 && type != GH_F16) refuse("unknown element type");
    if (rows < 0 || rows > (1 << 24)) refuse("rows must be 0 to 2^24");
    if (vocab < 1 || vocab > kMaxSampleVocab) refuse("vocab must be 1 to 2^20");
}

// Rows of one chunk are picked from by the workgroup that reads them.  Longer ones are read in chunks by as many workgroups, wide chunks where
// they keep every compute unit busy.  Rows of more groups than a list holds are looked through by up to eight workgroups, as many as the GPU has room for.
// (Flat rows, fp32, top-p 0.98, 1 and 64 of them: 140000 tokens 51 and 83 us.  Below that border one workgroup does it from a list of groups: 32000 tokens 62 and
// 65, 64000 93 and 104, 128000 161 and 175.)
constexpr int kUnits = 256, kMostShared = 512;
struct SampleForm {
    int chunk = kChunk;
    int chunks = 1;
    int shares = 1;  // workgroups that look through a row
    size_t group_tops = 0, chunk_tops = 0, segment_sums = 0, masses = 0, counters = 0, lists = 0, bytes = 0;  // places in the workspace
};

static SampleForm form_of(int rows, int vocab) {
    SampleForm f;
    if (vocab <= kChunk) return f;
    const auto chunks = [&](int length) { return (vocab + length - 1) / length; };
    if (static_cast<long long>(rows) * chunks(kWideChunk) >= kUnits) f.chunk = kWideChunk;
    f.chunks = chunks(f.chunk);
    const auto place = [&](size_t per_row) {
        const size_t at = f.bytes;
        f.bytes += (per_row * static_cast<size_t>(rows) + 15) / 16 * 16;
        return at;
    };
    f.group_tops = place(sizeof(float) * groups_of(vocab));
    f.chunk_tops = place(sizeof(float) * f.chunks);
    f.segment_sums = place(sizeof(double) * segments_of(vocab));
    f.masses = place(sizeof(unsigned long long) * kMassBuckets * f.chunks);
    if (rows > 0 && groups_of(vocab) > kListed && rows < kMostShared) {
        f.shares = std::min(8, kMostShared / rows);
        f.counters = place(2 * sizeof(unsigned));
        f.lists = place(sizeof(unsigned long long) * kListed);
    }
    return f;
}

// Enough for so many rows and for fewer: between the borders of the rules more rows need more.
static size_t workspace_of(int rows, int vocab) {
    size_t bytes = 0;
    const int wide = (kUnits - 1) / ((vocab + kWideChunk - 1) / kWideChunk);  // rows: the most of smaller chunks
    for (int n : {rows, std::min(rows, wide), std::min(rows, kMostShared - 1)}) bytes = std::max(bytes, form_of(n, vocab).bytes);
    return bytes;
}

template <int TYPE>
static void launch_sample(SampleParams p, const SampleForm& f, int rows, hipStream_t stream) {
    // (a launch holds at most 2^32 threads)
    const int slice = (1 << 21) / f.chunks;
    for (p.first_row = 0; p.first_row < rows; p.first_row += slice) {
        const int n = std::min(slice, rows - p.first_row);
        if (p.vocab <= kChunk) {
            hipLaunchKernelGGL(sample_row_kernel<TYPE>, dim3(n), dim3(kSampleThreads), 0, stream, p);
        } else {
            if (f.chunk == kChunk) {
                hipLaunchKernelGGL((sample_scan_kernel<TYPE, kSampleThreads>), dim3(n * f.chunks), dim3(kSampleThreads), 0, stream, p);
            } else {
                hipLaunchKernelGGL((sample_scan_kernel<TYPE, kWideThreads>), dim3(n * f.chunks), dim3(kWideThreads), 0, stream, p);
            }
            HIP_CHECK(hipGetLastError());
            hipLaunchKernelGGL(sample_pick_kernel<TYPE>, dim3(n * f.shares), dim3(kSampleThreads), 0, stream, p, f.chunk);
        }
        HIP_CHECK(hipGetLastError());
    }
}

static void sample(const gh_sample_args& a, hipStream_t stream) {
    check_sizes(a.type, a.rows, a.vocab);
    const SampleForm f = form_of(a.rows, a.vocab);
    if (a.row_stride < 0) refuse("negative row_stride");
    if (a.rows == 0) return;
    if (!a.logits || !a.uniforms || !a.ids) throw ApiError{GH_ERR_INVALID_ARGUMENT, "null argument"};
    if (f.bytes > 0 && (!a.workspace || a.workspace_bytes < f.bytes)) refuse("a workspace of " + std::to_string(f.bytes) + " bytes is needed");
    if (f.bytes > 0 && reinterpret_cast<uintptr_t>(a.workspace) % 16 != 0) refuse("the workspace is not aligned to 16 bytes");
    require_gpu();
    hipPointerAttribute_t at{};
    if (hipPointerGetAttributes(&at, a.logits) != hipSuccess || (at.type != hipMemoryTypeDevice && at.type != hipMemoryTypeManaged)) {
        (void)hipGetLastError();
        refuse("logits are not device memory");
    }
    const DeviceScope on(at.device);
    SampleParams p{};
    p.logits = a.logits;
    p.row_stride = a.row_stride;
    p.vocab = a.vocab;
    int bits = 0;
    while ((1 << bits) < a.vocab) bits++;
    p.scale_bits = std::min(51, 62 - bits);
    p.temperature = a.temperature;
    p.top_k = a.top_k;
    p.top_p = a.top_p;
    p.min_p = a.min_p;
    p.uniforms = a.uniforms;
    p.ids = a.ids;
    p.probs = a.probs;
    static const std::array<double, kPowers> powers = [] {
        std::array<double, kPowers> t;
        for (int j = 0; j < kPowers; j++) t[static_cast<size_t>(j)] = std::exp2(static_cast<double>(j) / kPowers);
        return t;
    }();
    std::copy(powers.begin(), powers.end(), p.powers);
    char* const work = static_cast<char*>(a.workspace);
    p.chunks = f.chunks;
    p.group_tops = reinterpret_cast<float*>(work + f.group_tops);
    p.chunk_tops = reinterpret_cast<float*>(work + f.chunk_tops);
    p.segment_sums = reinterpret_cast<double*>(work + f.segment_sums);
    p.masses = reinterpret_cast<unsigned long long*>(work + f.masses);
    p.shares = f.shares;
    p.counters = reinterpret_cast<unsigned*>(work + f.counters);
    p.lists = reinterpret_cast<unsigned long long*>(work + f.lists);
    if (a.type == GH_F32) launch_sample<kCacheF32>(p, f, a.rows, stream);
    else if (a.type == GH_BF16) launch_sample<kCacheBf16>(p, f, a.rows, stream);
    else launch_sample<kCacheF16>(p, f, a.rows, stream);
}

}  // namespace gh

using namespace gh;

extern "C" {

gh_status gh_sample_workspace(int32_t type, int32_t rows, int32_t vocab, size_t* bytes) {
    return guard([&] {
        if (!bytes) throw ApiError{GH_ERR_INVALID_ARGUMENT, "null argument"};
        check_sizes(type, rows, vocab);
        *bytes = workspace_of(rows, vocab);
    });
}

gh_status gh_sample(const gh_sample_args* args, void* hip_stream) {
    return guard([&] {
        if (!args) throw ApiError{GH_ERR_INVALID_ARGUMENT, "null argument"};
        sample(*args, static_cast<hipStream_t>(hip_stream));
    });
}

}  // extern "C"
