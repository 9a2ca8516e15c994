// Picks from rows of logits with settings of each row's own (gh_sample).
#include "device_scope.h"
#include "kernels_sample.h"

namespace gh {

[[noreturn]] static void refuse(const std::string& why) { throw ApiError{GH_ERR_INVALID_ARGUMENT, "gh_sample: " + why}; }

static void check_sizes(int type, int rows, int vocab) {
    if (type != GH_F32 && type != GH_BF16 && type != GH_F16) refuse("unknown element type");
    if (rows < 0 || rows > (1 << 24)) refuse("rows must be 0 to 2^24");
    if (vocab < 1 || vocab > kMaxSampleVocab) refuse("vocab must be 1 to 2^20");
}

static size_t sample_workspace(int type, int rows, int vocab) {
    check_sizes(type, rows, vocab);
    return 0;
}

static void sample(const gh_sample_args& a, hipStream_t stream) {
    const size_t need = sample_workspace(a.type, a.rows, a.vocab);
    if (a.row_stride < 0) refuse("negative row_stride");
    if (a.rows == 0) return;
    if (!a.logits || !a.uniforms || !a.ids) throw ApiError{GH_ERR_INVALID_ARGUMENT, "null argument"};
    if (need > 0 && (!a.workspace || a.workspace_bytes < need)) refuse("a workspace of " + std::to_string(need) + " bytes is needed");
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
    const auto kernel = a.type == GH_F32 ? sample_row_kernel<kCacheF32> : a.type == GH_BF16 ? sample_row_kernel<kCacheBf16> : sample_row_kernel<kCacheF16>;
    hipLaunchKernelGGL(kernel, dim3(a.rows), dim3(kSampleThreads), 0, stream, p);
    HIP_CHECK(hipGetLastError());
}

}  // namespace gh

using namespace gh;

extern "C" {

gh_status gh_sample_workspace(int32_t type, int32_t rows, int32_t vocab, size_t* bytes) {
    return guard([&] {
        if (!bytes) throw ApiError{GH_ERR_INVALID_ARGUMENT, "null argument"};
        *bytes = sample_workspace(type, rows, vocab);
    });
}

gh_status gh_sample(const gh_sample_args* args, void* hip_stream) {
    return guard([&] {
        if (!args) throw ApiError{GH_ERR_INVALID_ARGUMENT, "null argument"};
        sample(*args, static_cast<hipStream_t>(hip_stream));
    });
}

}  // extern "C"
