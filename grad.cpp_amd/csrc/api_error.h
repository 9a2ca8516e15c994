// How the C entry points report failures: an exception inside the library, a status code and a
// message of the calling thread outside.  Nothing is thrown through an entry point.
#pragma once

#include "../../include/gradhip.h"

#include <hip/hip_runtime.h>

#include <new>
#include <stdexcept>
#include <string>

namespace gh {

struct ApiError {
    gh_status code;
    std::string msg;
};

inline thread_local std::string g_last_error;

[[noreturn]] inline void throw_device(hipError_t e, const char* what, const char* file, int line) {
    throw ApiError{GH_ERR_DEVICE, std::string("HIP error in ") + what + ": " + hipGetErrorString(e)
                                      + " (" + file + ":" + std::to_string(line) + ")"};
}

#define HIP_CHECK(expr)                                                        \
    do {                                                                       \
        hipError_t e_ = (expr);                                                \
        if (e_ != hipSuccess) gh::throw_device(e_, #expr, __FILE__, __LINE__); \
    } while (0)

template <typename F>
inline gh_status guard(F&& f) {
    try {
        f();
        return GH_OK;
    } catch (const ApiError& e) {
        g_last_error = e.msg;
        return e.code;
    } catch (const std::out_of_range& e) {
        g_last_error = e.what();
        return GH_ERR_OUT_OF_RANGE;
    } catch (const std::invalid_argument& e) {
        g_last_error = e.what();
        return GH_ERR_INVALID_ARGUMENT;
    } catch (const std::bad_alloc&) {
        g_last_error = "out of host memory";
        return GH_ERR_RUNTIME;
    } catch (const std::exception& e) {
        g_last_error = e.what();
        return GH_ERR_RUNTIME;
    }
}

inline void require_gpu() {
    int n = 0;
    hipError_t e = hipGetDeviceCount(&n);
    if (e != hipSuccess || n <= 0) {
        throw ApiError{GH_ERR_DEVICE,
                       "gradhip needs a gfx950 GPU: no HIP device is usable and there is no CPU "
                       "fallback"};
    }
}

}  // namespace gh
