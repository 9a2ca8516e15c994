// Which attention kernel takes a pass; one translation unit per element type makes them.
#pragma once

#include "kernels_cache_tile.h"

namespace gh {

using AttendKernel = void (*)(AttendParams);

struct AttendForm {
    AttendKernel kernel = nullptr;
    int height = 0;       // rows of a tile
    int threads = 0;
    int part_floats = 0;  // of a tile's part in memory
};

// The kernel for sequences of so many rows (tokens times query heads of a kv head) at heads of `dim` dims.
AttendForm attend_form_f32(int dim, int rows);
AttendForm attend_form_bf16(int dim, int rows);
AttendForm attend_form_f16(int dim, int rows);

template <int TYPE, int DH, bool FULL>
AttendForm attend_form_at(int rows) {
    const auto form = [](AttendKernel kernel, int height, int waves) { return AttendForm{kernel, height, 64 * waves, height * (DH + 4)}; };
    if (rows > 64) {
        if constexpr (TYPE == kCacheF32) {
            return form(attend_wide_kernel<DH, FULL, DH == 64 ? 64 : 32>, kTileRows, kTileWaves);
        } else {
            return form(attend_tile_kernel<TYPE, DH, FULL, DH == 256 ? 32 : 64>, kTileRows, kTileWaves);
        }
    }
    if constexpr (DH < 256)
        if (rows > 16) return form(attend_rows_kernel<TYPE, DH, FULL, 2>, 32, attend_waves(TYPE, DH, 2));
    return form(attend_rows_kernel<TYPE, DH, FULL, 1>, 16, attend_waves(TYPE, DH, 1));
}

template <int TYPE>
AttendForm attend_form_of(int dim, int rows) {
    if (dim > 128) return attend_form_at<TYPE, 256, false>(rows);
    if (dim == 128) return attend_form_at<TYPE, 128, true>(rows);
    if (dim > 64) return attend_form_at<TYPE, 128, false>(rows);
    if (dim == 64) return attend_form_at<TYPE, 64, true>(rows);
    return attend_form_at<TYPE, 64, false>(rows);
}

}  // namespace gh
