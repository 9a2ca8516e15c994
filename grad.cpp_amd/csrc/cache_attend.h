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

// Rows of a sequence (tokens times query heads of a kv head) up to which tiles of 16 rows, whose wavefronts read the cache
// themselves, take it; more go to tiles of 128 rows that share what is read.  Tiles of 16 rows read the cache once each, which
// is nearly free for one sequence (its rows are in the L2s) and is not for many.  us, tiles of 16 and of 128: bf16, 32/8 heads of 128,
// 16 sequences of 4 k positions: 16 rows 77 and 93, 32 rows 108 and 95, 64 rows 166 and 83; one sequence: 32 rows 17 and 28, 64 rows
// 25 and 32.  fp32, 12 heads of 64, 16 sequences of 2 k positions: 32 rows 65 and 100, 64 rows 112 and 115, 128 rows 203 and 124; one
// sequence: 64 rows 17 and 29, 128 rows over 4 k positions 36 and 48, over 16 k 105 and 90.
constexpr int few_rows(int type) { return type == kCacheF32 ? 64 : 32; }
constexpr int kFewTile = 16;

// The kernel for sequences of so many rows (tokens times query heads of a kv head) at heads of `dim` dims.
AttendForm attend_form_f32(int dim, int rows);
AttendForm attend_form_bf16(int dim, int rows);
AttendForm attend_form_f16(int dim, int rows);
// ... whose rows see the first positions beside a window.
AttendForm attend_form_sinks_f32(int dim, int rows);
AttendForm attend_form_sinks_bf16(int dim, int rows);
AttendForm attend_form_sinks_f16(int dim, int rows);

template <int TYPE, int DH, bool FULL, bool SINKS>
AttendForm attend_form_at(int rows) {
    const auto form = [](AttendKernel kernel, int height, int waves) { return AttendForm{kernel, height, 64 * waves, height * (DH + 4)}; };
    if (rows > few_rows(TYPE)) {
        if constexpr (TYPE == kCacheF32) {
            return form(attend_wide_kernel<DH, FULL, DH == 64 ? 64 : 32, SINKS>, kTileRows, kTileWaves);
        } else {
            return form(attend_tile_kernel<TYPE, DH, FULL, DH == 256 ? 32 : 64, SINKS>, kTileRows, kTileWaves);
        }
    }
    return form(attend_rows_kernel<TYPE, DH, FULL, SINKS>, kFewTile, attend_waves(TYPE, DH));
}

template <int TYPE, bool SINKS>
AttendForm attend_form_of(int dim, int rows) {
    if (dim > 128) return attend_form_at<TYPE, 256, false, SINKS>(rows);
    if (dim == 128) return attend_form_at<TYPE, 128, true, SINKS>(rows);
    if (dim > 64) return attend_form_at<TYPE, 128, false, SINKS>(rows);
    if (dim == 64) return attend_form_at<TYPE, 64, true, SINKS>(rows);
    return attend_form_at<TYPE, 64, false, SINKS>(rows);
}

}  // namespace gh
