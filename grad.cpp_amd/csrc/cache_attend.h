// Which attention kernel takes a pass; one translation unit per element type makes them.
#pragma once

#include "kernels_cache_attn.h"

namespace gh {

using AttendKernel = void (*)(AttendParams);

struct AttendForm {
    AttendKernel kernel;
    int height;      // rows of a tile
    int part_floats; // of a tile's part in memory
};

// The form for tiles of up to 16 * tiles rows of heads of `dim` dims.
AttendForm attend_form_f32(int dim, int tiles);
AttendForm attend_form_bf16(int dim, int tiles);
AttendForm attend_form_f16(int dim, int tiles);

template <int TYPE>
AttendForm attend_form_of(int dim, int tiles) {
    const auto form = [](AttendKernel kernel, int width, int t) { return AttendForm{kernel, 16 * t, 16 * t * (width + 4)}; };
    if (dim > 128) return form(attend_rows_kernel<TYPE, 256, false, 1>, 256, 1);
    if (dim == 128)
        return tiles > 1 ? form(attend_rows_kernel<TYPE, 128, true, 2>, 128, 2) : form(attend_rows_kernel<TYPE, 128, true, 1>, 128, 1);
    if (dim > 64)
        return tiles > 1 ? form(attend_rows_kernel<TYPE, 128, false, 2>, 128, 2) : form(attend_rows_kernel<TYPE, 128, false, 1>, 128, 1);
    if (dim == 64)
        return tiles > 1 ? form(attend_rows_kernel<TYPE, 64, true, 2>, 64, 2) : form(attend_rows_kernel<TYPE, 64, true, 1>, 64, 1);
    return tiles > 1 ? form(attend_rows_kernel<TYPE, 64, false, 2>, 64, 2) : form(attend_rows_kernel<TYPE, 64, false, 1>, 64, 1);
}

}  // namespace gh
