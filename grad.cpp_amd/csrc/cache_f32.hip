// Attention over paged caches of f32: the kernels of this element type.
#include "cache_attend.h"

namespace gh {

AttendForm attend_form_f32(int dim, int rows) { return attend_form_of<kCacheF32, false>(dim, rows); }

}  // namespace gh
