// Attention over paged caches of f32, with a window and the first positions beside it: the kernels of this element type.
#include "cache_attend.h"

namespace gh {

AttendForm attend_form_sinks_f32(int dim, int rows) { return attend_form_of<kCacheF32, true>(dim, rows); }

}  // namespace gh
