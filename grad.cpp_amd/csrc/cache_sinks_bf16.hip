// Attention over paged caches of bf16, with a window and the first positions beside it: the kernels of this element type.
#include "cache_attend.h"

namespace gh {

AttendForm attend_form_sinks_bf16(int dim, int rows) { return attend_form_of<kCacheBf16, true>(dim, rows); }

}  // namespace gh
