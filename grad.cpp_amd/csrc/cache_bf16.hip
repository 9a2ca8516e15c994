// Attention over paged caches of bf16: the kernels of this element type.
#include "cache_attend.h"

namespace gh {

AttendForm attend_form_bf16(int dim, int rows) { return attend_form_of<kCacheBf16, false>(dim, rows); }

}  // namespace gh
