// Attention over paged caches of f16: the kernels of this element type.
#include "cache_attend.h"

namespace gh {

AttendForm attend_form_f16(int dim, int rows) { return attend_form_of<kCacheF16, false>(dim, rows); }

}  // namespace gh
