// The attention kernel's instances for q of GSK_BF16 over a cache of GSK_I8.
#include "gsk_attend_body.h"

namespace gse {

void launch_attend_bf16_i8(const AttendArgs &p, int mt, dim3 grid, hipStream_t s) { launch_attend_types<GSK_BF16, GSK_I8>(p, mt, grid, s); }

}  // namespace gse
