// The attention kernel's instances for q of GSK_BF16 over a cache of GSK_E4M3.
#include "gsk_attend_body.h"

namespace gse {

void launch_attend_bf16_e4m3(const AttendArgs &p, int mt, dim3 grid, hipStream_t s) { launch_attend_types<GSK_BF16, GSK_E4M3>(p, mt, grid, s); }

}  // namespace gse
