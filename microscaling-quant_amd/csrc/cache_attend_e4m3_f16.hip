#include "cache_attend_impl.h"

namespace mxq {
void launch_attend_e4m3_f16(const AttendArgs& a, bool many, bool wide, int64_t groups, hipStream_t st) { launch_attend<kE4M3, MXQ_DT_F16>(a, many, wide, groups, st); }
}  // namespace mxq
