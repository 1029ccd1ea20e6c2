#include "cache_attend_impl.h"

namespace mxq {
void launch_attend_e5m2_bf16(const AttendArgs& a, bool many, bool wide, int64_t groups, hipStream_t st) { launch_attend<kE5M2, MXQ_DT_BF16>(a, many, wide, groups, st); }
}  // namespace mxq
