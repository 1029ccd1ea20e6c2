#include "cache_attend_impl.h"

namespace mxq {
void launch_attend_pairs_f16(const AttendArgs& a, bool many, bool wide, int64_t groups, hipStream_t st) { launch_attend<kPairs, MXQ_DT_F16>(a, many, wide, groups, st); }
}  // namespace mxq
