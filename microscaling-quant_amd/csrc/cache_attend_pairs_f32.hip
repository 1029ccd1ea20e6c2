#include "cache_attend_impl.h"

namespace mxq {
void launch_attend_pairs_f32(const AttendArgs& a, bool many, bool wide, int64_t groups, hipStream_t st) { launch_attend<kPairs, MXQ_DT_F32>(a, many, wide, groups, st); }
}  // namespace mxq
