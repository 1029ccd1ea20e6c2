#include "cache_attend_few_impl.h"

namespace mxq {
void launch_attend_few_e4m3(const AttendArgs& a, int64_t units, int least, hipStream_t st) { launch_attend_few<kE4M3>(a, units, least, st); }
}  // namespace mxq
