#include "cache_attend_few_impl.h"

namespace mxq {
void launch_attend_few_pairs(const AttendArgs& a, int64_t units, int least, hipStream_t st) { launch_attend_few<kPairs>(a, units, least, st); }
}  // namespace mxq
