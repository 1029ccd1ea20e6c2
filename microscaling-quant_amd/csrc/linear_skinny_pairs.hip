#include "linear_skinny_impl.h"

namespace mxq {
void launch_skinny_pairs(const LinearArgs& a, int64_t tiles, hipStream_t st) { launch_skinny_family<kPairs>(a, tiles, st); }
}  // namespace mxq
