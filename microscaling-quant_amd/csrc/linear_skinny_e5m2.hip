#include "linear_skinny_impl.h"

namespace mxq {
void launch_skinny_e5m2(const LinearArgs& a, int64_t tiles, hipStream_t st) { launch_skinny_family<kE5M2>(a, tiles, st); }
}  // namespace mxq
