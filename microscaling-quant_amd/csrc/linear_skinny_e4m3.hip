#include "linear_skinny_impl.h"

namespace mxq {
void launch_skinny_e4m3(const LinearArgs& a, int64_t tiles, hipStream_t st) { launch_skinny_family<kE4M3>(a, tiles, st); }
}  // namespace mxq
