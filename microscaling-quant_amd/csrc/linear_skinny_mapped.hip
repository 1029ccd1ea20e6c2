#include "linear_skinny_impl.h"

namespace mxq {
void launch_skinny_mapped(const LinearArgs& a, int64_t tiles, hipStream_t st) { launch_skinny_family<kMapped>(a, tiles, st); }
}  // namespace mxq
