#include "linear_tile_impl.h"

namespace mxq {
void launch_tile_e5m2(const TileArgs& a, const TilePlan& p, hipStream_t st) { launch_tile_family<kE5M2>(a, p, st); }
}  // namespace mxq
