#include "linear_tile_impl.h"

namespace mxq {
void launch_tile_pairs(const TileArgs& a, const TilePlan& p, hipStream_t st) { launch_tile_family<kPairs>(a, p, st); }
}  // namespace mxq
