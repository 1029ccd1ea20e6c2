#include "linear_tile_impl.h"

namespace mxq {
void launch_tile_e4m3(const TileArgs& a, const TilePlan& p, hipStream_t st) { launch_tile_family<kE4M3>(a, p, st); }
}  // namespace mxq
