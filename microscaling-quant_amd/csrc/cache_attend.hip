// Attention over a cache in MX formats (include/mxq_hip.h, mxq_cache_attend): which kernel takes a call, and the sums of
// the sequences whose keys were cut into runs.
#include "cache_common.h"

namespace mxq {

void launch_attend_few_e4m3(const AttendArgs&, int64_t, int, hipStream_t);
void launch_attend_few_e5m2(const AttendArgs&, int64_t, int, hipStream_t);
void launch_attend_few_pairs(const AttendArgs&, int64_t, int, hipStream_t);

namespace {

constexpr int kFewRows = 16, kFewLeast = 8, kUnits = 256;   // rows a tile, steps a workgroup at least, CUs

// The rows of tiles that were cut, from their parts' sums, and zeros for rows of no sequence.  A workgroup takes every
// gridDim.y-th row of a tile of rows, its waves the runs in turn, then the waves' sums in their order.
template <int COLUMNS>
__global__ __launch_bounds__(256) void k_attend_join(AttendArgs a, int unit_rows, int least) {
  constexpr int V = COLUMNS / 64;
  __shared__ float sums[4][COLUMNS];
  __shared__ float weights[4];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, D = a.c.head_dim;
  if (a.starts) {
    // queries [0, starts[0]) and [starts[B], T) are no sequence's
    const int T = (int)a.a.T, x = a.a.B ? a.starts[0] : T, y = a.a.B ? a.starts[a.a.B] : T;
    const int64_t head = (int64_t)(x < 0 ? 0 : x > T ? T : x) * a.a.heads, tail = (int64_t)(y < 0 ? 0 : y > T ? T : y) * a.a.heads;
    const int64_t from = tail < head ? head : tail, all = head + (a.a.T * a.a.heads - from);
    const int64_t groups = (int64_t)gridDim.x * gridDim.y, me = (int64_t)blockIdx.y * gridDim.x + blockIdx.x;
    for (int64_t i = me * 4 + wave; i < all; i += groups * 4) {
      const int64_t row = i < head ? i : from + i - head;
      for (int d = lane; d < D; d += 64) store_elem(a.out, a.a.dtype, row * D + d, 0.0f);
      if (a.lse && lane == 0) a.lse[row] = -__builtin_inff();
    }
  }
  if (!a.partial) return;
  const Tile u = tile_of(a, unit_rows, blockIdx.x, true);
  if (u.b < 0) return;
  const Line line = line_of(a, unit_rows, least);
  const int g0 = same(line.group_at(u.first)), runs = same(line.group_at(u.first + u.steps - 1)) - g0 + 1;
  if (runs == 1) return;
  const bool at_begin = line.begin(g0) == u.first;          // of the first group's piece the tile is the first
  const Sequence s = same(sequence(a, u.b));
  const int rows = s.n * a.group, row_tiles = (rows + unit_rows - 1) / unit_rows, kv_head = u.index / row_tiles;
  const int row0 = (u.index - kv_head * row_tiles) * unit_rows, last = rows - row0 < unit_rows ? rows - row0 : unit_rows;
  for (int r = blockIdx.y; r < last; r += gridDim.y) {
    auto part_of = [&](int i) { return a.partial + (part_slot(g0 + i, i || at_begin) * unit_rows + r) * (COLUMNS + 2); };
    float best = -__builtin_inff(), all = 0.0f, v[V];
#pragma unroll
    for (int k = 0; k < V; ++k) v[k] = 0.0f;
    for (int i = lane; i < runs; i += 64) best = __builtin_fmaxf(best, part_of(i)[COLUMNS]);
    for (int o = 32; o; o >>= 1) best = __builtin_fmaxf(best, __shfl_xor(best, o));
#pragma unroll 4
    for (int i = wave; i < runs; i += 4) {
      const float* part = part_of(i);
      const float top = part[COLUMNS], sum = part[COLUMNS + 1];
      // a run without a maximum has seen no key, or only scores of NaN, which its sum is then
      const float factor = top == -__builtin_inff() ? sum : __builtin_amdgcn_exp2f(top - best);
      float x[V];
#pragma unroll
      for (int k = 0; k < V; ++k) x[k] = part[lane * V + k];
      all += top == -__builtin_inff() ? sum : factor * sum;
#pragma unroll
      for (int k = 0; k < V; ++k) v[k] += factor == 0.0f ? 0.0f : factor * x[k];
    }
    if (lane == 0) weights[wave] = all;
#pragma unroll
    for (int k = 0; k < V; ++k) sums[wave][lane * V + k] = v[k];
    __syncthreads();
    const int t = (int)divu31(row0 + r, a.by_group), h = kv_head * a.group + row0 + r - t * a.group;
    const int64_t row = (int64_t)(s.start + t) * a.a.heads + h;
    all = ((weights[0] + weights[1]) + weights[2]) + weights[3];
    const float inv = all == 0.0f ? 0.0f : 1.0f / all;
    for (int d = threadIdx.x; d < D; d += 256)
      store_elem(a.out, a.a.dtype, row * D + d, (((sums[0][d] + sums[1][d]) + sums[2][d]) + sums[3][d]) * inv);
    if (a.lse && threadIdx.x == 0) a.lse[row] = log_sum(best, all);
    __syncthreads();
  }
}

int check(const mxq_cache_spec* c, const mxq_attend_spec* a) {
  const std::string who = "mxq_cache_attend";
  if (!c || !a) return invalid(who + ": NULL spec");
  if (c->format != MXQ_FMT_E4M3 && c->format != MXQ_FMT_E5M2 && c->format != MXQ_FMT_E2M1_PAIRS) return invalid(who + ": unknown format");
  if (c->head_dim < 1 || c->head_dim > 256) return invalid(who + ": head_dim must be 1 to 256");
  if (c->pages < 1 || c->page_size < 1 || c->pages > 0x7fffffff || c->page_size > 0x7fffffff || c->pages * c->page_size > 0x7fffffff ||
      c->kv_heads < 1 || c->kv_heads > 65535)
    return invalid(who + ": cache size out of range");
  if (a->dtype < MXQ_DT_F32 || a->dtype > MXQ_DT_F16) return invalid(who + ": unknown dtype");
  if (a->T < 0 || a->B < 0 || a->heads < 1 || a->T > 0x3fffffff || a->B > 0x3fffffff || a->heads > 0x3fffffff || a->T * a->heads > 0x3fffffff)
    return invalid(who + ": size out of range");
  if (a->heads % c->kv_heads) return invalid(who + ": heads must be a multiple of kv_heads");
  if (!(a->scale > 0.0f) || a->scale > 3.4e38f) return invalid(who + ": scale must be positive and finite");
  if (a->window < 0 || a->window > 0x7fffffff) return invalid(who + ": window out of range");
  if (a->table_pages < 0 || a->table_pages > 0x7fffffff) return invalid(who + ": table out of range");
  return MXQ_OK;
}

// Tiles of `rows` rows that a call may have, and whether they may be cut: not where no sequence has keys for it.
struct Plan {
  int64_t tiles;
  bool split;
};
Plan plan_of(const mxq_cache_spec& c, const mxq_attend_spec& a, bool ragged, int rows, int least) {
  const int64_t group = a.heads / c.kv_heads;
  int64_t tiles;
  if (ragged) tiles = a.T * group / rows + (a.B < a.T ? a.B : a.T);
  else tiles = a.B * ceil_div(a.T / a.B * group, rows);
  const int64_t keys = a.table_pages * c.page_size, seen = a.window && a.window < keys ? a.window + (ragged ? a.T : a.T / a.B) : keys;
  return Plan{tiles * c.kv_heads, (keys < seen ? keys : seen) > (int64_t)(least - 1) * kStep};
}
int columns_of(int head_dim) { return head_dim <= 64 ? 64 : head_dim <= 128 ? 128 : 256; }

}  // namespace
}  // namespace mxq

extern "C" int64_t mxq_cache_attend_workspace(const mxq_cache_spec* cache, const mxq_attend_spec* spec, int32_t ragged) {
  using namespace mxq;
  if (check(cache, spec) || spec->T == 0 || spec->B == 0) return 0;
  const Plan p = plan_of(*cache, *spec, ragged, kFewRows, kFewLeast);
  const int64_t groups = kUnits * few_groups(spec->dtype, (cache->head_dim + 31) / 32);
  return p.split ? 2 * groups * kFewRows * (columns_of(cache->head_dim) + 2) * (int64_t)sizeof(float) : 0;
}

extern "C" int mxq_cache_attend(const void* q, const uint8_t* k_codes, const uint8_t* k_scales, const uint8_t* v_codes,
                                const uint8_t* v_scales, const mxq_cache_spec* cache, const int32_t* table, const int32_t* lengths,
                                const int32_t* starts, void* out, float* lse, const mxq_attend_spec* spec, void* workspace,
                                mxq_stream_t stream) {
  using namespace mxq;
  if (int rc = check(cache, spec)) return rc;
  if (spec->T == 0) return MXQ_OK;
  if (!starts && (spec->B == 0 || spec->T % spec->B)) return invalid("mxq_cache_attend: T must be a multiple of B without starts");
  if (!q || !k_codes || !k_scales || !v_codes || !v_scales || !out || (spec->B && (!lengths || (spec->table_pages && !table))))
    return invalid("mxq_cache_attend: NULL pointer");
  const int columns = columns_of(cache->head_dim);
  const int64_t group = spec->heads / cache->kv_heads;
  AttendArgs a = {};
  a.q = q, a.kc = k_codes, a.ks = k_scales, a.vc = v_codes, a.vs = v_scales;
  a.table = table, a.lengths = lengths, a.starts = starts, a.out = out, a.lse = lse;
  a.c = *cache, a.a = *spec;
  a.by_page = make_divu31((uint32_t)cache->page_size), a.by_group = make_divu31((uint32_t)group);
  a.group = (int)group, a.blocks = (cache->head_dim + 31) / 32;
  a.wanted = kUnits * few_groups(spec->dtype, a.blocks);
  a.aligned = cache->page_size % 16 == 0;
  for (int64_t r : cache->row_stride) a.aligned = a.aligned && r >= 0 && r < 1 << 26;
  a.scale2 = spec->scale * 1.44269504088896341f;
  hipStream_t st = as_stream(stream);
  Plan p = {};
  if (spec->B) {
    p = plan_of(*cache, *spec, starts != nullptr, kFewRows, kFewLeast);
    if (p.split && !workspace) return invalid("mxq_cache_attend: NULL workspace");
    if (p.tiles * 256 > kMaxThreads) return invalid("mxq_cache_attend: too many tiles for a launch");
    a.partial = p.split ? (float*)workspace : nullptr;
    auto launch = cache->format == MXQ_FMT_E4M3 ? launch_attend_few_e4m3 : cache->format == MXQ_FMT_E5M2 ? launch_attend_few_e5m2 : launch_attend_few_pairs;
    launch(a, p.tiles, kFewLeast, st);
    if (int rc = check_launch("mxq_cache_attend")) return rc;
  }
  if (a.partial || starts) {
    // few tiles: a workgroup for each of their rows
    const int64_t tiles = a.partial ? p.tiles : blocks_for(ceil_div(spec->T * spec->heads, 64));
    const dim3 grid((unsigned)tiles, (unsigned)(tiles >= 2048 ? 1 : tiles >= 512 ? 4 : 16));
    if (columns == 64) k_attend_join<64><<<grid, 256, 0, st>>>(a, kFewRows, kFewLeast);
    else if (columns == 128) k_attend_join<128><<<grid, 256, 0, st>>>(a, kFewRows, kFewLeast);
    else k_attend_join<256><<<grid, 256, 0, st>>>(a, kFewRows, kFewLeast);
    return check_launch("mxq_cache_attend");
  }
  return MXQ_OK;
}
