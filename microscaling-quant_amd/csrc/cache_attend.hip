// Attention over a cache in MX formats (include/mxq_hip.h, mxq_cache_attend): which kernel takes a call, and the sums of
// the sequences whose keys were cut into runs.
#include "cache_common.h"

namespace mxq {

#define MXQ_LAUNCH(NAME) void NAME(const AttendArgs&, bool many, bool wide, int64_t groups, hipStream_t);
MXQ_LAUNCH(launch_attend_e4m3_f32)
MXQ_LAUNCH(launch_attend_e4m3_bf16)
MXQ_LAUNCH(launch_attend_e4m3_f16)
MXQ_LAUNCH(launch_attend_e5m2_f32)
MXQ_LAUNCH(launch_attend_e5m2_bf16)
MXQ_LAUNCH(launch_attend_e5m2_f16)
MXQ_LAUNCH(launch_attend_pairs_f32)
MXQ_LAUNCH(launch_attend_pairs_bf16)
MXQ_LAUNCH(launch_attend_pairs_f16)
#undef MXQ_LAUNCH

namespace {

constexpr int64_t kMostKeys = 0x7fff0000;     // of a sequence, as its table has room for them
constexpr int kUnits = 256;                   // CUs
// Steps of 32 keys that a workgroup takes at least: one token's 8000 keys 19.1 us, with 4 steps 20.4, with 16 21.0.
constexpr int kLeast = 8;
// Rows a sequence up to which its keys are what a call costs, and tiles of few rows take them.  Eight sequences of 4096 keys
// with 32, 64 and 128 rows of each head: 37, 43 and 58 us by tiles of few rows, 42, 52 and 62 by tiles of many; past 64 rows
// each 32 of them read the keys again.
constexpr int kFewRows = 64;

// Whether tiles stay whole, `steps` of keys each at most.  Workgroups that take equal pieces end together, however unlike the
// tiles are, but parts and their join cost about as long as kCutFew or kCutMany steps.
// Many rows: four prompts of 512, 1024 and 2048 tokens (one, two and four tiles of 128 rows a workgroup; 32 heads of 128
// columns, 8 of MXFP4 keys): 39, 86 and 242 us whole, 68, 116 and 292 cut.  With fewer tiles than workgroups: one prompt of
// 1024, half a tile each, 43 us whole and 60 cut; four of 256 that end contexts of 8192, 295 and 240.  Sequences of unlike
// lengths and numbers of queries, 2.5 tiles a workgroup: 198 and 182.
// Few rows, one token of each sequence, the same heads: one sequence of 500, 1500 and 3000 keys 11, 18 and 29 us whole, 18, 19
// and 20 cut; 16 of 1000, 2000 and 3000 15, 25 and 33, and 24, 27 and 30; 48 of 2000 and 3000 30 and 40, and 43 and 51.  Past
// twice that many steps one sequence's length could make whole tiles the slower ones by more than cutting costs.
constexpr int kWholeTiles = 3, kCutMany = 24, kCutFew = 56;
bool stay_whole(bool many, int64_t tiles, int64_t wanted, int64_t steps, bool unlike) {
  if (!many) return steps <= 2 * kCutFew && steps * (wanted - (unlike ? 0 : tiles)) <= kCutFew * wanted;
  if (tiles >= wanted) return !unlike || tiles >= kWholeTiles * wanted;
  return steps * (wanted - tiles) <= kCutMany * wanted;
}
// Sequences up to which each workgroup of a whole tile looks for it among all of them, 64 at once; with more, workgroups take
// pieces of the line, and find the tile behind one where it is.  2048 sequences of 128 tokens: 2.0 ms, and 8.6 of whole tiles;
// 128 of 128: 0.17 and 0.18; 4096 sequences' tokens over 200 keys: 0.75 and 2.3; but 128 of them 34 us and 21 of whole tiles.
constexpr int kLookFew = 256, kLookMany = 64;

int wanted_of(int dtype, int blocks, int rows, bool many) { return kUnits * attend_groups(dtype, blocks, rows / 16 / (many ? kWaves : 1)); }

// What differs between the two ways that a call's sequences are taken.
struct JoinWay {
  float* partial;
  int32_t above, upto, wanted, size;
  int32_t places, shares;    // workgroups: tiles, or pieces of the line where they are fewer, and what shares one's rows
  bool by_tile;
};
struct JoinWays {
  JoinWay way[2];
};
// The rows of tiles that lie in two pieces of the line and more, from their parts' sums in the pieces' order.  A workgroup takes rows of a tile, or of the tile that a piece ends in, if that is the tile's first end
// of a piece: sixteen lanes a row, or the workgroup a row, its sixteens of lanes the parts in turn, whichever waits less often
// for loads.  One token's 131072 keys of 8 heads, in 64 parts a head, take 44 us by workgroups and 55 by sixteens; prompts in
// two to four parts a tile 67 by sixteens and 219 by workgroups.
// It is bound by its parts' bytes where they are many (23 sequences of up to 512 tokens, 1000 parts of 128 rows of 128 columns:
// 67 MB in 20 us) and by four loads one behind another else: 6 to 9 us.
// Workgroups that share what there is to join, twice as many of tiles of many rows: 64 sequences' 512 tiles of 4 to 8 rows took
// 128 us with 512 of them, 131 with 1024 and 139 with 2048 (most find nothing), prompts of 128 rows a tile 198, 193 and 198.
constexpr int kJoins = 512;
constexpr int kAtOnce = 4;                    // parts asked for together
// Sums of weights and of values relative to 2^best, and those of a part relative to its own maximum, `best` at most.  A part
// that has seen no key has sums of zero; any other's are taken with a factor of zero too, so that NaN of a value stays NaN.
template <int V> __device__ __forceinline__ void add_part(float& all, float (&v)[V], float top, float weight, float best, const float (&x)[V]) {
  // a part without a maximum has seen no key, or only scores of NaN, which its sum is then
  const bool none = top == -__builtin_inff();
  const float factor = none ? weight : __builtin_amdgcn_exp2f(top - best);
  all += none ? weight : factor * weight;
#pragma unroll
  for (int k = 0; k < V; ++k) v[k] += factor * x[k];
}
template <int COLUMNS>
__global__ __launch_bounds__(256) void k_attend_join(AttendArgs a, JoinWays ways) {
  constexpr int V = COLUMNS / 16;
  __shared__ float sums[16][COLUMNS];
  __shared__ float weights[16], maxima[16];
  struct Found {
    Tile u;
    int group, runs;           // its first piece, and in how many it lies
    bool at_begin;
  };
  __shared__ Found found;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, D = a.c.head_dim, c = lane & 15, sixteen = threadIdx.x >> 4;
  const int first_way = ways.way[0].places * ways.way[0].shares, which = (int)blockIdx.x >= first_way;
  const JoinWay& w = ways.way[which];
  const int index = (int)blockIdx.x - (which ? first_way : 0);
  if (index >= w.places * w.shares) return;
  const int share = index / w.places, place = index - share * w.places, size = w.size;
  a.above = w.above, a.upto = w.upto, a.wanted = w.wanted;
  if (a.fill) fill_rows(a);
  // one wave finds the tile: what it takes to find it is most of what a workgroup computes
  if (wave == 0) {
    Member own = member(a, lane, size, 0.0);
    const Line line = line_of(a, size, own);
    Found f{};
    if (w.by_tile || place + 1 < line.groups) {
      f.u = tile_of(a, size, own, line.unit, w.by_tile ? place : line.begin(place + 1), w.by_tile);
      if (f.u.b >= 0 && (w.by_tile || (f.u.first != line.begin(place + 1) && f.u.first >= line.begin(place)))) {
        f.group = w.by_tile ? line.group_at(f.u.first) : place;
        f.runs = line.group_at(f.u.first + f.u.weight - 1) - f.group + 1;
        f.at_begin = line.begin(f.group) == f.u.first;          // of the first piece it is the first tile
      }
    }
    if (lane == 0) found = f;
  }
  __syncthreads();
  const Tile u = found.u;
  const int g0 = same(found.group), runs = same(found.runs);
  if (runs < 2) return;
  const bool at_begin = found.at_begin;
  const int rows = u.s.n * a.group, row0 = u.row * size, last = rows - row0 < size ? rows - row0 : size;
  const int shares = w.shares, by_rows = (last + 16 * shares - 1) / (16 * shares) * (runs / kAtOnce + 1);
  const bool many = (last + shares - 1) / shares * (runs / (16 * kAtOnce) + 2) < by_rows;
  for (int r = many ? share : share * 16 + sixteen; r < last; r += many ? shares : shares * 16) {
    auto part_of = [&](int i) { return w.partial + (part_slot(g0 + i, i || at_begin) * size + r) * (COLUMNS + 2); };
    float best = -__builtin_inff(), all = 0.0f, v[V];
#pragma unroll
    for (int k = 0; k < V; ++k) v[k] = 0.0f;
    const int by = many ? 16 : 1;
    for (int i0 = many ? sixteen : 0; i0 < runs; i0 += kAtOnce * by) {
      float x[kAtOnce][V], tops[kAtOnce], weight[kAtOnce];
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u) {
        const int i = i0 + u * by;
        const float* part = part_of(i < runs ? i : i0);
        tops[u] = i < runs ? part[COLUMNS] : -__builtin_inff(), weight[u] = i < runs ? part[COLUMNS + 1] : 0.0f;
#pragma unroll
        for (int k = 0; k < V; k += 4) __builtin_memcpy(x[u] + k, part + k * 16 + c * 4, 16);
      }
      float now = best;
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u) now = __builtin_fmaxf(now, tops[u]);
      const float keep = best == now ? 1.0f : __builtin_amdgcn_exp2f(best - now);
      all *= keep;
#pragma unroll
      for (int k = 0; k < V; ++k) v[k] = keep * v[k];
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u)
        if (i0 + u * by < runs) add_part(all, v, tops[u], weight[u], now, x[u]);
      best = now;
    }
    if (many) {
      if (c == 0) weights[sixteen] = all, maxima[sixteen] = best;
#pragma unroll
      for (int k = 0; k < V; ++k) sums[sixteen][k / 4 * 64 + c * 4 + k % 4] = v[k];
      __syncthreads();
      if (sixteen == 0) {
        best = maxima[0], all = 0.0f;
#pragma unroll
        for (int j = 1; j < 16; ++j) best = __builtin_fmaxf(best, maxima[j]);
#pragma unroll
        for (int k = 0; k < V; ++k) v[k] = 0.0f;
        for (int j = 0; j < 16; ++j) {
          float x[V];
#pragma unroll
          for (int k = 0; k < V; ++k) x[k] = sums[j][k / 4 * 64 + c * 4 + k % 4];
          add_part(all, v, maxima[j], weights[j], best, x);
        }
      }
      __syncthreads();
      if (sixteen) continue;
    }
    const float inv = all == 0.0f ? 0.0f : 1.0f / all;
    const int t = (int)divu31(row0 + r, a.by_group), h = u.head * a.group + row0 + r - t * a.group;
    const int64_t row = (int64_t)(u.s.start + t) * a.a.heads + h;
#pragma unroll
    for (int k = 0; k < V; k += 4) {
      const int d = k * 16 + c * 4;
      const float y[4] = {v[k] * inv, v[k + 1] * inv, v[k + 2] * inv, v[k + 3] * inv};
      if (a.a.dtype == MXQ_DT_F32) store_four<MXQ_DT_F32>(a.out, row * D + d, D - d, y);
      else if (a.a.dtype == MXQ_DT_BF16) store_four<MXQ_DT_BF16>(a.out, row * D + d, D - d, y);
      else store_four<MXQ_DT_F16>(a.out, row * D + d, D - d, y);
    }
    if (a.lse && c == 0) a.lse[row] = log_sum(best, all);
  }
}

__global__ __launch_bounds__(256) void k_attend_none(AttendArgs a) { fill_rows(a); }

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
  if (!(a->scale > 0.0f) || a->scale > 0x1p127f) return invalid(who + ": scale must be positive, and 2^127 at most");
  if (a->window < 0 || a->window > 0x7fffffff) return invalid(who + ": window out of range");
  // keys are counted in 32 bits, also those that a wave looks for ahead of its last one
  if (a->table_pages < 0 || a->table_pages > 0x7fffffff || a->table_pages * c->page_size > kMostKeys) return invalid(who + ": table out of range");
  return MXQ_OK;
}

// How a call is taken: sequences of few rows (queries times the heads that share one of keys) by tiles whose keys the waves
// share, others by tiles whose waves have rows of their own.  Without starts every sequence has as many, so that one of the
// two does it.
struct Way {
  int rows;                  // of a tile; 0: nothing goes this way
  int64_t tiles, groups;     // as many as there may be, of all heads; workgroups
  int64_t bytes;             // workspace; 0: no tile is cut
};
struct Plan {
  int limit;                 // rows a sequence that are few
  Way way[2];
};
Plan plan_of(const mxq_cache_spec& c, const mxq_attend_spec& a, bool ragged) {
  const int64_t group = a.heads / c.kv_heads, n = ragged ? a.T : a.T / a.B, rows = n * group, least = ragged ? group : rows;
  const int blocks = blocks_class((c.head_dim + 31) / 32);
  Plan p = {};
  // 32 rows share a step's conversions and loads: 64 sequences of 4096 keys with 32 rows a head take 91 us so and 126 by 16 rows
  // a tile, but eight of them, which do not fill the card, 37 and 34.
  if (least <= kFewRows) p.limit = kFewRows, p.way[0].rows = least <= 16 || blocks == 8 ? 16 : 32;
  if (rows > p.limit) p.way[1].rows = 16 * kWaves * attend_rows(a.dtype, blocks);
  const int64_t keys = a.table_pages * c.page_size, seen = a.window && a.window < keys ? a.window + n : keys;
  for (int many = 0; many < 2; ++many) {
    Way& w = p.way[many];
    if (!w.rows) continue;
    // of sequences that may go this way, each with a tile that is not full
    const int64_t most = many ? rows / (p.limit + 1) : a.T, sequences = most < a.B ? most : a.B;
    w.tiles = ragged ? rows / w.rows + sequences : a.B * ceil_div(rows, w.rows);
    if (ragged && !many && w.tiles > a.B * ceil_div(p.limit, w.rows)) w.tiles = a.B * ceil_div(p.limit, w.rows);
    w.tiles *= c.kv_heads;
    w.groups = w.tiles;
    const int64_t wanted = wanted_of(a.dtype, blocks, w.rows, many);
    if (a.B <= (many ? kLookMany : kLookFew) && stay_whole(many, w.tiles, wanted, ceil_div(keys < seen ? keys : seen, kStep), ragged && a.B > 1)) continue;
    w.groups = wanted;
    w.bytes = 2 * w.groups * w.rows * (32 * blocks + 2) * (int64_t)sizeof(float);
  }
  return p;
}

}  // namespace
}  // namespace mxq

extern "C" int64_t mxq_cache_attend_workspace(const mxq_cache_spec* cache, const mxq_attend_spec* spec, int32_t ragged) {
  using namespace mxq;
  if (check(cache, spec) || spec->T == 0 || spec->B == 0) return 0;
  const Plan p = plan_of(*cache, *spec, ragged);
  return p.way[0].bytes + p.way[1].bytes;
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
  const int64_t group = spec->heads / cache->kv_heads;
  AttendArgs a = {};
  a.q = q, a.kc = k_codes, a.ks = k_scales, a.vc = v_codes, a.vs = v_scales;
  a.table = table, a.lengths = lengths, a.starts = starts, a.out = out, a.lse = lse;
  a.c = *cache, a.a = *spec;
  a.by_page = make_divu31((uint32_t)cache->page_size), a.by_group = make_divu31((uint32_t)group);
  a.group = (int)group, a.blocks = (cache->head_dim + 31) / 32;
  a.aligned = cache->page_size % 16 == 0;
  for (int64_t r : cache->row_stride) a.aligned = a.aligned && r >= 0 && r < 1 << 26;
  a.scale2 = spec->scale * 1.44269504088896341f;
  hipStream_t st = as_stream(stream);
  a.least = kLeast;
  const Plan p = spec->B ? plan_of(*cache, *spec, starts != nullptr) : Plan{};
  const bool cut = p.way[0].bytes || p.way[1].bytes;
  if (cut && !workspace) return invalid("mxq_cache_attend: NULL workspace");
  for (const Way& w : p.way)
    if (w.groups * 64 * kWaves > kMaxThreads) return invalid("mxq_cache_attend: too many tiles for a launch");
  const int blocks = blocks_class(a.blocks);
  constexpr decltype(&launch_attend_e4m3_f32) launches[3][3] = {{launch_attend_e4m3_f32, launch_attend_e4m3_bf16, launch_attend_e4m3_f16},
                                                                {launch_attend_e5m2_f32, launch_attend_e5m2_bf16, launch_attend_e5m2_f16},
                                                                {launch_attend_pairs_f32, launch_attend_pairs_bf16, launch_attend_pairs_f16}};
  const auto launch = launches[cache->format == MXQ_FMT_E4M3 ? 0 : cache->format == MXQ_FMT_E5M2 ? 1 : 2][spec->dtype];
  a.fill = starts && !cut;
  if (!spec->B) {
    KernelTimer timer("k_attend_none", st);
    k_attend_none<<<dim3(blocks_for(ceil_div(spec->T * spec->heads, 64))), 256, 0, st>>>(a);
    return check_launch("mxq_cache_attend");
  }
  JoinWays ways = {};
  int64_t joins = 0;
  char* work = (char*)workspace;
  for (int many = 0; many < 2; ++many) {
    const Way& w = p.way[many];
    if (!w.rows) continue;
    a.partial = w.bytes ? (float*)work : nullptr;
    work += w.bytes;
    a.above = many ? p.limit : 0, a.upto = many ? 0x7fffffff : p.limit;
    a.wanted = wanted_of(spec->dtype, blocks, w.rows, many);
    {
      KernelTimer timer("k_attend", st);
      launch(a, many, w.rows == 32, w.groups, st);
    }
    if (int rc = check_launch("mxq_cache_attend")) return rc;
    a.fill = 0;
    if (!a.partial) continue;
    const bool by_tile = w.tiles <= a.wanted;
    const int places = by_tile ? (int)w.tiles : a.wanted, most = many ? w.rows / 16 : 16, spare = (many ? 2 : 1) * kJoins / places;
    const int shares = spare < 1 ? 1 : spare < most ? spare : most;
    ways.way[many] = JoinWay{a.partial, a.above, a.upto, a.wanted, w.rows, places, shares, by_tile};
    joins += places * shares;
  }
  if (joins) {
    a.fill = starts != nullptr;
    const auto join = blocks == 2 ? k_attend_join<64> : blocks == 4 ? k_attend_join<128> : k_attend_join<256>;
    KernelTimer timer("k_attend_join", st);
    join<<<dim3((unsigned)joins), 256, 0, st>>>(a, ways);
    return check_launch("mxq_cache_attend");
  }
  return MXQ_OK;
}
