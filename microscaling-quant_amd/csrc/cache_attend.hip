// Attention over a cache in MX formats (include/mxq_hip.h, mxq_cache_attend): which kernel takes a call, and the sums of
// the sequences whose keys were cut into runs.
#include "cache_common.h"

namespace mxq {

void launch_attend_few_e4m3(const AttendArgs&, int64_t, int, hipStream_t);
void launch_attend_few_e5m2(const AttendArgs&, int64_t, int, hipStream_t);
void launch_attend_few_pairs(const AttendArgs&, int64_t, int, hipStream_t);

namespace {

constexpr int kFewRows = 16, kFewLeast = 8, kFewWanted = 1024;

// The rows of sequences that were cut, from their units' sums in the order of the runs, and zeros for rows of no sequence.
// A wave a row.
__global__ __launch_bounds__(256) void k_attend_join(AttendArgs a, int unit_rows, int least, int columns) {
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int lane = threadIdx.x & 63, H = (int)a.a.heads, D = a.c.head_dim;
  if (row >= a.a.T * H) return;
  const int t = (int)(row / H), h = (int)(row - (int64_t)t * H);
  int b;
  if (a.starts) {
    int low = -1, high = (int)a.a.B;                        // the last sequence that starts at t or before
    while (high - low > 1) {
      const int mid = (low + high) >> 1;
      if (a.starts[mid] <= t) low = mid;
      else high = mid;
    }
    b = low;
  } else {
    b = t / (int)(a.a.T / a.a.B);
  }
  const Sequence s = b < 0 ? Sequence{0, 0, 0, 0, 0} : sequence(a, b);
  if (t < s.start || t >= s.start + s.n) {
    for (int d = lane; d < D; d += 64) store_elem(a.out, a.a.dtype, row * D + d, 0.0f);
    if (a.lse && lane == 0) a.lse[row] = -__builtin_inff();
    return;
  }
  if (!a.partial) return;
  const int quota = quota_of(a, unit_rows, least);
  const Cut c = cut(a, s, unit_rows, quota);
  if (c.runs == 1) return;
  int first = 0;
  for (int i = lane; i < b; i += 64) {
    const Cut o = cut(a, sequence(a, i), unit_rows, quota);
    first += o.tiles * o.runs;
  }
  first = wave_sum(first);
  const int head = h / a.group, r = (t - s.start) * a.group + h - head * a.group, tile = r / unit_rows;
  const int64_t stride = (int64_t)a.c.kv_heads * unit_rows * (columns + 2);
  const float* part = a.partial + (((int64_t)(first + tile * c.runs) * a.c.kv_heads + head) * unit_rows + r - tile * unit_rows) * (columns + 2);
  float best = -__builtin_inff(), all = 0.0f;
  for (int i = lane; i < c.runs; i += 64) best = __builtin_fmaxf(best, part[i * stride + columns]);
  for (int o = 32; o; o >>= 1) best = __builtin_fmaxf(best, __shfl_xor(best, o));
  float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int i = 0; i < c.runs; ++i) {
    const float top = part[i * stride + columns], sum = part[i * stride + columns + 1];
    // a run without a maximum has seen no key, or only scores of NaN
    const float factor = top == -__builtin_inff() ? sum : __builtin_amdgcn_exp2f(top - best);
    if (factor == 0.0f) continue;
    all += top == -__builtin_inff() ? sum : factor * sum;
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (lane + 64 * k < D) v[k] += factor * part[i * stride + lane + 64 * k];
  }
  const float inv = all == 0.0f ? 0.0f : 1.0f / all;
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (lane + 64 * k < D) store_elem(a.out, a.a.dtype, row * D + lane + 64 * k, v[k] * inv);
  if (a.lse && lane == 0)
    a.lse[row] = all == 0.0f ? -__builtin_inff() : best == -__builtin_inff() ? all : (best + __builtin_amdgcn_logf(all)) * 0.693147180559945309f;
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

// Units of `rows` rows that a call may have: tiles of rows, and with runs of keys as many as are wanted besides.
struct Plan {
  int64_t units;
  bool split;
};
Plan plan_of(const mxq_cache_spec& c, const mxq_attend_spec& a, bool ragged, int rows, int least, int wanted) {
  const int64_t group = a.heads / c.kv_heads;
  int64_t tiles;
  if (ragged) tiles = a.T * group / rows + (a.B < a.T ? a.B : a.T);
  else tiles = a.B * ceil_div(a.T / a.B * group, rows);
  const int64_t keys = a.table_pages * c.page_size, seen = a.window && a.window < keys ? a.window + (ragged ? a.T : a.T / a.B) : keys;
  const bool split = (keys < seen ? keys : seen) > (int64_t)(least - 1) * kStep;
  // the quota is a float32 sum's, a part of 2^-16 too small at worst
  return Plan{tiles * c.kv_heads + (split ? wanted + wanted / 64 : 0), split};
}
int columns_of(int head_dim) { return head_dim <= 64 ? 64 : head_dim <= 128 ? 128 : 256; }

}  // namespace
}  // namespace mxq

extern "C" int64_t mxq_cache_attend_workspace(const mxq_cache_spec* cache, const mxq_attend_spec* spec, int32_t ragged) {
  using namespace mxq;
  if (check(cache, spec) || spec->T == 0 || spec->B == 0) return 0;
  const Plan p = plan_of(*cache, *spec, ragged, kFewRows, kFewLeast, kFewWanted);
  return p.split ? p.units * kFewRows * (columns_of(cache->head_dim) + 2) * (int64_t)sizeof(float) : 0;
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
  a.wanted = kFewWanted;
  a.aligned = cache->page_size % 16 == 0;
  for (int64_t r : cache->row_stride) a.aligned = a.aligned && r >= 0 && r < 1 << 26;
  a.scale2 = spec->scale * 1.44269504088896341f;
  hipStream_t st = as_stream(stream);
  if (spec->B) {
    const Plan p = plan_of(*cache, *spec, starts != nullptr, kFewRows, kFewLeast, kFewWanted);
    if (p.split && !workspace) return invalid("mxq_cache_attend: NULL workspace");
    if (p.units * 256 > kMaxThreads) return invalid("mxq_cache_attend: too many units for a launch");
    a.partial = p.split ? (float*)workspace : nullptr;
    auto launch = cache->format == MXQ_FMT_E4M3 ? launch_attend_few_e4m3 : cache->format == MXQ_FMT_E5M2 ? launch_attend_few_e5m2 : launch_attend_few_pairs;
    launch(a, p.units, kFewLeast, st);
    if (int rc = check_launch("mxq_cache_attend")) return rc;
  }
  if (a.partial || starts) {
    k_attend_join<<<dim3((unsigned)ceil_div(spec->T * spec->heads, 4)), 256, 0, st>>>(a, kFewRows, kFewLeast, columns);
    return check_launch("mxq_cache_attend");
  }
  return MXQ_OK;
}
