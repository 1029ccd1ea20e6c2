// Products with packed MX weights and their epilogue (include/mxq_hip.h, mxq_packed_linear and mxq_expert_linear): which
// kernel takes a call, and what runs before and after it.
//
//   z[m, n] = sum_k x[m, k] code[n, k] 2^(scale[n, k / 32] - 127);  y = act(z + b) [* (z' + b')] + residual
#include "packed_linear_common.h"

namespace mxq {

void launch_skinny_e4m3(const LinearArgs&, int64_t, hipStream_t);
void launch_skinny_e5m2(const LinearArgs&, int64_t, hipStream_t);
void launch_skinny_mapped(const LinearArgs&, int64_t, hipStream_t);
void launch_skinny_pairs(const LinearArgs&, int64_t, hipStream_t);
void launch_tile_e4m3(const TileArgs&, const TilePlan&, hipStream_t);
void launch_tile_e5m2(const TileArgs&, const TilePlan&, hipStream_t);
void launch_tile_mapped(const TileArgs&, const TilePlan&, hipStream_t);
void launch_tile_pairs(const TileArgs&, const TilePlan&, hipStream_t);

namespace {

// What k_linear_tile's direct loads cannot take as it lies is laid out first, by one launch.
//   x: bfloat16 planes of kp values, one after another along a row, zeros past K: each plane the leading bits of what the
//      ones before leave, so that their sum is the value (of a float32, down to bfloat16's smallest step of 2^-133).
//   codes: rows of whole 128 columns, zeros past K.
//   scales: rows of whole words.
// Experts without rows are left out.
struct PrepareArgs {
  LinearArgs l;
  int64_t kp, x_rows, w_rows, first;   // columns a plane, rows of x (0: stays), rows of one weight, this launch's first row
  int32_t planes;
  uint16_t* x;
  uint8_t *codes, *scales;             // NULL: stay
};
// A workgroup a row of x, then a row of the weight.
__global__ __launch_bounds__(256) void k_prepare(PrepareArgs p) {
  const LinearArgs& a = p.l;
  int64_t row = p.first + blockIdx.x;
  const bool pairs = a.sp.format == MXQ_FMT_E2M1_PAIRS;
  if (row < p.x_rows) {
    for (int64_t k = threadIdx.x * 8; k < p.kp; k += 256 * 8) {
      float v[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = 0.0f;
      if (k + 8 <= a.K) {
        add_eight(v, a.x, a.sp.x_dtype, row * a.sp.ld_x + k);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (k + e < a.K) v[e] = load_elem(a.x, a.sp.x_dtype, row * a.sp.ld_x + k + e);
      }
      for (int q = 0; q < p.planes; ++q) {
        u32x4 w;
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = __builtin_amdgcn_perm(__float_as_uint(v[2 * e + 1]), __float_as_uint(v[2 * e]), 0x07060302u);
        *(u32x4*)(p.x + (row * p.planes + q) * p.kp + k) = w;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float hi = __uint_as_float(__float_as_uint(v[e]) & 0xFFFF0000u);
          v[e] = v[e] == hi ? 0.0f : v[e] - hi;                          // infinities leave nothing
        }
      }
    }
    return;
  }
  const int64_t all = row - p.x_rows, e = all / p.w_rows;
  row = all - e * p.w_rows;
  if (a.offsets && a.offsets[e + 1] <= a.offsets[e]) return;
  const int64_t bytes = pairs ? p.kp / 2 : p.kp, have = pairs ? (a.K + 1) / 2 : a.K;
  const uint8_t* codes = a.codes + e * a.sp.batch_codes + row * a.sp.ld_codes;
  if (p.codes)
    for (int64_t at = threadIdx.x * 16; at < bytes; at += 256 * 16) {
      const int64_t left = have - at;
      u32x4 v;
      if (left >= 16) v = *(const u32x4_any*)(codes + at);
      else v = load_part(codes + at, left < 0 ? 0 : (int)left);
      if (pairs && (a.K & 1) && left > 0 && left <= 16) clear_odd(v, (int)left * 2 - 1);
      *(u32x4*)(p.codes + all * bytes + at) = v;
    }
  const uint8_t* scales = a.scales + e * a.sp.batch_scales + row * a.sp.ld_scales;
  if (p.scales)
    for (int64_t at = threadIdx.x * 4; at < p.kp / 32; at += 256 * 4) {
      uint32_t v = 0;
#pragma unroll
      for (int b = 0; b < 4; ++b)
        if (at + b < (a.K + 31) / 32) v |= (uint32_t)scales[at + b] << 8 * b;
      *(uint32_t*)(p.scales + all * (p.kp / 32) + at) = v;
    }
}

// The splits' sums in their order, and the epilogue: eight outputs a thread.
__global__ __launch_bounds__(256) void k_linear_finish(LinearArgs a, const float* partial, int split) {
  const int64_t row = blockIdx.x, width = a.sp.gated ? 2 * a.N : a.N;
  for (int64_t n = ((int64_t)blockIdx.y * 256 + threadIdx.x) * 8; n < a.N; n += (int64_t)gridDim.y * 256 * 8) {
    const RowTile t{0, 0, 0, false};
    const float* p = partial + row * width + n;
    if (n + 8 > a.N) {
      for (int64_t e = n; e < a.N; ++e, ++p) {
        float z = 0.0f, up = 0.0f;
        for (int s = 0; s < split; ++s) {
          z += p[s * a.M * width];
          if (a.sp.gated) up += p[s * a.M * width + a.N];
        }
        store_elem(a.y, a.sp.y_dtype, row * a.sp.ld_y + e, epilogue(a, t, row, e, z, up));
      }
      continue;
    }
    float z[8], up[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) z[e] = up[e] = 0.0f;
    for (int s = 0; s < split; ++s, p += a.M * width) {
      add_eight(z, p, MXQ_DT_F32, 0);
      if (a.sp.gated) add_eight(up, p + a.N, MXQ_DT_F32, 0);
    }
    Eight residual = {};
    if (a.residual) residual = load_eight(a.residual, a.sp.residual_dtype, row * a.sp.ld_residual + n);
    finish_eight(a, t, row, n, z, up, load_bias(a, t, n), residual);
  }
}

int check_spec(const std::string& who, int64_t M, int64_t N, int64_t K, const mxq_linear_spec* sp) {
  if (!sp) return invalid(who + ": NULL spec");
  for (int32_t d : {sp->x_dtype, sp->bias_dtype, sp->residual_dtype, sp->y_dtype})
    if (d < MXQ_DT_F32 || d > MXQ_DT_F16) return invalid(who + ": unknown dtype");
  if (sp->format < MXQ_FMT_E4M3 || sp->format > MXQ_FMT_E2M1_PAIRS) return invalid(who + ": unknown format");
  if (sp->activation < MXQ_ACT_NONE || sp->activation > MXQ_ACT_RELU) return invalid(who + ": unknown activation");
  if (sp->top_k < 0 || sp->top_k > 64) return invalid(who + ": top_k must be 0 to 64");
  if (M < 0 || N < 0 || K < 0 || M > 0x7fffffff || N > 0x3fffffff || K > 0x7fffff00) return invalid(who + ": size out of range");
  return MXQ_OK;
}

int family(int format) {
  return format == MXQ_FMT_E4M3 ? kE4M3 : format == MXQ_FMT_E5M2 ? kE5M2 : format == MXQ_FMT_E2M1_PAIRS ? kPairs : kMapped;
}

struct Plan {
  bool few;                    // k_linear_skinny, 16 rows a workgroup; k_linear_tile otherwise
  TilePlan tile;
  int64_t tiles_m, tiles_n;    // of either
  int steps, planes;
  bool lay_x, lay_codes, lay_scales;                  // what goes through k_prepare
  int64_t x_rows, w_rows;
  int64_t at_codes, at_scales, at_partial, bytes;     // workspace: x, codes, scales, partial sums
};

constexpr int kTileM[4] = {256, 128, 64, 64}, kTileN[4] = {256, 128, 128, 128};

// a.E = 0: one matrix.
Plan plan_of(const LinearArgs& a) {
  const mxq_linear_spec& sp = a.sp;
  const int64_t M = a.M, N = a.N, K = a.K, E = a.E;
  Plan p{};
  const int64_t each = E ? ceil_div(M, E) : M, width = sp.gated ? 2 * N : N;
  auto row_tiles = [&](int64_t bm) { return E ? M / bm + (M < E + 1 ? M : E + 1) : ceil_div(M, bm); };
  const bool pairs = sp.format == MXQ_FMT_E2M1_PAIRS;
  p.lay_codes = K % (pairs ? 32 : 16) || (uintptr_t)a.codes % 16 || sp.ld_codes % 16 || sp.batch_codes % 16;
  p.lay_scales = K % 128 || (uintptr_t)a.scales % 4 || sp.ld_scales % 4 || sp.batch_scales % 4;
  // by the sizes alone: strides and addresses do not change a result's bits
  if (each <= 16) {
    p.few = true;
    p.tiles_m = row_tiles(16);
    return p;
  }
  p.steps = (int)(2 * ceil_div(K, 128));
  p.planes = sp.x_dtype == MXQ_DT_BF16 ? 1 : sp.x_dtype == MXQ_DT_F16 ? 2 : 3;
  auto tiles = [&](int s) { return ceil_div(each, kTileM[s]) * (E ? E : 1) * ceil_div(width, kTileN[s]); };
  // By rows alone, measured with one weight of 4096 columns and 8192 rows, us on 256 x 256, 128 x 128, 64 x 128: 200 rows 39, 32, 31; 500
  // rows 54, 49, 46; 1000 rows 80, 72, 90; 2000 rows 114, 138, 166; 512 rows an expert 228, 206, 212, 1024 346, 351, 377.
  p.tile.shape = tiles(0) >= 192 && each > 1000 ? 0 : each > 500 ? 1 : 2;
  p.tiles_m = row_tiles(kTileM[p.tile.shape]);
  p.tiles_n = ceil_div(width, kTileN[p.tile.shape]);
  p.tile.split = 1;
  if (!E) {
    const int64_t have = p.tiles_m * p.tiles_n, all = (int64_t)p.steps * p.planes;
    while (p.tile.split < 8 && have * p.tile.split * 2 <= (p.tile.shape == 0 ? 256 : 512) && all / (p.tile.split * 2) >= 8) p.tile.split *= 2;
  }
  p.lay_x = sp.x_dtype != MXQ_DT_BF16 || K % 8 || sp.ld_x % 8 || (uintptr_t)a.x % 16;
  p.x_rows = E && sp.top_k ? ceil_div(M, sp.top_k) : M;
  p.w_rows = width;
  auto whole = [](int64_t bytes) { return ceil_div(bytes, 256) * 256; };
  const int64_t kp = (int64_t)p.steps * 64, matrices = (E ? E : 1) * width;
  // a tile's rows from its first one (x's of experts: from the first of all)
  const int64_t x_row = 2 * (p.lay_x ? kp * p.planes : sp.ld_x), w_row = p.lay_codes ? (pairs ? kp / 2 : kp) : sp.ld_codes;
  const int64_t s_row = p.lay_scales ? kp / 32 : sp.ld_scales, apart = sp.gated ? N + 256 : 256;
  const int64_t far = 0xFFFF0000;
  if (x_row > far / (E && sp.top_k ? p.x_rows : 256) || w_row > far / apart || s_row > far / apart) {
    p.tile.shape = 3;                                                    // the same sums: a split and its order are the others'
    p.tiles_m = row_tiles(kTileM[3]);
    p.tiles_n = ceil_div(width, kTileN[3]);
  }
  p.at_codes = p.lay_x ? whole(p.x_rows * p.planes * kp * 2) : 0;
  p.at_scales = p.at_codes + (p.lay_codes ? whole(matrices * (pairs ? kp / 2 : kp)) : 0);
  p.at_partial = p.at_scales + (p.lay_scales ? whole(matrices * (kp / 32)) : 0);
  p.bytes = p.at_partial + (p.tile.split > 1 ? p.tile.split * M * width * 4 : 0);
  return p;
}

int launch(const char* who, const LinearArgs& a, void* workspace, hipStream_t st) {
  const Plan p = plan_of(a);
  if (p.bytes && !workspace) return invalid(std::string(who) + ": NULL workspace");
  const int fam = family(a.sp.format);
  const int64_t threads = p.few ? (ceil_div(a.N, 16) * p.tiles_m >= 1024 ? 256 : 512) * ceil_div(a.N, 16)
                                : (p.tile.shape == 0 ? 512 : 256) * p.tiles_m * p.tiles_n;
  if (threads > kMaxThreads) return invalid(std::string(who) + ": too many outputs");
  if (p.few) {
    (fam == kE4M3 ? launch_skinny_e4m3 : fam == kE5M2 ? launch_skinny_e5m2 : fam == kPairs ? launch_skinny_pairs : launch_skinny_mapped)(
        a, p.tiles_m, st);
    return check_launch(who);
  }
  uint8_t* work = (uint8_t*)workspace;
  const bool pairs = fam == kPairs;
  const int64_t kp = (int64_t)p.steps * 64, matrices = (a.E ? a.E : 1) * p.w_rows;
  TileArgs t{a, (const uint16_t*)a.x, a.sp.ld_x, p.steps, p.planes, (int32_t)a.K, (int32_t)a.K, (int32_t)p.tiles_m, (int32_t)p.tiles_n,
             p.tile.split, (float*)(work + p.at_partial), code_map(a.sp.format)};
  if (kp && (p.lay_x || p.lay_codes || p.lay_scales)) {
    const int64_t x_rows = p.lay_x ? p.x_rows : 0, w_rows = p.lay_codes || p.lay_scales ? matrices : 0;
    PrepareArgs q{a, kp, x_rows, p.w_rows, 0, p.planes, (uint16_t*)work, p.lay_codes ? work + p.at_codes : nullptr,
                        p.lay_scales ? work + p.at_scales : nullptr};
    for (; q.first < x_rows + w_rows; q.first += kMaxBlocks) {
      KernelTimer timer("k_prepare", st);
      k_prepare<<<dim3(blocks_for(x_rows + w_rows - q.first)), 256, 0, st>>>(q);
    }
    if (p.lay_x) t.x = q.x, t.ld_x = kp * p.planes, t.x_columns = (int32_t)kp;
    if (p.lay_codes) {
      t.l.codes = q.codes, t.l.sp.ld_codes = pairs ? kp / 2 : kp, t.l.sp.batch_codes = t.l.sp.ld_codes * p.w_rows;
      t.w_columns = (int32_t)kp;
    }
    if (p.lay_scales) t.l.scales = q.scales, t.l.sp.ld_scales = kp / 32, t.l.sp.batch_scales = kp / 32 * p.w_rows;
  }
  (fam == kE4M3 ? launch_tile_e4m3 : fam == kE5M2 ? launch_tile_e5m2 : fam == kPairs ? launch_tile_pairs : launch_tile_mapped)(t, p.tile, st);
  if (p.tile.split > 1) {
    KernelTimer timer("k_linear_finish", st);
    const int64_t blocks = ceil_div(a.N, 256 * 8);
    k_linear_finish<<<dim3((unsigned)a.M, (unsigned)(blocks < 65535 ? blocks : 65535)), 256, 0, st>>>(a, t.partial, p.tile.split);
  }
  return check_launch(who);
}

}  // namespace
}  // namespace mxq

using namespace mxq;

extern "C" int64_t mxq_packed_linear_workspace(const void* x, const uint8_t* codes, const uint8_t* scales, int64_t M, int64_t N,
                                               int64_t K, const mxq_linear_spec* spec) {
  if (check_spec("mxq_packed_linear_workspace", M, N, K, spec) || !M || !N) return 0;
  return plan_of(LinearArgs{x, codes, scales, nullptr, nullptr, nullptr, nullptr, nullptr, M, N, K, 0, *spec}).bytes;
}
extern "C" int64_t mxq_expert_linear_workspace(const void* x, const uint8_t* codes, const uint8_t* scales, int64_t n, int64_t N,
                                               int64_t K, int64_t E, const mxq_linear_spec* spec) {
  if (check_spec("mxq_expert_linear_workspace", n, N, K, spec) || !n || !N || E < 1 || E > 1024) return 0;
  return plan_of(LinearArgs{x, codes, scales, nullptr, nullptr, nullptr, nullptr, nullptr, n, N, K, (int32_t)E, *spec}).bytes;
}

extern "C" int mxq_packed_linear(const void* x, const uint8_t* codes, const uint8_t* scales, const void* bias,
                                 const void* residual, void* y, int64_t M, int64_t N, int64_t K,
                                 const mxq_linear_spec* spec, void* workspace, mxq_stream_t stream) {
  if (int rc = check_spec("mxq_packed_linear", M, N, K, spec)) return rc;
  if (M == 0 || N == 0) return MXQ_OK;
  if (!y || (K && (!x || !codes || !scales))) return invalid("mxq_packed_linear: NULL argument");
  const LinearArgs a{x, codes, scales, bias, residual, y, nullptr, nullptr, M, N, K, 0, *spec};
  return launch("mxq_packed_linear", a, workspace, as_stream(stream));
}

extern "C" int mxq_expert_linear(const void* x, const uint8_t* codes, const uint8_t* scales, const void* bias, void* y,
                                 int64_t n, int64_t N, int64_t K, int64_t E, const int32_t* order, const int32_t* offsets,
                                 const mxq_linear_spec* spec, void* workspace, mxq_stream_t stream) {
  if (int rc = check_spec("mxq_expert_linear", n, N, K, spec)) return rc;
  if (E < 1 || E > 1024) return invalid("mxq_expert_linear: 1 to 1024 experts");
  if (n == 0 || N == 0) return MXQ_OK;
  if (!y || !offsets || (spec->top_k && !order) || (K && (!x || !codes || !scales)))
    return invalid("mxq_expert_linear: NULL argument");
  const LinearArgs a{x, codes, scales, bias, nullptr, y, order, offsets, n, N, K, (int32_t)E, *spec};
  return launch("mxq_expert_linear", a, workspace, as_stream(stream));
}
