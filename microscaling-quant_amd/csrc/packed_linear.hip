// Products with packed MX weights and their epilogue (include/mxq_hip.h, mxq_packed_linear and mxq_expert_linear): which
// kernel takes a call, and what runs before and after it.
//
//   z[m, n] = sum_k x[m, k] code[n, k] 2^(scale[n, k / 32] - 127);  y = act(z + b) [* (z' + b')] + residual
#include "packed_linear_common.h"

namespace mxq {

void launch_skinny_e4m3(const LinearArgs&, int, int64_t, hipStream_t);
void launch_skinny_e5m2(const LinearArgs&, int, int64_t, hipStream_t);
void launch_skinny_mapped(const LinearArgs&, int, int64_t, hipStream_t);
void launch_skinny_pairs(const LinearArgs&, int, int64_t, hipStream_t);
void launch_tile_e4m3(const TileArgs&, const TilePlan&, hipStream_t);
void launch_tile_e5m2(const TileArgs&, const TilePlan&, hipStream_t);
void launch_tile_mapped(const TileArgs&, const TilePlan&, hipStream_t);
void launch_tile_pairs(const TileArgs&, const TilePlan&, hipStream_t);

namespace {

// x's rows as bfloat16 planes of kp = 64 steps values, one after another along a row, zeros past K: each plane the leading
// bits of what the ones before leave, so that their sum is the value.
__global__ __launch_bounds__(256) void k_planes(const void* x, int dtype, int64_t ld, int64_t rows, int64_t K, int64_t kp, int planes,
                                                uint16_t* out) {
  const int64_t groups = kp / 8;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < rows * groups; i += (int64_t)gridDim.x * 256) {
    const int64_t row = i / groups, k = i % groups * 8;
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = 0.0f;
    if (k + 8 <= K) {
      add_eight(v, x, dtype, row * ld + k);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (k + e < K) v[e] = load_elem(x, dtype, row * ld + k + e);
    }
    for (int p = 0; p < planes; ++p) {
      u32x4 w;
#pragma unroll
      for (int e = 0; e < 4; ++e) w[e] = __builtin_amdgcn_perm(__float_as_uint(v[2 * e + 1]), __float_as_uint(v[2 * e]), 0x07060302u);
      *(u32x4*)(out + (row * planes + p) * kp + k) = w;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float hi = __uint_as_float(__float_as_uint(v[e]) & 0xFFFF0000u);
        v[e] = v[e] == hi ? 0.0f : v[e] - hi;                            // infinities leave nothing
      }
    }
  }
}

// The splits' sums in their order, and the epilogue: eight outputs a thread.
__global__ __launch_bounds__(256) void k_linear_finish(LinearArgs a, const float* partial, int split) {
  const int64_t groups = (a.N + 7) / 8, width = a.sp.gated ? 2 * a.N : a.N;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < a.M * groups; i += (int64_t)gridDim.x * 256) {
    const int64_t row = i / groups, n = i % groups * 8;
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
    finish_eight(a, t, row, n, z, up, residual);
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
  int mt;                      // rows of a k_linear_skinny workgroup / 16, or 0: k_linear_tile
  TilePlan tile;
  int64_t tiles_m, tiles_n;    // of either
  int steps, planes;
  bool convert;                // x goes through k_planes
  int64_t plane_bytes, bytes;  // workspace: the planes, everything
};

constexpr int kTileM[3] = {256, 128, 64}, kTileN[3] = {256, 128, 128};

// E = 0: one matrix.
Plan plan_of(const void* x, int64_t M, int64_t N, int64_t K, int64_t E, const mxq_linear_spec& sp) {
  Plan p{};
  const int64_t each = E ? ceil_div(M, E) : M, width = sp.gated ? 2 * N : N;
  auto row_tiles = [&](int64_t bm) { return E ? M / bm + (M < E + 1 ? M : E + 1) : ceil_div(M, bm); };
  if (each <= 64) {
    const int most = sp.x_dtype == MXQ_DT_F32 ? 2 : 4;
    p.mt = each <= 16 ? 1 : each <= 32 || most == 2 ? 2 : 4;
    p.tiles_m = row_tiles(16 * p.mt);
    return p;
  }
  p.steps = (int)ceil_div(K, 64);
  p.planes = sp.x_dtype == MXQ_DT_BF16 ? 1 : sp.x_dtype == MXQ_DT_F16 ? 2 : 3;
  auto tiles = [&](int s) { return ceil_div(each, kTileM[s]) * (E ? E : 1) * ceil_div(width, kTileN[s]); };
  p.tile.shape = tiles(0) >= 192 && each > 128 ? 0 : tiles(1) >= 128 && each > 64 ? 1 : 2;
  p.tiles_m = row_tiles(kTileM[p.tile.shape]);
  p.tiles_n = ceil_div(width, kTileN[p.tile.shape]);
  p.tile.split = 1;
  if (!E) {
    const int64_t have = p.tiles_m * p.tiles_n, all = (int64_t)p.steps * p.planes;
    while (p.tile.split < 8 && have * p.tile.split * 2 <= 512 && all / (p.tile.split * 2) >= 8) p.tile.split *= 2;
  }
  p.convert = sp.x_dtype != MXQ_DT_BF16 || K % 64 || sp.ld_x % 8 || (uintptr_t)x % 16;
  const int64_t rows = E && sp.top_k ? ceil_div(M, sp.top_k) : M;
  if (p.convert) p.plane_bytes = ceil_div(rows * p.planes * p.steps * 128, 256) * 256;
  p.bytes = p.plane_bytes + (p.tile.split > 1 ? p.tile.split * M * width * 4 : 0);
  return p;
}

int launch(const char* who, const LinearArgs& a, void* workspace, hipStream_t st) {
  const Plan p = plan_of(a.x, a.M, a.N, a.K, a.E, a.sp);
  if (p.bytes && !workspace) return invalid(std::string(who) + ": NULL workspace");
  const int fam = family(a.sp.format);
  if (p.mt) {
    (fam == kE4M3 ? launch_skinny_e4m3 : fam == kE5M2 ? launch_skinny_e5m2 : fam == kPairs ? launch_skinny_pairs : launch_skinny_mapped)(
        a, p.mt, p.tiles_m, st);
    return check_launch(who);
  }
  if (p.tiles_m * p.tiles_n > 0x7fffffff) return invalid(std::string(who) + ": too many outputs");
  TileArgs t{a, (const uint16_t*)a.x, a.sp.ld_x, p.steps, p.planes, (int32_t)p.tiles_m, (int32_t)p.tiles_n, p.tile.split,
             (float*)((uint8_t*)workspace + p.plane_bytes), code_map(a.sp.format)};
  if (p.convert) {
    const int64_t kp = (int64_t)p.steps * 64, rows = a.E && a.sp.top_k ? ceil_div(a.M, a.sp.top_k) : a.M;
    if (kp) {
      KernelTimer timer("k_planes", st);
      const int64_t blocks = ceil_div(rows * kp / 8, 256);
      k_planes<<<dim3((unsigned)(blocks < 16384 ? blocks : 16384)), 256, 0, st>>>(a.x, a.sp.x_dtype, a.sp.ld_x, rows, a.K, kp, p.planes,
                                                                               (uint16_t*)workspace);
    }
    t.x = (const uint16_t*)workspace;
    t.ld_x = kp * p.planes;
  }
  TilePlan tp = p.tile;
  tp.direct = a.K % 128 == 0 && (uintptr_t)a.codes % 16 == 0 && a.sp.ld_codes % 16 == 0 && a.sp.batch_codes % 16 == 0 &&
              (uintptr_t)a.scales % 4 == 0 && a.sp.ld_scales % 4 == 0 && a.sp.batch_scales % 4 == 0;
  (fam == kE4M3 ? launch_tile_e4m3 : fam == kE5M2 ? launch_tile_e5m2 : fam == kPairs ? launch_tile_pairs : launch_tile_mapped)(t, tp, st);
  if (tp.split > 1) {
    KernelTimer timer("k_linear_finish", st);
    const int64_t blocks = ceil_div(a.M * ceil_div(a.N, 8), 256);
    k_linear_finish<<<dim3((unsigned)(blocks < 65536 ? blocks : 65536)), 256, 0, st>>>(a, t.partial, tp.split);
  }
  return check_launch(who);
}

}  // namespace
}  // namespace mxq

using namespace mxq;

extern "C" int64_t mxq_packed_linear_workspace(const void* x, int64_t M, int64_t N, int64_t K, const mxq_linear_spec* spec) {
  return check_spec("mxq_packed_linear_workspace", M, N, K, spec) || !M || !N ? 0 : plan_of(x, M, N, K, 0, *spec).bytes;
}
extern "C" int64_t mxq_expert_linear_workspace(const void* x, int64_t n, int64_t N, int64_t K, int64_t E, const mxq_linear_spec* spec) {
  return check_spec("mxq_expert_linear_workspace", n, N, K, spec) || !n || !N || E < 1 || E > 1024 ? 0 : plan_of(x, n, N, K, E, *spec).bytes;
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
