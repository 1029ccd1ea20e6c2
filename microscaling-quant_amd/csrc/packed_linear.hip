// Products with packed MX weights and their epilogue (include/mxq_hip.h, mxq_packed_linear and mxq_expert_linear).
//
//   z[m, n] = sum_k x[m, k] code[n, k] 2^(scale[n, k / 32] - 127);  y = act(z + b) [* (z' + b')] + residual
#include "packed_linear_common.h"

namespace mxq {
namespace {

constexpr int kTile = 64, kStep = 16;

// 64 x 64 outputs a workgroup, 4 x 4 a thread, 16 columns of the contraction at a time through LDS in float32.
template <bool GATED>
__global__ __launch_bounds__(256) void k_linear_any(LinearArgs a) {
  constexpr int W = GATED ? 2 : 1;
  __shared__ float xs[kStep][kTile + 1], ws[W][kStep][kTile + 1];
  const RowTile t = row_tile(a, kTile, blockIdx.y);
  if (t.expert < 0) return;
  const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
  const int64_t n0 = (int64_t)blockIdx.x * kTile;
  const uint8_t* codes = a.codes + t.expert * a.sp.batch_codes;
  const uint8_t* scales = a.scales + t.expert * a.sp.batch_scales;
  float acc[W][4][4] = {};
  if (!t.zeros)
    for (int64_t k0 = 0; k0 < a.K; k0 += kStep) {
      for (int i = tid; i < kTile * kStep; i += 256) {
        const int r = i / kStep, c = i % kStep;
        const int64_t k = k0 + c;
        float v = 0.0f;
        if (r < t.rows && k < a.K) v = load_elem(a.x, a.sp.x_dtype, x_row(a, t.row0 + r) * a.sp.ld_x + k);
        xs[c][r] = v;
        for (int w = 0; w < W; ++w) {
          const int64_t n = n0 + r;
          v = 0.0f;
          if (n < a.N && k < a.K) {
            const int64_t row = n + w * a.N;
            v = code_value(codes + row * a.sp.ld_codes, k, a.sp.format) * scale_value(scales[row * a.sp.ld_scales + k / 32]);
          }
          ws[w][c][r] = v;
        }
      }
      __syncthreads();
      for (int c = 0; c < kStep; ++c)
        for (int i = 0; i < 4; ++i)
          for (int j = 0; j < 4; ++j)
            for (int w = 0; w < W; ++w)
              acc[w][i][j] = __builtin_fmaf(xs[c][ty * 4 + i], ws[w][c][tx * 4 + j], acc[w][i][j]);
      __syncthreads();
    }
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < 4; ++j) {
      const int r = ty * 4 + i;
      const int64_t n = n0 + tx * 4 + j;
      if (r >= t.rows || n >= a.N) continue;
      const float up = GATED ? acc[W - 1][i][j] : 0.0f;
      store_elem(a.y, a.sp.y_dtype, (t.row0 + r) * a.sp.ld_y + n, epilogue(a, t, t.row0 + r, n, acc[0][i][j], up));
    }
}

int check_spec(const std::string& who, int64_t M, int64_t N, int64_t K, const mxq_linear_spec* sp) {
  if (!sp) return invalid(who + ": NULL spec");
  for (int32_t d : {sp->x_dtype, sp->bias_dtype, sp->residual_dtype, sp->y_dtype})
    if (d < MXQ_DT_F32 || d > MXQ_DT_F16) return invalid(who + ": unknown dtype");
  if (sp->format < MXQ_FMT_E4M3 || sp->format > MXQ_FMT_E2M1_PAIRS) return invalid(who + ": unknown format");
  if (sp->activation < MXQ_ACT_NONE || sp->activation > MXQ_ACT_RELU) return invalid(who + ": unknown activation");
  if (M < 0 || N < 0 || K < 0 || M > 0x7fffffff || N > 0x3fffffff || K > 0x7fffffff) return invalid(who + ": size out of range");
  return MXQ_OK;
}

int launch(const char* who, const LinearArgs& a, int64_t tiles, mxq_stream_t stream) {
  if (tiles > 65535 * (int64_t)kTile) return invalid(std::string(who) + ": too many rows");
  const dim3 grid((unsigned)ceil_div(a.N, kTile), (unsigned)tiles);
  KernelTimer timer("k_linear_any", as_stream(stream));
  if (a.sp.gated) k_linear_any<true><<<grid, 256, 0, as_stream(stream)>>>(a);
  else k_linear_any<false><<<grid, 256, 0, as_stream(stream)>>>(a);
  return check_launch(who);
}

}  // namespace
}  // namespace mxq

using namespace mxq;

extern "C" int64_t mxq_packed_linear_workspace(int64_t, int64_t, int64_t, const mxq_linear_spec*) { return 0; }
extern "C" int64_t mxq_expert_linear_workspace(int64_t, int64_t, int64_t, int64_t, const mxq_linear_spec*) { return 0; }

extern "C" int mxq_packed_linear(const void* x, const uint8_t* codes, const uint8_t* scales, const void* bias,
                                 const void* residual, void* y, int64_t M, int64_t N, int64_t K,
                                 const mxq_linear_spec* spec, void* workspace, mxq_stream_t stream) {
  if (int rc = check_spec("mxq_packed_linear", M, N, K, spec)) return rc;
  if (M == 0 || N == 0) return MXQ_OK;
  if (!y || (K && (!x || !codes || !scales))) return invalid("mxq_packed_linear: NULL argument");
  const LinearArgs a{x, codes, scales, bias, residual, y, nullptr, nullptr, M, N, K, 0, *spec};
  return launch("mxq_packed_linear", a, ceil_div(M, kTile), stream);
}

extern "C" int mxq_expert_linear(const void* x, const uint8_t* codes, const uint8_t* scales, const void* bias, void* y,
                                 int64_t n, int64_t N, int64_t K, int64_t E, const int32_t* order, const int32_t* offsets,
                                 const mxq_linear_spec* spec, void* workspace, mxq_stream_t stream) {
  if (int rc = check_spec("mxq_expert_linear", n, N, K, spec)) return rc;
  if (E < 1 || E > 1024) return invalid("mxq_expert_linear: 1 to 1024 experts");
  if (spec->top_k < 0 || spec->top_k > 64) return invalid("mxq_expert_linear: top_k must be 0 to 64");
  if (n == 0 || N == 0) return MXQ_OK;
  if (!y || !offsets || (spec->top_k && !order) || (K && (!x || !codes || !scales)))
    return invalid("mxq_expert_linear: NULL argument");
  const LinearArgs a{x, codes, scales, bias, nullptr, y, order, offsets, n, N, K, (int32_t)E, *spec};
  return launch("mxq_expert_linear", a, n / kTile + (n < E + 1 ? n : E + 1), stream);
}
