// What the kernels of products with packed weights share: arguments, the tiles of rows by expert, codes as values, the
// epilogue.
#pragma once

#include "mxq_common.h"

namespace mxq {

struct LinearArgs {
  const void* x;
  const uint8_t *codes, *scales;
  const void *bias, *residual;
  void* y;
  const int32_t *order, *offsets;   // of the experts' product; NULL offsets: one matrix
  int64_t M, N, K;                  // rows of y, outputs, contraction
  int32_t E;
  mxq_linear_spec sp;
};

__device__ __forceinline__ float load_elem(const void* p, int dtype, int64_t i) {
  if (dtype == MXQ_DT_F32) return ((const float*)p)[i];
  if (dtype == MXQ_DT_BF16) return __uint_as_float((uint32_t)((const uint16_t*)p)[i] << 16);
  return (float)((const _Float16*)p)[i];
}

__device__ __forceinline__ void store_elem(void* p, int dtype, int64_t i, float v) {
  if (dtype == MXQ_DT_F32) ((float*)p)[i] = v;
  else if (dtype == MXQ_DT_BF16) ((__bf16*)p)[i] = (__bf16)v;
  else ((_Float16*)p)[i] = (_Float16)v;
}

// Up to BM rows of one matrix: expert -1 where there is no such tile; `zeros`: the rows of no expert.
struct RowTile {
  int expert, rows;
  int64_t row0;
  bool zeros;
};

// The index-th tile, the experts' tiles one expert after another and the rows of no expert last.  Every wave finds it by
// itself: a lane counts the tiles of (E + 1) / 64 neighbouring experts, a prefix sum over the lanes names the lane, which
// goes through its own.  Offsets are held to [0, M], whatever the caller's array says.
__device__ __forceinline__ RowTile row_tile(const LinearArgs& a, int BM, int index) {
  if (!a.offsets) {
    const int64_t row0 = (int64_t)index * BM, left = a.M - row0;
    return RowTile{0, left < BM ? (int)left : BM, row0, false};
  }
  const int lane = threadIdx.x & 63, M = (int)a.M, per = (a.E + 64) >> 6;
  auto offset = [&](int e) {
    if (e > a.E) return M;
    const int o = a.offsets[e];
    return o < 0 ? 0 : o > M ? M : o;
  };
  auto tiles_of = [&](int e) {
    const int rows = offset(e + 1) - offset(e);
    return rows > 0 ? (rows + BM - 1) / BM : 0;
  };
  int mine = 0;
  for (int i = 0; i < per; ++i) {
    const int e = lane * per + i;
    if (e <= a.E) mine += tiles_of(e);
  }
  int upto = mine;
  for (int o = 1; o < 64; o <<= 1) {
    const int q = __shfl_up(upto, o);
    if (lane >= o) upto += q;
  }
  const uint64_t at = __ballot(index >= upto - mine && index < upto);
  if (!at) return RowTile{-1, 0, 0, false};
  const int owner = __builtin_ctzll(at);
  int e = lane * per, left = index - (upto - mine), row0 = 0, rows = 0;
  if (lane == owner) {
    for (;; ++e) {
      const int k = tiles_of(e);
      if (left < k) break;
      left -= k;
    }
    row0 = offset(e) + left * BM;
    rows = offset(e + 1) - row0;
    if (rows > BM) rows = BM;
  }
  e = __shfl(e, owner), row0 = __shfl(row0, owner), rows = __shfl(rows, owner);
  return RowTile{e == a.E ? 0 : e, rows, row0, e == a.E};
}

// x's row for row r of y.
__device__ __forceinline__ int64_t x_row(const LinearArgs& a, int64_t r) {
  if (!a.offsets || !a.sp.top_k) return r;
  const int slot = a.order[r];
  return (slot < 0 || slot >= a.M ? 0 : slot) / a.sp.top_k;
}

__device__ __forceinline__ float code_value(const uint8_t* row, int64_t k, int format) {
  if (format == MXQ_FMT_E4M3) return __builtin_amdgcn_cvt_f32_fp8(row[k], 0);
  if (format == MXQ_FMT_E5M2) return __builtin_amdgcn_cvt_f32_bf8(row[k], 0);
  const int e = format == MXQ_FMT_E3M2 ? 3 : 2, m = format == MXQ_FMT_E3M2 ? 2 : format == MXQ_FMT_E2M3 ? 3 : 1;
  const int c = format == MXQ_FMT_E2M1_PAIRS ? row[k >> 1] >> (k & 1) * 4 : row[k];
  const int exponent = c >> m & ((1 << e) - 1), fraction = c & ((1 << m) - 1), bias = (1 << (e - 1)) - 1;
  const float v = exponent ? ldexpf((float)(fraction + (1 << m)), exponent - bias - m) : ldexpf((float)fraction, 1 - bias - m);
  return c >> (e + m) & 1 ? -v : v;
}

__device__ __forceinline__ float scale_value(int s) { return s == 255 ? NAN : ldexpf(1.0f, s - 127); }

__device__ __forceinline__ float activate(float z, int activation) {
  switch (activation) {
    case MXQ_ACT_SILU: return z / (1.0f + expf(-z));
    case MXQ_ACT_GELU: return 0.5f * z * (1.0f + erff(z * 0.70710678118654752f));
    case MXQ_ACT_GELU_TANH: {
      const float t = 0.79788456080286536f * (z + 0.044715f * z * z * z);
      return 0.5f * z * (1.0f + tanhf(t));
    }
    case MXQ_ACT_RELU: return z < 0.0f ? 0.0f : z;
    default: return z;
  }
}

// The value stored at (row, n), float32; z, up: the contractions with row n and, gated, with row N + n of the weight.
__device__ __forceinline__ float epilogue(const LinearArgs& a, const RowTile& t, int64_t row, int64_t n, float z, float up) {
  if (t.zeros) return 0.0f;
  if (a.bias) {
    const int64_t first = t.expert * a.sp.batch_bias;
    z += load_elem(a.bias, a.sp.bias_dtype, first + n);
    if (a.sp.gated) up += load_elem(a.bias, a.sp.bias_dtype, first + a.N + n);
  }
  z = activate(z, a.sp.activation);
  if (a.sp.gated) z *= up;
  if (a.residual) z += load_elem(a.residual, a.sp.residual_dtype, row * a.sp.ld_residual + n);
  return z;
}

}  // namespace mxq
