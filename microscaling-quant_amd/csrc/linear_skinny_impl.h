// Products of up to 16 rows (generated tokens, an expert's few) with packed weights: reading the weight is what they cost.
//
// A workgroup owns 16 outputs (gated: 16 rows of either half of the weight) of 16 rows of x; its waves divide the
// contraction, 128 columns at a time each, so that nothing is staged in LDS, no wave waits for another before the end, and
// a row's bytes are read in whole 128-byte lines, the next ones asked for before these are multiplied.  Lane (r, g) of a
// wave holds block g of row r: 32 codes, one scale, four operands of mfma_f32_16x16x32_bf16 (whose order of the contraction
// is free, as long as x's follows).  Weights become bfloat16 exactly; float16 and float32 activations are taken as the sum
// of two and three bfloat16, one product each, also exact but for what a float32 has below 2^-133, bfloat16's smallest step.
// The waves' sums meet in LDS, in the order of the waves; biases and residual are asked for at the start.
//
// Measured, us: 4096 x 4096 in E4M3 with one row 7.5 (2.3 TB/s; a launch and two trips to memory are what is left), 8
// experts of 4096 x 4096 36 (3.8 TB/s).  Eight waves a workgroup, or four where there are workgroups enough to fill the
// card four times: four take 36.3 there, eight 39.0, and for the one row 8.2 and 7.5.
#pragma once

#include "packed_linear_common.h"

namespace mxq {

template <int DT> constexpr int kPlanes = DT == MXQ_DT_BF16 ? 1 : DT == MXQ_DT_F16 ? 2 : 3;

// 32 values of one row of x.
template <int DT> struct XBlock {
  static constexpr int kLoads = DT == MXQ_DT_F32 ? 8 : 4, kEach = DT == MXQ_DT_F32 ? 4 : 8;
  u32x4 v[kLoads];

  __device__ __forceinline__ void load(const void* x, int64_t at) {
    const uint8_t* p = (const uint8_t*)x + at * (DT == MXQ_DT_F32 ? 4 : 2);
#pragma unroll
    for (int i = 0; i < kLoads; ++i) v[i] = *(const u32x4_any*)(p + 16 * i);
  }
  __device__ __forceinline__ void load_first(const void* x, int64_t at, int valid) {
    constexpr int size = DT == MXQ_DT_F32 ? 4 : 2;
    const uint8_t* p = (const uint8_t*)x + at * size;
#pragma unroll
    for (int i = 0; i < kLoads; ++i) v[i] = load_part(p + 16 * i, valid * size - 16 * i);
  }

  // The j-th eight values as kPlanes bfloat16 operands: each plane the leading bits of what the ones before leave.
  __device__ __forceinline__ void planes(int j, bf16x8 (&out)[kPlanes<DT>]) const {
    if constexpr (DT == MXQ_DT_BF16) {
      __builtin_memcpy(&out[0], &v[j], 16);
    } else {
      float f[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if constexpr (DT == MXQ_DT_F32) {
          f[i] = __uint_as_float(v[2 * j + (i >> 2)][i & 3]);
        } else {
          const uint16_t h = (uint16_t)(v[j][i >> 1] >> (i & 1) * 16);
          _Float16 t;
          __builtin_memcpy(&t, &h, 2);
          f[i] = (float)t;
        }
      }
#pragma unroll
      for (int p = 0; p < kPlanes<DT>; ++p) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
          w[i] = __builtin_amdgcn_perm(__float_as_uint(f[2 * i + 1]), __float_as_uint(f[2 * i]), 0x07060302u);
        __builtin_memcpy(&out[p], w, 16);
        if (p + 1 < kPlanes<DT>) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float hi = __uint_as_float(__float_as_uint(f[i]) & 0xFFFF0000u);
            f[i] = f[i] == hi ? 0.0f : f[i] - hi;                      // infinities leave nothing
          }
        }
      }
    }
  }
};

constexpr int kUnit = 128;

template <int FAM, int DT, bool GATED, int WAVES>
__global__ __launch_bounds__(64 * WAVES, 2) void k_linear_skinny(LinearArgs a, CodeMap map) {
  constexpr int P = kPlanes<DT>, BB = kBlockBytes<FAM>, NT = GATED ? 2 : 1, U = GATED ? 1 : 2;
  constexpr int64_t kStride = WAVES * U * kUnit;
  __shared__ f32x4 sums[WAVES][NT][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, g = lane >> 4;
  const int64_t n0 = (int64_t)blockIdx.x * 16;
  const RowTile t = row_tile(a, 16, blockIdx.y);
  if (t.expert < 0) return;

  // the output that this thread finishes
  const int n_out = threadIdx.x & 15, m_out = threadIdx.x >> 4;
  const bool mine = m_out < t.rows && n0 + n_out < a.N;
  float bias = 0.0f, bias_up = 0.0f, residual = 0.0f;
  if (mine && !t.zeros) {
    const int64_t first = t.expert * a.sp.batch_bias + n0 + n_out;
    if (a.bias) bias = load_elem(a.bias, a.sp.bias_dtype, first);
    if (a.bias && GATED) bias_up = load_elem(a.bias, a.sp.bias_dtype, first + a.N);
    if (a.residual) residual = load_elem(a.residual, a.sp.residual_dtype, (t.row0 + m_out) * a.sp.ld_residual + n0 + n_out);
  }

  f32x4 acc[NT];
#pragma unroll
  for (int i = 0; i < NT; ++i) acc[i] = f32x4{0, 0, 0, 0};

  if (!t.zeros) {
    const uint8_t *wp[NT], *sp[NT];
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      int64_t n = n0 + r < a.N ? n0 + r : a.N - 1;                     // a row that exists; its sums are not stored
      if (i) n += a.N;
      wp[i] = a.codes + t.expert * a.sp.batch_codes + n * a.sp.ld_codes + g * BB;
      sp[i] = a.scales + t.expert * a.sp.batch_scales + n * a.sp.ld_scales + g;
    }
    const int64_t xp = x_row(a, t.row0 + (r < t.rows ? r : t.rows - 1)) * a.sp.ld_x + g * 32;
    uint32_t w[2][U][NT][kWords<FAM>], s[2][U][NT];
    XBlock<DT> x[U];

    auto load_w = [&](int64_t k, uint32_t (&w)[U][NT][kWords<FAM>], uint32_t (&s)[U][NT]) {
      if (k + U * kUnit <= a.K) {
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int i = 0; i < NT; ++i) {
            const int64_t at = (k + u * kUnit) / 32 * BB;
#pragma unroll
            for (int c = 0; c < kWords<FAM> / 4; ++c) {
              const u32x4 v = *(const u32x4_any*)(wp[i] + at + 16 * c);
              __builtin_memcpy(&w[u][i][4 * c], &v, 16);
            }
            s[u][i] = sp[i][(k + u * kUnit) / 32];
          }
        return;
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int i = 0; i < NT; ++i) {
          const int64_t first = k + u * kUnit, left = a.K - (first + g * 32);
          const int valid = left < 0 ? 0 : left < 32 ? (int)left : 32;
          const int bytes = FAM == kPairs ? (valid + 1) / 2 : valid;
#pragma unroll
          for (int c = 0; c < kWords<FAM> / 4; ++c) {
            u32x4 v = load_part(wp[i] + first / 32 * BB + 16 * c, bytes - 16 * c);
            if (FAM == kPairs && (valid & 1)) clear_odd(v, valid);
            __builtin_memcpy(&w[u][i][4 * c], &v, 16);
          }
          s[u][i] = valid ? sp[i][first / 32] : 127;
        }
    };
    auto load_x = [&](int64_t k) {
      if (k + U * kUnit <= a.K) {
#pragma unroll
        for (int u = 0; u < U; ++u) x[u].load(a.x, xp + k + u * kUnit);
        return;
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int64_t left = a.K - (k + u * kUnit + g * 32);
        x[u].load_first(a.x, xp + k + u * kUnit, left < 0 ? 0 : left < 32 ? (int)left : 32);
      }
    };
    auto multiply = [&](const uint32_t (&w)[U][NT][kWords<FAM>], const uint32_t (&s)[U][NT]) {
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int i = 0; i < NT; ++i) {
          uint32_t left;
          const float scale = scale_of<FAM>(s[u][i], w[u][i], map, left, P > 1);
          const bool seldom = (FAM == kMapped || P > 1) && __builtin_expect(__any(left), 0);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            bf16x8 wv = eight<FAM>(w[u][i], scale, j, map), xv[P];
            if (FAM == kMapped && seldom) apply_left(wv, left);
            x[u].planes(j, xv);
            acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wv, xv[0], acc[i], 0, 0, 0);
            if constexpr (P > 1) {
              if (seldom) finite_only(wv);
#pragma unroll
              for (int p = 1; p < P; ++p) acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wv, xv[p], acc[i], 0, 0, 0);
            }
          }
        }
    };

    int64_t k = (int64_t)wave * U * kUnit;
    if (k < a.K) load_w(k, w[0], s[0]);
    for (; k < a.K; k += 2 * kStride) {
      load_x(k);
      if (k + kStride < a.K) load_w(k + kStride, w[1], s[1]);
      multiply(w[0], s[0]);
      if (k + kStride >= a.K) break;
      load_x(k + kStride);
      if (k + 2 * kStride < a.K) load_w(k + 2 * kStride, w[0], s[0]);
      multiply(w[1], s[1]);
    }
  }

#pragma unroll
  for (int i = 0; i < NT; ++i) sums[wave][i][lane] = acc[i];
  __syncthreads();
  if (!mine) return;
  // element (row m, weight row n) of a tile's sums: lane m + 16 (n / 4), component n % 4
  float z[NT];
#pragma unroll
  for (int i = 0; i < NT; ++i) {
    z[i] = 0.0f;
#pragma unroll
    for (int v = 0; v < WAVES; ++v) z[i] += ((const float*)&sums[v][i][m_out + 16 * (n_out >> 2)])[n_out & 3];
  }
  float y = activate(z[0] + bias, a.sp.activation);
  if (GATED) y *= z[NT - 1] + bias_up;
  if (a.residual) y += residual;
  if (t.zeros) y = 0.0f;
  store_elem(a.y, a.sp.y_dtype, (t.row0 + m_out) * a.sp.ld_y + n0 + n_out, y);
}

template <int FAM, int DT> void launch_skinny_dt(const LinearArgs& a, int64_t tiles, hipStream_t st) {
  const CodeMap map = code_map(a.sp.format);
  const dim3 grid((unsigned)ceil_div(a.N, 16), (unsigned)tiles);
  KernelTimer timer("k_linear_skinny", st);
  if ((int64_t)grid.x * grid.y >= 1024) {
    if (a.sp.gated) k_linear_skinny<FAM, DT, true, 4><<<grid, 256, 0, st>>>(a, map);
    else k_linear_skinny<FAM, DT, false, 4><<<grid, 256, 0, st>>>(a, map);
  } else {
    if (a.sp.gated) k_linear_skinny<FAM, DT, true, 8><<<grid, 512, 0, st>>>(a, map);
    else k_linear_skinny<FAM, DT, false, 8><<<grid, 512, 0, st>>>(a, map);
  }
}

template <int FAM> void launch_skinny_family(const LinearArgs& a, int64_t tiles, hipStream_t st) {
  if (a.sp.x_dtype == MXQ_DT_BF16) launch_skinny_dt<FAM, MXQ_DT_BF16>(a, tiles, st);
  else if (a.sp.x_dtype == MXQ_DT_F16) launch_skinny_dt<FAM, MXQ_DT_F16>(a, tiles, st);
  else launch_skinny_dt<FAM, MXQ_DT_F32>(a, tiles, st);
}

}  // namespace mxq
