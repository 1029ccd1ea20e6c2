// Products of few rows (a batch of generated tokens, an expert's few) with packed weights: reading the weight is what
// they cost.
//
// A workgroup owns 16 NT rows of the weight and 16 MT rows of x; its eight waves divide the contraction, 128 columns at a
// time each, so that nothing is staged in LDS, no wave waits for another before the end, and a row's bytes are read in
// whole 128-byte lines.  Lane (r, g) of a wave holds block g of row r: 32 codes, one scale, four operands of
// mfma_f32_16x16x32_bf16 (whose order of the contraction is free, as long as x's follows).  Weights become bfloat16 exactly;
// float16 and float32 activations are taken as the sum of two and three bfloat16, also exact, one product each.
// The waves' sums meet in LDS, in the order of the waves.
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

constexpr int kSkinnyWaves = 8, kUnit = 128;

template <int FAM, int DT, int MT, int NT, int U>
__global__ __launch_bounds__(64 * kSkinnyWaves, 2) void k_linear_skinny(LinearArgs a, CodeMap map) {
  constexpr int P = kPlanes<DT>, BB = kBlockBytes<FAM>;
  __shared__ f32x4 sums[kSkinnyWaves][NT * MT][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, g = lane >> 4;
  const bool gated = a.sp.gated;
  const int outputs = gated ? NT * 8 : NT * 16;                        // a workgroup's
  const int64_t n0 = (int64_t)blockIdx.x * outputs;
  const RowTile t = row_tile(a, MT * 16, blockIdx.y);
  if (t.expert < 0) return;

  f32x4 acc[NT][MT];
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int m = 0; m < MT; ++m) acc[i][m] = f32x4{0, 0, 0, 0};

  if (!t.zeros) {
    const uint8_t *wp[NT], *sp[NT];
    int64_t xp[MT];
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      const bool up = gated && i >= NT / 2;
      int64_t n = n0 + 16 * (up ? i - NT / 2 : i) + r;
      if (n >= a.N) n = a.N - 1;                                       // a row that exists; its sums are not stored
      if (up) n += a.N;
      wp[i] = a.codes + t.expert * a.sp.batch_codes + n * a.sp.ld_codes + g * BB;
      sp[i] = a.scales + t.expert * a.sp.batch_scales + n * a.sp.ld_scales + g;
    }
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      const int row = 16 * m + r;
      xp[m] = x_row(a, t.row0 + (row < t.rows ? row : t.rows - 1)) * a.sp.ld_x + g * 32;
    }
    uint32_t w[2][U][NT][kWords<FAM>], s[2][U][NT];
    XBlock<DT> x[U][MT];

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
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int m = 0; m < MT; ++m) x[u][m].load(a.x, xp[m] + k + u * kUnit);
        return;
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          const int64_t left = a.K - (k + u * kUnit + g * 32);
          x[u][m].load_first(a.x, xp[m] + k + u * kUnit, left < 0 ? 0 : left < 32 ? (int)left : 32);
        }
    };
    auto multiply = [&](const uint32_t (&w)[U][NT][kWords<FAM>], const uint32_t (&s)[U][NT]) {
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int i = 0; i < NT; ++i) {
          bf16x8 wv[4], wl[4];
          uint32_t left;
          const float scale = scale_of<FAM>(s[u][i], map, left);
#pragma unroll
          for (int j = 0; j < 4; ++j) wv[j] = eight<FAM>(w[u][i], scale, j, map);
          if (FAM == kMapped && __builtin_expect(__any(left), 0)) {
#pragma unroll
            for (int j = 0; j < 4; ++j) apply_left(wv[j], left);
          }
          if constexpr (P > 1 && FAM == kE5M2) {                       // an infinite weight meets no zero of a lower plane
            uint32_t f[8];
#pragma unroll
            for (int c = 0; c < 8; ++c) f[c] = without_infinities(w[u][i][c], ~0u);
#pragma unroll
            for (int j = 0; j < 4; ++j) wl[j] = eight<FAM>(f, scale, j, map);
          }
#pragma unroll
          for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              bf16x8 xv[P];
              x[u][m].planes(j, xv);
#pragma unroll
              for (int p = 0; p < P; ++p)
                acc[i][m] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(P > 1 && FAM == kE5M2 && p ? wl[j] : wv[j], xv[p], acc[i][m], 0, 0, 0);
            }
        }
    };

    constexpr int64_t stride = kSkinnyWaves * U * kUnit;
    int64_t k = (int64_t)wave * U * kUnit;
    if (k < a.K) load_w(k, w[0], s[0]);
    for (; k < a.K; k += 2 * stride) {
      load_x(k);
      if (k + stride < a.K) load_w(k + stride, w[1], s[1]);
      multiply(w[0], s[0]);
      if (k + stride >= a.K) break;
      load_x(k + stride);
      if (k + 2 * stride < a.K) load_w(k + 2 * stride, w[0], s[0]);
      multiply(w[1], s[1]);
    }
  }

#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int m = 0; m < MT; ++m) sums[wave][i * MT + m][lane] = acc[i][m];
  __syncthreads();

  // element (row m, weight row i 16 + n) of the tile's sums: lane (m & 15) + 16 (n / 4), component n % 4
  auto total = [&](int i, int m, int n) {
    const float* p = (const float*)&sums[0][i * MT + (m >> 4)][(m & 15) + 16 * (n >> 2)] + (n & 3);
    float z = p[0];
#pragma unroll
    for (int v = 1; v < kSkinnyWaves; ++v) z += p[(size_t)v * (NT * MT * 64 * 4)];
    return z;
  };
  for (int at = threadIdx.x; at < outputs * MT * 16; at += 64 * kSkinnyWaves) {
    const int n = at % outputs, m = at / outputs;
    if (m >= t.rows || n0 + n >= a.N) continue;
    const float z = total(n >> 4, m, n & 15), up = gated ? total(NT / 2 + (n >> 4), m, n & 15) : 0.0f;
    store_elem(a.y, a.sp.y_dtype, (t.row0 + m) * a.sp.ld_y + n0 + n, epilogue(a, t, t.row0 + m, n0 + n, z, up));
  }
}

template <int FAM, int DT> void launch_skinny_dt(const LinearArgs& a, int mt, int64_t tiles, hipStream_t st) {
  const CodeMap map = code_map(a.sp.format);
  auto go = [&](auto MT, auto NT, auto U) {
    const int outputs = a.sp.gated ? NT.value * 8 : NT.value * 16;
    const dim3 grid((unsigned)ceil_div(a.N, outputs), (unsigned)tiles);
    KernelTimer timer("k_linear_skinny", st);
    k_linear_skinny<FAM, DT, MT.value, NT.value, U.value><<<grid, 64 * kSkinnyWaves, 0, st>>>(a, map);
  };
  std::integral_constant<int, 1> one;
  std::integral_constant<int, 2> two;
  std::integral_constant<int, 4> four;
  if (mt == 1) {
    if (a.sp.gated) go(one, two, one);
    else go(one, one, two);
  } else if (mt == 2 || DT == MXQ_DT_F32) {
    go(two, two, one);
  } else {
    if constexpr (DT != MXQ_DT_F32) go(four, two, one);
  }
}

template <int FAM> void launch_skinny_family(const LinearArgs& a, int mt, int64_t tiles, hipStream_t st) {
  if (a.sp.x_dtype == MXQ_DT_BF16) launch_skinny_dt<FAM, MXQ_DT_BF16>(a, mt, tiles, st);
  else if (a.sp.x_dtype == MXQ_DT_F16) launch_skinny_dt<FAM, MXQ_DT_F16>(a, mt, tiles, st);
  else launch_skinny_dt<FAM, MXQ_DT_F32>(a, mt, tiles, st);
}

}  // namespace mxq
