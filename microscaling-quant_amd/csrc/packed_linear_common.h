// What the kernels of products with packed weights share: arguments, the tiles of rows by expert, codes as bfloat16
// values, the epilogue.
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
  e = __builtin_amdgcn_readlane(e, owner), row0 = __builtin_amdgcn_readlane(row0, owner), rows = __builtin_amdgcn_readlane(rows, owner);
  return RowTile{e == a.E ? 0 : e, rows, row0, e == a.E};
}

// x's row for row r of y.
__device__ __forceinline__ int64_t x_row(const LinearArgs& a, int64_t r) {
  if (!a.offsets || !a.sp.top_k) return r;
  const int slot = a.order[r];
  return (slot < 0 || slot >= a.M ? 0 : slot) / a.sp.top_k;
}

typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2;
typedef __attribute__((ext_vector_type(2))) _Float16 f16x2;
typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;
typedef __attribute__((ext_vector_type(4))) float f32x4;
typedef __attribute__((ext_vector_type(16))) float f32x16;
typedef __attribute__((ext_vector_type(4))) uint32_t u32x4;
typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(1)));       // at any address

// How a format's bytes become bfloat16.  kMapped: the formats of 4 and 6 bits a byte, put into E4M3's fields first.
enum Family { kE4M3 = 0, kE5M2 = 1, kMapped = 2, kPairs = 3 };

// 32 codes of one row with one scale: eight words, four of MXFP4's pairs.
template <int FAM> constexpr int kWords = FAM == kPairs ? 4 : 8;
template <int FAM> constexpr int kBlockBytes = FAM == kPairs ? 16 : 32;

// E3M2 and E2M1 move up to E4M3's fields, E2M3 keeps its place.  The exponents' biases differ, so that the fields alone
// are 2^4 or 2^6 too small; the scale makes up for it.
struct CodeMap {
  uint32_t mask;        // magnitude bits, in every byte
  int shift, sign;      // how far they and the sign move up
  uint32_t power;       // what the scale's exponent gains
};
inline CodeMap code_map(int format) {
  if (format == MXQ_FMT_E3M2) return CodeMap{0x1F1F1F1Fu, 1, 2, 4};
  if (format == MXQ_FMT_E2M3) return CodeMap{0x1F1F1F1Fu, 0, 2, 6};
  return CodeMap{0x07070707u, 2, 4, 6};
}

// Activations of several planes meet an infinite weight in the first one; the lower ones, which are zero where an activation
// has no more bits, see the largest finite value in its place (finite_only), or zero times infinity would make a NaN.  From
// this scale byte on a code's largest value is 2^128 or more, infinite in bfloat16 as in float32; a value of a code's few
// bits below 2^128 is finite in both.
template <int FAM> constexpr uint32_t kPastFloat = FAM == kE4M3 ? 247 : FAM == kE5M2 ? 240 : FAM == kMapped ? 251 : 253;
constexpr uint32_t kFinite = 0x80000000u;

// The E8M0 byte as the conversions take it: a float's exponent field, 0 standing for 2^-127 and 255 for NaN.  `left` holds
// what a block seldom needs besides.  kMapped: the excess of a scale past 2^127 with the map's power, for apply_left.
// lower, the block's codes for a lower plane: a bit above the lowest eight where one of them may be an infinity.
template <int FAM> __device__ __forceinline__ float scale_of(uint32_t s, const uint32_t (&codes)[kWords<FAM>], const CodeMap& map,
                                                             uint32_t& left, bool lower) {
  left = 0;
  uint32_t infinite = s >= kPastFloat<FAM> ? kFinite : 0;
  if constexpr (FAM == kMapped) {
    const uint32_t t = s + map.power;
    left = s != 255 && t > 254 ? t - 254 : 0;
    s = s == 255 ? 255 : t < 254 ? t : 254;
  }
  if constexpr (FAM == kE5M2) {
    uint32_t none = ~0u;                                           // a byte's highest bit: no code 0x7C or 0xFC there
#pragma unroll
    for (int i = 0; i < kWords<FAM>; ++i) none &= ((codes[i] & 0x7F7F7F7Fu) ^ 0x7C7C7C7Cu) + 0x7F7F7F7Fu;
    infinite |= (~none & 0x80808000u) | (~none & 0x80u) << 1;
  }
  if (lower) left |= infinite;
  return __uint_as_float(s << 23);
}
__device__ __forceinline__ void apply_left(bf16x8& w, uint32_t left) {
  const float more = __uint_as_float((127 + (left & 255)) << 23);
#pragma unroll
  for (int i = 0; i < 8; ++i) w[i] = (__bf16)((float)w[i] * more);
}
// Magnitudes past bfloat16's largest become it, NaN too, which the first plane has shown.
__device__ __forceinline__ void finite_only(bf16x8& w) {
  typedef uint16_t u16x8 __attribute__((ext_vector_type(8)));
  u16x8 u;
  __builtin_memcpy(&u, &w, 16);
  u = __builtin_elementwise_min(u & (uint16_t)0x7FFF, (u16x8)(uint16_t)0x7F7F) | (u & (uint16_t)0x8000);
  __builtin_memcpy(&w, &u, 16);
}

// The j-th eight of the 32 codes as bfloat16, times the scale: exact (a code has at most 4 significant bits), but for
// values below 2^-126, rounded to bfloat16's subnormals.  One instruction makes two values.
template <int FAM> __device__ __forceinline__ bf16x8 eight(const uint32_t (&w)[kWords<FAM>], float scale, int j, const CodeMap& map) {
  bf16x2 v[4];
  if constexpr (FAM == kPairs) {
    v[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[j], scale, 0);
    v[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[j], scale, 1);
    v[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[j], scale, 2);
    v[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[j], scale, 3);
  } else {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      uint32_t c = w[2 * j + i];
      if constexpr (FAM == kE5M2) {
        v[2 * i] = __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(c, scale, false);
        v[2 * i + 1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(c, scale, true);
      } else {
        if constexpr (FAM == kMapped) c = (c & map.mask) << map.shift | (c << map.sign & 0x80808080u);
        v[2 * i] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c, scale, false);
        v[2 * i + 1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c, scale, true);
      }
    }
  }
  bf16x8 r;
  __builtin_memcpy(&r, v, 16);
  return r;
}

// The arguments of k_linear_tile.
struct TileArgs {
  LinearArgs l;
  const uint16_t* x;      // bfloat16 planes one after another along a row, rows of ld_x, 16-byte aligned
  int64_t ld_x;
  int32_t steps, planes;  // 64 columns a step, an even number of steps a plane
  int32_t x_columns, w_columns;   // that exist in a plane of x and in a row of codes; the others are zeros
  int32_t tiles_m, tiles_n, split;
  float* partial;         // split > 1: split x M x rows of the weight
  CodeMap map;
};

struct TilePlan {
  int shape;              // 0: 256 x 256, 1: 128 x 128, 2: 64 x 128, 3: as 2, for rows 2^32 bytes apart
  int split;
};

// 16 bytes of which the first `valid` exist; zeros for the others.
__device__ __forceinline__ u32x4 load_part(const uint8_t* p, int valid) {
  u32x4 v = {0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < 16; ++i)
    if (i < valid) v[i >> 2] |= (uint32_t)p[i] << (i & 3) * 8;
  return v;
}

// sigmoid by the hardware's exp2 and reciprocal, each within one unit in the last place.
__device__ __forceinline__ float sigmoid(float z) {
  return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(z * -1.44269504088896341f));
}

// Of an odd number of MXFP4 codes the last byte's high half is no code.
__device__ __forceinline__ void clear_odd(u32x4& v, int valid) {
  const uint32_t keep = ~(0xF0u << (valid >> 1 & 3) * 8);
#pragma unroll
  for (int c = 0; c < 4; ++c)
    if (c == valid >> 3) v[c] &= keep;
}

// The normal distribution's share below z: with t = 1 / (1 + 0.39 |z| / sqrt 2), half of erfc(|z| / sqrt 2) is
// t p(t) exp(-z^2 / 2), p fitted here to 8e-9 of erfc; z times it is off by at most 2.2e-7 |z|.
__device__ __forceinline__ float normal_below(float z) {
  const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.27577164f, __builtin_fabsf(z), 1.0f));
  float p = __builtin_fmaf(-0.113768743f, t, 0.443332924f);
  p = __builtin_fmaf(p, t, -0.317701341f);
  p = __builtin_fmaf(p, t, 0.32478067f);
  p = __builtin_fmaf(p, t, 0.0456938178f);
  p = __builtin_fmaf(p, t, 0.117662672f);
  const float q = t * p * __builtin_amdgcn_exp2f(z * z * -0.72134752f);
  return z < 0.0f ? q : 1.0f - q;
}

__device__ __forceinline__ float activate(float z, int activation) {
  switch (activation) {
    case MXQ_ACT_SILU: return z * sigmoid(z);
    case MXQ_ACT_GELU: return z * normal_below(z);
    case MXQ_ACT_GELU_TANH: return z * sigmoid(1.59576912160573071f * (z + 0.044715f * z * z * z));
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

// Eight neighbours as they lie in memory (float32's second half in `more`), and their sum with v.
struct Eight {
  u32x4 first, more;
};
__device__ __forceinline__ Eight load_eight(const void* p, int dtype, int64_t at) {
  Eight e;
  if (dtype == MXQ_DT_F32) {
    e.first = *(const u32x4_any*)((const float*)p + at);
    e.more = *(const u32x4_any*)((const float*)p + at + 4);
  } else {
    e.first = *(const u32x4_any*)((const uint16_t*)p + at);
  }
  return e;
}
__device__ __forceinline__ void add_eight(float (&v)[8], const Eight& e, int dtype) {
  if (dtype == MXQ_DT_F32) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] += __uint_as_float(e.first[i]), v[i + 4] += __uint_as_float(e.more[i]);
  } else if (dtype == MXQ_DT_BF16) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] += __uint_as_float(e.first[i] << 16);
      v[2 * i + 1] += __uint_as_float(e.first[i] & 0xFFFF0000u);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f16x2 b;
      __builtin_memcpy(&b, (const char*)&e.first + 4 * i, 4);
      v[2 * i] += (float)b[0];
      v[2 * i + 1] += (float)b[1];
    }
  }
}
__device__ __forceinline__ void add_eight(float (&v)[8], const void* p, int dtype, int64_t at) { add_eight(v, load_eight(p, dtype, at), dtype); }

__device__ __forceinline__ void activate_eight(float (&v)[8], int activation) {
  switch (activation) {
#define MXQ_EACH(ACT)                                        \
  case ACT:                                                  \
    _Pragma("unroll") for (int i = 0; i < 8; ++i) v[i] = activate(v[i], ACT); \
    break;
    MXQ_EACH(MXQ_ACT_SILU)
    MXQ_EACH(MXQ_ACT_GELU)
    MXQ_EACH(MXQ_ACT_GELU_TANH)
    MXQ_EACH(MXQ_ACT_RELU)
#undef MXQ_EACH
  }
}

// The biases of eight neighbouring outputs, all below N: of z and, gated, of up.
struct Bias {
  float z[8], up[8];
};
__device__ __forceinline__ Bias load_bias(const LinearArgs& a, const RowTile& t, int64_t n) {
  Bias b = {};
  const int64_t first = t.expert * a.sp.batch_bias + n;
  if (a.bias) add_eight(b.z, a.bias, a.sp.bias_dtype, first);
  if (a.bias && a.sp.gated) add_eight(b.up, a.bias, a.sp.bias_dtype, first + a.N);
  return b;
}

// epilogue and store of eight neighbouring outputs of a row, all below N; residual: theirs, if there is one.
__device__ __forceinline__ void finish_eight(const LinearArgs& a, const RowTile& t, int64_t row, int64_t n, float (&z)[8], float (&up)[8],
                                             const Bias& bias, const Eight& residual) {
  if (t.zeros) {
#pragma unroll
    for (int i = 0; i < 8; ++i) z[i] = 0.0f;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) z[i] += bias.z[i];
    activate_eight(z, a.sp.activation);
    if (a.sp.gated) {
#pragma unroll
      for (int i = 0; i < 8; ++i) z[i] *= up[i] + bias.up[i];
    }
    if (a.residual) add_eight(z, residual, a.sp.residual_dtype);
  }
  const int64_t at = row * a.sp.ld_y + n;
  if (a.sp.y_dtype == MXQ_DT_F32) {
    u32x4 p, q;
#pragma unroll
    for (int i = 0; i < 4; ++i) p[i] = __float_as_uint(z[i]), q[i] = __float_as_uint(z[i + 4]);
    *(u32x4_any*)((float*)a.y + at) = p;
    *(u32x4_any*)((float*)a.y + at + 4) = q;
    return;
  }
  u32x4 p;
  if (a.sp.y_dtype == MXQ_DT_BF16) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const bf16x2 b = {(__bf16)z[2 * i], (__bf16)z[2 * i + 1]};
      __builtin_memcpy((char*)&p + 4 * i, &b, 4);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const f16x2 b = {(_Float16)z[2 * i], (_Float16)z[2 * i + 1]};
      __builtin_memcpy((char*)&p + 4 * i, &b, 4);
    }
  }
  *(u32x4_any*)((uint16_t*)a.y + at) = p;
}

}  // namespace mxq
