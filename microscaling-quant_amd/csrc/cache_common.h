// What the kernels of a key and value cache in MX formats share: codes as bfloat16 values, slots, how attention's work is
// cut.
#pragma once

#include "mxq_common.h"
#include "packed_linear_common.h"

namespace mxq {

// A row's block of 32 codes: 32 bytes, 16 of MXFP4's pairs.  FAM: kE4M3, kE5M2 or kPairs.
constexpr int kCacheBlock = 32;

// Codes 2 j and 2 j + 1 of some words times the scale as two bfloat16: exact (a code has at most 4 significant bits) but for
// values below 2^-126, rounded to bfloat16's subnormals.  scale: 2^(byte - 127) as the conversions take it, the byte in a
// float's exponent field.
template <int FAM> __device__ __forceinline__ uint32_t two_codes(const uint32_t* w, int j, float scale) {
  bf16x2 v;
  if constexpr (FAM == kPairs) {
    switch (j & 3) {
      case 0: v = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[j >> 2], scale, 0); break;
      case 1: v = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[j >> 2], scale, 1); break;
      case 2: v = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[j >> 2], scale, 2); break;
      default: v = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[j >> 2], scale, 3); break;
    }
  } else if constexpr (FAM == kE5M2) {
    v = j & 1 ? __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(w[j >> 1], scale, true) : __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(w[j >> 1], scale, false);
  } else {
    v = j & 1 ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[j >> 1], scale, true) : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[j >> 1], scale, false);
  }
  uint32_t u;
  __builtin_memcpy(&u, &v, 4);
  return u;
}
template <int FAM> __device__ __forceinline__ bf16x8 eight_codes(const uint32_t* w, float scale) {
  uint32_t v[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) v[j] = two_codes<FAM>(w, j, scale);
  bf16x8 r;
  __builtin_memcpy(&r, v, 16);
  return r;
}

// Whether some value of a word of codes under this scale byte is, or may be, an infinity or a NaN in bfloat16.
template <int FAM> __device__ __forceinline__ bool may_be_odd(uint32_t w, uint32_t scale) {
  if (scale >= kPastFloat<FAM>) return true;
  if constexpr (FAM == kPairs) return false;
  constexpr uint32_t special = FAM == kE4M3 ? 0x7F7F7F7Fu : 0x7C7C7C7Cu;
  const uint32_t x = (w & special) ^ special;               // a byte of zeros: E4M3's NaN, E5M2's infinities and NaNs
  return (x - 0x01010101u & ~x & 0x80808080u) != 0;
}
// Ones in the place of those of codes 2 j and 2 j + 1 whose value is no finite number, zeros in that of others; the codes
// become zeros.
template <int FAM> __device__ __forceinline__ uint32_t take_odd(uint32_t* w, int j, float scale) {
  const uint32_t x = two_codes<FAM>(w, j, scale);
  const bool low = (x & 0x7F80u) == 0x7F80u, high = (x & 0x7F800000u) == 0x7F800000u;
  constexpr int bits = FAM == kPairs ? 4 : 8, each = 32 / bits;
  const uint32_t code = (1u << bits) - 1, at = 2 * j % each * bits;
  w[2 * j / each] &= ~((low ? code << at : 0u) | (high ? code << (at + bits) : 0u));
  return (low ? 0x3F80u : 0u) | (high ? 0x3F800000u : 0u);
}

// Of pairs of neighbouring columns, a pair a key of eight keys, the keys of the first or the second column: an operand of
// the product with values.
__device__ __forceinline__ bf16x8 keys_of_column(const uint32_t (&x)[8], int second) {
  uint32_t y[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) y[i] = __builtin_amdgcn_perm(x[2 * i + 1], x[2 * i], second ? 0x07060302u : 0x05040100u);
  bf16x8 v;
  __builtin_memcpy(&v, y, 16);
  return v;
}

__device__ __forceinline__ float scale_field(uint32_t byte) { return __uint_as_float(byte << 23); }

struct AttendArgs {
  const void* q;
  const uint8_t *kc, *ks, *vc, *vs;
  const int32_t *table, *lengths, *starts;
  void* out;
  float* lse;
  float* partial;        // a unit's unnormalised sums, maxima and sums of weights; NULL: no sequence is split
  mxq_cache_spec c;
  mxq_attend_spec a;
  DivU31 by_page, by_group;
  int32_t group, blocks; // heads of q a head of keys; blocks a row
  int32_t aligned;       // pages of whole 16 rows, whose rows are less than 2^26 bytes apart
  int32_t wanted;        // workgroups that fill the card
  float scale2;          // scale times log2 e
};

// Sequence b as its lengths and starts say, held to what there is.  [lo, hi): the keys that some query of it sees.
struct Sequence {
  int start, n, length, lo, hi;
};
__device__ __forceinline__ Sequence sequence(const AttendArgs& a, int b) {
  Sequence s;
  const int T = (int)a.a.T;
  if (a.starts) {
    const int x = a.starts[b], y = a.starts[b + 1];
    s.start = x < 0 ? 0 : x > T ? T : x;
    s.n = (y > T ? T : y) - s.start;
    if (s.n < 0) s.n = 0;
  } else {
    s.n = T / (int)a.a.B;
    s.start = b * s.n;
  }
  const int64_t most = a.a.table_pages * a.c.page_size;
  const int l = a.lengths[b];
  s.length = l < 0 ? 0 : l > most ? (int)most : l;
  s.hi = s.n ? s.length : 0;
  s.lo = 0;
  if (a.a.window) {
    const int64_t lo = (int64_t)s.length - s.n + 1 - a.a.window;
    s.lo = lo <= 0 ? 0 : lo < s.hi ? (int)lo : s.hi;
  }
  return s;
}

// How the work is cut.  A unit is `rows` rows (a head of keys' queries, token by token, its heads within) and a run of
// keys; a sequence's keys are cut into runs of whole `steps` of 32, as many as make the units about fill the card, however
// its sequences' lengths differ.  Every wave finds its unit by itself from the lengths.
constexpr int kStep = 32;
__device__ __forceinline__ int same(int v) { return __builtin_amdgcn_readfirstlane(v); }   // of a wave's lanes, as it is in all of them
__device__ __forceinline__ Sequence same(const Sequence& s) { return Sequence{same(s.start), same(s.n), same(s.length), same(s.lo), same(s.hi)}; }
struct Cut {
  int tiles, runs;       // tiles of rows, runs of keys of each
};
__device__ __forceinline__ int steps_of(const Sequence& s) { return s.hi > s.lo ? (s.hi - (s.lo & ~(kStep - 1)) + kStep - 1) / kStep : 0; }
__device__ __forceinline__ Cut cut(const AttendArgs& a, const Sequence& s, int rows, int quota) {
  Cut c;
  c.tiles = (int)(((int64_t)s.n * a.group + rows - 1) / rows);
  const int steps = steps_of(s);
  c.runs = a.partial && steps > quota ? (steps + quota - 1) / quota : 1;
  return c;
}
__device__ __forceinline__ int wave_sum(int v) {
  for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
  return v;
}
// Steps a unit should take: the batch's steps over the units wanted, `least` at least.
__device__ __forceinline__ int quota_of(const AttendArgs& a, int rows, int least) {
  if (!a.partial) return least;
  const int lane = threadIdx.x & 63;
  float total = 0.0f;                                       // a number of the batch's steps, not a sum that results depend on
  for (int b = lane; b < a.a.B; b += 64) {
    const Sequence s = sequence(a, b);
    total += (float)cut(a, s, rows, 1 << 30).tiles * (float)steps_of(s);
  }
  for (int o = 32; o; o >>= 1) total += __shfl_xor(total, o);
  const float each = total * (float)a.c.kv_heads / (float)a.wanted;
  const int quota = each < 1e9f ? (int)__builtin_ceilf(each) : 1000000000;
  return quota < least ? least : quota;
}
struct Unit {
  int b, tile, run, runs, head;   // b < 0: there is none
};
__device__ __forceinline__ Unit unit_of(const AttendArgs& a, int rows, int quota, int index) {
  const int lane = threadIdx.x & 63, heads = (int)a.c.kv_heads;
  const int which = index / heads, head = index - which * heads;
  int before = 0;
  for (int b0 = 0; b0 < a.a.B; b0 += 64) {
    Cut c{0, 1};
    if (b0 + lane < a.a.B) c = cut(a, sequence(a, b0 + lane), rows, quota);
    const int mine = c.tiles * c.runs;
    int upto = mine;
    for (int o = 1; o < 64; o <<= 1) {
      const int v = __shfl_up(upto, o);
      if (lane >= o) upto += v;
    }
    const uint64_t at = __ballot(which < before + upto && which >= before + upto - mine);
    if (at) {
      const int owner = __builtin_ctzll(at);
      const int within = which - before - __builtin_amdgcn_readlane(upto - mine, owner);
      const int runs = __builtin_amdgcn_readlane(c.runs, owner), tile = within / runs;
      return Unit{same(b0 + owner), same(tile), same(within - tile * runs), same(runs), head};
    }
    before += __builtin_amdgcn_readlane(upto, 63);
  }
  return Unit{-1, 0, 0, 1, 0};
}

template <int DT> constexpr int kAttendPlanes = DT == MXQ_DT_BF16 ? 1 : DT == MXQ_DT_F16 ? 2 : 3;

// Eight float32 as bfloat16 planes, each the leading bits of what the ones before leave: three hold all of a float32 down
// to 2^-133, two hold a float16.  A single plane is rounded to the nearest.
template <int P> __device__ __forceinline__ void planes_of(float (&f)[8], bf16x8 (&out)[P]) {
  if constexpr (P == 1) {
    bf16x2 w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = bf16x2{(__bf16)f[2 * i], (__bf16)f[2 * i + 1]};
    __builtin_memcpy(&out[0], w, 16);
  } else {
#pragma unroll
    for (int p = 0; p < P; ++p) {
      uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        w[i] = __builtin_amdgcn_perm(__float_as_uint(f[2 * i + 1]), __float_as_uint(f[2 * i]), 0x07060302u);
      __builtin_memcpy(&out[p], w, 16);
      if (p + 1 < P) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float hi = __uint_as_float(__float_as_uint(f[i]) & 0xFFFF0000u);
          f[i] = f[i] == hi ? 0.0f : f[i] - hi;                          // infinities leave nothing
        }
      }
    }
  }
}

// Eight neighbouring columns of a row of q as planes, the first `valid` of them there.
template <int DT> __device__ __forceinline__ void load_query(const void* q, int64_t at, int valid, bf16x8 (&out)[kAttendPlanes<DT>]) {
  float f[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = 0.0f;
  if (valid >= 8) {
    add_eight(f, q, DT, at);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < valid) f[i] = load_elem(q, DT, at + i);
  }
  planes_of(f, out);
}

}  // namespace mxq
