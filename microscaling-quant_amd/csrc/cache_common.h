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
  float* partial;        // sums, maxima and sums of weights of parts of tiles; NULL: a workgroup has one whole tile
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

// How the work of few queries is cut.  A tile is `rows` rows of one head of keys (queries token by token, the heads that
// share it within) and its steps of 32 keys, one at least.  The batch's tiles, a sequence's with equal numbers of steps, lie
// one behind another on a line of steps, and every workgroup takes an equal piece of it, however lengths differ: a number of
// whole tiles, and a part of one before and behind them, whose sums are joined later.  Every wave finds its way by itself from
// the lengths.
constexpr int kStep = 32;
__device__ __forceinline__ int same(int v) { return __builtin_amdgcn_readfirstlane(v); }   // of a wave's lanes, as it is in all of them
__device__ __forceinline__ int64_t same(int64_t v) { return (int64_t)((uint64_t)(uint32_t)same((int)(v >> 32)) << 32 | (uint32_t)same((int)v)); }
__device__ __forceinline__ Sequence same(const Sequence& s) { return Sequence{same(s.start), same(s.n), same(s.length), same(s.lo), same(s.hi)}; }

struct Share {
  int tiles, steps;      // of a sequence: its tiles (of all heads), steps of each
};
__device__ __forceinline__ Share share_of(const AttendArgs& a, const Sequence& s, int rows) {
  const int tiles = (int)(((int64_t)s.n * a.group + rows - 1) / rows) * (int)a.c.kv_heads;
  return Share{tiles, s.hi > s.lo ? (s.hi - (s.lo & ~(kStep - 1)) + kStep - 1) / kStep : 1};
}
struct Line {
  int64_t total;         // steps
  int groups;            // workgroups that have a piece
  __device__ int64_t begin(int i) const { return total * i / groups; }
  __device__ int group_at(int64_t step) const { return (int)(((step + 1) * groups - 1) / total); }
};
__device__ __forceinline__ Line line_of(const AttendArgs& a, int rows, int least) {
  int64_t total = 0;
  for (int b = threadIdx.x & 63; b < a.a.B; b += 64) {
    const Share h = share_of(a, sequence(a, b), rows);
    total += (int64_t)h.tiles * h.steps;
  }
  for (int o = 32; o; o >>= 1) total += __shfl_xor(total, o);
  total = same(total);
  const int64_t most = (total + least - 1) / least;
  return Line{total, most < a.wanted ? (int)most : a.wanted};
}
// A tile: of sequence b (-1: there is none) the index-th, and the place of its first step on the line.
struct Tile {
  int b, index, steps;
  int64_t first;
};
// The tile at a step of the line, or the one with this number.
__device__ __forceinline__ Tile tile_of(const AttendArgs& a, int rows, int64_t at, bool number) {
  const int lane = threadIdx.x & 63;
  int64_t before = 0, steps_before = 0;
  for (int b0 = 0; b0 < a.a.B; b0 += 64) {
    Share h{0, 1};
    if (b0 + lane < a.a.B) h = share_of(a, sequence(a, b0 + lane), rows);
    const int64_t steps = (int64_t)h.tiles * h.steps, mine = number ? h.tiles : steps;
    int64_t upto = mine, steps_upto = steps;
    for (int o = 1; o < 64; o <<= 1) {
      const int64_t v = __shfl_up(upto, o), w = __shfl_up(steps_upto, o);
      if (lane >= o) upto += v, steps_upto += w;
    }
    upto += before, steps_upto += steps_before;
    const uint64_t found = __ballot(at < upto && at >= upto - mine);
    if (found) {
      const int owner = __builtin_ctzll(found);
      const int each = __shfl(h.steps, owner);
      const int64_t first = __shfl(steps_upto - steps, owner), within = at - __shfl(upto - mine, owner);
      const int index = same((int)(number ? within : within / each));
      return Tile{same(b0 + owner), index, same(each), same(first + (int64_t)index * each)};
    }
    before = __shfl(upto, 63), steps_before = __shfl(steps_upto, 63);
  }
  return Tile{-1, 0, 1, 0};
}
// Workgroups a CU (of a wave for each of its SIMDs) that the registers of the kernel of few queries are held to, and the
// steps that it asks for ahead.
constexpr int few_groups(int dtype, int blocks) { return blocks <= 2 ? 3 : blocks <= 4 || dtype == MXQ_DT_BF16 ? 2 : 1; }
constexpr int few_depth(int dtype, int blocks) { return blocks <= 4 ? 2 : 1; }

// Where the sums of a piece's parts of tiles lie: of the tile that its first step is in, and of its last one.
__device__ __forceinline__ int64_t part_slot(int group, bool first) { return 2 * (int64_t)group + !first; }

// The logarithm of a sum of weights relative to 2^top; of no weights -inf.
__device__ __forceinline__ float log_sum(float top, float sum) {
  if (sum == 0.0f) return -__builtin_inff();
  return top == -__builtin_inff() ? sum : (top + __builtin_amdgcn_logf(sum)) * 0.693147180559945309f;
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
