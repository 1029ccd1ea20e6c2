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
  int32_t wanted, least; // workgroups that fill the card, and steps that one takes at least
  int32_t above, upto;   // the numbers of rows a sequence that this launch takes: (above, upto]
  int32_t fill;          // whether this launch writes the rows of no sequence
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

// Zeros for the queries of no sequence: [0, starts[0]) and [starts[B], T).  By all workgroups of a launch together.
__device__ __forceinline__ void fill_rows(const AttendArgs& a) {
  const int T = (int)a.a.T, x = a.a.B ? a.starts[0] : T, y = a.a.B ? a.starts[a.a.B] : T, D = a.c.head_dim;
  const int64_t head = (int64_t)(x < 0 ? 0 : x > T ? T : x) * a.a.heads, tail = (int64_t)(y < 0 ? 0 : y > T ? T : y) * a.a.heads;
  const int64_t from = tail < head ? head : tail, all = head + (a.a.T * a.a.heads - from);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
  for (int64_t i = (int64_t)blockIdx.x * waves + wave; i < all; i += (int64_t)gridDim.x * waves) {
    const int64_t row = i < head ? i : from + i - head;
    for (int d = lane; d < D; d += 64) store_elem(a.out, a.a.dtype, row * D + d, 0.0f);
    if (a.lse && lane == 0) a.lse[row] = -__builtin_inff();
  }
}

// How the work is cut.  A tile is `size` rows of one head of keys (queries token by token, the heads that share it within).  A
// tile's weight is about the keys that its queries see, times the heads that share one, and what starting it costs.  The
// batch's tiles lie one behind another on a line, and every workgroup takes an equal piece of it, however lengths differ: a
// number of whole tiles, and a part of one before and behind them, whose sums are joined later.  Where tiles are few, each is cut
// into pieces of its own: a part's beginning and end cost a workgroup about as much as the pieces' unlike sizes (16 sequences
// of 700 to 8192 keys, 128 tiles: 37 us, and 45 by equal pieces of the line; one token's 2000 keys of 8 heads 19 and 18).
// Where there are tiles enough, a workgroup takes one whole tile instead, a sequence's last ones, which see most, first, and
// heads in turn, so that with eight of them each part of the card reads one head's keys.  Every wave finds its way by itself
// from the lengths, by the same arithmetic, so that all agree: no call waits for the host to read lengths, and a captured one
// follows them.
constexpr int kStep = 32;
__device__ __forceinline__ int same(int v) { return __builtin_amdgcn_readfirstlane(v); }   // of a wave's lanes, as it is in all of them
__device__ __forceinline__ int64_t same(int64_t v) { return (int64_t)((uint64_t)(uint32_t)same((int)(v >> 32)) << 32 | (uint32_t)same((int)v)); }

// The weights of a sequence's tiles of one head: `base` and 2^shift more for each tile before and itself, `most` at most.
struct Weights {
  int tiles, shift;      // shift < 0: all of weight `base`
  int64_t base, most, start;
  __device__ __forceinline__ int64_t of(int j) const {
    const int64_t w = shift < 0 ? base : base + ((int64_t)(j + 1) << shift);
    return (w < most ? w : most) + start;
  }
  __device__ __forceinline__ int64_t before(int j) const {          // of the first j together
    int64_t grow = shift < 0 ? 0 : (most - base) >> shift;          // tiles whose weight still grows
    grow = grow < 0 ? 0 : grow < j ? grow : j;
    return grow * base + (grow * (grow + 1) / 2 << (shift & 63)) + (j - grow) * most + j * start;
  }
};
// Of this lane: a sequence and its weights.  unit: 0, or what the tiles of a sequence, all as heavy as its last one, are cut
// into: a tile's weight is then its pieces.
struct Member {
  Sequence s;
  Weights w;
};
__device__ __forceinline__ Weights in_pieces(const Weights& w, double unit) {
  const int64_t pieces = w.tiles ? (int64_t)((double)w.of(w.tiles - 1) / unit) + 1 : 0;
  return Weights{w.tiles, -1, pieces, pieces, 0};
}
__device__ __forceinline__ Member member(const AttendArgs& a, int b, int size, double unit) {
  constexpr int64_t kMost = (int64_t)1 << 34;                       // so that no sum of weights passes 63 bits
  auto hold = [](int64_t v) { return v < kMost ? v : kMost; };
  Member m{};
  if (b >= a.a.B) return m;
  m.s = sequence(a, b);
  const Sequence& s = m.s;
  Weights& w = m.w;
  const int rows = s.n * a.group;
  w.tiles = rows > a.above && rows <= a.upto ? (rows + size - 1) / size : 0;
  w.start = hold((int64_t)4 * kStep * a.group);
  if (a.a.causal) {
    w.shift = __builtin_ctz(size);
    w.base = s.length > s.n ? hold((int64_t)(s.length - s.n) * a.group) : 0;
    w.most = a.a.window ? hold(a.a.window * a.group + size) : 2 * kMost;
  } else {
    const int64_t keys = a.a.window && a.a.window < s.length - s.n ? a.a.window + s.n : s.length;
    w.shift = -1, w.base = w.most = hold(keys * a.group);
  }
  if (unit != 0.0) w = in_pieces(w, unit);
  return m;
}
struct Line {
  int64_t total;
  double each;           // weight of a piece
  int groups;            // workgroups that have one
  double unit;           // weight that a piece is of, where no piece is of two tiles; else 0
  // begin(groups) is the total exactly while that is below 2^51 steps, which no call lives to see the end of.
  __device__ __forceinline__ int64_t begin(int i) const { return (int64_t)(each * i + 0.5); }
  __device__ __forceinline__ int group_at(int64_t at) const {
    int i = (int)((double)at / each);
    i = i < groups ? i : groups - 1;
    while (i > 0 && begin(i) > at) --i;
    while (i + 1 < groups && begin(i + 1) <= at) ++i;
    return i;
  }
};
// own: of lane l sequence l; its weights become the line's.
__device__ __forceinline__ Line line_of(const AttendArgs& a, int size, Member& own) {
  const int lane = threadIdx.x & 63, heads = (int)a.c.kv_heads;
  auto sum = [&](int64_t v) {
    for (int o = 1; o < 64 && o < a.a.B; o <<= 1) v += __shfl_xor(v, o);
    return same(v) * heads;
  };
  auto even_weight = [](const Weights& w) { return w.tiles ? w.tiles * w.of(w.tiles - 1) : 0; };
  int64_t total = own.w.before(own.w.tiles), even = even_weight(own.w), all = own.w.tiles;
  for (int b = 64 + lane; b < a.a.B; b += 64) {
    const Weights w = member(a, b, size, 0.0).w;
    total += w.before(w.tiles), even += even_weight(w), all += w.tiles;
  }
  total = sum(total), even = sum(even), all = sum(all);
  const double least = (double)a.least * kStep * a.group;
  if (2 * all <= a.wanted && even <= total + total / 4) {
    // w / unit + 1 pieces of each tile are `wanted` together
    const double share = (double)even / (double)(a.wanted - all), unit = share < least ? least : share;
    own.w = in_pieces(own.w, unit);
    int64_t pieces = own.w.before(own.w.tiles);
    for (int b = 64 + lane; b < a.a.B; b += 64) {
      const Weights w = member(a, b, size, unit).w;
      pieces += w.before(w.tiles);
    }
    pieces = sum(pieces);
    return Line{pieces, 1.0, (int)pieces, unit};
  }
  const double most = (double)total / least + 1.0;
  int n = most < a.wanted ? (int)most : a.wanted;
  // less work than fills the card: a whole number of pieces a tile, so that equal tiles' ends are pieces' ends
  if (n < a.wanted && all <= a.wanted) n = all ? (int)all * (n > all ? n / (int)all : 1) : 1;
  return Line{total, (double)total / n, n, 0.0};
}
// A tile: of sequence b (-1: there is none) and a head of keys, and its place on the line.
struct Tile {
  int b, head, row;
  int64_t first, weight;
  Sequence s;
};
// The tile at a point of the line or, `number`, the one with this number.
__device__ __forceinline__ Tile tile_of(const AttendArgs& a, int size, const Member& own, double unit, int64_t at, bool number) {
  const int lane = threadIdx.x & 63, heads = (int)a.c.kv_heads;
  int64_t before = 0, weight_before = 0;
  for (int b0 = 0; b0 < a.a.B; b0 += 64) {
    const Member m = b0 ? member(a, b0 + lane, size, unit) : own;
    const Weights& w = m.w;
    const int64_t of_head = w.before(w.tiles), weight = of_head * heads, mine = number ? (int64_t)w.tiles * heads : weight;
    int64_t upto = mine, weight_upto = weight;
    for (int o = 1; o < 64 && o < a.a.B; o <<= 1) {
      const int64_t v = __shfl_up(upto, o), x = __shfl_up(weight_upto, o);
      if (lane >= o) upto += v, weight_upto += x;
    }
    upto += before, weight_upto += weight_before;
    const uint64_t found = __ballot(at < upto && at >= upto - mine);
    if (found) {
      const int owner = __builtin_ctzll(found);
      int head = 0, row = 0;
      int64_t first = 0, its = 0;
      if (lane == owner) {
        int64_t in = at - (upto - mine);
        if (number) {
          row = (int)((uint32_t)in / (uint32_t)heads), head = (int)in - row * heads, row = w.tiles - 1 - row;
        } else {
          head = (int)((double)in / (double)of_head);
          while (head > 0 && head * of_head > in) --head;
          while ((head + 1) * of_head <= in) ++head;
          in -= head * of_head;
          int low = 0, high = w.tiles;                              // the last tile that begins at `in` or before
          while (high - low > 1) {
            const int mid = (low + high) >> 1;
            if (w.before(mid) <= in) low = mid;
            else high = mid;
          }
          row = low;
        }
        first = weight_upto - weight + head * of_head + w.before(row), its = w.of(row);
      }
      auto its_own = [&](int v) { return __builtin_amdgcn_readlane(v, owner); };
      auto its_own64 = [&](int64_t v) { return (int64_t)((uint64_t)(uint32_t)its_own((int)(v >> 32)) << 32 | (uint32_t)its_own((int)v)); };
      return Tile{same(b0 + owner), its_own(head), its_own(row), its_own64(first), its_own64(its),
                  Sequence{its_own(m.s.start), its_own(m.s.n), its_own(m.s.length), its_own(m.s.lo), its_own(m.s.hi)}};
    }
    before = __shfl(upto, 63), weight_before = __shfl(weight_upto, 63);
  }
  return Tile{-1, 0, 0, 0, 1, {}};
}
// The tile behind a tile on the line.
__device__ __forceinline__ Tile next_tile(const AttendArgs& a, int size, double unit, const Tile& u) {
  const int lane = threadIdx.x & 63, B = (int)a.a.B;
  Tile v = u;
  v.first = u.first + u.weight;
  Weights w = member(a, u.b, size, unit).w;
  if (u.row + 1 < w.tiles) {
    ++v.row;
  } else if (u.head + 1 < (int)a.c.kv_heads) {
    ++v.head, v.row = 0;
  } else {
    v.b = -1, v.head = v.row = 0;
    for (int b0 = u.b + 1; b0 < B && v.b < 0; b0 += 64) {
      const uint64_t found = __ballot(member(a, b0 + lane, size, unit).w.tiles > 0);
      if (found) v.b = b0 + __builtin_ctzll(found);
    }
    if (v.b < 0) return v;
    const Member m = member(a, v.b, size, unit);
    v.s = Sequence{same(m.s.start), same(m.s.n), same(m.s.length), same(m.s.lo), same(m.s.hi)};
    w = m.w;
  }
  v.weight = same(w.of(v.row));
  return v;
}
// Of `steps` those before a share of a tile's weight.
__device__ __forceinline__ int steps_before(int steps, int64_t share, int64_t weight) {
  if (share >= weight) return steps;
  const int n = (int)((float)steps * ((float)share * __builtin_amdgcn_rcpf((float)weight)));
  return n < steps ? n : steps;
}
// Where the sums of a piece's parts of tiles lie: of the tile that its first point is in, and of its last one.
__device__ __forceinline__ int64_t part_slot(int group, bool first) { return 2 * (int64_t)group + !first; }

constexpr int kWaves = 4;
// Sixteens of rows that a wave of many queries has: about as many as let two waves share a SIMD's registers (of float32's three
// planes half as many).  Not all forms fit.  Bytes a lane in scratch memory, of bfloat16 queries: up to 64 columns 40 to 64 where
// tiles are whole and 92 to 136 where they are cut, up to 128 none and 8 to 24, past that, of MXFP8 keys, 80 to 96 and 204 to 212
// (a prompt of 4096 tokens, 32 heads of 64, takes 211 us, 16 heads of 256 take 376).  What finds a piece's tiles, live through
// its steps, is most of it.
constexpr int attend_rows(int dtype, int blocks) { return blocks == 8 ? 1 : dtype == MXQ_DT_F32 ? 4 / blocks : 8 / blocks; }
// Workgroups a CU (of a wave for each of its SIMDs) that the registers are held to; with sixteen rows of 64 columns, where three
// would nearly fit, 64 sequences' 512 and 1024 tiles took 55 and 92 us of three, 51 and 97 of two.  Bytes a lane in scratch
// memory, of tiles of few rows: bfloat16 queries of more than 128 columns 80 to 84 over MXFP8 keys and 264 to 272 where tiles
// are cut, over MXFP4 keys 16 there (64 single tokens over 4096 MXFP8 keys of 4 heads of 256: 167 us; float32 ones, of one
// workgroup a CU, 126); 32 rows of 128 columns 16 to 72 where they are cut; float32 queries of 64 columns 16.
constexpr int attend_groups(int dtype, int blocks, int tiles) { return dtype == MXQ_DT_BF16 || tiles * blocks < 8 ? 2 : 1; }
constexpr int blocks_class(int blocks) { return blocks <= 2 ? 2 : blocks <= 4 ? 4 : 8; }

// The logarithm of a sum of weights relative to 2^top; of no weights -inf.
__device__ __forceinline__ float log_sum(float top, float sum) {
  if (sum == 0.0f) return -__builtin_inff();
  return top == -__builtin_inff() ? sum : (top + __builtin_amdgcn_logf(sum)) * 0.693147180559945309f;
}

template <int DT> constexpr int kAttendPlanes = DT == MXQ_DT_BF16 ? 1 : DT == MXQ_DT_F16 ? 2 : 3;   // of queries
// Planes of their weights, of tiles of many rows or of few.  bfloat16 queries' weights in one plane, rounded by 2^-9 on the
// average of each, add about as much to an output as its own rounding does; a second plane takes that away (an error of 2.6
// thousandths becomes 1.6, one token's 1000 keys of 64 columns).  Few rows, where the cache's bytes are the cost, have it: 64
// sequences of 4 to 8 thousand keys 112.7 us, 109.8 without; eight of 4096 with 64 rows a head 43.5 and 40.6.  Many rows, where
// products are, do not: a prompt of 8192 would take 958 us for 802, for 1.6 thousandths instead of 2.0.
constexpr int weight_planes_of(int dtype, bool many) { return dtype == MXQ_DT_F32 ? 3 : dtype == MXQ_DT_F16 || !many ? 2 : 1; }

// Eight float32 as bfloat16 planes, each the leading bits of what the ones before leave, the last one rounded to the nearest:
// three hold all of a float32 down to 2^-133, two all of a float16.
template <int P> __device__ __forceinline__ void planes_of(float (&f)[8], bf16x8 (&out)[P]) {
#pragma unroll
  for (int p = 0; p + 1 < P; ++p) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      w[i] = __builtin_amdgcn_perm(__float_as_uint(f[2 * i + 1]), __float_as_uint(f[2 * i]), 0x07060302u);
    __builtin_memcpy(&out[p], w, 16);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float hi = __uint_as_float(__float_as_uint(f[i]) & 0xFFFF0000u);
      f[i] = f[i] == hi ? 0.0f : f[i] - hi;                              // infinities leave nothing
    }
  }
  bf16x2 w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = bf16x2{(__bf16)f[2 * i], (__bf16)f[2 * i + 1]};
  __builtin_memcpy(&out[P - 1], w, 16);
}

// Eight weights (finite or NaN) as bfloat16 planes: all of them in three; else each plane to the nearest, all but 2^-16 in two
// and all but 2^-8 in one.
template <int P> __device__ __forceinline__ void weight_planes(float (&f)[8], bf16x8 (&out)[P]) {
  if constexpr (P == 3) {
    planes_of(f, out);
  } else {
#pragma unroll
    for (int p = 0; p < P; ++p) {
      uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const bf16x2 two = {(__bf16)f[2 * i], (__bf16)f[2 * i + 1]};
        __builtin_memcpy(&w[i], &two, 4);
        if (p + 1 < P) f[2 * i] -= __uint_as_float(w[i] << 16), f[2 * i + 1] -= __uint_as_float(w[i] & 0xFFFF0000u);
      }
      __builtin_memcpy(&out[p], w, 16);
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

// Four neighbouring columns of a row of the output, the first `valid` of them there.
template <int DT> __device__ __forceinline__ void store_four(void* p, int64_t at, int valid, const float (&v)[4]) {
  if (valid >= 4) {
    if constexpr (DT == MXQ_DT_F32) {
      __builtin_memcpy((float*)p + at, v, 16);
    } else if constexpr (DT == MXQ_DT_BF16) {
      const bf16x2 w[2] = {{(__bf16)v[0], (__bf16)v[1]}, {(__bf16)v[2], (__bf16)v[3]}};
      __builtin_memcpy((uint16_t*)p + at, w, 8);
    } else {
      const f16x2 w[2] = {{(_Float16)v[0], (_Float16)v[1]}, {(_Float16)v[2], (_Float16)v[3]}};
      __builtin_memcpy((uint16_t*)p + at, w, 8);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < valid) store_elem(p, DT, at + i, v[i]);
  }
}

}  // namespace mxq
