// Attention over a cache in MX formats.
//
//   s = scale q k^T;  out = sum_i 2^(s_i log2 e - m) v_i / sum_i 2^(s_i log2 e - m),  m the running maximum
//
// A tile is some rows (queries, token by token, of the heads that share a head of keys) and the keys that they see, taken 32 a
// step.  Of few rows (16 or 32 a tile) reading the cache is the cost, and the tile's four waves take its steps in turn, all with
// the same rows, and add their sums at the end; of many (64 to 256) the matrix cores' rate and what feeds them is, and each wave
// has rows of its own.  No wave waits for another before the end and nothing but what lanes hand each other passes through
// LDS on the way: the scores are computed transposed, S^T = K Q^T by mfma_f32_16x16x32_bf16, so that the lane that has four
// keys' scores of a query is the one whose operand of out^T = V^T P^T they are.  Orders of keys and columns are free as long
// as both products agree on them: key 16 t + 4 r + g is row 4 g + r of tile t, so that four neighbouring rows of the cache are
// read by one load, lane (g, c) has the g-th share of a row of keys (whole blocks, 128 columns and more) and the c-th sixteenth
// of four rows of values, whose pairs of keys v_perm puts next to each other.
// Codes become bfloat16 exactly by the scaled conversions, and float16 and float32 queries are taken as the sum of two and three
// bfloat16, so that the products are exact.  Weights are taken as three bfloat16 of float32 queries, which is all of them, and as
// two, all but 2^-16 of them, of others; of bfloat16 queries in tiles of many rows as one, as precise as their output
// (weight_planes_of).  The sum of weights is of the unrounded ones.
//
// Few rows: 64 sequences of 4 to 8 thousand keys (32 heads on 8, 128 columns, MXFP4, 429 MB): 116 us traced, 3.7 TB/s of the 5.2
// that a copy reaches, and 9 us of joining; one sequence of 131072: 40 us, 3.6 TB/s, and 8.  A step asks for its 32 keys a step
// ahead (two and three steps ahead gained nothing), which two workgroups a CU do not keep up with the memory's latency.
// Many rows: a prompt of 8192 tokens (32 heads on 8, 128 columns, MXFP8): 798 us, 690 TFLOP/s, of the 1350 of a large library
// product.  Of its cycles 73% issue vector instructions (286 a step of a wave's 32 rows: 96 make bfloat16 of the codes, 16 are
// exponentials at a quarter of the rate, 32 are the products, which keep the matrix cores busy for 27%).  Rows that share a
// step's conversions are as many as two waves a SIMD have registers for, or nearly (attend_rows): twice the rows with one wave
// took 2450 us.  Keys and values converted once for the four waves, in LDS, a barrier a step, were fewer instructions (223) and
// slower, 860 us, the waves waiting for each other.
#pragma once

#include "cache_common.h"

namespace mxq {

// PAGES16: pages of whole 16 rows that are less than 2^26 bytes apart: one page a tile of 16 keys, and a lane's place within it
// the same in every step.  64 sequences of 4096 keys take 72 us in pages of 16 and 85 in pages of 24.
// RT: sixteens of rows a wave; WR: waves with rows of their own; LINE: a piece of the line of tiles, not a tile by its number.
template <int FAM, int DT, int NB, bool PAGES16, int RT, int WR, bool LINE>
__global__ __launch_bounds__(64 * kWaves, attend_groups(DT, NB, RT)) void k_attend(AttendArgs a) {
  constexpr int P = kAttendPlanes<DT>, PW = weight_planes_of(DT, WR > 1), BB = FAM == kPairs ? 16 : 32;
  constexpr int KW = NB * BB / 16;                        // words of keys' codes a lane and tile of 16 keys
  constexpr int EW = FAM == kPairs ? 1 : 2;               // words of eight codes
  constexpr int VB = NB * BB / 16, VW = VB / 4 < EW ? EW : VB / 4;   // bytes and words of values' codes a lane and key
  constexpr int SW = NB == 8 ? 2 : 1;                     // words of a row's scales
  constexpr int OT = 2 * NB, DP = 32 * NB;                // tiles of out^T, columns
  constexpr int WK = kWaves / WR, ROWS = 16 * RT * WR;    // waves that share a row's keys; rows of a workgroup
  __shared__ __attribute__((aligned(16))) float sums[WK > 1 ? WK : 1][WK > 1 ? 16 : 1][WK > 1 ? DP + 4 : 1];
  __shared__ float tops[kWaves][16], weights[kWaves][16];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c = lane & 15, g = lane >> 4;
  const int D = a.c.head_dim;

  if constexpr (!LINE) {
    if (a.fill) fill_rows(a);
  }

  // this workgroup's piece of the line
  int piece = blockIdx.x;
  int64_t at = blockIdx.x, end_at = 0;
  double unit = 0.0;
  if constexpr (LINE) {
    Member own = member(a, lane, ROWS, 0.0);
    const Line line = line_of(a, ROWS, own);
    if ((int)blockIdx.x >= line.groups) return;
    // neighbouring pieces, which may share keys, on one of the card's eight parts
    if (line.groups == a.wanted) piece = (int)(blockIdx.x & 7) * (a.wanted >> 3) + (int)(blockIdx.x >> 3);
    at = line.begin(piece), end_at = line.begin(piece + 1), unit = line.unit;
  }
  Tile u = tile_of(a, ROWS, member(a, lane, ROWS, unit), unit, at, !LINE);
  for (bool first_part = true;; first_part = false) {
  if (u.b < 0) return;
  // this piece's share of the tile's weight
  const int64_t share_from = LINE ? at - u.first : 0, share_to = LINE && end_at - u.first < u.weight ? end_at - u.first : u.weight;
  const bool whole = !LINE || (share_from == 0 && share_to == u.weight);
  const int kv_head = u.head;
  const Sequence& s = u.s;
  const int rows = s.n * a.group, row0 = u.row * ROWS + (WR > 1 ? wave * 16 * RT : 0);   // of this wave

  // this lane's queries, and the keys they see: [lo, hi]
  auto first_key = [&](int t) {
    const int64_t f = (int64_t)s.length - s.n + t + 1 - a.a.window;
    return a.a.window && f > 0 ? (f < s.length ? (int)f : s.length) : 0;
  };
  auto last_key = [&](int t) { return a.a.causal ? s.length - s.n + t : s.length - 1; };
  int lo[RT], hi[RT];
  bf16x8 q[RT][P][NB];
  int64_t q_at[RT];
#pragma unroll
  for (int m = 0; m < RT; ++m) {
    const int row = row0 + 16 * m + c, held = row < rows ? row : rows - 1;
    const int token = (int)divu31(held, a.by_group), head = kv_head * a.group + held - token * a.group;
    lo[m] = row < rows ? first_key(token) : 1, hi[m] = row < rows ? last_key(token) : 0;
    q_at[m] = (int64_t)(s.start + token) * a.a.q_token + head * a.a.q_head;
  }
  auto q_column = [&](int i) { return NB == 2 ? 16 * g + 8 * i : 32 * (g + 4 * (i >> 2)) + 8 * (i & 3); };
  if (D & 7) {
#pragma unroll
    for (int m = 0; m < RT; ++m)
#pragma unroll
      for (int i = 0; i < NB; ++i) {
        bf16x8 p[P];
        load_query<DT>(a.q, q_at[m] + q_column(i), D - q_column(i), p);
#pragma unroll
        for (int j = 0; j < P; ++j) q[m][j][i] = p[j];
      }
  } else {
    // all on their way before the first is looked at
    Eight x[RT][NB];
#pragma unroll
    for (int m = 0; m < RT; ++m)
#pragma unroll
      for (int i = 0; i < NB; ++i) x[m][i] = load_eight(a.q, DT, q_at[m] + (q_column(i) < D ? q_column(i) : 0));
#pragma unroll
    for (int m = 0; m < RT; ++m)
#pragma unroll
      for (int i = 0; i < NB; ++i) {
        float f[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) f[k] = 0.0f;
        add_eight(f, x[m][i], DT);
#pragma unroll
        for (int k = 0; k < 8; ++k) f[k] = q_column(i) < D ? f[k] : 0.0f;
        bf16x8 p[P];
        planes_of(f, p);
#pragma unroll
        for (int j = 0; j < P; ++j) q[m][j][i] = p[j];
      }
  }
  const int end_row = row0 + 16 * RT < rows ? row0 + 16 * RT : rows;       // no row is this wave's where it is not past row0
  const int t_first = (int)divu31(row0 < rows ? row0 : rows - 1, a.by_group), t_last = (int)divu31((row0 < end_row ? end_row : rows) - 1, a.by_group);
  const int from = first_key(t_first), to = row0 < end_row ? last_key(t_last) + 1 : 0;   // some row sees them
  const int all_from = first_key(t_last), all_to = last_key(t_first) + 1;   // every row does

  f32x4 o[RT][OT];
  float top[RT], total[RT];
#pragma unroll
  for (int m = 0; m < RT; ++m) {
    top[m] = -__builtin_inff(), total[m] = 0.0f;
#pragma unroll
    for (int t = 0; t < OT; ++t) o[m][t] = f32x4{0, 0, 0, 0};
  }

  // of the tile's steps those that are this piece's and that some row of the wave sees, of which every WK-th is the wave's
  const int base = s.lo & ~(kStep - 1);
  int begin, end;
  {
    const int tile_last = (u.row + 1) * ROWS < rows ? (u.row + 1) * ROWS - 1 : rows - 1;
    const int tile_from = first_key((int)divu31(u.row * ROWS, a.by_group)), tile_to = last_key((int)divu31(tile_last, a.by_group)) + 1;
    const int low = (tile_from - base) / kStep, high = tile_to > tile_from ? (tile_to - base + kStep - 1) / kStep : low;
    const int sees_from = (from - base) / kStep, sees_to = to > from ? (to - base + kStep - 1) / kStep : 0;
    begin = low + steps_before(high - low, share_from, u.weight), end = low + steps_before(high - low, share_to, u.weight);
    begin = same(begin > sees_from ? begin : sees_from), end = same(end < sees_to ? end : sees_to);
  }
  const int mine = WK > 1 ? begin + wave : begin;

  // Where a lane reads within a row.  Keys: lane l asks for share l % 4 of tile row l / 4, so that four lanes read a row's
  // neighbouring bytes, and hands it to lane (l % 4, l / 4).  Values: the c-th sixteenth.  Scales: lane l those of key l % 32,
  // of values and, from lane 32 on, of keys.
  const int share = lane & 3, kbyte = NB == 2 ? share * (BB / 2) : share * BB, vblock = c * NB / 16;
  const bool kthere = (NB == 2 ? share >> 1 : share) < a.blocks, kthere2 = NB == 8 && share + 4 < a.blocks, vthere = vblock < a.blocks;
  const uint8_t *kc = a.kc + kv_head * a.c.head_stride[0], *ks = a.ks + kv_head * a.c.head_stride[1];
  const uint8_t *vc = a.vc + kv_head * a.c.head_stride[2], *vs = a.vs + kv_head * a.c.head_stride[3];
  const int32_t* table = a.table + (int64_t)u.b * a.a.table_row;
  // Codes and scales of the keys and values of a step, as they lie in memory, asked for a step ahead.
  struct Ahead {
    uint32_t kw[2][KW], sw[SW], vw[8][VW];
    uint32_t there;                                       // bit i: key i of this lane's eight
  };
  constexpr int first = NB == 8 ? KW / 2 : KW;            // words of keys' codes in one piece
  auto read_keys = [&](Ahead& b, int t, const uint8_t* p, uint32_t code) {
    if (a.blocks < NB) {
#pragma unroll
      for (int i = 0; i < KW; ++i) b.kw[t][i] = 0;
    }
    if (a.blocks == NB || kthere) __builtin_memcpy(&b.kw[t][0], p + code, 4 * first);
    if constexpr (NB == 8) {
      if (a.blocks == NB || kthere2) __builtin_memcpy(&b.kw[t][first], p + code + 4 * BB, 4 * first);
    }
  };
  auto read_scales = [&](Ahead& b, const uint8_t* p) {
    if (a.blocks == NB) {
      b.sw[0] = 0;
      __builtin_memcpy(&b.sw[0], p, NB);
    } else {
      b.sw[0] = p[0];
      if constexpr (NB == 8) b.sw[1] = 0;
#pragma unroll
      for (int i = 1; i < NB - 1; ++i)
        if (i < a.blocks) b.sw[i >> 2] |= (uint32_t)p[i] << 8 * (i & 3);
    }
  };
  // A lane's scale bytes of what lane `from` holds: of block `block`.
  auto scale_from = [&](const Ahead& b, int from, int block) {
    uint32_t w = (uint32_t)__builtin_amdgcn_ds_bpermute(4 * from, (int)b.sw[0]);
    if constexpr (NB == 8) {
      const uint32_t high = (uint32_t)__builtin_amdgcn_ds_bpermute(4 * from, (int)b.sw[1]);
      w = block & 4 ? high : w;
    }
    return w >> 8 * (block & 3) & 255u;
  };
  const uint32_t krow = 4 * ((lane >> 2) & 3) + (lane >> 4);
  // Where the 32 keys of a step lie.  PAGES16: each tile of 16 keys has a page; lane l finds tile l % 2 of this wave's step
  // l / 2 from `upto` on, 32 steps at once, and a lane's place within a tile is the same in every step; rows past the length
  // are read as they are, and masked.  Otherwise lane l finds key l % 32 of one step, whose page it asked for a step ahead,
  // and the others ask it.
  int64_t tile[4] = {0, 0, 0, 0};                         // bytes to a tile's first row, of each of the cache's tensors
  uint64_t tiles_there = 0;
  int upto = mine, page_ahead = 0;
  auto key_of = [&](int step) { return base + step * kStep + (PAGES16 ? 16 * (lane & 1) : lane & 31); };
  auto page_of = [&](int key) { return table[(int)divu31(key < s.length ? key : s.length - 1, a.by_page)]; };
  auto find_tiles = [&](int step) {
    const int key = key_of(step + (lane >> 1) * WK), page = page_of(key), k = key < s.length ? key : s.length - 1;
    const bool yes = key < s.length && (uint32_t)page < (uint32_t)a.c.pages;
    const int at = k - (int)divu31(k, a.by_page) * (int)a.c.page_size;
#pragma unroll
    for (int i = 0; i < 4; ++i) tile[i] = yes ? page * a.c.page_stride[i] + at * a.c.row_stride[i] : 0;
    tiles_there = __ballot(yes);
    upto = step;
  };
  auto tile_at = [&](int i, int l) {
    const uint32_t low = __builtin_amdgcn_readlane((int)(uint32_t)tile[i], l), high = __builtin_amdgcn_readlane((int)(uint32_t)(tile[i] >> 32), l);
    return (int64_t)((uint64_t)high << 32 | low);
  };
  struct Places {
    int lane;                                             // PAGES16: the first tile's
    int page, at;                                         // otherwise this lane's key's
    uint32_t there;
  };
  auto places_of = [&](int step) {
    Places p{};
    if constexpr (PAGES16) {
      if (step - upto >= 32 * WK) find_tiles(step);
      p.lane = (step - upto) / WK * 2;
      p.there = (uint32_t)(tiles_there >> p.lane) & 3u;
    } else {
      const int key = key_of(step), k = key < s.length ? key : s.length - 1;
      const bool yes = key < s.length && (uint32_t)page_ahead < (uint32_t)a.c.pages;
      p.page = yes ? page_ahead : 0;
      p.at = yes ? k - (int)divu31(k, a.by_page) * (int)a.c.page_size : 0;
      p.there = yes;
      page_ahead = page_of(key_of(step + WK));
    }
    return p;
  };
  const uint32_t kcode = (PAGES16 ? krow * (uint32_t)a.c.row_stride[0] : 0) + kbyte;
  // columns of blocks that a row does not have are not stored: the first block does for them
  const uint32_t vcode = (PAGES16 ? g * (uint32_t)a.c.row_stride[2] : 0) + (vthere ? c * VB : 0);
  const uint32_t vcode4 = 4 * (uint32_t)a.c.row_stride[2], scale_row = (lane & 15) * (uint32_t)a.c.row_stride[lane < 32 ? 3 : 1];
  auto load_keys = [&](Ahead& b, const Places& p) {
    if constexpr (PAGES16) {
#pragma unroll
      for (int t = 0; t < 2; ++t) read_keys(b, t, kc + tile_at(0, p.lane + t), kcode);
      const int64_t v0 = tile_at(3, p.lane), v1 = tile_at(3, p.lane + 1), k0 = tile_at(1, p.lane), k1 = tile_at(1, p.lane + 1);
      const uint8_t *vp = vs + (lane & 16 ? v1 : v0), *kp = ks + (lane & 16 ? k1 : k0);
      read_scales(b, (lane < 32 ? vp : kp) + scale_row);
    } else {
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const int page = __shfl(p.page, 16 * t + krow), at = __shfl(p.at, 16 * t + krow);
        read_keys(b, t, kc + page * a.c.page_stride[0] + at * a.c.row_stride[0], kcode);
      }
      read_scales(b, lane < 32 ? vs + p.page * a.c.page_stride[3] + p.at * a.c.row_stride[3] : ks + p.page * a.c.page_stride[1] + p.at * a.c.row_stride[1]);
    }
  };
  auto load_values = [&](Ahead& b, const Places& p) {
    b.there = 0;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      if constexpr (PAGES16) {
        b.there |= p.there >> t & 1 ? 0xFu << 4 * t : 0u;
        const uint8_t* code = vc + tile_at(2, p.lane + t);
#pragma unroll
        for (int r = 0; r < 4; ++r) __builtin_memcpy(&b.vw[4 * t + r][0], code + (vcode + r * vcode4), VB);
      } else {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int from = 16 * t + 4 * r + g, page = __shfl(p.page, from), at = __shfl(p.at, from);
          b.there |= (uint32_t)__shfl((int)p.there, from) << (4 * t + r);
          __builtin_memcpy(&b.vw[4 * t + r][0], vc + page * a.c.page_stride[2] + at * a.c.row_stride[2] + vcode, VB);
        }
      }
    }
  };

  // The scores of a step's keys once more, where one is NaN: a query's lower planes are zero where it has no more bits, and zero
  // times an infinite key is NaN, so infinite keys meet the first plane alone, the lower ones the largest finite value.  Seldom
  // needed, it takes the keys from memory again, eight columns at a time, so that no step holds registers for it.  Scores looked
  // at in every step, their keys kept, took 142 us where this takes 122 (64 single float32 tokens over 4096 keys, 256 columns of
  // E4M3) and 505 where it takes 470 (a float16 prompt of 4096, 128 columns).
  auto scores_with_care = [&](int k0, f32x4 (&z)[RT][2]) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int asked = k0 + 16 * t + 4 * (c & 3) + (c >> 2), key = asked < s.length ? asked : s.length - 1, of = page_of(key);
      const bool yes = (uint32_t)of < (uint32_t)a.c.pages;
      const int page = yes ? of : 0, at = yes ? key - (int)divu31(key, a.by_page) * (int)a.c.page_size : 0;
      const uint8_t *codes = kc + page * a.c.page_stride[0] + at * a.c.row_stride[0], *scales = ks + page * a.c.page_stride[1] + at * a.c.row_stride[1];
#pragma unroll
      for (int m = 0; m < RT; ++m) z[m][t] = f32x4{0, 0, 0, 0};
#pragma unroll
      for (int i = 0; i < NB; ++i) {
        uint32_t w[EW] = {}, scale = 0;
        if (q_column(i) / 32 < a.blocks) {
          __builtin_memcpy(w, codes + q_column(i) * BB / 32, BB / 4);
          scale = scales[q_column(i) / 32];
        }
        const bf16x8 k = eight_codes<FAM>(w, scale_field(scale));
        bf16x8 lower = k;
        finite_only(lower);
#pragma unroll
        for (int m = 0; m < RT; ++m)
#pragma unroll
          for (int p = P - 1; p >= 0; --p) z[m][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(p ? lower : k, q[m][p][i], z[m][t], 0, 0, 0);
      }
    }
  };

  Ahead ahead;
  if (begin < end) {                                      // there is a key, and so a page of it
    if constexpr (PAGES16) find_tiles(mine);
    else page_ahead = page_of(key_of(mine));
  }
#pragma unroll
  for (int k = 0; k < 8; ++k)
#pragma unroll
    for (int w = 0; w < VW; ++w) ahead.vw[k][w] = 0;
  if (mine < end) {
    const Places p = places_of(mine);
    load_keys(ahead, p);
    load_values(ahead, p);
  }
  for (int step = mine; step < end; step += WK) {
    const bool more = step + WK < end;
    const int k0 = base + step * kStep;
    uint32_t vsc[8];                                      // scale bytes of this lane's eight keys of values
    f32x4 z[RT][2];
    {
      uint32_t kw[2][KW], ksc[2][SW];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
#pragma unroll
        for (int i = 0; i < SW; ++i) ksc[t][i] = scale_from(ahead, 32 + 16 * t + 4 * (c & 3) + (c >> 2), NB == 2 ? g >> 1 : g + 4 * i);
#pragma unroll
        for (int i = 0; i < KW; ++i) kw[t][i] = (uint32_t)__builtin_amdgcn_ds_bpermute(4 * (4 * c + g), (int)ahead.kw[t][i]);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) vsc[i] = scale_from(ahead, 16 * (i >> 2) + 4 * (i & 3) + g, vblock);
#pragma unroll
      for (int m = 0; m < RT; ++m) z[m][0] = z[m][1] = f32x4{0, 0, 0, 0};
#pragma unroll
      for (int i = 0; i < NB; ++i) {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const bf16x8 k = eight_codes<FAM>(&kw[t][i * EW], scale_field(ksc[t][NB == 8 ? i >> 2 : 0]));
#pragma unroll
          for (int m = 0; m < RT; ++m)
#pragma unroll
            for (int p = P - 1; p >= 0; --p) z[m][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k, q[m][p][i], z[m][t], 0, 0, 0);
        }
      }
    }
    Places next{};
    if (more) {
      next = places_of(step + WK);
      load_keys(ahead, next);
    }

    const bool part = k0 < all_from || k0 + kStep > all_to || (PAGES16 ? ahead.there != 0xFF : __any(ahead.there != 0xFF));
    uint32_t seen[RT];
#pragma unroll
    for (int m = 0; m < RT; ++m) seen[m] = 0xFF;
    if (part) {
#pragma unroll
      for (int m = 0; m < RT; ++m) {
        seen[m] = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int key = k0 + 16 * (i >> 2) + 4 * (i & 3) + g;
          const bool yes = key >= lo[m] && key <= hi[m] && (ahead.there >> i & 1);
          seen[m] |= yes ? 1u << i : 0u;
          z[m][i >> 2][i & 3] = yes ? z[m][i >> 2][i & 3] : -__builtin_inff();
        }
      }
    }
    // The maximum follows only when a weight would pass 2^8: until then weights and sums are relative to an old one.  Of several
    // planes it is NaN where a score is.
    float most[RT];
    auto find_most = [&] {
      bool past = false;
#pragma unroll
      for (int m = 0; m < RT; ++m) {
        most[m] = z[m][0][0];
#pragma unroll
        for (int i = 1; i < 8; ++i)
          most[m] = P > 1 ? __builtin_elementwise_maximum(most[m], z[m][i >> 2][i & 3]) : __builtin_fmaxf(most[m], z[m][i >> 2][i & 3]);
        most[m] *= a.scale2;
        past |= P > 1 ? !(most[m] <= top[m] + 8.0f) : most[m] > top[m] + 8.0f;
      }
      return __any(past);
    };
    if (find_most()) {
      if constexpr (P > 1) {
        bool none = false;
#pragma unroll
        for (int m = 0; m < RT; ++m) none |= most[m] != most[m] && total[m] == total[m];   // a row that is NaN already stays it
        if (__builtin_expect(__any(none), 0)) {
          scores_with_care(k0, z);
#pragma unroll
          for (int m = 0; m < RT; ++m)
#pragma unroll
            for (int i = 0; i < 8; ++i) z[m][i >> 2][i & 3] = seen[m] >> i & 1 ? z[m][i >> 2][i & 3] : -__builtin_inff();
          find_most();
        }
      }
#pragma unroll
      for (int m = 0; m < RT; ++m) {
        most[m] = __builtin_fmaxf(most[m], __shfl_xor(most[m], 16));
        most[m] = __builtin_fmaxf(most[m], __shfl_xor(most[m], 32));
        const float now = __builtin_fmaxf(top[m], most[m]);
        const float factor = now == -__builtin_inff() ? 1.0f : __builtin_amdgcn_exp2f(top[m] - now);
        top[m] = now;
        total[m] *= factor;
#pragma unroll
        for (int t = 0; t < OT; ++t)
#pragma unroll
          for (int r = 0; r < 4; ++r) o[m][t][r] *= factor;
      }
    }
    bf16x8 pw[RT][PW];
#pragma unroll
    for (int m = 0; m < RT; ++m) {
      const float less = top[m] == -__builtin_inff() ? 0.0f : -top[m];
      float w[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        w[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(z[m][i >> 2][i & 3], a.scale2, less));
        total[m] += w[i];
      }
      weight_planes(w, pw[m]);
    }

    // Zero times infinity is no zero.  Where a key is hidden from some query, values that are no finite number are taken out,
    // and the sums of the queries that see one of them become NaN.
    if (part) {
      bool odd = false;
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int w = 0; w < VW; ++w) odd |= may_be_odd<FAM>(ahead.vw[i][w], vsc[i]);
      if (__any(odd)) {
        bf16x8 sw[RT];
#pragma unroll
        for (int m = 0; m < RT; ++m) {
          uint32_t sees[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) sees[i] = (seen[m] >> 2 * i & 1 ? 0x3F80u : 0u) | (seen[m] >> 2 * i & 2 ? 0x3F800000u : 0u);
          __builtin_memcpy(&sw[m], sees, 16);
        }
#pragma unroll
        for (int j = 0; j < OT / 2; ++j) {
          uint32_t x[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) x[i] = take_odd<FAM>(&ahead.vw[i][0], j, scale_field(vsc[i]));
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const bf16x8 v = keys_of_column(x, half);
#pragma unroll
            for (int m = 0; m < RT; ++m) {
              const f32x4 found = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, sw[m], f32x4{0, 0, 0, 0}, 0, 0, 0);
#pragma unroll
              for (int r = 0; r < 4; ++r) o[m][2 * j + half][r] = found[r] > 0.0f ? __builtin_nanf("") : o[m][2 * j + half][r];
            }
          }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) vsc[i] = vsc[i] == 255 ? 127 : vsc[i];        // whose codes are zeros now
      }
    }
#pragma unroll
    for (int j = 0; j < OT / 2; ++j) {
      uint32_t x[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = two_codes<FAM>(&ahead.vw[i][0], j, scale_field(vsc[i]));
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const bf16x8 v = keys_of_column(x, half);
#pragma unroll
        for (int m = 0; m < RT; ++m)
#pragma unroll
          for (int p = PW - 1; p >= 0; --p) o[m][2 * j + half] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, pw[m][p], o[m][2 * j + half], 0, 0, 0);
      }
    }
    if (more) load_values(ahead, next);
  }

#pragma unroll
  for (int m = 0; m < RT; ++m) {
    total[m] += __shfl_xor(total[m], 16);
    total[m] += __shfl_xor(total[m], 32);
    const int tile0 = row0 + 16 * m;                        // these rows' first
    // where row r of these 16 goes: the output's row, or the place of its part
    auto out_row = [&](int r) {
      const int t = (int)divu31(tile0 + r, a.by_group);
      return (int64_t)(s.start + t) * a.a.heads + kv_head * a.group + tile0 + r - t * a.group;
    };
    auto part_row = [&](int r) {
      return a.partial + (part_slot(piece, first_part) * ROWS + (WR > 1 ? wave * 16 * RT : 0) + 16 * m + r) * (DP + 2);
    };
    if constexpr (WK == 1) {
      if (tile0 + c >= rows) continue;
      const float inv = total[m] == 0.0f ? 0.0f : 1.0f / total[m];
      const int d0 = 4 * OT * g;
      if (whole) {
        const int64_t row = out_row(c);
#pragma unroll
        for (int e = 0; e < 4 * OT; e += 4) {
          float v[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) v[k] = o[m][(e + k) % OT][(e + k) / OT] * inv;
          store_four<DT>(a.out, row * D + d0 + e, D - d0 - e, v);
        }
        if (a.lse && g == 0) a.lse[row] = log_sum(top[m], total[m]);
      } else {
        float* part = part_row(c);
#pragma unroll
        for (int e = 0; e < 4 * OT; e += 2) {
          const float v[2] = {o[m][e % OT][e / OT], o[m][(e + 1) % OT][(e + 1) / OT]};
          __builtin_memcpy(part + d0 + e, v, 8);
        }
        if (g == 0) part[DP] = top[m], part[DP + 1] = total[m];
      }
    } else {
      // the waves' sums, relative to the largest of their maxima, in the order of the waves
      if (m || !first_part) __syncthreads();                // what the last round left has been read
      if (g == 0) tops[wave][c] = top[m], weights[wave][c] = total[m];
#pragma unroll
      for (int t = 0; t < OT; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) sums[wave][c][OT * (4 * g + r) + t] = o[m][t][r];
      __syncthreads();
      const int r = threadIdx.x >> 4, d0 = 4 * (threadIdx.x & 15);
      if (tile0 + r >= rows) continue;
      float best = tops[0][r], all = 0.0f, factor[WK];
#pragma unroll
      for (int w = 1; w < WK; ++w) best = __builtin_fmaxf(best, tops[w][r]);
#pragma unroll
      for (int w = 0; w < WK; ++w) {
        // a wave without a maximum has seen no key, or only scores of NaN, which its sum is then
        factor[w] = tops[w][r] == -__builtin_inff() ? weights[w][r] : __builtin_amdgcn_exp2f(tops[w][r] - best);
        all += tops[w][r] == -__builtin_inff() ? weights[w][r] : factor[w] * weights[w][r];
      }
      const float inv = all == 0.0f ? 0.0f : 1.0f / all;
      const int64_t row = out_row(r);
      float* part = part_row(r);
#pragma unroll
      for (int d = d0; d < DP; d += 64) {
        float v[4] = {0, 0, 0, 0};
#pragma unroll
        for (int w = 0; w < WK; ++w)
#pragma unroll
          for (int k = 0; k < 4; ++k) v[k] += factor[w] * sums[w][r][d + k];    // a factor of zero too: NaN stays NaN
        if (!whole) {
          __builtin_memcpy(part + d, v, 16);
        } else if (d < D) {
#pragma unroll
          for (int k = 0; k < 4; ++k) v[k] *= inv;
          store_four<DT>(a.out, row * D + d, D - d, v);
        }
      }
      if (d0 == 0) {
        if (!whole) part[DP] = best, part[DP + 1] = all;
        else if (a.lse) a.lse[row] = log_sum(best, all);
      }
    }
  }
  if constexpr (!LINE) return;
  at = u.first + u.weight;
  if (at >= end_at) return;
  u = next_tile(a, ROWS, unit, u);
  }
}

template <int FAM, int DT, int NB, int RT, int WR> void launch_attend_of(const AttendArgs& a, int64_t groups, hipStream_t st) {
  const dim3 grid((unsigned)groups), block(64 * kWaves);
  if (a.aligned && a.partial) k_attend<FAM, DT, NB, true, RT, WR, true><<<grid, block, 0, st>>>(a);
  else if (a.aligned) k_attend<FAM, DT, NB, true, RT, WR, false><<<grid, block, 0, st>>>(a);
  else if (a.partial) k_attend<FAM, DT, NB, false, RT, WR, true><<<grid, block, 0, st>>>(a);
  else k_attend<FAM, DT, NB, false, RT, WR, false><<<grid, block, 0, st>>>(a);
}
// many: tiles of many rows; wide: few queries' rows are 32.
template <int FAM, int DT, int NB> void launch_attend_by(const AttendArgs& a, bool many, bool wide, int64_t groups, hipStream_t st) {
  if (many) launch_attend_of<FAM, DT, NB, attend_rows(DT, NB), kWaves>(a, groups, st);
  else if (NB < 8 && wide) launch_attend_of<FAM, DT, NB < 8 ? NB : 4, 2, 1>(a, groups, st);
  else launch_attend_of<FAM, DT, NB, 1, 1>(a, groups, st);
}
template <int FAM, int DT> void launch_attend(const AttendArgs& a, bool many, bool wide, int64_t groups, hipStream_t st) {
  if (a.blocks <= 2) launch_attend_by<FAM, DT, 2>(a, many, wide, groups, st);
  else if (a.blocks <= 4) launch_attend_by<FAM, DT, 4>(a, many, wide, groups, st);
  else launch_attend_by<FAM, DT, 8>(a, many, wide, groups, st);
}

}  // namespace mxq
