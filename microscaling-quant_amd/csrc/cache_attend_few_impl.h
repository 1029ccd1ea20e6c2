// Attention of few queries over a cache in MX formats: reading the cache is what it costs.
//
//   s = scale q k^T;  out = sum_i 2^(s_i log2 e - m) v_i / sum_i 2^(s_i log2 e - m),  m the running maximum
//
// A workgroup takes 16 rows (queries of the heads that share a head of keys) and a run of keys, its four waves 32 keys in
// turn.  No wave waits for another before the end and nothing passes through LDS on the way: the scores are computed
// transposed, S^T = K Q^T by mfma_f32_16x16x32_bf16, so that the lane that has four keys' scores of a query is the one whose
// operand of out^T = V^T P^T they are.  Orders of keys and columns are free as long as both products agree on them: key
// 16 t + 4 r + g is row 4 g + r of tile t, so that four neighbouring rows of the cache are read by one load, lane (g, c) has
// the g-th share of a row of keys (whole blocks, 128 columns and more) and the c-th sixteenth of four rows of values,
// whose pairs of keys v_perm puts next to each other.
// Codes become bfloat16 exactly by the scaled conversions; float16 and float32 queries and their weights are taken as the
// sum of two and three bfloat16.
#pragma once

#include "cache_common.h"

namespace mxq {

constexpr int kFewRows = 16, kFewWaves = 4;

// PAGES16: pages of whole 16 rows that are less than 2^26 bytes apart.

template <int FAM, int DT, int NB, bool PAGES16>
__global__ __launch_bounds__(64 * kFewWaves, few_groups(DT, NB)) void k_attend_few(AttendArgs a, int least) {
  constexpr int P = kAttendPlanes<DT>, BB = FAM == kPairs ? 16 : 32;
  constexpr int KW = NB * BB / 16;                        // words of keys' codes a lane and tile of 16 keys
  constexpr int EW = FAM == kPairs ? 1 : 2;               // words of eight codes
  constexpr int VB = NB * BB / 16, VW = VB / 4 < EW ? EW : VB / 4;   // bytes and words of values' codes a lane and key
  constexpr int DEPTH = few_depth(DT, NB);                // steps asked for ahead
  constexpr int SW = NB == 8 ? 2 : 1;                     // words of a row's scales
  constexpr int OT = 2 * NB, DP = 32 * NB;                // tiles of out^T, columns
  __shared__ float sums[kFewWaves][16][DP + 4];
  __shared__ float tops[kFewWaves][16], weights[kFewWaves][16];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c = lane & 15, g = lane >> 4;

  int64_t at_step = 0, end_step = 0;
  if (a.partial) {
    const Line line = line_of(a, kFewRows, least);
    if ((int)blockIdx.x >= line.groups) return;
    at_step = line.begin(blockIdx.x), end_step = line.begin(blockIdx.x + 1);
  }
  for (bool first_part = true;; first_part = false) {
  const Tile u = tile_of(a, kFewRows, a.partial ? at_step : blockIdx.x, !a.partial);
  if (u.b < 0) return;
  const int begin_step = a.partial ? (int)(at_step - u.first) : 0;
  const int stop_step = a.partial && end_step - u.first < u.steps ? (int)(end_step - u.first) : u.steps;
  const Sequence s = same(sequence(a, u.b));
  const int rows = s.n * a.group, row_tiles = (rows + kFewRows - 1) / kFewRows, kv_head = u.index / row_tiles;
  const int row0 = (u.index - kv_head * row_tiles) * kFewRows;
  const int D = a.c.head_dim;

  // this lane's query, and the keys it sees: [lo, hi]
  const int row = row0 + c, token = (int)divu31(row < rows ? row : rows - 1, a.by_group), last_row = row0 + 15 < rows ? row0 + 15 : rows - 1;
  const int head = kv_head * a.group + (row < rows ? row : rows - 1) - token * a.group;
  auto first_key = [&](int t) {
    const int64_t f = (int64_t)s.length - s.n + t + 1 - a.a.window;
    return a.a.window && f > 0 ? (f < s.length ? (int)f : s.length) : 0;
  };
  auto last_key = [&](int t) { return a.a.causal ? s.length - s.n + t : s.length - 1; };
  const int lo = row < rows ? first_key(token) : 1, hi = row < rows ? last_key(token) : 0;
  const int t_first = (int)divu31(row0, a.by_group), t_last = (int)divu31(last_row, a.by_group);
  const int from = first_key(t_first), to = last_key(t_last) + 1;   // some row sees them
  const int all_from = first_key(t_last), all_to = last_key(t_first) + 1;   // every row does

  bf16x8 q[P][NB];
  {
    const int64_t at = (int64_t)(s.start + token) * a.a.q_token + head * a.a.q_head;
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      const int d = NB == 2 ? 16 * g + 8 * i : 32 * (g + 4 * (i >> 2)) + 8 * (i & 3);
      bf16x8 p[P];
      load_query<DT>(a.q, at + d, row < rows ? D - d : 0, p);
#pragma unroll
      for (int j = 0; j < P; ++j) q[j][i] = p[j];
    }
  }

  f32x4 o[OT];
#pragma unroll
  for (int t = 0; t < OT; ++t) o[t] = f32x4{0, 0, 0, 0};
  float top = -__builtin_inff(), total = 0.0f;

  // this part's steps that some row sees, of which every kFewWaves-th is this wave's
  const int base = s.lo & ~(kStep - 1), sees_from = (from - base) / kStep, sees_to = to > base ? (to - base + kStep - 1) / kStep : 0;
  const int begin = same(begin_step > sees_from ? begin_step : sees_from), end = same(to > from ? (stop_step < sees_to ? stop_step : sees_to) : 0);

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
  int upto = begin + wave, page_ahead = 0;
  auto key_of = [&](int step) { return base + step * kStep + (PAGES16 ? 16 * (lane & 1) : lane & 31); };
  auto page_of = [&](int key) { return table[(int)divu31(key < s.length ? key : s.length - 1, a.by_page)]; };
  auto find_tiles = [&](int step) {
    const int key = key_of(step + (lane >> 1) * kFewWaves), page = page_of(key), k = key < s.length ? key : s.length - 1;
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
      if (step - upto >= 32 * kFewWaves) find_tiles(step);
      p.lane = (step - upto) / kFewWaves * 2;
      p.there = (uint32_t)(tiles_there >> p.lane) & 3u;
    } else {
      const int key = key_of(step), k = key < s.length ? key : s.length - 1;
      const bool yes = key < s.length && (uint32_t)page_ahead < (uint32_t)a.c.pages;
      p.page = yes ? page_ahead : 0;
      p.at = yes ? k - (int)divu31(k, a.by_page) * (int)a.c.page_size : 0;
      p.there = yes;
      page_ahead = page_of(key_of(step + kFewWaves));
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

  Ahead ahead[DEPTH];
  if (begin < end) {                                      // there is a key, and so a page of it
    if constexpr (PAGES16) find_tiles(begin + wave);
    else page_ahead = page_of(key_of(begin + wave));
  }
#pragma unroll
  for (int i = 0; i < DEPTH; ++i) {
#pragma unroll
    for (int k = 0; k < 8; ++k)
#pragma unroll
      for (int w = 0; w < VW; ++w) ahead[i].vw[k][w] = 0;
    const int step = begin + wave + i * kFewWaves;
    if (step < end) {
      const Places p = places_of(step);
      load_keys(ahead[i], p);
      load_values(ahead[i], p);
    }
  }
  auto body = [&](Ahead& b, int step) {
    const bool more = step + DEPTH * kFewWaves < end;
    const int k0 = base + step * kStep;
    uint32_t vsc[8];                                      // scale bytes of this lane's eight keys of values
    f32x4 z[2];
    z[0] = z[1] = f32x4{0, 0, 0, 0};
    {
      uint32_t kw[2][KW], ksc[2][SW];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
#pragma unroll
        for (int i = 0; i < SW; ++i) ksc[t][i] = scale_from(b, 32 + 16 * t + 4 * (c & 3) + (c >> 2), NB == 2 ? g >> 1 : g + 4 * i);
#pragma unroll
        for (int i = 0; i < KW; ++i) kw[t][i] = (uint32_t)__builtin_amdgcn_ds_bpermute(4 * (4 * c + g), (int)b.kw[t][i]);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) vsc[i] = scale_from(b, 16 * (i >> 2) + 4 * (i & 3) + g, vblock);
#pragma unroll
      for (int i = 0; i < NB; ++i) {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const bf16x8 k = eight_codes<FAM>(&kw[t][i * EW], scale_field(ksc[t][NB == 8 ? i >> 2 : 0]));
#pragma unroll
          for (int p = P - 1; p >= 0; --p) z[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k, q[p][i], z[t], 0, 0, 0);
        }
      }
    }
    Places next{};
    if (more) {
      next = places_of(step + DEPTH * kFewWaves);
      load_keys(b, next);
    }

    const bool part = k0 < all_from || k0 + kStep > all_to || (PAGES16 ? b.there != 0xFF : __any(b.there != 0xFF));
    uint32_t seen = 0xFF;
    if (part) {
      seen = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int key = k0 + 16 * (i >> 2) + 4 * (i & 3) + g;
        const bool yes = key >= lo && key <= hi && (b.there >> i & 1);
        seen |= yes ? 1u << i : 0u;
        z[i >> 2][i & 3] = yes ? z[i >> 2][i & 3] : -__builtin_inff();
      }
    }
    float most = z[0][0];
#pragma unroll
    for (int i = 1; i < 8; ++i) most = __builtin_fmaxf(most, z[i >> 2][i & 3]);
    most *= a.scale2;
    // The maximum follows only when a weight would pass 2^8: until then weights and sums are relative to an old one.
    if (__any(most > top + 8.0f)) {
      most = __builtin_fmaxf(most, __shfl_xor(most, 16));
      most = __builtin_fmaxf(most, __shfl_xor(most, 32));
      const float now = __builtin_fmaxf(top, most);
      const float factor = now == -__builtin_inff() ? 1.0f : __builtin_amdgcn_exp2f(top - now);
      top = now;
      total *= factor;
#pragma unroll
      for (int t = 0; t < OT; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) o[t][r] *= factor;
    }
    const float less = top == -__builtin_inff() ? 0.0f : -top;
    float w[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      w[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(z[i >> 2][i & 3], a.scale2, less));
      total += w[i];
    }
    bf16x8 pw[P];
    planes_of(w, pw);

    // Zero times infinity is no zero.  Where a key is hidden from some query, values that are no finite number are taken out,
    // and the sums of the queries that see one of them become NaN.
    if (part) {
      bool odd = false;
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int w = 0; w < VW; ++w) odd |= may_be_odd<FAM>(b.vw[i][w], vsc[i]);
      if (__any(odd)) {
        uint32_t sees[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) sees[i] = (seen >> 2 * i & 1 ? 0x3F80u : 0u) | (seen >> 2 * i & 2 ? 0x3F800000u : 0u);
        bf16x8 sw;
        __builtin_memcpy(&sw, sees, 16);
#pragma unroll
        for (int j = 0; j < OT / 2; ++j) {
          uint32_t x[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) x[i] = take_odd<FAM>(&b.vw[i][0], j, scale_field(vsc[i]));
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const f32x4 found = __builtin_amdgcn_mfma_f32_16x16x32_bf16(keys_of_column(x, half), sw, f32x4{0, 0, 0, 0}, 0, 0, 0);
#pragma unroll
            for (int r = 0; r < 4; ++r) o[2 * j + half][r] = found[r] > 0.0f ? __builtin_nanf("") : o[2 * j + half][r];
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
      for (int i = 0; i < 8; ++i) x[i] = two_codes<FAM>(&b.vw[i][0], j, scale_field(vsc[i]));
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const bf16x8 v = keys_of_column(x, half);
#pragma unroll
        for (int p = P - 1; p >= 0; --p) o[2 * j + half] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, pw[p], o[2 * j + half], 0, 0, 0);
      }
    }
    if (more) load_values(b, next);
  };
  for (int step = begin + wave; step < end; step += DEPTH * kFewWaves) {
    body(ahead[0], step);
#pragma unroll
    for (int i = 1; i < DEPTH; ++i)
      if (step + i * kFewWaves < end) body(ahead[i], step + i * kFewWaves);
  }

  // the waves' sums, relative to the largest of their maxima, in the order of the waves
  total += __shfl_xor(total, 16);
  total += __shfl_xor(total, 32);
  if (g == 0) tops[wave][c] = top, weights[wave][c] = total;
#pragma unroll
  for (int t = 0; t < OT; ++t)
#pragma unroll
    for (int r = 0; r < 4; ++r) sums[wave][c][OT * (4 * g + r) + t] = o[t][r];
  __syncthreads();
  const int r = threadIdx.x >> 4, d0 = threadIdx.x & 15;
  const bool whole = begin_step == 0 && stop_step == u.steps;
  if (row0 + r < rows) {
  float best = tops[0][r], all = 0.0f, factor[kFewWaves];
#pragma unroll
  for (int w = 1; w < kFewWaves; ++w) best = __builtin_fmaxf(best, tops[w][r]);
#pragma unroll
  for (int w = 0; w < kFewWaves; ++w) {
    factor[w] = tops[w][r] == -__builtin_inff() ? (weights[w][r] == 0.0f ? 0.0f : weights[w][r]) : __builtin_amdgcn_exp2f(tops[w][r] - best);
    all += tops[w][r] == -__builtin_inff() ? weights[w][r] : factor[w] * weights[w][r];
  }
  const int t = (int)divu31(row0 + r, a.by_group), h = kv_head * a.group + row0 + r - t * a.group;
  const int64_t out_row = (int64_t)(s.start + t) * a.a.heads + h;
  float* part = a.partial + (part_slot(blockIdx.x, first_part) * kFewRows + r) * (DP + 2);
  const float inv = all == 0.0f ? 0.0f : 1.0f / all;
  for (int d = d0; d < D; d += 16) {
    float v = 0.0f;
#pragma unroll
    for (int w = 0; w < kFewWaves; ++w) v += factor[w] == 0.0f ? 0.0f : factor[w] * sums[w][r][d];
    if (whole) store_elem(a.out, DT, out_row * D + d, v * inv);
    else part[d] = v;
  }
  if (d0 == 0) {
    if (!whole) part[DP] = best, part[DP + 1] = all;
    else if (a.lse) a.lse[out_row] = log_sum(best, all);
  }
  }
  if (!a.partial) return;
  at_step = u.first + stop_step;
  if (at_step >= end_step) return;
  __syncthreads();
  }
}

template <int FAM, int DT, int NB> void launch_attend_few_of(const AttendArgs& a, int64_t tiles, int least, hipStream_t st) {
  const dim3 grid((unsigned)(a.partial ? a.wanted : tiles)), block(64 * kFewWaves);
  if (a.aligned) k_attend_few<FAM, DT, NB, true><<<grid, block, 0, st>>>(a, least);
  else k_attend_few<FAM, DT, NB, false><<<grid, block, 0, st>>>(a, least);
}
template <int FAM, int DT> void launch_attend_few_by(const AttendArgs& a, int64_t tiles, int least, hipStream_t st) {
  if (a.blocks <= 2) launch_attend_few_of<FAM, DT, 2>(a, tiles, least, st);
  else if (a.blocks <= 4) launch_attend_few_of<FAM, DT, 4>(a, tiles, least, st);
  else launch_attend_few_of<FAM, DT, 8>(a, tiles, least, st);
}
template <int FAM> void launch_attend_few(const AttendArgs& a, int64_t tiles, int least, hipStream_t st) {
  if (a.a.dtype == MXQ_DT_F32) launch_attend_few_by<FAM, MXQ_DT_F32>(a, tiles, least, st);
  else if (a.a.dtype == MXQ_DT_BF16) launch_attend_few_by<FAM, MXQ_DT_BF16>(a, tiles, least, st);
  else launch_attend_few_by<FAM, MXQ_DT_F16>(a, tiles, least, st);
}

}  // namespace mxq
