// Products of many rows with packed weights on the matrix cores.
//
// A workgroup owns BM rows of x by BN rows of the weight and goes through the contraction 64 columns at a time.  x (64
// bfloat16, 128 bytes a row) and the codes (64 or 32 bytes a row) come straight from global memory into LDS, three stages
// deep: while one is multiplied the next has landed and the third is on its way.  The codes stay codes in LDS, half the
// bytes, and become bfloat16 when a wave takes its operands: one conversion for two values with their scale, beside the
// matrix instructions.  Lane (r, h) takes block h of row r's 64 columns, so a lane's 32 codes share one scale.
// Chunks of 16 bytes are permuted within a row by its number, so that the sixteen rows an LDS cycle pair reads lie in
// different ones of the 64 banks.
// float16 and float32 activations have been split into bfloat16 planes one after another along a longer row: the walk
// goes through the weight, and converts it, once a plane.
//
// Measured, 8192 x 8192 x 4096 in E4M3 on 256 x 256: 436 us without an epilogue (1.26 PFLOP/s, what the library's product of
// bfloat16 weights reaches here), 488 with bias, gelu and residual.  The matrix pipes are busy for 524 K of 905 K cycles at
// 1.7 GHz; alone, the products of a 64-column step take 1.0 us, its loads 0.9 (0.4 where they hit the first cache), both
// together 1.5.  4096 x 4096 x 4096, a call, in E4M3, E5M2, E3M2 and MXFP4's pairs: bfloat16 114 and 116 (E4M3, pairs),
// float16 234, 236, 245, 221, float32 348, 358, 370, 336.  Tried and slower: four waves of 128 x 128 (no second wave to fill a wait), two halves of waves taking turns
// at products and loads, waves of 64 x 128, codes by whole lines of 128 columns two stages deep.
#pragma once

#include <type_traits>

#include "packed_linear_common.h"

namespace mxq {

__device__ __forceinline__ uint32_t lds_offset(const void* p) {
  return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const void*)p;
}
// Global memory straight into LDS, 16 or 4 bytes a lane, lane i's at base + 16 i or 4 i.  Written as
// assembly because the compiler would wait for all such loads before every LDS read; the waits are the kernel's.  m0 is
// reserved: the compiler keeps nothing in it, and warns of undefined behaviour where it is named as overwritten.
__device__ __forceinline__ void dma16(uint32_t base, const void* p) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(base), "v"(p) : "memory");
}

__device__ __forceinline__ void dma16(uint32_t to, const void* base, uint32_t offset) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(to), "v"(offset), "s"(base) : "memory");
}
__device__ __forceinline__ void dma4(uint32_t base, const void* p) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" ::"s"(base), "v"(p) : "memory");
}

// What a chunk past the last column is loaded from.
static __device__ const u32x4 kNothing = {0, 0, 0, 0};

// FAM: code family; WIDE: activations of several planes; BM x BN rows; WM x WN of 32 x 32 tiles a wave; STAGES of 64 columns in LDS; FAR: a tile's rows lie 2^32
// bytes apart or more.
template <int FAM, bool WIDE, int BM, int BN, int WM, int WN, int STAGES, bool FAR>
__global__ __launch_bounds__(64 * (BM / (32 * WM)) * (BN / (32 * WN)), 2) void k_linear_tile(TileArgs ta) {
  constexpr int WAVES_N = BN / (32 * WN), WAVES = BM / (32 * WM) * WAVES_N, THREADS = 64 * WAVES;
  constexpr int WB = 2 * kBlockBytes<FAM>, CH = WB / 16;                 // a weight row's bytes and chunks of one stage
  constexpr int XL = BM * 8 / THREADS, WL = BN * CH / THREADS;   // loads a thread and stage
  constexpr int SC = BN * 4 / THREADS;                                   // loads of scales a thread and eight steps
  static_assert(WN == 2, "a wave's two tiles are neighbours, or G's and U's of the same outputs");
  static_assert(XL >= 2 && WL >= 1 && SC >= 1 && BM * 8 % THREADS == 0, "whole loads");
  struct Stage {
    uint8_t x[BM * 128];
    uint8_t w[BN * WB];
  };
  constexpr int kScales = 2 * BN * 16;                                   // a ring of two times eight steps' scale bytes
  constexpr int PITCH = 32 * WN + 4;
  constexpr int kHeld = WM < 2 ? WM : 2;                                 // 32-row pieces of a wave's sums in LDS at a time
  constexpr size_t kEpilogue = (size_t)WAVES * kHeld * 32 * PITCH * 4, kStages = STAGES * sizeof(Stage) + kScales;
  __shared__ __attribute__((aligned(16))) uint8_t memory[kStages > kEpilogue ? kStages : kEpilogue];
  Stage* stage = (Stage*)memory;
  uint8_t* scale_ring = memory + STAGES * sizeof(Stage);

  const LinearArgs& a = ta.l;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r = lane & 31, h = lane >> 5, wm = wave / WAVES_N, wn = wave % WAVES_N;
  const bool gated = a.sp.gated;
  const int outputs = gated ? BN / 2 : BN;

  // Consecutive workgroups go to the eight XCDs in turn; each XCD gets a run of tiles, in strips of eight row tiles, so
  // that what its L2 holds serves its neighbours.
  const int total = ta.tiles_m * ta.tiles_n;
  int at = blockIdx.x;
  {
    const int xcd = at & 7, local = at >> 3, base = total >> 3, more = total & 7;
    at = xcd * base + (xcd < more ? xcd : more) + local;
  }
  const int strip = at / (8 * ta.tiles_n), in = at - strip * 8 * ta.tiles_n;
  const int deep = ta.tiles_m - strip * 8 < 8 ? ta.tiles_m - strip * 8 : 8;
  const int tile_n = in / deep;
  const RowTile t = row_tile(a, BM, strip * 8 + in % deep);
  if (t.expert < 0) return;
  const int64_t n0 = (int64_t)tile_n * outputs;

  // the weight row of LDS row q; gated: of every 64 rows the first 32 from G, the others the same outputs' from U
  auto weight_row = [&](int q) {
    int64_t n = gated ? n0 + (q >> 6) * 32 + (q & 31) : n0 + q;
    if (n >= a.N) n = a.N - 1;
    return gated && (q & 32) ? n + a.N : n;
  };

  f32x16 acc[WN][WM];
#pragma unroll
  for (int i = 0; i < WN; ++i)
#pragma unroll
    for (int m = 0; m < WM; ++m)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][m][e] = 0.0f;

  const int all = ta.steps * ta.planes, per = ((all + ta.split - 1) / ta.split + 1) & ~1;         // even: a word of scales is two steps'
  const int first = (int)blockIdx.y * per, last = first + per < all ? first + per : all;

  if (!t.zeros && first < last) {
    // A row's place from a scalar base, 32 bits of offset a lane where they suffice: a step then costs scalar additions only.
    typedef typename std::conditional<FAR, int64_t, uint32_t>::type Offset;
    Offset xo[XL], wo[WL], so[SC];
    const uint8_t* x = (const uint8_t*)(ta.x + (a.sp.top_k ? 0 : t.row0 * ta.ld_x));
    const uint8_t* codes = a.codes + t.expert * a.sp.batch_codes + n0 * a.sp.ld_codes;
    const uint8_t* scales = a.scales + t.expert * a.sp.batch_scales + n0 * a.sp.ld_scales;
    const int xc = (tid & 7) ^ (tid >> 4 & 7);                           // this thread's chunk of a row, the same in all its rows
    const int wc = (tid % CH) ^ (CH == 4 ? tid >> 4 & 3 : tid >> 4 & 1);
#pragma unroll
    for (int i = 0; i < XL; ++i) {
      const int row = (i * THREADS + tid) >> 3, r = row < t.rows ? row : t.rows - 1;
      xo[i] = (Offset)((a.sp.top_k ? x_row(a, t.row0 + r) : r) * ta.ld_x * 2 + xc * 16);
    }
#pragma unroll
    for (int i = 0; i < WL; ++i) wo[i] = (Offset)((weight_row((i * THREADS + tid) / CH) - n0) * a.sp.ld_codes + wc * 16);
#pragma unroll
    for (int i = 0; i < SC; ++i) so[i] = (Offset)((weight_row((i * THREADS + tid) >> 2) - n0) * a.sp.ld_scales);

    auto load = [&](uint32_t to, const uint8_t* base, Offset offset) {
      if constexpr (FAR) dma16(to, base + offset);
      else dma16(to, base, offset);
    };
    // A third of the next step's loads into stage b, in the order codes and scales, x, x: loads of a step issued at once
    // would keep the wave from its multiplications while the memory pipeline takes them.  The last step again after it, so
    // that every step waits for as many loads.
    int st = first, k = first % ta.steps;
    auto issue = [&](int b, int part) {
      const uint8_t* nothing = (const uint8_t*)&kNothing;
      if (part == 1 || part == 2) {
        const uint32_t to = lds_offset(stage[b].x) + wave * 1024;
        const uint8_t* from = x + (int64_t)st * 128;
        if (k * 64 + 64 <= ta.x_columns) {
#pragma unroll
          for (int i = (part - 1) * (XL / 2); i < part * (XL / 2); ++i) load(to + i * THREADS * 16, from, xo[i]);
        } else {
          const bool past = k * 64 + xc * 8 >= ta.x_columns;
#pragma unroll
          for (int i = (part - 1) * (XL / 2); i < part * (XL / 2); ++i) dma16(to + i * THREADS * 16, past ? nothing : from + xo[i]);
        }
        return;
      }
      const int chunk = st - first;
      if ((chunk & 7) == 0) {
        const uint32_t to = lds_offset(scale_ring) + (chunk >> 3 & 1) * BN * 16 + wave * 256;
        const int two = (k + 2 * (tid & 3)) % ta.steps;
#pragma unroll
        for (int i = 0; i < SC; ++i) dma4(to + i * THREADS * 4, scales + so[i] + two * 2);
      }
      const uint32_t to = lds_offset(stage[b].w) + wave * 1024;
      const uint8_t* from = codes + (int64_t)k * WB;
      if (k * 64 + 64 <= ta.w_columns) {
#pragma unroll
        for (int i = 0; i < WL; ++i) load(to + i * THREADS * 16, from, wo[i]);
      } else {
        const bool past = k * 64 + wc * (FAM == kPairs ? 32 : 16) >= ta.w_columns;
#pragma unroll
        for (int i = 0; i < WL; ++i) dma16(to + i * THREADS * 16, past ? nothing : from + wo[i]);
      }
    };
    auto advance = [&]() {
      if (st + 1 < last) ++st, k = k + 1 == ta.steps ? 0 : k + 1;
    };
    // the later stages' loads, without the scales that come before them every eighth time: the waits below then ask for a little
    // more than they need
    constexpr int kInFlight = (STAGES - 2) * (XL + WL);
    auto read_codes = [&](int b, int st, uint32_t (&code)[WN][kWords<FAM>], float (&scale)[WN], uint32_t (&left)[WN]) {
#pragma unroll
      for (int i = 0; i < WN; ++i) {
        const int row = (wn * WN + i) * 32 + r, since = st - first;
#pragma unroll
        for (int c = 0; c < kWords<FAM> / 4; ++c) {
          const int chunk = h * (CH / 2) + c;
          const u32x4 v = *(const u32x4*)&stage[b].w[row * WB + (chunk ^ (CH == 4 ? row >> 2 & 3 : row >> 3 & 1)) * 16];
          __builtin_memcpy(&code[i][4 * c], &v, 16);
        }
        const uint8_t* at = scale_ring + (since >> 3 & 1) * BN * 16 + row * 16 + (since & 7) * 2 + h;
        scale[i] = scale_of<FAM>(*at, code[i], ta.map, left[i], WIDE && st >= ta.steps);
      }
    };
    auto read_x = [&](int b, int j, bf16x8 (&x)[WM]) {
#pragma unroll
      for (int m = 0; m < WM; ++m) {
        const int row = (wm * WM + m) * 32 + r;
        x[m] = *(const bf16x8*)&stage[b].x[row * 128 + ((h * 4 + j) ^ (row >> 1 & 7)) * 16];
      }
    };
    auto convert = [&](const uint32_t (&code)[WN][kWords<FAM>], const float (&scale)[WN], const uint32_t (&left)[WN], int j, bf16x8 (&w)[WN]) {
#pragma unroll
      for (int i = 0; i < WN; ++i) w[i] = eight<FAM>(code[i], scale[i], j, ta.map);
      // (the whole step twice in the code, so that no branch parts its products, takes the registers of a workgroup: 1.1 to 1.8
      // times slower)
      if ((FAM == kMapped || WIDE) && __builtin_expect(__any(left[0] | left[1]), 0)) {
#pragma unroll
        for (int i = 0; i < WN; ++i) {
          if (FAM == kMapped) apply_left(w[i], left[i]);
          if (WIDE && __any(left[i] & ~255u)) finite_only(w[i]);
        }
      }
    };
    auto multiply = [&](const bf16x8 (&w)[WN], const bf16x8 (&x)[WM]) {
#pragma unroll
      for (int i = 0; i < WN; ++i)
#pragma unroll
        for (int m = 0; m < WM; ++m) acc[i][m] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(w[i], x[m], acc[i][m], 0, 0, 0);
    };
    auto next = [](int b) { return b == STAGES - 1 ? 0 : b + 1; };

    if constexpr (WM <= 2) {
      // Few rows: a step's operands are all read a step ahead, one wait for LDS a step, since a phase of the larger tile's
      // walk would hold too few products to hide it.
#pragma unroll
      for (int s = 0; s < STAGES; ++s) {
        if (s) advance();
#pragma unroll
        for (int p = 0; p < 3; ++p) issue(s, p);
      }
      asm volatile("s_waitcnt vmcnt(%0)" ::"n"(kInFlight + XL + WL) : "memory");
      asm volatile("s_barrier" ::: "memory");
      uint32_t code[2][WN][kWords<FAM>], left[2][WN];
      float scale[2][WN];
      bf16x8 xv[2][4][WM];
      auto read = [&](int b, int st, int turn) {
        read_codes(b, st, code[turn], scale[turn], left[turn]);
#pragma unroll
        for (int j = 0; j < 4; ++j) read_x(b, j, xv[turn][j]);
      };
      int b = 0;
      read(0, first, 0);
      for (int now = first; now < last; now += 2) {                      // an even number of steps
#pragma unroll
        for (int turn = 0; turn < 2; ++turn) {
          asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(kInFlight) : "memory");
          asm volatile("s_barrier" ::: "memory");
          advance();
#pragma unroll
          for (int p = 0; p < 3; ++p) issue(b, p);
          b = next(b);
          read(b, now + turn + 1, 1 - turn);                             // after the last step: what no sum takes
          __builtin_amdgcn_sched_barrier(0);                             // the compiler would sink the reads to their uses
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            bf16x8 w[WN];
            convert(code[turn], scale[turn], left[turn], j, w);
            multiply(w, xv[turn][j]);
          }
        }
      }
    } else {
      // A step is four phases of eight columns a lane.  A phase reads and converts the next one's operands while its own
      // are multiplied; the last phase of a step first waits for the next stage, whose loads began two steps ago, and
      // hands its own buffer to the stage after the one in flight.
      uint32_t code[WN][kWords<FAM>], left[WN];
      float scale[WN];
      bf16x8 wv[2][WN], xv[2][WM];
#pragma unroll
      for (int s = 0; s < STAGES; ++s) {
#pragma unroll
        for (int p = 0; p < 3; ++p)
          if (s < STAGES - 1 || p == 0) issue(s, p);
        if (s < STAGES - 1) advance();
      }
      asm volatile("s_waitcnt vmcnt(%0)" ::"n"(kInFlight + WL) : "memory");
      asm volatile("s_barrier" ::: "memory");
      read_codes(0, first, code, scale, left);
      read_x(0, 0, xv[0]);
      convert(code, scale, left, 0, wv[0]);
      int b = 0;
      for (int now = first; now < last; ++now) {
        const int nb = next(b), pb = b == 0 ? STAGES - 1 : b - 1;        // the stage whose loads are being issued
#pragma unroll
        for (int j = 0; j < 3; ++j) {
          read_x(b, j + 1, xv[(j + 1) & 1]);
          __builtin_amdgcn_sched_barrier(0);                             // the compiler would sink the reads to their uses
          if (j < 2) issue(pb, j + 1);
          multiply(wv[j & 1], xv[j & 1]);
          convert(code, scale, left, j + 1, wv[(j + 1) & 1]);
        }
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(kInFlight) : "memory");
        asm volatile("s_barrier" ::: "memory");
        advance();
        read_codes(nb, now + 1, code, scale, left);                      // after the last step: what no sum takes
        read_x(nb, 0, xv[0]);
        __builtin_amdgcn_sched_barrier(0);
        issue(b, 0);
        multiply(wv[1], xv[1]);
        convert(code, scale, left, 0, wv[0]);
        b = nb;
      }
    }
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
  }

  // acc[i][m][e]: row m * 32 + (lane & 31), weight row i * 32 + 8 (e / 4) + 4 h + e % 4.  The stages become the waves' own
  // transposes, from which a lane takes eight neighbouring outputs of a row.  The loop stays a loop: unrolled, its code was
  // read from memory once a workgroup, 5 us that nothing hid.
  __syncthreads();
  const int shift = gated ? 2 : 3, groups = 1 << shift, passes = groups / 2, group = lane & (groups - 1);       // of a row, of 32
  const int64_t n = n0 + wn * (gated ? 32 : 64) + group * 8, width = gated ? 2 * a.N : a.N;
  float* mine = (float*)memory + wave * (kHeld * 32 * PITCH);
  auto hold = [&](int m, int at) {
#pragma unroll
    for (int i = 0; i < WN; ++i)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const f32x16& v = acc[i][m];
        *(f32x4*)&mine[(at * 32 + r) * PITCH + i * 32 + 8 * q + 4 * h] = f32x4{v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]};
      }
  };
  auto in_order = [&]() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  };
  const bool split = ta.split > 1, whole = n + 8 <= a.N;
  Bias bias = {};
  if (whole && !split && !t.zeros) bias = load_bias(a, t, n);
  // a residual of 16 bits: these 32 rows', and the next's, asked for before them
  const bool early = a.residual && a.sp.residual_dtype != MXQ_DT_F32 && !split && whole;
  u32x4 residual[4], coming[4];
  auto ask = [&](int m) {
#pragma unroll
    for (int p = 0; p < 4; ++p) {
      const int row = (wm * WM + m) * 32 + ((p * 64 + lane) >> shift);
      if (early && p < passes && row < t.rows)
        coming[p] = *(const u32x4_any*)((const uint16_t*)a.residual + (t.row0 + row) * a.sp.ld_residual + n);
    }
  };
  ask(0);
#pragma unroll
  for (int some = 0; some < WM; some += kHeld) {
    if (some) in_order();
#pragma unroll
    for (int m = 0; m < kHeld; ++m) hold(some + m, m);
    in_order();
#pragma unroll 1
    for (int held = 0; held < kHeld; ++held) {
#pragma unroll
      for (int p = 0; p < 4; ++p) residual[p] = coming[p];
      if (some + held + 1 < WM) ask(some + held + 1);
#pragma unroll
      for (int p = 0; p < 4; ++p) {
        const int line = (p * 64 + lane) >> shift, row = (wm * WM + some + held) * 32 + line;
        if (p >= passes || row >= t.rows || n >= a.N) continue;
        const float* at = &mine[(held * 32 + line) * PITCH + group * 8];
        float z[8], up[8];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const f32x4 u = *(const f32x4*)(at + 4 * i), v = *(const f32x4*)(at + 4 * i + (gated ? 32 : 0));
#pragma unroll
          for (int e = 0; e < 4; ++e) z[4 * i + e] = u[e], up[4 * i + e] = v[e];
        }
        const int64_t y = t.row0 + row;
        if (split) {
          float* out = ta.partial + ((int64_t)blockIdx.y * a.M + y) * width + n;
          if (whole) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              u32x4 first4, second4;
#pragma unroll
              for (int e = 0; e < 4; ++e) first4[e] = __float_as_uint(z[4 * i + e]), second4[e] = __float_as_uint(up[4 * i + e]);
              *(u32x4_any*)(out + 4 * i) = first4;
              if (gated) *(u32x4_any*)(out + a.N + 4 * i) = second4;
            }
          } else {
#pragma unroll 1
            for (int e = 0; n + e < a.N; ++e) {
              out[e] = at[e];
              if (gated) out[a.N + e] = at[32 + e];
            }
          }
        } else if (whole) {
          Eight r8;
          r8.first = residual[p];
          if (a.residual && !early) r8 = load_eight(a.residual, a.sp.residual_dtype, y * a.sp.ld_residual + n);
          finish_eight(a, t, y, n, z, up, bias, r8);
        } else {
#pragma unroll 1
          for (int e = 0; n + e < a.N; ++e) store_elem(a.y, a.sp.y_dtype, y * a.sp.ld_y + n + e, epilogue(a, t, y, n + e, at[e], at[gated ? 32 + e : 0]));
        }
      }
    }
  }
}

template <int FAM, bool WIDE> void launch_tile_planes(const TileArgs& ta, const TilePlan& p, hipStream_t st) {
  const dim3 grid((unsigned)(ta.tiles_m * ta.tiles_n), (unsigned)p.split);
  KernelTimer timer("k_linear_tile", st);
  if (p.shape == 0) k_linear_tile<FAM, WIDE, 256, 256, 4, 2, 3, false><<<grid, 512, 0, st>>>(ta);
  else if (p.shape == 1) k_linear_tile<FAM, WIDE, 128, 128, 2, 2, 3, false><<<grid, 256, 0, st>>>(ta);
  else if (p.shape == 2) k_linear_tile<FAM, WIDE, 64, 128, 1, 2, 3, false><<<grid, 256, 0, st>>>(ta);
  else k_linear_tile<FAM, WIDE, 64, 128, 1, 2, 3, true><<<grid, 256, 0, st>>>(ta);
}

template <int FAM> void launch_tile_family(const TileArgs& ta, const TilePlan& p, hipStream_t st) {
  if (ta.planes > 1) launch_tile_planes<FAM, true>(ta, p, st);
  else launch_tile_planes<FAM, false>(ta, p, st);
}

}  // namespace mxq
