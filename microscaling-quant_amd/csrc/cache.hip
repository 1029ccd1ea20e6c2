// Rows of a key and value cache in MX formats (include/mxq_hip.h): quantized as they are written, and read back as values.
// Both are bound by memory: a row of 128 bfloat16 is 256 bytes in and 68 (MXFP4) or 132 (MXFP8) out.  Four lanes take a block of 32 columns,
// eight columns a lane, so that a wave reads and writes runs of whole rows, 16 bytes a lane on the side of the values.
#include "cache_common.h"
#include "mxq_numerics.h"
#include "ocp_hw.h"

namespace mxq {
namespace {

struct RowsArgs {
  const void *k, *v;              // written from
  void *k_out, *v_out;            // read to
  int64_t token[2], head[2];      // strides of k and v, in elements
  uint8_t *codes[2], *scales[2];
  const void* slots;
  int64_t first, T;               // tokens [first, T) of this launch
  mxq_cache_spec c;
  DivU31 by_page;
  int32_t wide, per_group;        // int64 slots; tokens a workgroup
  DivU31 by_token, by_row;        // items a token, and a row
};

__device__ __forceinline__ int slot_of(const RowsArgs& a, int64_t t) {
  const int64_t s = a.wide ? ((const int64_t*)a.slots)[t] : ((const int32_t*)a.slots)[t];
  return s >= 0 && s < a.c.pages * a.c.page_size ? (int)s : -1;
}

// Eight columns of a block of a row of keys (which 0) or values are an item of a token; a thread has the same item of one
// token after another, so that what it takes from the item alone is found once.  Where a token has fewer items than the
// workgroup threads, several tokens are taken together; where it has more, its items in turns.
struct Lane {
  int item, token, tokens;        // this thread's first item and token, and how many tokens are taken together
};
template <int THREADS> __device__ __forceinline__ Lane lane_of(const RowsArgs& a) {
  const int items = (int)a.by_token.d;
  if (items > THREADS) return Lane{(int)threadIdx.x, 0, 1};
  const int token = (int)divu31(threadIdx.x, a.by_token), tokens = THREADS / items;
  return Lane{token < tokens ? (int)threadIdx.x - token * items : items, token, tokens};
}
struct Item {
  int which, head, block, quarter, d;   // d: its first column
  int64_t code, scale;                  // bytes from a row of head 0 to its codes and its block's scale
};
template <int BB> __device__ __forceinline__ Item item_of(const RowsArgs& a, int i) {
  const int row = (int)divu31(i, a.by_row), in = i - row * (int)a.by_row.d;
  const int which = row >= (int)a.c.kv_heads, head = row - which * (int)a.c.kv_heads, block = in >> 2, quarter = in & 3;
  return Item{which, head, block, quarter, block * kCacheBlock + quarter * 8, head * a.c.head_stride[2 * which] + block * BB + quarter * (BB / 4),
              head * a.c.head_stride[2 * which + 1] + block};
}
// A token's page and row; page -1 where its slot is not in the cache.
struct Place {
  int page, at;
};
__device__ __forceinline__ Place place_of(const RowsArgs& a, int slot) {
  if (slot < 0) return Place{-1, 0};
  const int page = (int)divu31(slot, a.by_page);
  return Place{page, slot - page * (int)a.c.page_size};
}

// 2^(floor(log2 amax) - emax) as an E8M0 byte, the logarithm rounded to float32 as the block quantizers take it; 255 where
// amax (its bits) is an infinity or a NaN.
template <int DT> __device__ __forceinline__ int scale_byte(uint32_t amax, int emax) {
  if (amax >= 0x7F800000u) return 255;
  int e;
  if (DT != MXQ_DT_F32 && amax >= 0x00800000u) e = (int)(amax >> 23) - 127;      // no 16-bit value is near enough below a power of two
  else e = amax ? floor_log2_pos(u2f(amax)) : -126;
  e -= emax;
  return e < -127 ? 0 : e + 127;
}

// The largest of four neighbouring lanes' values.
__device__ __forceinline__ uint32_t quad_max(uint32_t v) {
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xF, 0xF, true));          // lanes 1, 0, 3, 2
  return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xF, 0xF, true));       // lanes 2, 3, 0, 1
}

// Few tokens: one a workgroup of 256 threads, to be done soonest.  Otherwise up to kTokens a workgroup of 512, each thread with
// kAhead of its items in flight.  16384 tokens of 8 heads of 128 bfloat16 columns to MXFP8: 41 us, 102 MB at 2.5 TB/s (32
// tokens a workgroup 47; 16 with four items ahead, which leaves half the waves, 53).  About 8 us of it is looking for later
// tokens with the same slots, which each workgroup does for itself: the call needs no workspace and no second launch, and
// no order of the workgroups matters.
// Written and read back, 1021 tokens of 5 heads of 80 float32 columns take 10.3 us by the one and 14.0 by the other, the 16384
// tokens 127 and 60.6: a workgroup a token reads all slots once a token.
constexpr int kTokens = 16, kFewTokens = 1024, kFilter = 2048;
template <bool FEW> constexpr int kThreads = FEW ? 256 : 512;
template <bool FEW> constexpr int kAhead = FEW ? 1 : 2;

template <int FAM, int DT, bool FEW> __global__ __launch_bounds__(kThreads<FEW>) void k_cache_write(RowsArgs a) {
  constexpr int THREADS = kThreads<FEW>, AHEAD = kAhead<FEW>;
  constexpr int EMAX = FAM == kE4M3 ? 8 : FAM == kE5M2 ? 15 : 2, BB = FAM == kPairs ? 16 : 32, SIZE = DT == MXQ_DT_F32 ? 4 : 2;
  constexpr float TOP = FAM == kE4M3 ? 448.0f : FAM == kE5M2 ? 57344.0f : 6.0f;
  __shared__ uint32_t filter[FEW ? 1 : kFilter];
  __shared__ int slots[kTokens];
  __shared__ Place places[kTokens];
  const int64_t t0 = a.first + (int64_t)blockIdx.x * a.per_group;
  const int mine = a.T - t0 < a.per_group ? (int)(a.T - t0) : a.per_group;
  const int items = (int)a.by_token.d, D = a.c.head_dim;
  const Lane lane = lane_of<THREADS>(a);

  // eight columns as they lie in memory, zeros past the row's end
  auto load = [&](const Item& it, int token) {
    Eight x{};
    if (token >= mine) return x;
    const uint8_t* p = (const uint8_t*)(it.which ? a.v : a.k) + ((t0 + token) * a.token[it.which] + it.head * a.head[it.which] + it.d) * SIZE;
    if (it.d + 8 <= D) {
      x = load_eight(p, DT, 0);
    } else {
      const int left = it.d < D ? (D - it.d) * SIZE : 0;
      x.first = load_part(p, left);
      if (DT == MXQ_DT_F32) x.more = load_part(p + 16, left - 16);
    }
    return x;
  };
  Item it{};
  Eight ahead[AHEAD] = {};
  if (lane.item < items) {
    it = item_of<BB>(a, lane.item);
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) ahead[u] = load(it, lane.token + u * lane.tokens);
  }

  // A slot that a later token has is that token's.
  if constexpr (FEW) {
    const int slot = slot_of(a, t0);
    bool later = false;
    for (int64_t t = t0 + 1 + threadIdx.x; t < a.T; t += THREADS) later |= slot_of(a, t) == slot;
    later = __syncthreads_or(later);
    if (threadIdx.x == 0) places[0] = place_of(a, later ? -1 : slot);
  } else {
    for (int i = threadIdx.x; i < kFilter; i += THREADS) filter[i] = 0;
    if (threadIdx.x < kTokens) slots[threadIdx.x] = (int)threadIdx.x < mine ? slot_of(a, t0 + threadIdx.x) : -1;
    __syncthreads();
    // A bit for each of these tokens' slots, of as many that seldom one of a wave's 64 slots meets one by chance.
    if ((int)threadIdx.x < mine && slots[threadIdx.x] >= 0) atomicOr(&filter[slots[threadIdx.x] >> 5 & kFilter - 1], 1u << (slots[threadIdx.x] & 31));
    __syncthreads();
    constexpr int kAtOnce = 8;
    for (int64_t t = t0 + 1 + threadIdx.x; t < a.T; t += THREADS * kAtOnce) {
      int s[kAtOnce];
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u) s[u] = t + THREADS * u < a.T ? slot_of(a, t + THREADS * u) : -1;
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u)
        if (s[u] >= 0 && (filter[s[u] >> 5 & kFilter - 1] >> (s[u] & 31) & 1))
          for (int i = 0; i < mine && t0 + i < t + THREADS * u; ++i)
            if (slots[i] == s[u]) slots[i] = -1;             // every thread that finds it writes the same
    }
    __syncthreads();
    if ((int)threadIdx.x < mine) places[threadIdx.x] = place_of(a, slots[threadIdx.x]);
  }
  __syncthreads();

  for (int i = lane.item; i < items; i += THREADS) {
    if (i != lane.item) {
      it = item_of<BB>(a, i);
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) ahead[u] = load(it, lane.token + u * lane.tokens);
    }
    for (int token = lane.token; token < mine; token += lane.tokens * AHEAD) {
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) {
        const int now = token + u * lane.tokens;
        const Eight x = ahead[u];
        ahead[u] = load(it, now + AHEAD * lane.tokens);
        float f[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) f[k] = 0.0f;
        add_eight(f, x, DT);
        uint32_t amax = 0;
#pragma unroll
        for (int k = 0; k < 8; ++k) amax = max(amax, __float_as_uint(f[k]) & 0x7FFFFFFFu);
        amax = quad_max(amax);
        const Place place = now < mine ? places[now] : Place{-1, 0};
        if (place.page < 0) continue;
        const int byte = scale_byte<DT>(amax, EMAX);
        // times the scale's reciprocal, 2^(127 - byte): exact, byte 254 is not reached
        const float inv = byte == 255 ? 0.0f : __uint_as_float((uint32_t)(254 - byte) << 23);
#pragma unroll
        for (int k = 0; k < 8; ++k) f[k] = byte == 255 ? 0.0f : __builtin_amdgcn_fmed3f(f[k] * inv, -TOP, TOP);
        uint32_t w[2];
        mxq_ocp_hw::codes<8>(f, FAM == kE4M3 ? 4 : FAM == kE5M2 ? 5 : 2, FAM == kE4M3 ? 3 : FAM == kE5M2 ? 2 : 1, w);
        const int part = 2 * it.which;
        uint8_t* out = a.codes[it.which] + (place.page * a.c.page_stride[part] + place.at * a.c.row_stride[part] + it.code);
        if constexpr (FAM == kPairs) {
          const uint32_t n = w[0] | w[0] >> 4, m = w[1] | w[1] >> 4;
          const uint32_t both = (n & 0xFFu) | (n >> 8 & 0xFF00u) | (m & 0xFFu) << 16 | (m >> 8 & 0xFF00u) << 16;
          __builtin_memcpy(out, &both, 4);
        } else {
          __builtin_memcpy(out, w, 8);
        }
        if (it.quarter == 0)
          a.scales[it.which][place.page * a.c.page_stride[part + 1] + place.at * a.c.row_stride[part + 1] + it.scale] = (uint8_t)byte;
      }
    }
  }
}

// Values of many rows go past the caches: 268 MB of bfloat16 from 65536 rows of 8 heads of 128 MXFP4 columns take 52 us, 6.5
// TB/s with what is read, and took 95 through them.  777 rows take 3.7 us through the caches and 4.1 past them.
template <bool FEW> __device__ __forceinline__ void store_sixteen(void* p, const u32x4& v) {
  if constexpr (FEW) *(u32x4_any*)p = v;
  else __builtin_nontemporal_store(v, (u32x4_any*)p);
}

template <int FAM, int DT, bool FEW> __global__ __launch_bounds__(kThreads<FEW>) void k_cache_read(RowsArgs a) {
  constexpr int THREADS = kThreads<FEW>, AHEAD = kAhead<FEW>, BB = FAM == kPairs ? 16 : 32;
  __shared__ Place places[kTokens];
  const int items = (int)a.by_token.d, D = a.c.head_dim;
  const int64_t t0 = a.first + (int64_t)blockIdx.x * a.per_group;
  const int mine = a.T - t0 < a.per_group ? (int)(a.T - t0) : a.per_group;
  if ((int)threadIdx.x < mine) places[threadIdx.x] = place_of(a, slot_of(a, t0 + threadIdx.x));
  __syncthreads();
  const Lane lane = lane_of<THREADS>(a);
  for (int i = lane.item; i < items; i += THREADS) {
    const Item it = item_of<BB>(a, i);
    if (it.d >= D) continue;
    const int part = 2 * it.which;
    const uint8_t *codes = a.codes[it.which] + it.code, *scales = a.scales[it.which] + it.scale;
    for (int token = lane.token; token < mine; token += lane.tokens * AHEAD) {
      uint32_t w[AHEAD][2], byte[AHEAD];
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) {
        w[u][0] = w[u][1] = 0, byte[u] = 127;
        const int now = token + u * lane.tokens;
        const Place place = now < mine ? places[now] : Place{-1, 0};
        if (place.page < 0) continue;
        __builtin_memcpy(w[u], codes + (place.page * a.c.page_stride[part] + place.at * a.c.row_stride[part]), BB / 4);
        byte[u] = scales[place.page * a.c.page_stride[part + 1] + place.at * a.c.row_stride[part + 1]];
      }
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) {
        const int now = token + u * lane.tokens;
        if (now >= mine) continue;
        void* out = it.which ? a.v_out : a.k_out;
        const int64_t at = ((t0 + now) * a.c.kv_heads + it.head) * D + it.d;
        u32x4 half;                                       // eight values of 16 bits
        float f[8];
        if constexpr (DT == MXQ_DT_BF16) {
          const bf16x8 v = eight_codes<FAM>(w[u], scale_field(byte[u]));
          __builtin_memcpy(&half, &v, 16);
        } else {
          const float scale = e8m0_decode(byte[u]);
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            mxq_ocp_hw::f2v v;
            if constexpr (FAM == kPairs) {
              if (k == 0) v = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[u][0], 1.0f, 0);
              else if (k == 1) v = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[u][0], 1.0f, 1);
              else if (k == 2) v = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[u][0], 1.0f, 2);
              else v = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[u][0], 1.0f, 3);
            } else if constexpr (FAM == kE4M3) {
              v = k & 1 ? __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w[u][k >> 1], 1.0f, true) : __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w[u][k >> 1], 1.0f, false);
            } else {
              v = k & 1 ? __builtin_amdgcn_cvt_scalef32_pk_f32_bf8(w[u][k >> 1], 1.0f, true) : __builtin_amdgcn_cvt_scalef32_pk_f32_bf8(w[u][k >> 1], 1.0f, false);
            }
            f[2 * k] = v.x * scale, f[2 * k + 1] = v.y * scale;
            if constexpr (DT == MXQ_DT_F16) {
              const f16x2 h = {(_Float16)f[2 * k], (_Float16)f[2 * k + 1]};
              uint32_t both;
              __builtin_memcpy(&both, &h, 4);
              half[k] = both;
            }
          }
        }
        if (it.d + 8 <= D) {
          if constexpr (DT == MXQ_DT_F32) {
            u32x4 p, q;
            __builtin_memcpy(&p, f, 16);
            __builtin_memcpy(&q, f + 4, 16);
            store_sixteen<FEW>((float*)out + at, p);
            store_sixteen<FEW>((float*)out + at + 4, q);
          } else {
            store_sixteen<FEW>((uint16_t*)out + at, half);
          }
        } else {
#pragma unroll
          for (int k = 0; k < 8; ++k)
            if (it.d + k < D) {
              if constexpr (DT == MXQ_DT_F32) ((float*)out)[at + k] = f[k];
              else ((uint16_t*)out)[at + k] = (uint16_t)(half[k >> 1] >> (k & 1) * 16);
            }
        }
      }
    }
  }
}

int check(const std::string& who, const mxq_cache_spec* c, int32_t dtype, int64_t T, bool pointers) {
  if (!c) return invalid(who + ": NULL spec");
  if (c->format != MXQ_FMT_E4M3 && c->format != MXQ_FMT_E5M2 && c->format != MXQ_FMT_E2M1_PAIRS) return invalid(who + ": unknown format");
  if (c->head_dim < 1 || c->head_dim > 256) return invalid(who + ": head_dim must be 1 to 256");
  if (c->pages < 1 || c->page_size < 1 || c->pages > 0x7fffffff || c->page_size > 0x7fffffff || c->pages * c->page_size > 0x7fffffff ||
      c->kv_heads < 1 || c->kv_heads > 65535)
    return invalid(who + ": cache size out of range");
  if (dtype < MXQ_DT_F32 || dtype > MXQ_DT_F16) return invalid(who + ": unknown dtype");
  if (T < 0 || T > 0x7fffffff) return invalid(who + ": size out of range");
  if (T && !pointers) return invalid(who + ": NULL pointer");
  return MXQ_OK;
}

RowsArgs rows_args(const mxq_cache_spec* c, const void* slots, int32_t wide, uint8_t* kc, uint8_t* ks, uint8_t* vc, uint8_t* vs) {
  RowsArgs a = {};
  a.codes[0] = kc, a.codes[1] = vc, a.scales[0] = ks, a.scales[1] = vs;
  a.slots = slots, a.wide = wide, a.c = *c;
  const int blocks = (c->head_dim + kCacheBlock - 1) / kCacheBlock;
  a.by_page = make_divu31((uint32_t)c->page_size);
  a.by_row = make_divu31((uint32_t)(4 * blocks));
  a.by_token = make_divu31((uint32_t)(2 * c->kv_heads * 4 * blocks));
  return a;
}

#define MXQ_EACH_TYPE(KERNEL, FAM, FEW)                                                                       \
  (dtype == MXQ_DT_F32 ? KERNEL<FAM, MXQ_DT_F32, FEW> : dtype == MXQ_DT_BF16 ? KERNEL<FAM, MXQ_DT_BF16, FEW> \
                                                                             : KERNEL<FAM, MXQ_DT_F16, FEW>)
#define MXQ_EACH_FORMAT(KERNEL, FEW)                                          \
  (a.c.format == MXQ_FMT_E4M3   ? MXQ_EACH_TYPE(KERNEL, kE4M3, FEW)           \
   : a.c.format == MXQ_FMT_E5M2 ? MXQ_EACH_TYPE(KERNEL, kE5M2, FEW)           \
                                : MXQ_EACH_TYPE(KERNEL, kPairs, FEW))

// Tokens in launches of at most `most` (2^26: 2^31 threads, half of what a launch can have), one behind another.
template <typename Kernel> int launch_rows(RowsArgs a, Kernel one, Kernel many, int64_t T, int64_t most, hipStream_t st, const char* who,
                                       const char* name) {
  for (int64_t first = 0; first < T; first += most) {
    a.first = first, a.T = T - first < most ? T : first + most;
    const int64_t n = a.T - first;
    const bool few = n <= kFewTokens;
    a.per_group = few ? 1 : (int)(ceil_div(n, 1024) < kTokens ? ceil_div(n, 1024) : kTokens);
    {
      KernelTimer timer(name, st);
      (few ? one : many)<<<dim3((unsigned)ceil_div(n, a.per_group)), few ? kThreads<true> : kThreads<false>, 0, st>>>(a);
    }
    if (int rc = check_launch(who)) return rc;
  }
  return MXQ_OK;
}

}  // namespace
}  // namespace mxq

extern "C" int mxq_cache_write(const void* k, const void* v, int32_t dtype, int64_t T, int64_t k_token, int64_t k_head, int64_t v_token,
                               int64_t v_head, const void* slots, int32_t slots_wide, uint8_t* k_codes, uint8_t* k_scales, uint8_t* v_codes,
                               uint8_t* v_scales, const mxq_cache_spec* cache, mxq_stream_t stream) {
  using namespace mxq;
  if (int rc = check("mxq_cache_write", cache, dtype, T, k && v && slots && k_codes && k_scales && v_codes && v_scales)) return rc;
  RowsArgs a = rows_args(cache, slots, slots_wide, k_codes, k_scales, v_codes, v_scales);
  a.k = k, a.v = v;
  a.token[0] = k_token, a.token[1] = v_token, a.head[0] = k_head, a.head[1] = v_head;
  // A launch looks through its own later tokens for each of its slots; launches follow one another.
  return launch_rows(a, MXQ_EACH_FORMAT(k_cache_write, true), MXQ_EACH_FORMAT(k_cache_write, false), T, 1 << 15, as_stream(stream), "mxq_cache_write",
                     "k_cache_write");
}

extern "C" int mxq_cache_read(const uint8_t* k_codes, const uint8_t* k_scales, const uint8_t* v_codes, const uint8_t* v_scales,
                              const mxq_cache_spec* cache, const void* slots, int32_t slots_wide, int64_t T, void* k, void* v, int32_t dtype,
                              mxq_stream_t stream) {
  using namespace mxq;
  if (int rc = check("mxq_cache_read", cache, dtype, T, k && v && slots && k_codes && k_scales && v_codes && v_scales)) return rc;
  if (T == 0) return MXQ_OK;
  RowsArgs a = rows_args(cache, slots, slots_wide, const_cast<uint8_t*>(k_codes), const_cast<uint8_t*>(k_scales), const_cast<uint8_t*>(v_codes),
                         const_cast<uint8_t*>(v_scales));
  a.k_out = k, a.v_out = v;
  return launch_rows(a, MXQ_EACH_FORMAT(k_cache_read, true), MXQ_EACH_FORMAT(k_cache_read, false), T, 1 << 26, as_stream(stream), "mxq_cache_read",
                     "k_cache_read");
}
