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
  int32_t wide, blocks, per_group;  // int64 slots; blocks a row; tokens a workgroup
  DivU31 by_token, by_row, by_heads;  // items a token, a row, and heads
};

__device__ __forceinline__ int slot_of(const RowsArgs& a, int64_t t) {
  const int64_t s = a.wide ? ((const int64_t*)a.slots)[t] : ((const int32_t*)a.slots)[t];
  return s >= 0 && s < a.c.pages * a.c.page_size ? (int)s : -1;
}

// Item i of a token: eight columns of a block of a row of keys (which 0) or values.
struct Item {
  int which, head, block, quarter;
};
__device__ __forceinline__ Item item_of(const RowsArgs& a, int i) {
  const int row = (int)divu31(i, a.by_row), in = i - row * (int)a.by_row.d;
  const int which = row >= (int)a.c.kv_heads;
  return Item{which, row - which * (int)a.c.kv_heads, in >> 2, in & 3};
}
__device__ __forceinline__ int64_t at_row(const RowsArgs& a, int part, int slot, int head) {
  const int page = (int)divu31(slot, a.by_page), at = slot - page * (int)a.c.page_size;
  return page * a.c.page_stride[part] + head * a.c.head_stride[part] + at * a.c.row_stride[part];
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

template <int FAM, int DT> __global__ __launch_bounds__(256) void k_cache_write(RowsArgs a) {
  constexpr int EMAX = FAM == kE4M3 ? 8 : FAM == kE5M2 ? 15 : 2, BB = FAM == kPairs ? 16 : 32;
  constexpr float TOP = FAM == kE4M3 ? 448.0f : FAM == kE5M2 ? 57344.0f : 6.0f;
  __shared__ uint32_t filter[64];
  __shared__ int slots[64];
  const int64_t t0 = a.first + (int64_t)blockIdx.x * a.per_group;
  const int mine = a.T - t0 < a.per_group ? (int)(a.T - t0) : a.per_group;
  if (threadIdx.x < 64) {
    filter[threadIdx.x] = 0;
    slots[threadIdx.x] = (int)threadIdx.x < mine ? slot_of(a, t0 + threadIdx.x) : -1;
  }
  __syncthreads();
  // A slot that a later token has is that token's: a bit of 2048 for each of these tokens' slots sorts out nearly all others.
  if (a.T - t0 > 1) {
    if ((int)threadIdx.x < mine && slots[threadIdx.x] >= 0) atomicOr(&filter[slots[threadIdx.x] >> 5 & 63], 1u << (slots[threadIdx.x] & 31));
    __syncthreads();
    for (int64_t t = t0 + 1 + threadIdx.x; t < a.T; t += 256) {
      const int s = slot_of(a, t);
      if (s >= 0 && (filter[s >> 5 & 63] >> (s & 31) & 1))
        for (int i = 0; i < mine && t0 + i < t; ++i)
          if (slots[i] == s) slots[i] = -1;                  // every thread that finds it writes the same
    }
    __syncthreads();
  }
  const int items = (int)a.by_token.d, D = a.c.head_dim;
  for (int j = threadIdx.x; j < mine * items; j += 256) {
    const int t = (int)divu31(j, a.by_token), slot = slots[t];
    const Item it = item_of(a, j - t * items);
    const int d = it.block * kCacheBlock + it.quarter * 8;
    float f[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = 0.0f;
    if (slot >= 0) {
      const void* x = it.which ? a.v : a.k;
      const int64_t at = (t0 + t) * a.token[it.which] + it.head * a.head[it.which] + d;
      if (d + 8 <= D) {
        add_eight(f, x, DT, at);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (d + i < D) f[i] = load_elem(x, DT, at + i);
      }
    }
    uint32_t amax = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) amax = max(amax, __float_as_uint(f[i]) & 0x7FFFFFFFu);
    amax = max(amax, (uint32_t)__shfl_xor((int)amax, 1));
    amax = max(amax, (uint32_t)__shfl_xor((int)amax, 2));
    if (slot < 0) continue;
    const int byte = scale_byte<DT>(amax, EMAX);
    // times the scale's reciprocal, 2^(127 - byte): exact, byte 254 is not reached
    const float inv = byte == 255 ? 0.0f : __uint_as_float((uint32_t)(254 - byte) << 23);
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = byte == 255 ? 0.0f : __builtin_amdgcn_fmed3f(f[i] * inv, -TOP, TOP);
    uint32_t w[2];
    mxq_ocp_hw::codes<8>(f, FAM == kE4M3 ? 4 : FAM == kE5M2 ? 5 : 2, FAM == kE4M3 ? 3 : FAM == kE5M2 ? 2 : 1, w);
    uint8_t* out = a.codes[it.which] + at_row(a, 2 * it.which, slot, it.head) + it.block * BB + it.quarter * (BB / 4);
    if constexpr (FAM == kPairs) {
      const uint32_t n = w[0] | w[0] >> 4, m = w[1] | w[1] >> 4;
      const uint32_t p = (n & 0xFFu) | (n >> 8 & 0xFF00u) | (m & 0xFFu) << 16 | (m >> 8 & 0xFF00u) << 16;
      __builtin_memcpy(out, &p, 4);
    } else {
      __builtin_memcpy(out, w, 8);
    }
    if (it.quarter == 0) a.scales[it.which][at_row(a, 2 * it.which + 1, slot, it.head) + it.block] = (uint8_t)byte;
  }
}

template <int FAM, int DT> __global__ __launch_bounds__(256) void k_cache_read(RowsArgs a) {
  constexpr int BB = FAM == kPairs ? 16 : 32;
  const int items = (int)a.by_token.d, D = a.c.head_dim;
  const int64_t t0 = a.first + (int64_t)blockIdx.x * a.per_group;
  const int mine = a.T - t0 < a.per_group ? (int)(a.T - t0) : a.per_group;
  for (int j = threadIdx.x; j < mine * items; j += 256) {
    const int t = (int)divu31(j, a.by_token), slot = slot_of(a, t0 + t);
    const Item it = item_of(a, j - t * items);
    const int d = it.block * kCacheBlock + it.quarter * 8;
    if (d >= D) continue;
    uint32_t w[2] = {0, 0}, byte = 127;
    if (slot >= 0) {
      __builtin_memcpy(w, a.codes[it.which] + at_row(a, 2 * it.which, slot, it.head) + it.block * BB + it.quarter * (BB / 4), BB / 4);
      byte = a.scales[it.which][at_row(a, 2 * it.which + 1, slot, it.head) + it.block];
    }
    void* out = it.which ? a.v_out : a.k_out;
    const int64_t at = ((t0 + t) * a.c.kv_heads + it.head) * D + d;
    uint32_t half[4];                                     // eight values of 16 bits
    float f[8];
    if constexpr (DT == MXQ_DT_BF16) {
      const bf16x8 v = eight_codes<FAM>(w, scale_field(byte));
      __builtin_memcpy(half, &v, 16);
    } else {
      const float scale = e8m0_decode(byte);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        mxq_ocp_hw::f2v v;
        if constexpr (FAM == kPairs) {
          if (i == 0) v = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[0], 1.0f, 0);
          else if (i == 1) v = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[0], 1.0f, 1);
          else if (i == 2) v = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[0], 1.0f, 2);
          else v = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[0], 1.0f, 3);
        } else if constexpr (FAM == kE4M3) {
          v = i & 1 ? __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w[i >> 1], 1.0f, true) : __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w[i >> 1], 1.0f, false);
        } else {
          v = i & 1 ? __builtin_amdgcn_cvt_scalef32_pk_f32_bf8(w[i >> 1], 1.0f, true) : __builtin_amdgcn_cvt_scalef32_pk_f32_bf8(w[i >> 1], 1.0f, false);
        }
        f[2 * i] = v.x * scale, f[2 * i + 1] = v.y * scale;
        if constexpr (DT == MXQ_DT_F16) {
          const f16x2 h = {(_Float16)f[2 * i], (_Float16)f[2 * i + 1]};
          __builtin_memcpy(&half[i], &h, 4);
        }
      }
    }
    if (d + 8 <= D) {
      if constexpr (DT == MXQ_DT_F32) __builtin_memcpy((float*)out + at, f, 32);
      else __builtin_memcpy((uint16_t*)out + at, half, 16);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (d + i < D) {
          if constexpr (DT == MXQ_DT_F32) ((float*)out)[at + i] = f[i];
          else ((uint16_t*)out)[at + i] = (uint16_t)(half[i >> 1] >> (i & 1) * 16);
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
  a.blocks = (c->head_dim + kCacheBlock - 1) / kCacheBlock;
  a.by_page = make_divu31((uint32_t)c->page_size);
  a.by_row = make_divu31((uint32_t)(4 * a.blocks));
  a.by_token = make_divu31((uint32_t)(2 * c->kv_heads * 4 * a.blocks));
  return a;
}

#define MXQ_EACH_TYPE(KERNEL, FAM)                                                          \
  (dtype == MXQ_DT_F32 ? KERNEL<FAM, MXQ_DT_F32> : dtype == MXQ_DT_BF16 ? KERNEL<FAM, MXQ_DT_BF16> : KERNEL<FAM, MXQ_DT_F16>)
#define MXQ_EACH_FORMAT(KERNEL) \
  (a.c.format == MXQ_FMT_E4M3 ? MXQ_EACH_TYPE(KERNEL, kE4M3) : a.c.format == MXQ_FMT_E5M2 ? MXQ_EACH_TYPE(KERNEL, kE5M2) : MXQ_EACH_TYPE(KERNEL, kPairs))

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
  auto kernel = MXQ_EACH_FORMAT(k_cache_write);
  // A launch looks through its own later tokens for each of its slots; launches follow one another.
  constexpr int64_t kMost = 1 << 15;
  for (int64_t first = 0; first < T; first += kMost) {
    a.first = first, a.T = T - first < kMost ? T : first + kMost;
    const int64_t n = a.T - first;
    a.per_group = n <= 1024 ? 1 : n <= 16384 ? (int)ceil_div(n, 1024) : 16;
    kernel<<<dim3((unsigned)ceil_div(n, a.per_group)), 256, 0, as_stream(stream)>>>(a);
    if (int rc = check_launch("mxq_cache_write")) return rc;
  }
  return MXQ_OK;
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
  auto kernel = MXQ_EACH_FORMAT(k_cache_read);
  // workgroups of 256 threads, so that a launch stays below 2^32 threads
  a.T = T;
  a.per_group = (int)ceil_div(T, 1 << 20);
  kernel<<<dim3((unsigned)ceil_div(T, a.per_group)), 256, 0, as_stream(stream)>>>(a);
  return check_launch("mxq_cache_read");
}
