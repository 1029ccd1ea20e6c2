// Tokens' slots sorted by expert, and the weighted sum that brings the experts' rows back (include/mxq_hip.h,
// mxq_dispatch and mxq_combine).  Slot i = t k + j is token t's j-th choice.
#include "mxq_common.h"

namespace mxq {
namespace {

constexpr int kMaxExperts = 1024, kMaxTopK = 64;
constexpr int kSortThreads = 1024, kSortWaves = kSortThreads / 64;

// A stable counting sort by one workgroup: counts, their prefix, then 1024 slots at a time each to its expert's next
// places.  A slot's rank among its wave's equal ones is a population count of the lanes with the same key; the waves
// before it add theirs from LDS.  Integer sums throughout: the same order whatever the timing.
__global__ __launch_bounds__(kSortThreads) void k_dispatch(const int32_t* experts, int n, int E, int bits,
                                                           int32_t* order, int32_t* offsets, int32_t* positions) {
  __shared__ int base[kMaxExperts + 1];
  __shared__ int scan[kSortWaves];
  __shared__ uint16_t cnt[kSortWaves][kMaxExperts + 1];      // a wave's counts, at most 64 each
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  auto key_of = [&](int i) {
    const int e = experts[i];
    return (unsigned)e < (unsigned)E ? e : E;                     // E: the slots of no expert, sorted last
  };
  for (int e = tid; e <= E; e += kSortThreads) base[e] = 0;
  __syncthreads();
  for (int i = tid; i < n; i += kSortThreads) atomicAdd(&base[key_of(i)], 1);
  __syncthreads();
  // exclusive prefix over the E + 1 <= 1025 counts: one a thread, the last by itself
  int c = tid < E ? base[tid] : 0, p = c;
  for (int o = 1; o < 64; o <<= 1) {
    const int q = __shfl_up(p, o);
    if (lane >= o) p += q;
  }
  if (lane == 63) scan[wave] = p;
  __syncthreads();
  int before = 0;
  for (int w = 0; w < wave; ++w) before += scan[w];
  p += before;
  __syncthreads();
  if (tid < E) base[tid] = p - c, offsets[tid] = p - c;
  if (tid == kSortThreads - 1) base[E] = p, offsets[E] = p;
  __syncthreads();
  for (int first = 0; first < n; first += kSortThreads) {
    for (int w = 0; w < kSortWaves; ++w)
      for (int e = tid; e <= E; e += kSortThreads) cnt[w][e] = 0;
    __syncthreads();
    const int i = first + tid;
    const int key = i < n ? key_of(i) : -1;
    uint64_t same = __ballot(i < n);
    for (int b = 0; b < bits; ++b) {
      const uint64_t set = __ballot(key >> b & 1);
      same &= key >> b & 1 ? set : ~set;
    }
    const int rank = __popcll(same & ((1ull << lane) - 1));
    if (i < n && rank == 0) cnt[wave][key] = (uint16_t)__popcll(same);
    __syncthreads();
    int place = 0;
    if (i < n) {
      place = base[key] + rank;
      for (int w = 0; w < wave; ++w) place += cnt[w][key];
      order[place] = i;
      positions[i] = key < E ? place : -1 - place;
    }
    __syncthreads();
    for (int e = tid; e <= E; e += kSortThreads)
      for (int w = 0; w < kSortWaves; ++w) base[e] += cnt[w][e];
    __syncthreads();
  }
}

template <int DT> struct Elem;
template <> struct Elem<MXQ_DT_F32> { typedef float type; };
template <> struct Elem<MXQ_DT_BF16> { typedef __bf16 type; };
template <> struct Elem<MXQ_DT_F16> { typedef _Float16 type; };

// out[t] = residual[t] + sum_j w[t, j] y[position[t, j]] in float32, j in order, rounded once.
template <int DT> __global__ __launch_bounds__(256) void k_combine(const void* y_, const float* weights, const int32_t* positions,
                                                                   const void* residual_, void* out_, int64_t T, int k, int64_t D) {
  typedef typename Elem<DT>::type E;
  const E *y = (const E*)y_, *residual = (const E*)residual_;
  E* out = (E*)out_;
  for (int64_t t = blockIdx.x; t < T; t += gridDim.x)
    for (int64_t d = (int64_t)blockIdx.y * 256 + threadIdx.x; d < D; d += (int64_t)gridDim.y * 256) {
      float sum = residual ? (float)residual[t * D + d] : 0.0f;
      for (int j = 0; j < k; ++j) {
        const float w = weights[t * k + j];
        const int p = positions[t * k + j];
        if (p >= 0) sum = __builtin_fmaf(w, (float)y[p * D + d], sum);
        else if (w != w) sum = w;                               // a NaN weight of no expert stays visible
      }
      out[t * D + d] = (E)sum;
    }
}

// dy[position] = w g[t] (zeros for a slot of no expert), dw = <g[t], y[position]>: a workgroup a token.
template <int DT> __global__ __launch_bounds__(256) void k_combine_grad(const void* grad_, const void* y_, const float* weights,
                                                                        const int32_t* positions, void* dy_, float* dw, int64_t T,
                                                                        int k, int64_t D) {
  typedef typename Elem<DT>::type E;
  __shared__ float part[4];
  const E *y = (const E*)y_, *grad = (const E*)grad_;
  E* dy = (E*)dy_;
  for (int64_t t = blockIdx.x; t < T; t += gridDim.x)
    for (int j = 0; j < k; ++j) {
      const int p = positions[t * k + j];
      const int64_t row = p >= 0 ? p : -1 - (int64_t)p;
      const float w = p >= 0 ? weights[t * k + j] : 0.0f;
      float dot = 0.0f;
      for (int64_t d = threadIdx.x; d < D; d += 256) {
        const float g = (float)grad[t * D + d];
        if (dw && p >= 0) dot = __builtin_fmaf(g, (float)y[row * D + d], dot);
        if (dy) dy[row * D + d] = (E)(p >= 0 ? w * g : 0.0f);
      }
      if (!dw) continue;
      for (int o = 32; o; o >>= 1) dot += __shfl_xor(dot, o);
      if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = dot;
      __syncthreads();
      if (threadIdx.x == 0) dw[t * k + j] = part[0] + part[1] + part[2] + part[3];
      __syncthreads();
    }
}

int check_combine(const char* who, int32_t dtype, int64_t T, int64_t k, int64_t D) {
  const std::string w(who);
  if (dtype < MXQ_DT_F32 || dtype > MXQ_DT_F16) return invalid(w + ": unknown dtype");
  if (T < 0 || D < 0) return invalid(w + ": negative size");
  if (k < 1 || k > kMaxTopK) return invalid(w + ": top_k must be 1 to 64");
  if (T > 0x7fffffff / k) return invalid(w + ": at most 2^31 - 1 slots");
  return MXQ_OK;
}

template <typename F> void with_dtype(int32_t dtype, F f) {
  if (dtype == MXQ_DT_F32) f(std::integral_constant<int, MXQ_DT_F32>());
  else if (dtype == MXQ_DT_BF16) f(std::integral_constant<int, MXQ_DT_BF16>());
  else f(std::integral_constant<int, MXQ_DT_F16>());
}

}  // namespace
}  // namespace mxq

using namespace mxq;

extern "C" int mxq_dispatch(const int32_t* experts, int64_t n, int64_t E, int32_t* order, int32_t* offsets,
                            int32_t* positions, mxq_stream_t stream) {
  if (n < 0 || n > 0x7fffffff - kSortThreads) return invalid("mxq_dispatch: n out of range");
  if (E < 1 || E > kMaxExperts) return invalid("mxq_dispatch: 1 to 1024 experts");
  if (!offsets || (n && (!experts || !order || !positions))) return invalid("mxq_dispatch: NULL argument");
  int bits = 0;
  while ((E >> bits) != 0) ++bits;                                // keys 0 .. E
  KernelTimer timer("k_dispatch", as_stream(stream));
  k_dispatch<<<1, kSortThreads, 0, as_stream(stream)>>>(experts, (int)n, (int)E, bits, order, offsets, positions);
  return check_launch("mxq_dispatch");
}

extern "C" int mxq_combine(const void* y, int32_t dtype, const float* weights, const int32_t* positions,
                           const void* residual, void* out, int64_t T, int64_t k, int64_t D, mxq_stream_t stream) {
  if (int rc = check_combine("mxq_combine", dtype, T, k, D)) return rc;
  if (T == 0 || D == 0) return MXQ_OK;
  if (!y || !weights || !positions || !out) return invalid("mxq_combine: NULL argument");
  const dim3 grid((unsigned)T, (unsigned)(ceil_div(D, 256) < 65535 ? ceil_div(D, 256) : 65535));
  with_dtype(dtype, [&](auto dt) {
    KernelTimer timer("k_combine", as_stream(stream));
    k_combine<decltype(dt)::value><<<grid, 256, 0, as_stream(stream)>>>(y, weights, positions, residual, out, T, (int)k, D);
  });
  return check_launch("mxq_combine");
}

extern "C" int mxq_combine_grad(const void* grad, int32_t dtype, const void* y, const float* weights, const int32_t* positions,
                                void* dy, float* dw, int64_t T, int64_t k, int64_t D, mxq_stream_t stream) {
  if (int rc = check_combine("mxq_combine_grad", dtype, T, k, D)) return rc;
  if (T == 0 || (!dy && !dw)) return MXQ_OK;
  if (!positions || (D && (!grad || !y || !weights))) return invalid("mxq_combine_grad: NULL argument");
  with_dtype(dtype, [&](auto dt) {
    KernelTimer timer("k_combine_grad", as_stream(stream));
    k_combine_grad<decltype(dt)::value><<<dim3((unsigned)T), 256, 0, as_stream(stream)>>>(grad, y, weights, positions, dy, dw, T,
                                                                                         (int)k, D);
  });
  return check_launch("mxq_combine_grad");
}
