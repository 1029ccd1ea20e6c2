// Tokens' slots sorted by expert, and the weighted sum that brings the experts' rows back (include/mxq_hip.h,
// mxq_dispatch and mxq_combine).  Slot i = t k + j is token t's j-th choice.
#include "mxq_common.h"

namespace mxq {
namespace {

constexpr int kMaxExperts = 1024, kMaxTopK = 64;
constexpr int kSortThreads = 1024, kSortWaves = kSortThreads / 64, kAhead = 4;

// A stable counting sort.  A workgroup owns 16 runs of whole 64s of the slots, one a wave.  It counts the whole array's
// experts itself, those before its runs apart from the others (reading 4 bytes a slot again costs less than a second
// launch and a workspace), and each wave its own run's; prefix sums over the experts and the waves turn the counts into the
// places where each wave's slots go.  A slot's rank among its wave's equal ones is a population count of the lanes with
// the same key, which ballots over the key's bits find.  Integer sums throughout: the same order whatever the timing.
// 16384 slots of 32 experts 8.6 us, 32 slots 3.7: round trips to memory.  Counting everything in each workgroup grows beyond
// that, and additions to few experts' counts wait for each other: 65,536 slots of 32 experts 14 us, 262,144 36, 1,048,576 122;
// of 2 experts 39, 133 and 513.
__global__ __launch_bounds__(kSortThreads) void k_dispatch(const int32_t* experts, int n, int E, int bits, int run,
                                                           int32_t* order, int32_t* offsets, int32_t* positions) {
  __shared__ int place[kSortWaves][kMaxExperts + 1];
  __shared__ int before_me[kMaxExperts + 1], others[kMaxExperts + 1];
  __shared__ int scan[kSortWaves];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, begin = blockIdx.x * (kSortWaves * run);
  const int left = n - begin, used = left <= 0 ? 0 : left > (kSortWaves - 1) * run ? kSortWaves : (left - 1) / run + 1;
  const int first = begin + wave * run, last = wave >= used ? first : n - first < run ? n : first + run;
  volatile int* mine = place[wave];
  auto key_of = [&](int e) { return (unsigned)e < (unsigned)E ? e : E; };        // E: the slots of no expert, sorted last
  for (int e = tid; e <= E; e += kSortThreads) before_me[e] = others[e] = 0;
  if (wave < used)
    for (int e = lane; e <= E; e += 64) mine[e] = 0;
  __syncthreads();
  const int own = first + lane < last ? experts[first + lane] : 0;
  typedef int int4_any __attribute__((ext_vector_type(4), aligned(4)));
  // 16 slots a thread asked for at once; a single workgroup's runs are the whole array
  for (int i = gridDim.x > 1 ? tid * 4 : n; i < n; i += kSortThreads * 4 * kAhead) {
    int4_any e[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int at = i + u * kSortThreads * 4;
      if (at + 4 <= n) {
        e[u] = *(const int4_any*)(experts + at);
      } else {
#pragma unroll
        for (int c = 0; c < 4; ++c) e[u][c] = at + c < n ? experts[at + c] : 0;
      }
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int at = i + u * kSortThreads * 4 + c;
        if (at < n) atomicAdd(at < begin ? &before_me[key_of(e[u][c])] : &others[key_of(e[u][c])], 1);
      }
  }
  if (first + lane < last) atomicAdd(&place[wave][key_of(own)], 1);
  for (int i = first + lane + 64; i < last; i += 64) atomicAdd(&place[wave][key_of(experts[i])], 1);
  __syncthreads();
  // one expert a thread: its count, the prefix over the experts, then the runs' places; slots of none follow all others
  int c = 0;
  if (tid < E) {
    c = before_me[tid] + others[tid];
    if (gridDim.x == 1)
      for (int w = 0; w < used; ++w) c += place[w][tid];
  }
  int p = c;
  for (int o = 1; o < 64; o <<= 1) {
    const int q = __shfl_up(p, o);
    if (lane >= o) p += q;
  }
  if (lane == 63) scan[wave] = p;
  __syncthreads();
  int ahead = 0, all = 0;
  for (int w = 0; w < kSortWaves; ++w) {
    if (w == wave) ahead = all;
    all += scan[w];
  }
  p += ahead - c;
  if (blockIdx.x == 0 && tid < E) offsets[tid] = p;
  if (blockIdx.x == 0 && tid == 0) offsets[E] = all;
  auto runs = [&](int e, int at) {
    for (int w = 0; w < used; ++w) {
      const int q = place[w][e];
      place[w][e] = at;
      at += q;
    }
  };
  if (tid < E) runs(tid, p + before_me[tid]);
  if (tid == kSortThreads - 1) runs(E, all + before_me[E]);
  __syncthreads();
  if (wave >= used) return;
  for (int i0 = first; i0 < last; i0 += 64 * kAhead) {
    int e[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) e[u] = i0 + u * 64 + lane < last ? experts[i0 + u * 64 + lane] : 0;
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int i = i0 + u * 64 + lane, key = key_of(e[u]);
      uint64_t same = __ballot(i < last);
      for (int b = 0; b < bits; ++b) {
        const uint64_t set = __ballot(key >> b & 1);
        same &= key >> b & 1 ? set : ~set;
      }
      if (i < last) {
        const int rank = __popcll(same & ((1ull << lane) - 1)), at = mine[key] + rank;
        order[at] = i;
        positions[i] = key < E ? at : -1 - at;
        if (rank == 0) mine[key] = at + __popcll(same);
      }
    }
  }
}

template <int DT> struct Elem;
template <> struct Elem<MXQ_DT_F32> { typedef float type; };
template <> struct Elem<MXQ_DT_BF16> { typedef __bf16 type; };
template <> struct Elem<MXQ_DT_F16> { typedef _Float16 type; };

// 16 bytes of a row at any address, element i of them as float32; the row's last ones one by one.
template <int DT> struct Pack {
  typedef typename Elem<DT>::type E;
  static constexpr int N = 16 / sizeof(E);
  typedef E Any __attribute__((ext_vector_type(N), aligned(sizeof(E))));
  E v[N];
  __device__ __forceinline__ void load(const E* p, int64_t left) {
    if (left >= N) {
      const Any a = *(const Any*)p;
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = a[i];
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = i < left ? p[i] : (E)0.0f;
    }
  }
  __device__ __forceinline__ void store(E* p, int64_t left) const {
    if (left >= N) {
      Any a;
#pragma unroll
      for (int i = 0; i < N; ++i) a[i] = v[i];
      *(Any*)p = a;
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (i < left) p[i] = v[i];
    }
  }
};

constexpr int kRows = 4;                                          // experts' rows in flight

// Whether a slot's position is a row of y's, and not that of a slot of none, below zero, or past the rows, the caller's
// mistake, which must not reach memory.
__device__ __forceinline__ bool is_row(int position, int rows) { return (uint32_t)position < (uint32_t)rows; }

// out[t] = residual[t] + sum_j w[t, j] y[position[t, j]] in float32, j in order, rounded once.  Reading y bounds it: 16
// bytes a thread, four rows' loads in flight before the first is added.  4096 tokens x 4 x 2048 bfloat16 22.4 us, 4.5 TB/s.
template <int DT> __global__ __launch_bounds__(256) void k_combine(const void* y_, const float* weights, const int32_t* positions,
                                                                   const void* residual_, void* out_, int64_t T, int k, int rows,
                                                                   int64_t D) {
  typedef Pack<DT> P;
  typedef typename P::E E;
  const E *y = (const E*)y_, *residual = (const E*)residual_;
  E* out = (E*)out_;
  const int64_t groups = (D + P::N - 1) / P::N;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < T * groups; i += (int64_t)gridDim.x * 256) {
    const int64_t t = i / groups, d = (i - t * groups) * P::N, left = D - d;
    float sum[P::N];
    P res, row[kRows];
    if (residual) res.load(residual + t * D + d, left);
#pragma unroll
    for (int e = 0; e < P::N; ++e) sum[e] = 0.0f;
    for (int j0 = 0; j0 < k; j0 += kRows) {
      float w[kRows];
      int p[kRows];
#pragma unroll
      for (int j = 0; j < kRows; ++j) {
        const bool in = j0 + j < k;
        w[j] = in ? weights[t * k + j0 + j] : 0.0f;
        p[j] = in ? positions[t * k + j0 + j] : -1;
      }
#pragma unroll
      for (int j = 0; j < kRows; ++j)
        if (is_row(p[j], rows)) row[j].load(y + p[j] * D + d, left);
      if (residual && j0 == 0) {
#pragma unroll
        for (int e = 0; e < P::N; ++e) sum[e] = (float)res.v[e];
      }
#pragma unroll
      for (int j = 0; j < kRows; ++j) {
        if (is_row(p[j], rows)) {
#pragma unroll
          for (int e = 0; e < P::N; ++e) sum[e] = __builtin_fmaf(w[j], (float)row[j].v[e], sum[e]);
        } else if (w[j] != w[j]) {                                // a NaN weight of no expert stays visible
#pragma unroll
          for (int e = 0; e < P::N; ++e) sum[e] = w[j];
        }
      }
    }
    P o;
#pragma unroll
    for (int e = 0; e < P::N; ++e) o.v[e] = (E)sum[e];
    o.store(out + t * D + d, left);
  }
}

// dy[position] = w g[t] (zeros for a slot of no expert), dw = <g[t], y[position]>: a workgroup a token, the gradient's row
// read once for four slots, their rows' loads in flight together.  4096 tokens x 4 x 2048 bfloat16 29.8 us, 5.1 TB/s.
template <int DT> __global__ __launch_bounds__(256) void k_combine_grad(const void* grad_, const void* y_, const float* weights,
                                                                        const int32_t* positions, void* dy_, float* dw, int64_t T,
                                                                        int k, int64_t D) {
  typedef Pack<DT> P;
  typedef typename P::E E;
  __shared__ float part[2][kRows][4];
  const E *y = (const E*)y_, *grad = (const E*)grad_;
  E* dy = (E*)dy_;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int turn = 0;
  for (int64_t t = blockIdx.x; t < T; t += gridDim.x)
    for (int j0 = 0; j0 < k; j0 += kRows, turn ^= 1) {
      float w[kRows], dot[kRows];
      int64_t at[kRows];
      bool there[kRows], live[kRows];                             // a row of dy, one of y
#pragma unroll
      for (int j = 0; j < kRows; ++j) {
        const int p = j0 + j < k ? positions[t * k + j0 + j] : 0, row = p < 0 ? -1 - p : p;
        there[j] = j0 + j < k && row < T * k;
        live[j] = there[j] && p >= 0;
        at[j] = (int64_t)row * D;
        w[j] = live[j] ? weights[t * k + j0 + j] : 0.0f;
        dot[j] = 0.0f;
      }
      for (int64_t d = (int64_t)threadIdx.x * P::N; d < D; d += 256 * P::N) {
        const int64_t left = D - d;
        P g, row[kRows];
        g.load(grad + t * D + d, left);
#pragma unroll
        for (int j = 0; j < kRows; ++j)
          if (dw && live[j]) row[j].load(y + at[j] + d, left);
#pragma unroll
        for (int j = 0; j < kRows; ++j) {
          if (dw && live[j]) {
#pragma unroll
            for (int e = 0; e < P::N; ++e) dot[j] = __builtin_fmaf((float)g.v[e], (float)row[j].v[e], dot[j]);
          }
          if (dy && there[j]) {
            P o;
#pragma unroll
            for (int e = 0; e < P::N; ++e) o.v[e] = (E)(live[j] ? w[j] * (float)g.v[e] : 0.0f);
            o.store(dy + at[j] + d, left);
          }
        }
      }
      if (!dw) continue;
#pragma unroll
      for (int j = 0; j < kRows; ++j) {
        for (int o = 32; o; o >>= 1) dot[j] += __shfl_xor(dot[j], o);
        if (lane == 0) part[turn][j][wave] = dot[j];
      }
      __syncthreads();                                            // the other half of `part` is the next turn's
      if (threadIdx.x < kRows && j0 + (int)threadIdx.x < k) {
        const float* p = part[turn][threadIdx.x];
        dw[t * k + j0 + threadIdx.x] = p[0] + p[1] + p[2] + p[3];
      }
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
  if (n < 0 || n > 0x7fffffff - 8 * kSortThreads * kAhead) return invalid("mxq_dispatch: n out of range");
  if (E < 1 || E > kMaxExperts) return invalid("mxq_dispatch: 1 to 1024 experts");
  if (!offsets || (n && (!experts || !order || !positions))) return invalid("mxq_dispatch: NULL argument");
  int bits = 0;
  while ((E >> bits) != 0) ++bits;                                // keys 0 .. E
  // a workgroup has 1024 slots, or more where that would be over 256 workgroups counting
  const int64_t run = n ? ceil_div(n, 256 * kSortThreads) * 64 : 64, blocks = n ? ceil_div(n, run * kSortWaves) : 1;
  KernelTimer timer("k_dispatch", as_stream(stream));
  k_dispatch<<<dim3((unsigned)blocks), kSortThreads, 0, as_stream(stream)>>>(experts, (int)n, (int)E, bits, (int)run, order, offsets, positions);
  return check_launch("mxq_dispatch");
}

extern "C" int mxq_combine(const void* y, int32_t dtype, const float* weights, const int32_t* positions,
                           const void* residual, void* out, int64_t T, int64_t k, int64_t D, mxq_stream_t stream) {
  if (int rc = check_combine("mxq_combine", dtype, T, k, D)) return rc;
  if (T == 0 || D == 0) return MXQ_OK;
  if (!y || !weights || !positions || !out) return invalid("mxq_combine: NULL argument");
  const int64_t blocks = ceil_div(T * ceil_div(D, dtype == MXQ_DT_F32 ? 4 : 8), 256);
  const dim3 grid(blocks_for(blocks));
  with_dtype(dtype, [&](auto dt) {
    KernelTimer timer("k_combine", as_stream(stream));
    k_combine<decltype(dt)::value><<<grid, 256, 0, as_stream(stream)>>>(y, weights, positions, residual, out, T, (int)k, (int)(T * k), D);
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
    k_combine_grad<decltype(dt)::value><<<dim3(blocks_for(T)), 256, 0, as_stream(stream)>>>(grad, y, weights, positions, dy, dw, T,
                                                                                         (int)k, D);
  });
  return check_launch("mxq_combine_grad");
}
