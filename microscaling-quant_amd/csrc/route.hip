// Routing of tokens to experts, and the gradient of its weights (include/mxq_hip.h, mxq_route).
//
//   s_e = softmax(l)_e or 1 / (1 + exp(-l_e));  r_e = s_e + bias_e, -inf where l_e = -inf
//   groups > 1: a group's score is the sum of its two best r; experts outside the top_groups best groups: r = -inf
//   the k experts of largest r, ties to the lowest index;  w_j = scale s_{e_j} [/ sum of the k s]
//
// Scores are 64-bit: an expert is taken or left by values that lie close together (16384 tokens of 256 experts hold a pair
// of neighbours at rank k within 1e-8 of each other), and float32's exp would decide those by its rounding.
//
// Up to 512 experts a token has 16 lanes, so that a maximum over its lanes is four rotations within a row of lanes and a
// wave chooses for four tokens at once; beyond, a whole wave.  Expert e is register e / L of lane e % L.  What bounds it is
// instructions, most of them of 64 bits: of four tokens of 256 experts a wave issues 990 vector instructions for the scores,
// 380 for 8 groups and 150 a choice, 2571 with 8 of them, counted.  16384 such tokens: the SIMDs issue them in 42 of the 51
// thousand cycles a CU is busy, 24 us; reading the logits would take 4.
#include "mxq_common.h"

namespace mxq {
namespace {

constexpr int kWaves = 4;
constexpr int kMaxExperts = 1024, kMaxTopK = 64, kMaxGroups = 64;

template <int DT> __device__ __forceinline__ float load_as_float(const void* p, int64_t i) {
  if constexpr (DT == MXQ_DT_F32) return ((const float*)p)[i];
  if constexpr (DT == MXQ_DT_BF16) return __uint_as_float((uint32_t)((const uint16_t*)p)[i] << 16);
  return (float)((const _Float16*)p)[i];
}

template <int DT> __device__ __forceinline__ void store_from_float(void* p, int64_t i, float v) {
  if constexpr (DT == MXQ_DT_F32) ((float*)p)[i] = v;
  if constexpr (DT == MXQ_DT_BF16) ((__bf16*)p)[i] = (__bf16)v;
  if constexpr (DT == MXQ_DT_F16) ((_Float16*)p)[i] = (_Float16)v;
}

// Rotation by N within each row of 16 lanes.
template <int N> __device__ __forceinline__ int rotate(int v) { return __builtin_amdgcn_update_dpp(v, v, 0x120 + N, 0xF, 0xF, false); }
template <int N> __device__ __forceinline__ float rotate(float v) { return __int_as_float(rotate<N>(__float_as_int(v))); }
template <int N> __device__ __forceinline__ double rotate(double v) {
  const uint64_t b = __double_as_longlong(v);
  const uint32_t lo = rotate<N>((int)(uint32_t)b), hi = rotate<N>((int)(uint32_t)(b >> 32));
  return __longlong_as_double((uint64_t)hi << 32 | lo);
}
// f over the L lanes of a token, the same value in each.
template <int L, typename T, typename F> __device__ __forceinline__ T over_lanes(T v, F f) {
  v = f(v, rotate<8>(v));
  v = f(v, rotate<4>(v));
  v = f(v, rotate<2>(v));
  v = f(v, rotate<1>(v));
  if constexpr (L == 64) {
    v = f(v, __shfl_xor(v, 16));
    v = f(v, __shfl_xor(v, 32));
  }
  return v;
}
template <int L> __device__ __forceinline__ double lanes_max(double v) {
  return over_lanes<L>(v, [](double a, double b) { return fmax(a, b); });
}
template <int L> __device__ __forceinline__ double lanes_sum(double v) {
  return over_lanes<L>(v, [](double a, double b) { return a + b; });
}
template <int L> __device__ __forceinline__ int lanes_min(int v) {
  return over_lanes<L>(v, [](int a, int b) { return a < b ? a : b; });
}
template <int L> __device__ __forceinline__ bool lanes_any(bool b) {
  const uint64_t all = __ballot(b);
  if constexpr (L == 64) return all != 0;
  return (all >> (threadIdx.x & 48) & 0xFFFF) != 0;
}

// x[i] = e^x[i] for x <= 709, zero below -746: x = n ln 2 + r with |r| <= ln(2) / 2, Taylor's series of e^r to r^13 (the
// next term is below 4e-18), times 2^n.  Up to eight at a time, so that a coefficient is put into registers once for them.
template <int V> __device__ __forceinline__ void exp64(double (&x)[V]) {
  constexpr int G = V < 8 ? V : 8;
  constexpr double kFactorials[14] = {1.0, 1.0, 2.0, 6.0, 24.0, 120.0, 720.0, 5040.0, 40320.0, 362880.0, 3628800.0, 39916800.0, 479001600.0,
                                      6227020800.0};
#pragma unroll
  for (int v = 0; v < V; v += G) {
    double r[G], p[G];
    int n[G];
#pragma unroll
    for (int i = 0; i < G; ++i) {
      const double y = fmin(fmax(x[v + i], -746.0), 709.0), whole = rint(y * 1.4426950408889634);
      r[i] = fma(whole, -2.3190468138462996e-17, fma(whole, -0.69314718055994531, y));
      n[i] = (int)whole;
      p[i] = 1.0 / kFactorials[13];
    }
#pragma unroll
    for (int c = 12; c >= 0; --c) {
      double coefficient = 1.0 / kFactorials[c];
      asm("" : "+v"(coefficient));                                // once for all, not once an element
#pragma unroll
      for (int i = 0; i < G; ++i) p[i] = fma(p[i], r[i], coefficient);
    }
#pragma unroll
    for (int i = 0; i < G; ++i) x[v + i] = __builtin_ldexp(p[i], n[i]);
  }
}

// 1 / d for 1 <= d < 2^1000: the hardware's estimate and two steps of Newton's iteration.
__device__ __forceinline__ double inverse(double d) {
  double y = __builtin_amdgcn_rcp(d);
  y = fma(fma(-d, y, 1.0), y, y);
  return fma(fma(-d, y, 1.0), y, y);
}

// The row's largest logit and the inverse of its sum of powers, under softmax.
struct Norm {
  double top, inverse;
};

// s[i]: the scores of the logits l[i].
template <int V> __device__ __forceinline__ void scores_of(const float (&l)[V], int softmax, const Norm& n, double (&s)[V]) {
#pragma unroll
  for (int v = 0; v < V; ++v) s[v] = softmax ? (double)l[v] - n.top : -(double)l[v];
  exp64(s);
#pragma unroll
  for (int v = 0; v < V; ++v) s[v] = softmax ? s[v] * n.inverse : -l[v] > 709.0f ? 0.0 : inverse(1.0 + s[v]);
}

// l[]: the lane's logits, s[]: their scores; true if the row holds a NaN, or +inf under softmax, which has no score.
template <int DT, int L, int V> __device__ __forceinline__ bool row_scores(const void* logits, int64_t row, int E, int softmax, float (&l)[V],
                                                                           double (&s)[V], Norm& n) {
  const int lane = threadIdx.x & (L - 1);
  bool bad = false;
  float top = -INFINITY;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int e = v * L + lane;
    l[v] = load_as_float<DT>(logits, row * E + (e < E ? e : E - 1));
  }
#pragma unroll
  for (int v = 0; v < V; ++v) {
    if (v * L + lane >= E) l[v] = -INFINITY;
    bad |= l[v] != l[v] || (softmax && l[v] == INFINITY);
    top = fmaxf(top, l[v]);
  }
  bad = lanes_any<L>(bad);
  n = Norm{0.0, 1.0};
  if (softmax) {
    top = over_lanes<L>(top, [](float a, float b) { return fmaxf(a, b); });
    n.top = top == -INFINITY ? 0.0 : (double)top;
  }
  scores_of(l, softmax, n, s);
  if (softmax) {
    double sum = 0.0;
#pragma unroll
    for (int v = 0; v < V; ++v) sum += s[v];
    sum = lanes_sum<L>(sum);
    n.inverse = sum < 1.0 ? 1.0 : inverse(sum);                   // an open row's sum is at least 1
#pragma unroll
    for (int v = 0; v < V; ++v) s[v] *= n.inverse;
  }
  return bad;
}

template <int DT, int L, int V, int SLOTS>
__global__ __launch_bounds__(64 * kWaves) void k_route(const void* logits, const float* bias, int64_t T, int E,
                                                       mxq_route_spec sp, DivU31 per, float* weights, int32_t* experts) {
  extern __shared__ double shared[];                              // groups > 1: E ranks and 64 scores a token
  const int lane = threadIdx.x & (L - 1), token = threadIdx.x / L;
  const int64_t at = (int64_t)blockIdx.x * (blockDim.x / L) + token, row = at < T ? at : T - 1;
  const bool softmax = sp.score == MXQ_SCORE_SOFTMAX, out = at < T;     // lanes past the end go along: the row's lanes work together
  const int k = sp.top_k;
  float l[V];
  double r[V];
  Norm norm;
  bool bad = row_scores<DT, L, V>(logits, row, E, softmax, l, r, norm);
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int e = v * L + lane;
    if (bias && e < E) r[v] += (double)bias[e];
    if (l[v] == -INFINITY) r[v] = -INFINITY;
    bad |= r[v] != r[v];
  }
  bad = lanes_any<L>(bad);
  if (sp.groups > 1) {
    double* ranks = shared + (size_t)token * (E + kMaxGroups);
    double* scores = ranks + E;
    auto in_order = [&]() {                                       // the wave's own LDS writes before its reads
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
    };
#pragma unroll
    for (int v = 0; v < V; ++v)
      if (v * L + lane < E) ranks[v * L + lane] = r[v];
    in_order();
    for (int g = lane; g < sp.groups; g += L) {
      double a = -INFINITY, b = -INFINITY;
#pragma unroll 4
      for (int j = 0; j < (int)per.d; ++j) {
        const double x = ranks[g * per.d + j];
        b = fmax(b, fmin(a, x));
        a = fmax(a, x);
      }
      scores[g] = b == -INFINITY ? a : a + b;
    }
    in_order();
    // a group is kept if fewer than top_groups come before it
    uint64_t kept = 0;
    for (int g0 = 0; g0 < sp.groups; g0 += L) {
      const int g = g0 + lane;
      const double mine = g < sp.groups ? scores[g] : 0.0;
      int before = 0;
#pragma unroll 4
      for (int h = 0; h < sp.groups; ++h) {
        const double x = scores[h];
        before += x > mine || (x == mine && h < g);
      }
      const uint64_t all = __ballot(g < sp.groups && before < sp.top_groups);
      kept |= (L == 64 ? all : all >> (threadIdx.x & 48) & 0xFFFF) << g0;
    }
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const uint32_t g = divu31(v * L + lane, per);
      if (!(kept >> (g & 63) & 1)) r[v] = -INFINITY;
    }
  }
  int pick[SLOTS];
#pragma unroll
  for (int q = 0; q < SLOTS; ++q) {
    pick[q] = -1;
    for (int j = q * L; j < k && j < (q + 1) * L; ++j) {
      double best = r[0];
#pragma unroll
      for (int v = 1; v < V; ++v) best = fmax(best, r[v]);
      best = lanes_max<L>(best);
      int i = 0x7fffffff;
#pragma unroll
      for (int v = V - 1; v >= 0; --v)
        if (r[v] == best) i = v * L + lane;
      i = lanes_min<L>(i);
      if (lane == j - q * L && best > -INFINITY) pick[q] = i;
#pragma unroll
      for (int v = 0; v < V; ++v)
        if (i == v * L + lane) r[v] = -INFINITY;
    }
  }
  double total = 0.0;
  float chosen[SLOTS];
  double own[SLOTS];
#pragma unroll
  for (int q = 0; q < SLOTS; ++q) chosen[q] = load_as_float<DT>(logits, row * E + (pick[q] >= 0 && !bad ? pick[q] : 0));
  scores_of(chosen, softmax, norm, own);                          // the bits they were chosen by
#pragma unroll
  for (int q = 0; q < SLOTS; ++q) {
    if (pick[q] < 0 || bad) own[q] = 0.0;
    total += own[q];
  }
  total = lanes_sum<L>(total);
  if (!sp.renormalize || total == 0.0) total = 1.0;
#pragma unroll
  for (int q = 0; q < SLOTS; ++q) {
    const int j = q * L + lane;
    if (j >= k || !out) continue;
    weights[row * k + j] = bad ? NAN : (float)(own[q] / total * (double)sp.scale);
    experts[row * k + j] = bad ? -1 : pick[q];
  }
}

// The gradient of the logits: with u_j the chosen scores and U their sum, du_j = scale (g_j - sum_i g_i u_i / U) / U
// where renormalized, scale g_j otherwise; softmax: dl_e = s_e (du_e - sum_j du_j u_j); sigmoid: dl_e = du_e s_e (1 - s_e).
template <int DT, int L, int V, int SLOTS>
__global__ __launch_bounds__(64 * kWaves) void k_route_grad(const void* logits, const int32_t* experts, const float* grad,
                                                            int64_t T, int E, mxq_route_spec sp, void* out) {
  const int lane = threadIdx.x & (L - 1), first = threadIdx.x & 63 & ~(L - 1);
  const int64_t at = (int64_t)blockIdx.x * (64 * kWaves / L) + threadIdx.x / L, row = at < T ? at : T - 1;
  const bool softmax = sp.score == MXQ_SCORE_SOFTMAX;
  const int k = sp.top_k;
  float l[V];
  double s[V], d[V];
  Norm norm;
  const bool bad = row_scores<DT, L, V>(logits, row, E, softmax, l, s, norm);
  int pick[SLOTS];
  float chosen[SLOTS];
  double u[SLOTS], du[SLOTS], U = 0.0, gu = 0.0;
#pragma unroll
  for (int q = 0; q < SLOTS; ++q) {
    const int j = q * L + lane;
    const int e = j < k ? experts[row * k + j] : -1;
    pick[q] = e < E ? e : -1;
    chosen[q] = load_as_float<DT>(logits, row * E + (pick[q] >= 0 ? pick[q] : 0));
  }
  scores_of(chosen, softmax, norm, u);
#pragma unroll
  for (int q = 0; q < SLOTS; ++q) {
    const int j = q * L + lane;
    if (pick[q] < 0) u[q] = 0.0;
    du[q] = pick[q] >= 0 ? (double)grad[row * k + j] * (double)sp.scale : 0.0;
    U += u[q];
    gu += du[q] * u[q];
  }
  if (sp.renormalize) {
    U = lanes_sum<L>(U);
    gu = lanes_sum<L>(gu);
    if (U == 0.0) U = 1.0;
    const double mean = gu / U;
#pragma unroll
    for (int q = 0; q < SLOTS; ++q) du[q] = pick[q] >= 0 ? (du[q] - mean) / U : 0.0;
  }
  double dot = 0.0;
#pragma unroll
  for (int q = 0; q < SLOTS; ++q) dot += du[q] * u[q];
  dot = softmax ? lanes_sum<L>(dot) : 0.0;
#pragma unroll
  for (int v = 0; v < V; ++v) d[v] = 0.0;
#pragma unroll
  for (int q = 0; q < SLOTS; ++q)
    for (int j = q * L; j < k && j < (q + 1) * L; ++j) {
      const int e = __shfl(pick[q], first + j - q * L);
      const double x = __shfl(du[q], first + j - q * L);
#pragma unroll
      for (int v = 0; v < V; ++v)
        if (e == v * L + lane) d[v] = x;
    }
  if (at >= T) return;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int e = v * L + lane;
    const double x = softmax ? s[v] * (d[v] - dot) : d[v] * s[v] * (1.0 - s[v]);
    if (e < E) store_from_float<DT>(out, row * E + e, bad ? NAN : (float)x);
  }
}

int check_spec(const char* who, int32_t dtype, int64_t T, int64_t E, const mxq_route_spec* sp) {
  const std::string w(who);
  if (!sp) return invalid(w + ": NULL spec");
  if (dtype < MXQ_DT_F32 || dtype > MXQ_DT_F16) return invalid(w + ": unknown dtype");
  if (T < 0 || T > (int64_t)kWaves * 0x7fffffff) return invalid(w + ": T out of range");
  if (E < 1 || E > kMaxExperts) return invalid(w + ": 1 to 1024 experts");
  if (sp->top_k < 1 || sp->top_k > kMaxTopK || sp->top_k > E) return invalid(w + ": top_k must be 1 to min(64, experts)");
  if (sp->groups < 1 || sp->groups > kMaxGroups || E % sp->groups) return invalid(w + ": groups must divide the experts, at most 64");
  if (sp->top_groups < 1 || sp->top_groups > sp->groups) return invalid(w + ": top_groups must be 1 to groups");
  if (sp->score != MXQ_SCORE_SOFTMAX && sp->score != MXQ_SCORE_SIGMOID) return invalid(w + ": unknown score");
  return MXQ_OK;
}

// f(DT, L, V, SLOTS): the dtype, the lanes of a token, the registers and the choices of a lane, as compile-time constants.
template <typename F> void with_shape(int32_t dtype, int64_t E, int k, F f) {
  auto by_choices = [&](auto dt, auto v) {
    std::integral_constant<int, 16> row;
    if (k <= 16) f(dt, row, v, std::integral_constant<int, 1>());
    else f(dt, row, v, std::integral_constant<int, 4>());
  };
  auto by_experts = [&](auto dt) {
    if (E <= 16) f(dt, std::integral_constant<int, 16>(), std::integral_constant<int, 1>(), std::integral_constant<int, 1>());
    else if (E <= 32) by_choices(dt, std::integral_constant<int, 2>());
    else if (E <= 64) by_choices(dt, std::integral_constant<int, 4>());
    else if (E <= 128) by_choices(dt, std::integral_constant<int, 8>());
    else if (E <= 256) by_choices(dt, std::integral_constant<int, 16>());
    else if (E <= 512) by_choices(dt, std::integral_constant<int, 32>());
    else f(dt, std::integral_constant<int, 64>(), std::integral_constant<int, 16>(), std::integral_constant<int, 1>());
  };
  if (dtype == MXQ_DT_F32) by_experts(std::integral_constant<int, MXQ_DT_F32>());
  else if (dtype == MXQ_DT_BF16) by_experts(std::integral_constant<int, MXQ_DT_BF16>());
  else by_experts(std::integral_constant<int, MXQ_DT_F16>());
}

}  // namespace
}  // namespace mxq

using namespace mxq;

extern "C" int mxq_route(const void* logits, int32_t dtype, const float* bias, int64_t T, int64_t E,
                         const mxq_route_spec* spec, float* weights, int32_t* experts, mxq_stream_t stream) {
  if (int rc = check_spec("mxq_route", dtype, T, E, spec)) return rc;
  if (T == 0) return MXQ_OK;
  if (!logits || !weights || !experts) return invalid("mxq_route: NULL argument");
  with_shape(dtype, E, spec->top_k, [&](auto dt, auto lanes, auto v, auto slots) {
    constexpr int L = decltype(lanes)::value;
    const int threads = spec->groups > 1 && E > 256 ? 32 * kWaves : 64 * kWaves, tokens = threads / L;   // below 64 KB of LDS
    constexpr size_t size = decltype(dt)::value == MXQ_DT_F32 ? 4 : 2;
    const size_t lds = spec->groups > 1 ? tokens * (size_t)(E + kMaxGroups) * sizeof(double) : 0;
    for (int64_t t = 0, n; t < T; t += n) {
      n = T - t < kMaxBlocks * tokens ? T - t : kMaxBlocks * tokens;
      KernelTimer timer("k_route", as_stream(stream));
      k_route<decltype(dt)::value, L, decltype(v)::value, decltype(slots)::value><<<dim3((unsigned)ceil_div(n, tokens)), threads, lds, as_stream(stream)>>>(
          (const char*)logits + t * E * size, bias, n, (int)E, *spec, make_divu31((uint32_t)(E / spec->groups)), weights + t * spec->top_k,
          experts + t * spec->top_k);
    }
  });
  return check_launch("mxq_route");
}

extern "C" int mxq_route_grad(const void* logits, int32_t dtype, const int32_t* experts, const float* grad, int64_t T,
                              int64_t E, const mxq_route_spec* spec, void* out, mxq_stream_t stream) {
  if (int rc = check_spec("mxq_route_grad", dtype, T, E, spec)) return rc;
  if (T == 0) return MXQ_OK;
  if (!logits || !experts || !grad || !out) return invalid("mxq_route_grad: NULL argument");
  with_shape(dtype, E, spec->top_k, [&](auto dt, auto lanes, auto v, auto slots) {
    constexpr int L = decltype(lanes)::value, kTokens = 64 * kWaves / L;
    constexpr size_t size = decltype(dt)::value == MXQ_DT_F32 ? 4 : 2;
    for (int64_t t = 0, n; t < T; t += n) {
      n = T - t < kMaxBlocks * kTokens ? T - t : kMaxBlocks * kTokens;
      KernelTimer timer("k_route_grad", as_stream(stream));
      k_route_grad<decltype(dt)::value, L, decltype(v)::value, decltype(slots)::value><<<dim3((unsigned)ceil_div(n, kTokens)), 64 * kWaves, 0, as_stream(stream)>>>(
          (const char*)logits + t * E * size, experts + t * spec->top_k, grad + t * spec->top_k, n, (int)E, *spec, (char*)out + t * E * size);
    }
  });
  return check_launch("mxq_route_grad");
}
