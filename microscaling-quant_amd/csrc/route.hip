// Routing of tokens to experts, and the gradient of its weights (include/mxq_hip.h, mxq_route).
//
//   s_e = softmax(l)_e or 1 / (1 + exp(-l_e));  r_e = s_e + bias_e, -inf where l_e = -inf
//   groups > 1: a group's score is the sum of its two best r; experts outside the top_groups best groups: r = -inf
//   the k experts of largest r, ties to the lowest index;  w_j = scale s_{e_j} [/ sum of the k s]
//
// One wave a token, expert e in register e / 64 of lane e % 64.  Scores are 64-bit: an expert is taken or left by values
// that lie close together (16384 tokens of 256 experts hold a pair of neighbours at rank k within 1e-8 of each other),
// and float32's exp would decide those by its rounding.
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

__device__ __forceinline__ double wave_max(double v) {
  for (int o = 32; o; o >>= 1) v = fmax(v, __shfl_xor(v, o));
  return v;
}
__device__ __forceinline__ double wave_sum(double v) {
  for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
  return v;
}

// The wave's best (value, index), the larger value first, the lower index among equals.
__device__ __forceinline__ void wave_best(double& v, int& i) {
  for (int o = 32; o; o >>= 1) {
    const double ov = __shfl_xor(v, o);
    const int oi = __shfl_xor(i, o);
    if (ov > v || (ov == v && oi < i)) v = ov, i = oi;
  }
}

// s[]: the scores of the lane's experts; true if the row holds a NaN, or +inf under softmax, which has no score.
template <int DT, int V> __device__ __forceinline__ bool scores_of(const void* logits, int64_t row, int E, int softmax,
                                                                   float (&l)[V], double (&s)[V]) {
  const int lane = threadIdx.x & 63;
  double top = -INFINITY;
  bool bad = false;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int e = v * 64 + lane;
    l[v] = e < E ? load_as_float<DT>(logits, row * E + e) : -INFINITY;
    bad |= l[v] != l[v] || (softmax && l[v] == INFINITY);
    top = fmax(top, (double)l[v]);
  }
  bad = __any(bad);
  if (softmax) {
    top = wave_max(top);
    if (top == -INFINITY) top = 0.0;
    double sum = 0.0;
#pragma unroll
    for (int v = 0; v < V; ++v) sum += s[v] = exp((double)l[v] - top);
    sum = wave_sum(sum);
    if (sum == 0.0) sum = 1.0;
#pragma unroll
    for (int v = 0; v < V; ++v) s[v] /= sum;
  } else {
#pragma unroll
    for (int v = 0; v < V; ++v) s[v] = 1.0 / (1.0 + exp(-(double)l[v]));
  }
  return bad;
}

template <int DT, int V>
__global__ __launch_bounds__(64 * kWaves) void k_route(const void* logits, const float* bias, int64_t T, int E,
                                                       mxq_route_spec sp, float* weights, int32_t* experts) {
  __shared__ double ranked[kWaves][V * 64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t row = (int64_t)blockIdx.x * kWaves + wave;
  if (row >= T) return;
  const int k = sp.top_k;
  float l[V];
  double s[V], r[V];
  bool bad = scores_of<DT, V>(logits, row, E, sp.score == MXQ_SCORE_SOFTMAX, l, s);
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int e = v * 64 + lane;
    r[v] = bias && e < E ? s[v] + (double)bias[e] : s[v];
    if (l[v] == -INFINITY) r[v] = -INFINITY;
    bad |= r[v] != r[v];
  }
  if (__any(bad)) {
    if (lane < k) weights[row * k + lane] = NAN, experts[row * k + lane] = -1;
    return;
  }
  if (sp.groups > 1) {
    double* mine = ranked[wave];
#pragma unroll
    for (int v = 0; v < V; ++v) mine[v * 64 + lane] = r[v];
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    const int per = E / sp.groups;
    double a = -INFINITY, b = -INFINITY;
    if (lane < sp.groups)
      for (int j = 0; j < per; ++j) {
        const double x = mine[lane * per + j];
        if (x > a) b = a, a = x;
        else if (x > b) b = x;
      }
    double score = a == -INFINITY ? a : b == -INFINITY ? a : a + b;
    uint64_t kept = 0;
    for (int j = 0; j < sp.top_groups; ++j) {
      double x = score;
      int i = lane < sp.groups && !(kept >> lane & 1) ? lane : 64;
      if (i == 64) x = -INFINITY;
      wave_best(x, i);
      if (i < 64) kept |= 1ull << i;
    }
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int g = (v * 64 + lane) / per;
      if (g >= sp.groups || !(kept >> g & 1)) r[v] = -INFINITY;
    }
  }
  double own = 0.0;
  int pick = -1;
  for (int j = 0; j < k; ++j) {
    double x = r[0], sx = s[0];
    int i = lane;
#pragma unroll
    for (int v = 1; v < V; ++v)
      if (r[v] > x) x = r[v], sx = s[v], i = v * 64 + lane;
    wave_best(x, i);
    if (x == -INFINITY) break;
    sx = __shfl(sx, i & 63);
    if (lane == j) own = sx, pick = i;
#pragma unroll
    for (int v = 0; v < V; ++v)
      if (i == v * 64 + lane) r[v] = -INFINITY;
  }
  double total = 1.0;
  if (sp.renormalize) {
    total = wave_sum(own);
    if (total == 0.0) total = 1.0;
  }
  if (lane < k) {
    weights[row * k + lane] = (float)(own / total * (double)sp.scale);
    experts[row * k + lane] = pick;
  }
}

// The gradient of the logits: with u_j the chosen scores and U their sum, du_j = scale (g_j - sum_i g_i u_i / U) / U
// where renormalized, scale g_j otherwise; softmax: dl_e = s_e (du_e - sum_j du_j u_j); sigmoid: dl_e = du_e s_e (1 - s_e).
template <int DT, int V>
__global__ __launch_bounds__(64 * kWaves) void k_route_grad(const void* logits, const int32_t* experts, const float* grad,
                                                            int64_t T, int E, mxq_route_spec sp, void* out) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t row = (int64_t)blockIdx.x * kWaves + wave;
  if (row >= T) return;
  const int k = sp.top_k;
  float l[V];
  double s[V], d[V];
  const bool bad = scores_of<DT, V>(logits, row, E, sp.score == MXQ_SCORE_SOFTMAX, l, s);
  const int pick = lane < k ? experts[row * k + lane] : -1;
  const double g = lane < k && pick >= 0 ? (double)grad[row * k + lane] : 0.0;
  double u = 0.0;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const double x = __shfl(s[v], pick & 63);
    if (pick >= 0 && pick >> 6 == v) u = x;
    d[v] = 0.0;
  }
  double du = g * (double)sp.scale;
  if (sp.renormalize) {
    double U = wave_sum(u);
    if (U == 0.0) U = 1.0;
    du = (du - wave_sum(du * u) / U) / U;
    if (pick < 0) du = 0.0;
  }
  const double dot = sp.score == MXQ_SCORE_SOFTMAX ? wave_sum(du * u) : 0.0;
  for (int j = 0; j < k; ++j) {
    const int e = __shfl(pick, j);
    const double x = __shfl(du, j);
#pragma unroll
    for (int v = 0; v < V; ++v)
      if (e == v * 64 + lane) d[v] = x;
  }
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int e = v * 64 + lane;
    double x = sp.score == MXQ_SCORE_SOFTMAX ? s[v] * (d[v] - dot) : d[v] * s[v] * (1.0 - s[v]);
    if (bad) x = NAN;
    if (e < E) store_from_float<DT>(out, row * E + e, (float)x);
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

// f(DT, V) with the dtype and the registers a lane needs for E experts as compile-time constants.
template <typename F> void with_shape(int32_t dtype, int64_t E, F f) {
  auto by_v = [&](auto dt) {
    if (E <= 64) f(dt, std::integral_constant<int, 1>());
    else if (E <= 128) f(dt, std::integral_constant<int, 2>());
    else if (E <= 256) f(dt, std::integral_constant<int, 4>());
    else if (E <= 512) f(dt, std::integral_constant<int, 8>());
    else f(dt, std::integral_constant<int, 16>());
  };
  if (dtype == MXQ_DT_F32) by_v(std::integral_constant<int, MXQ_DT_F32>());
  else if (dtype == MXQ_DT_BF16) by_v(std::integral_constant<int, MXQ_DT_BF16>());
  else by_v(std::integral_constant<int, MXQ_DT_F16>());
}

}  // namespace
}  // namespace mxq

using namespace mxq;

extern "C" int mxq_route(const void* logits, int32_t dtype, const float* bias, int64_t T, int64_t E,
                         const mxq_route_spec* spec, float* weights, int32_t* experts, mxq_stream_t stream) {
  if (int rc = check_spec("mxq_route", dtype, T, E, spec)) return rc;
  if (T == 0) return MXQ_OK;
  if (!logits || !weights || !experts) return invalid("mxq_route: NULL argument");
  with_shape(dtype, E, [&](auto dt, auto v) {
    KernelTimer timer("k_route", as_stream(stream));
    k_route<decltype(dt)::value, decltype(v)::value><<<dim3((unsigned)ceil_div(T, kWaves)), 64 * kWaves, 0, as_stream(stream)>>>(
        logits, bias, T, (int)E, *spec, weights, experts);
  });
  return check_launch("mxq_route");
}

extern "C" int mxq_route_grad(const void* logits, int32_t dtype, const int32_t* experts, const float* grad, int64_t T,
                              int64_t E, const mxq_route_spec* spec, void* out, mxq_stream_t stream) {
  if (int rc = check_spec("mxq_route_grad", dtype, T, E, spec)) return rc;
  if (T == 0) return MXQ_OK;
  if (!logits || !experts || !grad || !out) return invalid("mxq_route_grad: NULL argument");
  with_shape(dtype, E, [&](auto dt, auto v) {
    KernelTimer timer("k_route_grad", as_stream(stream));
    k_route_grad<decltype(dt)::value, decltype(v)::value><<<dim3((unsigned)ceil_div(T, kWaves)), 64 * kWaves, 0, as_stream(stream)>>>(
        logits, experts, grad, T, (int)E, *spec, out);
  });
  return check_launch("mxq_route_grad");
}
