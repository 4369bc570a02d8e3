// libqbnn_hip.so: the router of a layer of experts and the sum of the experts' results.
//   scores    s = softmax(l) or sigmoid(l) over a row's E logits;  key = s + bias (what is compared), weight = s (what is multiplied)
//   groups    E / groups neighbouring experts each; a group counts its two largest keys, the best `top_groups` groups stay
//   choice    the top_k largest keys, ties to the lowest index; weights optionally divided by their sum, times `scale`
//   order     the (row, choice) pairs of a sample sorted by expert, stable: what the experts' products walk
// Keys are compared as 64-bit values: two experts whose scores differ only behind fp32's last place are still told apart, so the choice
// does not depend on the order in which a row's sum was taken.
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <stdio.h>
#include <float.h>
#include <math.h>

#include "../../include/qbnn.h"
#include "qbnn_common.h"
#include "qbnn_f8.h"

using namespace qbnn;

namespace {

static inline int route_fail(const char* fmt, long a = 0, long b = 0) {
  char buf[512];
  snprintf(buf, sizeof(buf), fmt, a, b);
  return qbnn_fail_msg(QBNN_E_INVALID, buf);
}

constexpr int ROUTE_ROWS = 64;         // rows of a sample per workgroup = the unit of the counting sort

struct RouteArgs {
  const void* logits; int64_t l_ss, l_rs;
  const float* bias;
  float* weights; int32_t* experts; int32_t* offsets; int32_t* rows; int32_t* counts;      // counts [S][blocks][E]
  int S, T, E, k, groups, kept, sigmoid, renorm, blocks;
  float scale;
};

template <int T> __device__ __forceinline__ float route_lowest() {
  if constexpr (T == QBNN_BF16) return -3.3895313892515355e38f;
  else if constexpr (T == QBNN_F16) return -65504.f;
  else return -FLT_MAX;
}
__device__ __forceinline__ double shfl_xor_f64(double v, int d) { return __shfl_xor(v, d); }

template <int T, int CH> __global__ __launch_bounds__(256) void route_kernel(const RouteArgs a) {
  __shared__ int hist[CH * 64];
  __shared__ double keys[4][CH * 64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int s = blockIdx.y, t0 = blockIdx.x * ROUTE_ROWS, t1 = min(a.T, t0 + ROUTE_ROWS);
  for (int i = threadIdx.x; i < a.E; i += 256) hist[i] = 0;
  __syncthreads();
  const int per = a.E / a.groups;
  const bool by_logit = !a.bias && a.groups == 1;             // both scores increase with the logit
  for (int t = t0 + wave; t < t1; t += 4) {
    const f8_type<T>* l = (const f8_type<T>*)a.logits + s * a.l_ss + t * a.l_rs;
    float v[CH];
    bool open[CH], nan = false;
    float top = -INFINITY;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int e = c * 64 + lane;
      v[c] = e < a.E ? f8_load<T>(l[e]) : -INFINITY;
      open[c] = v[c] > route_lowest<T>();                     // -inf, the type's lowest value and NaN are masked
      nan |= v[c] != v[c];
      if (open[c]) top = fmaxf(top, v[c]);
    }
    nan = __any(nan);
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) top = fmaxf(top, __shfl_xor(top, d));
    double p[CH], sum = 0.;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      p[c] = !open[c] ? 0. : a.sigmoid ? 1. / (1. + exp(-(double)v[c])) : exp((double)v[c] - (double)top);
      sum += p[c];
    }
    if (!a.sigmoid) {
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) sum += shfl_xor_f64(sum, d);
#pragma unroll
      for (int c = 0; c < CH; ++c) if (open[c]) p[c] /= sum;
    }
    double key[CH];
    int idx[CH];
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int e = c * 64 + lane;
      double q = by_logit ? (double)v[c] : p[c] + (a.bias && e < a.E ? (double)a.bias[e] : 0.);
      key[c] = open[c] && q == q ? q : -INFINITY;
      idx[c] = e < a.E ? e : 0x7fffffff;
    }
    if (a.groups > 1) {
      // lane g sums group g's two largest keys (masked experts left out; a group of masked experts ranks last)
#pragma unroll
      for (int c = 0; c < CH; ++c) keys[wave][c * 64 + lane] = key[c];
      __builtin_amdgcn_wave_barrier();
      double a1 = -INFINITY, a2 = -INFINITY;
      if (lane < a.groups)
        for (int i = 0; i < per; ++i) {
          const double q = keys[wave][lane * per + i];
          if (q > a1) { a2 = a1; a1 = q; } else if (q > a2) a2 = q;
        }
      const double g = a1 == -INFINITY ? -INFINITY : a2 == -INFINITY ? a1 : a1 + a2;
      int rank = 0;
      for (int i = 0; i < a.groups; ++i) {
        const double o = __shfl(g, i);
        rank += o > g || (o == g && i < lane) ? 1 : 0;
      }
      const unsigned long long stay = __ballot(lane < a.groups && rank < a.kept);
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        const int e = c * 64 + lane;
        if (e < a.E && !((stay >> (e / per)) & 1)) { key[c] = -INFINITY; idx[c] = 0x7fffffff; }
      }
      __builtin_amdgcn_wave_barrier();
    }
    int my_e = 0;
    double my_p = 0.;
    for (int j = 0; j < a.k; ++j) {
      double b = key[0], bp = p[0];
      int bi = idx[0];
#pragma unroll
      for (int c = 1; c < CH; ++c)
        if (key[c] > b || (key[c] == b && idx[c] < bi)) { b = key[c]; bi = idx[c]; bp = p[c]; }
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) {
        const double ob = shfl_xor_f64(b, d), op = shfl_xor_f64(bp, d);
        const int oi = __shfl_xor(bi, d);
        if (ob > b || (ob == b && oi < bi)) { b = ob; bi = oi; bp = op; }
      }
#pragma unroll
      for (int c = 0; c < CH; ++c) if (idx[c] == bi) { key[c] = -INFINITY; idx[c] = 0x7fffffff; }
      if (lane == j) { my_e = bi; my_p = bp; }
    }
    double total = 0.;
    if (a.renorm) {
      total = lane < a.k ? my_p : 0.;
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) total += shfl_xor_f64(total, d);
    }
    if (lane < a.k) {
      const double w = a.renorm ? (total == 0. ? 0. : my_p / total) : my_p;
      const int64_t at = ((int64_t)s * a.T + t) * a.k + lane;
      a.weights[at] = nan ? NAN : (float)(w * (double)a.scale);
      a.experts[at] = my_e;
      atomicAdd(&hist[my_e], 1);                             // (a count: its value does not depend on the order)
    }
  }
  __syncthreads();
  int32_t* out = a.counts + ((int64_t)s * a.blocks + blockIdx.x) * a.E;
  for (int i = threadIdx.x; i < a.E; i += 256) out[i] = hist[i];
}

// counts -> exclusive prefix over a sample's workgroups, per expert; offsets -> exclusive prefix over its experts
__global__ __launch_bounds__(256) void route_scan_kernel(const RouteArgs a) {
  __shared__ int total[1024];
  const int s = blockIdx.x;
  for (int e = threadIdx.x; e < a.E; e += 256) {
    int run = 0;
    for (int b = 0; b < a.blocks; ++b) {
      int32_t* c = a.counts + ((int64_t)s * a.blocks + b) * a.E + e;
      const int n = *c;
      *c = run;
      run += n;
    }
    total[e] = run;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    int run = s * a.T * a.k;
    for (int e = 0; e < a.E; ++e) { a.offsets[s * a.E + e] = run; run += total[e]; }
    if (s == a.S - 1) a.offsets[a.S * a.E] = run;
  }
}

__global__ __launch_bounds__(256) void route_scatter_kernel(const RouteArgs a) {
  extern __shared__ int32_t mine[];
  const int s = blockIdx.y, t0 = blockIdx.x * ROUTE_ROWS, n = (min(a.T, t0 + ROUTE_ROWS) - t0) * a.k;
  const int64_t first = ((int64_t)s * a.T + t0) * a.k;
  for (int i = threadIdx.x; i < n; i += 256) mine[i] = a.experts[first + i];
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += 256) {
    const int e = mine[i];
    int rank = 0;
    for (int j = 0; j < i; ++j) rank += mine[j] == e ? 1 : 0;
    a.rows[a.offsets[s * a.E + e] + a.counts[((int64_t)s * a.blocks + blockIdx.x) * a.E + e] + rank] = (int32_t)(first + i);
  }
}

template <int T> int launch_route(const RouteArgs& a, hipStream_t st) {
  const dim3 grid((unsigned)a.blocks, (unsigned)a.S);
  if (a.E <= 64) hipLaunchKernelGGL((route_kernel<T, 1>), grid, dim3(256), 0, st, a);
  else if (a.E <= 128) hipLaunchKernelGGL((route_kernel<T, 2>), grid, dim3(256), 0, st, a);
  else if (a.E <= 256) hipLaunchKernelGGL((route_kernel<T, 4>), grid, dim3(256), 0, st, a);
  else if (a.E <= 512) hipLaunchKernelGGL((route_kernel<T, 8>), grid, dim3(256), 0, st, a);
  else hipLaunchKernelGGL((route_kernel<T, 16>), grid, dim3(256), 0, st, a);
  if (int rc = qbnn_check_launch_msg("qbnn_route_experts")) return rc;
  hipLaunchKernelGGL(route_scan_kernel, dim3((unsigned)a.S), dim3(256), 0, st, a);
  if (int rc = qbnn_check_launch_msg("qbnn_route_experts (scan)")) return rc;
  hipLaunchKernelGGL(route_scatter_kernel, grid, dim3(256), ROUTE_ROWS * a.k * sizeof(int32_t), st, a);
  return qbnn_check_launch_msg("qbnn_route_experts (order)");
}

// ---- y[t] = sum over the row's top_k results, in the order of choice --------------------------------------------------------------
// The results come in fp32: rounded to 16 bits first, each would cost as much as the one rounding of the sum does.
template <int T> __global__ __launch_bounds__(256) void combine_kernel(const float* __restrict__ o, f8_type<T>* __restrict__ y, int rows, int k, int N) {
  const int n0 = (blockIdx.x * 256 + threadIdx.x) * 4;
  const int64_t t = blockIdx.y + (int64_t)blockIdx.z * 32768;
  if (n0 >= N || t >= rows) return;
  float sum[4] = {0.f, 0.f, 0.f, 0.f};
  const bool whole = n0 + 4 <= N;
  for (int j = 0; j < k; ++j) {
    const float* r = o + (t * k + j) * N + n0;
    float v[4];
    if (whole) __builtin_memcpy(v, r, sizeof(v));
    else
      for (int i = 0; i < 4; ++i) v[i] = n0 + i < N ? r[i] : 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) sum[i] += v[i];
  }
  f8_type<T> v[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = f8_store<T>(sum[i]);
  f8_type<T>* out = y + t * N + n0;
  if (whole) __builtin_memcpy(out, v, sizeof(v));
  else
    for (int i = 0; i < 4; ++i) if (n0 + i < N) out[i] = v[i];
}

}  // namespace

QBNN_EXPORT int64_t qbnn_route_workspace_ints(int32_t S, int32_t T, int32_t E) {
  return S <= 0 || T <= 0 || E <= 0 ? 0 : (int64_t)S * ((T + ROUTE_ROWS - 1) / ROUTE_ROWS) * E;
}

QBNN_EXPORT int qbnn_route_experts(const qbnn_route* r, void* stream) {
  if (!r || r->S < 0 || r->T < 0 || r->E <= 0 || r->E > QBNN_ROUTE_MAX_EXPERTS || r->top_k <= 0 || r->top_k > QBNN_ROUTE_MAX_CHOICES || r->groups <= 0 || r->groups > 64 ||
      r->E % r->groups || r->top_groups <= 0 || r->top_groups > r->groups || r->top_k > r->E / r->groups * r->top_groups || r->type < QBNN_F32 || r->type > QBNN_F16 ||
      !r->offsets)
    return route_fail("qbnn_route_experts: bad argument (E %ld, top_k %ld)", r ? r->E : 0, r ? r->top_k : 0);
  const int64_t rows = (int64_t)r->S * r->T * r->top_k;
  if (rows > 0x7fffffff || (int64_t)r->S * r->E >= 0x7fffffff) return route_fail("qbnn_route_experts: %ld routed rows do not fit 31 bits", (long)rows);
  if (rows == 0) return route_fail("qbnn_route_experts: no rows");
  if (!r->logits || !r->weights || !r->experts || !r->rows || !r->workspace || r->S > 65535) return route_fail("qbnn_route_experts: bad argument");
  RouteArgs a;
  a.logits = r->logits; a.l_ss = r->logits_ss; a.l_rs = r->logits_rs; a.bias = r->bias;
  a.weights = r->weights; a.experts = r->experts; a.offsets = r->offsets; a.rows = r->rows; a.counts = r->workspace;
  a.S = r->S; a.T = r->T; a.E = r->E; a.k = r->top_k; a.groups = r->groups; a.kept = r->top_groups; a.sigmoid = r->sigmoid; a.renorm = r->renormalize; a.scale = r->scale;
  a.blocks = (r->T + ROUTE_ROWS - 1) / ROUTE_ROWS;
  switch (r->type) {
    case QBNN_F32: return launch_route<QBNN_F32>(a, (hipStream_t)stream);
    case QBNN_BF16: return launch_route<QBNN_BF16>(a, (hipStream_t)stream);
    default: return launch_route<QBNN_F16>(a, (hipStream_t)stream);
  }
}

QBNN_EXPORT int qbnn_combine_routed(const float* o, int32_t rows, int32_t top_k, int32_t N, void* y, int32_t y_type, void* stream) {
  if (rows < 0 || top_k <= 0 || N <= 0 || y_type < QBNN_F32 || y_type > QBNN_F16) return route_fail("qbnn_combine_routed: bad argument");
  if (rows == 0) return QBNN_OK;
  if (!o || !y) return route_fail("qbnn_combine_routed: bad argument");
  const dim3 grid((unsigned)((N + 1023) / 1024), (unsigned)(rows < 32768 ? rows : 32768), (unsigned)((rows + 32767) / 32768));
  switch (y_type) {
    case QBNN_F32: hipLaunchKernelGGL((combine_kernel<QBNN_F32>), grid, dim3(256), 0, (hipStream_t)stream, o, (float*)y, rows, top_k, N); break;
    case QBNN_BF16: hipLaunchKernelGGL((combine_kernel<QBNN_BF16>), grid, dim3(256), 0, (hipStream_t)stream, o, (uint16_t*)y, rows, top_k, N); break;
    default: hipLaunchKernelGGL((combine_kernel<QBNN_F16>), grid, dim3(256), 0, (hipStream_t)stream, o, (_Float16*)y, rows, top_k, N); break;
  }
  return qbnn_check_launch_msg("qbnn_combine_routed");
}
