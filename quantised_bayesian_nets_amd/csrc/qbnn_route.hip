// libqbnn_hip.so: the router of a layer of experts.
//   scores    s = softmax(l) or sigmoid(l) over a row's E logits;  key = s + bias (what is compared), weight = s (what is multiplied)
//   groups    E / groups neighbouring experts each; a group counts its two largest keys, the best `top_groups` groups stay
//   choice    the top_k largest keys; of equal ones with one group the larger logit first, then the lowest index; weights optionally divided by their sum, times `scale`
//   order     the (row, choice) pairs of a sample sorted by expert, stable: what the experts' products walk
// The choice is that of 64-bit keys: two experts whose scores differ only behind fp32's last place are still told apart, so it does not depend on
// the order in which a row's sum was taken.  Both scores increase with the logit, so without a bias and groups the logits are compared themselves; the rule for equal
// keys makes that the same choice as under a bias of zeros, also where scores are equal to the last bit of 64 (sigmoid above 37, softmax 746 below the largest).
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <stdio.h>
#include <float.h>
#include <math.h>
#include <atomic>

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
constexpr int ROUTE_BLOCKS = 128;      // up to so many workgroups per sample, each sums the others' counts itself; beyond, a kernel between does

struct RouteArgs {
  const void* logits; int64_t l_ss, l_rs;
  const float* bias;
  float* weights; int32_t* experts; int32_t* offsets; int32_t* rows; int32_t* counts;      // counts [S][blocks][E]
  int S, T, E, k, groups, kept, sigmoid, renorm, blocks, bits;                             // bits: of an expert's index
  float scale;
};

template <int T> __device__ __forceinline__ float route_lowest() {
  if constexpr (T == QBNN_BF16) return -3.3895313892515355e38f;
  else if constexpr (T == QBNN_F16) return -65504.f;
  else return -FLT_MAX;
}
__device__ __forceinline__ float route_exp(float v) { return __builtin_amdgcn_exp2f(v * 1.44269504088896340736f); }      // off by at most (|v| + 2) 2^-23 of it

// e^(l - top) to a unit or two in the last place wherever it lies: the difference's rounding, |l - top| 2^-24 of the result, is put back
__device__ __forceinline__ float route_softmax_term(float l, float top) {
  const float d = l - top, b = d - l, lost = (l - (d - b)) - (top + b), z = expf(d);
  return z > 0.f && z < 1.f ? z + z * lost : z;                 // (0: past the range, and lost may be NaN)
}

// ---- reductions over the L lanes (a power of two) of a row: each step's partner holds what the step before left in all lanes of its half ------------
template <int CTRL> __device__ __forceinline__ uint32_t route_dpp(uint32_t v) { return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, true); }
template <int STEP> __device__ __forceinline__ uint32_t route_partner(uint32_t v) {
  if constexpr (STEP == 1) return route_dpp<0xB1>(v);              // quad_perm 1 0 3 2
  else if constexpr (STEP == 2) return route_dpp<0x4E>(v);         // quad_perm 2 3 0 1
  else if constexpr (STEP == 4) return route_dpp<0x141>(v);        // row_half_mirror
  else if constexpr (STEP == 8) return route_dpp<0x140>(v);        // row_mirror
  else return (uint32_t)__shfl_xor((int)v, STEP);
}
template <int L, class F> __device__ __forceinline__ uint32_t route_reduce(uint32_t v, F f) {
  if constexpr (L > 1) v = f(v, route_partner<1>(v));
  if constexpr (L > 2) v = f(v, route_partner<2>(v));
  if constexpr (L > 4) v = f(v, route_partner<4>(v));
  if constexpr (L > 8) v = f(v, route_partner<8>(v));
  if constexpr (L > 16) v = f(v, route_partner<16>(v));
  if constexpr (L > 32) v = f(v, route_partner<32>(v));
  return v;
}
template <int L> __device__ __forceinline__ uint32_t route_max(uint32_t v) { return route_reduce<L>(v, [](uint32_t a, uint32_t b) { return max(a, b); }); }
template <int L> __device__ __forceinline__ float route_maxf(float v) {
  return __uint_as_float(route_reduce<L>(__float_as_uint(v), [](uint32_t a, uint32_t b) { return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b))); }));
}
template <int L> __device__ __forceinline__ float route_sumf(float v) {
  return __uint_as_float(route_reduce<L>(__float_as_uint(v), [](uint32_t a, uint32_t b) { return __float_as_uint(__uint_as_float(a) + __uint_as_float(b)); }));
}
// order-preserving bits of a float and back
__device__ __forceinline__ uint32_t route_order(float v) { const uint32_t b = __float_as_uint(v); return b ^ ((uint32_t)((int)b >> 31) | 0x80000000u); }
__device__ __forceinline__ float route_value(uint32_t o) { return __uint_as_float(o ^ ((uint32_t)((int)~o >> 31) | 0x80000000u)); }

// What a group of keys counts: its two largest summed, masked ones left out; a group of masked keys ranks last.
template <class FLT> __device__ __forceinline__ FLT route_score(FLT a1, FLT a2) { return a1 == -INFINITY ? a1 : a2 == -INFINITY ? a1 : a1 + a2; }

// score[row][group] of the wave's rows from their keys in LDS, 2^parts lanes per (row, group)
template <class FLT> __device__ __forceinline__ void route_group_scores(const RouteArgs& a, const FLT* keys, int rows, int pitch, FLT* score) {
  const int per = a.E / a.groups, lane = threadIdx.x & 63;
  int parts = 0;
  while ((rows * a.groups << (parts + 1)) <= 64) ++parts;
  for (int q = lane >> parts; q < rows * a.groups; q += 64 >> parts) {
    const int r = q / a.groups, g = q - r * a.groups;
    const FLT* k = keys + r * pitch + g * per;
    FLT a1 = -INFINITY, a2 = -INFINITY;
#pragma unroll 4
    for (int i = lane & ((1 << parts) - 1); i < per; i += 1 << parts) {
      const FLT v = k[i];
      a2 = fmax(a2, fmin(a1, v));
      a1 = fmax(a1, v);
    }
    for (int d = 0; d < parts; ++d) {
      const FLT b1 = __shfl_xor(a1, 1 << d), b2 = __shfl_xor(a2, 1 << d);
      a2 = fmax(fmin(a1, b1), fmax(a2, b2));
      a1 = fmax(a1, b1);
    }
    if ((lane & ((1 << parts) - 1)) == 0) score[q] = route_score(a1, a2);
  }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
}
// Which groups stay, by comparing each with its row's others; slack[row]: the score of the last group kept minus the best one left out.
template <class FLT> __device__ __forceinline__ void route_keep_groups(const RouteArgs& a, int rows, const FLT* score, uint32_t* stay, FLT* slack) {
  for (int q = threadIdx.x & 63; q < rows * a.groups; q += 64) {
    const int r = q / a.groups, g = q - r * a.groups;
    const FLT mine = score[q];
    int rank = 0;
    FLT next = -INFINITY;                                       // the best score behind mine
#pragma unroll 4
    for (int i = 0; i < a.groups; ++i) {
      const FLT o = score[r * a.groups + i];
      const bool ahead = o > mine || (o == mine && i < g);
      rank += ahead ? 1 : 0;
      if (!ahead && i != g && o > next) next = o;
    }
    stay[q] = rank < a.kept ? 1u : 0u;
    if (rank == a.kept - 1) slack[r] = a.kept == a.groups ? (FLT)INFINITY : mine == next ? (FLT)0 : mine - next;
  }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
}

// ---- the order of the rows -----------------------------------------------------------------------------------------------------
// A counting sort, stable: a workgroup's n choices in four quarters, one per wave; count[wave][E] holds each quarter's number of every expert and then the
// position of its next one.  Within 64 choices a lane's rank is the number of lanes below it with the same expert, from one ballot per index bit.
__device__ __forceinline__ int route_quarter(int n) { return ((n + 255) >> 8) << 6; }
__device__ __forceinline__ void route_count(const uint32_t* choice, int* count, int n, int E) {      // count is 0
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, q = route_quarter(n);
  for (int i = wave * q + lane; i < min(n, (wave + 1) * q); i += 64) atomicAdd(&count[wave * E + choice[i]], 1);      // (a number: no order)
  __syncthreads();
}
// exclusive prefix over E values, four per thread and pass; at(e) reads, put(e, prefix) takes
template <class At, class Put> __device__ __forceinline__ void route_prefix(int E, At at, Put put) {
  __shared__ int sums[8];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, e0 = threadIdx.x * 4;
  int v[4], mine = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) { v[i] = e0 + i < E ? at(e0 + i) : 0; mine += v[i]; }
  int incl = mine;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) { const int u = __shfl_up(incl, d); if (lane >= d) incl += u; }
  if (lane == 63) sums[wave] = incl;
  __syncthreads();
  int run = incl - mine;
  for (int w = 0; w < wave; ++w) run += sums[w];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (e0 + i < E) { put(e0 + i, run); run += v[i]; }
}
// count: each quarter's position of its next choice of e
__device__ __forceinline__ void route_place(const RouteArgs& a, const uint32_t* choice, int* count, int n, int first) {
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, q = route_quarter(n);
  int* mine = count + wave * a.E;
  for (int i0 = wave * q; i0 < min(n, (wave + 1) * q); i0 += 64) {
    const int i = i0 + lane;
    const bool in = i < n;
    const uint32_t e = in ? choice[i] : 0u;
    unsigned long long same = __ballot(in);
    for (int b = 0; b < a.bits; ++b) {
      const unsigned long long ones = __ballot((e >> b) & 1);
      same &= (e >> b) & 1 ? ones : ~ones;
    }
    const int rank = __popcll(same & ((1ull << lane) - 1));
    const int at = in ? mine[e] : 0;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    if (in) {
      a.rows[at + rank] = first + i;
      if (rank == 0) mine[e] = at + __popcll(same);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  }
}
// start(e): position of the workgroup's first choice of e -> the quarters' own positions
template <class F> __device__ __forceinline__ void route_starts(int* count, int E, F start) {
  for (int e = threadIdx.x; e < E; e += blockDim.x) {
    int run = start(e);
#pragma unroll
    for (int w = 0; w < 4; ++w) { const int c = count[w * E + e]; count[w * E + e] = run; run += c; }
  }
  __syncthreads();
}

__host__ __device__ __forceinline__ bool route_whole(const RouteArgs& a) { const int per = a.E / a.groups; return per >= 16 && (per & (per - 1)) == 0; }
// LDS of a wave: for its rows' groups fp32 keys [64 / L][L 16 + 2] where a group is not whole lanes, scores, masks and slack of 64 / L rows; or 64-bit ones of one row
template <int L> __host__ __device__ constexpr int route_wave_bytes(int groups, bool whole) {
  const int fast = groups > 1 ? (64 / L) * (((whole ? 0 : L * 16 + 2) + 2 * groups) * 4 + 4) : 0, exact = (L * 16 + 1) * 8 + groups * 12;
  return ((fast > exact ? fast : exact) + 15) & ~15;
}

// One step of a choice over a wave: the larger key, and of equal ones the lower index
template <int STEP> __device__ __forceinline__ void route_join(double& b, int& bi) {
  const double ob = __hiloint2double((int)route_partner<STEP>((uint32_t)__double2hiint(b)), (int)route_partner<STEP>((uint32_t)__double2loint(b)));
  const int oi = (int)route_partner<STEP>((uint32_t)bi);
  if (ob > b || (ob == b && oi < bi)) { b = ob; bi = oi; }
}

// One row by a whole wave with 64-bit keys, NP experts per lane.  They are made one by one, through LDS: NP exponentials at once would halve the waves of the fast pass.
template <int T, int NP> __device__ __forceinline__ void route_exact_row(const RouteArgs& a, const f8_type<T>* l, bool by_logit, double* keys, double* score, uint32_t* choice) {
  const int lane = threadIdx.x & 63, per = a.E / a.groups;
  double* slack = score + a.groups;
  uint32_t* stay = (uint32_t*)(slack + 1);
  double top = -INFINITY, total = 0.;
#pragma unroll 1
  for (int e = lane; e < a.E; e += 64) {
    const float v = f8_load<T>(l[e]);
    keys[e] = v > route_lowest<T>() ? (double)v : -INFINITY;    // (false for NaN)
    top = fmax(top, keys[e]);
  }
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) top = fmax(top, __shfl_xor(top, d));
  if (!by_logit) {
#pragma unroll 1
    for (int e = lane; e < a.E; e += 64) {
      const double x = keys[e], z = exp(a.sigmoid ? -x : x == top ? 0. : x - top), p = a.sigmoid ? 1. / (1. + z) : z;      // (infinite logits share the row)
      keys[e] = x > -INFINITY ? p : -1.;
      total += x > -INFINITY ? p : 0.;
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) total += __shfl_xor(total, d);
    total = a.sigmoid ? 1. : 1. / total;
#pragma unroll 1
    for (int e = lane; e < a.E; e += 64) {
      const double p = keys[e], q = p * total + (a.bias ? (double)a.bias[e] : 0.);
      keys[e] = p >= 0. && q == q ? q : -INFINITY;
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    if (a.groups > 1) {
      route_group_scores<double>(a, keys, 1, 0, score);
      route_keep_groups<double>(a, 1, score, stay, slack);
    }
  }
  double key[NP];
  int idx[NP];
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    const int e = i * 64 + lane;
    const bool in = e < a.E && (a.groups == 1 || stay[e / per]);
    key[i] = in ? keys[e] : -INFINITY;
    idx[i] = in ? e : 0x7fffffff;
  }
  const bool by_score = !by_logit && a.groups == 1;
  for (int j = 0; j < a.k; ++j) {
    double b = key[0];
    int bi = idx[0];
#pragma unroll
    for (int i = 1; i < NP; ++i)
      if (key[i] > b || (key[i] == b && idx[i] < bi)) { b = key[i]; bi = idx[i]; }
    route_join<1>(b, bi);
    route_join<2>(b, bi);
    route_join<4>(b, bi);
    route_join<8>(b, bi);
    route_join<16>(b, bi);
    route_join<32>(b, bi);
    if (by_score && b > -INFINITY) {                            // of equal keys the one with the larger logit, as without a bias
      bool tied = false;
#pragma unroll
      for (int i = 0; i < NP; ++i) tied |= key[i] == b && idx[i] != bi && idx[i] != 0x7fffffff;
      if (__any(tied)) {
        double most = -INFINITY;
        bi = 0x7fffffff;
#pragma unroll
        for (int i = 0; i < NP; ++i) {
          const bool in = key[i] == b && idx[i] != 0x7fffffff;
          const double v = in ? (double)f8_load<T>(l[idx[i]]) : -INFINITY;
          if (in && (v > most || (v == most && idx[i] < bi))) { most = v; bi = idx[i]; }
        }
        route_join<1>(most, bi);
        route_join<2>(most, bi);
        route_join<4>(most, bi);
        route_join<8>(most, bi);
        route_join<16>(most, bi);
        route_join<32>(most, bi);
      }
    }
#pragma unroll
    for (int i = 0; i < NP; ++i) if (idx[i] == bi) { key[i] = -INFINITY; idx[i] = 0x7fffffff; }
    if (lane == 0) choice[j] = (uint32_t)bi;
  }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
}

// L lanes per row, 16 neighbouring experts per lane.
//
// Fast pass: keys in fp32 as ordered integers whose low bits say which expert they are (its complement: ties go to the lowest index), so that a round of the
// choice is one integer maximum.  Logits of 16 bits compare exactly as they are and carry the whole index; other keys give up only 4 bits, for the place
// in their lane, and the choice must be proved: each chosen key has to lie above the next one by more than the keys' error and the bits given up (and
// likewise the last group kept above the next), and one lane alone may hold it.  Rows without that proof (1 in 1000 of 256 continuous fp32 logits; without a bias each
// row with equal ones among its first, 37 in 100 where the logits were rounded to bf16 before, 42 -> 67 us) are listed and done again, a whole wave each, with 64-bit keys.  Masked experts are the integers below all keys, lowest index first.
// A key that was chosen is not taken out: the next round looks for the largest below it, as the smallest unsigned m - 1 - w (what lies above wraps).
// Bound: vector issue.  A round is 50 instructions for 64 / L rows, all of a row of 256 with groups and 8 choices 1,000 for 4 rows: 32768 x 256 take 38 us at 2 GHz, where
// reading them takes 7; 22 - 28 of it are these rounds, the rest waits for the waves that do a row again (10 us each).  Registers held to 128, for 4 waves per SIMD.
constexpr uint32_t ROUTE_MASKED = 0x00800000u;                  // the order of the lowest finite float: masked experts lie below

// Waves of a workgroup: 64 rows are 64 L / 64 of them, done in turn by 4 where that is all and by 8 where there are more
constexpr int route_waves(int L) { return L < 8 ? 4 : 8; }

// KEY: what is compared
enum { KEY_LOGIT, KEY_SIGMOID, KEY_SOFTMAX };

template <int T, int L, int KEY> __global__ __launch_bounds__(route_waves(L) * 64, L >= 8 ? 4 : 2) void route_kernel(const RouteArgs a) {
  constexpr int RPW = 64 / L, NW = route_waves(L);              // rows per wave, waves
  constexpr int NP = L < 4 ? 1 : L / 4;                         // experts per lane where a wave does one row
  constexpr int PITCH = L * 16 + 2;
  extern __shared__ __attribute__((aligned(16))) uint8_t dyn[];
  __shared__ float row_top[ROUTE_ROWS], row_sum[ROUTE_ROWS];
  __shared__ int again[ROUTE_ROWS], n_again;
  __shared__ __attribute__((aligned(16))) float bias[KEY == KEY_LOGIT ? 1 : L * 16];
  // dynamic: choices and their scores [64][k], the quarters' counts [4][E], starts [E], and with groups each wave's keys, scores, masks
  uint32_t* choice = (uint32_t*)dyn;
  float* part = (float*)(choice + ROUTE_ROWS * a.k);
  int* count = (int*)(part + ROUTE_ROWS * a.k);
  int* start = count + 4 * a.E;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, sub = lane / L, li = lane % L;
  uint8_t* more = (uint8_t*)(start + a.E);
  more += (-(uintptr_t)more) & 15;

  const int s = blockIdx.y, t0 = blockIdx.x * ROUTE_ROWS, rows = min(a.T - t0, ROUTE_ROWS);
  constexpr bool exact = KEY == KEY_LOGIT && T != QBNN_F32;
  const uint32_t low = exact ? (1u << a.bits) - 1 : 15u;
  const f8_type<T>* base = (const f8_type<T>*)a.logits + s * a.l_ss + t0 * a.l_rs;
  for (int i = threadIdx.x; i < 4 * a.E; i += NW * 64) count[i] = 0;
  if constexpr (KEY != KEY_LOGIT)                               // (each lane's 16 straight from memory: 16 loads of 16 lines each, by every wave)
    for (int i = threadIdx.x; i < L * 16; i += NW * 64) {
      const float b = a.bias && i < a.E ? a.bias[i] : 0.f;
      bias[i] = b == b ? b : -INFINITY;
    }
  if (threadIdx.x == 0) n_again = 0;
  __syncthreads();

  int e0 = li * 16;
  const int per = KEY == KEY_LOGIT ? a.E : a.E / a.groups, g0 = e0 / per, p0 = e0 - g0 * per;      // the lane's first group, and the place in it
  const bool whole = route_whole(a);                            // a group is whole lanes (and a power of two of them): its two largest without LDS
  more += (size_t)wave * route_wave_bytes<L>(a.groups, whole);
  for (int r0 = wave * RPW; r0 < rows; r0 += NW * RPW) {
    asm volatile("" : "+v"(e0));                                // (or 16 of everything that depends on it alone are kept over the loop: 50 registers)
    const int r = r0 + sub;
    const bool valid = r < rows;
    const f8_type<T>* l = base + (int64_t)min(r, rows - 1) * a.l_rs;
    f8_type<T> raw[16];
    if (e0 + 16 <= a.E) __builtin_memcpy(raw, l + e0, sizeof(raw));
    else {
#pragma unroll
      for (int i = 0; i < 16; ++i) raw[i] = l[min(e0 + i, a.E - 1)];
    }
    float v[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = e0 + i < a.E ? f8_load<T>(raw[i]) : -INFINITY;
    bool nan = false;
    float top = -INFINITY, sum = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) nan |= v[i] != v[i];
    if (!a.sigmoid) {
#pragma unroll
      for (int i = 0; i < 16; ++i) top = fmaxf(top, v[i] > route_lowest<T>() ? v[i] : -INFINITY);
      top = route_maxf<L>(top);
    }
    uint32_t w[16];
    bool unsure = false;
    float worst = 0.f;                                          // two scores' errors
    if constexpr (KEY == KEY_LOGIT) {
      if (!a.sigmoid) {
#pragma unroll
        for (int i = 0; i < 16; ++i) sum += v[i] > route_lowest<T>() ? route_exp(v[i] - top) : 0.f;
        sum = route_sumf<L>(sum);
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) {                            // (-0 ties with 0)
        const uint32_t order = (route_order(v[i] + 0.f) & ~low) | (exact ? low - (uint32_t)(e0 + i) : 15u - i);
        w[i] = v[i] > route_lowest<T>() ? order : (uint32_t)max(a.E - e0 - i, 0);
      }
    } else {
      // exp is off by (|x| + 2) 2^-23 of it.  Sigmoid: p (1 - p) |x| < 0.23, p (1 - p) <= 1/4, 1 + z half a step, its reciprocal one: 2.3 2^-23, 3 taken.
      // Softmax, x = v - top <= 0 off by half a step, p <= 1 / sum: a term by (1.5 |x| + 2), e^x |x| < 0.37; the sum by 15 + 6 additions (10.5) and its terms'
      // own (sum p |x| <= ln E < 7: 12.5); the reciprocal and the product 1.5: 27.1 2^-23 / sum, 32 taken.
      constexpr bool SIG = KEY == KEY_SIGMOID;
      float key[16];
      if constexpr (SIG) {
        worst = 2 * 3 * 1.1920929e-7f;
#pragma unroll
        for (int i = 0; i < 16; ++i) key[i] = v[i] > route_lowest<T>() ? __builtin_amdgcn_rcpf(1.f + route_exp(-v[i])) + bias[e0 + i] : -INFINITY;
      } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          key[i] = v[i] > route_lowest<T>() ? route_exp(v[i] - top) : 0.f;
          sum += key[i];
        }
        sum = route_sumf<L>(sum);
        unsure = !(top < INFINITY);                             // infinite logits share the row: not a sum of these terms
        const float over = __builtin_amdgcn_rcpf(sum);
        worst = 2 * 32 * 1.1920929e-7f * over;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const float q = key[i] * over + bias[e0 + i];
          key[i] = v[i] > route_lowest<T>() && q == q ? q : -INFINITY;
        }
      }
      uint32_t in = 0xffffu;
      if (a.groups > 1) {
        float* score = (float*)more;                            // [RPW][groups]
        uint32_t* stay = (uint32_t*)(score + RPW * a.groups);
        float* slack = (float*)(stay + RPW * a.groups);
        float large = 0.f;                                      // the largest key that counts
        if (whole) {
          float a1 = -INFINITY, a2 = -INFINITY;
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            a2 = __builtin_amdgcn_fmed3f(a1, a2, key[i]);
            a1 = fmaxf(a1, key[i]);
          }
          auto join = [&](uint32_t p1, uint32_t p2) {
            const float b1 = __uint_as_float(p1), b2 = __uint_as_float(p2);
            a2 = fmaxf(fminf(a1, b1), fmaxf(a2, b2));
            a1 = fmaxf(a1, b1);
          };
          if (L > 1 && per > 16) join(route_partner<1>(__float_as_uint(a1)), route_partner<1>(__float_as_uint(a2)));
          if (L > 2 && per > 32) join(route_partner<2>(__float_as_uint(a1)), route_partner<2>(__float_as_uint(a2)));
          if (L > 4 && per > 64) join(route_partner<4>(__float_as_uint(a1)), route_partner<4>(__float_as_uint(a2)));
          if (L > 8 && per > 128) join(route_partner<8>(__float_as_uint(a1)), route_partner<8>(__float_as_uint(a2)));
          if (L > 16 && per > 256) join(route_partner<16>(__float_as_uint(a1)), route_partner<16>(__float_as_uint(a2)));
          large = fmaxf(a1 > -INFINITY ? fabsf(a1) : 0.f, a2 > -INFINITY ? fabsf(a2) : 0.f);
          if (p0 == 0 && e0 < a.E) score[sub * a.groups + g0] = route_score(a1, a2);
          __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        } else {
          float* keys = slack + RPW;
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            keys[sub * PITCH + e0 + i] = e0 + i < a.E ? key[i] : -INFINITY;
            large = e0 + i < a.E && key[i] > -INFINITY ? fmaxf(large, fabsf(key[i])) : large;
          }
          __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
          route_group_scores<float>(a, keys, RPW, PITCH, score);
        }
        route_keep_groups<float>(a, RPW, score, stay, slack);
        // sums of two keys each (score and bias), and the sums' rounding
        unsure |= !(slack[sub] > 2.f * worst + route_maxf<L>(large) * 9.6e-7f);
        if (whole) in = e0 < a.E && stay[sub * a.groups + g0] ? 0xffffu : 0u;
        else {
#pragma unroll
          for (int i = 0, g = g0, p = p0; i < 16; ++i) {
            in ^= (stay[sub * a.groups + min(g, a.groups - 1)] ^ 1u) << i;
            g += p + 1 == per ? 1 : 0;
            p = p + 1 == per ? 0 : p + 1;
          }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const uint32_t order = (route_order(key[i]) & ~15u) | (15u - i);
        w[i] = (key[i] > -INFINITY ? order : (uint32_t)max(a.E - e0 - i, 0)) & (uint32_t)((int)(in << (31 - i)) >> 31);
      }
    }
    if (li == 0 && valid) {
      row_top[r] = top;
      row_sum[r] = sum;
    }
    if (route_max<L>(nan ? 1u : 0u) && li == 0 && valid) row_top[r] = NAN;

    // k rounds, and one more to see that the last choice was none too close
    uint32_t before = 0;
    float above = 0.f;
    for (int j = 0; j < a.k + (exact ? 0 : 1); ++j) {
      const uint32_t c = before - 1;
      uint32_t near = 0xffffffffu;
#pragma unroll
      for (int i = 0; i < 16; ++i) near = min(near, c - w[i]);
      const uint32_t mine = near <= c ? c - near : 0u;          // the lane's largest below `before`; 0: none
      const uint32_t m = route_max<L>(mine);
      if (j < a.k) {
        const bool own = mine == m;
        if (own && valid) choice[r * a.k + j] = m < ROUTE_MASKED ? a.E - m : exact ? low - (m & low) : e0 + 15u - (m & 15u);
        if (!exact && L > 1) {
          const unsigned long long owners = __ballot(own);
          if (__popcll(owners) != RPW) unsure |= __popcll((owners >> (sub * L % 64)) & (L < 64 ? (1ull << (L % 64)) - 1 : ~0ull)) > 1;
        }
      }
      if constexpr (KEY == KEY_LOGIT) {
        if (!exact && j > 0 && m >= ROUTE_MASKED) unsure |= ((before ^ m) & ~15u) == 0;
      } else {                                                  // each key gave up 15 last places at most and its bias half of one: 16 2^-23 of it
        const float at = route_value(m);
        if (j > 0 && m >= ROUTE_MASKED) unsure |= !(above - at > __builtin_fmaf(fmaxf(fabsf(above), fabsf(at)), 32 * 1.1920929e-7f, worst));
        above = at;
      }
      before = m;
    }
    if (unsure && li == 0 && valid) again[atomicAdd(&n_again, 1)] = r;      // (their order does not matter)
  }
  __syncthreads();
  if constexpr (!exact) {
    for (int i = wave; i < n_again; i += NW)
      route_exact_row<T, NP>(a, base + (int64_t)again[i] * a.l_rs, KEY == KEY_LOGIT, (double*)more, (double*)more + L * 16, choice + again[i] * a.k);
    __syncthreads();
  }

  // weights: a thread per choice, scores taken again from the logits
  const int n = rows * a.k;
  const int64_t first = ((int64_t)s * a.T + t0) * a.k;
  for (int i = threadIdx.x; i < n; i += NW * 64) {
    const int r = i / a.k, e = (int)choice[i];
    const float l = f8_load<T>(base[(int64_t)r * a.l_rs + e]), top = row_top[r];
    float p = a.sigmoid ? 1.f / (1.f + expf(-l)) : route_softmax_term(l, top) / row_sum[r];
    if (!(l > route_lowest<T>())) p = 0.f;
    if (top != top) p = NAN;
    part[i] = p;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += NW * 64) {
    float p = part[i];
    if (a.renorm) {
      const int r = i / a.k;
      float total = 0.f;
      for (int j = 0; j < a.k; ++j) total += part[r * a.k + j];
      p = total == 0.f ? 0.f : p / total;
    }
    a.weights[first + i] = p * a.scale;
    a.experts[first + i] = (int32_t)choice[i];
  }
  route_count(choice, count, n, a.E);
  auto total = [&](int e) { return count[e] + count[a.E + e] + count[2 * a.E + e] + count[3 * a.E + e]; };
  if (a.blocks > 1) {
    int32_t* out = a.counts + ((int64_t)s * (a.blocks + 1) + blockIdx.x) * a.E;
    for (int e = threadIdx.x; e < a.E; e += NW * 64) out[e] = total(e);
    return;
  }
  const int all = s * a.T * a.k;
  route_prefix(a.E, total, [&](int e, int before) { a.offsets[s * a.E + e] = start[e] = all + before; });
  if (s == a.S - 1 && threadIdx.x == 0) a.offsets[a.S * a.E] = all + n;
  __syncthreads();
  route_starts(count, a.E, [&](int e) { return start[e]; });
  route_place(a, choice, count, n, (int)first);
}

// counts [blocks + 1][E] of a sample: each workgroup's -> the workgroups' before it, and the sum in the last row.  4 experts per workgroup, 64 runs of rows (16 and 16
// took 13 us for 512 x 256: their loads waited for one another).
__global__ __launch_bounds__(256) void route_scan_kernel(const RouteArgs a) {
  __shared__ int sums[4][4];
  const int col = threadIdx.x & 3, r = threadIdx.x >> 2, wave = threadIdx.x >> 6, lane = threadIdx.x & 63, e = blockIdx.x * 4 + col, per = (a.blocks + 63) / 64;
  int32_t* c = a.counts + (int64_t)blockIdx.y * (a.blocks + 1) * a.E + e;
  const int b0 = r * per, b1 = e < a.E ? min(a.blocks, b0 + per) : 0;
  int sum = 0;
#pragma unroll 8
  for (int b = b0; b < b1; ++b) sum += c[(int64_t)b * a.E];
  int incl = sum;
#pragma unroll
  for (int d = 4; d < 64; d <<= 1) { const int u = __shfl_up(incl, d); if (lane >= d) incl += u; }
  if (lane >= 60) sums[wave][col] = incl;
  __syncthreads();
  int at = incl - sum;
  for (int i = 0; i < wave; ++i) at += sums[i][col];
  if (r == 63 && e < a.E) c[(int64_t)a.blocks * a.E] = at + sum;
#pragma unroll 8
  for (int b = b0; b < b1; ++b) { const int v = c[(int64_t)b * a.E]; c[(int64_t)b * a.E] = at; at += v; }
}

__global__ __launch_bounds__(256) void route_scatter_kernel(const RouteArgs a) {
  extern __shared__ __attribute__((aligned(16))) uint8_t dyn[];
  uint32_t* choice = (uint32_t*)dyn;
  int* count = (int*)(choice + ROUTE_ROWS * a.k);
  int* before = count + 4 * a.E;                                // of the sample's workgroups before this one
  int* sums = before + a.E;
  const int s = blockIdx.y, blk = blockIdx.x, t0 = blk * ROUTE_ROWS, n = (min(a.T, t0 + ROUTE_ROWS) - t0) * a.k;
  const int64_t first = ((int64_t)s * a.T + t0) * a.k;
  for (int i = threadIdx.x; i < 4 * a.E; i += 256) count[i] = 0;
  for (int i = threadIdx.x; i < n; i += 256) choice[i] = (uint32_t)a.experts[first + i];
  const int32_t* c = a.counts + (int64_t)s * (a.blocks + 1) * a.E;
  for (int e = threadIdx.x; e < a.E; e += 256) {
    if (a.blocks > ROUTE_BLOCKS) {
      before[e] = c[(int64_t)blk * a.E + e];
      sums[e] = c[(int64_t)a.blocks * a.E + e];
    } else {
      int lower = 0, all = 0;
#pragma unroll 8
      for (int b = 0; b < a.blocks; ++b) {
        const int v = c[(int64_t)b * a.E + e];
        lower += b < blk ? v : 0;
        all += v;
      }
      before[e] = lower;
      sums[e] = all;
    }
  }
  __syncthreads();
  route_count(choice, count, n, a.E);
  const int all = s * a.T * a.k;
  route_prefix(a.E, [&](int e) { return sums[e]; }, [&](int e, int lower) {
    before[e] += all + lower;
    if (blk == 0) a.offsets[s * a.E + e] = all + lower;
  });
  if (blk == 0 && s == a.S - 1 && threadIdx.x == 0) a.offsets[a.S * a.E] = all + a.T * a.k;
  __syncthreads();
  route_starts(count, a.E, [&](int e) { return before[e]; });
  route_place(a, choice, count, n, (int)first);
}

template <int T, int L, int KEY> int launch_route_by(const RouteArgs& a, hipStream_t st) {
  static std::atomic<uint64_t> attr{0};
  const int lds = ROUTE_ROWS * a.k * 8 + a.E * 20 + 16 + (KEY == KEY_LOGIT && T != QBNN_F32 ? 0 : route_waves(L) * route_wave_bytes<L>(a.groups, route_whole(a)));
  if (int rc = qbnn_ensure_dyn_lds((const void*)route_kernel<T, L, KEY>, &attr, 128 * 1024)) return rc;
  hipLaunchKernelGGL((route_kernel<T, L, KEY>), dim3((unsigned)a.blocks, (unsigned)a.S), dim3(route_waves(L) * 64), lds, st, a);
  return qbnn_check_launch_msg("qbnn_route_experts");
}
template <int T, int L> int launch_route_as(const RouteArgs& a, hipStream_t st) {
  if (!a.bias && a.groups == 1) return launch_route_by<T, L, KEY_LOGIT>(a, st);      // both scores increase with the logit
  return a.sigmoid ? launch_route_by<T, L, KEY_SIGMOID>(a, st) : launch_route_by<T, L, KEY_SOFTMAX>(a, st);
}
template <int T> int launch_route(const RouteArgs& a, hipStream_t st) {
  int rc;
  if (a.E <= 16) rc = launch_route_as<T, 1>(a, st);
  else if (a.E <= 32) rc = launch_route_as<T, 2>(a, st);
  else if (a.E <= 64) rc = launch_route_as<T, 4>(a, st);
  else if (a.E <= 128) rc = launch_route_as<T, 8>(a, st);
  else if (a.E <= 256) rc = launch_route_as<T, 16>(a, st);
  else if (a.E <= 512) rc = launch_route_as<T, 32>(a, st);
  else rc = launch_route_as<T, 64>(a, st);
  if (rc || a.blocks == 1) return rc;
  if (a.blocks > ROUTE_BLOCKS) {
    hipLaunchKernelGGL(route_scan_kernel, dim3((unsigned)((a.E + 3) / 4), (unsigned)a.S), dim3(256), 0, st, a);
    if ((rc = qbnn_check_launch_msg("qbnn_route_experts (scan)"))) return rc;
  }
  hipLaunchKernelGGL(route_scatter_kernel, dim3((unsigned)a.blocks, (unsigned)a.S), dim3(256), ROUTE_ROWS * a.k * 4 + a.E * 24, st, a);
  return qbnn_check_launch_msg("qbnn_route_experts (order)");
}

}  // namespace

QBNN_EXPORT int64_t qbnn_route_workspace_ints(int32_t S, int32_t T, int32_t E) {
  return S <= 0 || T <= 0 || E <= 0 ? 0 : (int64_t)S * ((T + ROUTE_ROWS - 1) / ROUTE_ROWS + 1) * E;
}

QBNN_EXPORT int qbnn_route_experts(const qbnn_route* r, void* stream) {
  if (!r || r->S < 0 || r->T < 0 || r->E <= 0 || r->E > QBNN_ROUTE_MAX_EXPERTS || r->top_k <= 0 || r->top_k > QBNN_ROUTE_MAX_CHOICES || r->groups <= 0 || r->groups > 64 ||
      r->E % r->groups || r->top_groups <= 0 || r->top_groups > r->groups || r->top_k > r->E / r->groups * r->top_groups || r->type < QBNN_F32 || r->type > QBNN_F16 ||
      !r->offsets)
    return route_fail("qbnn_route_experts: bad argument (E %ld, top_k %ld)", r ? r->E : 0, r ? r->top_k : 0);
  const int64_t rows = (int64_t)r->S * r->T * r->top_k;
  if (rows > 0x7fffffff || (int64_t)r->S * r->E >= 0x7fffffff) return route_fail("qbnn_route_experts: %ld routed rows do not fit 31 bits", (long)rows);
  if (r->T >= 1 << 29) return route_fail("qbnn_route_experts: %ld rows of a sample are more than a launch has threads for", r->T);      // 512 for each 64 of them, 2^32 in all
  if (rows == 0) return route_fail("qbnn_route_experts: no rows");
  if (!r->logits || !r->weights || !r->experts || !r->rows || !r->workspace || r->S > 65535) return route_fail("qbnn_route_experts: bad argument");
  RouteArgs a;
  a.logits = r->logits; a.l_ss = r->logits_ss; a.l_rs = r->logits_rs; a.bias = r->bias;
  a.weights = r->weights; a.experts = r->experts; a.offsets = r->offsets; a.rows = r->rows; a.counts = r->workspace;
  a.S = r->S; a.T = r->T; a.E = r->E; a.k = r->top_k; a.groups = r->groups; a.kept = r->top_groups; a.sigmoid = r->sigmoid; a.renorm = r->renormalize; a.scale = r->scale;
  a.blocks = (r->T + ROUTE_ROWS - 1) / ROUTE_ROWS;
  for (a.bits = 0; (1 << a.bits) < r->E; ++a.bits) {}
  switch (r->type) {
    case QBNN_F32: return launch_route<QBNN_F32>(a, (hipStream_t)stream);
    case QBNN_BF16: return launch_route<QBNN_BF16>(a, (hipStream_t)stream);
    default: return launch_route<QBNN_F16>(a, (hipStream_t)stream);
  }
}
