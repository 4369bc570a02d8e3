// libqbnn_hip.so: 8-bit floating-point linear layers with one scale for each block of 128 (format: qbnn_f8.h).
//   quantiser   float rows / weights -> e4m3 + block exponents
//   product     y[s][b][n] = act( sum_k x[s][b][k] w[s][n][k] + bias[n] ) for S Monte-Carlo samples in one launch, or over ragged
//               groups of rows, one weight set each (the experts of a routed layer)
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <stdio.h>
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "../../include/qbnn.h"
#include "qbnn_common.h"
#include "qbnn_conv.h"          // LDS-DMA requests, their counted waits, LDS-only barrier
#include "qbnn_f8.h"

using namespace qbnn;

namespace {

static inline int f8_fail(const char* fmt, long a = 0, long b = 0) {
  char buf[512];
  snprintf(buf, sizeof(buf), fmt, a, b);
  return qbnn_fail_msg(QBNN_E_INVALID, buf);
}

// ================================================================================================================================
// Quantiser.  ROWS = 1: a block is 128 columns of one row, 16 lanes x 8 columns; ROWS = 128: a block is 128 x 128, a workgroup each,
// held in registers between the maximum and the conversion, so that the input is read once.
// ================================================================================================================================
struct QuantF8Args {
  const void* x; int64_t x_bs, x_rs;       // batch / row stride in elements; columns are contiguous
  uint8_t* q; uint8_t* e;                  // [batch][R][Kp], [batch][Rb][Sp]
  int R, K, Kb, Sp; int64_t blocks, first; // blocks = batch * Rb * Kb; first: that of the launch (blocks form)
  uint32_t kb_magic, r_magic; int kb_shift, r_shift;      // division by Kb and R: n * magic >> (31 + shift), n < 2^31 (rows form)
};
// n / d for n < 2^31: the smallest p with 2^p >= d gives an error below 1 / d
static void f8_magic(uint32_t d, uint32_t& magic, int& shift) {
  shift = 0;
  while ((1u << shift) < d) ++shift;
  magic = (uint32_t)((((uint64_t)1 << (31 + shift)) + d - 1) / d);
}
__device__ __forceinline__ uint32_t f8_divide(uint32_t n, uint32_t magic, int shift) { return (uint32_t)(((uint64_t)n * magic) >> (31 + shift)); }

// A 16-bit result with block exponents, as the experts' sums take it: fp16 of v 2^-e, e the block's exponent as of e4m3 (so at most 448; inf and NaN stay)
constexpr int F8_HALF = 4;

// 8 columns from `col` of a row of K (zeros behind the last); rows may start at any element's address
template <int T> __device__ __forceinline__ void f8_load8(const f8_type<T>* row, int col, int K, float (&v)[8]) {
  if (col + 8 <= K) {
    f8_type<T> t[8];
    __builtin_memcpy(t, row + col, sizeof(t));
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = f8_load<T>(t[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = col + i < K ? f8_load<T>(row[col + i]) : 0.f;
  }
}
__device__ __forceinline__ uint32_t f8_max8(const float (&v)[8]) {      // of what is finite; a maximum passes NaN over, only infinities need a second look
  float f = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) f = fmaxf(f, fabsf(v[i]));
  uint32_t m = __float_as_uint(f);
  if (m == 0x7f800000u) {
    m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, f8_magnitude(v[i]));
  }
  return m;
}
template <int CTRL> __device__ __forceinline__ uint32_t f8_max_dpp(uint32_t m) { return max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, CTRL, 0xf, 0xf, true)); }
__device__ __forceinline__ uint32_t f8_max16(uint32_t m) {      // over the 16 lanes of a row's block: quads, then halves and rows mirrored
  return f8_max_dpp<0x140>(f8_max_dpp<0x141>(f8_max_dpp<0x4E>(f8_max_dpp<0xB1>(m))));
}
__device__ __forceinline__ f8_v2i f8_scale8(const float (&v)[8], float down) {
  return (f8_v2i){(int)f8_pack4(v[0] * down, v[1] * down, v[2] * down, v[3] * down), (int)f8_pack4(v[4] * down, v[5] * down, v[6] * down, v[7] * down)};
}
// the exponent of block kb; the lane that writes the last block's also clears the pad behind it
__device__ __forceinline__ void f8_put_exponent(uint8_t* row, int kb, int Kb, int Sp, int e) {
  row[kb] = (uint8_t)(e + 127);
  if (kb == Kb - 1)
    for (int i = Kb; i < Sp; ++i) row[i] = 0;
}

// U blocks, 16 apart, in flight per 16 lanes (4 for large inputs, 1 where there are too few blocks to fill the card); TAIL: K is not a multiple of 8
template <int T, int U, bool TAIL> __global__ __launch_bounds__(256) void quantize_f8_rows_kernel(const QuantF8Args a) {
  const int j = threadIdx.x & 15;
  const uint32_t b0 = blockIdx.x * (16 * U) + (threadIdx.x >> 4), blocks = (uint32_t)a.blocks;
  float v[U][8];
  uint32_t r[U];
  int kb[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const uint32_t b = min(b0 + 16 * u, blocks - 1);                // (past the last: done again, to the same bytes)
    r[u] = f8_divide(b, a.kb_magic, a.kb_shift);
    kb[u] = (int)(b - r[u] * (uint32_t)a.Kb);
    const uint32_t bt = f8_divide(r[u], a.r_magic, a.r_shift);
    const f8_type<T>* row = (const f8_type<T>*)a.x + bt * a.x_bs + (int64_t)(r[u] - bt * (uint32_t)a.R) * a.x_rs;
    const int col = kb[u] * 128 + j * 8;
    if constexpr (TAIL) f8_load8<T>(row, col, a.K, v[u]);
    else {
      f8_type<T> t[8] = {};
      if (col < a.K) __builtin_memcpy(t, row + col, sizeof(t));
#pragma unroll
      for (int i = 0; i < 8; ++i) v[u][i] = f8_load<T>(t[i]);
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int e = f8_exponent(f8_max16(f8_max8(v[u])));
    *(f8_v2i*)(a.q + (int64_t)r[u] * ((int64_t)a.Kb * 128) + kb[u] * 128 + j * 8) = f8_scale8(v[u], f8_pow2(-e));
    if (j == 0) f8_put_exponent(a.e + (int64_t)r[u] * a.Sp, kb[u], a.Kb, a.Sp, e);
  }
}

template <int T> __global__ __launch_bounds__(256) void quantize_f8_blocks_kernel(const QuantF8Args a) {
  __shared__ uint32_t red[4];
  const int Rb = (a.R + 127) >> 7;
  const int64_t b = a.first + blockIdx.x;
  const int64_t br = b / a.Kb;
  const int kb = (int)(b - br * a.Kb), j = threadIdx.x & 15, sub = threadIdx.x >> 4;
  const int64_t bt = br / Rb;
  const int r0 = (int)(br - bt * Rb) * 128;
  const f8_type<T>* x = (const f8_type<T>*)a.x + bt * a.x_bs;
  float v[8][8];
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int r = r0 + 16 * i + sub;
    if (r < a.R) f8_load8<T>(x + r * a.x_rs, kb * 128 + j * 8, a.K, v[i]);
    else
#pragma unroll
      for (int c = 0; c < 8; ++c) v[i][c] = 0.f;
    m = max(m, f8_max8(v[i]));
  }
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) m = max(m, (uint32_t)__shfl_xor((int)m, d));
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = m;
  __syncthreads();
  const int e = f8_exponent(max(max(red[0], red[1]), max(red[2], red[3])));
  const float down = f8_pow2(-e);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int r = r0 + 16 * i + sub;
    if (r < a.R) *(f8_v2i*)(a.q + (bt * a.R + r) * ((int64_t)a.Kb * 128) + kb * 128 + j * 8) = f8_scale8(v[i], down);
  }
  if (threadIdx.x == 0) f8_put_exponent(a.e + br * a.Sp, kb, a.Kb, a.Sp, e);
}

template <int T> int launch_quantize_rows(QuantF8Args a, int64_t batch, hipStream_t st) {
  if (a.x_bs == a.R * a.x_rs && batch * a.R < ((int64_t)1 << 31)) { a.R = (int)(batch * a.R); batch = 1; }      // one matrix
  f8_magic((uint32_t)a.Kb, a.kb_magic, a.kb_shift);
  // launches of up to 2^29 blocks and rows: fewer than 2^32 threads
  const int64_t rows = batch * a.R, most = ((int64_t)1 << 29) / a.Kb;
  const int64_t step = rows <= most ? rows : batch == 1 ? most : (most / a.R ? most / a.R * a.R : 0);
  if (step == 0) return f8_fail("qbnn_quantize_f8: a matrix of %ld blocks in a batch", (long)((int64_t)a.R * a.Kb));
  f8_magic((uint32_t)(batch == 1 ? (step < a.R ? step : a.R) : a.R), a.r_magic, a.r_shift);
  for (int64_t r0 = 0; r0 < rows; r0 += step) {
    QuantF8Args c = a;
    const int64_t n = rows - r0 < step ? rows - r0 : step;
    c.blocks = n * a.Kb;
    c.x = (const char*)a.x + (batch == 1 ? r0 * a.x_rs : r0 / a.R * a.x_bs) * (int64_t)sizeof(f8_type<T>);
    if (batch == 1) { c.R = (int)n; f8_magic((uint32_t)n, c.r_magic, c.r_shift); }
    c.q = a.q + r0 * ((int64_t)a.Kb * 128);
    c.e = a.e + r0 * a.Sp;
    const bool many = c.blocks >= 65536;
    const dim3 grid((unsigned)((c.blocks + (many ? 63 : 15)) / (many ? 64 : 16)));
    if (a.K % 8) {
      if (many) hipLaunchKernelGGL((quantize_f8_rows_kernel<T, 4, true>), grid, dim3(256), 0, st, c);
      else hipLaunchKernelGGL((quantize_f8_rows_kernel<T, 1, true>), grid, dim3(256), 0, st, c);
    } else {
      if (many) hipLaunchKernelGGL((quantize_f8_rows_kernel<T, 4, false>), grid, dim3(256), 0, st, c);
      else hipLaunchKernelGGL((quantize_f8_rows_kernel<T, 1, false>), grid, dim3(256), 0, st, c);
    }
    if (int rc = qbnn_check_launch_msg("qbnn_quantize_f8")) return rc;
  }
  return QBNN_OK;
}
template <int T> int launch_quantize(const QuantF8Args& a, int64_t batch, int block_rows, hipStream_t st) {
  if (block_rows == 1) return launch_quantize_rows<T>(a, batch, st);
  QuantF8Args c = a;
  for (c.first = 0; c.first < a.blocks; c.first += 1 << 23) {      // (2^31 threads: a launch of 2^32 or more loses the rest of them without an error)
    hipLaunchKernelGGL((quantize_f8_blocks_kernel<T>), dim3((unsigned)std::min(a.blocks - c.first, (int64_t)1 << 23)), dim3(256), 0, st, c);
    if (int rc = qbnn_check_launch_msg("qbnn_quantize_f8")) return rc;
  }
  return QBNN_OK;
}

// ================================================================================================================================
// Product
// ================================================================================================================================
struct F8Args {
  const uint8_t* x; const uint8_t* xe; int64_t x_ss, xe_ss;
  const uint8_t* w; const uint8_t* we; int64_t w_ss, we_ss;
  const float* bias; int64_t bias_ss;
  uint8_t* y; uint8_t* ye; int64_t y_ss;        // y_ss in elements
  int M, N, Kb, Sp, relu, y_rs, ye_rs;          // y row pitch in elements, exponent pitch of an e4m3 result
  int samples, fold;                            // direct form: fold != 0: row tiles of a sample, tiles of all samples numbered over blockIdx.y and z
  // ragged groups: rows offsets[g] .. offsets[g + 1] of the routed order, with weight set g % w_groups
  const int32_t* offsets; int groups, w_groups;
  const int32_t* rows; int topk, x_rows;        // rows != null: x row of routed row i = (rows[i] / topk) % x_rows, else i
  const int32_t* y_rows; const float* scale;    // y_rows != null: result row i goes to y_rows[i], times scale[y_rows[i]]
};

constexpr int F8_FOLD = 32768;

struct F8Tile { int m0, m1, set, sample; };     // rows m0 .. m1 - 1, weight set, sample (0 for groups: rows are global)

// Groups: the tiles of every group's rows in a row, ceil(rows / TM) each.  One wave-wide pass over the offsets, 64 groups at a time.
template <int TM> __device__ __forceinline__ int f8_group_tiles(const F8Args& a, int g, int& b, int& n) {
  b = 0; n = 0;
  if (g < a.groups) { b = a.offsets[g]; n = a.offsets[g + 1] - b; }
  return (n + TM - 1) / TM;
}
template <int TM> __device__ __forceinline__ int f8_count_tiles(const F8Args& a) {
  const int lane = threadIdx.x & 63;
  int sum = 0, b, n;
  for (int g0 = 0; g0 < a.groups; g0 += 64) sum += f8_group_tiles<TM>(a, g0 + lane, b, n);
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) sum += __shfl_xor(sum, d);
  return __builtin_amdgcn_readfirstlane(sum);
}
// tile t (of a grid sized for the worst split of the rows); false if there are fewer
template <int TM, bool GROUPED> __device__ __forceinline__ bool f8_find_tile(const F8Args& a, int t, int z, F8Tile& o) {
  if constexpr (!GROUPED) {
    o.m0 = t * TM; o.m1 = min(a.M, o.m0 + TM); o.set = z; o.sample = z;
    return true;
  } else {
    const int lane = threadIdx.x & 63;
    int before = 0;
    for (int g0 = 0; g0 < a.groups; g0 += 64) {
      int b, n;
      const int tiles = f8_group_tiles<TM>(a, g0 + lane, b, n);
      int incl = tiles;
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) { const int u = __shfl_up(incl, d); if (lane >= d) incl += u; }
      const int total = __shfl(incl, 63);
      if (t < before + total) {
        const int mine = before + incl - tiles;
        const unsigned long long hit = __ballot(t >= mine && t < mine + tiles);
        const int src = __ffsll(hit) - 1;
        const int k = t - __shfl(mine, src), bb = __shfl(b, src), nn = __shfl(n, src);
        o.m0 = __builtin_amdgcn_readfirstlane(bb + k * TM);
        o.m1 = __builtin_amdgcn_readfirstlane(min(bb + nn, bb + k * TM + TM));
        o.set = __builtin_amdgcn_readfirstlane((g0 + src) % a.w_groups); o.sample = 0;
        return true;
      }
      before += total;
    }
    return false;
  }
}
// The row that offsets into x count from: the tile's first, or x's own first where rows are gathered
template <bool GROUPED> __device__ __forceinline__ int f8_x_base(const F8Args& a, const F8Tile& t) {
  if constexpr (GROUPED) { if (a.rows) return 0; }
  return t.m0;
}
template <bool GROUPED> __device__ __forceinline__ int f8_x_row(const F8Args& a, int i) {
  if constexpr (GROUPED) { if (a.rows) return (a.rows[i] / a.topk) % a.x_rows; }
  return i;
}

// four consecutive results (weight rows n .. n + 3) of activation row i
template <int OUT, bool GROUPED> __device__ __forceinline__ void f8_put4(const F8Args& a, const F8Tile& t, int i, int n, f8_v4f v) {
  const float* bias = a.bias ? a.bias + (int64_t)t.set * a.bias_ss : nullptr;
  int64_t row = i;
  float s = 1.f;
  bool weighed = false;
  if constexpr (GROUPED) { if (a.y_rows) { row = a.y_rows[i]; s = a.scale[row]; weighed = true; } }
  f8_type<OUT> o[4];
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    float u = v[c];
    if (bias && n + c < a.N) u += bias[n + c];
    if (a.relu) u = u > 0.f ? u : (u != u ? u : 0.f);          // (a NaN stays one)
    if (weighed) u = s == 0.f ? 0.f : u * s;                   // (an expert of weight 0 adds nothing, whatever it computed)
    o[c] = f8_store<OUT>(u);
  }
  f8_type<OUT>* y = (f8_type<OUT>*)a.y + (int64_t)t.sample * a.y_ss + row * a.y_rs + n;
  if (n + 4 <= a.N) __builtin_memcpy(y, o, sizeof(o));
  else
    for (int c = 0; c < 4; ++c) if (n + c < a.N) y[c] = o[c];
}

// Direct form: operands straight from memory into the matrix instruction's registers, the waves of a workgroup split the columns and
// join their sums in LDS in a fixed order.  For few rows, where the weights are read once and nothing is used twice: what counts is bytes in flight, so a
// wave asks for D blocks of columns (1, 2 or 4: one dword of exponents) before it multiplies the first.
template <int MT, int NT, int NW, int D, int OUT, bool EXACT, bool GROUPED>
__global__ __launch_bounds__(NW * 64) void linear_f8_direct_kernel(const F8Args a) {
  __shared__ __attribute__((aligned(16))) f8_v4f red[NW > 1 ? NW : 1][MT * NT * 64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r16 = lane & 15, h = lane >> 4;
  F8Tile t;
  int row_tile = blockIdx.y, sample = blockIdx.z;
  if (a.fold) {
    const int64_t q = (int64_t)blockIdx.z * F8_FOLD + blockIdx.y;
    sample = (int)(q / a.fold);
    row_tile = (int)(q - (int64_t)sample * a.fold);
    if (sample >= a.samples) return;
  }
  if (!f8_find_tile<16 * MT, GROUPED>(a, row_tile, sample, t)) return;
  const int n0 = blockIdx.x * (16 * NT);
  const int64_t pitch = (int64_t)a.Kb * 128;
  const uint8_t* xp[MT]; const uint8_t* xep[MT];
  const uint8_t* wp[NT]; const uint8_t* wep[NT];
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    const int row = min(n0 + 16 * j + r16, a.N - 1);
    wp[j] = a.w + (int64_t)t.set * a.w_ss + row * pitch + h * 16;
    wep[j] = a.we + (int64_t)t.set * a.we_ss + (int64_t)(row >> 7) * a.Sp;
  }
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    const int row = f8_x_row<GROUPED>(a, min(t.m0 + 16 * i + r16, t.m1 - 1));      // a row behind the last repeats it: its result is not stored
    xp[i] = a.x + (int64_t)t.sample * a.x_ss + row * pitch + h * 16;
    xep[i] = a.xe + (int64_t)t.sample * a.xe_ss + (int64_t)row * a.Sp;
  }
  f8_v4f acc[MT][NT];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) acc[i][j] = (f8_v4f){0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
  for (int k0 = wave * D; k0 < a.Kb; k0 += NW * D) {
    f8_v8i xf[D][MT], wf[D][NT];
    uint32_t xs[MT], ws[NT];
#pragma unroll
    for (int d = 0; d < D; ++d) {
      const int at = min(k0 + d, a.Kb - 1) * 128;               // (past the last block: read again, not multiplied)
#pragma unroll
      for (int j = 0; j < NT; ++j) wf[d][j] = f8_join(*(const f8_v4i*)(wp[j] + at), *(const f8_v4i*)(wp[j] + at + 64));
    }
#pragma unroll
    for (int d = 0; d < D; ++d) {
      const int at = min(k0 + d, a.Kb - 1) * 128;
#pragma unroll
      for (int i = 0; i < MT; ++i) xf[d][i] = f8_join(*(const f8_v4i*)(xp[i] + at), *(const f8_v4i*)(xp[i] + at + 64));
    }
#pragma unroll
    for (int j = 0; j < NT; ++j) ws[j] = *(const uint32_t*)(wep[j] + (k0 & ~3)) >> ((k0 & 3) * 8);
#pragma unroll
    for (int i = 0; i < MT; ++i) xs[i] = *(const uint32_t*)(xep[i] + (k0 & ~3)) >> ((k0 & 3) * 8);
    auto multiply = [&](auto Dc) {
      constexpr int d = decltype(Dc)::value;
      if constexpr (EXACT) {
        F8Wide xw[MT];
#pragma unroll
        for (int i = 0; i < MT; ++i) xw[i] = f8_widen(xf[d][i], xs[i] >> (8 * d));
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          const F8Wide ww = f8_widen(wf[d][j], ws[j] >> (8 * d));
#pragma unroll
          for (int i = 0; i < MT; ++i) acc[i][j] = f8_mfma_exact(ww, xw[i], acc[i][j]);
        }
      } else {
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int j = 0; j < NT; ++j) acc[i][j] = f8_mfma<d>(wf[d][j], xf[d][i], acc[i][j], ws[j], xs[i]);
      }
    };
    multiply(std::integral_constant<int, 0>{});
    if constexpr (D > 1) { if (k0 + 1 < a.Kb) multiply(std::integral_constant<int, 1>{}); }
    if constexpr (D > 2) { if (k0 + 2 < a.Kb) multiply(std::integral_constant<int, 2>{}); }
    if constexpr (D > 2) { if (k0 + 3 < a.Kb) multiply(std::integral_constant<int, 3>{}); }
  }
  if constexpr (OUT == QBNN_F8) {
    static_assert(NT == 8, "a block of an e4m3 result is 128 columns of a row");
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int j = 0; j < NT; ++j) red[wave][(i * NT + j) * 64 + lane] = acc[i][j];
    __syncthreads();
    // 16 threads per row: thread c sums and converts columns 8 c .. + 7 = parts 2 (c & 1), + 1 of weight tile c / 2
    const float* bias = a.bias ? a.bias + (int64_t)t.set * a.bias_ss : nullptr;
    for (int u = threadIdx.x; u < MT * 256; u += NW * 64) {
      const int i = u >> 8, r = (u >> 4) & 15, c = u & 15, row = t.m0 + 16 * i + r;
      float v[8];
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        const int at = (i * NT + (c >> 1)) * 64 + (2 * (c & 1) + p) * 16 + r;
        f8_v4f s = red[0][at];
#pragma unroll
        for (int k = 1; k < NW; ++k) s += red[k][at];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int n = n0 + c * 8 + p * 4 + q;
          float o = s[q];
          if (bias && n < a.N) o += bias[n];
          if (a.relu) o = o > 0.f ? o : (o != o ? o : 0.f);
          v[p * 4 + q] = n < a.N ? o : 0.f;
        }
      }
      const int e = f8_exponent(f8_max16(f8_max8(v)));
      if (row < t.m1) {
        *(f8_v2i*)(a.y + (int64_t)t.sample * a.y_ss + (int64_t)row * a.y_rs + n0 + c * 8) = f8_scale8(v, f8_pow2(-e));
        if (c == 0) f8_put_exponent(a.ye + ((int64_t)t.sample * a.M + row) * a.ye_rs, blockIdx.x, gridDim.x, a.ye_rs, e);
      }
    }
  } else {
    if constexpr (NW > 1) {
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) red[wave][(i * NT + j) * 64 + lane] = acc[i][j];
      __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        if ((i * NT + j) % NW != wave) continue;
        f8_v4f s = acc[i][j];
        if constexpr (NW > 1) {
          s = red[0][(i * NT + j) * 64 + lane];
#pragma unroll
          for (int k = 1; k < NW; ++k) s += red[k][(i * NT + j) * 64 + lane];
        }
        const int row = t.m0 + 16 * i + r16, n = n0 + 16 * j + 4 * h;
        if (row < t.m1 && n < a.N) f8_put4<OUT == QBNN_F8 ? QBNN_F32 : OUT, GROUPED>(a, t, row, n, s);
      }
  }
}

template <int MT, int NT, int NW, int D, int OUT, bool EXACT, bool GROUPED> int launch_direct(const F8Args& a, int64_t tiles, int z, hipStream_t st) {
  F8Args c = a;
  dim3 grid((unsigned)((a.N + 16 * NT - 1) / (16 * NT)), (unsigned)tiles, (unsigned)z);
  if (tiles > 65535 || z > 65535) {                             // (f8_fits: fewer than 2^31 of them)
    c.samples = z; c.fold = (int)tiles;
    grid.y = F8_FOLD; grid.z = (unsigned)((tiles * z + F8_FOLD - 1) / F8_FOLD);
  }
  hipLaunchKernelGGL((linear_f8_direct_kernel<MT, NT, NW, D, OUT, EXACT, GROUPED>), grid, dim3(NW * 64), 0, st, c);
  return qbnn_check_launch_msg("qbnn_linear_f8");
}

// Tiled form: TM activation rows x TN weight rows per workgroup, WM x WN waves of (32 MI) x 128 each, one block of 128 columns per step.
// Both operands' rows go to LDS by DMA, two steps in two buffers; a row's eight 16-byte pieces lie permuted (piece c of row r at c ^ f(r)), f such that the
// 16 lanes whose 16 bytes the LDS serves in one cycle (0-3, 12-15, 20-27 and 4-11, 16-19, 28-31 of each half wave) hit 16 different places modulo 256.  What bounds it at large sizes is the matrix unit: 4 waves of 128 x 128 read 2 x 16 KiB each and step, 128 KiB at
// 128 B/clk = 1024 cycles, for 32 instructions of 64 cycles; with waves of 128 x 64 the LDS would be the bound.  The 32 x 32 form of the instruction, because
// its accumulators are tied in place (the 16 x 16 form's are renamed, which cost 3 register moves per instruction here) and it reads half the operand registers.
// One barrier per step, in front of the last activation fragment's products: before it the wave waits for its share of the next step's bytes; behind it
// the buffer just read is requested again and the next step's first fragments are read, each weight fragment's registers as soon as their products are issued.
constexpr int F8_PITCH = 132, F8_STAGE = 32 * F8_PITCH * 4 + 128 * 8;      // a wave's stage behind the products, see f8_finish
template <int MI, int WM, int WN> struct F8Tiled {
  static constexpr int TM = 32 * MI * WM, TN = 128 * WN, WAVES = WM * WN, XB = TM * 128, WB = TN * 128;
  static constexpr int LDS = 2 * (XB + WB) > WAVES * F8_STAGE ? 2 * (XB + WB) : WAVES * F8_STAGE;      // the operands, and then the stages
  static constexpr int PX = TM / 8 / WAVES, PW = TN / 8 / WAVES;      // DMA requests (8 rows each) per wave and step
  static_assert(TM % (8 * WAVES) == 0 && TN % (8 * WAVES) == 0 && LDS <= 160 * 1024 && 2 * XB <= 65536 && 2 * WB <= 65536, "immediate offsets of the reads");
};
typedef float f8_v16f __attribute__((ext_vector_type(16)));

// Workgroups of one XCD (every eighth) take neighbouring tiles, in columns of 4 row tiles, sample after sample: what they read at a time shares its L2.
// false: no tile.
template <int TM, int TN, bool GROUPED> __device__ __forceinline__ bool f8_locate(const F8Args& a, int tiles_m, int tiles_n, int samples, F8Tile& t, int& n0) {
  const int tm = GROUPED ? f8_count_tiles<TM>(a) : tiles_m, each = tm * tiles_n, total = each * samples;
  const int p = blockIdx.x;
  if (p >= total) return false;
  const int per = total >> 3, rest = total & 7, xcd = p & 7;
  int q = xcd * per + min(xcd, rest) + (p >> 3);
  const int z = GROUPED ? 0 : q / each;
  q -= z * each;
  const int band = q / (4 * tiles_n), in = q - band * (4 * tiles_n), rows = min(4, tm - band * 4);
  const int col = in / rows;
  n0 = col * TN;
  return f8_find_tile<TM, GROUPED>(a, band * 4 + in - col * rows, z, t);
}

// Results of a wave's (32 G) x 128 tile from row m, weight row nw on, 32 rows at a time through `stage` (F8_STAGE bytes of LDS of this wave's own, no longer read
// by anyone; put(i, st) writes rows 32 i .. + 31 there, F8_PITCH floats each): 16 lanes then write 128 neighbouring columns of a row.  Stored from the
// accumulators' layout they were 32 bytes of each of 32 rows per instruction, and with the bounds unrolled 30 KiB of code: 27,000 cycles a tile, as much as 11 steps.
// AT_ONCE passes of 4 rows without a branch between them: one by one each waited for its own reads (30,900 cycles of a routed 256 x 256 tile, now 18,300).
__device__ __forceinline__ float f8_relu(float u) { return __builtin_elementwise_maximum(u, 0.f); }      // (a NaN stays one)
// Where a wave's 32 G rows go and their weights (G = 4: two rows a lane).  Two dependent loads: in front of the products where registers are left, so that they are not waited for behind them.
template <int G> struct F8Moves {
  int to[(G + 1) / 2];
  float weight[(G + 1) / 2];
  __device__ __forceinline__ void rows(const F8Args& a, const F8Tile& t, int m) {
#pragma unroll
    for (int i = 0; i < (G + 1) / 2; ++i) to[i] = a.y_rows[min(m + i * 64 + (int)(threadIdx.x & 63), t.m1 - 1)];
  }
  __device__ __forceinline__ void weights(const F8Args& a) {
#pragma unroll
    for (int i = 0; i < (G + 1) / 2; ++i) weight[i] = a.scale[to[i]];
  }
};
template <int OUT, bool GROUPED> constexpr bool f8_moves() { return GROUPED && OUT != QBNN_F8; }
template <int G, int OUT, bool GROUPED, bool WHOLE, class Put>
__device__ __forceinline__ void f8_finish_as(const F8Args& a, const F8Tile& t, int m, int nw, uint8_t* stage, const F8Moves<G>& moves, Put put) {
  const int lane = threadIdx.x & 63, n = (lane & 15) * 8;
  const int in = WHOLE ? 8 : a.N - nw - n;                      // columns of this lane that exist
  float b[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  if (a.bias) {
    const float* bias = a.bias + (int64_t)t.set * a.bias_ss + nw + n;
    if constexpr (WHOLE) __builtin_memcpy(b, bias, sizeof(b));
    else
#pragma unroll
      for (int c = 0; c < 8; ++c) b[c] = c < in ? bias[c] : 0.f;
  }
  float* st = (float*)stage;
  int* const to_row = (int*)(stage + 32 * F8_PITCH * 4);
  float* const to_weight = (float*)(to_row + 32 * G);
  constexpr bool moved = f8_moves<OUT, GROUPED>();
  const bool relu = GROUPED ? OUT == QBNN_F8 : a.relu != 0;     // (experts: behind the first product)
  if constexpr (moved) {
#pragma unroll
    for (int i = 0; i < (G + 1) / 2; ++i)
      if (i * 64 + lane < 32 * G) { to_row[i * 64 + lane] = moves.to[i]; to_weight[i * 64 + lane] = moves.weight[i]; }
  }
#pragma unroll
  for (int i = 0; i < G; ++i) {
    put(i, st);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");      // (the wave's own LDS: no barrier)
    constexpr int AT_ONCE = WHOLE ? 4 : 2;
#pragma unroll 1
    for (int p0 = 0; p0 < 8; p0 += AT_ONCE) {
      const int r0 = p0 * 4 + (lane >> 4);
      float v[AT_ONCE][8], s[AT_ONCE];
      int64_t to[AT_ONCE];
#pragma unroll
      for (int p = 0; p < AT_ONCE; ++p) {
        const int r = r0 + p * 4;
        const f8_v4f lo = *(const f8_v4f*)(st + r * F8_PITCH + n), hi = *(const f8_v4f*)(st + r * F8_PITCH + n + 4);
#pragma unroll
        for (int c = 0; c < 4; ++c) { v[p][c] = lo[c]; v[p][4 + c] = hi[c]; }
        to[p] = m + i * 32 + r;
        s[p] = 1.f;
        if constexpr (moved) { to[p] = to_row[i * 32 + r]; s[p] = to_weight[i * 32 + r]; }
      }
#pragma unroll
      for (int p = 0; p < AT_ONCE; ++p)
#pragma unroll
        for (int c = 0; c < 8; ++c) v[p][c] += b[c];
      if (relu) {
#pragma unroll
        for (int p = 0; p < AT_ONCE; ++p)
#pragma unroll
          for (int c = 0; c < 8; ++c) v[p][c] = f8_relu(v[p][c]);
      }
      if constexpr (moved) {
        bool none = false;
#pragma unroll
        for (int p = 0; p < AT_ONCE; ++p) none |= s[p] == 0.f;
        if (__any(none)) {                                      // (an expert of weight 0 adds nothing, whatever it computed)
#pragma unroll
          for (int p = 0; p < AT_ONCE; ++p)
#pragma unroll
            for (int c = 0; c < 8; ++c) v[p][c] = s[p] == 0.f ? 0.f : v[p][c];
        }
        if constexpr (OUT != F8_HALF) {                         // (there it is one factor with the block's)
#pragma unroll
          for (int p = 0; p < AT_ONCE; ++p)
#pragma unroll
            for (int c = 0; c < 8; ++c) v[p][c] *= s[p];
        }
      }
      if constexpr (OUT == QBNN_F8 || OUT == F8_HALF) {
        uint32_t top[AT_ONCE];
        bool inf = false;
#pragma unroll
        for (int p = 0; p < AT_ONCE; ++p) {
          float f = 0.f;
#pragma unroll
          for (int c = 0; c < 8; ++c) {
            if (!WHOLE && c >= in) v[p][c] = 0.f;
            f = fmaxf(f, fabsf(v[p][c]));
          }
          top[p] = __float_as_uint(f);
          inf |= top[p] == 0x7f800000u;
        }
        if (__any(inf)) {
#pragma unroll
          for (int p = 0; p < AT_ONCE; ++p) top[p] = f8_max8(v[p]);
        }
#pragma unroll
        for (int p = 0; p < AT_ONCE; ++p) {
          top[p] = f8_max16(top[p]);
          if constexpr (OUT == F8_HALF) top[p] = min(__float_as_uint(__uint_as_float(top[p]) * s[p]) & 0x7fffffffu, 0x7f7fffffu);      // (an overflow: the largest scale, the others stay finite)
        }
        int e[AT_ONCE];
        float by[AT_ONCE];
        f8_v4i o[AT_ONCE];
        bool far = false;
#pragma unroll
        for (int p = 0; p < AT_ONCE; ++p) {
          e[p] = f8_exponent(top[p]);
          by[p] = OUT == F8_HALF ? s[p] * f8_pow2(-e[p]) : f8_pow2(-e[p]);
          far |= OUT == F8_HALF && !(fabsf(by[p]) < INFINITY);
        }
        if (OUT == F8_HALF && __any(far)) {                     // tiny results under a large weight: one after the other
#pragma unroll
          for (int p = 0; p < AT_ONCE; ++p) {
            by[p] = f8_pow2(-e[p]);
#pragma unroll
            for (int c = 0; c < 8; ++c) v[p][c] *= s[p];
          }
        }
#pragma unroll
        for (int p = 0; p < AT_ONCE; ++p) {
          const float down = by[p];
          if constexpr (OUT == QBNN_F8) {
            const f8_v2i q = f8_scale8(v[p], down);
            o[p][0] = q[0];
            o[p][1] = q[1];
          } else {
#pragma unroll
            for (int c = 0; c < 4; ++c) o[p][c] = f8_store2<QBNN_F16>(v[p][2 * c] * down, v[p][2 * c + 1] * down);
          }
        }
#pragma unroll
        for (int p = 0; p < AT_ONCE; ++p) {
          if (m + i * 32 + r0 + p * 4 >= t.m1) continue;
          if constexpr (OUT == QBNN_F8) {
            *(f8_v2i*)(a.y + (int64_t)t.sample * a.y_ss + to[p] * a.y_rs + nw + n) = (f8_v2i){o[p][0], o[p][1]};
            if (n == 0) f8_put_exponent(a.ye + ((int64_t)t.sample * a.M + to[p]) * a.ye_rs, nw >> 7, (a.N + 127) >> 7, a.ye_rs, e[p]);
          } else {
            *(f8_v4i*)(a.y + (to[p] * a.y_rs + nw + n) * 2) = o[p];
            if (n == 0) a.ye[to[p] * a.ye_rs + (nw >> 7)] = (uint8_t)(e[p] + 127);
          }
        }
      } else {
#pragma unroll
        for (int p = 0; p < AT_ONCE; ++p) {
          const int r = r0 + p * 4;
          if (m + i * 32 + r >= t.m1) continue;
          f8_type<OUT>* y = (f8_type<OUT>*)a.y + (int64_t)t.sample * a.y_ss + to[p] * a.y_rs + nw + n;
          if (!WHOLE && in < 8) {                               // the lane at the end: its values by way of the stage, one by one
            *(f8_v4f*)(st + r * F8_PITCH + n) = (f8_v4f){v[p][0], v[p][1], v[p][2], v[p][3]};
            *(f8_v4f*)(st + r * F8_PITCH + n + 4) = (f8_v4f){v[p][4], v[p][5], v[p][6], v[p][7]};
#pragma unroll 1
            for (int c = 0; c < in; ++c) y[c] = f8_store<OUT>(st[r * F8_PITCH + n + c]);
          } else if constexpr (OUT == QBNN_F32) {
            __builtin_memcpy(y, v[p], sizeof(v[p]));
          } else {
            f8_v4i o;
#pragma unroll
            for (int c = 0; c < 4; ++c) o[c] = f8_store2<OUT>(v[p][2 * c], v[p][2 * c + 1]);
            __builtin_memcpy(y, &o, sizeof(o));
          }
        }
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  }
}
template <int G, int OUT, bool GROUPED, class Put>
__device__ __forceinline__ void f8_finish(const F8Args& a, const F8Tile& t, int m, int nw, uint8_t* stage, const F8Moves<G>& moves, Put put) {
  if (nw >= a.N || m >= t.m1) return;
  if (nw + 128 <= a.N) f8_finish_as<G, OUT, GROUPED, true>(a, t, m, nw, stage, moves, put);
  else f8_finish_as<G, OUT, GROUPED, false>(a, t, m, nw, stage, moves, put);
}

// The exponents of 16 steps of a row: four dwords, used from the bottom and moved down two bytes every two steps.  A load's result may only be waited for
// together with every request issued before it, so they are loaded 16 steps at a time and waited for at once, outside of the loop over the steps.
struct F8Exponents {
  uint32_t d[4];
  __device__ __forceinline__ void load(const uint8_t* row, int kb, int Sp) {
#pragma unroll
    for (int i = 0; i < 4; ++i) d[i] = *(const uint32_t*)(row + min(kb + 4 * i, Sp - 4));
  }
  __device__ __forceinline__ void arrive() {
#pragma unroll
    for (int i = 0; i < 4; ++i) asm volatile("" : "+v"(d[i]));
  }
  __device__ __forceinline__ void down() {
#pragma unroll
    for (int i = 0; i < 3; ++i) d[i] = __builtin_amdgcn_alignbit(d[i + 1], d[i], 16);
    d[3] >>= 16;
  }
};

template <int MI, int WM, int WN, int OUT, bool EXACT, bool GROUPED>
__global__ __launch_bounds__(WM * WN * 64, 1) void linear_f8_tiled_kernel(const F8Args a, int tiles_m, int tiles_n, int samples) {
  using C = F8Tiled<MI, WM, WN>;
  extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r32 = lane & 31, h = lane >> 5;
  const int wm = wave / WN, wn = wave % WN;

  F8Tile t;
  int n0;
  if (!f8_locate<C::TM, C::TN, GROUPED>(a, tiles_m, tiles_n, samples, t, n0)) return;
  const int64_t pitch = (int64_t)a.Kb * 128;
  const int base = f8_x_base<GROUPED>(a, t);
  const uint8_t* xg = a.x + (int64_t)t.sample * a.x_ss + base * pitch;
  const uint8_t* wg = a.w + (int64_t)t.set * a.w_ss + n0 * pitch;

  // per-lane byte offsets of this wave's DMA requests; rows behind the last repeat it (their results are not stored)
  uint32_t xo[C::PX], wo[C::PW];
#pragma unroll
  for (int p = 0; p < C::PX; ++p) {
    const int r = (p * C::WAVES + wave) * 8 + (lane >> 3), i = min(t.m0 + r, t.m1 - 1);
    xo[p] = (uint32_t)((f8_x_row<GROUPED>(a, i) - base) * pitch) + (((lane & 7) ^ ((r >> 1) & 7)) << 4);
  }
#pragma unroll
  for (int p = 0; p < C::PW; ++p) {
    const int r = (p * C::WAVES + wave) * 8 + (lane >> 3);
    wo[p] = (uint32_t)(min(r, a.N - 1 - n0) * pitch) + (((lane & 7) ^ ((r >> 1) & 7)) << 4);
  }
  const uint32_t lds0 = lds_addr_of(lds);
  auto request = [&](int kb, int buf) {
    const uint32_t at = lds0 + wave * 1024;
#pragma unroll
    for (int p = 0; p < C::PX; ++p) f8_dma16(xg + kb * 128, xo[p], at + buf * C::XB + p * (C::WAVES * 1024));
#pragma unroll
    for (int p = 0; p < C::PW; ++p) f8_dma16(wg + kb * 128, wo[p], at + 2 * C::XB + buf * C::WB + p * (C::WAVES * 1024));
  };

  const uint8_t* xeg = a.xe + (int64_t)t.sample * a.xe_ss + (int64_t)base * a.Sp;
  uint32_t xeo[MI];
#pragma unroll
  for (int i = 0; i < MI; ++i) xeo[i] = (uint32_t)(f8_x_row<GROUPED>(a, min(t.m0 + (wm * MI + i) * 32 + r32, t.m1 - 1)) - base) * (uint32_t)a.Sp;
  const uint8_t* we = a.we + (int64_t)t.set * a.we_ss + (int64_t)min((n0 >> 7) + wn, (a.N - 1) >> 7) * a.Sp;
  F8Exponents xs[MI], ws;

  // a fragment of 32 rows x 128 columns: instruction s = 0, 1 of the two takes pieces 4 s + h and 4 s + 2 + h
  struct Frag { f8_v8i k[2]; };
  const uint8_t* xl = lds + wm * MI * 4096 + r32 * 128;
  const uint8_t* wl = lds + 2 * C::XB + wn * 16384 + r32 * 128;
  const int piece = (h ^ ((r32 >> 1) & 7)) << 4;
  const uint8_t *x0 = xl + piece, *x1 = xl + (piece ^ 32), *x2 = xl + (piece ^ 64), *x3 = xl + (piece ^ 96);
  const uint8_t *w0 = wl + piece, *w1 = wl + (piece ^ 32), *w2 = wl + (piece ^ 64), *w3 = wl + (piece ^ 96);
  auto read_x = [&](int buf, int i) {
    const int at = buf * C::XB + i * 4096;
    return Frag{{f8_join(*(const f8_v4i*)(x0 + at), *(const f8_v4i*)(x1 + at)), f8_join(*(const f8_v4i*)(x2 + at), *(const f8_v4i*)(x3 + at))}};
  };
  auto read_w = [&](int buf, int j) {
    const int at = buf * C::WB + j * 4096;
    return Frag{{f8_join(*(const f8_v4i*)(w0 + at), *(const f8_v4i*)(w1 + at)), f8_join(*(const f8_v4i*)(w2 + at), *(const f8_v4i*)(w3 + at))}};
  };
  f8_v16f acc[MI][4];
#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int c = 0; c < 16; ++c) acc[i][j][c] = 0.f;

  // a request past the last step repeats the last one's bytes, into a buffer that is not read again: the loop stays free of branches, over which the
  // compiler would move the matrix instructions and spill their operands
  const int last = a.Kb - 1;
  request(0, 0);
  request(min(1, last), 1);
  wait_vmcnt<C::PX + C::PW>();
  lds_barrier();

  if constexpr (!EXACT) {
    Frag wf[4], xf[2];
#pragma unroll
    for (int j = 0; j < 4; ++j) wf[j] = read_w(0, j);
    xf[0] = read_x(0, 0);
    // even and odd steps differ in the buffer and in the byte B of xs / ws that holds their exponents
    auto step = [&](auto Bc, int kb) {
      constexpr int B = decltype(Bc)::value;
      constexpr int X0 = MI & 1 ? B : 0;      // registers of the step's first activation fragment
      auto mfma = [&](int i, int j, int s) {
        acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(wf[j].k[s], xf[(i + X0) & 1].k[s], acc[i][j], 0, 0, B, (int)ws.d[0], B, (int)xs[i].d[0]);
      };
#pragma unroll
      for (int i = 0; i < MI - 1; ++i) {
        xf[(i + 1 + X0) & 1] = read_x(B, i + 1);
#pragma unroll
        for (int u = 0; u < 8; ++u) mfma(i, u & 3, u >> 2);
        __builtin_amdgcn_sched_barrier(0);
      }
      wait_vmcnt<0>();
      lds_barrier();
      xf[(MI + X0) & 1] = read_x(B ^ 1, 0);
      request(min(kb + 2, last), B);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int j = 0; j < 4; j += 2) {
#pragma unroll
        for (int u = 0; u < 4; ++u) mfma(MI - 1, j + (u & 1), u >> 1);
        wf[j] = read_w(B ^ 1, j);
        wf[j + 1] = read_w(B ^ 1, j + 1);
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    for (int k0 = 0; k0 < a.Kb; k0 += 16) {
#pragma unroll
      for (int i = 0; i < MI; ++i) xs[i].load(xeg + xeo[i], k0, a.Sp);
      ws.load(we, k0, a.Sp);
#pragma unroll
      for (int i = 0; i < MI; ++i) xs[i].arrive();
      ws.arrive();
      const int end = min(k0 + 16, a.Kb);
      int kb = k0;
      for (; kb + 1 < end; kb += 2) {
        step(std::integral_constant<int, 0>{}, kb);
        step(std::integral_constant<int, 1>{}, kb + 1);
#pragma unroll
        for (int i = 0; i < MI; ++i) xs[i].down();
        ws.down();
      }
      if (kb < end) step(std::integral_constant<int, 0>{}, kb);
    }
  } else {
    for (int kb = 0; kb < a.Kb; ++kb) {
      const int buf = kb & 1;
      if ((kb & 15) == 0) {
#pragma unroll
        for (int i = 0; i < MI; ++i) xs[i].load(xeg + xeo[i], kb, a.Sp);
        ws.load(we, kb, a.Sp);
#pragma unroll
        for (int i = 0; i < MI; ++i) xs[i].arrive();
        ws.arrive();
      }
      const int byte = (kb & 1) * 8;
      F8Wide xw[MI][2], ww[4][2];
#pragma unroll
      for (int i = 0; i < MI; ++i) {
        const Frag f = read_x(buf, i);
        xw[i][0] = f8_widen(f.k[0], xs[i].d[0] >> byte);
        xw[i][1] = f8_widen(f.k[1], xs[i].d[0] >> byte);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const Frag f = read_w(buf, j);
        ww[j][0] = f8_widen(f.k[0], ws.d[0] >> byte);
        ww[j][1] = f8_widen(f.k[1], ws.d[0] >> byte);
      }
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int g = 0; g < 4; ++g)
#pragma unroll
          for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int i = 0; i < MI; ++i) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(ww[j][s].part[g], xw[i][s].part[g], acc[i][j], 0, 0, 0);
      if (kb & 1) {
#pragma unroll
        for (int i = 0; i < MI; ++i) xs[i].down();
        ws.down();
      }
      wait_vmcnt<0>();
      lds_barrier();
      request(min(kb + 2, last), buf);
    }
  }
  wait_vmcnt<0>();          // (no request outlives the workgroup's LDS)

  lds_barrier();            // ... and no wave reads another's operands any more
  // lane: activation row r32 of fragment i, weight rows 8 q + 4 h .. + 3 of fragment j in registers 4 q .. + 3
  F8Moves<MI> moves;
  if constexpr (f8_moves<OUT, GROUPED>()) { moves.rows(a, t, t.m0 + wm * MI * 32); moves.weights(a); }
  f8_finish<MI, OUT, GROUPED>(a, t, t.m0 + wm * MI * 32, n0 + wn * 128, lds + wave * F8_STAGE, moves, [&](int i, float* st) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q)
        *(f8_v4f*)(st + r32 * F8_PITCH + j * 32 + q * 8 + h * 4) = (f8_v4f){acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
  });
}

template <int MI, int WM, int WN, int OUT, bool EXACT, bool GROUPED> int launch_tiled(const F8Args& a, int rows, int z, hipStream_t st) {
  using C = F8Tiled<MI, WM, WN>;
  static std::atomic<uint64_t> attr{0};
  if (int rc = qbnn_ensure_dyn_lds((const void*)linear_f8_tiled_kernel<MI, WM, WN, OUT, EXACT, GROUPED>, &attr, C::LDS)) return rc;
  const int64_t tm = ((int64_t)rows + C::TM - 1) / C::TM + (GROUPED ? std::min(a.groups, rows) : 0), tn = (a.N + C::TN - 1) / C::TN;
  hipLaunchKernelGGL((linear_f8_tiled_kernel<MI, WM, WN, OUT, EXACT, GROUPED>), dim3((unsigned)(tm * tn * z)), dim3(C::WAVES * 64), C::LDS, st, a, (int)tm, (int)tn, z);
  return qbnn_check_launch_msg("qbnn_linear_f8");
}

// The largest tile, 256 x 256, 4 waves of 128 x 128, two steps of operands (64 KiB each) in LDS.  What the wave issues between two matrix instructions has 32 cycles,
// so requests and reads go one by one behind one instruction each (eight requests in a row held the wave at the address unit for longer than the
// matrix unit had work: 528 -> 476 us at 8192^3), and the loop holds nothing that waits for memory but the barrier that hands over a step:
//   first half   x0 .. x3 times w; reads x4 .. x7; then everything of this step is in registers: barrier, its buffer is requested for the step after the next
//   second half  wait for the next step, barrier; x4 .. x7 times w; reads the next step's x0 .. x3 and w, each fragment into its registers behind its last product
// The exponents come the same way, a dword (four steps) of each row every two steps: as loads into registers they were waited for together with every
// request issued before them, which emptied the ring.
// 8192^3: 370 us replayed from a graph, 2.97 PFLOP/s (447 under the profiler from idle).  At this rate the card is bound by power (1.5 - 1.9 GHz on normal data), and the 16 x 16 x 128 form draws less of it than 32 x 32 x 64 (alone: 4,080 against
// 3,500 TFLOP/s).  The compiler gives its result other registers than its addend, for which 256 accumulators leave none; so the instruction is written
// out, in place.  An accumulator is read again 32 instructions later or behind the wait at the end, which is what its hazards ask for.
template <int B> __device__ __forceinline__ void f8_mfma_in_place(f8_v4f& acc, const f8_v8i& w, const f8_v8i& x, uint32_t ws, uint32_t xs) {      // exponents: byte B
  static_assert(B == 0 || B == 1, "");
  if constexpr (B == 0) asm volatile("v_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel_hi:[0,0,0]" : "+a"(acc) : "v"(w), "v"(x), "v"(ws), "v"(xs));
  else asm volatile("v_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel:[1,1,0] op_sel_hi:[0,0,0]" : "+a"(acc) : "v"(w), "v"(x), "v"(ws), "v"(xs));
}

static_assert(4 * F8_STAGE <= 131072, "the stages lie where the operands were");
constexpr int F8_BIG_LDS = 131072 + 2 * 2048;      // two steps of x and w, two sets of exponents (1 KiB of x, 256 bytes for each wave of w)

template <int OUT, bool GROUPED>
__global__ __launch_bounds__(256, 1) void linear_f8_big_kernel(const F8Args a, int tiles_m, int tiles_n, int samples) {
  constexpr int W0 = 65536, E0 = 131072;             // x at 0 and 32768, w at W0 and W0 + 32768, exponents at E0 and E0 + 2048
  extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r16 = lane & 15, h = lane >> 4;
  const int wm = wave >> 1, wn = wave & 1;
  F8Tile t;
  int n0;
  if (!f8_locate<256, 256, GROUPED>(a, tiles_m, tiles_n, samples, t, n0)) return;
  const int64_t pitch = (int64_t)a.Kb * 128;
  const int base = f8_x_base<GROUPED>(a, t);
  const uint8_t* xg = a.x + (int64_t)t.sample * a.x_ss + base * pitch;
  const uint8_t* wg = a.w + (int64_t)t.set * a.w_ss + n0 * pitch;
  uint32_t xo[8], wo[8];
#pragma unroll
  for (int p = 0; p < 8; ++p) {
    const int r = (p * 4 + wave) * 8 + (lane >> 3), i = min(t.m0 + r, t.m1 - 1), piece = ((lane & 7) ^ ((r >> 1) & 7)) << 4;
    xo[p] = (uint32_t)((f8_x_row<GROUPED>(a, i) - base) * pitch) + piece;
    wo[p] = (uint32_t)(min(r, a.N - 1 - n0) * pitch) + piece;
  }
  const uint8_t* xeg = a.xe + (int64_t)t.sample * a.xe_ss + (int64_t)base * a.Sp;
  const uint8_t* weg = a.we + (int64_t)t.set * a.we_ss + (int64_t)min((n0 >> 7) + wn, (a.N - 1) >> 7) * a.Sp;
  const uint32_t xeo = (uint32_t)(f8_x_row<GROUPED>(a, min(t.m0 + (int)threadIdx.x, t.m1 - 1)) - base) * (uint32_t)a.Sp;      // of row threadIdx.x
  const uint32_t lds0 = lds_addr_of(lds) + wave * 1024, ldse = lds_addr_of(lds) + E0 + wave * 256;
  const int last = a.Kb - 1;
  // requests past the last step repeat its bytes, into buffers that are not read again (no branch in the loop)
  auto request = [&](int kb, int buf, int p) {       // 16 of a step
    const int at = min(kb, last) * 128;
    if (p < 8) f8_dma16(xg + at, xo[p], lds0 + buf * 32768 + p * 4096);
    else f8_dma16(wg + at, wo[p - 8], lds0 + W0 + buf * 32768 + (p - 8) * 4096);
  };
  auto request_exponents = [&](int kb, int set) {    // of step kb (a multiple of 2) and the next
    const int at = min(kb, last) & ~3;
    f8_dma4(xeg + at, xeo, ldse + set * 2048);
    f8_dma4(weg + at, 0, ldse + set * 2048 + 1024);
  };

  const int fl = r16 * 128 + ((h ^ ((r16 >> 1) & 7)) << 4);
  const uint8_t *xl = lds + wm * 16384 + fl, *xh = lds + wm * 16384 + (fl ^ 64), *wl = lds + W0 + wn * 16384 + fl, *wh = lds + W0 + wn * 16384 + (fl ^ 64);
  auto half = [](f8_v8i& o, int s, const uint8_t* p) {      // a fragment: pieces h and 4 + h of its rows
    const f8_v4i v = *(const f8_v4i*)p;
#pragma unroll
    for (int c = 0; c < 4; ++c) o[4 * s + c] = v[c];
  };
  f8_v8i wf[8], xf[8];
  auto read_x = [&](int buf, int f, int s) { half(xf[f], s, (s ? xh : xl) + buf * 32768 + f * 2048); };
  auto read_w = [&](int buf, int f, int s) { half(wf[f], s, (s ? wh : wl) + buf * 32768 + f * 2048); };
  uint32_t xs[8], ws;
  const uint8_t *xel = lds + E0 + (wm * 128 + r16) * 4, *wel = lds + E0 + 1024 + wave * 256 + lane * 4;
  auto read_exponents = [&](int set, int by) {
#pragma unroll
    for (int i = 0; i < 8; ++i) xs[i] = *(const uint32_t*)(xel + set * 2048 + i * 64) >> by;
    ws = *(const uint32_t*)(wel + set * 2048) >> by;
  };
  f8_v4f acc[8][8];
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[i][j] = (f8_v4f){0.f, 0.f, 0.f, 0.f};

  F8Moves<4> moves;
  if constexpr (f8_moves<OUT, GROUPED>()) moves.rows(a, t, t.m0 + wm * 128);
  request_exponents(0, 0);
#pragma unroll
  for (int p = 0; p < 16; ++p) request(0, 0, p);
#pragma unroll
  for (int p = 0; p < 16; ++p) request(1, 1, p);
  if constexpr (f8_moves<OUT, GROUPED>()) moves.weights(a);
  wait_vmcnt<16>();
  lds_barrier();
#pragma unroll
  for (int f = 0; f < 8; ++f) { read_w(0, f, 0); read_w(0, f, 1); }
#pragma unroll
  for (int f = 0; f < 4; ++f) { read_x(0, f, 0); read_x(0, f, 1); }
  read_exponents(0, 0);
  // even and odd steps differ in the buffer and in the byte of xs / ws; the even one requests the next two steps' exponents, into set `set`
  auto step = [&](auto Bc, int kb, int set) {
    constexpr int B = decltype(Bc)::value;
    auto mfma = [&](int i, int j) { f8_mfma_in_place<B>(acc[i][j], wf[j], xf[i], ws, xs[i]); };
    asm volatile("s_nop 3" : "+v"(ws), "+v"(xs[0]), "+a"(acc[0][0]));      // behind the vector unit's last writes of what the first instructions read
#pragma unroll
    for (int u = 0; u < 32; ++u) {
      if (u == 12) lds_barrier();            // the reads above are back
      mfma(u >> 3, u & 7);
      if (u < 8) read_x(B, 4 + (u >> 1), u & 1);
      if (u >= 12 && u % 2 == 1) request(kb + 2, B, (u - 13) / 2);
      if (u == 31 && B == 0) request_exponents(kb + 2, set);
      __builtin_amdgcn_sched_barrier(0);
    }
    wait_vmcnt<B == 0 ? 12 : 10>();          // the next step's operands have landed (what this half requested may be in flight)
    lds_barrier();
#pragma unroll
    for (int u = 0; u < 32; ++u) {
      const int g = u >> 2;
      mfma(4 + (u & 3), g);
      if (u < 12 && u % 2 == 0) request(kb + 2, B, 10 + u / 2);
      else if (u < 12 && u % 2 == 1) read_x(B ^ 1, (u / 2) >> 1, (u / 2) & 1);
      if (u == 12 || u == 13) read_x(B ^ 1, 3, u & 1);
      if ((u & 1) == 0 && u >= 4) { read_w(B ^ 1, (u - 4) >> 2, 0); }
      if ((u & 1) == 1 && u >= 4) { read_w(B ^ 1, (u - 4) >> 2, 1); }
      __builtin_amdgcn_sched_barrier(0);
    }
    read_w(B ^ 1, 7, 0);
    read_w(B ^ 1, 7, 1);
  };
  int kb = 0;
  for (; kb < last; kb += 2) {
    const int set = (~kb >> 1) & 1;
    step(std::integral_constant<int, 0>{}, kb, set);
    step(std::integral_constant<int, 1>{}, kb + 1, set);
    read_exponents(set, ((kb + 2) & 2) * 8);
  }
  if (kb == last) step(std::integral_constant<int, 0>{}, kb, (~kb >> 1) & 1);
  wait_vmcnt<0>();          // (no request outlives the workgroup's LDS)
  lds_barrier();            // ... and no wave reads another's operands any more
  asm volatile("s_nop 15\n\ts_nop 15");      // the last products are in their registers
  __builtin_amdgcn_sched_barrier(0);
  // lane: activation row r16 of fragment i, weight rows 4 h .. + 3 of fragment j
  f8_finish<4, OUT, GROUPED>(a, t, t.m0 + wm * 128, n0 + wn * 128, lds + wave * F8_STAGE, moves, [&](int g, float* st) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) *(f8_v4f*)(st + (i * 16 + r16) * F8_PITCH + j * 16 + h * 4) = acc[2 * g + i][j];
  });
}

template <int OUT, bool GROUPED> int launch_big(const F8Args& a, int rows, int z, hipStream_t st) {
  static std::atomic<uint64_t> attr{0};
  if (int rc = qbnn_ensure_dyn_lds((const void*)linear_f8_big_kernel<OUT, GROUPED>, &attr, F8_BIG_LDS)) return rc;
  const int64_t tm = ((int64_t)rows + 255) / 256 + (GROUPED ? std::min(a.groups, rows) : 0), tn = (a.N + 255) / 256;
  hipLaunchKernelGGL((linear_f8_big_kernel<OUT, GROUPED>), dim3((unsigned)(tm * tn * z)), dim3(256), F8_BIG_LDS, st, a, (int)tm, (int)tn, z);
  return qbnn_check_launch_msg("qbnn_linear_f8");
}

// Whether the products go through LDS tiles.  rows: the rows of one sample, or all routed rows.  Offsets are 32 bits wide there: of a gathered row's bytes from the
// first, of a row's in its tile.
template <bool GROUPED> int f8_rows_each(const F8Args& a, int rows) { return GROUPED ? (int)(((int64_t)rows + a.groups - 1) / a.groups) : rows; }
template <bool GROUPED> bool f8_tiled(const F8Args& a, int rows) {
  const int64_t far = GROUPED && a.rows ? (int64_t)a.x_rows * a.Kb * 128 : 0;
  return f8_rows_each<GROUPED>(a, rows) > 32 && far < ((int64_t)1 << 32) && a.Kb < (1 << 16);
}
// The form of a call: rows x weight rows of a tile, the direct form up to 32 rows and through LDS from 64 on.
struct F8Form { int tm, tn; };
template <bool GROUPED> F8Form f8_form(const F8Args& a, int rows, int z, int type, bool exact) {
  const int spare = GROUPED ? std::min(a.groups, rows) : 0;      // each group with rows may end inside a tile
  const int per = f8_rows_each<GROUPED>(a, rows);
  const auto tiles = [&](int tm, int tn) { return (__int128)z * (((int64_t)rows + tm - 1) / tm + spare / 2) * (((int64_t)a.N + tn - 1) / tn); };
  // The largest tile that still gives the 256 CUs work: fewer bytes through LDS per product, but 256 x 256 holds a CU for itself.  Measured the other way round (us):
  // 128 x 128 for 64 x 128 with 330 - 600 tiles 69 -> 58 (5 x 12 groups of 75, fp16) and 28.6 -> 23.8 (100 x 128 x 500 x 800, fp32), with 32 - 64 tiles 22.6 -> 25.7.
  if (f8_tiled<GROUPED>(a, rows)) {
    if (!exact && per > 128 && tiles(256, 256) >= 192) return {256, 256};
    if (per > 64 && tiles(128, 256) >= 384) return {128, 256};
    if (tiles(128, 128) >= 256) return {128, 128};
    return {64, 128};
  }
  const int tm = per <= 16 ? 16 : 32;
  if (type == QBNN_F8) return {tm, 128};
  return {tm, GROUPED || tm == 32 ? 64 : 16};
}
// Whether the form's workgroups fit a grid (2^32 threads along x, 2^31 pairs of row tile and sample in the direct form): asked before a call's first launch
template <bool GROUPED> int f8_fits(const F8Args& a, int rows, int z, int type, bool exact) {
  const F8Form f = f8_form<GROUPED>(a, rows, z, type, exact);
  const int64_t tm = ((int64_t)rows + f.tm - 1) / f.tm + (GROUPED ? std::min(a.groups, rows) : 0), tn = ((int64_t)a.N + f.tn - 1) / f.tn;
  const __int128 along = f.tm <= 32 ? (__int128)tn * 512 : (__int128)tm * tn * z * 256;
  if (along >= ((int64_t)1 << 32) || tm * z >= ((int64_t)1 << 31) - F8_FOLD) return f8_fail("qbnn_linear_f8: %ld tiles x %ld samples do not fit a grid", (long)(tm * tn), z);
  return QBNN_OK;
}
template <int OUT, bool EXACT, bool GROUPED> int launch_linear(const F8Args& a, int rows, int z, hipStream_t st) {
  const F8Form f = f8_form<GROUPED>(a, rows, z, OUT, EXACT);
  if constexpr (!EXACT) {
    if (f.tm == 256) return launch_big<OUT, GROUPED>(a, rows, z, st);
  }
  if (f.tm == 128 && f.tn == 256) return launch_tiled<2, 2, 2, OUT, EXACT, GROUPED>(a, rows, z, st);
  if (f.tm == 128) return launch_tiled<1, 4, 1, OUT, EXACT, GROUPED>(a, rows, z, st);
  if (f.tm == 64) return launch_tiled<1, 2, 1, OUT, EXACT, GROUPED>(a, rows, z, st);
  const int64_t tiles = ((int64_t)rows + f.tm - 1) / f.tm + (GROUPED ? std::min(a.groups, rows) : 0);
  // Tiles of 16 rows are exact whatever the result: they wait for memory, and the widening is done beside it (us, cut -> exact: 1 x 1024 x 1024 4.7 -> 5.0, 4 x 8192 x 8192
  // 18.2 -> 18.9, with an e4m3 result 55.8 -> 40.3, 61 rows through 6 of 64 experts 60.8 -> 58.8).  With 32 rows the vector unit is in the way: 32 x 8192 x 8192 34.2 -> 40.5.
  if constexpr (OUT == F8_HALF) return f8_fail("qbnn_experts_f8: no direct form of this result");
  else if constexpr (OUT == QBNN_F8) {
    if (f.tm == 16) return launch_direct<1, 8, 4, 2, OUT, true, GROUPED>(a, tiles, z, st);
    return launch_direct<2, 8, 4, 1, OUT, EXACT, GROUPED>(a, tiles, z, st);
  } else {
    if (f.tm == 16) {
      if constexpr (GROUPED) return launch_direct<1, 4, 4, 2, OUT, true, GROUPED>(a, tiles, z, st);
      else return launch_direct<1, 1, 8, 4, OUT, true, GROUPED>(a, tiles, z, st);
    }
    return launch_direct<2, 4, 4, 2, OUT, EXACT, GROUPED>(a, tiles, z, st);
  }
}
// what the two entries ask for: every type for dense rows (fp32 exact), e4m3 and fp32 of either form and halves for groups
template <bool GROUPED> int launch_linear_any(const F8Args& a, int rows, int z, int y_type, int exact, hipStream_t st) {
  switch (y_type) {
    case QBNN_F32: if constexpr (!GROUPED) return launch_linear<QBNN_F32, true, GROUPED>(a, rows, z, st);
      else return exact ? launch_linear<QBNN_F32, true, GROUPED>(a, rows, z, st) : launch_linear<QBNN_F32, false, GROUPED>(a, rows, z, st);
    case QBNN_BF16: if constexpr (!GROUPED) return launch_linear<QBNN_BF16, false, GROUPED>(a, rows, z, st);
    case QBNN_F16: if constexpr (!GROUPED) return launch_linear<QBNN_F16, false, GROUPED>(a, rows, z, st);
    case F8_HALF: if constexpr (GROUPED) return launch_linear<F8_HALF, false, GROUPED>(a, rows, z, st);
    default:
      if constexpr (GROUPED) { if (exact) return launch_linear<QBNN_F8, true, GROUPED>(a, rows, z, st); }
      return launch_linear<QBNN_F8, false, GROUPED>(a, rows, z, st);
  }
}

// ---- y[t] = sum over the row's top_k results, in the order of choice --------------------------------------------------------------
// The results come in fp32: rounded to the 16 bits of y first, each would cost as much as the one rounding of the sum does.  For a bf16 y, halves with block exponents
// cost 2^-11 of each term beside the sum's 2^-8 and are half of the bytes, which bound this kernel (32768 x 4096: 115 us from fp32, 55 from halves, 6.1 TB/s).
constexpr int COMBINE_COLUMNS = 8;
template <int T, bool HALF> __global__ __launch_bounds__(256) void combine_kernel(const uint8_t* __restrict__ o, const uint8_t* __restrict__ oe, f8_type<T>* __restrict__ y, int rows, int k, int N) {
  const int n0 = (blockIdx.x * 256 + threadIdx.x) * COMBINE_COLUMNS;
  const int64_t t = blockIdx.y + (int64_t)blockIdx.z * 32768;
  if (n0 >= N || t >= rows) return;
  const int Nb = (N + 127) >> 7;
  float sum[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  const bool whole = n0 + 8 <= N;
#pragma unroll 4
  for (int j = 0; j < k; ++j) {
    const int64_t r = t * k + j;
    if constexpr (HALF) {                                       // (rows are padded to whole blocks)
      const f8_v4i p = *(const f8_v4i*)(o + (r * (Nb * 128) + n0) * 2);
      const float up = f8_pow2((int)oe[r * Nb + (n0 >> 7)] - 127);
      _Float16 h[8];
      __builtin_memcpy(h, &p, sizeof(h));
#pragma unroll
      for (int i = 0; i < 8; ++i) sum[i] += (float)h[i] * up;
    } else {
      const float* p = (const float*)o + r * N + n0;
      float v[8];
      if (whole) __builtin_memcpy(v, p, sizeof(v));
      else
        for (int i = 0; i < 8; ++i) v[i] = n0 + i < N ? p[i] : 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) sum[i] += v[i];
    }
  }
  f8_type<T> v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = f8_store<T>(sum[i]);
  f8_type<T>* out = y + t * N + n0;
  if (whole) __builtin_memcpy(out, v, sizeof(v));
  else
    for (int i = 0; i < 8; ++i) if (n0 + i < N) out[i] = v[i];
}

int launch_combine(const void* o, const uint8_t* oe, int rows, int k, int N, void* y, int y_type, hipStream_t st) {
  const dim3 grid((unsigned)((N + 256 * COMBINE_COLUMNS - 1) / (256 * COMBINE_COLUMNS)), (unsigned)(rows < 32768 ? rows : 32768), (unsigned)((rows + 32767) / 32768));
  const uint8_t* in = (const uint8_t*)o;
  if (oe) hipLaunchKernelGGL((combine_kernel<QBNN_BF16, true>), grid, dim3(256), 0, st, in, oe, (uint16_t*)y, rows, k, N);
  else if (y_type == QBNN_F32) hipLaunchKernelGGL((combine_kernel<QBNN_F32, false>), grid, dim3(256), 0, st, in, oe, (float*)y, rows, k, N);
  else if (y_type == QBNN_BF16) hipLaunchKernelGGL((combine_kernel<QBNN_BF16, false>), grid, dim3(256), 0, st, in, oe, (uint16_t*)y, rows, k, N);
  else hipLaunchKernelGGL((combine_kernel<QBNN_F16, false>), grid, dim3(256), 0, st, in, oe, (_Float16*)y, rows, k, N);
  return qbnn_check_launch_msg("qbnn_experts_f8 (sum)");
}

int quantize(const void* x, int x_type, int64_t bs, int64_t rs, int64_t batch, int R, int K, int block_rows, uint8_t* q, uint8_t* e, hipStream_t st) {
  QuantF8Args a = {};
  a.x = x; a.x_bs = bs; a.x_rs = rs; a.q = q; a.e = e;
  a.R = R; a.K = K; a.Kb = (K + 127) / 128; a.Sp = (a.Kb + 3) / 4 * 4;
  a.blocks = batch * (block_rows == 1 ? R : (R + 127) / 128) * a.Kb;
  switch (x_type) {
    case QBNN_F32: return launch_quantize<QBNN_F32>(a, batch, block_rows, st);
    case QBNN_BF16: return launch_quantize<QBNN_BF16>(a, batch, block_rows, st);
    default: return launch_quantize<QBNN_F16>(a, batch, block_rows, st);
  }
}
bool aligned(const void* p, int64_t stride, int to) { return !(((uintptr_t)p | (uintptr_t)stride) & (to - 1)); }
bool float_type(int t) { return t >= QBNN_F32 && t <= QBNN_F16; }
void set_columns(F8Args& a, int K) {
  a.Kb = (int)(((int64_t)K + 127) / 128);
  a.Sp = (a.Kb + 3) / 4 * 4;
}
void set_result(F8Args& a, void* y, uint8_t* ye, int M, int N, int type) {
  const int Nb = (int)(((int64_t)N + 127) / 128);
  a.y = (uint8_t*)y; a.ye = ye; a.M = M; a.N = N;
  a.y_rs = type == QBNN_F8 ? Nb * 128 : N;
  a.ye_rs = (Nb + 3) / 4 * 4;
  a.y_ss = (int64_t)M * a.y_rs;
}

}  // namespace

QBNN_EXPORT int qbnn_quantize_f8(const void* x, int32_t x_type, int64_t x_batch_stride, int64_t x_row_stride, int64_t batch, int32_t R, int32_t K,
                                 int32_t block_rows, uint8_t* q, uint8_t* exponents, void* stream) {
  if (!float_type(x_type) || batch < 0 || R < 0 || K <= 0 || (block_rows != 1 && block_rows != 128)) return f8_fail("qbnn_quantize_f8: bad argument");
  if (batch == 0 || R == 0) return QBNN_OK;
  if (!x || !q || !exponents || !aligned(q, 0, 16) || K > 0x7fffff00) return f8_fail("qbnn_quantize_f8: bad argument (q starts at a multiple of 16 bytes)");
  return quantize(x, x_type, x_batch_stride, x_row_stride, batch, R, K, block_rows, q, exponents, (hipStream_t)stream);
}

namespace {
// A call's arguments checked and laid out; whether its launches fit is known before the first
int linear_args(const qbnn_f8_linear* d, F8Args& a) {
  if (!d || d->N <= 0 || d->K <= 0 || d->K > 0x7fffff00 || d->N > 0x7fffff00 || d->M < 0 || d->n_samples < 0 || d->y_type < QBNN_F32 || d->y_type > QBNN_F8 ||
      (d->x_float && !float_type(d->x_type)))
    return f8_fail("qbnn_linear_f8_mc: bad argument");
  a = {};
  if (d->M == 0 || d->n_samples == 0) return QBNN_OK;
  if (!d->x || !d->x_exp || !d->w || !d->w_exp || !d->y || (d->y_type == QBNN_F8 && !d->y_exp)) return f8_fail("qbnn_linear_f8_mc: bad argument");
  if (!aligned(d->x, d->x_ss, 16) || !aligned(d->w, d->w_ss, 16) || !aligned(d->x_exp, d->x_exp_ss, 4) || !aligned(d->w_exp, d->w_exp_ss, 4) ||
      (d->y_type == QBNN_F8 && !aligned(d->y, 0, 16)))
    return f8_fail("qbnn_linear_f8_mc: e4m3 operands start at multiples of 16 bytes, exponents of 4");
  set_columns(a, d->K);
  a.x = d->x; a.xe = d->x_exp; a.x_ss = d->x_ss; a.xe_ss = d->x_exp_ss;
  a.w = d->w; a.we = d->w_exp; a.w_ss = d->w_ss; a.we_ss = d->w_exp_ss;
  a.bias = d->bias; a.bias_ss = d->bias_ss; a.relu = d->relu;
  set_result(a, d->y, d->y_exp, d->M, d->N, d->y_type);
  return f8_fits<false>(a, a.M, d->n_samples, d->y_type, d->y_type == QBNN_F32);
}
// half: the second product's results wait for their sum as halves.  They do where the result is bf16, behind tiles, and take R Nb 257 bytes of the R N 4.
int experts_args(const qbnn_f8_experts* d, F8Args& up, F8Args& down, int& rows, bool& half) {
  rows = 0;
  if (!d || d->S < 0 || d->T < 0 || d->E <= 0 || d->top_k <= 0 || d->D <= 0 || d->H <= 0 || d->N <= 0 || d->D > 0x7fffff00 || d->H > 0x7fffff00 || d->N > 0x7fffff00 ||
      !float_type(d->y_type) || (d->x_float && !float_type(d->x_type)) || (d->up_sets != d->E && d->up_sets != d->S * d->E) ||
      (d->down_sets != d->E && d->down_sets != d->S * d->E) || (int64_t)d->S * d->T * d->top_k > 0x7fffffff || (int64_t)d->S * d->E > 0x7fffffff)
    return f8_fail("qbnn_experts_f8: bad argument");
  const int n = d->S * d->T * d->top_k;
  if (n == 0) return QBNN_OK;
  if (!d->x || !d->x_exp || !d->offsets || !d->rows || !d->weights || !d->w_up || !d->up_exp || !d->w_down || !d->down_exp || !d->h || !d->h_exp || !d->o || !d->y ||
      (d->x_rows != d->T && d->x_rows != d->S * d->T))
    return f8_fail("qbnn_experts_f8: bad argument");
  if (!aligned(d->x, 0, 16) || !aligned(d->w_up, d->up_ss, 16) || !aligned(d->w_down, d->down_ss, 16) || !aligned(d->h, 0, 16) || !aligned(d->x_exp, 0, 4) ||
      !aligned(d->up_exp, d->up_exp_ss, 4) || !aligned(d->down_exp, d->down_exp_ss, 4) || !aligned(d->h_exp, 0, 4) || !aligned(d->o, 0, 16))
    return f8_fail("qbnn_experts_f8: e4m3 operands start at multiples of 16 bytes, exponents of 4");
  up = {};
  up.offsets = d->offsets; up.groups = d->S * d->E;
  down = up;
  set_columns(up, d->D);
  up.x = d->x; up.xe = d->x_exp; up.rows = d->rows; up.topk = d->top_k; up.x_rows = d->x_rows;
  up.w = d->w_up; up.we = d->up_exp; up.w_ss = d->up_ss; up.we_ss = d->up_exp_ss; up.w_groups = d->up_sets;
  up.bias = d->b_up; up.bias_ss = d->b_up_ss; up.relu = 1;
  set_result(up, d->h, d->h_exp, n, d->H, QBNN_F8);
  set_columns(down, d->H);
  down.x = d->h; down.xe = d->h_exp;
  down.w = d->w_down; down.we = d->down_exp; down.w_ss = d->down_ss; down.we_ss = d->down_exp_ss; down.w_groups = d->down_sets;
  down.bias = d->b_down; down.bias_ss = d->b_down_ss;
  down.y_rows = d->rows; down.scale = d->weights;
  set_result(down, d->o, nullptr, n, d->N, QBNN_F32);
  half = d->y_type == QBNN_BF16 && !(d->exact & 2) && d->N >= 128 && f8_tiled<true>(down, n);
  if (half) {
    const int Nb = (d->N + 127) / 128;
    down.y_rs = Nb * 128; down.ye_rs = Nb;
    down.ye = (uint8_t*)d->o + (int64_t)n * down.y_rs * 2;
  }
  if (int rc = f8_fits<true>(up, n, 1, QBNN_F8, d->exact & 1)) return rc;
  if (int rc = f8_fits<true>(down, n, 1, half ? F8_HALF : QBNN_F32, d->exact >> 1 & 1)) return rc;
  rows = n;
  return QBNN_OK;
}
int32_t tile_of(F8Form f) { return f.tm << 16 | f.tn; }
}  // namespace

QBNN_EXPORT int qbnn_linear_f8_mc(const qbnn_f8_linear* d, void* stream) {
  F8Args a;
  if (int rc = linear_args(d, a)) return rc;
  if (a.M == 0) return QBNN_OK;
  if (d->x_float)
    if (int rc = quantize(d->x_float, d->x_type, d->x_float_ss, d->x_float_rs, d->x_ss ? d->n_samples : 1, d->M, d->K, 1, d->x, d->x_exp, (hipStream_t)stream)) return rc;
  return launch_linear_any<false>(a, a.M, d->n_samples, d->y_type, 0, (hipStream_t)stream);
}

QBNN_EXPORT int32_t qbnn_linear_f8_tile(const qbnn_f8_linear* d) {
  F8Args a;
  if (int rc = linear_args(d, a)) return rc;
  return a.M == 0 ? 0 : tile_of(f8_form<false>(a, a.M, d->n_samples, d->y_type, d->y_type == QBNN_F32));
}

QBNN_EXPORT int qbnn_experts_f8(const qbnn_f8_experts* d, void* stream) {
  F8Args up, down;
  int rows;
  bool half;
  if (int rc = experts_args(d, up, down, rows, half)) return rc;
  if (rows == 0) return QBNN_OK;
  hipStream_t st = (hipStream_t)stream;
  if (d->x_float)
    if (int rc = quantize(d->x_float, d->x_type, d->x_float_ss, d->x_float_rs, d->x_rows / d->T, d->T, d->D, 1, d->x, d->x_exp, st)) return rc;
  if (int rc = launch_linear_any<true>(up, rows, 1, QBNN_F8, d->exact & 1, st)) return rc;
  if (int rc = launch_linear_any<true>(down, rows, 1, half ? F8_HALF : QBNN_F32, d->exact >> 1 & 1, st)) return rc;
  return launch_combine(d->o, half ? down.ye : nullptr, d->S * d->T, d->top_k, d->N, d->y, d->y_type, st);
}

QBNN_EXPORT int qbnn_experts_f8_tiles(const qbnn_f8_experts* d, int32_t* tiles) {
  F8Args up, down;
  int rows;
  bool half;
  if (int rc = experts_args(d, up, down, rows, half)) return rc;
  if (!tiles) return f8_fail("qbnn_experts_f8_tiles: bad argument");
  tiles[0] = rows ? tile_of(f8_form<true>(up, rows, 1, QBNN_F8, d->exact & 1)) : 0;
  tiles[1] = rows ? tile_of(f8_form<true>(down, rows, 1, half ? F8_HALF : QBNN_F32, d->exact >> 1 & 1)) : 0;
  return QBNN_OK;
}
