// Device code shared by the 8-bit floating-point kernels (qbnn_f8.hip, qbnn_route.hip): the block format's conversions and the
// block-scaled matrix instruction.
//
// Format: e4m3 values [rows][Kp] (Kp = K up to a multiple of 128, zeros behind the last column) and one biased exponent byte per block
// (127 = 2^0) [row blocks][Sp] (Sp = blocks of 128 columns up to a multiple of 4: a lane fetches the scales of four blocks as one dword).
// The scale of a block is the smallest power of two, at least 2^-126, that brings its largest finite magnitude to 448 or below; 1 for a
// block of zeros.  A power of two because v_mfma_scale_f32_16x16x128_f8f6f4 applies one per operand row and 32 columns at no cost, because
// v * 2^-e is exact (one rounding in all, no division: the bits are defined), and because a float's relative step does not depend on it.
#ifndef QBNN_F8_H_
#define QBNN_F8_H_
#include <hip/hip_runtime.h>
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <stdint.h>

#include "../../include/qbnn.h"
#include "qbnn_common.h"

namespace qbnn {

typedef int f8_v8i __attribute__((ext_vector_type(8)));
typedef int f8_v4i __attribute__((ext_vector_type(4)));
typedef int f8_v2i __attribute__((ext_vector_type(2)));
typedef float f8_v4f __attribute__((ext_vector_type(4)));

// ---- floating types at the interface (QBNN_F32 / QBNN_BF16 / QBNN_F16) --------------------------------------------------------
template <int T> struct F8Type;
template <> struct F8Type<QBNN_F32> { typedef float type; };
template <> struct F8Type<QBNN_BF16> { typedef uint16_t type; };
template <> struct F8Type<QBNN_F16> { typedef _Float16 type; };
template <int T> using f8_type = typename F8Type<T>::type;

template <int T> __device__ __forceinline__ float f8_load(f8_type<T> v) {
  if constexpr (T == QBNN_BF16) return __uint_as_float((uint32_t)v << 16);
  else return (float)v;
}
// round to nearest, ties to even (the one rounding of a 16-bit result)
template <int T> __device__ __forceinline__ f8_type<T> f8_store(float v) {
  if constexpr (T == QBNN_BF16) {
    const __bf16 b = (__bf16)v;
    return __builtin_bit_cast(uint16_t, b);
  } else return (f8_type<T>)v;
}

template <int T> __device__ __forceinline__ int f8_store2(float a, float b) {      // two 16-bit results in a dword
  if constexpr (T == QBNN_BF16) {
    typedef __bf16 v2 __attribute__((ext_vector_type(2)));
    typedef float f2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(int, __builtin_convertvector((f2){a, b}, v2));
  } else {
    typedef _Float16 v2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(int, (v2){(_Float16)a, (_Float16)b});
  }
}

// ---- block scale ---------------------------------------------------------------------------------------------------------------
// bits of the largest finite magnitude -> unbiased exponent: the smallest e >= -126 with a <= 448 2^e = 1.75 2^(e + 8); 0 for a = 0
__device__ __forceinline__ int f8_exponent(uint32_t bits) {
  const int e = (int)(bits >> 23) - 135 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  return bits == 0 ? 0 : (e < -126 ? -126 : e);
}
__device__ __forceinline__ float f8_pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }      // -126 <= e <= 127
// |v| as bits where it is finite, 0 where it is not: unsigned maximum = largest finite magnitude
__device__ __forceinline__ uint32_t f8_magnitude(float v) {
  const uint32_t b = __float_as_uint(v) & 0x7fffffffu;
  return b < 0x7f800000u ? b : 0u;
}
// four values already scaled to [-448, 448] -> four e4m3 bytes; the conversion makes a NaN of what is not finite
__device__ __forceinline__ uint32_t f8_pack4(float a, float b, float c, float d) {
  const int r = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, r, true);
}

// ---- matrix instruction --------------------------------------------------------------------------------------------------------
// D[16 weight rows][16 activation rows] += (128 columns of both) with one power of two per operand row; lane l supplies row l & 15 of
// both operands, 32 of the 128 columns -- any 32, as long as the four lane groups of both operands agree on them, since all 128 columns of a
// row share its scale (a byte of ws / xs).  D: lane l holds weight rows 4 (l >> 4) .. + 3 of activation row l & 15.
//
// f8_mfma: the e4m3 instruction.  It adds the products of 8 neighbouring bytes after aligning them to the largest, what lies 2^-13 below it cut
// off, and keeps fp32 from there on (probed): 1.3e-5 of the result's norm on normal data, an eightieth of half a step of fp16 and a
// hundred-and-fiftieth of bf16's -- the form for results of 16 and 8 bits, from 17 rows on.
// f8_mfma_exact: the operands widened to bf16 times their block's scale (both exact down to exponents of -117; below, bf16 ends at 2^-133) and multiplied by the bf16 instruction, whose sums are fp32
// throughout: half the matrix rate, the widening beside it on the vector unit; the form for fp32 results, and for few rows, which wait
// for memory either way.
template <int BYTE> __device__ __forceinline__ f8_v4f f8_mfma(f8_v8i w, f8_v8i x, f8_v4f acc, uint32_t ws, uint32_t xs) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, x, acc, 0, 0, BYTE, (int)ws, BYTE, (int)xs);
}
typedef __bf16 f8_v8b __attribute__((ext_vector_type(8)));
typedef __bf16 f8_v2b __attribute__((ext_vector_type(2)));
struct F8Wide { f8_v8b part[4]; };
// exponent: biased, in the lowest byte
__device__ __forceinline__ F8Wide f8_widen(f8_v8i v, uint32_t exponent) {
  const float s = __uint_as_float((exponent & 255) << 23);
  F8Wide o;
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    const f8_v2b a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(v[2 * g], s, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(v[2 * g], s, true);
    const f8_v2b c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(v[2 * g + 1], s, false), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(v[2 * g + 1], s, true);
    o.part[g] = (f8_v8b){a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
  }
  return o;
}
__device__ __forceinline__ f8_v4f f8_mfma_exact(const F8Wide& w, const F8Wide& x, f8_v4f acc) {
#pragma unroll
  for (int g = 0; g < 4; ++g) acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w.part[g], x.part[g], acc, 0, 0, 0);
  return acc;
}

// 16 bytes per lane from a uniform address + a 32-bit offset per lane to LDS at lds_addr + 16 * lane; counted by the caller (wait_vmcnt).  m0 is given up, not kept
// as dma16_s does: two scalar instructions fewer in a gap of 32 cycles.
__device__ __forceinline__ void f8_dma16(const uint8_t* base, uint32_t lane_off, uint32_t lds_addr) {
  const uint64_t g = (uint64_t)base;
  const uint64_t gs = ((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(g >> 32)) << 32) | (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)g);
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" : : "v"(lane_off), "s"(gs), "s"(lds_addr) : "memory", "m0");
}

__device__ __forceinline__ void f8_dma4(const uint8_t* base, uint32_t lane_off, uint32_t lds_addr) {      // 4 bytes per lane
  const uint64_t g = (uint64_t)base;
  const uint64_t gs = ((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(g >> 32)) << 32) | (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)g);
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dword %0, %1" : : "v"(lane_off), "s"(gs), "s"(lds_addr) : "memory", "m0");
}

__device__ __forceinline__ f8_v8i f8_join(f8_v4i lo, f8_v4i hi) { return (f8_v8i){lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w}; }

}  // namespace qbnn
#endif
