// Shared pieces of the e4m3 key / value cache: code conversions and the block scale.
//
// A block of tokens of one head stores codes x / s rounded to e4m3, with s the smallest power of two for which the
// block's largest magnitude is at most 448 s.  A power of two makes the division exact, so the only rounding is the
// one to e4m3, and raising the scale of a block that already holds codes moves them by an exact factor before they
// are rounded again.  Against a scale of amax / 448 it costs at most one binade of range and no precision above the
// subnormal codes (e4m3 keeps three mantissa bits at every scale).
#pragma once
#include "common.cuh"
#include <cuda_fp8.h>

namespace ob {
namespace kvfp8 {

// Exponents of a block scale.  Below: the smallest code times 2^-112 is 2^-121, a normal fp32 number, so flushing
// subnormal fp32 changes nothing.  Above: 448 * 2^119 is finite in fp32; larger values saturate.
constexpr int EXP_MIN = -112, EXP_MAX = 119;

__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

__device__ __forceinline__ float inverse_pow2(float s) { return __uint_as_float((254u << 23) - __float_as_uint(s)); }

__device__ __forceinline__ float needed_scale(float amax) {
  // ceil(log2(amax / 448)): 448 = 1.75 * 2^8, so the exponent goes up by one where the mantissa is above 1.75
  const int e = (int)((__float_as_uint(amax) + 0x1fffffu) >> 23) - 127 - 8;
  return pow2(amax > 0.f ? min(max(e, EXP_MIN), EXP_MAX) : EXP_MIN);
}

// two floats to two codes, nearest even; NaN stays NaN, finite values saturate at 448
__device__ __forceinline__ uint32_t to_codes(float a, float b) {
  return (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
}
// two codes (low 16 bits) to an f16 pair, exact
__device__ __forceinline__ uint32_t to_half2(uint32_t codes) {
  uint32_t r;
  asm("{\n\t.reg .b16 l;\n\tcvt.u16.u32 l, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\t}" : "=r"(r) : "r"(codes));
  return r;
}
__device__ __forceinline__ uint32_t to_half2_hi(uint32_t codes) {
  uint32_t r;
  asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, h;\n\t}" : "=r"(r) : "r"(codes));
  return r;
}
__device__ __forceinline__ float2 half2_to_float2(uint32_t h) {
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

// Launch of the append kernel (kv_fp8.cu), also used in front of the decode attention.
struct AppendParams {
  const void *k_new, *v_new;
  long long new_batch, new_tok, new_head;      // elements
  void *k, *v;
  long long batch, tok, head;                  // bytes
  float *k_scale, *v_scale;
  long long scale_batch, scale_head;           // elements
  const int *lens, *n_new;                     // n_new may be null
  int* status;
  int B, T, Hk, hd, capacity, block;
  // set by the launcher: blocks that a run of T tokens can touch, the launch's first sequence, log2 of block and of a
  // row's 8-element chunks
  int span, b0, block_shift, row_shift;
};
int launch_append(AppendParams p, int dtype, cudaStream_t stream);

}  // namespace kvfp8
}  // namespace ob
