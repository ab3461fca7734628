// Rows and weights in 8-bit floating point (e4m3) with scales: what the kernels that write them and the products share.
#pragma once
#include <cuda_fp8.h>

#include <algorithm>

#include "typed.cuh"

namespace zse {

constexpr int kFp8Block = 128;                  // columns of a scale, and rows of a weight's
constexpr float kFp8Top = 448.f;                // the largest e4m3
constexpr float kFp8Least = 1e-30f;             // a block whose largest number is not above it is written as zeros
constexpr int kFp8Most = 1 << 30;               // rows or columns of a call: their numbers, rounded up to a tile, stay ints

enum Fp8Type : int { kFp8F16 = 0, kFp8BF16 = 1, kFp8F32 = 2 };
enum Fp8Act : int { kFp8None = 0, kFp8Silu = 1, kFp8Gelu = 2 };

// The order of these is that of |x|, with infinity above every number and NaN above infinity.
__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// `top`: the largest |y| of a block (NaN where it has one)
__device__ __forceinline__ float fp8_steps(float top) { return top <= kFp8Least ? 0.f : __fdiv_rn(kFp8Top, top); }
__device__ __forceinline__ float fp8_scale(float top) { return top <= kFp8Least ? 0.f : __fdiv_rn(top, kFp8Top); }
// (steps * |y| <= 448 up to rounding, which e4m3 rounds back to 448)
__device__ __forceinline__ uint32_t fp8_pack4(const float* y, float steps) {
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(__fmul_rn(y[0], steps), __fmul_rn(y[1], steps)), __NV_SATFINITE, __NV_E4M3);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(__fmul_rn(y[2], steps), __fmul_rn(y[3], steps)), __NV_SATFINITE, __NV_E4M3);
  return lo | hi << 16;
}

// act(g) * u.  gelu's tanh form is g * sigmoid(2 z).  The special-function unit's sigmoid is off by a few units in the last place of fp32,
// 2^-17 of half a step of e4m3; with expf and a division rows of 13824 took a third longer.
template <int ACT>
__device__ __forceinline__ float fp8_gated(float g, float u) {
  const float z = ACT == kFp8Silu ? g : 1.5957691216057308f * (g + 0.044715f * g * g * g);
  return g * sigmoid_fast(z) * u;
}

// two numbers in 16 bits each; fp16 is held within its largest, and a NaN stays one
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack2<bf16>(float a, float b) { return pack_bf16(a, b); }
__device__ __forceinline__ float hold_f16(float x) {
  float r;
  asm("{\n\t.reg .f32 t;\n\tmax.NaN.f32 t, %1, 0fC77FE000;\n\tmin.NaN.f32 %0, t, 0f477FE000;\n\t}" : "=f"(r) : "f"(x));  // +-65504
  return r;
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float a, float b) { return pack_half2(hold_f16(a), hold_f16(b)); }

// Whether `rows` rows of `bytes` bytes, ld bytes apart, at p share none with those at q: apart as a whole, or columns of the same rows.
inline bool rows_apart(const void* p, long long bytes, long long ld, const void* q, long long q_bytes, long long q_ld, int rows) {
  const long long d = reinterpret_cast<const uint8_t*>(q) - reinterpret_cast<const uint8_t*>(p);
  if (d >= (rows - 1) * ld + bytes || -d >= (rows - 1) * q_ld + q_bytes) return true;
  if (rows == 1 || ld != q_ld || ld <= 0) return false;
  const long long column = (d % ld + ld) % ld;
  return column >= bytes && column + q_bytes <= ld;
}

}  // namespace zse
