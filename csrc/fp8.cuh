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

// act(g) * u.  gelu's tanh form is g * sigmoid(2 z).  The sigmoid is the special-function unit's: 2^x within 2^-22, a reciprocal, and for negative z
// an argument whose rounding weighs as much as |z| is large.  With the products the result is off by up to (10 + 1.25 |z|) 2^-24 of itself (gelu's z
// comes out of five roundings: 10 + 6.25 |z|): 2^-19 at z = -20, 2^-17 at z = -80, where half a step of e4m3 is 2^-4; below z = -87 the
// sigmoid is 0.  With expf and a division rows of 13824 took a third longer.
// (Where `act` is not a constant both z are computed and one is taken, without a branch.)
__device__ __forceinline__ float fp8_gated(int act, float g, float u) {
  const float z = act == kFp8Silu ? g : 1.5957691216057308f * (g + 0.044715f * g * g * g);
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

// What a call reads or writes: rows of `bytes` bytes, ld bytes apart (p null: nothing).
struct Fp8Span {
  const void* p;
  long long bytes, ld, rows;
};
// Whether two share no byte: apart as a whole, or columns side by side of the same rows (a single row may be one of any distance).
inline bool spans_apart(const Fp8Span& a, const Fp8Span& b) {
  if (a.p == nullptr || b.p == nullptr) return true;
  const long long d = reinterpret_cast<const uint8_t*>(b.p) - reinterpret_cast<const uint8_t*>(a.p);
  if (d >= (a.rows - 1) * a.ld + a.bytes || -d >= (b.rows - 1) * b.ld + b.bytes) return true;
  const long long ld = a.rows == 1 ? b.ld : a.ld;
  if ((a.rows == 1 && b.rows == 1) || (a.rows > 1 && b.rows > 1 && a.ld != b.ld) || ld <= 0) return false;
  const long long column = (d % ld + ld) % ld;
  return column >= a.bytes && column + b.bytes <= ld;
}
// Whether what is written shares no byte with anything else of the call: CTAs work on rows in any order.
template <int W, int R>
bool written_apart(const Fp8Span (&written)[W], const Fp8Span (&read)[R]) {
  for (int i = 0; i < W; ++i) {
    for (int j = 0; j < i; ++j)
      if (!spans_apart(written[i], written[j])) return false;
    for (int j = 0; j < R; ++j)
      if (!spans_apart(written[i], read[j])) return false;
  }
  return true;
}

}  // namespace zse
