// Rows in 8-bit floating point (e4m3) with one fp32 scale for each block of 128 columns: what the products of gemm_fp8.cu read.
//
// A block's scale is max|y| / 448 and its numbers are e4m3(y * (448 / max|y|)): three bits behind the leading one, so that a number
// is off by at most 2^-4 of itself, or by 2^-10 of the scale where it is smaller than 2^-6 scale.  The scale of a block that holds an infinity or a
// NaN is infinite or NaN, and so are its products.  Both kernels round once, from fp32: y is never a 16-bit number on the way.
#include <cuda_fp8.h>

#include "api.h"
#include "fp8.cuh"

namespace zse {

namespace {

// ---- residual += planes + 16-bit rows; out = RMSNorm(residual) * weight in 8 bits --------------------------------------------------
// A warp has blocks of 128 columns, four columns a lane, which stay in registers between the sum and the rounding: every number is read once
// and written once.  More than one addend is summed in 64 bits and the squares always are, a block's by itself and then the blocks' in an
// order of their own, so that the same row gives the same bytes however it is split over warps (8192 x 5120, one 16-bit addend: 98 us, and 95 with
// sums by warp, whose order goes by the launch).  Bound by memory where there are many rows: with the norm in 16 bits as well 105 us, 5.2 TB/s.
struct NormFp8 {
  float* residual;
  const float* planes;
  const void *add, *weight;
  void* normed;
  uint8_t* data;
  float* scale;
  long long ld_data, ld_scale;
  double eps;
  int n_planes, M, H;
};

template <typename T>
__device__ __forceinline__ float4 load4(const T* p);
template <>
__device__ __forceinline__ float4 load4<float>(const float* p) { return *reinterpret_cast<const float4*>(p); }
template <>
__device__ __forceinline__ float4 load4<__half>(const __half* p) {
  const uint2 v = *reinterpret_cast<const uint2*>(p);
  const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&v.x)), b = __half22float2(*reinterpret_cast<const __half2*>(&v.y));
  return make_float4(a.x, a.y, b.x, b.y);
}
template <>
__device__ __forceinline__ float4 load4<bf16>(const bf16* p) {
  const uint2 v = *reinterpret_cast<const uint2*>(p);
  return make_float4(__uint_as_float(v.x << 16), __uint_as_float(v.x & 0xffff0000u), __uint_as_float(v.y << 16), __uint_as_float(v.y & 0xffff0000u));
}

// s[j], j < J: a lane's part of the sum of block j of the warp's.  Returns the whole sum of block lane >> (5 - log2 J), J rounded up to a power of
// two: lanes whose numbers differ in one bit are added, from bit 4 down, the same way for every J.  Where a lane still has several blocks,
// it keeps half of them and sends the other half: 9 exchanges for eight blocks, not 40.
template <int J>
__device__ __forceinline__ double block_sums(const double (&s)[J], int lane) {
  constexpr int P = J == 1 ? 1 : J == 2 ? 2 : J <= 4 ? 4 : 8;
  double t[P];
#pragma unroll
  for (int j = 0; j < P; ++j) t[j] = j < J ? s[j < J ? j : 0] : 0.;
  int o = 16;
#pragma unroll
  for (int n = P / 2; n > 0; n /= 2, o /= 2) {
#pragma unroll
    for (int j = 0; j < n; ++j) {
      const bool upper = lane & o;
      t[j] = (upper ? t[j + n] : t[j]) + __shfl_xor_sync(0xffffffffu, upper ? t[j] : t[j + n], o);
    }
  }
#pragma unroll
  for (; o > 0; o /= 2) t[0] += __shfl_xor_sync(0xffffffffu, t[0], o);
  return t[0];
}

// SEVERAL: more than one addend.  (One, and 256 threads: as many rows on an SM as registers allow.)
template <typename T, int J, int THREADS, bool SEVERAL>
__global__ void __launch_bounds__(THREADS, THREADS > 256 || SEVERAL ? 1 : J <= 5 ? 6 : 4)
add_rmsnorm_fp8_kernel(const NormFp8 a) {
  __shared__ double red[256];                                  // a block's sum of squares
  pdl_launch_dependents();
  pdl_wait();
  const int warps = blockDim.x >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int row = blockIdx.x, H = a.H, blocks = (H + kFp8Block - 1) / kFp8Block;
  const size_t base = size_t(row) * H, plane = size_t(a.M) * H;
  float4 x[J];
#pragma unroll
  for (int j = 0; j < J; ++j) {
    const int c = (warp + j * warps) * kFp8Block + lane * 4;
    x[j] = c < H ? load4(a.residual + base + c) : make_float4(0, 0, 0, 0);
  }
  if (a.n_planes + (a.add != nullptr) > 0) {
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const int c = (warp + j * warps) * kFp8Block + lane * 4;
      if (c < H) {
        if constexpr (SEVERAL) {
          double s[4] = {x[j].x, x[j].y, x[j].z, x[j].w};
#pragma unroll 4
          for (int p = 0; p < a.n_planes; ++p) {
            const float4 y = load4(a.planes + p * plane + base + c);
            s[0] += y.x, s[1] += y.y, s[2] += y.z, s[3] += y.w;
          }
          if (a.add != nullptr) {
            const float4 y = load4(static_cast<const T*>(a.add) + base + c);
            s[0] += y.x, s[1] += y.y, s[2] += y.z, s[3] += y.w;
          }
          x[j] = make_float4(float(s[0]), float(s[1]), float(s[2]), float(s[3]));
        } else {
          const float4 y = a.add != nullptr ? load4(static_cast<const T*>(a.add) + base + c) : load4(a.planes + base + c);
          x[j] = make_float4(x[j].x + y.x, x[j].y + y.y, x[j].z + y.z, x[j].w + y.w);
        }
        *reinterpret_cast<float4*>(a.residual + base + c) = x[j];
      }
    }
  }
  double ss[J];
#pragma unroll
  for (int j = 0; j < J; ++j) {
    const double b[4] = {x[j].x, x[j].y, x[j].z, x[j].w};
    ss[j] = fma(b[0], b[0], fma(b[1], b[1], fma(b[2], b[2], b[3] * b[3])));
  }
  constexpr int kLanes = J == 1 ? 32 : J == 2 ? 16 : J <= 4 ? 8 : 4;         // that have the same block's sum
  const double sum = block_sums<J>(ss, lane);
  const int mine = warp + lane / kLanes * warps;
  if (lane % kLanes == 0 && lane / kLanes < J && mine < blocks) red[mine] = sum;
  __syncthreads();
  double total = 0;
  for (int b = lane; b < blocks; b += 32) total += red[b];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
  const float inv = float(rsqrt(total / H + a.eps));
#pragma unroll
  for (int j = 0; j < J; ++j) {
    const int b = warp + j * warps, c = b * kFp8Block + lane * 4;
    if (b < blocks) {
      float y[4] = {0, 0, 0, 0};
      if (c < H) {
        const float4 w = load4(static_cast<const T*>(a.weight) + c);
        y[0] = x[j].x * inv * w.x, y[1] = x[j].y * inv * w.y, y[2] = x[j].z * inv * w.z, y[3] = x[j].w * inv * w.w;
        if (a.normed != nullptr) {
          uint2 v;
          v.x = pack2<T>(y[0], y[1]), v.y = pack2<T>(y[2], y[3]);
          *reinterpret_cast<uint2*>(static_cast<T*>(a.normed) + base + c) = v;
        }
      }
      const uint32_t top = __reduce_max_sync(0xffffffffu, max(max(abs_bits(y[0]), abs_bits(y[1])), max(abs_bits(y[2]), abs_bits(y[3]))));
      const float steps = fp8_steps(__uint_as_float(top));
      if (c < H) *reinterpret_cast<uint32_t*>(a.data + row * a.ld_data + c) = fp8_pack4(y, steps);
      if (lane == 0) a.scale[b * a.ld_scale + row] = fp8_scale(__uint_as_float(top));
    }
  }
}

// ---- rows, or act(gate) * up of their halves, in 8 bits ------------------------------------------------------------------------------
// 16 threads have a block, eight columns each.
template <typename T>
struct Eight {
  uint4 raw[sizeof(T) / 2];
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < int(sizeof(T) / 2); ++i) raw[i] = __ldcs(reinterpret_cast<const uint4*>(p) + i);
  }
  __device__ __forceinline__ void values(float* v) const {
    const float4 a = load4(reinterpret_cast<const T*>(raw)), b = load4(reinterpret_cast<const T*>(raw) + 4);
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
  }
};

template <typename T, int ACT>
__global__ void __launch_bounds__(256)
quant_fp8_kernel(const T* __restrict__ x, long long ldx, uint8_t* __restrict__ data, long long ld_data, float* __restrict__ scale,
                 long long ld_scale, int M, int C) {
  constexpr int kRows = 2;                                     // read before the first of them is worked on
  pdl_launch_dependents();
  pdl_wait();
  const int t = threadIdx.x & 15, b = blockIdx.x * 16 + (threadIdx.x >> 4), c = b * kFp8Block + t * 8;
  const bool inside = c < C;
  for (int row0 = blockIdx.y * kRows; row0 < M; row0 += gridDim.y * kRows) {
    Eight<T> g[kRows], u[kRows];
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      if (inside && row0 + r < M) {
        g[r].load(x + (row0 + r) * ldx + c);
        if (ACT != kFp8None) u[r].load(x + (row0 + r) * ldx + C + c);
      }
    }
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      const long long row = row0 + r;
      const bool live = inside && row < M;
      float y[8], v[8];
      g[r].values(y);
      if constexpr (ACT != kFp8None) {
        u[r].values(v);
#pragma unroll
        for (int k = 0; k < 8; ++k) y[k] = fp8_gated(ACT, y[k], v[k]);
      }
      uint32_t top = 0;
#pragma unroll
      for (int k = 0; k < 8; ++k) top = max(top, abs_bits(y[k]));
      if (!live) top = 0;
#pragma unroll
      for (int o = 1; o < 16; o <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
      const float steps = fp8_steps(__uint_as_float(top));
      if (live) *reinterpret_cast<uint2*>(data + row * ld_data + c) = make_uint2(fp8_pack4(y, steps), fp8_pack4(y + 4, steps));
      if (live && t == 0) scale[b * ld_scale + row] = fp8_scale(__uint_as_float(top));
    }
  }
}

template <typename T, bool SEVERAL>
int norm_fp8(const NormFp8& a, cudaStream_t st) {
  const int blocks = (a.H + kFp8Block - 1) / kFp8Block, least = (blocks + 31) / 32;
  auto go = [&](auto kernel, int J) {
    return launch_pdl(kernel, dim3(a.M), dim3(32 * ((blocks + J - 1) / J)), 0, st, a) == cudaSuccess ? 1 : ZSE_ERR_LAUNCH;
  };
  // many rows: eight warps a row, so that several rows are under way on an SM; few: as soon as possible done with each
  if (a.M >= 4 * sm_count() && blocks <= 64) {
    const int J = (blocks + 7) / 8;
    if (J == 1) return go(add_rmsnorm_fp8_kernel<T, 1, 256, SEVERAL>, 1);
    if (J == 2) return go(add_rmsnorm_fp8_kernel<T, 2, 256, SEVERAL>, 2);
    if (J == 3) return go(add_rmsnorm_fp8_kernel<T, 3, 256, SEVERAL>, 3);
    if (J == 4) return go(add_rmsnorm_fp8_kernel<T, 4, 256, SEVERAL>, 4);
    if (J == 5) return go(add_rmsnorm_fp8_kernel<T, 5, 256, SEVERAL>, 5);
    return go(add_rmsnorm_fp8_kernel<T, 8, 256, SEVERAL>, 8);
  }
  if (least == 1) return go(add_rmsnorm_fp8_kernel<T, 1, 1024, SEVERAL>, 1);
  if (least == 2) return go(add_rmsnorm_fp8_kernel<T, 2, 1024, SEVERAL>, 2);
  if (least <= 4) return go(add_rmsnorm_fp8_kernel<T, 4, 1024, SEVERAL>, 4);
  return go(add_rmsnorm_fp8_kernel<T, 8, 1024, SEVERAL>, 8);
}

template <typename T>
int quant_fp8(const ZseQuantFp8& q, cudaStream_t st) {
  const int across = ((q.C + kFp8Block - 1) / kFp8Block + 15) / 16;
  const dim3 grid(across, std::min((q.M + 1) / 2, 65535));
  auto go = [&](auto kernel) {
    return launch_pdl(kernel, grid, dim3(256), 0, st, static_cast<const T*>(q.x), q.ldx, static_cast<uint8_t*>(q.data), q.ld_data,
                      static_cast<float*>(q.scale), q.ld_scale, q.M, q.C) == cudaSuccess
               ? 1
               : ZSE_ERR_LAUNCH;
  };
  return q.act == kFp8None ? go(quant_fp8_kernel<T, kFp8None>) : q.act == kFp8Silu ? go(quant_fp8_kernel<T, kFp8Silu>) : go(quant_fp8_kernel<T, kFp8Gelu>);
}

bool aligned(const void* p, int bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

}  // namespace
}  // namespace zse

using namespace zse;

extern "C" int zse_add_rmsnorm_fp8(const ZseNormFp8* n) {
  if (n->M <= 0) return 0;
  if (n->H <= 0 || n->H % 16 || n->n_planes < 0 || n->residual == nullptr || n->weight == nullptr || (n->n_planes > 0 && n->planes == nullptr))
    return ZSE_ERR_SHAPE;
  if (n->H > 32768 || n->M > kFp8Most) return ZSE_ERR_LIMIT;
  const int64_t ld_data = n->M == 1 ? 0 : n->ld_data;          // (a single row may have any)
  if (!aligned(n->residual, 16) || !aligned(n->planes, 16) || !aligned(n->add, 8) || !aligned(n->weight, 8) || !aligned(n->normed, 8) ||
      !aligned(n->data, 16) || ld_data % 16 || !aligned(n->scale, 4))
    return ZSE_ERR_ALIGN;
  const NormFp8 a{static_cast<float*>(n->residual), static_cast<const float*>(n->planes), n->add, n->weight, n->normed,
                  static_cast<uint8_t*>(n->data), static_cast<float*>(n->scale), ld_data, n->ld_scale, n->eps, n->n_planes, n->M, n->H};
  const long long M = n->M, H = n->H, blocks = (H + kFp8Block - 1) / kFp8Block;
  const void* add = n->add == n->normed ? nullptr : n->add;                 // (normed in its place: each thread reads its own columns first)
  const Fp8Span written[] = {{n->residual, M * H * 4, 0, 1}, {n->data, H, ld_data, M}, {n->scale, M * 4, n->ld_scale * 4, blocks}, {n->normed, M * H * 2, 0, 1}};
  const Fp8Span read[] = {{n->n_planes > 0 ? n->planes : nullptr, M * H * 4 * n->n_planes, 0, 1}, {add, M * H * 2, 0, 1}, {n->weight, H * 2, 0, 1}};
  if (!written_apart(written, read)) return ZSE_ERR_SHAPE;
  const cudaStream_t st = static_cast<cudaStream_t>(n->stream);
  const bool several = n->n_planes + (n->add != nullptr) > 1;
  if (n->type == kFp8F16) return several ? norm_fp8<__half, true>(a, st) : norm_fp8<__half, false>(a, st);
  if (n->type == kFp8BF16) return several ? norm_fp8<bf16, true>(a, st) : norm_fp8<bf16, false>(a, st);
  return ZSE_ERR_SHAPE;
}

extern "C" int zse_quant_fp8(const ZseQuantFp8* q) {
  if (q->M <= 0) return 0;
  if (q->C <= 0 || q->C % 16 || q->act < kFp8None || q->act > kFp8Gelu) return ZSE_ERR_SHAPE;
  if (q->M > kFp8Most || q->C > kFp8Most) return ZSE_ERR_LIMIT;
  ZseQuantFp8 one = *q;
  if (q->M == 1) one.ldx = one.ld_data = 0, q = &one;          // (a single row may have any)
  const int item = q->type == kFp8F32 ? 4 : 2;
  if (!aligned(q->x, 16) || q->ldx * item % 16 || !aligned(q->data, 16) || q->ld_data % 16 || !aligned(q->scale, 4)) return ZSE_ERR_ALIGN;
  const Fp8Span written[] = {{q->data, q->C, q->ld_data, q->M}, {q->scale, q->M * 4ll, q->ld_scale * 4, (q->C + kFp8Block - 1) / kFp8Block}};
  const Fp8Span read[] = {{q->x, (q->act == kFp8None ? 1ll : 2ll) * q->C * item, q->ldx * item, q->M}};
  if (!written_apart(written, read)) return ZSE_ERR_SHAPE;
  const cudaStream_t st = static_cast<cudaStream_t>(q->stream);
  switch (q->type) {
    case kFp8F16: return quant_fp8<__half>(*q, st);
    case kFp8BF16: return quant_fp8<bf16>(*q, st);
    case kFp8F32: return quant_fp8<float>(*q, st);
    default: return ZSE_ERR_SHAPE;
  }
}
