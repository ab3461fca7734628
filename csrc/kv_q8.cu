// The 8-bit KV cache: written (rotation, quantisation) and read back.
//
// An element is stored as a byte u and stands for (u - 128) * scale, with one fp32 scale per (token, kv head), K and V apart.  A
// scale per token and head costs 4 bytes per head_dim and keeps a token's error within max|x| / 254 of its own values; attention
// takes it out of its products (q . (u - 128) times the scale of K; weight times the scale of V), so no element is multiplied.
#include <algorithm>

#include "api.h"
#include "common.cuh"

namespace zse {

namespace {

constexpr double kTurn = 6.283185307179586, kTurnLow = 2.4492935982947064e-16;   // 2 pi in two parts

// max and clamp that keep a NaN: a row that holds one is stored with a NaN scale and reads back as NaN, as it would in fp16
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float clamp_nan(float x) {
  float r;
  asm("{\n\t.reg .f32 t;\n\tmax.NaN.f32 t, %1, 0fC77FE000;\n\tmin.NaN.f32 %0, t, 0f477FE000;\n\t}" : "=f"(r) : "f"(x));  // +-65504
  return r;
}
__device__ __forceinline__ uint32_t half2_bits(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// bytes of eight values: rint(x * steps) + 128; steps * |x| <= 127 up to rounding, so the sum is within 1 .. 255 (NaN: 128)
__device__ __forceinline__ uint2 quantise8(const float* x, float steps) {
  uint32_t w[2] = {0u, 0u};
#pragma unroll
  for (int j = 0; j < 8; ++j) w[j >> 2] |= uint32_t(__float2int_rn(x[j] * steps) + 128) << (8 * (j & 3));
  return make_uint2(w[0], w[1]);
}

template <int HD>
constexpr int kLanes = HD <= 64 ? 4 : HD <= 128 ? 8 : 16;      // threads of a head, a power of two; HD / 16 of them work

// A CTA has one token and blockIdx.y's share of its heads; a thread has 16 elements of a head, two runs of eight that rotate with
// each other (or neighbouring runs of the part that does not rotate).  Angles are products in 64 bits brought into one turn, so a
// rotation is as exact at position 10^9 as at 0; they are computed once per CTA.
template <int HD>
__global__ void __launch_bounds__(256)
rope_kv_write_q8_kernel(const __half* qkv, int ld, __half* q_out, int ld_q, const float* __restrict__ planes, int n_planes,
                        const __half* __restrict__ bias, uint8_t* __restrict__ data, float* __restrict__ scale,
                        const int* __restrict__ positions, const long long* __restrict__ slots,
                        const float* __restrict__ inv_freq, int nh, int nkv, int rot, int block_size, long long num_slots,
                        Status* st) {
  pdl_launch_dependents();
  pdl_wait();
  constexpr int L = kLanes<HD>;
  constexpr int kHeads = 256 / L;
  __shared__ float sin_t[HD / 2], cos_t[HD / 2];
  const int t = blockIdx.x, M = gridDim.x, half = rot / 2;
  if (threadIdx.x < half) {
    const double turns = double(positions[t]) * double(inv_freq[threadIdx.x]);
    const double n = rint(turns * (1.0 / kTurn));
    sincosf(float(fma(-n, kTurnLow, fma(-n, kTurn, turns))), &sin_t[threadIdx.x], &cos_t[threadIdx.x]);
  }
  __syncthreads();
  const int c = threadIdx.x % L;
  const bool works = c < HD / 16, turns = works && c < rot / 16;
  const int ia = turns ? c * 8 : works ? rot + (c - rot / 16) * 16 : 0, ib = turns ? half + c * 8 : ia + 8;
  const int heads = nh + 2 * nkv, cols = heads * HD;
  long long slot = slots[t];
  if (slot >= num_slots) {
    if (threadIdx.x == 0 && blockIdx.y == 0) report(st, kBadArgument, 70, unsigned(t));
    slot = -1;
  }
  const long long blk = slot >= 0 ? slot / block_size : 0;
  const int off = slot >= 0 ? int(slot - blk * block_size) : 0;
  for (int base = blockIdx.y * kHeads; base < heads; base += gridDim.y * kHeads) {     // the same rounds for the whole CTA
    const int head = base + threadIdx.x / L;
    const bool live = works && head < heads;
    float a[8], b[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) a[j] = b[j] = 0.f;
    if (live) {
      if (planes != nullptr) {
        if (bias != nullptr) {
#pragma unroll
          for (int j = 0; j < 8; ++j) a[j] = __half2float(bias[head * HD + ia + j]), b[j] = __half2float(bias[head * HD + ib + j]);
        }
        for (int p = 0; p < n_planes; ++p) {
          const float* src = planes + (size_t(p) * M + t) * cols + size_t(head) * HD;
#pragma unroll
          for (int j = 0; j < 8; ++j) a[j] += src[ia + j], b[j] += src[ib + j];
        }
      } else {
        const __half* src = qkv + size_t(t) * ld + size_t(head) * HD;
#pragma unroll
        for (int j = 0; j < 8; ++j) a[j] = __half2float(src[ia + j]), b[j] = __half2float(src[ib + j]);
      }
      if (turns && head < nh + nkv) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float s = sin_t[c * 8 + j], k = cos_t[c * 8 + j], x = a[j], y = b[j];
          a[j] = x * k - y * s;
          b[j] = y * k + x * s;
        }
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) a[j] = clamp_nan(a[j]), b[j] = clamp_nan(b[j]);
    }
    float top = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) top = max_nan(top, max_nan(fabsf(a[j]), fabsf(b[j])));
#pragma unroll
    for (int o = 1; o < L; o <<= 1) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (!live) continue;
    if (head < nh) {
      __half* dst = q_out + size_t(t) * ld_q + size_t(head) * HD;
#pragma unroll
      for (int j = 0; j < 8; ++j) dst[ia + j] = __float2half_rn(a[j]), dst[ib + j] = __float2half_rn(b[j]);
    } else if (slot >= 0) {
      const bool none = top <= 1e-30f;
      const float steps = none ? 0.f : __fdiv_rn(127.f, top);
      const size_t row = ((size_t(blk) * 2) * nkv + (head - nh)) * block_size + off;     // K heads, then V heads
      uint8_t* dst = data + row * HD;
      *reinterpret_cast<uint2*>(dst + ia) = quantise8(a, steps);
      *reinterpret_cast<uint2*>(dst + ib) = quantise8(b, steps);
      if (c == 0) scale[row] = none ? 0.f : __fdiv_rn(top, 127.f);
    }
  }
}

// A CTA takes page after page: the sequence a page belongs to is the number of sequences that end at or before it.  A thread
// reads 16 bytes and writes 32.
__global__ void __launch_bounds__(256)
kv_read_q8_kernel(const uint8_t* __restrict__ data, const float* __restrict__ scale, int num_blocks, int nkv, int block_size,
                  int hd, const int* __restrict__ tables, int table_ld, int max_blocks, const int* __restrict__ seq_lens,
                  const int* __restrict__ cu_blocks, int num_seqs, __half* __restrict__ out, int out_blocks,
                  int* __restrict__ out_tables, int out_table_ld, int out_max_blocks, Status* st) {
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const long long entries = (long long)num_seqs * out_max_blocks;
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < entries; i += (long long)gridDim.x * 256) {
    const int s = int(i / out_max_blocks), j = int(i - (long long)s * out_max_blocks);
    const int len = seq_lens[s], first = cu_blocks[s], pages = (max(len, 0) + block_size - 1) / block_size;
    const bool fits = first >= 0 && pages <= min(min(max_blocks, out_max_blocks), cu_blocks[s + 1] - first) && first + pages <= out_blocks;
    if (j == 0 && (!fits || len < 0)) report(st, kBadArgument, 71, unsigned(s));
    const int blk = fits && j < pages ? tables[size_t(s) * table_ld + j] : -1;
    if (blk >= num_blocks) report(st, kBadArgument, 72, unsigned(blk));
    out_tables[size_t(s) * out_table_ld + j] = blk >= 0 && blk < num_blocks ? first + j : -1;
  }
  const int total = min(cu_blocks[num_seqs], out_blocks);
  const int runs = 2 * nkv * block_size * hd / 16, row16 = hd / 16;
  for (int page = blockIdx.x; page < total; page += gridDim.x) {
    int s = 0;
    for (int i = lane; i - lane < num_seqs; i += 32)
      s += __popc(__ballot_sync(0xffffffffu, i < num_seqs && cu_blocks[i + 1] <= page));
    if (s >= num_seqs) continue;
    const int first = cu_blocks[s], j = page - first, len = seq_lens[s], pages = (max(len, 0) + block_size - 1) / block_size;
    if (first < 0 || j < 0 || j >= pages || pages > min(min(max_blocks, out_max_blocks), cu_blocks[s + 1] - first) ||
        first + pages > out_blocks)
      continue;
    const int blk = tables[size_t(s) * table_ld + j];
    if (blk < 0 || blk >= num_blocks) continue;
    const uint4* src = reinterpret_cast<const uint4*>(data) + size_t(blk) * runs;
    const float* sc = scale + size_t(blk) * 2 * nkv * block_size;
    uint4* dst = reinterpret_cast<uint4*>(out) + size_t(page) * runs * 2;
    for (int i = threadIdx.x; i < runs; i += 256) {
      const int row = i / row16;
      const bool in = j * block_size + row % block_size < len;
      const float f = sc[row];
      const uint4 v = src[i];
      const uint32_t w[4] = {v.x, v.y, v.z, v.w};
      uint32_t h[8];
#pragma unroll
      for (int k = 0; k < 4; ++k)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float x = float(int((w[k] >> (16 * e)) & 255u) - 128) * f, y = float(int((w[k] >> (16 * e + 8)) & 255u) - 128) * f;
          h[2 * k + e] = in ? half2_bits(x, y) : 0u;
        }
      dst[2 * i] = make_uint4(h[0], h[1], h[2], h[3]);
      dst[2 * i + 1] = make_uint4(h[4], h[5], h[6], h[7]);
    }
  }
}

bool cache_ok(const ZseKvQ8* kv) {
  return kv->num_blocks > 0 && kv->nkv > 0 && kv->block_size > 0 && kv->block_size % 16 == 0 &&
         (kv->hd == 64 || kv->hd == 96 || kv->hd == 128 || kv->hd == 256);
}
bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
int sm_count() {
  static int counts[kMaxDevices];
  const int slot = current_device_slot();
  if (counts[slot] == 0 && cudaDeviceGetAttribute(&counts[slot], cudaDevAttrMultiProcessorCount, slot) != cudaSuccess) return 148;
  return counts[slot];
}

}  // namespace
}  // namespace zse

using namespace zse;

extern "C" int zse_rope_kv_write_q8(const ZseKvQ8* kv, const void* qkv, int ld, void* q_out, int ld_q, const void* planes,
                                    int n_planes, const void* bias, const void* positions, const void* slots,
                                    const void* inv_freq, int M, int nh, int rotary_dim, void* status, void* stream) {
  if (M <= 0) return 0;
  if (!cache_ok(kv) || nh <= 0 || rotary_dim < 0 || rotary_dim % 16 || rotary_dim > kv->hd || (planes == nullptr && qkv == nullptr))
    return ZSE_ERR_SHAPE;
  if (!aligned16(kv->data) || !aligned16(kv->scale) || !aligned16(q_out) || ld_q % 8 ||
      (planes != nullptr ? !aligned16(planes) || (bias != nullptr && !aligned16(bias)) : !aligned16(qkv) || ld % 8))
    return ZSE_ERR_ALIGN;
  auto go = [&](auto kernel, int lanes) {
    const int rounds = (nh + 2 * kv->nkv + 256 / lanes - 1) / (256 / lanes);
    return launch_pdl(kernel, dim3(M, M < sm_count() ? rounds : 1), dim3(256), 0, static_cast<cudaStream_t>(stream),
                      static_cast<const __half*>(qkv), ld, static_cast<__half*>(q_out), ld_q, static_cast<const float*>(planes),
                      n_planes, static_cast<const __half*>(bias), static_cast<uint8_t*>(kv->data), static_cast<float*>(kv->scale),
                      static_cast<const int*>(positions), static_cast<const long long*>(slots),
                      static_cast<const float*>(inv_freq), nh, kv->nkv, rotary_dim, kv->block_size,
                      (long long)kv->num_blocks * kv->block_size, static_cast<Status*>(status)) == cudaSuccess
               ? 0
               : ZSE_ERR_LAUNCH;
  };
  switch (kv->hd) {
    case 64: return go(rope_kv_write_q8_kernel<64>, kLanes<64>);
    case 96: return go(rope_kv_write_q8_kernel<96>, kLanes<96>);
    case 128: return go(rope_kv_write_q8_kernel<128>, kLanes<128>);
    default: return go(rope_kv_write_q8_kernel<256>, kLanes<256>);
  }
}

extern "C" int zse_kv_read_q8(const ZseKvQ8* kv, const void* tables, int table_ld, int max_blocks, const void* seq_lens,
                              const void* cu_blocks, int num_seqs, void* out, int out_blocks, void* out_tables, int out_table_ld,
                              int out_max_blocks, void* status, void* stream) {
  if (num_seqs <= 0) return 0;
  if (!cache_ok(kv) || max_blocks < 0 || out_blocks < 0 || out_max_blocks < 0) return ZSE_ERR_SHAPE;
  if (!aligned16(kv->data) || !aligned16(kv->scale) || !aligned16(out)) return ZSE_ERR_ALIGN;
  const long long entries = ((long long)num_seqs * out_max_blocks + 255) / 256;
  const int grid = int(std::max(1ll, std::min((long long)sm_count() * 8, std::max((long long)out_blocks, entries))));
  return launch_pdl(kv_read_q8_kernel, dim3(grid), dim3(256), 0, static_cast<cudaStream_t>(stream),
                    static_cast<const uint8_t*>(kv->data), static_cast<const float*>(kv->scale), kv->num_blocks, kv->nkv,
                    kv->block_size, kv->hd, static_cast<const int*>(tables), table_ld, max_blocks, static_cast<const int*>(seq_lens),
                    static_cast<const int*>(cu_blocks), num_seqs, static_cast<__half*>(out), out_blocks,
                    static_cast<int*>(out_tables), out_table_ld, out_max_blocks, static_cast<Status*>(status)) == cudaSuccess
             ? 0
             : ZSE_ERR_LAUNCH;
}
