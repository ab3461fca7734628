// Attention of new tokens (one, or a few, of every sequence) over the 8-bit KV cache.
#include "api.h"
#include "common.cuh"

namespace zse {

namespace {

constexpr float kLog2e = 1.4426950408889634f;

// The plain form: a CTA has one row of one head, a thread one token of a tile of 128.
template <int HD>
__global__ void __launch_bounds__(128)
attn_q8_kernel(const uint8_t* __restrict__ data, const float* __restrict__ scale, int num_blocks, int nkv, int block_size,
               const __half* __restrict__ q, int ldq, const int* __restrict__ tables, int max_blocks,
               const int* __restrict__ seq_lens, const int* __restrict__ cu_q, const int* __restrict__ q_pos0,
               __half* __restrict__ out, int ldo, int nh, float scale_log2, int window, Status* st) {
  pdl_launch_dependents();
  pdl_wait();
  __shared__ float qs[HD], ps[128], red[128];
  const int head = blockIdx.x, s = blockIdx.z, tid = threadIdx.x, kvh = head / (nh / nkv);
  const int row = cu_q != nullptr ? cu_q[s] + blockIdx.y : s;
  if (cu_q != nullptr && row >= cu_q[s + 1]) return;
  int len = cu_q != nullptr ? q_pos0[s] + int(blockIdx.y) + 1 : seq_lens[s];
  if (len < 0 || (len + block_size - 1) / block_size > max_blocks) {
    if (tid == 0) report(st, kBadArgument, 75, unsigned(s));
    len = max(0, min(len, max_blocks * block_size));
  }
  for (int d = tid; d < HD; d += 128) qs[d] = __half2float(q[size_t(row) * ldq + size_t(head) * HD + d]);
  __syncthreads();
  float m = -INFINITY, l = 0.f, acc[(HD + 127) / 128] = {};
  for (int t0 = window > 0 ? max(0, len - window) : 0; t0 < len; t0 += 128) {
    const int t = t0 + tid;
    float z = -INFINITY, vs = 0.f;
    if (t < len) {
      const int blk = tables[size_t(s) * max_blocks + t / block_size];
      if (blk >= num_blocks) report(st, kBadArgument, 76, unsigned(blk));
      if (blk >= 0 && blk < num_blocks) {
        const size_t r = ((size_t(blk) * 2) * nkv + kvh) * block_size + t % block_size;
        float dot = 0.f;
        for (int d = 0; d < HD; ++d) dot += qs[d] * float(int(data[r * HD + d]) - 128);
        z = dot * scale[r] * scale_log2;
        vs = scale[r + size_t(nkv) * block_size];
      }
    }
    red[tid] = z;
    __syncthreads();
    float top = m;
    for (int i = 0; i < 128; ++i) top = fmaxf(top, red[i]);
    __syncthreads();
    const float base = top == -INFINITY ? 0.f : top, fade = exp2f(m - base), p = exp2f(z - base);
    m = top;
    red[tid] = p;
    ps[tid] = z == -INFINITY ? 0.f : p * vs;
    __syncthreads();
    l *= fade;
    for (int i = 0; i < 128; ++i) l += red[i];
    for (int k = 0; k * 128 + tid < HD; ++k) acc[k] *= fade;
    for (int i = 0; i < min(128, len - t0); ++i) {
      const int t1 = t0 + i, blk = tables[size_t(s) * max_blocks + t1 / block_size];
      if (blk < 0 || blk >= num_blocks) continue;
      const size_t r = ((size_t(blk) * 2 + 1) * nkv + kvh) * block_size + t1 % block_size;
      for (int k = 0; k * 128 + tid < HD; ++k) acc[k] += ps[i] * float(int(data[r * HD + k * 128 + tid]) - 128);
    }
    __syncthreads();
  }
  for (int k = 0; k * 128 + tid < HD; ++k)
    out[size_t(row) * ldo + size_t(head) * HD + k * 128 + tid] = __float2half_rn(l == 0.f ? 0.f : acc[k] / l);
}

}  // namespace
}  // namespace zse

using namespace zse;

extern "C" int zse_attn_decode_q8_splits(int, int, int, int, int, int, int, int, int) { return 1; }
extern "C" int64_t zse_attn_decode_q8_scratch_floats(int, int, int, int, int) { return 0; }

extern "C" int zse_attn_decode_q8(const ZseKvQ8* kv, const void* q, int ldq, const void* tables, int max_blocks,
                                  const void* seq_lens, const void* cu_q, const void* q_pos0, int num_seqs, int max_q, void* out,
                                  int ldo, int nh, void* scratch, int64_t scratch_floats, int num_splits, float scale, int window,
                                  void* status, void* stream) {
  if (num_seqs <= 0 || max_q <= 0) return 0;
  if (kv->num_blocks <= 0 || kv->nkv <= 0 || kv->block_size <= 0 || kv->block_size % 16 || nh <= 0 || nh % kv->nkv ||
      nh / kv->nkv > 16 || num_seqs > 65535)
    return ZSE_ERR_SHAPE;
  auto go = [&](auto kernel) {
    return launch_pdl(kernel, dim3(nh, max_q, num_seqs), dim3(128), 0, static_cast<cudaStream_t>(stream),
                      static_cast<const uint8_t*>(kv->data), static_cast<const float*>(kv->scale), kv->num_blocks, kv->nkv,
                      kv->block_size, static_cast<const __half*>(q), ldq, static_cast<const int*>(tables), max_blocks,
                      static_cast<const int*>(seq_lens), static_cast<const int*>(cu_q), static_cast<const int*>(q_pos0),
                      static_cast<__half*>(out), ldo, nh, scale * kLog2e, window, static_cast<Status*>(status)) == cudaSuccess
               ? 0
               : ZSE_ERR_LAUNCH;
  };
  switch (kv->hd) {
    case 64: return go(attn_q8_kernel<64>);
    case 96: return go(attn_q8_kernel<96>);
    case 128: return go(attn_q8_kernel<128>);
    case 256: return go(attn_q8_kernel<256>);
    default: return ZSE_ERR_SHAPE;
  }
}
