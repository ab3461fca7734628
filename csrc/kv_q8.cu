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
// bytes of eight values: rint(x * steps) + 128, in the low byte of a float between 2^23 and 2^24; steps * |x| <= 127 up to
// rounding, so they are within 1 .. 255
__device__ __forceinline__ uint2 quantise8(const float* x, float steps) {
  uint32_t b[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) b[j] = __float_as_uint(__fadd_rn(__fmul_rn(x[j], steps), 8388736.f));
  return make_uint2(__byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410),
                    __byte_perm(__byte_perm(b[4], b[5], 0x0040), __byte_perm(b[6], b[7], 0x0040), 0x5410));
}
__device__ __forceinline__ void unpack8(const uint4& v, float* x) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[j]));
    x[2 * j] = f.x;
    x[2 * j + 1] = f.y;
  }
}
__device__ __forceinline__ uint4 pack8(const float* x) {
  return make_uint4(half2_bits(x[0], x[1]), half2_bits(x[2], x[3]), half2_bits(x[4], x[5]), half2_bits(x[6], x[7]));
}

template <int HD>
constexpr int kLanes = HD / 16;                                // threads of a head: 4, 6, 8 or 16
template <int HD>
constexpr int kWarpHeads = 32 / kLanes<HD>;                    // heads of a warp.  Of 96: five, and two threads idle; as eight
                                                               // threads a head, two of them idle, 8080 rows of 96 heads took 60 us instead of 53

// What the two write kernels do with a head of a token: a thread has 16 of its elements, two runs of eight that rotate with each
// other (or neighbouring runs of the part that does not rotate).
struct Write {
  __half* q_out;
  uint8_t* data;
  float* scale;
  int ld_q, nh, nkv;
};
template <int HD>
struct Lane {
  static constexpr int L = kLanes<HD>;
  int group, c, ia, ib;                                                // head of the CTA's at a time, thread of it; first elements of the two runs
  bool works, turns;
  __device__ __forceinline__ explicit Lane(int rot) {
    const int lane = threadIdx.x & 31;
    group = (threadIdx.x >> 5) * kWarpHeads<HD> + lane / L;
    c = lane % L;
    works = lane < kWarpHeads<HD> * L;
    turns = works && c < rot / 16;
    ia = turns ? c * 8 : works ? rot + (c - rot / 16) * 16 : 0;
    ib = turns ? rot / 2 + c * 8 : ia + 8;
  }
};
// `stored`: the cache row of K head 0 of the token, or -1; the whole warp calls it (live: this thread has something)
template <int HD>
__device__ __forceinline__ void put_head(const Write& w, const Lane<HD>& lane, float* a, float* b, const float* sn, const float* cs,
                                         bool live, int t, int head, long long stored, int block_size) {
  if (live && lane.turns && head < w.nh + w.nkv) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float x = a[j], y = b[j], s = sn[lane.c * 8 + j], c = cs[lane.c * 8 + j];
      a[j] = x * c - y * s;
      b[j] = y * c + x * s;
    }
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) a[j] = clamp_nan(a[j]), b[j] = clamp_nan(b[j]);
  const bool cached = live && head >= w.nh && stored >= 0;
  if (__any_sync(0xffffffffu, cached)) {
    float top = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) top = max_nan(top, max_nan(fabsf(a[j]), fabsf(b[j])));
    if constexpr (Lane<HD>::L == 6) {                                  // the thread three on, then the two that are one and two on
      const int first = (threadIdx.x & 31) - lane.c;
      top = max_nan(top, __shfl_sync(0xffffffffu, top, first + (lane.c + 3) % 6));
      top = max_nan(top, max_nan(__shfl_sync(0xffffffffu, top, first + (lane.c + 1) % 6), __shfl_sync(0xffffffffu, top, first + (lane.c + 2) % 6)));
    } else {
#pragma unroll
      for (int o = 1; o < Lane<HD>::L; o <<= 1) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
    }
    if (cached) {
      const bool none = top <= 1e-30f;
      const float steps = none ? 0.f : __fdiv_rn(127.f, top);
      const size_t row = size_t(stored) + size_t(head - w.nh) * block_size;            // K heads, then V heads
      uint8_t* dst = w.data + row * HD;
      *reinterpret_cast<uint2*>(dst + lane.ia) = quantise8(a, steps);
      *reinterpret_cast<uint2*>(dst + lane.ib) = quantise8(b, steps);
      if (lane.c == 0) w.scale[row] = none ? 0.f : __fdiv_rn(top, 127.f);
    }
  }
  if (live && head < w.nh) {
    __half* dst = w.q_out + size_t(t) * w.ld_q + size_t(head) * HD;
    *reinterpret_cast<uint4*>(dst + lane.ia) = pack8(a);
    *reinterpret_cast<uint4*>(dst + lane.ib) = pack8(b);
  }
}
// Sine and cosine of a token's angle for pair i: the product in 64 bits, brought into one turn, so that a rotation is as exact at
// position 10^9 as at 0.
__device__ __forceinline__ void turn_of(int position, float freq, float* s, float* c) {
  const double turn = double(position) * double(freq), n = rint(turn * (1.0 / kTurn));
  sincosf(float(fma(-n, kTurnLow, fma(-n, kTurn, turn))), s, c);
}
// The cache row of K head 0 of a slot, or -1.
__device__ __forceinline__ long long row_of_slot(long long slot, int t, int nkv, int block_size, long long num_slots, Status* st) {
  if (slot >= num_slots) {
    report(st, kBadArgument, 70, unsigned(t));
    return -1;
  }
  if (slot < 0) return -1;
  const long long blk = slot / block_size;
  return blk * 2 * nkv * block_size + (slot - blk * block_size);
}

// Rows of fp16.  A CTA has `tokens` neighbouring tokens: their angles (one per thread), then their heads, each thread's next 32 bytes
// loaded before those at hand are turned.  With one token a CTA (48 heads of 64 are 3 KB) it is all start: 8080 such tokens took 34 us,
// eight a CTA 20 (4.5 TB/s of 91 MB); 2590 tokens of 56 heads of 128 14 (4.9 TB/s).  Bound by launch and memory latency, not by its
// instructions: half of them, at the same CTAs an SM, took the same time.
template <int HD>
__global__ void __launch_bounds__(256)
rope_kv_write_q8_kernel(const __half* qkv, int ld, Write w, const int* __restrict__ positions, const long long* __restrict__ slots,
                        const float* __restrict__ inv_freq, int M, int tokens, int rot, int block_size, long long num_slots, Status* st) {
  pdl_launch_dependents();
  pdl_wait();
  constexpr int kGroups = 8 * kWarpHeads<HD>, kMost = 16;
  __shared__ float sin_t[256], cos_t[256];                             // [token][rot / 2]
  __shared__ long long stored[kMost];
  const Lane<HD> lane(rot);
  const int half = rot / 2, heads = w.nh + 2 * w.nkv, t0 = blockIdx.x * tokens, n = min(tokens, M - t0);
  // this thread's heads: every kGroups-th of the tokens' heads in a row (with gridDim.y > 1: of one token, its share)
  int head = blockIdx.y * kGroups + lane.group, t = 0;
  const int step = gridDim.y * kGroups;
  uint4 va = make_uint4(0, 0, 0, 0), vb = va;
  auto fetch = [&]() {
    while (head >= heads && t < n) head -= heads, ++t;
    if (t < n && lane.works) {
      const __half* src = qkv + size_t(t0 + t) * ld + size_t(head) * HD;
      va = *reinterpret_cast<const uint4*>(src + lane.ia);
      vb = *reinterpret_cast<const uint4*>(src + lane.ib);
    }
  };
  if (gridDim.y > 1 && head >= heads) t = n;
  fetch();
  for (int i = threadIdx.x; i < n * half; i += 256) {
    const int k = i / half;
    turn_of(positions[t0 + k], inv_freq[i - k * half], &sin_t[i], &cos_t[i]);
  }
  if (threadIdx.x < n) stored[threadIdx.x] = row_of_slot(slots[t0 + threadIdx.x], t0 + threadIdx.x, w.nkv, block_size, num_slots, st);
  __syncthreads();
  while (__any_sync(0xffffffffu, t < n)) {
    const int now = t, at = head;
    const bool live = t < n && lane.works;
    float a[8], b[8];
    unpack8(va, a);
    unpack8(vb, b);
    head += step;
    if (gridDim.y > 1 && head >= heads) t = n;
    fetch();
    put_head<HD>(w, lane, a, b, sin_t + now * half, cos_t + now * half, live, t0 + now, at, live ? stored[now] : -1, block_size);
  }
}

// Sums of planes (few rows: a decode step; 64 rows of 56 heads from four planes 4.7 us, 1.2 at the rate of a copy).  A CTA has one token
// and blockIdx.y's share of its heads; four planes are loaded before the first is added.
template <int HD>
__global__ void __launch_bounds__(256)
rope_kv_write_q8_planes_kernel(const float* __restrict__ planes, int n_planes, const __half* __restrict__ bias, Write w,
                               const int* __restrict__ positions, const long long* __restrict__ slots,
                               const float* __restrict__ inv_freq, int rot, int block_size, long long num_slots, Status* st) {
  pdl_launch_dependents();
  pdl_wait();
  constexpr int kHeads = 8 * kWarpHeads<HD>, kPlanes = 4;
  __shared__ float sin_t[HD / 2], cos_t[HD / 2];
  __shared__ long long stored;
  const Lane<HD> lane(rot);
  const int t = blockIdx.x, M = gridDim.x, heads = w.nh + 2 * w.nkv, cols = heads * HD;
  float a[8], b[8];
  auto load = [&](int head) {
#pragma unroll
    for (int j = 0; j < 8; ++j) a[j] = b[j] = 0.f;
    if (!lane.works || head >= heads) return;
    if (bias != nullptr) {
      unpack8(*reinterpret_cast<const uint4*>(bias + head * HD + lane.ia), a);
      unpack8(*reinterpret_cast<const uint4*>(bias + head * HD + lane.ib), b);
    }
    const float* src = planes + size_t(t) * cols + size_t(head) * HD;
    const size_t next = size_t(M) * cols;
    for (int p = 0; p < n_planes; p += kPlanes) {
      float4 x[kPlanes][4];
#pragma unroll
      for (int k = 0; k < kPlanes; ++k)
        if (p + k < n_planes) {
          const float* from = src + (p + k) * next;
          x[k][0] = __ldcs(reinterpret_cast<const float4*>(from + lane.ia));
          x[k][1] = __ldcs(reinterpret_cast<const float4*>(from + lane.ia + 4));
          x[k][2] = __ldcs(reinterpret_cast<const float4*>(from + lane.ib));
          x[k][3] = __ldcs(reinterpret_cast<const float4*>(from + lane.ib + 4));
        }
#pragma unroll
      for (int k = 0; k < kPlanes; ++k)
        if (p + k < n_planes) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            a[e] += (&x[k][0].x)[e];
            a[4 + e] += (&x[k][1].x)[e];
            b[e] += (&x[k][2].x)[e];
            b[4 + e] += (&x[k][3].x)[e];
          }
        }
    }
  };
  int head = blockIdx.y * kHeads + lane.group;
  load(head);
  if (threadIdx.x < rot / 2) turn_of(positions[t], inv_freq[threadIdx.x], &sin_t[threadIdx.x], &cos_t[threadIdx.x]);
  if (threadIdx.x == 0) stored = row_of_slot(slots[t], t, w.nkv, block_size, num_slots, st);
  __syncthreads();
  for (int base = blockIdx.y * kHeads; base < heads; base += gridDim.y * kHeads) {     // the same rounds for the whole CTA
    put_head<HD>(w, lane, a, b, sin_t, cos_t, lane.works && head < heads, t, head, stored, block_size);
    head += gridDim.y * kHeads;
    load(head);
  }
}

// Eight bytes -> eight fp16: a byte below 0x4B0000 is 2^23 + u in fp32, so the difference is exact and the product rounded once
// before the rounding to fp16.
__device__ __forceinline__ uint4 values8(const uint2& v, float f) {
  const uint32_t w[2] = {v.x, v.y};
  float x[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) x[j] = (__uint_as_float(__byte_perm(w[j >> 2], 0x4B000000u, 0x7540 + (j & 3))) - 8388736.f) * f;
  return pack8(x);
}

// A CTA takes part after part of the pages (a page is `parts` of them, for few pages): the sequence a page belongs to is the number of
// sequences that end at or before it.  Where the next part lies is looked up before this one is copied.  A thread reads 8 bytes and
// writes 16, so that a warp's stores are one run; four such pieces are loaded before the first is converted.  109 k tokens of 8 heads of
// 128, a few blocks dropped: 99 us, 5.7 TB/s of one byte in and two out (16-byte loads with 32-byte stores 113 us).
template <int HD>
__global__ void __launch_bounds__(256)
kv_read_q8_kernel(const uint8_t* __restrict__ data, const float* __restrict__ scale, int num_blocks, int nkv, int block_size,
                  const int* __restrict__ tables, int table_ld, int max_blocks, const int* __restrict__ seq_lens,
                  const int* __restrict__ cu_blocks, int num_seqs, __half* __restrict__ out, int out_blocks,
                  int* __restrict__ out_tables, int out_table_ld, int out_max_blocks, int parts, Status* st) {
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const long long entries = (long long)num_seqs * out_max_blocks;
  auto pages_of = [&](int len) { return max(len, 0) / block_size + (max(len, 0) % block_size > 0); };
  auto fit = [&](int first, int pages, int last) {                     // (no sum of these overflows)
    return first >= 0 && pages <= min(max_blocks, out_max_blocks) && first <= out_blocks - pages && first + pages <= last;
  };
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < entries; i += (long long)gridDim.x * 256) {
    const int s = int(i / out_max_blocks), j = int(i - (long long)s * out_max_blocks);
    const int len = seq_lens[s], first = cu_blocks[s], pages = pages_of(len);
    const bool fits = fit(first, pages, cu_blocks[s + 1]);
    if (j == 0 && (!fits || len < 0)) report(st, kBadArgument, 71, unsigned(s));
    const int blk = fits && j < pages ? tables[size_t(s) * table_ld + j] : -1;
    if (blk >= num_blocks) report(st, kBadArgument, 72, unsigned(blk));
    out_tables[size_t(s) * out_table_ld + j] = blk >= 0 && blk < num_blocks ? first + j : -1;
  }
  constexpr int kRow = HD / 8, kAhead = 4;                             // pieces of a row
  const int total = min(cu_blocks[num_seqs], out_blocks) * parts;
  const int pieces = 2 * nkv * block_size * kRow, per_part = (pieces + parts - 1) / parts;
  struct Part {
    int blk, page, inside;                                             // blk -1: nothing to copy; tokens of the sequence in the page
  };
  auto look_up = [&](int part) {
    Part u{-1, part / parts, 0};
    if (part >= total) return u;
    int s = 0;
    for (int i = lane; i - lane < num_seqs; i += 32)
      s += __popc(__ballot_sync(0xffffffffu, i < num_seqs && cu_blocks[i + 1] <= u.page));
    if (s >= num_seqs) return u;
    const int first = cu_blocks[s], len = seq_lens[s], pages = pages_of(len);
    if (!fit(first, pages, cu_blocks[s + 1]) || u.page < first || u.page - first >= pages) return u;
    const int j = u.page - first;
    const int blk = tables[size_t(s) * table_ld + j];
    if (blk >= 0 && blk < num_blocks) u.blk = blk;
    u.inside = min(block_size, len - j * block_size);
    return u;
  };
  Part now = look_up(blockIdx.x);
  for (int part = blockIdx.x; part < total; part += gridDim.x) {
    const Part next = look_up(part + gridDim.x);
    if (now.blk >= 0) {
      const uint2* src = reinterpret_cast<const uint2*>(data) + size_t(now.blk) * pieces;
      const float* sc = scale + size_t(now.blk) * 2 * nkv * block_size;
      uint4* dst = reinterpret_cast<uint4*>(out) + size_t(now.page) * pieces;
      const int begin = (part - now.page * parts) * per_part, end = min(pieces, begin + per_part);
      for (int i0 = begin + threadIdx.x; i0 < end; i0 += 256 * kAhead) {
        uint2 v[kAhead];
        float f[kAhead];
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
          const int i = i0 + k * 256;
          if (i < end) {
            v[k] = __ldcs(src + i);
            f[k] = sc[i / kRow];
          }
        }
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
          const int i = i0 + k * 256;
          if (i < end)
            dst[i] = now.inside == block_size || (i / kRow) % block_size < now.inside ? values8(v[k], f[k]) : make_uint4(0, 0, 0, 0);
        }
      }
    }
    now = next;
  }
}

bool cache_ok(const ZseKvQ8& kv) {
  return kv.num_blocks > 0 && kv.nkv > 0 && kv.block_size > 0 && kv.block_size % 16 == 0 &&
         (kv.hd == 64 || kv.hd == 96 || kv.hd == 128 || kv.hd == 256);
}
bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace
}  // namespace zse

using namespace zse;

extern "C" int zse_rope_kv_write_q8(const ZseWriteQ8* w) {
  const ZseKvQ8& kv = w->kv;
  if (w->M <= 0) return 0;
  if (!cache_ok(kv) || w->nh <= 0 || w->rotary_dim < 0 || w->rotary_dim % 16 || w->rotary_dim > kv.hd ||
      (w->planes == nullptr && w->qkv == nullptr))
    return ZSE_ERR_SHAPE;
  if (!aligned16(kv.data) || !aligned16(kv.scale) || !aligned16(w->q_out) || w->ld_q % 8 ||
      (w->planes != nullptr ? !aligned16(w->planes) || (w->bias != nullptr && !aligned16(w->bias)) : !aligned16(w->qkv) || w->ld % 8))
    return ZSE_ERR_ALIGN;
  const Write to{static_cast<__half*>(w->q_out), static_cast<uint8_t*>(kv.data), static_cast<float*>(kv.scale), w->ld_q, w->nh, kv.nkv};
  const long long num_slots = (long long)kv.num_blocks * kv.block_size;
  const auto* positions = static_cast<const int*>(w->positions);
  const auto* slots = static_cast<const long long*>(w->slots);
  const auto* freqs = static_cast<const float*>(w->inv_freq);
  auto* status = static_cast<Status*>(w->status);
  const cudaStream_t st = static_cast<cudaStream_t>(w->stream);
  auto go = [&](auto from_rows, auto from_planes, int warp_heads) {
    const int rounds = (w->nh + 2 * kv.nkv + 8 * warp_heads - 1) / (8 * warp_heads);
    cudaError_t e;
    if (w->planes != nullptr) {
      e = launch_pdl(from_planes, dim3(w->M, w->M < 2 * sm_count() ? rounds : 1), dim3(256), 0, st,
                     static_cast<const float*>(w->planes), w->n_planes, static_cast<const __half*>(w->bias), to, positions, slots,
                     freqs, w->rotary_dim, kv.block_size, num_slots, status);
    } else {
      // as many tokens a CTA as its threads have angles, while three CTAs an SM are left; few tokens: a CTA per 256 threads' worth of heads
      int tokens = 1;
      while (tokens < 16 && tokens * 2 * std::max(w->rotary_dim / 2, 1) <= 256 && w->M / (tokens * 2) >= 3 * sm_count()) tokens *= 2;
      e = launch_pdl(from_rows, dim3((w->M + tokens - 1) / tokens, w->M < 2 * sm_count() ? rounds : 1), dim3(256), 0, st,
                     static_cast<const __half*>(w->qkv), w->ld, to, positions, slots, freqs, w->M, tokens, w->rotary_dim,
                     kv.block_size, num_slots, status);
    }
    return e == cudaSuccess ? 1 : ZSE_ERR_LAUNCH;
  };
  switch (kv.hd) {
    case 64: return go(rope_kv_write_q8_kernel<64>, rope_kv_write_q8_planes_kernel<64>, kWarpHeads<64>);
    case 96: return go(rope_kv_write_q8_kernel<96>, rope_kv_write_q8_planes_kernel<96>, kWarpHeads<96>);
    case 128: return go(rope_kv_write_q8_kernel<128>, rope_kv_write_q8_planes_kernel<128>, kWarpHeads<128>);
    default: return go(rope_kv_write_q8_kernel<256>, rope_kv_write_q8_planes_kernel<256>, kWarpHeads<256>);
  }
}

extern "C" int zse_kv_read_q8(const ZseReadQ8* r) {
  const ZseKvQ8& kv = r->kv;
  if (r->num_seqs <= 0) return 0;
  if (!cache_ok(kv) || r->max_blocks < 0 || r->out_blocks < 0 || r->out_max_blocks < 0) return ZSE_ERR_SHAPE;
  if (!aligned16(kv.data) || !aligned16(kv.scale) || !aligned16(r->out)) return ZSE_ERR_ALIGN;
  // five CTAs an SM fit; pages in parts of 1024 pieces or more where there are fewer pages than that
  const long long entries = ((long long)r->num_seqs * r->out_max_blocks + 255) / 256, room = (long long)sm_count() * 5;
  const long long pieces = 2ll * kv.nkv * kv.block_size * kv.hd / 8;
  if (pieces * 8 > 0x7fffffffll) return ZSE_ERR_LIMIT;
  const int parts = int(std::max(1ll, std::min((16 * room + r->out_blocks - 1) / std::max(r->out_blocks, 1), pieces / 1024)));
  const int grid = int(std::max(1ll, std::min(room, std::max((long long)r->out_blocks * parts, entries))));
  auto go = [&](auto kernel) {
    return launch_pdl(kernel, dim3(grid), dim3(256), 0, static_cast<cudaStream_t>(r->stream), static_cast<const uint8_t*>(kv.data),
                      static_cast<const float*>(kv.scale), kv.num_blocks, kv.nkv, kv.block_size,
                      static_cast<const int*>(r->tables), r->table_ld, r->max_blocks, static_cast<const int*>(r->seq_lens),
                      static_cast<const int*>(r->cu_blocks), r->num_seqs, static_cast<__half*>(r->out), r->out_blocks,
                      static_cast<int*>(r->out_tables), r->out_table_ld, r->out_max_blocks, parts,
                      static_cast<Status*>(r->status)) == cudaSuccess
               ? 1
               : ZSE_ERR_LAUNCH;
  };
  switch (kv.hd) {
    case 64: return go(kv_read_q8_kernel<64>);
    case 96: return go(kv_read_q8_kernel<96>);
    case 128: return go(kv_read_q8_kernel<128>);
    default: return go(kv_read_q8_kernel<256>);
  }
}
