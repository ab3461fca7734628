// Products of rows and weights in 8-bit floating point, a scale for each block of 128.
//
//   P[t, n] = sum_b sx[b, t] * sw[n / 128, b] * sum_{k in block b} x[t, k] * w[n, k]
//
// x, w e4m3, sx a scale per row and 128 columns, sw per 128 x 128 block.  The scales differ from block to block of k, so the inner sum of
// a block is a product by itself (four tcgen05.mma of 32 columns) in one of two TMEM accumulators, and the warps that own its rows add it,
// times both scales, to fp32 sums in their registers while the next block's product runs in the other.
//
// Tokens lie on the TMEM lanes: a thread has one row, so both scales are one number of its own per block, the gated activation pairs columns
// of the same thread, and the largest number of a row's 128 outputs needs two threads.
#include "api.h"
#include "fp8.cuh"
#include "gemm_common.cuh"
#include "pair.cuh"

namespace zse {

namespace {

constexpr int kThreads = 320;                    // warp 0 loads, warp 1 issues the products, warps 2 .. 9 add them up
constexpr int kStageMax = 8;

struct Fp8Bars {
  uint64_t full[kStageMax], empty[kStageMax];
  uint64_t acc_full[2], acc_empty[2];
  uint32_t tmem_base;
  int abort_flag;
  float top[2][128];                             // largest of a row's 64 outputs, for the warps that have the other 64
};

struct Fp8Args {
  const float *sx, *sw;
  const void* bias;
  void* out;
  float* out_scale;
  long long ldo, ld_sx, ld_os;
  int M, N, K;                                   // N: output columns
  int type, bias_type, act;
  Status* status;
};

__device__ __forceinline__ void umma_fp8(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

__device__ __forceinline__ float bias_of(const Fp8Args& a, int n) {
  return a.bias_type == kFp8F32    ? static_cast<const float*>(a.bias)[n]
         : a.bias_type == kFp8BF16 ? to_f32(static_cast<const bf16*>(a.bias)[n])
                                   : __half2float(static_cast<const __half*>(a.bias)[n]);
}

__device__ __forceinline__ float gated(int act, float g, float u) { return act == kFp8Silu ? fp8_gated<kFp8Silu>(g, u) : fp8_gated<kFp8Gelu>(g, u); }

__device__ __forceinline__ void store32(void* p, const uint32_t* v) {
  asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]),
               "r"(v[6]), "r"(v[7])
               : "memory");
}
// The row's columns n .. n + C - 1 to memory, rounded to the output's type: 32 bytes, a sector, at a time where the row lies so.
template <int C>
__device__ __forceinline__ void put_row(const Fp8Args& a, float* y, int t, int n) {
  if (a.bias != nullptr) {
#pragma unroll
    for (int i = 0; i < C; ++i)
      if (n + i < a.N) y[i] += bias_of(a, n + i);
  }
  const size_t at = size_t(t) * a.ldo + n;
  const bool whole = n + C <= a.N;
  if (a.type == kFp8F32) {
    float* o = static_cast<float*>(a.out) + at;
    if (whole && (reinterpret_cast<uintptr_t>(o) & 31) == 0) {
#pragma unroll
      for (int i = 0; i < C; i += 8) store32(o + i, reinterpret_cast<const uint32_t*>(y + i));
    } else {
#pragma unroll
      for (int i = 0; i < C; ++i)
        if (n + i < a.N) o[i] = y[i];
    }
    return;
  }
  uint16_t* o = static_cast<uint16_t*>(a.out) + at;
  const bool wide = whole && (reinterpret_cast<uintptr_t>(o) & 31) == 0;
#pragma unroll
  for (int i = 0; i < C; i += 16) {
    uint32_t v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j)
      v[j] = a.type == kFp8BF16 ? pack2<bf16>(y[i + 2 * j], y[i + 2 * j + 1]) : pack2<__half>(y[i + 2 * j], y[i + 2 * j + 1]);
    if (wide) {
      store32(o + i, v);
    } else {
#pragma unroll
      for (int j = 0; j < 16; ++j)
        if (n + i + j < a.N) o[i + j] = uint16_t(v[j >> 1] >> (16 * (j & 1)));
    }
  }
}

// act(gate) * up of 64 neighbouring outputs of a row (acc: gates, then ups), the other 64 of their block in the thread of the other half.
// `live` is false where the sums are not there; every warp of the barrier calls it.
__device__ __forceinline__ void put_gated(const Fp8Args& a, float* acc, int t, int n, int half, float (*tops)[128], int row, int barrier,
                                          int threads, bool live) {
  constexpr int O = 64;
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < O; ++i) {
    acc[i] = n + i < a.N ? gated(a.act, acc[i], acc[O + i]) : 0.f;
    top = max(top, abs_bits(acc[i]));
  }
  tops[half][row] = __uint_as_float(top);
  asm volatile("bar.sync %0, %1;" ::"r"(barrier), "r"(threads) : "memory");
  top = max(top, __float_as_uint(tops[half ^ 1][row]));
  if (live && t < a.M) {
    const float steps = fp8_steps(__uint_as_float(top));
    uint8_t* o = static_cast<uint8_t*>(a.out) + t * a.ldo + n;
#pragma unroll
    for (int i = 0; i < O; i += 16)                            // (N is a multiple of 16)
      if (n + i < a.N)
        *reinterpret_cast<uint4*>(o + i) =
            make_uint4(fp8_pack4(acc + i, steps), fp8_pack4(acc + i + 4, steps), fp8_pack4(acc + i + 8, steps), fp8_pack4(acc + i + 12, steps));
    if (half == 0) a.out_scale[(n / kFp8Block) * a.ld_os + t] = fp8_scale(__uint_as_float(top));
  }
}

// Waits for the loads from TMEM; what they brought are operands, so that nothing that uses it moves before the wait.
__device__ __forceinline__ void tc_wait_ld16(uint32_t* r) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]),
                 "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])::"memory");
}
// acc += s (s_up from column SPLIT on) * the accumulator's columns: sixteen are read while the sixteen before are added.  (Packed pairs,
// fma.rn.f32x2, took longer: they have to be brought together first.)
template <int C, int SPLIT>
__device__ __forceinline__ void add_block(float* acc, uint32_t taddr, float s, float s_up) {
  uint32_t r[2][16];
  ZSE_TMEM_LD_X16(r[0], taddr);
#pragma unroll
  for (int c = 0; c < C; c += 16) {
    uint32_t* now = r[(c >> 4) & 1];
    tc_wait_ld16(now);
    if (c + 16 < C) ZSE_TMEM_LD_X16(r[((c >> 4) & 1) ^ 1], taddr + c + 16);
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[c + i] = fmaf(__uint_as_float(now[i]), c < SPLIT ? s : s_up, acc[c + i]);
  }
}

// A CTA has 128 tokens and NT weight rows (GLU: NT / 2 gate rows and their up rows, in runs of 64 that alternate).
template <int NT, bool GLU>
__global__ void __launch_bounds__(kThreads, 1)
gemm_fp8_kernel(const __grid_constant__ CUtensorMap tmap_x, const __grid_constant__ CUtensorMap tmap_w, const Fp8Args a) {
  constexpr int kA = 128 * 128, kB = NT * 128, kStages = NT == 256 ? 4 : 6;
  constexpr int C = NT / 2;                                    // columns of a thread
  extern __shared__ uint8_t smem_raw[];
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  Fp8Bars* bars = reinterpret_cast<Fp8Bars*>(ring + kStages * (kA + kB));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int t0 = blockIdx.y * 128, n_kb = (a.K + kFp8Block - 1) / kFp8Block;
  const int n0 = blockIdx.x * (GLU ? NT / 2 : NT);             // first output column
  const int quarters = min(4, (a.M - t0 + 31) / 32);           // warps of TMEM lanes that have a row
  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&bars->full[i], 1);
      mbar_init(&bars->empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bars->acc_full[i], 1);
      mbar_init(&bars->acc_empty[i], 2 * quarters);
    }
    bars->abort_flag = 0;
    mbar_fence_init();
    prefetch_tmap(&tmap_x);
    prefetch_tmap(&tmap_w);
  }
  if (warp == 1) {
    tmem_alloc(&bars->tmem_base, 2 * NT);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = bars->tmem_base;
  volatile int* abort_flag = &bars->abort_flag;
  pdl_launch_dependents();                                     // (the TMEM is ours: a dependent cannot take it first)

  if (warp == 0) {
    if (lane == 0) {
      pdl_wait();
      for (int k = 0; k < n_kb; ++k) {
        const int s = k % kStages;
        if (k >= kStages && !mbar_wait(&bars->empty[s], ((k / kStages) & 1) ^ 1, abort_flag, a.status, 80, k)) break;
        mbar_arrive_expect_tx(&bars->full[s], kA + kB);
        uint8_t* to = ring + s * (kA + kB);
        tma_load_2d(to, &tmap_x, k * kFp8Block, t0, &bars->full[s]);
        if constexpr (GLU) {
#pragma unroll
          for (int h = 0; h < NT / 128; ++h) {
            tma_load_2d(to + kA + h * 16384, &tmap_w, k * kFp8Block, n0 + h * 64, &bars->full[s]);
            tma_load_2d(to + kA + h * 16384 + 8192, &tmap_w, k * kFp8Block, a.N + n0 + h * 64, &bars->full[s]);
          }
        } else {
#pragma unroll
          for (int h = 0; h < NT / 64; ++h) tma_load_2d(to + kA + h * 8192, &tmap_w, k * kFp8Block, n0 + h * 64, &bars->full[s]);
        }
      }
    }
  } else if (warp == 1) {
    constexpr uint32_t idesc = make_idesc_f16(128, NT);        // (format 0 of kind::f8f6f4 is e4m3)
    const uint64_t desc = make_desc_sw128(smem_u32(ring));
    for (int k = 0; k < n_kb; ++k) {
      const int s = k % kStages, buf = k & 1;
      bool ok = k < 2 || mbar_wait_spin(&bars->acc_empty[buf], ((k >> 1) & 1) ^ 1, abort_flag, a.status, 81, k);
      ok = ok && mbar_wait_spin(&bars->full[s], (k / kStages) & 1, abort_flag, a.status, 82, k);
      if (!__all_sync(0xffffffffu, ok)) break;
      tc_fence_after_sync();
      const uint64_t da = desc + uint64_t((s * (kA + kB)) >> 4), db = da + (kA >> 4);
      if (elect_one()) {
#pragma unroll
        for (int j = 0; j < 4; ++j) umma_fp8(tmem + buf * NT, da + j * 2, db + j * 2, idesc, j != 0);
        tc_commit(&bars->empty[s]);
        tc_commit(&bars->acc_full[buf]);
      }
      __syncwarp();
    }
  } else {
    const int q = warp & 3, half = (warp - 2) >> 2, row = q * 32 + lane, t = t0 + row;
    if (q < quarters) {
      const uint32_t taddr = tmem + (uint32_t(q * 32) << 16) + half * C;
      pdl_wait();
      // the scales of this thread's columns: all of one block of weight rows, or (GLU) of a gate and an up block
      const int nb = (n0 + (GLU ? 0 : half * C)) / kFp8Block, nbs = (a.N + kFp8Block - 1) / kFp8Block;
      const float* sw = a.sw + size_t(min(nb, nbs - 1)) * n_kb;
      const float* sw_up = sw + size_t(nbs) * n_kb;
      const float* sx = a.sx + min(t, a.M - 1);
      float acc[C];
#pragma unroll
      for (int i = 0; i < C; ++i) acc[i] = 0.f;
      bool live = true;
      for (int k = 0; k < n_kb && live; ++k) {
        const float x = sx[size_t(k) * a.ld_sx], s = x * sw[k], s_up = GLU ? x * sw_up[k] : s;
        const int buf = k & 1;
        live = __all_sync(0xffffffffu, mbar_wait(&bars->acc_full[buf], (k >> 1) & 1, abort_flag, a.status, 83, k));
        if (!live) break;
        tc_fence_after_sync();
        add_block<C, GLU ? C / 2 : C>(acc, taddr + buf * NT, s, s_up);
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars->acc_empty[buf]);
      }
      if constexpr (GLU) {
        put_gated(a, acc, t, n0 + half * 64, half, bars->top, row, 1, 64 * quarters, live);
      } else if (live && t < a.M && n0 + half * C < a.N) {
        put_row<C>(a, acc, t, n0 + half * C);
      }
    }
  }
  __syncthreads();
  if (*abort_flag) {                                           // copies in flight must land before the CTA may leave
    const uint64_t began = globaltimer_ns();
    while (globaltimer_ns() - began < 1000000ull) {
    }
  }
  tc_fence_before_sync();
  __syncthreads();
  if (warp == 1) tmem_dealloc(tmem, 2 * NT);
}

// ---- many tokens: pairs of CTAs, persistent ------------------------------------------------------------------------------------------
// 256 tokens and NT weight rows a pair (cta_group::2): a CTA has 128 of the tokens, loads those and half of the weight rows, and owns the
// sums of its tokens.
constexpr int kPairThreads = 384;                // warp 0 loads, warp 1 issues the products, warps 4 .. 11 add them up
// Registers: 168 a thread at launch (64512), then 56 for the first four warps and 216 for the other eight (62464): 128 sums and two reads of 16
// columns do not fit 168.
constexpr int kPairStages = 6, kPairStage = 2 * 128 * 128;

struct Fp8PairBars {
  uint64_t full[kPairStages], done[kPairStages];   // done: a stage's products are complete: it may be filled again, its accumulator read
  uint64_t acc_empty[2];
  uint32_t tmem_base;
  int abort_flag;
  float top[2][2][128];                          // two units: a warp may be a unit ahead of the one that has the other 64 outputs
};

// Units (256 tokens x a tile of weight rows) in an order that keeps m_group token tiles in L2 while the weights stream past them once.
struct Fp8Units {
  int n_tiles, m_tiles, m_group;
  __device__ __forceinline__ void at(int i, int* n, int* m) const {
    const int g = i / (n_tiles * m_group), r = i - g * n_tiles * m_group, gm = min(m_group, m_tiles - g * m_group);
    *n = r / gm;
    *m = g * m_group + r % gm;
  }
};

__device__ __forceinline__ void umma_fp8_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

template <bool GLU>
__global__ void __launch_bounds__(kPairThreads, 1) __cluster_dims__(2, 1, 1)
gemm_fp8_pair_kernel(const __grid_constant__ CUtensorMap tmap_x, const __grid_constant__ CUtensorMap tmap_w, const Fp8Args a,
                     const Fp8Units units) {
  constexpr int kA = 128 * 128, C = 128;                       // C: columns of a thread
  extern __shared__ uint8_t smem_raw[];
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  Fp8PairBars* bars = reinterpret_cast<Fp8PairBars*>(ring + kPairStages * kPairStage);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint32_t crank;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(crank));
  const int pair = blockIdx.x >> 1, workers = gridDim.x >> 1, n_units = units.n_tiles * units.m_tiles;
  const int n_kb = (a.K + kFp8Block - 1) / kFp8Block;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kPairStages; ++i) {
      mbar_init(&bars->full[i], 1);
      mbar_init(&bars->done[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bars->acc_empty[i], 16);
    }
    bars->abort_flag = 0;
    mbar_fence_init();
    prefetch_tmap(&tmap_x);
    prefetch_tmap(&tmap_w);
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&bars->tmem_base)), "r"(512) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tc_fence_before_sync();
  __syncthreads();
  pair_cluster_sync();                                         // both CTAs' barriers exist before anybody signals them
  tc_fence_after_sync();
  const uint32_t tmem = bars->tmem_base;
  volatile int* abort_flag = &bars->abort_flag;
  pdl_launch_dependents();                                     // (the TMEM is ours: a dependent cannot take it first)

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
    if (warp == 0 && lane == 0) {
      pdl_wait();
      int s = 0, c = 0;
      uint32_t ph = 1;
      bool live = true;
      for (int i = pair; i < n_units && live; i += workers) {
        int n, m;
        units.at(i, &n, &m);
        const int t0 = m * 256 + int(crank) * 128;
        for (int k = 0; k < n_kb; ++k, ++c) {
          if (c >= kPairStages && !mbar_wait(&bars->done[s], ph, abort_flag, a.status, 90, c)) {
            live = false;
            break;
          }
          const uint32_t full = map_to_rank(smem_u32(&bars->full[s]), 0);
          if (crank == 0) mbar_arrive_expect_tx(&bars->full[s], 2 * kPairStage);
          const uint32_t to = smem_u32(ring) + s * kPairStage;
          tma_load_2d_pair(to, &tmap_x, k * kFp8Block, t0, full);
          if constexpr (GLU) {                                 // columns 0 .. 127 of the product: 64 gate rows and their up rows; the rest: the next
            const int g = n * 128 + int(crank) * 64;
            tma_load_2d_pair(to + kA, &tmap_w, k * kFp8Block, g, full);
            tma_load_2d_pair(to + kA + 8192, &tmap_w, k * kFp8Block, a.N + g, full);
          } else {
            tma_load_2d_pair(to + kA, &tmap_w, k * kFp8Block, n * 256 + int(crank) * 128, full);
          }
          if (++s == kPairStages) { s = 0; ph ^= 1; }
        }
      }
    } else if (warp == 1 && crank == 0) {
      constexpr uint32_t idesc = make_idesc_f16(256, 256);      // (format 0 of kind::f8f6f4 is e4m3)
      const uint64_t desc = make_desc_sw128(smem_u32(ring));
      int s = 0, c = 0;
      uint32_t ph = 0;
      bool live = true;
      for (int i = pair; i < n_units && live; i += workers) {
        for (int k = 0; k < n_kb; ++k, ++c) {
          const int buf = c & 1;
          bool ok = mbar_wait_cluster(&bars->full[s], ph, abort_flag, a.status, 92, c);
          ok = ok && (c < 2 || mbar_wait_cluster(&bars->acc_empty[buf], ((c >> 1) & 1) ^ 1, abort_flag, a.status, 91, c));
          live = __all_sync(0xffffffffu, ok);
          if (!live) break;
          tc_fence_after_sync();
          const uint64_t da = desc + uint64_t((s * kPairStage) >> 4), db = da + (kA >> 4);
          if (elect_one()) {
#pragma unroll
            for (int j = 0; j < 4; ++j) umma_fp8_pair(tmem + buf * 256, da + j * 2, db + j * 2, idesc, j != 0);
            tc_commit_pair(&bars->done[s]);
          }
          __syncwarp();
          if (++s == kPairStages) { s = 0; ph ^= 1; }
        }
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
    const int q = warp & 3, half = (warp - 4) >> 2, row = q * 32 + lane;
    const uint32_t taddr = tmem + (uint32_t(q * 32) << 16) + half * C;
    const uint32_t empty_bar = map_to_rank(smem_u32(&bars->acc_empty[0]), 0);
    const int nbs = (a.N + kFp8Block - 1) / kFp8Block;
    bool live = true;
    int c = 0, unit = 0, es = 0;
    uint32_t eph = 0;
    pdl_wait();
    for (int i = pair; i < n_units; i += workers, ++unit) {
      int n, m;
      units.at(i, &n, &m);
      const int t = m * 256 + int(crank) * 128 + row;
      const int nb = GLU ? n : (n * 256 + half * C) / kFp8Block;
      const float* sw = a.sw + size_t(min(nb, nbs - 1)) * n_kb;
      const float* sw_up = GLU ? sw + size_t(nbs) * n_kb : sw;
      const float* sx = a.sx + min(t, a.M - 1);
      float acc[C];
#pragma unroll
      for (int j = 0; j < C; ++j) acc[j] = 0.f;
      float x = sx[0], w = sw[0], w_up = sw_up[0];             // scales of a block are loaded while the one before is added
      for (int k = 0; k < n_kb; ++k, ++c) {
        const float f = x * w, f_up = GLU ? x * w_up : f;
        if (k + 1 < n_kb) {
          x = sx[size_t(k + 1) * a.ld_sx];
          w = sw[k + 1];
          if (GLU) w_up = sw_up[k + 1];
        }
        const int buf = c & 1;
        live = live && __all_sync(0xffffffffu, mbar_wait(&bars->done[es], eph, abort_flag, a.status, 93, c));
        tc_fence_after_sync();
        add_block<C, GLU ? C / 2 : C>(acc, taddr + buf * 256, f, f_up);
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(empty_bar + buf * 8);
        if (++es == kPairStages) { es = 0; eph ^= 1; }
      }
      if constexpr (GLU) {
        put_gated(a, acc, t, n * 128 + half * 64, half, bars->top[unit & 1], row, 1 + q, 64, live);
      } else if (live && t < a.M && n * 256 + half * C < a.N) {
        put_row<C>(a, acc, t, n * 256 + half * C);
      }
    }
  }
  __syncthreads();
  if (*abort_flag) {                                           // copies in flight must land before the CTA may leave
    const uint64_t began = globaltimer_ns();
    while (globaltimer_ns() - began < 1000000ull) {
    }
  }
  tc_fence_before_sync();
  __syncthreads();
  pair_cluster_sync();                                         // nobody leaves while the other CTA may still signal it
  if (warp == 1)
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
}

// e4m3 rows [rows, K], ld bytes apart: box = 128 columns x box_rows rows, 128-byte swizzle, zeros out of bounds
int make_map(const void* p, uint64_t rows, uint64_t K, uint64_t ld, uint32_t box_rows, CUtensorMap* out) {
  const EncodeTiledFn fn = encode_fn();
  if (fn == nullptr) return ZSE_ERR_DRIVER;
  const cuuint64_t dims[2] = {K, rows}, strides[1] = {ld};
  const cuuint32_t box[2] = {kFp8Block, box_rows}, each[2] = {1, 1};
  return fn(out, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(p), dims, strides, box, each, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS
             ? 0
             : ZSE_ERR_DRIVER;
}

template <int NT, bool GLU>
int launch(const ZseGemmFp8& g, const Fp8Args& a, cudaStream_t st) {
  CUtensorMap tx, tw;
  if (int rc = make_map(g.x, g.M, g.K, g.ldx, 128, &tx)) return rc;
  if (int rc = make_map(g.w, GLU ? 2ull * g.N : g.N, g.K, g.ldw, 64, &tw)) return rc;
  constexpr int smem = (NT == 256 ? 4 : 6) * (128 + NT) * 128 + int(sizeof(Fp8Bars)) + 1024;
  auto kern = gemm_fp8_kernel<NT, GLU>;
  static bool attr_done[kMaxDevices] = {};
  const int dev = current_device_slot();
  if (!attr_done[dev]) {
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess) return ZSE_ERR_LAUNCH;
    attr_done[dev] = true;
  }
  const int cols = GLU ? NT / 2 : NT;
  return launch_pdl(kern, dim3((g.N + cols - 1) / cols, (g.M + 127) / 128), dim3(kThreads), smem, st, tx, tw, a) == cudaSuccess ? 1 : ZSE_ERR_LAUNCH;
}

template <bool GLU>
int launch_pair(const ZseGemmFp8& g, const Fp8Args& a, cudaStream_t st) {
  CUtensorMap tx, tw;
  if (int rc = make_map(g.x, g.M, g.K, g.ldx, 128, &tx)) return rc;
  if (int rc = make_map(g.w, GLU ? 2ull * g.N : g.N, g.K, g.ldw, GLU ? 64 : 128, &tw)) return rc;
  constexpr int smem = kPairStages * kPairStage + int(sizeof(Fp8PairBars)) + 1024;
  auto kern = gemm_fp8_pair_kernel<GLU>;
  static bool attr_done[kMaxDevices] = {};
  const int dev = current_device_slot();
  if (!attr_done[dev]) {
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess) return ZSE_ERR_LAUNCH;
    attr_done[dev] = true;
  }
  const int cols = GLU ? 128 : 256, m_tiles = (g.M + 255) / 256, n_tiles = (g.N + cols - 1) / cols, groups = (m_tiles + 7) / 8;
  const Fp8Units u{n_tiles, m_tiles, (m_tiles + groups - 1) / groups};        // about 2048 tokens at a time
  const int pairs = std::min<long long>(sm_count() / 2, (long long)n_tiles * m_tiles);
  return launch_pdl(kern, dim3(2 * pairs), dim3(kPairThreads), smem, st, tx, tw, a, u) == cudaSuccess ? 1 : ZSE_ERR_LAUNCH;
}

}  // namespace
}  // namespace zse

using namespace zse;

extern "C" int zse_gemm_fp8(const ZseGemmFp8* g) {
  if (g->M <= 0) return 0;
  const bool glu = g->act != kFp8None;
  if (g->N <= 0 || g->K <= 0 || g->K % 16 || g->act < kFp8None || g->act > kFp8Gelu || g->type < kFp8F16 || g->type > kFp8F32 ||
      g->bias_type < kFp8F16 || g->bias_type > kFp8F32 || (glu && (g->N % 16 || g->bias != nullptr || g->out_scale == nullptr)))
    return ZSE_ERR_SHAPE;
  if (g->M > 65535 * 128) return ZSE_ERR_LIMIT;
  auto aligned = [](const void* p, int bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; };
  if (!aligned(g->x, 16) || !aligned(g->w, 16) || g->ldx % 16 || g->ldw % 16 || !aligned(g->sx, 4) || !aligned(g->sw, 4) ||
      (glu ? !aligned(g->out, 16) || g->ldo % 16 : !aligned(g->out, g->type == kFp8F32 ? 4 : 2)))
    return ZSE_ERR_ALIGN;
  const Fp8Args a{static_cast<const float*>(g->sx), static_cast<const float*>(g->sw), g->bias, g->out, static_cast<float*>(g->out_scale),
                  g->ldo, g->ld_sx, g->ld_os, g->M, g->N, g->K, g->type, g->bias_type, g->act, static_cast<Status*>(g->status)};
  const cudaStream_t st = static_cast<cudaStream_t>(g->stream);
  if (g->M > 256) return glu ? launch_pair<true>(*g, a, st) : launch_pair<false>(*g, a, st);
  return glu ? launch<256, true>(*g, a, st) : launch<128, false>(*g, a, st);
}
