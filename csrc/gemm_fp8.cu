// Products of rows and weights in 8-bit floating point, a scale for each block of 128.
//
//   P[t, n] = sum_b sx[b, t] * sw[n / 128, b] * sum_{k in block b} x[t, k] * w[n, k]
//
// x, w e4m3, sx a scale per row and 128 columns, sw per 128 x 128 block.  The scales differ from block to block of k, so the inner sum of
// a block is a product by itself (four tcgen05.mma of 32 columns) in one of two TMEM accumulators, and the warps that own its rows add it,
// times both scales, to fp32 sums in their registers while the next block's product runs in the other.
//
// Two kernels.  For many tokens pairs of CTAs have the tokens on the TMEM lanes: a thread has one row, so both scales are one number of its own
// per block, the gated activation pairs columns of the same thread, and the largest number of a row's 128 outputs needs two threads.  For few
// tokens the weight rows lie on the lanes.
#include <type_traits>

#include "api.h"
#include "fp8.cuh"
#include "gemm_common.cuh"
#include "pair.cuh"

namespace zse {

namespace {

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

__device__ __forceinline__ void store32(void* p, const uint32_t* v) {
  asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]),
               "r"(v[6]), "r"(v[7])
               : "memory");
}
// y[0 .. 15] += the bias of columns n .. n + 15
__device__ __forceinline__ void add_bias(const Fp8Args& a, float* y, int n) {
  if (a.bias == nullptr) return;
#pragma unroll
  for (int j = 0; j < 16; ++j)
    if (n + j < a.N) y[j] += bias_of(a, n + j);
}
template <int TYPE>
__device__ __forceinline__ void put_one(const Fp8Args& a, float y, size_t at) {
  if (TYPE == kFp8F32) static_cast<float*>(a.out)[at] = y;
  else if (TYPE == kFp8BF16) static_cast<bf16*>(a.out)[at] = __float2bfloat16_rn(y);
  else static_cast<__half*>(a.out)[at] = __float2half_rn(hold_f16(y));
}
// f(the type as a constant): one branch a row of outputs, not one an output
template <typename F>
__device__ __forceinline__ void of_type(int type, F f) {
  if (type == kFp8F32) f(std::integral_constant<int, kFp8F32>());
  else if (type == kFp8BF16) f(std::integral_constant<int, kFp8BF16>());
  else f(std::integral_constant<int, kFp8F16>());
}
// Columns n .. n + C - 1 of a warp's 32 rows t - lane .. to memory, rounded to the output's type.  WIDE: the output, its rows and N are multiples of
// 32 bytes, a sector, which are written at a time; else sixteen columns of two rows at a time, by way of `stage`.  The whole warp calls it.
template <int C, bool WIDE, int TYPE>
__device__ __forceinline__ void put_rows(const Fp8Args& a, float* y, int t, int n, float (*stage)[17]) {
  if constexpr (WIDE) {
    const int item = TYPE == kFp8F32 ? 4 : 2;
    uint8_t* o = static_cast<uint8_t*>(a.out) + (size_t(min(t, a.M - 1)) * a.ldo + n) * item;
#pragma unroll
    for (int i = 0; i < C; i += 16) {
      if (n + i < a.N && t < a.M) {
        add_bias(a, y + i, n + i);
        if (TYPE == kFp8F32) {
          store32(o + i * 4, reinterpret_cast<const uint32_t*>(y + i));
          if (n + i + 8 < a.N) store32(o + i * 4 + 32, reinterpret_cast<const uint32_t*>(y + i + 8));
        } else {
          uint32_t v[8];
#pragma unroll
          for (int j = 0; j < 8; ++j)
            v[j] = TYPE == kFp8BF16 ? pack2<bf16>(y[i + 2 * j], y[i + 2 * j + 1]) : pack2<__half>(y[i + 2 * j], y[i + 2 * j + 1]);
          store32(o + i * 2, v);
        }
      }
    }
  } else {
    const int lane = threadIdx.x & 31, t0 = t - lane;
#pragma unroll
    for (int i = 0; i < C; i += 16) {
      add_bias(a, y + i, n + i);
      __syncwarp();
#pragma unroll
      for (int j = 0; j < 16; ++j) stage[lane][j] = y[i + j];
      __syncwarp();
      const int col = n + i + (lane & 15);
      of_type(a.type, [&](auto type) {
#pragma unroll
        for (int r = 0; r < 32; r += 2) {
          const int row = r + (lane >> 4);
          if (t0 + row < a.M && col < a.N) put_one<decltype(type)::value>(a, stage[row][lane & 15], size_t(t0 + row) * a.ldo + col);
        }
      });
    }
  }
}

// act(gate) * up of 64 neighbouring outputs of a row (acc: gates, then ups), the other 64 of their block in the thread of the other half.
// No branch an output: with one, each had to be done before the next began, 9000 cycles a unit instead of 1500 (4096 x 2 x 13824 x 5120 651 us
// instead of 594).
// `live` is false where the sums are not there; every warp of the barrier calls it.
__device__ __forceinline__ void put_gated(const Fp8Args& a, float* acc, int t, int n, int half, float (*tops)[128], int row, int barrier,
                                          int threads, bool live) {
  constexpr int O = 64;
  uint32_t top = 0;
  auto gate = [&](auto act) {
#pragma unroll
    for (int i = 0; i < O; ++i) {
      const float y = fp8_gated(decltype(act)::value, acc[i], acc[O + i]);
      acc[i] = n + (i & ~15) < a.N ? y : 0.f;
      top = max(top, abs_bits(acc[i]));
    }
  };
  if (a.act == kFp8Silu) gate(std::integral_constant<int, kFp8Silu>());
  else gate(std::integral_constant<int, kFp8Gelu>());
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

// ---- few tokens: weight rows on the lanes --------------------------------------------------------------------------------------------
// The product the other way around: 128 weight rows on the TMEM lanes, NT tokens as columns, so that a thread adds NT / 2 numbers a block
// whatever the rows are, and the weights, whose bytes are the time of such a pass, stream past once.  A step is two tiles of 128 x 128 weights:
// two blocks of K of the same rows, or (GLU) gate and up rows of one block.  Where there are fewer tiles of rows than SMs, the CTAs of a
// cluster have a part of K each and add their sums through distributed shared memory: each finishes a run of the tokens, from the parts in
// rank order.  Bound by the weights' bytes where there are many steps (5 tokens of 2 x 13824 x 5120 26 us, 5.4 TB/s), by the steps' handshakes with
// 64 columns (5120 x 13824 19.6 us, 3.7 TB/s), by the start and the cluster's three barriers with few (one token of 5120 x 5120 8.4 us).
template <int NT, bool GLU>
struct Few {
  static constexpr int kX = NT * 128, kW = 128 * 128;
  static constexpr int kStage = 2 * kW + (GLU ? 1 : 2) * kX;
  static constexpr int kBars = 8704;
  static constexpr int kRoom = (232448 - 1024 - kBars) / kStage, kStages = kRoom < 6 ? kRoom : 6;
  static constexpr int kBufs = NT <= 64 && kStages >= 4 ? 4 : 2;           // accumulators of two tiles
  static constexpr int kSmem = kStages * kStage + kBars + 1024;
  static_assert(kStages >= kBufs && 2 * NT * kBufs <= 512, "a stage's barrier stands for its accumulator too");
  static_assert((NT + 8) * 512 * (GLU ? 2 : 1) <= kStages * kStage, "the ring has room for the other CTAs' sums");
};

struct FewBars {
  uint64_t full[6], done[6], sc_full[6], sc_empty[6], acc_empty[4];
  uint32_t tmem_base;
  int abort_flag;
  float sw[6][2];
  alignas(16) float sx[6][2][128];
  float top[4][128];
};
static_assert(sizeof(FewBars) <= 8704, "barriers and scales fit their place");

__device__ __forceinline__ void tmem_ld8(uint32_t* r, uint32_t taddr) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(taddr)
               : "memory");
}
// four bytes of global memory to shared memory, and an arrival at `bar` when this thread's copies so far are there
__device__ __forceinline__ void copy4(void* to, const void* from) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(to)), "l"(from) : "memory");
}
__device__ __forceinline__ void copies_arrive(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}

struct FewUnits {
  int n_tiles, m_tiles, ks;                      // units: tiles of 128 rows x tiles of NT tokens; CTAs of a unit (= cluster size)
};

template <int NT, bool GLU>
__global__ void __launch_bounds__(384, 1)
gemm_fp8_few_kernel(const __grid_constant__ CUtensorMap tmap_x, const __grid_constant__ CUtensorMap tmap_w, const Fp8Args a, const FewUnits u) {
  using F = Few<NT, GLU>;
  constexpr int J = GLU ? 2 : 1, H = NT / 2;                   // sums of a thread: J x H
  extern __shared__ uint8_t smem_raw[];
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  float* red = reinterpret_cast<float*>(ring);                 // once all products of the cluster are done
  FewBars* bars = reinterpret_cast<FewBars*>(ring + F::kStages * F::kStage);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = int(blockIdx.x) % u.ks, first = int(blockIdx.x) / u.ks, stride = int(gridDim.x) / u.ks, n_units = u.n_tiles * u.m_tiles;
  const int n_kb = (a.K + kFp8Block - 1) / kFp8Block, steps = GLU ? n_kb : (n_kb + 1) / 2;
  const int s0 = int((long long)steps * rank / u.ks), s1 = int((long long)steps * (rank + 1) / u.ks);
  if (threadIdx.x == 0) {
    for (int i = 0; i < F::kStages; ++i) {
      mbar_init(&bars->full[i], 1);
      mbar_init(&bars->done[i], 1);
      mbar_init(&bars->sc_full[i], 32);
      mbar_init(&bars->sc_empty[i], 8);
    }
    for (int i = 0; i < F::kBufs; ++i) mbar_init(&bars->acc_empty[i], 8);
    bars->abort_flag = 0;
    mbar_fence_init();
    prefetch_tmap(&tmap_x);
    prefetch_tmap(&tmap_w);
  }
  if (warp == 1) {
    tmem_alloc(&bars->tmem_base, 2 * NT * F::kBufs);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  if (u.ks > 1) pair_cluster_sync();                           // every CTA of the cluster runs before anybody writes to it
  tc_fence_after_sync();
  const uint32_t tmem = bars->tmem_base;
  volatile int* abort_flag = &bars->abort_flag;
  pdl_launch_dependents();                                     // (the TMEM is ours: a dependent cannot take it first)

  if (warp == 0) {
    if (lane == 0) {
      pdl_wait();
      int s = 0, c = 0;
      uint32_t ph = 1;
      bool live = true;
      for (int i = first; i < n_units && live; i += stride) {
        for (int st = s0; st < s1; ++st, ++c) {
          if (c >= F::kStages && !mbar_wait(&bars->done[s], ph, abort_flag, a.status, 80, c)) {
            live = false;
            break;
          }
          mbar_arrive_expect_tx(&bars->full[s], F::kStage);
          uint8_t* to = ring + s * F::kStage;
          const int n0 = i / u.m_tiles * 128, t0 = i % u.m_tiles * NT, k = (GLU ? st : 2 * st) * kFp8Block;
          tma_load_2d(to, &tmap_w, k, n0, &bars->full[s]);
          tma_load_2d(to + F::kW, &tmap_w, GLU ? k : k + kFp8Block, GLU ? a.N + n0 : n0, &bars->full[s]);
          tma_load_2d(to + 2 * F::kW, &tmap_x, k, t0, &bars->full[s]);
          if (!GLU) tma_load_2d(to + 2 * F::kW + F::kX, &tmap_x, k + kFp8Block, t0, &bars->full[s]);
          if (++s == F::kStages) { s = 0; ph ^= 1; }
        }
      }
    }
  } else if (warp == 1) {
    constexpr uint32_t idesc = make_idesc_f16(128, NT);        // (format 0 of kind::f8f6f4 is e4m3)
    const uint64_t desc = make_desc_sw128(smem_u32(ring));
    int s = 0, c = 0;
    uint32_t ph = 0;
    bool live = true;
    for (int i = first; i < n_units && live; i += stride) {
      for (int st = s0; st < s1; ++st, ++c) {
        const int buf = c % F::kBufs;
        bool ok = mbar_wait_spin(&bars->full[s], ph, abort_flag, a.status, 82, c);
        ok = ok && (c < F::kBufs || mbar_wait_spin(&bars->acc_empty[buf], ((c / F::kBufs) & 1) ^ 1, abort_flag, a.status, 81, c));
        live = __all_sync(0xffffffffu, ok);
        if (!live) break;
        tc_fence_after_sync();
        const uint64_t dw = desc + uint64_t((s * F::kStage) >> 4), dx = dw + (2 * F::kW >> 4);
        if (elect_one()) {
#pragma unroll
          for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int k = 0; k < 4; ++k)
              umma_fp8(tmem + (buf * 2 + j) * NT, dw + ((j * F::kW) >> 4) + k * 2, dx + ((GLU ? 0 : j * F::kX) >> 4) + k * 2, idesc, k != 0);
          tc_commit(&bars->done[s]);
        }
        __syncwarp();
        if (++s == F::kStages) { s = 0; ph ^= 1; }
      }
    }
  } else if (warp == 2) {
    const int nbs = (a.N + kFp8Block - 1) / kFp8Block;
    int s = 0, c = 0;
    uint32_t ph = 1;
    bool live = true;
    pdl_wait();
    for (int i = first; i < n_units && live; i += stride) {
      const int nb = i / u.m_tiles, t0 = i % u.m_tiles * NT;
      for (int st = s0; st < s1; ++st, ++c) {
        live = c < F::kStages || __all_sync(0xffffffffu, mbar_wait(&bars->sc_empty[s], ph, abort_flag, a.status, 84, c));
        if (!live) break;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int k = GLU ? st : 2 * st + j;
          if (k < n_kb) {
            if (!GLU || j == 0)
#pragma unroll
              for (int l = 0; l < NT; l += 32)
                if (l + lane < NT) copy4(&bars->sx[s][j][l + lane], a.sx + size_t(k) * a.ld_sx + min(t0 + l + lane, a.M - 1));
            if (lane == 0) copy4(&bars->sw[s][j], a.sw + size_t(nb + (GLU ? j * nbs : 0)) * n_kb + k);
          }
        }
        copies_arrive(&bars->sc_full[s]);
        if (++s == F::kStages) { s = 0; ph ^= 1; }
      }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
  }

  const int q = warp & 3, half = (warp - 4) >> 2, row = q * 32 + lane;
  // one output's byte; `c`: the token's place in bars->top
  auto put_byte = [&](float y, int c, int n, int t) {
    uint32_t top = 0;
#pragma unroll
    for (int w = 0; w < 4; ++w) top = max(top, __float_as_uint(bars->top[w][c]));
    y = __fmul_rn(y, fp8_steps(__uint_as_float(top)));
    if (n < a.N) static_cast<uint8_t*>(a.out)[t * a.ldo + n] = __nv_cvt_float_to_fp8(y, __NV_SATFINITE, __NV_E4M3);
    if (row == 0) a.out_scale[(n / kFp8Block) * a.ld_os + t] = fp8_scale(__uint_as_float(top));
  };
  bool live = true;
  if (warp >= 4) {
    const uint32_t taddr = tmem + (uint32_t(q * 32) << 16) + half * H;
    int s = 0, c = 0;
    uint32_t ph = 0;
    pdl_wait();
    for (int i = first; i < n_units; i += stride) {
      float acc[J * H];
#pragma unroll
      for (int j = 0; j < J * H; ++j) acc[j] = 0.f;
      for (int st = s0; st < s1; ++st, ++c) {
        const int buf = c % F::kBufs;
        live = live && __all_sync(0xffffffffu, mbar_wait(&bars->sc_full[s], ph, abort_flag, a.status, 85, c) &&
                                                   mbar_wait(&bars->done[s], ph, abort_flag, a.status, 83, c));
        tc_fence_after_sync();
        constexpr int B = H < 16 ? 8 : 16, R = H < 32 ? H : 32;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          if (GLU || j == 0 || 2 * st + 1 < n_kb) {            // (uniform)
            const float w = bars->sw[s][j];
            float* sum = acc + (GLU ? j * H : 0);
#pragma unroll
            for (int l0 = 0; l0 < H; l0 += R) {
              uint32_t r[R / B][B];
#pragma unroll
              for (int l = 0; l < R; l += B) {
                if constexpr (B == 8) tmem_ld8(r[l / B], taddr + (buf * 2 + j) * NT + l0 + l);
                else ZSE_TMEM_LD_X16(r[l / B], taddr + (buf * 2 + j) * NT + l0 + l);
              }
              float f[R];
#pragma unroll
              for (int l = 0; l < R; l += 4) {
                const float4 x = *reinterpret_cast<const float4*>(&bars->sx[s][GLU ? 0 : j][half * H + l0 + l]);
                f[l] = x.x * w, f[l + 1] = x.y * w, f[l + 2] = x.z * w, f[l + 3] = x.w * w;
              }
              tc_wait_ld();
#pragma unroll
              for (int l = 0; l < R; ++l) {
                asm volatile("" : "+r"(r[l / B][l % B]));      // behind the wait
                sum[l0 + l] = fmaf(__uint_as_float(r[l / B][l % B]), f[l], sum[l0 + l]);
              }
            }
          }
        }
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&bars->acc_empty[buf]);
          mbar_arrive(&bars->sc_empty[s]);
        }
        if (++s == F::kStages) { s = 0; ph ^= 1; }
      }
      if (u.ks == 1) {
        const int n = i / u.m_tiles * 128 + row, t0 = i % u.m_tiles * NT + half * H;
        if constexpr (GLU) {
#pragma unroll
          for (int l = 0; l < H; ++l) {
            const float y = fp8_gated(a.act, acc[l], acc[H + l]);
            acc[l] = n < a.N ? y : 0.f;
            const uint32_t top = __reduce_max_sync(0xffffffffu, abs_bits(acc[l]));
            if (lane == 0) bars->top[q][half * H + l] = __uint_as_float(top);
          }
          asm volatile("bar.sync %0, 128;" ::"r"(1 + half) : "memory");
#pragma unroll
          for (int l = 0; l < H; ++l)
            if (live && t0 + l < a.M) put_byte(acc[l], half * H + l, n, t0 + l);
          asm volatile("bar.sync %0, 128;" ::"r"(1 + half) : "memory");    // before the next unit's
        } else if (live && n < a.N) {
          const float b = a.bias != nullptr ? bias_of(a, n) : 0.f;
          of_type(a.type, [&](auto type) {
#pragma unroll
            for (int l = 0; l < H; ++l)
              if (t0 + l < a.M) put_one<decltype(type)::value>(a, a.bias != nullptr ? acc[l] + b : acc[l], size_t(t0 + l) * a.ldo + n);
          });
        }
      } else {
        pair_cluster_sync();                                   // nothing is read from or loaded into a ring of the cluster any more
        // tokens owner * share .. of this thread's row go to the CTA `owner`
        const int share = (NT + u.ks - 1) / u.ks, there = min(NT, a.M - i % u.m_tiles * NT);
        const uint32_t mine = smem_u32(red + (rank * J * share) * 128 + row);
        int owner = half * H / share, slot = half * H - owner * share;
        uint32_t to = map_to_rank(mine, owner) + slot * 512;
#pragma unroll
        for (int l = 0; l < H; ++l) {
          if (half * H + l < there) {
#pragma unroll
            for (int j = 0; j < J; ++j)
              asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(to + j * share * 512), "f"(acc[j * H + l]) : "memory");
            to += 512;
            if (++slot == share) slot = 0, to = map_to_rank(mine, ++owner < u.ks ? owner : 0);
          }
        }
      }
    }
  }
  if (u.ks > 1) {                                              // one unit a cluster
    __syncwarp();
    if (warp < 4) pair_cluster_sync();
    pair_cluster_sync();
    if (warp >= 4) {
      const int share = (NT + u.ks - 1) / u.ks, n = first / u.m_tiles * 128 + row, t0 = first % u.m_tiles * NT + rank * share;
      const int mine = min(min(share, NT - rank * share), a.M - t0);          // tokens; the two halves of the warps take turns
      auto sum_of = [&](int j, int slot) {
        const float* from = red + (j * share + slot) * 128 + row;
        float sum = 0.f;
#pragma unroll 4
        for (int r = 0; r < u.ks; ++r) sum += from[r * J * share * 128];
        return sum;
      };
      if constexpr (GLU) {
        for (int i = half; i < mine; i += 2) {
          const float y = n < a.N ? fp8_gated(a.act, sum_of(0, i), sum_of(1, i)) : 0.f;
          red[i * 128 + row] = y;                              // (where this thread read its own part of the first sum)
          const uint32_t top = __reduce_max_sync(0xffffffffu, abs_bits(y));
          if (lane == 0) bars->top[q][i] = __uint_as_float(top);
        }
        asm volatile("bar.sync %0, 128;" ::"r"(1 + half) : "memory");
        for (int i = half; live && i < mine; i += 2) put_byte(red[i * 128 + row], i, n, t0 + i);
      } else if (live && n < a.N) {
        const float b = a.bias != nullptr ? bias_of(a, n) : 0.f;
        of_type(a.type, [&](auto type) {
#pragma unroll 4
          for (int i = half; i < mine; i += 2) {
            const float y = sum_of(0, i);
            put_one<decltype(type)::value>(a, a.bias != nullptr ? y + b : y, size_t(t0 + i) * a.ldo + n);
          }
        });
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
  if (warp == 1) tmem_dealloc(tmem, 2 * NT * F::kBufs);
}

// ---- many tokens: pairs of CTAs, persistent ------------------------------------------------------------------------------------------
// 256 tokens and 256 weight rows a pair (cta_group::2): a CTA has 128 of the tokens, loads those and half of the weight rows, and owns the
// sums of its tokens.  Bound by the way from a product to the next but one, 785 to 810 cycles a block where the product takes 512, and by the card's
// power (8192 x 5120 x 5120 190 us cold, 2260 TFLOP/s; 217 warm).  Units that do not fill a round of all pairs take a launch of their own with
// KS pairs a unit, clusters of 2 KS: each pair
// has a part of K, and the sums of 128 / KS rows go to each of the CTAs that have the same tokens.
constexpr int kPairThreads = 384;                // warp 0 loads, warp 1 issues the products, warps 4 .. 11 add them up
// Registers: 168 a thread at launch (64512), then 56 for the first four warps and 216 for the other eight (62464): 128 sums and two reads of 16
// columns do not fit 168.
constexpr int kPairStages = 6, kPairStage = 2 * 128 * 128;

struct Fp8PairBars {
  uint64_t full[kPairStages], done[kPairStages];   // done: a stage's products are complete: it may be filled again, its accumulator read
  uint64_t acc_empty[2];
  uint32_t tmem_base;
  int abort_flag;
  float stage[8][32][17];
  float top[2][2][128];                          // two units: a warp may be a unit ahead of the one that has the other 64 outputs
};

// Units (256 tokens x a tile of weight rows) in an order that keeps m_group token tiles in L2 while the weights stream past them once.
struct Fp8Units {
  int n_tiles, m_tiles, m_group, first, end;     // units first .. end - 1 belong to this launch
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

// WIDE: see put_rows (true for GLU); TYPE: of the output, where WIDE (its own kernel for each type: the sums come out 2 to 4 % faster).
template <bool GLU, int KS, bool WIDE, int TYPE>
__global__ void __launch_bounds__(kPairThreads, 1) __cluster_dims__(2 * KS, 1, 1)
gemm_fp8_pair_kernel(const __grid_constant__ CUtensorMap tmap_x, const __grid_constant__ CUtensorMap tmap_w, const Fp8Args a,
                     const Fp8Units units) {
  constexpr int kA = 128 * 128, C = 128;                       // C: columns of a thread
  extern __shared__ uint8_t smem_raw[];
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  Fp8PairBars* bars = reinterpret_cast<Fp8PairBars*>(ring + kPairStages * kPairStage);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint32_t rank;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  const uint32_t crank = rank & 1, leader = KS > 1 ? rank & ~1u : 0;       // of the pair
  const int part = KS > 1 ? int(rank >> 1) : 0;
  const int pair = units.first + int(blockIdx.x) / (2 * KS), workers = int(gridDim.x) / (2 * KS), n_units = units.end;
  const int all_kb = (a.K + kFp8Block - 1) / kFp8Block;
  const int kb0 = KS > 1 ? all_kb * part / KS : 0, n_kb = KS > 1 ? all_kb * (part + 1) / KS - kb0 : all_kb;
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
          const uint32_t full = map_to_rank(smem_u32(&bars->full[s]), leader);
          if (crank == 0) mbar_arrive_expect_tx(&bars->full[s], 2 * kPairStage);
          const uint32_t to = smem_u32(ring) + s * kPairStage;
          tma_load_2d_pair(to, &tmap_x, (kb0 + k) * kFp8Block, t0, full);
          if constexpr (GLU) {                                 // columns 0 .. 127 of the product: 64 gate rows and their up rows; the rest: the next
            const int g = n * 128 + int(crank) * 64;
            tma_load_2d_pair(to + kA, &tmap_w, (kb0 + k) * kFp8Block, g, full);
            tma_load_2d_pair(to + kA + 8192, &tmap_w, (kb0 + k) * kFp8Block, a.N + g, full);
          } else {
            tma_load_2d_pair(to + kA, &tmap_w, (kb0 + k) * kFp8Block, n * 256 + int(crank) * 128, full);
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
            tc_commit_pair(&bars->done[s], uint16_t(3u << leader));
          }
          __syncwarp();
          if (++s == kPairStages) { s = 0; ph ^= 1; }
        }
      }
    }
    if constexpr (KS > 1) {                                    // (the sums' two)
      __syncwarp();
      pair_cluster_sync();
      pair_cluster_sync();
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
    const int q = warp & 3, half = (warp - 4) >> 2, row = q * 32 + lane;
    const uint32_t taddr = tmem + (uint32_t(q * 32) << 16) + half * C;
    const uint32_t empty_bar = map_to_rank(smem_u32(&bars->acc_empty[0]), leader);
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
      const float* sw = a.sw + size_t(min(nb, nbs - 1)) * all_kb + kb0;
      const float* sw_up = GLU ? sw + size_t(nbs) * all_kb : sw;
      const float* sx = a.sx + size_t(kb0) * a.ld_sx + min(t, a.M - 1);
      float acc[C];
#pragma unroll
      for (int j = 0; j < C; ++j) acc[j] = 0.f;
      // One block.  Its rows' scale is in x, where that of the next but one is loaded when it has been used: it comes from the L2, which can take
      // longer than a block.  (Two blocks a turn of the loop, so that no register with a load under way is copied; from shared memory, which the
      // products keep busy, the scales took longer: 567 us instead of 536 for 8192 x 5120 x 13824, 595 with loads one block ahead.)
      float w32 = 0.f, u32 = 0.f;                              // weight scales of 32 blocks, one a lane
      auto block = [&](int k, float& x) {
        const float f = x * __shfl_sync(0xffffffffu, w32, k & 31), f_up = GLU ? x * __shfl_sync(0xffffffffu, u32, k & 31) : f;
        x = sx[size_t(min(k + 2, n_kb - 1)) * a.ld_sx];
        const int buf = c & 1;
        live = live && __all_sync(0xffffffffu, mbar_wait_spin(&bars->done[es], eph, abort_flag, a.status, 93, c));
        tc_fence_after_sync();
        add_block<C, GLU ? C / 2 : C>(acc, taddr + buf * 256, f, f_up);
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(empty_bar + buf * 8);
        if (++es == kPairStages) { es = 0; eph ^= 1; }
        ++c;
      };
      float x0 = sx[0], x1 = sx[size_t(min(1, n_kb - 1)) * a.ld_sx];
      for (int k0 = 0; k0 < n_kb; k0 += 32) {                  // (no way out of these loops but their end: with one, the sums were moved about)
        const int end = min(k0 + 32, n_kb);
        w32 = sw[min(k0 + lane, n_kb - 1)];
        if (GLU) u32 = sw_up[min(k0 + lane, n_kb - 1)];
        int k = k0;
        for (; k + 1 < end; k += 2) {
          block(k, x0);
          block(k + 1, x1);
        }
        if (k < end) block(k, x0);
      }
      if constexpr (KS > 1) {
        // 32 rows of a quarter go to the CTA `owner` of those with the same tokens, from the others in the order of their parts
        constexpr int kQuarters = 4 / KS;                      // of a CTA
        const int owner = q / kQuarters;
        auto place = [&](int src) { return smem_u32(ring) + ((src * kQuarters + q % kQuarters) * 2 + half) * 16384 + lane * 16; };
        pair_cluster_sync();                                   // nothing is read from or loaded into a ring of the cluster any more
        if (owner != part) {
          const uint32_t to = map_to_rank(place(part < owner ? part : part - 1), uint32_t(owner) * 2 + crank);
#pragma unroll
          for (int j = 0; j < C; j += 4)
            asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(to + j * 128), "f"(acc[j]), "f"(acc[j + 1]), "f"(acc[j + 2]),
                         "f"(acc[j + 3])
                         : "memory");
        }
        pair_cluster_sync();
        if (owner != part) continue;
#pragma unroll
        for (int src = 0; src < KS - 1; ++src) {
#pragma unroll
          for (int j = 0; j < C; j += 4) {
            float4 v;
            asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(place(src) + j * 128));
            acc[j] += v.x, acc[j + 1] += v.y, acc[j + 2] += v.z, acc[j + 3] += v.w;
          }
        }
      }
      if constexpr (GLU) {
        put_gated(a, acc, t, n * 128 + half * 64, half, bars->top[unit & 1], row, 1 + q, 64, live);
      } else if (live && n * 256 + half * C < a.N) {
        put_rows<C, WIDE, TYPE>(a, acc, t, n * 256 + half * C, bars->stage[WIDE ? 0 : warp - 4]);
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

struct Gpu {
  int slot, sms;                                               // of the current device
};

// Clusters of `ctas` CTAs of a kernel that run on the GPU at a time.
template <typename Kernel>
int clusters_at_a_time(Kernel kern, int ctas, int smem) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(384);
  cfg.dynamicSmemBytes = smem;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ctas, attr[0].val.clusterDim.y = 1, attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr, cfg.numAttrs = 1;
  int got = 0;
  return cudaOccupancyMaxActiveClusters(&got, kern, &cfg) == cudaSuccess ? got : 0;
}

constexpr int kPairSmem = kPairStages * kPairStage + int(sizeof(Fp8PairBars)) + 1024;

template <bool GLU, int KS, bool WIDE, int TYPE>
int pair_fit(const Gpu& gpu) {                                 // units of this form that run at a time
  static int fit[kMaxDevices];                                 // + 1
  int& n = fit[gpu.slot];
  if (n == 0) {
    auto kern = gemm_fp8_pair_kernel<GLU, KS, WIDE, TYPE>;
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kPairSmem) != cudaSuccess) return 0;
    n = 1 + (KS == 1 ? gpu.sms / 2 : clusters_at_a_time(kern, 2 * KS, kPairSmem));
  }
  return n - 1;
}

template <bool GLU, int KS, bool WIDE, int TYPE>
int launch_pair(const Gpu& gpu, const CUtensorMap& tx, const CUtensorMap& tw, const Fp8Args& a, Fp8Units u, int first, int end, cudaStream_t st) {
  if (first == end) return 0;
  const int fit = pair_fit<GLU, KS, WIDE, TYPE>(gpu);
  if (fit == 0) return ZSE_ERR_LAUNCH;
  u.first = first, u.end = end;
  const int clusters = KS == 1 ? std::min(fit, end - first) : end - first;
  return launch_pdl(gemm_fp8_pair_kernel<GLU, KS, WIDE, TYPE>, dim3(2 * KS * clusters), dim3(kPairThreads), kPairSmem, st, tx, tw, a, u) == cudaSuccess
             ? 1
             : ZSE_ERR_LAUNCH;
}

// ---- which kernel ------------------------------------------------------------------------------------------------------------------------
// Times in microseconds, from layers of 1 to 4096 tokens (those of gate and up weights in brackets).  A pair of CTAs takes 0.44 (0.6) a block of K
// whatever part of its 256 tokens there is, and 5 besides; the kernel for few tokens 0.6 a step with 16 token columns, 0.65 with 32, 0.78 (0.87)
// with 64 and 1.25 with 128 (gate and up weights: 1.9, which pairs beat), but not less than its weights take from memory, and 2 besides.  Sums over
// a cluster cost 3 or 4.  Both sides of the line, measured: 128 tokens of 5120 x 13824 29 us with 128 columns and 31 in pairs, 128 of 10240 x 8192 38
// and 32; 64 of 5120 x 13824 20 and 31, of 2 x 13824 x 5120 36 and 46, 128 70 and 49.
struct Fp8Plan {
  int nt;                                                      // token columns of the kernel for few tokens; 0: pairs
  int ks;                                                      // pairs: parts of K of the units behind the last whole round
  float us;
};
template <bool GLU>
Fp8Plan plan_pairs(const Gpu& gpu, int units, int n_kb) {
  const float kb = GLU ? 0.6f : 0.44f;
  const int at_once = std::max(1, pair_fit<GLU, 1, true, 0>(gpu)), rest = units % at_once;
  Fp8Plan p{0, 1, 5 + kb * n_kb * ((units + at_once - 1) / at_once)};
  if (rest == 0) return p;
  auto with = [&](int ks, int fit) {
    const float us = 5 + kb * n_kb * (units / at_once) + (units > rest ? 3 : 0) + 4 + kb * ((n_kb + ks - 1) / ks);
    if (rest <= fit && n_kb >= 4 * ks && us < p.us) p.ks = ks, p.us = us;
  };
  with(2, pair_fit<GLU, 2, true, 0>(gpu));
  with(4, pair_fit<GLU, 4, true, 0>(gpu));
  return p;
}

template <int NT, bool GLU>
int few_ready(const Gpu& gpu) {                                // 0, or an error
  static bool done[kMaxDevices];
  bool& d = done[gpu.slot];
  if (!d && cudaFuncSetAttribute(gemm_fp8_few_kernel<NT, GLU>, cudaFuncAttributeMaxDynamicSharedMemorySize, Few<NT, GLU>::kSmem) != cudaSuccess)
    return ZSE_ERR_LAUNCH;
  d = true;
  return 0;
}
// CTAs of a unit: as many as leave every one an SM of its own and a step of K.
template <int NT, bool GLU>
int few_splits(const Gpu& gpu, int units, int steps) {
  static int fit[kMaxDevices][9];                              // clusters of a size that run at a time, + 1
  if (few_ready<NT, GLU>(gpu)) return 1;
  for (int ks = std::min(std::min(8, steps), gpu.sms / std::max(units, 1)); ks > 1; --ks) {
    int& n = fit[gpu.slot][ks];
    if (n == 0) n = 1 + clusters_at_a_time(gemm_fp8_few_kernel<NT, GLU>, ks, Few<NT, GLU>::kSmem);
    if (units <= n - 1) return ks;
  }
  return 1;
}
template <int NT, bool GLU>
void plan_few(const Gpu& gpu, int M, int N, int n_kb, Fp8Plan* best) {
  if (M > 4 * NT) return;
  const int units = (N + 127) / 128 * ((M + NT - 1) / NT), steps = GLU ? n_kb : (n_kb + 1) / 2, ks = few_splits<NT, GLU>(gpu, units, steps);
  const float step = NT == 16 ? 0.6f : NT == 32 ? 0.65f : NT == 64 ? (GLU ? 0.87f : 0.78f) : 1.25f;
  const float us = 2 + (ks > 1 ? 3 : 0) + std::max(step * ((steps + ks - 1) / ks) * ((units + gpu.sms - 1) / gpu.sms), 2.f * N * n_kb * (GLU ? 1 : 0.5f) * 128 / 6e6f);
  if (us < best->us) *best = Fp8Plan{NT, ks, us};
}

template <int NT, bool GLU>
int launch_few(const Gpu& gpu, const ZseGemmFp8& g, const Fp8Args& a, int ks, cudaStream_t st) {
  using F = Few<NT, GLU>;
  if (int rc = few_ready<NT, GLU>(gpu)) return rc;
  CUtensorMap tx, tw;
  if (int rc = make_map(g.x, g.M, g.K, g.ldx, NT, &tx)) return rc;
  if (int rc = make_map(g.w, GLU ? 2ull * g.N : g.N, g.K, g.ldw, 128, &tw)) return rc;
  const FewUnits u{(g.N + 127) / 128, (g.M + NT - 1) / NT, ks};
  const int units = u.n_tiles * u.m_tiles;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ks > 1 ? units * ks : std::min(units, gpu.sms));
  cfg.blockDim = dim3(384);
  cfg.dynamicSmemBytes = F::kSmem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ks, attr[0].val.clusterDim.y = 1, attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_enabled() ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, gemm_fp8_few_kernel<NT, GLU>, tx, tw, a, u) == cudaSuccess ? 1 : ZSE_ERR_LAUNCH;
}

template <bool GLU, bool WIDE, int TYPE>
int run_pairs(const Gpu& gpu, const ZseGemmFp8& g, const Fp8Args& a, const Fp8Units& u, int units, int ks, cudaStream_t st) {
  CUtensorMap tx, tw;
  if (int rc = make_map(g.x, g.M, g.K, g.ldx, 128, &tx)) return rc;
  if (int rc = make_map(g.w, GLU ? 2ull * g.N : g.N, g.K, g.ldw, GLU ? 64 : 128, &tw)) return rc;
  const int whole = ks > 1 ? units - units % std::max(1, pair_fit<GLU, 1, WIDE, TYPE>(gpu)) : units;
  const int first = launch_pair<GLU, 1, WIDE, TYPE>(gpu, tx, tw, a, u, 0, whole, st);
  if (first < 0) return first;
  const int rest = ks == 4 ? launch_pair<GLU, 4, WIDE, TYPE>(gpu, tx, tw, a, u, whole, units, st) : launch_pair<GLU, 2, WIDE, TYPE>(gpu, tx, tw, a, u, whole, units, st);
  return rest < 0 ? rest : first + rest;
}

template <bool GLU>
int plan(const Gpu& gpu, const ZseGemmFp8& g, Fp8Units* u, int* units, Fp8Plan* p) {
  const int cols = GLU ? 128 : 256, m_tiles = (g.M + 255) / 256, n_tiles = (g.N + cols - 1) / cols, groups = (m_tiles + 7) / 8;
  const int n_kb = (g.K + kFp8Block - 1) / kFp8Block;
  if ((long long)m_tiles * n_tiles > 0x3fffffff) return ZSE_ERR_LIMIT;
  *u = Fp8Units{n_tiles, m_tiles, (m_tiles + groups - 1) / groups, 0, 0};      // about 2048 tokens at a time
  *units = m_tiles * n_tiles;
  *p = plan_pairs<GLU>(gpu, *units, n_kb);
  plan_few<16, GLU>(gpu, g.M, g.N, n_kb, p);
  plan_few<32, GLU>(gpu, g.M, g.N, n_kb, p);
  plan_few<64, GLU>(gpu, g.M, g.N, n_kb, p);
  if constexpr (!GLU) plan_few<128, GLU>(gpu, g.M, g.N, n_kb, p);
  return 0;
}

template <bool GLU>
int run(const ZseGemmFp8& g, const Fp8Args& a, cudaStream_t st) {
  const Gpu gpu{current_device_slot(), sm_count()};
  Fp8Units u;
  Fp8Plan p;
  int units;
  if (int rc = plan<GLU>(gpu, g, &u, &units, &p)) return rc;
  switch (p.nt) {
    case 16: return launch_few<16, GLU>(gpu, g, a, p.ks, st);
    case 32: return launch_few<32, GLU>(gpu, g, a, p.ks, st);
    case 64: return launch_few<64, GLU>(gpu, g, a, p.ks, st);
    case 128:
      if constexpr (!GLU) return launch_few<128, GLU>(gpu, g, a, p.ks, st);
  }
  const int item = a.type == kFp8F32 ? 4 : 2;
  if (GLU || ((reinterpret_cast<uintptr_t>(a.out) | size_t(a.ldo) * item | size_t(a.N) * item) & 31) == 0)
    return GLU || a.type == kFp8F16 ? run_pairs<GLU, true, kFp8F16>(gpu, g, a, u, units, p.ks, st)
           : a.type == kFp8BF16     ? run_pairs<GLU, true, GLU ? 0 : kFp8BF16>(gpu, g, a, u, units, p.ks, st)
                                    : run_pairs<GLU, true, GLU ? 0 : kFp8F32>(gpu, g, a, u, units, p.ks, st);
  return run_pairs<GLU, GLU, kFp8F16>(gpu, g, a, u, units, p.ks, st);
}

}  // namespace
}  // namespace zse

using namespace zse;

namespace {
int fp8_shape(const ZseGemmFp8* g) {
  const bool glu = g->act != kFp8None;
  return g->N <= 0 || g->K <= 0 || g->K % 16 || g->act < kFp8None || g->act > kFp8Gelu || g->type < kFp8F16 || g->type > kFp8F32 ||
                 g->bias_type < kFp8F16 || g->bias_type > kFp8F32 || (glu && (g->N % 16 || g->bias != nullptr))
             ? ZSE_ERR_SHAPE
         : g->M > kFp8Most || g->N > (glu ? kFp8Most / 2 : kFp8Most) || g->K > kFp8Most ? ZSE_ERR_LIMIT
                                                                                       : 0;
}
}  // namespace

extern "C" int zse_gemm_fp8_plan(const ZseGemmFp8* g, int32_t* tokens, int32_t* parts) {
  if (g->M <= 0) return ZSE_ERR_SHAPE;
  if (int rc = fp8_shape(g)) return rc;
  const Gpu gpu{current_device_slot(), sm_count()};
  Fp8Units u;
  Fp8Plan p;
  int units;
  if (int rc = g->act != kFp8None ? plan<true>(gpu, *g, &u, &units, &p) : plan<false>(gpu, *g, &u, &units, &p)) return rc;
  *tokens = p.nt;
  *parts = p.ks;
  return 0;
}

extern "C" int zse_gemm_fp8(const ZseGemmFp8* g) {
  if (g->M <= 0) return 0;
  if (int rc = fp8_shape(g)) return rc;
  const bool glu = g->act != kFp8None;
  if (glu && g->out_scale == nullptr) return ZSE_ERR_SHAPE;
  ZseGemmFp8 one = *g;                                         // (a single row may be any distance from the next)
  if (g->M == 1) one.ldx = g->K, one.ldo = g->N;
  if (!glu && g->N == 1) one.ldw = g->K;
  g = &one;
  const int item = glu ? 1 : g->type == kFp8F32 ? 4 : 2;
  auto aligned = [](const void* p, int bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; };
  if (!aligned(g->x, 16) || !aligned(g->w, 16) || g->ldx % 16 || g->ldw % 16 || !aligned(g->sx, 4) || !aligned(g->sw, 4) ||
      (glu ? !aligned(g->out, 16) || g->ldo % 16 : !aligned(g->out, item) || !aligned(g->bias, g->bias_type == kFp8F32 ? 4 : 2)))
    return ZSE_ERR_ALIGN;
  const long long n_kb = (g->K + kFp8Block - 1) / kFp8Block, nbs = (g->N + kFp8Block - 1) / kFp8Block, parts = glu ? 2 : 1;
  const Fp8Span written[] = {{g->out, (long long)g->N * item, g->ldo * item, g->M}, {glu ? g->out_scale : nullptr, g->M * 4ll, g->ld_os * 4, nbs}};
  const Fp8Span read[] = {{g->x, g->K, g->ldx, g->M}, {g->sx, g->M * 4ll, g->ld_sx * 4, n_kb}, {g->w, g->K, g->ldw, parts * g->N},
                          {g->sw, parts * nbs * n_kb * 4, 0, 1}, {g->bias, g->N * (g->bias_type == kFp8F32 ? 4ll : 2ll), 0, 1}};
  if (!written_apart(written, read)) return ZSE_ERR_SHAPE;
  const Fp8Args a{static_cast<const float*>(g->sx), static_cast<const float*>(g->sw), g->bias, g->out, static_cast<float*>(g->out_scale),
                  g->ldo, g->ld_sx, g->ld_os, g->M, g->N, g->K, g->type, g->bias_type, g->act, static_cast<Status*>(g->status)};
  const cudaStream_t st = static_cast<cudaStream_t>(g->stream);
  return glu ? run<true>(*g, a, st) : run<false>(*g, a, st);
}
