// Attention of new tokens (one, or a few, of every sequence) over the 8-bit KV cache.
//
//   s[t][c] = scale * kscale[t] * (sum_d q[c][d] (uk[t][d] - 128)),   o[c][d] = sum_t p[t][c] vscale[t] (uv[t][d] - 128) / sum_t p[t][c]
//
// An item is one kv head of one sequence with up to 8 * NB columns c: query heads of the group, times rows of a draft.  Its tokens are
// cut into pieces, one per CTA; four warps of a CTA take every fourth tile of 16 tokens through rings of their own (cp.async) and
// keep a running maximum, sum and output in registers.  Tokens are the 16 rows of the products, columns their 8 columns.
//
// The pieces of an item are a thread-block cluster: its CTAs put what they have into shared memory and every CTA adds up a share
// of the result from all of them.  No scratch, no second kernel, nothing that two calls could share.  Only where a cluster of 16
// per item leaves most of the GPU idle (few sequences of few kv heads) are there several clusters per item, which meet in scratch.
//
// Bytes become fp16 numbers by byte permutations alone.  Keys: a byte in the low half of an fp16 number is u * 2^-24 (subnormal numbers
// are exact in the products), so a product sum that starts at -2^-17 sum(q) ends at 2^-24 (q . (uk - 128)): half an instruction per
// element.  Values: 0x64 above the byte makes 1024 + u, and a packed subtraction of 1152 the
// exact u - 128; with the subnormal form the weights' sum times 128 would cancel against a result that can be a thousand times smaller.
// Values come as pairs of dimensions of one token out of ldmatrix.trans, so the two rows of a thread are neighbouring dimensions.
#include <algorithm>

#include "api.h"
#include "common.cuh"
#include "typed.cuh"

namespace zse {

namespace {

constexpr int kWarps = 4;
constexpr int kStages = 3;
constexpr int kMostCluster = 16;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kNone = -1e30f;                          // below every score, finite so that no difference is not a number

struct Q8Args {
  const uint8_t* data;
  const float* scale;
  const __half* q;
  const int *tables, *seq_lens, *cu_q, *q_pos0;
  __half* out;
  float* scratch;
  Status* st;
  int ldq, ldo, q_rows, num_blocks, nkv, bpt, bpt_shift, table_ld, max_blocks, group, group_inv, max_q, rows_per, row_groups, window,
      pieces, cluster;
  float scale_log2;
};
// c / group for columns and c < 64: group_inv = ceil(2^16 / group)
__device__ __forceinline__ int row_of(const Q8Args& a, int c) { return (c * a.group_inv) >> 16; }
__device__ __noinline__ void complain(Status* st, unsigned where, unsigned detail) { report(st, kBadArgument, where, detail); }

__device__ __forceinline__ void mma_f16(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t turn_8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ uint32_t minus_1152(uint32_t x) {           // both halves
  uint32_t y;
  asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(y) : "r"(x), "r"(0x64806480u));
  return y;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t in_cta(uint32_t smem_addr, int rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_addr), "r"(rank));
  return r;
}
__device__ __forceinline__ float4 load_cluster4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ float load_cluster(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}

// Where 16-byte chunk c of a tile's row lies: any eight rows of one chunk are in eight different groups of four banks.  Written so
// that a thread's places follow from one of them by constants: copy j of a lane (chunk j * 32 + lane of the tile) and step kk of the
// matrix loads (chunks 2 kk, 2 kk + 1) are an exclusive or and an addition away from copy 0 and step 0.
template <int HD>
__device__ __forceinline__ uint32_t place(int row, int c) {
  if constexpr (HD == 64) return row * 64 + ((c ^ ((row >> 1) & 3)) << 4);
  if constexpr (HD == 96) return row * 96 + ((c ^ ((row >> 2) & 1)) << 4);
  return row * HD + ((c ^ (row & 7)) << 4);
}
template <int HD>
__device__ __forceinline__ uint32_t copy_place(uint32_t first, int lane, int j) {
  if constexpr (HD == 96) return first + place<96>((j * 32 + lane) / 6, (j * 32 + lane) % 6) - place<96>(lane / 6, lane % 6);
  if constexpr (HD == 128) return (first ^ (uint32_t(j & 1) << 6)) + j * 512;
  if constexpr (HD == 256) return (first ^ (uint32_t(j & 3) << 5)) + j * 512;
  return first + j * 512;
}
template <int HD>
__device__ __forceinline__ uint32_t step_place(uint32_t first, int kk) {
  if constexpr (HD == 96) return first + kk * 32;
  return first ^ (kk * 32);
}
__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ float load_shared(uint32_t addr) {
  float v;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}

template <int HD, int NB>
struct Q8Smem {
  static constexpr int kTile = 16 * HD;                                // K or V of 16 tokens
  static constexpr int kSlot = 2 * kTile + (HD == 256 ? 256 : 128);    // K, V, their scales
  static constexpr int kCols = 8 * NB;
  static constexpr int kPitch = HD + 4;                                // floats of a column of output
  static constexpr int kRing = kStages * kSlot > kCols * kPitch * 4 ? kStages * kSlot : kCols * kPitch * 4;   // of a warp
  static constexpr int kQPitch = HD * 2 + 32;                          // bytes: four columns in different groups of eight banks
  static constexpr bool kQShared = NB > 1;                             // queries in shared memory, or in registers
  static constexpr int kNumbers = kWarps * kRing;                      // own_m, own_l, own_ref, part_m, part_l
  static constexpr int kQ = kNumbers + ((kWarps + 1) * 2 * kCols + kWarps + 2 * kMostCluster * kCols) * 4;
  static constexpr int kTotal = kQ + (kQShared ? kCols * kQPitch : 0);
  static_assert(kQ % 16 == 0, "16-byte pieces");
};

template <int HD, int NB>
__global__ void __launch_bounds__(kWarps * 32, NB == 1 && HD <= 128 ? 4 : NB == 2 && HD <= 128 ? 3 : 1)
attn_q8_kernel(const Q8Args a) {
  using S = Q8Smem<HD, NB>;
  constexpr int kChunks = HD / 16;                                     // 16-byte chunks of a row, and 16-wide steps of the products
  constexpr int kChains = NB == 1 ? 2 : 1;                             // even and odd steps of a column apart
  extern __shared__ __align__(128) uint8_t smem[];
  float* own_m = reinterpret_cast<float*>(smem + S::kNumbers);         // [warp][column], then the CTA's
  float* own_l = own_m + (kWarps + 1) * S::kCols;
  float* own_ref = own_l + (kWarps + 1) * S::kCols;                    // [warp]
  pdl_launch_dependents();
  pdl_wait();
  // (what every CTA does once is kept short: with one tile per warp it is most of its instructions)
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t2 = (lane & 3) * 2;
  const int piece = blockIdx.x, s = blockIdx.z, kvh = a.row_groups == 1 ? blockIdx.y : blockIdx.y / a.row_groups;
  const int rg = blockIdx.y - kvh * a.row_groups, cap = a.max_blocks * a.bpt * 16;

  // rows of this item, and how many tokens its first row sees (each further row sees one more)
  int row0 = s, rows = 1, base_len;
  if (a.cu_q != nullptr) {
    const int first = a.cu_q[s], count = a.cu_q[s + 1] - first;
    row0 = first + rg * a.rows_per;
    rows = min(a.rows_per, count - rg * a.rows_per);
    base_len = a.q_pos0[s] + rg * a.rows_per + 1;
    if (count > 0 && (first < 0 || count > a.max_q || first + count > a.q_rows)) {
      if (tid == 0) complain(a.st, 73, s);
      rows = 0;
    }
  } else {
    base_len = a.seq_lens[s];
  }
  if (rows <= 0) return;                                               // the whole cluster
  if (base_len < (a.cu_q != nullptr ? 1 : 0) || base_len + rows - 1 > cap) {
    if (tid == 0) complain(a.st, 75, s);
    base_len = max(0, min(base_len, cap));
  }
  const int most_len = min(base_len + rows - 1, cap);
  const int first_tok = a.window > 0 ? max(0, base_len - a.window) : 0;
  const int last_first = a.window > 0 ? max(0, most_len - a.window) : 0;       // of the last row
  const int tile0 = first_tok >> 4, tiles = ((most_len + 15) >> 4) - tile0;
  const int per = unsigned(tiles + a.pieces - 1) / unsigned(a.pieces), lo = min(tiles, piece * per), hi = min(tiles, lo + per);
  const int mine = max(0, (hi - lo - warp + kWarps - 1) / kWarps);     // tiles lo + warp, lo + warp + 4, ...

  // places of the next 32 tiles in the cache, in units of 16 rows, one in every lane (-1: a hole)
  const int* table = a.tables + size_t(s) * a.table_ld;
  auto find = [&](int i0) {
    const int i = i0 + lane;
    int v = -1;
    if (i < mine) {
      const int tile = tile0 + lo + warp + i * kWarps, bi = a.bpt_shift >= 0 ? tile >> a.bpt_shift : tile / a.bpt;
      const int blk = table[bi];
      if (unsigned(blk) < unsigned(a.num_blocks)) v = (blk * 2 * a.nkv + kvh) * a.bpt + (tile - bi * a.bpt);
      else if (blk >= 0) complain(a.st, 76, blk);
    }
    return v;
  };
  const uint32_t ring = smem_u32(smem) + warp * S::kRing;
  int now = find(0), next = mine > 32 ? find(32) : -1;
  uint32_t holes = 0;                                                  // bit: ring slot whose tile is a hole
  const uint8_t* from = a.data + lane * 16;
  const uint32_t half = uint32_t(a.nkv * a.bpt) * S::kTile;            // from K to V of a page
  const float* from_scale = a.scale + (lane & 3) * 4 + (lane & 4 ? size_t(a.nkv * a.bpt) * 16 : 0);
  const uint32_t copy0 = place<HD>(lane / kChunks, lane % kChunks);
  auto issue = [&](int i, int slot) {                                  // always commits a group
    if (i < mine) {
      if ((i & 31) == 0 && i > 0) {
        now = next;
        next = find(i + 32);
      }
      const int at = __shfl_sync(0xffffffffu, now, i & 31);
      holes &= ~(1u << slot);
      if (at >= 0) {
        const uint32_t dst = ring + slot * S::kSlot;
        const uint8_t* k = from + size_t(uint32_t(at)) * S::kTile;
        const uint8_t* v = k + half;
#pragma unroll
        for (int j = 0; j < HD / 32; ++j) {
          const uint32_t to = copy_place<HD>(dst + copy0, lane, j);
          copy16(to, k + j * 512);
          copy16(to + S::kTile, v + j * 512);
        }
        if (lane < 8) copy16(dst + 2 * S::kTile + lane * 16, from_scale + size_t(uint32_t(at)) * 16);
      } else {
        holes |= 1u << slot;
      }
    }
    cpa_commit();
  };
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) issue(i, i);

  // queries, the B operand: column nb * 8 + g, dimensions 16 c + 4 (lane & 3) .. + 3 of a step; the order of the dimensions inside
  // a step is that of the keys' bytes
  uint32_t qb[S::kQShared ? 1 : kChunks][2];
  const uint8_t* qs = smem + S::kQ + g * S::kQPitch + t2 * 4;
  if constexpr (S::kQShared) {
    for (int i = tid; i < S::kCols * kChunks * 2; i += kWarps * 32) {
      const int c = i / (kChunks * 2), d = i % (kChunks * 2) * 8, r = row_of(a, c);
      uint4 v = make_uint4(0u, 0u, 0u, 0u);
      if (r < rows)
        v = *reinterpret_cast<const uint4*>(a.q + size_t(row0 + r) * a.ldq + size_t(kvh * a.group + c - r * a.group) * HD + d);
      *reinterpret_cast<uint4*>(smem + S::kQ + c * S::kQPitch + d * 2) = v;
    }
    __syncthreads();
  } else {
    const int r = row_of(a, g);
    const __half* src = a.q + size_t(row0 + r) * a.ldq + size_t(kvh * a.group + g - r * a.group) * HD + t2 * 2;
#pragma unroll
    for (int kk = 0; kk < kChunks; ++kk) {
      uint2 v = make_uint2(0u, 0u);
      if (r < rows) v = *reinterpret_cast<const uint2*>(src + kk * 16);
      qb[kk][0] = v.x;
      qb[kk][1] = v.y;
    }
  }
  auto query = [&](int nb, int kk) {
    if constexpr (S::kQShared) return *reinterpret_cast<const uint2*>(qs + nb * 8 * S::kQPitch + kk * 32);
    else return make_uint2(qb[kk][0], qb[kk][1]);
  };
  // -2^-17 times the sum over a query, of columns t2, t2 + 1: what the products start from, against the bytes' offset of 128
  float sum_q[NB][2];
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    const uint32_t ones[4] = {0x3C003C00u, 0x3C003C00u, 0x3C003C00u, 0x3C003C00u};
    float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int kk = 0; kk < kChunks; ++kk) {
      const uint2 x = query(nb, kk);
      mma_f16(sum, ones, x.x, x.y);
    }
    sum_q[nb][0] = sum[0] * -7.62939453125e-6f;
    sum_q[nb][1] = sum[1] * -7.62939453125e-6f;
  }

  // Weights are 2^(score - m): m is a score of the column that none so far exceeds by more than 6, so that it and what has been summed
  // change seldom (kNone: nothing seen).  ref: a power of two that no value's scale so far exceeds; o holds sums of weight * vscale /
  // ref, which fp16 takes.
  float o[NB][kChunks][4], m[NB][2], l[NB][2], ref = 0.f, inv_ref = 0.f;
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    m[nb][0] = m[nb][1] = kNone;
    l[nb][0] = l[nb][1] = 0.f;
#pragma unroll
    for (int d = 0; d < kChunks; ++d) o[nb][d][0] = o[nb][d][1] = o[nb][d][2] = o[nb][d][3] = 0.f;
  }
  const uint32_t step0 = place<HD>((lane >> 3 & 1) * 8 + (lane & 7), lane >> 4);
  int slot = 0;
#pragma unroll 1
  for (int i = 0; i < mine; ++i) {
    cpa_wait<kStages - 2>();
    __syncwarp();
    const bool hole = (holes >> slot) & 1u;
    issue(i + kStages - 1, slot == 0 ? kStages - 1 : slot - 1);        // the slot of the tile before this one
    const uint32_t at = ring + slot * S::kSlot, tile = at + step0, scales = at + 2 * S::kTile + g * 4;
    slot = slot + 1 == kStages ? 0 : slot + 1;
    if (hole) continue;
    const int tok = (tile0 + lo + warp + i * kWarps) << 4;
    const float k0 = load_shared(scales) * a.scale_log2, k1 = load_shared(scales + 32) * a.scale_log2;      // (with the 2^24 of the bytes)
    float w0 = load_shared(scales + 64), w1 = load_shared(scales + 96);
    float sc[NB][kChains][4];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        sc[nb][0][e] = sum_q[nb][e & 1];
        if (kChains > 1) sc[nb][kChains - 1][e] = 0.f;
      }
#pragma unroll
    for (int kk = 0; kk < kChunks / 2; ++kk) {
      uint32_t r[4];
      ldm_x4(step_place<HD>(tile, kk), r);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t f[4] = {__byte_perm(r[2 * h], 0u, 0x4140), __byte_perm(r[2 * h + 1], 0u, 0x4140),
                               __byte_perm(r[2 * h], 0u, 0x4342), __byte_perm(r[2 * h + 1], 0u, 0x4342)};
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
          const uint2 x = query(nb, kk * 2 + h);
          mma_f16(sc[nb][h & (kChains - 1)], f, x.x, x.y);
        }
      }
    }
    float t[NB][4];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (kChains > 1) sc[nb][0][e] += sc[nb][kChains - 1][e];
        t[nb][e] = fmaf(sc[nb][0][e], e < 2 ? k0 : k1, -m[nb][e & 1]);
      }
    uint32_t dead = 0;                                                 // bit nb * 4 + e: the column's row does not see the token
    if (tok + 16 > base_len || tok < last_first) {
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int len = min(base_len + row_of(a, nb * 8 + t2 + (e & 1)), cap), at_tok = tok + g + (e >> 1) * 8;
          if (at_tok >= len || (a.window > 0 && at_tok < len - a.window)) {
            dead |= 1u << (nb * 4 + e);
            t[nb][e] = -INFINITY;
          }
        }
      if (tok + g >= most_len) w0 = 0.f;                               // what lies behind the sequence may be anything
      if (tok + g + 8 >= most_len) w1 = 0.f;
    }
    bool over = fmaxf(w0, w1) > ref;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int e = 0; e < 4; ++e) over |= t[nb][e] > 6.f;
    if (__any_sync(0xffffffffu, over)) {
      // new references: the tile's maxima where they are above, and what has been summed scaled to them
      float wtop = fmaxf(fmaxf(w0, w1), 0.f);
#pragma unroll
      for (int sh = 4; sh < 32; sh <<= 1) wtop = fmaxf(wtop, __shfl_xor_sync(0xffffffffu, wtop, sh));
      float fade = 1.f;
      if (wtop > ref) {
        // the power of two above twice the scale, so that a slowly growing scale does not come here every time
        const float up = __uint_as_float(((__float_as_uint(fmaxf(wtop, 1e-30f)) >> 23) + 2u) << 23);
        inv_ref = 1.f / up;
        fade = ref * inv_ref;
        ref = up;
      }
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        float f[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float v0 = (dead >> (nb * 4 + e)) & 1u ? -INFINITY : sc[nb][0][e] * k0;
          const float v1 = (dead >> (nb * 4 + e + 2)) & 1u ? -INFINITY : sc[nb][0][e + 2] * k1;
          float x = fmaxf(v0, v1);
#pragma unroll
          for (int sh = 4; sh < 32; sh <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, sh));
          const float to = fmaxf(m[nb][e], x), drop = ex2(m[nb][e] - to);
          m[nb][e] = to;
          l[nb][e] *= drop;
          f[e] = drop * fade;
          t[nb][e] = v0 - to;
          t[nb][e + 2] = v1 - to;
        }
#pragma unroll
        for (int d = 0; d < kChunks; ++d) {
          o[nb][d][0] *= f[0];
          o[nb][d][1] *= f[1];
          o[nb][d][2] *= f[0];
          o[nb][d][3] *= f[1];
        }
      }
    }
    w0 *= inv_ref;
    w1 *= inv_ref;
    uint32_t pb[NB][2];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      float w[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float p = ex2(t[nb][e]);
        l[nb][e & 1] += p;
        w[e] = p * (e < 2 ? w0 : w1);
      }
      if (dead) {                                                      // (a weight of zero times a scale that is no number)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if ((dead >> (nb * 4 + e)) & 1u) w[e] = 0.f;
      }
      pb[nb][0] = turn_8x8(pack_half2(w[0], w[1]));                    // [token][column] -> [column][token], the B operand
      pb[nb][1] = turn_8x8(pack_half2(w[2], w[3]));
    }
#pragma unroll
    for (int dd = 0; dd < kChunks / 2; ++dd) {
      uint32_t r[4];
      ldm_x4_t(step_place<HD>(tile, dd) + S::kTile, r);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t f[4] = {minus_1152(__byte_perm(r[2 * h], 0x64646464u, 0x4240)), minus_1152(__byte_perm(r[2 * h], 0x64646464u, 0x4341)),
                               minus_1152(__byte_perm(r[2 * h + 1], 0x64646464u, 0x4240)),
                               minus_1152(__byte_perm(r[2 * h + 1], 0x64646464u, 0x4341))};
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) mma_f16(o[nb][dd * 2 + h], f, pb[nb][0], pb[nb][1]);
      }
    }
  }

  // ---- the warps' results side by side, in their rings
  cpa_wait<0>();
  __syncwarp();
  float* put = reinterpret_cast<float*>(smem + warp * S::kRing);
#pragma unroll
  for (int nb = 0; nb < NB; ++nb)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
#pragma unroll
      for (int sh = 4; sh < 32; sh <<= 1) l[nb][e] += __shfl_xor_sync(0xffffffffu, l[nb][e], sh);
      const int c = nb * 8 + t2 + e;
#pragma unroll
      for (int d = 0; d < kChunks; ++d)
        *reinterpret_cast<float2*>(put + c * S::kPitch + d * 16 + 2 * g) = make_float2(o[nb][d][e], o[nb][d][2 + e]);
      if (g == 0) {
        own_m[warp * S::kCols + c] = m[nb][e];
        own_l[warp * S::kCols + c] = l[nb][e];
      }
    }
  if (lane == 0) own_ref[warp] = ref;
  __syncthreads();
  const int cols = rows * a.group, item = (s * a.nkv + kvh) * a.row_groups + rg;
  constexpr int kQuads = HD / 4;
  auto finish = [&](int c, int d, const float4& acc, float top, float total) {
    const int r = row_of(a, c);
    if (a.pieces == a.cluster) {
      const float inv = total == 0.f ? 0.f : 1.f / total;              // nothing seen: zeros
      uint2 h = make_uint2(pack_half2(acc.x * inv, acc.y * inv), pack_half2(acc.z * inv, acc.w * inv));
      *reinterpret_cast<uint2*>(a.out + size_t(row0 + r) * a.ldo + size_t(kvh * a.group + c - r * a.group) * HD + d) = h;
    } else {
      float* to = a.scratch + ((size_t(item) * (a.pieces / a.cluster) + piece / a.cluster) * S::kCols + c) * (HD + 4);
      *reinterpret_cast<float4*>(to + d) = acc;
      if (d == 0) {
        to[HD] = top;
        to[HD + 1] = total;
      }
    }
  };
  for (int idx = tid; idx < cols * kQuads; idx += kWarps * 32) {
    const int c = idx / kQuads, d = (idx - c * kQuads) * 4;
    float top = kNone, total = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) top = fmaxf(top, own_m[w * S::kCols + c]);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float mw = own_m[w * S::kCols + c], f = ex2(mw - top);
      const float4 x = *reinterpret_cast<const float4*>(smem + w * S::kRing + (c * S::kPitch + d) * 4);
      total += own_l[w * S::kCols + c] * f;
      const float fo = f * own_ref[w];
      acc.x += x.x * fo;
      acc.y += x.y * fo;
      acc.z += x.z * fo;
      acc.w += x.w * fo;
    }
    if (a.cluster == 1) {
      finish(c, d, acc, top, total);
    } else {
      *reinterpret_cast<float4*>(smem + (c * S::kPitch + d) * 4) = acc;            // in place of the first warp's
      if (d == 0) {
        own_m[kWarps * S::kCols + c] = top;
        own_l[kWarps * S::kCols + c] = total;
      }
    }
  }
  if (a.cluster == 1) return;
  // Every CTA has a share of the elements and adds it up over the cluster.  A load from another CTA takes some 200 cycles, so they
  // go out together: first all references and sums of weights, then the results in batches.
  cluster_sync();
  const int rank = piece & (a.cluster - 1);
  const uint32_t base = smem_u32(smem), ma = smem_u32(own_m + kWarps * S::kCols), la = smem_u32(own_l + kWarps * S::kCols);
  float* part_m = own_ref + kWarps;                                    // [column][CTA]: factor of its result; sums of weights
  float* part_l = part_m + S::kCols * kMostCluster;
  for (int idx = tid; idx < cols * kMostCluster; idx += kWarps * 32) { // the CTAs of a column are neighbouring lanes
    const int c = idx / kMostCluster, w = idx % kMostCluster;
    const bool there = w < a.cluster;
    const float mw = there ? load_cluster(in_cta(ma + c * 4, w)) : kNone, lw = there ? load_cluster(in_cta(la + c * 4, w)) : 0.f;
    part_m[idx] = mw;
    part_l[idx] = lw;
  }
  __syncthreads();
  for (int idx = rank * kWarps * 32 + tid; idx < cols * kQuads; idx += a.cluster * kWarps * 32) {
    const int c = idx / kQuads, d = (idx - c * kQuads) * 4;
    float top = kNone, total = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kMostCluster; ++w) top = fmaxf(top, part_m[c * kMostCluster + w]);
#pragma unroll
    for (int w0 = 0; w0 < kMostCluster; w0 += 8) {
      if (w0 < a.cluster) {
        float4 x[8];
#pragma unroll
        for (int w = 0; w < 8; ++w) x[w] = load_cluster4(in_cta(base + (c * S::kPitch + d) * 4, min(w0 + w, a.cluster - 1)));
#pragma unroll
        for (int w = 0; w < 8; ++w) {
          const float mw = part_m[c * kMostCluster + w0 + w], f = ex2(mw - top);
          if (w0 + w < a.cluster) {
            total += part_l[c * kMostCluster + w0 + w] * f;
            acc.x += x[w].x * f;
            acc.y += x[w].y * f;
            acc.z += x[w].z * f;
            acc.w += x[w].w * f;
          }
        }
      }
    }
    finish(c, d, acc, top, total);
  }
  cluster_sync();                                                      // nobody leaves while others read its shared memory
}

// Joins the clusters of an item.  grid (kv heads * row groups, sequences), 128 threads.
template <int HD>
__global__ void __launch_bounds__(128)
attn_q8_join_kernel(const Q8Args a, int cols_kept) {
  pdl_launch_dependents();
  pdl_wait();
  const int s = blockIdx.y, item = s * gridDim.x + blockIdx.x, kvh = blockIdx.x / a.row_groups, rg = blockIdx.x - kvh * a.row_groups;
  const int G = a.group, clusters = a.pieces / a.cluster;
  int row0 = s, rows = 1;
  if (a.cu_q != nullptr) {
    const int first = a.cu_q[s], count = a.cu_q[s + 1] - first;
    row0 = first + rg * a.rows_per;
    rows = min(a.rows_per, count - rg * a.rows_per);
    if (first < 0 || count > a.max_q || first + count > a.q_rows) rows = 0;
  }
  for (int idx = threadIdx.x; idx < rows * G * (HD / 4); idx += 128) {
    const int c = idx / (HD / 4), d = (idx - c * (HD / 4)) * 4, r = row_of(a, c);
    const float* from = a.scratch + (size_t(item) * clusters * cols_kept + c) * (HD + 4);
    const size_t step = size_t(cols_kept) * (HD + 4);
    float top = kNone, total = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
    for (int w = 0; w < clusters; ++w) top = fmaxf(top, from[w * step + HD]);
#pragma unroll 4
    for (int w = 0; w < clusters; ++w) {
      const float mw = from[w * step + HD], f = ex2(mw - top);
      const float4 x = *reinterpret_cast<const float4*>(from + w * step + d);
      total += from[w * step + HD + 1] * f;
      acc.x += x.x * f;
      acc.y += x.y * f;
      acc.z += x.z * f;
      acc.w += x.w * f;
    }
    const float inv = total == 0.f ? 0.f : 1.f / total;
    *reinterpret_cast<uint2*>(a.out + size_t(row0 + r) * a.ldo + size_t(kvh * G + c - r * G) * HD + d) =
        make_uint2(pack_half2(acc.x * inv, acc.y * inv), pack_half2(acc.z * inv, acc.w * inv));
  }
}

int sm_count() {
  static int counts[kMaxDevices];
  const int slot = current_device_slot();
  if (counts[slot] == 0 && cudaDeviceGetAttribute(&counts[slot], cudaDevAttrMultiProcessorCount, slot) != cudaSuccess) return 148;
  return counts[slot];
}

struct Plan {
  int nb, rows_per, row_groups, pieces, cluster;
};
Plan plan_of(int num_seqs, int max_q, int nh, int nkv, int hd, int block_size, int max_blocks, int window, int num_splits) {
  Plan p;
  const int G = nh / nkv;
  p.nb = max_q * G <= 8 ? 1 : max_q * G <= 16 || hd > 128 ? 2 : 4;
  p.rows_per = std::max(1, 8 * p.nb / G);
  p.row_groups = (max_q + p.rows_per - 1) / p.rows_per;
  const long long items = (long long)num_seqs * nkv * p.row_groups;
  long long want = num_splits;
  if (num_splits <= 0) {
    long long tokens = (long long)max_blocks * block_size;
    if (window > 0) tokens = std::min(tokens, (long long)window + max_q + 16);
    const long long most = std::max(1ll, tokens / 64);                 // a tile for every warp of a piece
    want = std::min(most, (2ll * sm_count() + items - 1) / items);
  }
  if (want <= kMostCluster) {
    p.cluster = 1;
    while (p.cluster < want) p.cluster *= 2;
    p.pieces = p.cluster;
  } else {
    p.cluster = kMostCluster;
    p.pieces = int(std::min(64ll, (want + kMostCluster - 1) / kMostCluster) * kMostCluster);
  }
  return p;
}

template <int HD, int NB>
int launch(const Q8Args& a, int num_seqs, cudaStream_t st) {
  static bool ready[kMaxDevices];
  const int dev = current_device_slot();
  auto kernel = attn_q8_kernel<HD, NB>;
  constexpr int kBytes = Q8Smem<HD, NB>::kTotal;
  if (!ready[dev]) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kBytes) != cudaSuccess ||
        cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess)
      return ZSE_ERR_LAUNCH;
    ready[dev] = true;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(a.pieces, a.nkv * a.row_groups, num_seqs);
  cfg.blockDim = dim3(kWarps * 32);
  cfg.dynamicSmemBytes = kBytes;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (a.cluster > 1) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = a.cluster;
    attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
    ++n;
  }
  if (pdl_enabled()) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n].val.programmaticStreamSerializationAllowed = 1;
    ++n;
  }
  cfg.attrs = attr;
  cfg.numAttrs = n;
  if (cudaLaunchKernelEx(&cfg, kernel, a) != cudaSuccess) return ZSE_ERR_LAUNCH;
  if (a.pieces > a.cluster &&
      launch_pdl(attn_q8_join_kernel<HD>, dim3(a.nkv * a.row_groups, num_seqs), dim3(128), 0, st, a, 8 * NB) != cudaSuccess)
    return ZSE_ERR_LAUNCH;
  return 0;
}

}  // namespace
}  // namespace zse

using namespace zse;

extern "C" int zse_attn_decode_q8_pieces(int num_seqs, int max_q, int nh, int nkv, int hd, int block_size, int max_blocks, int window,
                                         int num_splits) {
  if (nkv <= 0 || nh < nkv || max_q <= 0 || num_seqs <= 0) return 1;
  return plan_of(num_seqs, max_q, nh, nkv, hd, block_size, max_blocks, window, num_splits).pieces;
}

extern "C" int64_t zse_attn_decode_q8_scratch_floats(int num_seqs, int max_q, int nh, int nkv, int hd, int block_size, int max_blocks,
                                                     int window, int num_splits) {
  if (nkv <= 0 || nh < nkv || max_q <= 0 || num_seqs <= 0) return 0;
  const Plan p = plan_of(num_seqs, max_q, nh, nkv, hd, block_size, max_blocks, window, num_splits);
  if (p.pieces == p.cluster) return 0;
  return int64_t(num_seqs) * nkv * p.row_groups * (p.pieces / p.cluster) * 8 * p.nb * (hd + 4);
}

extern "C" int zse_attn_decode_q8(const ZseKvQ8* kv, const void* q, int ldq, int q_rows, const void* tables, int table_ld, int max_blocks,
                                  const void* seq_lens, const void* cu_q, const void* q_pos0, int num_seqs, int max_q, void* out,
                                  int ldo, int nh, void* scratch, int64_t scratch_floats, int num_splits, float scale, int window,
                                  void* status, void* stream) {
  if (num_seqs <= 0 || max_q <= 0) return 0;
  const int bpt = kv->block_size / 16;
  if (kv->num_blocks <= 0 || kv->nkv <= 0 || kv->block_size <= 0 || kv->block_size % 16 || nh <= 0 || nh % kv->nkv ||
      nh / kv->nkv > 16 || max_blocks < 0 || max_q > 64 || (cu_q == nullptr && max_q != 1) ||
      (kv->hd != 64 && kv->hd != 96 && kv->hd != 128 && kv->hd != 256))
    return ZSE_ERR_SHAPE;
  if ((reinterpret_cast<uintptr_t>(kv->data) | reinterpret_cast<uintptr_t>(kv->scale) | reinterpret_cast<uintptr_t>(scratch) |
       reinterpret_cast<uintptr_t>(q)) & 15 || reinterpret_cast<uintptr_t>(out) & 7 || ldq % 8 || ldo % 4)
    return ZSE_ERR_ALIGN;
  const Plan p = plan_of(num_seqs, max_q, nh, kv->nkv, kv->hd, kv->block_size, max_blocks, window, num_splits);
  if (num_seqs > 65535 || (long long)kv->nkv * p.row_groups > 65535 || (long long)num_seqs * kv->nkv * p.row_groups > 0x7fffffffll ||
      (long long)kv->num_blocks * 2 * kv->nkv * bpt > 0x7fffffffll || (long long)max_blocks * kv->block_size > 0x7fffff00ll)
    return ZSE_ERR_LIMIT;
  if (p.pieces > p.cluster &&
      (scratch == nullptr || scratch_floats < (long long)num_seqs * kv->nkv * p.row_groups * (p.pieces / p.cluster) * 8 * p.nb * (kv->hd + 4)))
    return ZSE_ERR_LIMIT;
  const int group = nh / kv->nkv;
  int shift = 0;
  while ((1 << shift) < bpt) ++shift;
  const Q8Args a{static_cast<const uint8_t*>(kv->data), static_cast<const float*>(kv->scale), static_cast<const __half*>(q),
                 static_cast<const int*>(tables), static_cast<const int*>(seq_lens), static_cast<const int*>(cu_q),
                 static_cast<const int*>(q_pos0), static_cast<__half*>(out), static_cast<float*>(scratch),
                 static_cast<Status*>(status), ldq, ldo, q_rows, kv->num_blocks, kv->nkv, bpt, (1 << shift) == bpt ? shift : -1,
                 table_ld, max_blocks, group, (65536 + group - 1) / group, max_q, p.rows_per, p.row_groups, window, p.pieces,
                 p.cluster, scale * kLog2e * 16777216.f};
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
#define ZSE_Q8_WIDTH(HD) p.nb == 1 ? launch<HD, 1>(a, num_seqs, st) : p.nb == 2 ? launch<HD, 2>(a, num_seqs, st)
  switch (kv->hd) {
    case 64: return ZSE_Q8_WIDTH(64) : launch<64, 4>(a, num_seqs, st);
    case 96: return ZSE_Q8_WIDTH(96) : launch<96, 4>(a, num_seqs, st);
    case 128: return ZSE_Q8_WIDTH(128) : launch<128, 4>(a, num_seqs, st);
    default: return p.nb == 1 ? launch<256, 1>(a, num_seqs, st) : launch<256, 2>(a, num_seqs, st);
  }
#undef ZSE_Q8_WIDTH
}
