// Attention of new tokens (one, or a few, of every sequence) over the 8-bit KV cache.
//
//   s[t][c] = scale * kscale[t] * (sum_d q[c][d] (uk[t][d] - 128)),   o[c][d] = sum_t p[t][c] vscale[t] (uv[t][d] - 128) / sum_t p[t][c]
//
// An item is one kv head of one sequence with up to 16 columns c: query heads of the group, times rows of a draft.  More rows are more
// items, which read the keys and values again, from L2: with 32 columns a warp needs 240 registers, and 32 drafts of up to five rows of
// 40 heads over 2001 to 4094 tokens took 78 us instead of 66 (both with weights of one fp16 number, see below).  An item's tokens are
// cut into pieces, one per CTA; four warps of a CTA take every fourth tile of 16 tokens through rings of their own (cp.async) and keep
// running references, sums and outputs in registers.  Tokens are the 16 rows of the products, columns their 8 columns.
//
// Up to eight pieces of an item are a thread-block cluster: every CTA stores what it has into the shared memory of the CTAs that add it
// up, each a share of the elements.  No scratch, no second kernel, nothing that two calls could share.  Only where eight pieces per item
// leave most of the GPU idle (few long sequences of few kv heads) are there several clusters per item, which meet in scratch.
//
// Bytes become fp16 numbers by byte permutations.  Keys: a byte in the low half of an fp16 number is u * 2^-24 (subnormal numbers are
// exact in the products), so a sum that starts at -2^-17 sum(q) ends at 2^-24 (q . (uk - 128)): half an instruction per element.
// Values: 0x64 above the byte makes 1024 + u, and a packed subtraction of 1152 the exact u - 128; in the subnormal form 128 times the
// weights' sum would cancel against a result that can be a thousand times smaller.  Values come as pairs of dimensions of one token out
// of ldmatrix.trans, so the two rows of a thread are neighbouring dimensions.
//
// Weights go into the products as two fp16 numbers, rounded and what that leaves: with the first alone results were off by 3.0e-4 of
// themselves (2-norm), with both by the 2.1e-4 of their own rounding to fp16.  Up to four columns have the second numbers in the four
// that would be idle; else they are products more (a product of 16 x 8 x 16 keeps a quarter of an SM busy for some 8 cycles: the drafts
// 66 -> 77 us, 64 sequences of 128 to 2300 tokens of 40 heads 35.7 -> 38.2; longest first, as by_length() has them, 70 and 35).
//
// What bounds it: the cache's bytes where there are many of them (64 sequences of 6001 to 8190 tokens, 64 heads over 8: in a CUDA graph
// 148 us, 6.5 TB/s, the rate of a plain copy; in calls one by one 168 us, 5.8 TB/s); mixed lengths leave SMs idle at the end (128 to 2300
// tokens: 4.8 TB/s); drafts the products (71 us, of which 34 are product time); few short sequences the way length -> table -> tile ->
// merge (1 x 300 tokens of 28 heads over 4: 4.1 us).
#include <algorithm>

#include "api.h"
#include "common.cuh"
#include "typed.cuh"

namespace zse {

namespace {

constexpr int kWarps = 4;
constexpr int kStages = 3;
constexpr int kMostCluster = 8;
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
      pieces, cluster, sort;                                           // sort: sequences, to be taken the longest first (0: as they come)
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
__device__ __forceinline__ float lg2(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Barrier of the cluster in two halves: the relaxed form only says that a CTA has got there, the other one orders its writes.
__device__ __forceinline__ void cluster_arrive_relaxed() { asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ uint32_t in_cta(uint32_t smem_addr, int rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_addr), "r"(rank));
  return r;
}
__device__ __forceinline__ void store_cluster4(uint32_t addr, const float4& v) {
  asm volatile("st.shared::cluster.v4.f32 [%0], {%1,%2,%3,%4};" ::"r"(addr), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w) : "memory");
}
__device__ __forceinline__ void store_cluster2(uint32_t addr, float x, float y) {
  asm volatile("st.shared::cluster.v2.f32 [%0], {%1,%2};" ::"r"(addr), "f"(x), "f"(y) : "memory");
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

// The z-th longest of the (at most 64) sequences.  Items are handed to the SMs in the order of the grid: the longest first, every SM
// gets one of each size: with two pieces each, 64 sequences of 128 to 2300 tokens took 36.5 us and take 35.0, of 6001 to 8190 151 and 146.
__device__ __forceinline__ int by_length(const Q8Args& a, int z) {
  const int lane = threadIdx.x & 31;
  int key[2], rank[2] = {0, 0};
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int i = k * 32 + lane;
    key[k] = -1;
    if (i < a.sort) {
      const int len = a.cu_q != nullptr ? a.q_pos0[i] + (a.cu_q[i + 1] - a.cu_q[i]) : a.seq_lens[i];
      key[k] = (min(max(a.window > 0 ? min(len, a.window) : len, 0), (1 << 28) - 1) >> 4) * 64 + 63 - i;   // (no two alike)
    }
  }
#pragma unroll 8
  for (int j = 0; j < 32; ++j) {
    const int u = __shfl_sync(0xffffffffu, key[0], j), v = __shfl_sync(0xffffffffu, key[1], j);
#pragma unroll
    for (int k = 0; k < 2; ++k) rank[k] += (u > key[k]) + (v > key[k]);
  }
  const uint32_t low = __ballot_sync(0xffffffffu, key[0] >= 0 && rank[0] == z), high = __ballot_sync(0xffffffffu, key[1] >= 0 && rank[1] == z);
  return low != 0 ? __ffs(low) - 1 : __ffs(high) + 31;
}

constexpr int kQ8SmemAlign = 256;                                      // of the dynamic shared memory
template <int HD, int NB>
struct Q8Smem {
  static constexpr int kTile = 16 * HD;                                // K or V of 16 tokens
  static constexpr int kSlot = 2 * kTile + (HD == 256 ? 256 : 128);    // K, V, their scales
  static constexpr int kCols = 8 * NB;
  static constexpr int kPitch = HD + 4;                                // floats of a column of output
  static constexpr int kRing = kStages * kSlot > kCols * kPitch * 4 ? kStages * kSlot : kCols * kPitch * 4;   // of a warp
  static constexpr int kQPitch = HD * 2 + 32;                          // bytes: four columns in different groups of eight banks
  static constexpr bool kQShared = NB > 1;                             // queries in shared memory, or in registers
  static constexpr int kNumbers = kWarps * kRing;                      // own_m, own_l [warp][column]
  static constexpr int kGot = kNumbers + 2 * kWarps * kCols * 4;       // references and sums, [CTA][column][2]
  static constexpr int kGotO = kGot + 2 * kMostCluster * kCols * 4;                    // results, [CTA][its share here] of 16 bytes
  static constexpr int kQ = kGotO + (kCols * HD / 4 + kMostCluster) * 16;
  static constexpr int kTotal = kQ + (kQShared ? kCols * kQPitch : 0);
  static_assert(kGot % 16 == 0 && kGotO % 16 == 0 && kQ % 16 == 0, "16-byte pieces");
  // copy_place() and step_place() turn bits of whole shared addresses over, up to bit 7 for rows of 256 bytes and bit 6 for the others:
  // tiles begin where those bits are zero
  static constexpr int kAlign = HD == 256 ? 256 : 128;
  static_assert(kAlign <= kQ8SmemAlign && kTile % kAlign == 0 && kSlot % kAlign == 0 && kRing % kAlign == 0, "places of a tile");
};

// PACKED: up to four columns; they stand a second time in columns 4 .. 7, where the weights are what rounding leaves of the first.
template <int HD, int NB, bool PACKED>
__global__ void __launch_bounds__(kWarps * 32, HD > 128 ? 1 : NB == 1 || HD == 64 ? 4 : 3)
attn_q8_kernel(const Q8Args a) {
  using S = Q8Smem<HD, NB>;
  constexpr int kChunks = HD / 16;                                     // 16-byte chunks of a row, and 16-wide steps of the products
  constexpr int kChains = NB == 1 ? 2 : 1;                             // even and odd steps of a column apart
  extern __shared__ __align__(kQ8SmemAlign) uint8_t smem[];
  float* own_m = reinterpret_cast<float*>(smem + S::kNumbers);         // [warp][column]
  float* own_l = own_m + kWarps * S::kCols;
  pdl_launch_dependents();
  pdl_wait();
  // (what every CTA does once is kept short: with one tile per warp it is most of its instructions)
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t2 = (lane & 3) * 2;
  const int piece = blockIdx.x, s = a.sort > 0 ? by_length(a, blockIdx.z) : blockIdx.z;
  const int kvh = a.row_groups == 1 ? blockIdx.y : blockIdx.y / a.row_groups;
  const int rg = blockIdx.y - kvh * a.row_groups, cap = a.max_blocks * a.bpt * 16;

  // A warp's tile i is 4 (i * pieces + piece) + warp of the item: pieces are equally long, and without a window where the first tiles
  // lie is known before the length (the entries are loaded beside it, and used if the sequence is that long).
  const int* table = a.tables + size_t(s) * a.table_ld;
  const int stride = a.pieces * kWarps, ahead = piece * kWarps + warp + lane * stride;
  int early = -1;
  if (a.window == 0 && lane < 4 && ahead < a.max_blocks * a.bpt) early = table[a.bpt_shift >= 0 ? ahead >> a.bpt_shift : ahead / a.bpt];

  // rows of this item, and how many tokens its first row sees (each further row sees one more)
  int row0 = s, rows = 1, base_len;
  if (a.cu_q != nullptr) {
    const int first = a.cu_q[s], count = a.cu_q[s + 1] - first;
    row0 = first + rg * a.rows_per;
    rows = min(a.rows_per, count - rg * a.rows_per);
    base_len = min(a.q_pos0[s], 0x7fffff7f) + rg * a.rows_per + 1;     // (no sum of these overflows, and that is above every cap)
    if (count <= 0 || first < 0 || count > a.max_q || first + count > a.q_rows) {
      if (tid == 0 && count > 0) complain(a.st, 73, s);
      rows = 0;
    }
  } else {
    base_len = a.seq_lens[s];
  }
  if (rows <= 0) return;                                               // the whole cluster
  if (base_len < (a.cu_q != nullptr ? 1 : 0) || base_len > cap - (rows - 1)) {
    if (tid == 0) complain(a.st, 75, s);
    base_len = max(0, min(base_len, cap));
  }
  const int most_len = min(base_len + rows - 1, cap);
  const int first_tok = a.window > 0 ? max(0, base_len - a.window) : 0;
  const int last_first = a.window > 0 ? max(0, most_len - a.window) : 0;       // of the last row
  const int tile0 = first_tok >> 4, tiles = ((most_len + 15) >> 4) - tile0;
  const int first_tile = piece * kWarps + warp, mine = first_tile < tiles ? unsigned(tiles - first_tile - 1) / unsigned(stride) + 1 : 0;
  if (a.cluster > 1) cluster_arrive_relaxed();                         // (waited for before another CTA's memory is written)

  // places of the next 32 tiles in the cache, in units of 16 rows, one in every lane (-1: a hole)
  auto find = [&](int i0) {
    const int i = i0 + lane;
    int v = -1;
    if (i < mine) {
      const int tile = tile0 + first_tile + i * stride, bi = a.bpt_shift >= 0 ? tile >> a.bpt_shift : tile / a.bpt;
      const int blk = i < 4 && a.window == 0 ? early : table[bi];
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
    const int c = PACKED ? g & 3 : g, r = row_of(a, c);
    const __half* src = a.q + size_t(row0 + r) * a.ldq + size_t(kvh * a.group + c - r * a.group) * HD + t2 * 2;
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

  // Weights are 2^(score - m), and what goes into the products is weight * vscale, in fp16: so m, one for every column, is what makes the
  // largest of those 64 when it is set, and it and what has been summed change only where one comes out above 2^14 (kNone: nothing seen).
  // With the largest score and the largest vscale apart, a token of large values and little weight takes the others' bits (values 10^6
  // times the others': results off by a fifth).  Weights are at most 2^40 then, however small the values: below that fp16 has zero for
  // the result.
  constexpr float kMost = 16384.f, kMostSum = 1e27f;
  float o[NB][kChunks][4], m[NB][2], l[NB][2];
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
    const int tok = (tile0 + first_tile + i * stride) << 4;
    const float k0 = load_shared(scales) * a.scale_log2, k1 = load_shared(scales + 32) * a.scale_log2;      // (with the 2^24 of the bytes)
    const float w0 = load_shared(scales + 64), w1 = load_shared(scales + 96);
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
          const int c = PACKED ? (t2 & 2) + (e & 1) : nb * 8 + t2 + (e & 1);
          // (a column of no row sees nothing: a large value behind the sequence would move the references of them all)
          const int r = row_of(a, c), len = r < rows ? min(base_len + r, cap) : 0, at_tok = tok + g + (e >> 1) * 8;
          if (at_tok >= len || (a.window > 0 && at_tok < len - a.window)) {
            dead |= 1u << (nb * 4 + e);
            t[nb][e] = -INFINITY;
          }
        }
    }
    float w[NB][4], sum[NB][2];
    bool over = false;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float p0 = ex2(t[nb][e]), p1 = ex2(t[nb][e + 2]);
        w[nb][e] = p0 * w0;
        w[nb][e + 2] = p1 * w1;
        sum[nb][e] = l[nb][e] + (p0 + p1);
        over |= fmaxf(w[nb][e], w[nb][e + 2]) > kMost || sum[nb][e] > kMostSum;
      }
    if (__any_sync(0xffffffffu, over)) {
      // new references, where the tile's are above, and what has been summed scaled to them
      const float log0 = lg2(w0), log1 = lg2(w1);
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        float f[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float v0 = (dead >> (nb * 4 + e)) & 1u ? -INFINITY : sc[nb][0][e] * k0;
          const float v1 = (dead >> (nb * 4 + e + 2)) & 1u ? -INFINITY : sc[nb][0][e + 2] * k1;
          float to = fmaxf(fmaxf(v0, v1) - 40.f, fmaxf(v0 + log0, v1 + log1) - 6.f);   // (fmaxf passes over what is no number)
#pragma unroll
          for (int sh = 4; sh < 32; sh <<= 1) to = fmaxf(to, __shfl_xor_sync(0xffffffffu, to, sh));
          to = fmaxf(m[nb][e], to);
          f[e] = ex2(m[nb][e] - to);
          m[nb][e] = to;
          const float p0 = ex2(v0 - to), p1 = ex2(v1 - to);
          w[nb][e] = p0 * w0;
          w[nb][e + 2] = p1 * w1;
          sum[nb][e] = l[nb][e] * f[e] + (p0 + p1);
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
    uint32_t pb[NB][2], rest[NB][2];                                   // tokens 0..7 and 8..15, [column][token]: the B operand
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      l[nb][0] = sum[nb][0];
      l[nb][1] = sum[nb][1];
      if (dead) {                                                      // (a weight of zero times a scale that is no number)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if ((dead >> (nb * 4 + e)) & 1u) w[nb][e] = 0.f;
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t x = pack_half2(w[nb][2 * h], w[nb][2 * h + 1]);
        const float2 back = __half22float2(*reinterpret_cast<const __half2*>(&x));
        const uint32_t y = pack_half2(w[nb][2 * h] - back.x, w[nb][2 * h + 1] - back.y);
        pb[nb][h] = turn_8x8(PACKED && t2 >= 4 ? y : x);
        rest[nb][h] = PACKED ? 0u : turn_8x8(y);
      }
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
        if constexpr (!PACKED) {
#pragma unroll
          for (int nb = 0; nb < NB; ++nb) mma_f16(o[nb][dd * 2 + h], f, rest[nb][0], rest[nb][1]);
        }
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
        *reinterpret_cast<float2*>(to + HD) = make_float2(top, total);
      }
    }
  };
  const int rank = piece & (a.cluster - 1), shift = 31 - __clz(a.cluster), share = (cols * kQuads + a.cluster - 1) >> shift;
  const uint32_t got = smem_u32(smem) + S::kGot, got_o = smem_u32(smem) + S::kGotO;
  if (a.cluster > 1) cluster_wait();                                   // all CTAs of the cluster run
  for (int idx = tid; idx < cols * kQuads; idx += kWarps * 32) {
    const int c = idx / kQuads, d = (idx - c * kQuads) * 4;
    float top = kNone, total = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) top = fmaxf(top, own_m[w * S::kCols + c]);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float f = ex2(own_m[w * S::kCols + c] - top);
      float4 x = *reinterpret_cast<const float4*>(smem + w * S::kRing + (c * S::kPitch + d) * 4);
      if constexpr (PACKED) {
        const float4 y = *reinterpret_cast<const float4*>(smem + w * S::kRing + ((c + 4) * S::kPitch + d) * 4);
        x = make_float4(x.x + y.x, x.y + y.y, x.z + y.z, x.w + y.w);
      }
      total += own_l[w * S::kCols + c] * f;
      acc.x += x.x * f;
      acc.y += x.y * f;
      acc.z += x.z * f;
      acc.w += x.w * f;
    }
    if (a.cluster == 1) {
      finish(c, d, acc, top, total);
    } else {
      // to the CTA that adds up this element: every cluster-th is its own
      const uint32_t to = in_cta(got_o + ((rank * share) + (idx >> shift)) * 16, idx & (a.cluster - 1));
      store_cluster4(to, acc);
      if (d == 0)
        for (int w = 0; w < a.cluster; ++w) store_cluster2(in_cta(got + (rank * S::kCols + c) * 8, w), top, total);
    }
  }
  if (a.cluster == 1) return;
  cluster_arrive();
  cluster_wait();                                                      // nobody writes here any more, and nobody leaves before
  const float2* numbers = reinterpret_cast<const float2*>(smem + S::kGot);
  const float4* parts = reinterpret_cast<const float4*>(smem + S::kGotO);
  for (int at = tid; at * a.cluster + rank < cols * kQuads; at += kWarps * 32) {
    const int idx = at * a.cluster + rank, c = idx / kQuads, d = (idx - c * kQuads) * 4;
    float top = kNone, total = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kMostCluster; ++w)
      if (w < a.cluster) top = fmaxf(top, numbers[w * S::kCols + c].x);
#pragma unroll
    for (int w = 0; w < kMostCluster; ++w)
      if (w < a.cluster) {
        const float2 n = numbers[w * S::kCols + c];
        const float4 x = parts[w * share + at];
        const float f = ex2(n.x - top);
        total += n.y * f;
        acc.x += x.x * f;
        acc.y += x.y * f;
        acc.z += x.z * f;
        acc.w += x.w * f;
      }
    finish(c, d, acc, top, total);
  }
}

// Joins the clusters of an item.  grid (kv heads * row groups, sequences, columns), 128 threads: kGroups of them share a piece of a
// column, each takes every kGroups-th cluster.
template <int HD>
__global__ void __launch_bounds__(128)
attn_q8_join_kernel(const Q8Args a, int cols_kept) {
  pdl_launch_dependents();
  pdl_wait();
  constexpr int kQuads = HD / 4, kGroups = 128 / kQuads;
  __shared__ float4 part[kGroups][kQuads];
  __shared__ float2 number[kGroups];
  const int s = blockIdx.y, item = s * gridDim.x + blockIdx.x, kvh = blockIdx.x / a.row_groups, rg = blockIdx.x - kvh * a.row_groups;
  const int c = blockIdx.z, r = row_of(a, c), clusters = a.pieces / a.cluster;
  int row0 = s, rows = 1;
  if (a.cu_q != nullptr) {
    const int first = a.cu_q[s], count = a.cu_q[s + 1] - first;
    row0 = first + rg * a.rows_per;
    rows = min(a.rows_per, count - rg * a.rows_per);
    if (count <= 0 || first < 0 || count > a.max_q || first + count > a.q_rows) rows = 0;
  }
  if (r >= rows) return;
  const int grp = threadIdx.x / kQuads, d = (threadIdx.x - grp * kQuads) * 4;
  const float* from = a.scratch + (size_t(item) * clusters * cols_kept + c) * (HD + 4);
  const size_t step = size_t(cols_kept) * (HD + 4);
  float top = kNone, total = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  auto add = [&](float m, float l, const float4& x) {
    const float to = fmaxf(top, m), f = ex2(top - to), g = ex2(m - to);
    top = to;
    total = total * f + l * g;
    acc = make_float4(acc.x * f + x.x * g, acc.y * f + x.y * g, acc.z * f + x.z * g, acc.w * f + x.w * g);
  };
  if (grp < kGroups) {
#pragma unroll 4
    for (int w = grp; w < clusters; w += kGroups) {
      const float2 n = *reinterpret_cast<const float2*>(from + w * step + HD);
      add(n.x, n.y, *reinterpret_cast<const float4*>(from + w * step + d));
    }
    part[grp][d / 4] = acc;
    if (d == 0) number[grp] = make_float2(top, total);
  }
  __syncthreads();
  if (grp == 0) {
#pragma unroll
    for (int w = 1; w < kGroups; ++w) add(number[w].x, number[w].y, part[w][d / 4]);
    const float inv = total == 0.f ? 0.f : 1.f / total;
    *reinterpret_cast<uint2*>(a.out + size_t(row0 + r) * a.ldo + size_t(kvh * a.group + c - r * a.group) * HD + d) =
        make_uint2(pack_half2(acc.x * inv, acc.y * inv), pack_half2(acc.z * inv, acc.w * inv));
  }
}

struct Plan {
  int nb, rows_per, row_groups, pieces, cluster, sort;
  long long scratch_floats;
};
Plan plan_of(const ZseAttnQ8& a) {
  Plan p;
  const int G = a.nh / a.kv.nkv;
  p.nb = a.max_q * G <= 8 ? 1 : 2;
  p.rows_per = std::max(1, 8 * p.nb / G);
  p.row_groups = (a.max_q + p.rows_per - 1) / p.rows_per;
  const long long items = (long long)a.num_seqs * a.kv.nkv * p.row_groups;
  // Pieces: what fits the GPU at a time (CTAs an SM by registers and shared memory; an eighth less, for clusters need neighbouring
  // places), at least half a tile a warp.  Measured (HD 128, us by pieces): 1 x 1000 tokens of 8 kv heads 1: 11.1, 4: 5.9, 8: 5.0; 32 x 500
  // 1: 15.9, 2: 13.4, 4: 17.6.
  // Twice as many, a second wave, where there is little more than one (one) and a warp still has 16 (12) tiles: sequences of mixed length are then
  // shared out better, the longest first.  64 x 128 .. 2300 tokens of 8 kv heads 1: 38.5, 2: 35.0; 128 .. 4600 1: 71, 2: 55; of 32 heads over
  // 8 of 64 28 and 23; 48 x 100 .. 1700 of 40 over 8 28.5 and 23.8; 32 drafts of up to five rows 79 and 71; but 64 x 2300 1: 52.8, 2: 56.2, 64 x
  // 1300 .. 1600 36.7 and 40.9, 32 x 6000 .. 8000 of 28 over 4 4: 44.0, 8: 47.7 (the plan has the table's width, not the lengths), and windows make
  // sequences alike.
  // Several clusters (and the launch that joins them) where eight pieces leave a warp 12 tiles: 1 x 4000 of 4 kv heads 8: 8.4, 32: 7.8;
  // 1 x 32765 8: 38, 64: 15.5, 128: 14.0.
  const int per_sm = a.kv.hd > 128 ? (p.nb == 1 ? 2 : 1) : p.nb == 1 || a.kv.hd == 64 ? 4 : 3;
  const long long slots = (long long)sm_count() * per_sm;
  long long want = a.num_splits;
  if (want <= 0) {
    long long tiles = (long long)a.max_blocks * (a.kv.block_size / 16);
    if (a.window > 0) tiles = std::min(tiles, ((long long)a.window + a.max_q) / 16 + 2);
    const long long room = std::max(1ll, slots * 7 / 8 / items);
    want = 1;
    while (want < kMostCluster && want * 2 <= room && want * 2 <= (tiles + 1) / 2) want *= 2;
    if (want < kMostCluster && want * 2 > room && a.window == 0 && items * want * 4 <= 5 * slots &&
        tiles >= want * 2 * kWarps * (items * want <= slots ? 12 : 16))
      want *= 2;
    if (want == kMostCluster && room > kMostCluster && tiles >= kMostCluster * kWarps * 12)
      want = std::max(want, std::min(room, tiles / (4 * kWarps)) / kMostCluster * kMostCluster);
  }
  p.cluster = 1;
  while (p.cluster < want && p.cluster < kMostCluster) p.cluster *= 2;
  p.pieces = int(std::min(64ll, (want + p.cluster - 1) / p.cluster) * p.cluster);
  // The longest first where the CTAs do not all run at once.  More than 8 columns: 64 drafts of five rows of 28 heads over 4, 500 .. 2000
  // tokens, 1.7 waves 68.2 as they come, 57.4 the longest first; 48 of three rows of 64 over 8 53.7, 43.7.  Up to 8 columns from one
  // and a half waves on: 48 x 100 .. 1700 of 32 heads over 8 of 64, 1.3 waves, 15.4 and 18.0 (a step takes that long to find its sequence).
  p.sort = a.num_seqs > 1 && a.num_seqs <= 64 && 2 * items * p.pieces >= (p.nb == 1 ? 3 : 2) * slots ? a.num_seqs : 0;
  p.scratch_floats = p.pieces == p.cluster ? 0 : items * (p.pieces / p.cluster) * 8 * p.nb * (a.kv.hd + 4);
  return p;
}
bool shape_ok(const ZseAttnQ8& a) {
  const ZseKvQ8& kv = a.kv;
  return kv.num_blocks > 0 && kv.nkv > 0 && kv.block_size > 0 && kv.block_size % 16 == 0 && a.nh > 0 && a.nh % kv.nkv == 0 &&
         a.nh / kv.nkv <= 16 && a.max_blocks >= 0 && a.max_q <= 64 && (a.cu_q != nullptr || a.max_q == 1) &&
         (kv.hd == 64 || kv.hd == 96 || kv.hd == 128 || kv.hd == 256);
}

template <int HD, int NB, bool PACKED>
int launch(const Q8Args& a, int num_seqs, cudaStream_t st) {
  static bool ready[kMaxDevices];
  const int dev = current_device_slot();
  auto kernel = attn_q8_kernel<HD, NB, PACKED>;
  constexpr int kBytes = Q8Smem<HD, NB>::kTotal;
  if (!ready[dev]) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kBytes) != cudaSuccess) return ZSE_ERR_LAUNCH;
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
      launch_pdl(attn_q8_join_kernel<HD>, dim3(a.nkv * a.row_groups, num_seqs, a.rows_per * a.group), dim3(128), 0, st, a, 8 * NB) != cudaSuccess)
    return ZSE_ERR_LAUNCH;
  return a.pieces > a.cluster ? 2 : 1;
}

}  // namespace
}  // namespace zse

using namespace zse;

extern "C" int zse_attn_decode_q8_pieces(const ZseAttnQ8* x) {
  return x->num_seqs > 0 && x->max_q > 0 && shape_ok(*x) ? plan_of(*x).pieces : 0;
}
extern "C" int64_t zse_attn_decode_q8_scratch_floats(const ZseAttnQ8* x) {
  return x->num_seqs > 0 && x->max_q > 0 && shape_ok(*x) ? plan_of(*x).scratch_floats : 0;
}

extern "C" int zse_attn_decode_q8(const ZseAttnQ8* x) {
  const ZseKvQ8& kv = x->kv;
  if (x->num_seqs <= 0 || x->max_q <= 0) return 0;
  if (!shape_ok(*x)) return ZSE_ERR_SHAPE;
  if ((reinterpret_cast<uintptr_t>(kv.data) | reinterpret_cast<uintptr_t>(kv.scale) | reinterpret_cast<uintptr_t>(x->scratch) |
       reinterpret_cast<uintptr_t>(x->q)) & 15 || reinterpret_cast<uintptr_t>(x->out) & 7 || x->ldq % 8 || x->ldo % 4)
    return ZSE_ERR_ALIGN;
  const Plan p = plan_of(*x);
  const int bpt = kv.block_size / 16, group = x->nh / kv.nkv;
  if (x->num_seqs > 65535 || (long long)kv.nkv * p.row_groups > 65535 ||
      (long long)x->num_seqs * kv.nkv * p.row_groups > 0x7fffffffll || (long long)kv.num_blocks * 2 * kv.nkv * bpt > 0x7fffffffll ||
      (long long)x->max_blocks * kv.block_size > 0x7fffff00ll || (long long)kv.nkv * kv.block_size * kv.hd > 0x7fffffffll)
    return ZSE_ERR_LIMIT;
  if (p.scratch_floats > 0 && (x->scratch == nullptr || x->scratch_floats < p.scratch_floats)) return ZSE_ERR_SCRATCH;
  int shift = 0;
  while ((1 << shift) < bpt) ++shift;
  const Q8Args a{static_cast<const uint8_t*>(kv.data), static_cast<const float*>(kv.scale), static_cast<const __half*>(x->q),
                 static_cast<const int*>(x->tables), static_cast<const int*>(x->seq_lens), static_cast<const int*>(x->cu_q),
                 static_cast<const int*>(x->q_pos0), static_cast<__half*>(x->out), static_cast<float*>(x->scratch),
                 static_cast<Status*>(x->status), x->ldq, x->ldo, x->q_rows, kv.num_blocks, kv.nkv, bpt,
                 (1 << shift) == bpt ? shift : -1, x->table_ld, x->max_blocks, group, (65536 + group - 1) / group, x->max_q,
                 p.rows_per, p.row_groups, x->window, p.pieces, p.cluster, p.sort, x->scale * kLog2e * 16777216.f};
  const int n = x->num_seqs;
  const cudaStream_t st = static_cast<cudaStream_t>(x->stream);
  auto go = [&](auto packed, auto one, auto two) { return (x->max_q * group <= 4 ? packed : p.nb == 1 ? one : two)(a, n, st); };
  switch (kv.hd) {
    case 64: return go(launch<64, 1, true>, launch<64, 1, false>, launch<64, 2, false>);
    case 96: return go(launch<96, 1, true>, launch<96, 1, false>, launch<96, 2, false>);
    case 128: return go(launch<128, 1, true>, launch<128, 1, false>, launch<128, 2, false>);
    default: return go(launch<256, 1, true>, launch<256, 1, false>, launch<256, 2, false>);
  }
}
