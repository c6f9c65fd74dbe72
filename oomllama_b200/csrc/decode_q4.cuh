// K-B over a 4-bit cache (kv4.cuh): split-KV GQA decode, the schedule, the
// split merge and the outputs those of decode.cuh.
//
// Mathematics.  With K row r = o_g + (c - 8) s_g per group g of 32 dims,
//   q . K[r] = sum_g s_g (q_g . c_g) + sum_g (o_g sum(q_g) + s_g (-8 sum(q_g)))
// The first sum is a tensor-core product of q with the bare codes, scaled per
// group in f32; the second is one more product, of the four group sums of q
// (and -8 times them) with the token's eight stored numbers [o, s].  For V,
// (c - 8) s is exact in f16 (s has 8 bits), so
//   O = sum_r p_r (c - 8) s  +  sum_r p_r o
// is a product with the f16 values plus a small one with the offsets, which
// are one column per group.
//
// Tiles.  m16n8k16 with keys (K) or dims (V) as the 16 rows and four query
// heads as the 8 columns, column 2 h the f16 high part of head h's query (or
// probability), column 2 h + 1 the low part (x - high): one product carries 22
// bits of the f32 value, and the two columns of an accumulator, which lie in
// one lane, are added at the end.  A group of five to eight heads takes two
// such column sets (SETS = 2) over the same unpacked rows.  With the heads as
// rows instead (8 high, 8 low) a group of four would cost as many products as
// one of eight, and twice the softmax.  K codes enter as subnormal halves (code *
// 2^-24, or 2^-20 for the upper nibble of a byte, whose q is prescaled by
// 1/16): unpacking is one AND per two codes.  q is scaled by a power of two to
// [2^14, 2^15) per head so that its low part keeps its bits.
// The P V products of a 32-token tile start from zero and are added to O in
// f32 (one packed FMA with the softmax rescale): the tensor core truncates
// when it accumulates, which over a long context would shrink O.
//
// Each warp works alone: its own ring of tiles in shared memory, filled by
// bulk copies (one of 2560 bytes per page: K, then V) that one of its lanes issues, its
// own running maximum and sum; the four warps of a CTA join at the end.
#pragma once
#include "common.cuh"
#include "decode.cuh"
#include "kv4.cuh"
#include "params.cuh"
#include "rope_append.cuh"

namespace oomattn {

constexpr int kQ4Pages = 2;                              // pages per tile
constexpr int kQ4Tile = kQ4Pages * kPageSize;            // tokens per tile
constexpr int kQ4TileBytes = kQ4Pages * kQ4Pair;         // 5 KB
// One column set needs 128 registers and two need 168: four CTAs of two stages
// each, or three of three, per SM -- about 160 and 180 KB in flight.
__host__ __device__ constexpr int q4_stages(int sets) { return sets == 1 ? 2 : 3; }
__host__ __device__ constexpr int q4_ctas_per_sm(int sets) { return sets == 1 ? 4 : 3; }
__host__ __device__ constexpr int q4_ring_bytes(int sets) { return kDecWarps * q4_stages(sets) * kQ4TileBytes; }
__host__ __device__ constexpr int q4_smem_bytes(int sets) {
  return q4_ring_bytes(sets) + kDecWarps * q4_stages(sets) * 8 + 64 + kMaxGroup * 32 * 4;
}
static_assert(sizeof(MergeSmem) <= q4_ring_bytes(1), "the merge is staged over the ring");

__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                   smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}
__device__ __forceinline__ void mma_f16_16816(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// The same from zero: the accumulator's registers need no clearing.
__device__ __forceinline__ void mma_f16_16816_z(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ void mma_f16_1688_z(float* d, uint32_t a0, uint32_t a1, uint32_t b0) {
  asm(
      "mma.sync.aligned.m16n8k8.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5}, {%6}, {%7,%7,%7,%7};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(b0), "f"(0.f));
}
__device__ __forceinline__ uint32_t h2_add(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("add.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
__device__ __forceinline__ uint32_t h2_mul(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
__device__ __forceinline__ uint32_t h2_fma(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t d;
  asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
  return d;
}
// (x & mask) | magic in one instruction (with both as immediates it takes two).
__device__ __forceinline__ uint32_t and_or(uint32_t x, uint32_t mask, uint32_t magic) {
  uint32_t d;
  asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(d) : "r"(x), "r"(mask), "r"(magic));
  return d;
}
__device__ __forceinline__ float h_lo(uint32_t v) { return __half2float(__ushort_as_half((uint16_t)v)); }
__device__ __forceinline__ float h_hi(uint32_t v) { return __half2float(__ushort_as_half((uint16_t)(v >> 16))); }
// (a, b) rounded to f16, or (low) what that rounding leaves: exact in f32, rounded once.
__device__ __forceinline__ uint32_t f16_part(float a, float b, bool low) {
  const uint32_t hi = pack_f16(a, b);
  return low ? pack_f16(a - h_lo(hi), b - h_hi(hi)) : hi;
}

// decode.cuh's prefetch_then_wait for 4-bit chunks.
__device__ __forceinline__ void q4_prefetch_then_wait(const KVPool& pool, const DecodeArgs& a, int seq, int g, int pb,
                                                      int pe) {
  const int np = min(pe - pb, kDecPrefetchPages);
  if (np > 0) {
    constexpr int lines = kQ4Pair / 128;
    const int* bt = pool.block_table + (size_t)seq * pool.max_pages_per_seq;
    for (int i = threadIdx.x; i < np * lines; i += blockDim.x) {
      const int page = __ldg(bt + pb + i / lines), r = i % lines;
      if ((unsigned)page >= (unsigned)pool.n_pool_pages) continue;  // reported by the main loop
      const char* base = static_cast<const char*>(pool.k) + q4_chunk_off(pool, a.layer, page, g);
      asm volatile("prefetch.global.L2 [%0];" ::"l"(base + (size_t)r * 128));
    }
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");
}

// IO16: q and out in bf16 (the newest tokens of a sequence as one row each)
// instead of f32 (a generation step).
template <int SETS, bool IO16>
__global__ void __launch_bounds__(kDecWarps * 32, q4_ctas_per_sm(SETS))
    decode_q4_kernel(const KVPool pool, const DecodeArgs a, const __grid_constant__ SeqBatch sb,
                     const __grid_constant__ DecodeSched sched) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // as in decode_bf16_kernel
  constexpr int kStages = q4_stages(SETS), kRing = q4_ring_bytes(SETS);
  extern __shared__ __align__(128) uint8_t smem_q4[];
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem_q4 + kRing);
  int* s_last = reinterpret_cast<int*>(bars + kDecWarps * kStages);
  float* s_w = reinterpret_cast<float*>(s_last + 16);  // [kMaxGroup][32] merge weights

  const DecodeItem item = decode_item(sched, sb, blockIdx.x);
  const int g_kv = item.g, z = item.z;
  const int seq = sb.seq[z], L = sb.len[z];
  const int pb = item.pb, pe = item.pe;
  q4_prefetch_then_wait(pool, a, seq, g_kv, pb, pe);
  if (pb >= pe) {
    if (!IO16 && L <= 0 && item.split == 0) write_empty_row(a, z, g_kv);  // a bf16 row sees its own token at least
    return;
  }
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  uint8_t* ring = smem_q4 + warp * (kStages * kQ4TileBytes);
  uint64_t* full = bars + warp * kStages;
  if (lane == 0)
    for (int s = 0; s < kStages; ++s) mbar_init(&full[s], kQ4Pages);
  fence_mbar_init();
  __syncwarp();

  // ---- this warp's tiles: warp, warp + 4, ... of the CTA's pages; lane l holds
  // the ids of the warp's local pages l (mod 32), the next 32 loaded ahead
  const int n_tiles_cta = (pe - pb + kQ4Pages - 1) / kQ4Pages;
  const int n_tiles = n_tiles_cta > warp ? (n_tiles_cta - warp + kDecWarps - 1) / kDecWarps : 0;
  const int* bt = pool.block_table + (size_t)seq * pool.max_pages_per_seq;
  auto tile_page = [&](int k) { return pb + (warp + k * kDecWarps) * kQ4Pages; };  // first page of local tile k
  auto load_id = [&](int j) {  // id of local page j
    const int pi = tile_page(j / kQ4Pages) + j % kQ4Pages;
    int id = -1;
    if (j < n_tiles * kQ4Pages && pi < pe) {
      id = __ldg(bt + pi);
      if ((unsigned)id >= (unsigned)pool.n_pool_pages) {
        report_error(a.status, kDevErrBounds);
        id = pool.n_pool_pages - 1;
      }
    }
    return id;
  };
  int ids = load_id(lane), ids_next = load_id(lane + 32);
  int issued = 0;
  bool gave_up = false;
  // lane i copies K and V of a tile's page i: one chunk of the pool
  const uint8_t* base = static_cast<const uint8_t*>(pool.k) + q4_chunk_off(pool, a.layer, 0, g_kv);
  const uint32_t page_bytes = (uint32_t)pool.n_kv * kQ4Pair;
  uint8_t* dst0 = ring + (lane & 1) * kQ4Pair;
  const bool drop = (a.test_flags & kTestDropDecodeCopies) != 0;
  auto issue = [&](int k, int s) {  // all lanes; copies of local tile k into stage s
    const int j = (k * kQ4Pages) & 31;
    if (j == 0 && k > 0) {
      ids = ids_next;
      ids_next = load_id(k * kQ4Pages + 32 + lane);
    }
    const int id = __shfl_sync(0xffffffffu, ids, j + (lane & 1));
    if (drop) return;
    // each of the two lanes arrives for its own page (a missing second one: no bytes)
    if (lane < kQ4Pages) {
      mbar_arrive_expect_tx(&full[s], id >= 0 ? kQ4Pair : 0);
      if (id >= 0) bulk_load(dst0 + s * kQ4TileBytes, base + (size_t)(uint32_t)id * page_bytes, kQ4Pair, &full[s]);
    }
    issued = k + 1;
  };
  for (int k = 0; k < min(kStages, n_tiles); ++k) issue(k, k);

  // ---- the query as B operand: of set u, lane (g, t) holds column g, the high
  // (g even) or low part of head 4 u + g / 2, at dims 32 w + 8 t + 0..7; product
  // j of group w meets K nibbles (2j | 2j + 4) and (2j + 1 | 2j + 5) of the word
  uint32_t qb[SETS][8][2], bm[SETS];
  float f2[SETS];  // of head 4 u + t: score * f2 is the base-2 logit
#pragma unroll
  for (int u = 0; u < SETS; ++u) {
    const int j = 4 * u + (g >> 1);
    const bool valid = j < a.group, low = g & 1;
    const size_t q0 = ((size_t)z * a.n_heads + g_kv * a.group + (valid ? j : 0)) * kHeadDim;
    float x[4][8];
    float mx = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      load8<IO16>(a.q, q0 + 32 * w + 8 * t, x[w]);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (!valid) x[w][i] = 0.f;
        mx = fmaxf(mx, fabsf(x[w][i]));
      }
    }
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
    // 2^e brings the largest |q| to [2^14, 2^15); zero, subnormal and infinite q stay finite factors
    const int ex = (int)((__float_as_uint(mx) >> 23) & 255u);
    const int e = min(100, max(-100, 14 + 127 - (ex == 0 ? 127 : ex)));
    const float up = __uint_as_float((uint32_t)(127 + e) << 23);
    // codes enter as code * 2^-24: undo that and 2^e (both powers of two, f2 stays normal)
    const float f2_own = a.qscale * __uint_as_float((uint32_t)(127 + 24) << 23) * __uint_as_float((uint32_t)(127 - e) << 23);
    f2[u] = __shfl_sync(0xffffffffu, f2_own, 8 * t);
    float qs[4];
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        x[w][i] *= up;
        sum += x[w][i];
      }
      sum += __shfl_xor_sync(0xffffffffu, sum, 1);
      sum += __shfl_xor_sync(0xffffffffu, sum, 2);
      qs[w] = sum * (1.f / 4096.f);  // within f16: |sum| < 2^20, times 8 below
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        qb[u][2 * w + i][0] = f16_part(x[w][2 * i], x[w][2 * i + 4], low);
        qb[u][2 * w + i][1] = f16_part(x[w][2 * i + 1] * 0.0625f, x[w][2 * i + 5] * 0.0625f, low);
      }
    }
    // rows [o0 o1 | o2 o3 | s0 s1 | s2 s3] of the token's stored numbers, lane t has its two
    const float u0 = (t & 1) ? qs[2] : qs[0], u1 = (t & 1) ? qs[3] : qs[1];
    const float m8 = t < 2 ? 1.f : -8.f;
    bm[u] = f16_part(u0 * m8, u1 * m8, low);
  }

  uint64_t o[SETS][4][2];  // [group w][i]: head 4 u + t, dims 32 w + 4 g + 2 i and + 1
  float oo[SETS];          // sum p * offset of group g % 4, head 4 u + t
  float m[SETS], l[SETS];     // m: the running maximum as a base-2 logit
#pragma unroll
  for (int u = 0; u < SETS; ++u) {
#pragma unroll
    for (int w = 0; w < 4; ++w) o[u][w][0] = o[u][w][1] = 0;
    oo[u] = 0.f;
    m[u] = -INFINITY;
    l[u] = 0.f;
  }
  const int tok_end = min(pe * kPageSize, L);
  uint32_t magic;  // 1024.0 in both halves, in a register
  asm volatile("mov.b32 %0, 0x64006400;" : "=r"(magic));

  int s = 0;
  uint32_t phase = 0;
  for (int k = 0; k < n_tiles; ++k) {
    // all lanes leave together: the shuffles and products below are the whole warp's
    if (!__all_sync(0xffffffffu, mbar_wait(&full[s], phase, a.status, a.timeout_ns))) {
      gave_up = true;
      break;
    }
    uint8_t* st = ring + s * kQ4TileBytes;
    const int lim = tok_end - tile_page(k) * kPageSize;  // tokens of the tile that count: >= 1
    if (lim < kQ4Tile) {
      // the row's (or the split's) last tile: zero the V scales and offsets of the
      // tokens behind the end, which may be stale or never written; their scores
      // become -inf below.  (No copy follows into this stage.)
      if (lane >= lim) {
        uint8_t* mp = st + (lane >> 4) * kQ4Pair + kQ4Chunk + kQ4Meta + q4_v_meta(lane & 15) + 2 * (lane & 1);
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          *reinterpret_cast<uint16_t*>(mp + 4 * w) = 0;
          *reinterpret_cast<uint16_t*>(mp + kQ4VOffsets - kQ4Meta + 4 * w) = 0;
        }
      }
      __syncwarp();
    }
    // ---- scores of 2 x 16 tokens: rows g and g + 8 of a page, head 4 u + t
    float sc[SETS][4];
#pragma unroll
    for (int pg = 0; pg < 2; ++pg) {
      const uint8_t* kc = st + pg * kQ4Pair;
      const uint4 wa = *reinterpret_cast<const uint4*>(kc + lane * 16);
      const uint4 wb = *reinterpret_cast<const uint4*>(kc + 512 + lane * 16);
      const uint32_t am0 = *reinterpret_cast<const uint32_t*>(kc + kQ4Meta + g * 16 + t * 4);
      const uint32_t am1 = *reinterpret_cast<const uint32_t*>(kc + kQ4Meta + (g + 8) * 16 + t * 4);
      const uint2 sa = *reinterpret_cast<const uint2*>(kc + kQ4Meta + g * 16 + 8);
      const uint2 sb2 = *reinterpret_cast<const uint2*>(kc + kQ4Meta + (g + 8) * 16 + 8);
      float acc[SETS][2];
#pragma unroll
      for (int u = 0; u < SETS; ++u) {
        float d[4];
        mma_f16_1688_z(d, am0, am1, bm[u]);
        acc[u][0] = (d[0] + d[1]) * (1.f / 4096.f);  // 2^-24 / 2^-12
        acc[u][1] = (d[2] + d[3]) * (1.f / 4096.f);
      }
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const uint32_t xa = w == 0 ? wa.x : (w == 1 ? wa.y : (w == 2 ? wa.z : wa.w));
        const uint32_t xb = w == 0 ? wb.x : (w == 1 ? wb.y : (w == 2 ? wb.z : wb.w));
        const uint32_t ya = xa >> 8, yb = xb >> 8;
        const uint32_t f0[4] = {xa & 0x000f000fu, xb & 0x000f000fu, xa & 0x00f000f0u, xb & 0x00f000f0u};
        const uint32_t f1[4] = {ya & 0x000f000fu, yb & 0x000f000fu, ya & 0x00f000f0u, yb & 0x00f000f0u};
        const uint32_t ha = w < 2 ? sa.x : sa.y, hb = w < 2 ? sb2.x : sb2.y;
        const float s0 = (w & 1) ? h_hi(ha) : h_lo(ha), s1 = (w & 1) ? h_hi(hb) : h_lo(hb);
#pragma unroll
        for (int u = 0; u < SETS; ++u) {
          float e[4];
          mma_f16_16816_z(e, f0, qb[u][2 * w][0], qb[u][2 * w][1]);
          mma_f16_16816(e, f1, qb[u][2 * w + 1][0], qb[u][2 * w + 1][1]);
          acc[u][0] = fmaf(e[1], s0, fmaf(e[0], s0, acc[u][0]));
          acc[u][1] = fmaf(e[3], s1, fmaf(e[2], s1, acc[u][1]));
        }
      }
#pragma unroll
      for (int u = 0; u < SETS; ++u) {
        sc[u][2 * pg] = acc[u][0];
        sc[u][2 * pg + 1] = acc[u][1];
      }
    }
    if (lim < kQ4Tile) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (8 * i + g >= lim) {
#pragma unroll
          for (int u = 0; u < SETS; ++u) sc[u][i] = -INFINITY;
        }
    }
    // ---- online softmax of the lane's heads over the tile
    uint32_t pb2[SETS][4];  // B operands: (high | low) of tokens 2t, 2t + 1 of each half page, column g
    float alpha[SETS];
#pragma unroll
    for (int u = 0; u < SETS; ++u) {
      float mt = fmaxf(max3f(sc[u][0], sc[u][1], sc[u][2]), sc[u][3]);
#pragma unroll
      for (int off = 4; off < 32; off <<= 1) mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, off));
      // the running maximum is rounded: the same number enters every weight, so its rounding cancels
      const float mf = fmaxf(m[u], mt * f2[u]);
      alpha[u] = ex2_ftz(m[u] - mf);
      m[u] = mf;
      float ps = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float p = ex2_ftz(fmaf(sc[u][i], f2[u], -mf));
        ps += p;
        // token row g, columns (2t, 2t + 1) = (high, low) of the head; transposed: tokens 2t, 2t + 1 of column g
        pb2[u][i] = movmatrix_trans(pack_f16(p, p - h_lo(pack_f16(p, 0.f))));
      }
      l[u] = fmaf(l[u], alpha[u], ps);
    }
    // ---- O = O * alpha + V^T P
    uint4 vw[4], vs[4];  // [page, half]: the four groups' codes and scales of the lane's token pair
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint8_t* vc = st + (i >> 1) * kQ4Pair + kQ4Chunk;
      vw[i] = *reinterpret_cast<const uint4*>(vc + (i & 1) * 512 + lane * 16);
      vs[i] = *reinterpret_cast<const uint4*>(vc + kQ4Meta + (i & 1) * 64 + t * 16);
    }
    uint32_t ao[2][4];  // offsets as A operand: row g (and g + 8) = group g % 4
#pragma unroll
    for (int pg = 0; pg < 2; ++pg) {
      const uint8_t* vo = st + pg * kQ4Pair + kQ4Chunk + kQ4VOffsets + t * 16 + (g & 3) * 4;
      ao[pg][0] = ao[pg][1] = *reinterpret_cast<const uint32_t*>(vo);
      ao[pg][2] = ao[pg][3] = *reinterpret_cast<const uint32_t*>(vo + 64);
    }
#pragma unroll
    for (int u = 0; u < SETS; ++u) {
      float d[4];
      mma_f16_16816_z(d, ao[0], pb2[u][0], pb2[u][1]);
      mma_f16_16816(d, ao[1], pb2[u][2], pb2[u][3]);
      oo[u] = fmaf(oo[u], alpha[u], d[0] + d[1]);
    }
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      float e[SETS][2][4];
#pragma unroll
      for (int pg = 0; pg < 2; ++pg) {
        uint32_t b[2][4];  // [half][n]
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint4& c4 = vw[2 * pg + h];
          const uint4& s4 = vs[2 * pg + h];
          const uint32_t x = w == 0 ? c4.x : (w == 1 ? c4.y : (w == 2 ? c4.z : c4.w));
          const uint32_t s2 = w == 0 ? s4.x : (w == 1 ? s4.y : (w == 2 ? s4.z : s4.w));
          const uint32_t y = x >> 8;
          // 1024 + c, or 1024 + 16 c, to c - 8, times s: every step exact
          b[h][0] = h2_mul(h2_add(and_or(x, 0x000f000fu, magic), 0xe408e408u), s2);
          b[h][1] = h2_mul(h2_fma(and_or(x, 0x00f000f0u, magic), 0x2c002c00u, 0xd480d480u), s2);
          b[h][2] = h2_mul(h2_add(and_or(y, 0x000f000fu, magic), 0xe408e408u), s2);
          b[h][3] = h2_mul(h2_fma(and_or(y, 0x00f000f0u, magic), 0x2c002c00u, 0xd480d480u), s2);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint32_t av[4] = {b[0][2 * i], b[0][2 * i + 1], b[1][2 * i], b[1][2 * i + 1]};
#pragma unroll
          for (int u = 0; u < SETS; ++u) {
            if (pg == 0) mma_f16_16816_z(e[u][i], av, pb2[u][0], pb2[u][1]);
            else mma_f16_16816(e[u][i], av, pb2[u][2], pb2[u][3]);
          }
        }
      }
#pragma unroll
      for (int u = 0; u < SETS; ++u) {
        const uint64_t al2 = f2_pack(alpha[u], alpha[u]);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          o[u][w][i] = f2_fma(o[u][w][i], al2, f2_pack(e[u][i][0] + e[u][i][1], e[u][i][2] + e[u][i][3]));
        }
      }
    }
    __syncwarp();  // every lane has read the stage
    if (k + kStages < n_tiles) issue(k + kStages, s);
    if (++s == kStages) {
      s = 0;
      phase ^= 1;
    }
  }
  if (gave_up) {  // the copies that were issued land before the ring is used again
    for (int k = max(0, issued - kStages); k < issued; ++k)
      mbar_wait(&full[k % kStages], (k / kStages) & 1, a.status, a.timeout_ns);
  }

#pragma unroll
  for (int u = 0; u < SETS; ++u)
#pragma unroll
    for (int off = 4; off < 32; off <<= 1) l[u] += __shfl_xor_sync(0xffffffffu, l[u], off);
  consumer_bar();  // every warp is done with its ring
  MergeSmem& ms = *reinterpret_cast<MergeSmem*>(smem_q4);
#pragma unroll
  for (int u = 0; u < SETS; ++u) {
    if (g == 0) {
      ms.m[warp][4 * u + t] = m[u];
      ms.l[warp][4 * u + t] = l[u];
    }
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float off = __shfl_sync(0xffffffffu, oo[u], 4 * w + t);
      *reinterpret_cast<float4*>(&ms.o[warp][4 * u + t][32 * w + 4 * g]) =
          make_float4(f2_lo(o[u][w][0]) + off, f2_hi(o[u][w][0]) + off, f2_lo(o[u][w][1]) + off, f2_hi(o[u][w][1]) + off);
    }
  }
  consumer_bar();
  combine_and_store<IO16>(ms, a, z, g_kv, item.split, item.nsplit, pool.n_kv, threadIdx.x, s_last,
                          reinterpret_cast<float*>(smem_q4), kRing / 4, s_w);
}

}  // namespace oomattn
