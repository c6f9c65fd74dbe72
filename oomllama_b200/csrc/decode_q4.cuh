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
// Tiles.  m16n8k16 with the query heads of the group as rows: rows 0-7 hold
// the f16 high parts and rows 8-15 the low parts (x - high), so one product
// carries 22 bits of the f32 query (and probability) and the two halves of an
// accumulator are added at the end.  K codes enter as subnormal halves (code *
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
constexpr int kQ4Stages = 3;
constexpr int kQ4CtasPerSm = 3;
constexpr int kQ4RingBytes = kDecWarps * kQ4Stages * kQ4TileBytes;
constexpr int kQ4SmemBytes = kQ4RingBytes + kDecWarps * kQ4Stages * 8 + 64 + kMaxGroup * 32 * 4;
static_assert(sizeof(MergeSmem) <= kQ4RingBytes, "the merge is staged over the ring");

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
// (a, b) as f16 pairs hi + lo: lo = x - hi is exact in f32 and rounded once.
__device__ __forceinline__ void split_f16x2(float a, float b, uint32_t& hi, uint32_t& lo) {
  hi = pack_f16(a, b);
  lo = pack_f16(a - h_lo(hi), b - h_hi(hi));
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
template <bool IO16>
__global__ void __launch_bounds__(kDecWarps * 32, kQ4CtasPerSm)
    decode_q4_kernel(const KVPool pool, const DecodeArgs a, const __grid_constant__ SeqBatch sb,
                     const __grid_constant__ DecodeSched sched) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // as in decode_bf16_kernel
  extern __shared__ __align__(128) uint8_t smem_q4[];
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem_q4 + kQ4RingBytes);
  int* s_last = reinterpret_cast<int*>(bars + kDecWarps * kQ4Stages);
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
  uint8_t* ring = smem_q4 + warp * (kQ4Stages * kQ4TileBytes);
  uint64_t* full = bars + warp * kQ4Stages;
  if (lane == 0)
    for (int s = 0; s < kQ4Stages; ++s) mbar_init(&full[s], kQ4Pages);
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
  auto issue = [&](int k) {  // all lanes; copies of local tile k into its stage
    const int j = (k * kQ4Pages) & 31;
    if (j == 0 && k > 0) {
      ids = ids_next;
      ids_next = load_id(k * kQ4Pages + 32 + lane);
    }
    const int id = __shfl_sync(0xffffffffu, ids, j + (lane & 1));
    if (drop) return;
    const int s = k % kQ4Stages;
    // each of the two lanes arrives for its own page (a missing second one: no bytes)
    if (lane < kQ4Pages) {
      mbar_arrive_expect_tx(&full[s], id >= 0 ? kQ4Pair : 0);
      if (id >= 0) bulk_load(dst0 + s * kQ4TileBytes, base + (size_t)(uint32_t)id * page_bytes, kQ4Pair, &full[s]);
    }
    issued = k + 1;
  };
  for (int k = 0; k < min(kQ4Stages, n_tiles); ++k) issue(k);

  // ---- the query as A operand.  Of head g, lane t holds dims 32 w + 8 t + 0..7;
  // product j of group w takes K nibbles (2j | 2j + 4) and (2j + 1 | 2j + 5) of the word.
  uint32_t qa[8][4], am[2];
  float f2;  // score = accumulated * f2, base-2 logits
  {
    const bool valid = g < a.group;
    const size_t q0 = ((size_t)z * a.n_heads + g_kv * a.group + (valid ? g : 0)) * kHeadDim;
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
    // codes enter as code * 2^-24: undo that and 2^e in two exact steps (f2 stays normal)
    f2 = a.qscale * __uint_as_float((uint32_t)(127 + 24) << 23) * __uint_as_float((uint32_t)(127 - e) << 23);
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
      for (int j = 0; j < 2; ++j) {
        split_f16x2(x[w][2 * j], x[w][2 * j + 4], qa[2 * w + j][0], qa[2 * w + j][1]);
        split_f16x2(x[w][2 * j + 1] * 0.0625f, x[w][2 * j + 5] * 0.0625f, qa[2 * w + j][2], qa[2 * w + j][3]);
      }
    }
    // columns [o0 o1 | o2 o3 | s0 s1 | s2 s3] of the token's stored numbers, lane t has its two
    const float u0 = (t & 1) ? qs[2] : qs[0], u1 = (t & 1) ? qs[3] : qs[1];
    const float m8 = t < 2 ? 1.f : -8.f;
    split_f16x2(u0 * m8, u1 * m8, am[0], am[1]);
  }

  uint64_t o[4][4];  // [group w][n]: head g, dims 32 w + 8 t + n (low) and + 4 (high)
#pragma unroll
  for (int w = 0; w < 4; ++w)
#pragma unroll
    for (int n = 0; n < 4; ++n) o[w][n] = 0;
  uint64_t oo = 0;   // sum p * offset of groups 2 (t & 1), 2 (t & 1) + 1
  float m = -INFINITY, l = 0.f;
  const int tok_end = min(pe * kPageSize, L);
  uint32_t magic;  // 1024.0 in both halves, in a register
  asm volatile("mov.b32 %0, 0x64006400;" : "=r"(magic));
  const uint64_t kMetaUnit = f2_pack(1.f / 4096.f, 1.f / 4096.f);  // 2^-24 / 2^-12

  for (int k = 0; k < n_tiles; ++k) {
    const int s = k % kQ4Stages;
    // all lanes leave together: the shuffles and products below are the whole warp's
    if (!__all_sync(0xffffffffu, mbar_wait(&full[s], (k / kQ4Stages) & 1, a.status, a.timeout_ns))) {
      gave_up = true;
      break;
    }
    uint8_t* st = ring + s * kQ4TileBytes;
    const int lim = tok_end - tile_page(k) * kPageSize;  // tokens of the tile that count: >= 1
    if (lim < kQ4Tile) {
      // the row's (or the split's) last tile: zero the V scales and offsets of the
      // tokens behind the end, which may be stale or never written; their scores
      // become -inf below.  (No copy follows into this stage.)
      const int tok = lane;
      if (tok >= lim) {
        uint8_t* mp = st + (tok >> 4) * kQ4Pair + kQ4Chunk + kQ4Meta + q4_v_meta(tok & 15) + 2 * (tok & 1);
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          *reinterpret_cast<uint16_t*>(mp + 4 * w) = 0;
          *reinterpret_cast<uint16_t*>(mp + kQ4VOffsets - kQ4Meta + 4 * w) = 0;
        }
      }
      __syncwarp();
    }
    // ---- S = q K^T of 32 tokens: n-tile nt = tokens 8 nt .. + 7, lane's are 2t, 2t + 1
    float sc[8];
#pragma unroll
    for (int nt = 0; nt < 4; ++nt) {
      const uint8_t* kc = st + (nt >> 1) * kQ4Pair;
      const int h = nt & 1;
      const uint4 w4 = *reinterpret_cast<const uint4*>(kc + h * 512 + lane * 16);
      const uint32_t bm = *reinterpret_cast<const uint32_t*>(kc + kQ4Meta + (8 * h + g) * 16 + t * 4);
      const uint2 s0 = *reinterpret_cast<const uint2*>(kc + kQ4Meta + (8 * h + 2 * t) * 16 + 8);
      const uint2 s1 = *reinterpret_cast<const uint2*>(kc + kQ4Meta + (8 * h + 2 * t + 1) * 16 + 8);
      const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
      float d[4];
      mma_f16_1688_z(d, am[0], am[1], bm);
      uint64_t acc = f2_fma(f2_pack(d[0], d[1]), kMetaUnit, 0);
      acc = f2_fma(f2_pack(d[2], d[3]), kMetaUnit, acc);
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const uint32_t x = w[q], y = w[q] >> 8;
        float e[4];
        mma_f16_16816_z(e, qa[2 * q], x & 0x000f000fu, x & 0x00f000f0u);
        mma_f16_16816(e, qa[2 * q + 1], y & 0x000f000fu, y & 0x00f000f0u);
        const uint32_t a0 = q < 2 ? s0.x : s0.y, a1 = q < 2 ? s1.x : s1.y;
        const uint64_t sp = (q & 1) ? f2_pack(h_hi(a0), h_hi(a1)) : f2_pack(h_lo(a0), h_lo(a1));
        acc = f2_fma(f2_pack(e[0], e[1]), sp, acc);
        acc = f2_fma(f2_pack(e[2], e[3]), sp, acc);
      }
      sc[2 * nt] = f2_lo(acc);
      sc[2 * nt + 1] = f2_hi(acc);
    }
    if (lim < kQ4Tile) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (8 * (i >> 1) + 2 * t + (i & 1) >= lim) sc[i] = -INFINITY;
    }
    // ---- online softmax of head g over the tile
    float mt = fmaxf(max3f(sc[0], sc[1], sc[2]), max3f(sc[3], sc[4], sc[5]));
    mt = max3f(mt, sc[6], sc[7]);
    mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, 1));
    mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, 2));
    // m is the running maximum as a base-2 logit, rounded: the same number in
    // every weight, so its rounding cancels
    const float mf = fmaxf(m, mt * f2);
    const float alpha = ex2_ftz(m - mf);
    m = mf;
    float ps = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      sc[i] = ex2_ftz(fmaf(sc[i], f2, -mf));
      ps += sc[i];
    }
    l = fmaf(l, alpha, ps);
    uint32_t pa[2][4];  // A operands of the two pages: rows hi, lo x tokens (2t, 2t+1), (8 + 2t, + 1)
#pragma unroll
    for (int pg = 0; pg < 2; ++pg) {
      split_f16x2(sc[4 * pg], sc[4 * pg + 1], pa[pg][0], pa[pg][1]);
      split_f16x2(sc[4 * pg + 2], sc[4 * pg + 3], pa[pg][2], pa[pg][3]);
    }
    // ---- O = O * alpha + P V
    const uint64_t al2 = f2_pack(alpha, alpha);
    uint4 vw[4], vs[4];  // [page, half]: the four groups' codes and scales of the lane's token pair
    float d[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint8_t* vc = st + (i >> 1) * kQ4Pair + kQ4Chunk;
      vw[i] = *reinterpret_cast<const uint4*>(vc + (i & 1) * 512 + lane * 16);
      vs[i] = *reinterpret_cast<const uint4*>(vc + kQ4Meta + (i & 1) * 64 + t * 16);
    }
#pragma unroll
    for (int pg = 0; pg < 2; ++pg) {
      const uint8_t* vo = st + pg * kQ4Pair + kQ4Chunk + kQ4VOffsets + t * 16 + (g & 3) * 4;
      const uint32_t b0 = *reinterpret_cast<const uint32_t*>(vo), b1 = *reinterpret_cast<const uint32_t*>(vo + 64);
      if (pg == 0) mma_f16_16816_z(d, pa[pg], b0, b1);
      else mma_f16_16816(d, pa[pg], b0, b1);
    }
    oo = f2_fma(oo, al2, f2_pack(d[0], d[1]));
    oo = f2_add(oo, f2_pack(d[2], d[3]));
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      float e[4][4];
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
        for (int n = 0; n < 4; ++n) {
          if (pg == 0) mma_f16_16816_z(e[n], pa[pg], b[0][n], b[1][n]);
          else mma_f16_16816(e[n], pa[pg], b[0][n], b[1][n]);
        }
      }
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        o[w][n] = f2_fma(o[w][n], al2, f2_pack(e[n][0], e[n][1]));
        o[w][n] = f2_add(o[w][n], f2_pack(e[n][2], e[n][3]));
      }
    }
    __syncwarp();  // every lane has read the stage
    if (k + kQ4Stages < n_tiles) issue(k + kQ4Stages);
  }
  if (gave_up) {  // the copies that were issued land before the ring is used again
    for (int k = max(0, issued - kQ4Stages); k < issued; ++k)
      mbar_wait(&full[k % kQ4Stages], (k / kQ4Stages) & 1, a.status, a.timeout_ns);
  }

  l += __shfl_xor_sync(0xffffffffu, l, 1);
  l += __shfl_xor_sync(0xffffffffu, l, 2);
  consumer_bar();  // every warp is done with its ring
  MergeSmem& ms = *reinterpret_cast<MergeSmem*>(smem_q4);
  if (t == 0) {
    ms.m[warp][g] = m;
    ms.l[warp][g] = l;
  }
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const int src = (lane & ~3) | (w >> 1);
    const float olo = __shfl_sync(0xffffffffu, f2_lo(oo), src), ohi = __shfl_sync(0xffffffffu, f2_hi(oo), src);
    const float off = (w & 1) ? ohi : olo;
    float* row = &ms.o[warp][g][32 * w + 8 * t];
    *reinterpret_cast<float4*>(row) =
        make_float4(f2_lo(o[w][0]) + off, f2_lo(o[w][1]) + off, f2_lo(o[w][2]) + off, f2_lo(o[w][3]) + off);
    *reinterpret_cast<float4*>(row + 4) =
        make_float4(f2_hi(o[w][0]) + off, f2_hi(o[w][1]) + off, f2_hi(o[w][2]) + off, f2_hi(o[w][3]) + off);
  }
  consumer_bar();
  combine_and_store<IO16>(ms, a, z, g_kv, item.split, item.nsplit, pool.n_kv, threadIdx.x, s_last,
                    reinterpret_cast<float*>(smem_q4), kQ4RingBytes / 4, s_w);
}

}  // namespace oomattn
