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
// Tiles.  m16n8k16 with keys (K) or dims (V) as the 16 rows and query heads as
// the 8 columns; a query (or probability) enters as an f16 high part and a low
// one (x - high), 22 bits of the f32 value together.  Probabilities are held at
// 2^14 times their size (kQ4PBias): f16 ends at 2^-24, so a weight keeps its 22
// bits down to 2^-16 of the largest and is off by 2^-39 of it at most below that.
// (At their own size all below 2^-25 were lost from O but not from the sum l:
// beside a key 17.5 nats above 8191 others, a quarter of what those carry.)
// A group of up to four heads (WIDE = false) has both parts side by side, column
// 2 h the high part of head h, column 2 h + 1 the low: one product does both, and
// the two columns of an accumulator lie in one lane.  A group of five to eight
// (WIDE) has a column per head and a second product for the low parts.  (Heads as
// rows, eight high and eight low, would cost a group of four as many products as
// one of eight: 96.2 instead of 66.7 us for 8 x 32768 tokens of 32q/8kv.)
// K codes enter as subnormal halves (code * 2^-24, or 2^-20 for the upper nibble
// of a byte, whose q is prescaled by 1/16): unpacking is one AND per two codes.
// q is scaled by a power of two to [2^14, 2^15) per head, and its high part put
// on a grid on which the products' sums are exact (q_part).
// The P V products of a 32-token tile start from zero and are added to O in
// f32 (one packed FMA with the softmax rescale): the tensor core truncates
// when it accumulates, which over a long context would shrink O.
//
// Each warp works alone: its own ring of tiles in shared memory, filled by
// bulk copies (one of 2560 bytes per page: K, then V) that two of its lanes issue,
// its own running maximum and sum; the four warps of a CTA join at the end.
//
// Measured: 8 x 32768 tokens of 32q/8kv (335 MB) in 65 us, 5.13 TB/s, 0.78 of
// the copy rate (75 us under the 1000 W cap, 1.70 GHz, in a loop of seconds); 64
// ragged rows of 28q/4kv (209 MB) in 62 us, 0.51.  Copies alone take 53 and 38
// us, the arithmetic alone 58 and 52: about 320 (narrow) and 400 (wide)
// instructions per warp and 16 tokens -- 40 + 104 to unpack K and V, 18 or 36
// tensor products of 8.4 cycles each, which overlap the ALU and f16 pipes only
// in part (16 products with 64 LOP3 and 64 HMUL2: 196 cycles; 136, 126 and 125
// alone).  Neither two tiles in flight in one warp, nor 16 warps of the wide form
// (it spills), nor e4m3 digits of q (an exact product of K = 32, but slow as
// mma.sync) made it faster.
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
// The narrow form has 128 registers (8 bytes spilled) and the wide one 168: four
// CTAs of two stages each, or three of three, per SM -- about 160 and 180 KB in flight.
__host__ __device__ constexpr int q4_stages(bool wide) { return !wide ? 2 : 3; }
__host__ __device__ constexpr int q4_ctas_per_sm(bool wide) { return !wide ? 4 : 3; }
// The running maximum that weights are taken against lies this far (base 2) below
// the largest logit: weights in (0, 2^14], and so l and O, which cancels in O / l
// and in the lse.  It is rounded up, so that no weight passes 2^14 where a unit of
// its last place is large (logits of 2^25 and more), which f16 would not hold.
constexpr int kQ4PBias = 14;
__host__ __device__ constexpr int q4_ring_bytes(bool wide) { return kDecWarps * q4_stages(wide) * kQ4TileBytes; }
__host__ __device__ constexpr int q4_tail_bytes(bool wide) {  // barriers, a flag, merge weights
  return kDecWarps * q4_stages(wide) * 8 + 64 + kMaxGroup * 32 * 4;
}
__host__ __device__ constexpr int q4_smem_bytes(bool wide) {  // and the query
  return q4_ring_bytes(wide) + q4_tail_bytes(wide) + (wide ? 4096 : 2048);
}
static_assert(q4_tail_bytes(false) % 16 == 0 && q4_tail_bytes(true) % 16 == 0, "the query's alignment");
static_assert(sizeof(MergeSmem) <= q4_ring_bytes(false), "the merge is staged over the ring");

__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                   smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}
__device__ __forceinline__ void mma_f16_16816(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_f16_1688(float* d, uint32_t a0, uint32_t a1, uint32_t b0) {
  asm volatile(
      "mma.sync.aligned.m16n8k8.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5}, {%6}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(b0));
}
// The same from zero: the accumulator's registers need no clearing.
__device__ __forceinline__ void mma_f16_16816_z(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ void mma_f16_1688_z(float* d, uint32_t a0, uint32_t a1, uint32_t b0) {
  asm volatile(
      "mma.sync.aligned.m16n8k8.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5}, {%6}, {%7,%7,%7,%7};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(b0), "f"(0.f));
}
__device__ __forceinline__ float h_lo(uint32_t v) { return __half2float(__ushort_as_half((uint16_t)v)); }
__device__ __forceinline__ float h_hi(uint32_t v) { return __half2float(__ushort_as_half((uint16_t)(v >> 16))); }
// (a, b) rounded to f16, or (low) what that rounding leaves: exact in f32, rounded once.
__device__ __forceinline__ uint32_t f16_part(float a, float b, bool low) {
  const uint32_t hi = pack_f16(a, b);
  return low ? pack_f16(a - h_lo(hi), b - h_hi(hi)) : hi;
}
// The query's parts times `by` (1 or 1/16), |a|, |b| < 2^15: the high part a
// multiple of 16, so that its products with 32 codes add up to less than 2^20
// such units and the tensor core's accumulator holds the sum exactly (it
// truncates: with the high part rounded to its own 11 bits the decode's error
// was twice as large); the low part, at most 8, is rounded to 2^-9.
__device__ __forceinline__ uint32_t q_part(float a, float b, float by, bool low) {
  const float ha = rintf(a * 0.0625f) * 16.f, hb = rintf(b * 0.0625f) * 16.f;
  return low ? pack_f16((a - ha) * by, (b - hb) * by) : pack_f16(ha * by, hb * by);
}

// Q16, OUT16: q and out in bf16 (the newest tokens of a sequence as one row each)
// instead of f32 (a generation step).
template <bool WIDE, bool Q16, bool OUT16>
__global__ void __launch_bounds__(kDecWarps * 32, q4_ctas_per_sm(WIDE))
    decode_q4_kernel(const KVPool pool, const DecodeArgs a, const __grid_constant__ SeqBatch sb,
                     const __grid_constant__ DecodeSched sched) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // as in decode_bf16_kernel
  constexpr int kStages = q4_stages(WIDE), kRing = q4_ring_bytes(WIDE);
  extern __shared__ __align__(128) uint8_t smem_q4[];
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem_q4 + kRing);
  int* s_last = reinterpret_cast<int*>(bars + kDecWarps * kStages);
  float* s_w = reinterpret_cast<float*>(s_last + 16);  // [kMaxGroup][32] merge weights
  uint4* s_q = reinterpret_cast<uint4*>(smem_q4 + kRing + q4_tail_bytes(WIDE));  // [4][parts][32]: the query

  const DecodeItem item = decode_item(sched, sb, blockIdx.x);
  const int g_kv = item.g, z = item.z;
  const int seq = sb.seq[z], L = sb.len[z];
  const int pb = item.pb, pe = item.pe;
  if (pb >= pe) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (!OUT16 && L <= 0 && item.split == 0) write_empty_row(a, z, g_kv);  // a bf16 row sees its own token at least
    return;
  }
  const int warp = threadIdx.x >> 5;
  int lane;  // kept in a register
  asm volatile("mov.u32 %0, %%laneid;" : "=r"(lane));
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
  // Launched as a programmatic dependent of the kernel before it (the append):
  // while that one finishes, the first tiles' pages are pulled into L2 (20 lines
  // of 128 bytes each); q and the cache are read only after it.
#pragma unroll
  for (int j = 0; j < kStages * kQ4Pages; ++j) {
    const int id = __shfl_sync(0xffffffffu, ids, j);
    if (id >= 0 && lane < kQ4Pair / 128)
      asm volatile("prefetch.global.L2 [%0];" ::"l"(base + (size_t)(uint32_t)id * page_bytes + lane * 128));
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");
  for (int k = 0; k < min(kStages, n_tiles); ++k) issue(k, k);

  // ---- the query as B operand: lane (g, t) holds column g at dims 32 w + 8 t +
  // 0..7; product j of group w meets K nibbles (2j | 2j + 4) and (2j + 1 | 2j + 5)
  // of the word.  Wide: both parts of head g.  Narrow: a part of head g / 2.
  constexpr int HL = WIDE ? 2 : 1;  // heads of a lane's accumulators: 2 t and 2 t + 1, or t
  // It stays in shared memory (one copy for the CTA's warps) and is read per tile.
  uint32_t bm[HL];
  float f2[HL];  // score * f2 is the base-2 logit
  {
    const int j = WIDE ? g : g >> 1;
    const bool valid = j < a.group;
    const size_t q0 = ((size_t)z * a.n_heads + g_kv * a.group + (valid ? j : 0)) * kHeadDim;
    float x[4][8];
    float mx = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      load8<Q16>(a.q, q0 + 32 * w + 8 * t, x[w]);
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
#pragma unroll
    for (int h = 0; h < HL; ++h) f2[h] = __shfl_sync(0xffffffffu, f2_own, 8 * t + 4 * h);
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
    }
    // rows [o0 o1 | o2 o3 | s0 s1 | s2 s3] of the token's stored numbers, lane t has its two
    const float m8 = t < 2 ? 1.f : -8.f;
    const float u0 = ((t & 1) ? qs[2] : qs[0]) * m8, u1 = ((t & 1) ? qs[3] : qs[1]) * m8;
#pragma unroll
    for (int h = 0; h < HL; ++h) {
      const bool low = WIDE ? h == 1 : (g & 1) != 0;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        uint32_t v[4];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          v[2 * i] = q_part(x[w][2 * i], x[w][2 * i + 4], 1.f, low);
          v[2 * i + 1] = q_part(x[w][2 * i + 1], x[w][2 * i + 5], 0.0625f, low);
        }
        if (warp == 0) s_q[(w * HL + h) * 32 + lane] = make_uint4(v[0], v[1], v[2], v[3]);
      }
      bm[h] = f16_part(u0, u1, low);
    }
    consumer_bar();
  }

  // O of the lane: dims 32 w + 4 g + 2 i + r.  Wide: [w][2 i + r] of heads (2 t, 2 t + 1);
  // narrow: [w][i] of head t, r = 0 and 1.  oo: sum p * offset of groups 2 (g % 2) and + 1.
  uint64_t o[4][2 * HL];
  float oo[HL][2], m[HL], l[HL];  // m: the running maximum as a base-2 logit, less kQ4PBias
#pragma unroll
  for (int w = 0; w < 4; ++w)
#pragma unroll
    for (int i = 0; i < 2 * HL; ++i) o[w][i] = 0;
#pragma unroll
  for (int h = 0; h < HL; ++h) {
    oo[h][0] = oo[h][1] = 0.f;
    m[h] = -INFINITY;
    l[h] = 0.f;
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
    // ---- scores of 2 x 16 tokens: rows g and g + 8 of a page, the lane's heads
    float sc[HL][4];
#pragma unroll
    for (int pg = 0; pg < 2; ++pg) {
      const uint8_t* kc = st + pg * kQ4Pair;
      const uint32_t am0 = *reinterpret_cast<const uint32_t*>(kc + kQ4Meta + g * 16 + t * 4);
      const uint32_t am1 = *reinterpret_cast<const uint32_t*>(kc + kQ4Meta + (g + 8) * 16 + t * 4);
      float d[4];
      mma_f16_1688_z(d, am0, am1, bm[0]);
      if (WIDE) {
        mma_f16_1688(d, am0, am1, bm[HL - 1]);
        sc[0][2 * pg] = d[0] * (1.f / 4096.f);  // 2^-24 / 2^-12
        sc[HL - 1][2 * pg] = d[1] * (1.f / 4096.f);
        sc[0][2 * pg + 1] = d[2] * (1.f / 4096.f);
        sc[HL - 1][2 * pg + 1] = d[3] * (1.f / 4096.f);
      } else {
        sc[0][2 * pg] = (d[0] + d[1]) * (1.f / 4096.f);
        sc[0][2 * pg + 1] = (d[2] + d[3]) * (1.f / 4096.f);
      }
    }
#pragma unroll
    for (int wp = 0; wp < 2; ++wp) {  // two groups at a time: 64-bit loads of rows g and g + 8
      uint2 wk[4];
      uint32_t sk[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint8_t* kc = st + (i >> 1) * kQ4Pair;
        wk[i] = *reinterpret_cast<const uint2*>(kc + wp * 512 + (i & 1) * 256 + lane * 8);
        sk[i] = *reinterpret_cast<const uint32_t*>(kc + kQ4Meta + (g + 8 * (i & 1)) * 16 + 8 + wp * 4);
      }
#pragma unroll
      for (int wl = 0; wl < 2; ++wl) {
        const int w = 2 * wp + wl;
        const uint4 q0 = s_q[w * HL * 32 + lane], q1 = s_q[(w * HL + HL - 1) * 32 + lane];
#pragma unroll
        for (int pg = 0; pg < 2; ++pg) {
          const uint32_t xa = wl ? wk[2 * pg].y : wk[2 * pg].x, xb = wl ? wk[2 * pg + 1].y : wk[2 * pg + 1].x;
          const uint32_t ya = xa >> 8, yb = xb >> 8;
          const uint32_t f0[4] = {xa & 0x000f000fu, xb & 0x000f000fu, xa & 0x00f000f0u, xb & 0x00f000f0u};
          const uint32_t f1[4] = {ya & 0x000f000fu, yb & 0x000f000fu, ya & 0x00f000f0u, yb & 0x00f000f0u};
          const float s0 = wl ? h_hi(sk[2 * pg]) : h_lo(sk[2 * pg]), s1 = wl ? h_hi(sk[2 * pg + 1]) : h_lo(sk[2 * pg + 1]);
          float e[4];
          mma_f16_16816_z(e, f0, q0.x, q0.y);
          mma_f16_16816(e, f1, q0.z, q0.w);
          if (WIDE) {  // the low parts by themselves: added onto the high ones they would be truncated at those' size
            float el[4];
            mma_f16_16816_z(el, f0, q1.x, q1.y);
            mma_f16_16816(el, f1, q1.z, q1.w);
            sc[0][2 * pg] = fmaf(el[0], s0, sc[0][2 * pg]);
            sc[HL - 1][2 * pg] = fmaf(el[1], s0, sc[HL - 1][2 * pg]);
            sc[0][2 * pg + 1] = fmaf(el[2], s1, sc[0][2 * pg + 1]);
            sc[HL - 1][2 * pg + 1] = fmaf(el[3], s1, sc[HL - 1][2 * pg + 1]);
          }
          sc[0][2 * pg] = fmaf(e[0], s0, sc[0][2 * pg]);
          sc[HL - 1][2 * pg] = fmaf(e[1], s0, sc[HL - 1][2 * pg]);
          sc[0][2 * pg + 1] = fmaf(e[2], s1, sc[0][2 * pg + 1]);
          sc[HL - 1][2 * pg + 1] = fmaf(e[3], s1, sc[HL - 1][2 * pg + 1]);
        }
      }
    }
    if (lim < kQ4Tile) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (8 * i + g >= lim) {
#pragma unroll
          for (int h = 0; h < HL; ++h) sc[h][i] = -INFINITY;
        }
    }
    // ---- online softmax of the lane's heads over the tile
    float alpha[HL];
#pragma unroll
    for (int h = 0; h < HL; ++h) {
      float mt = fmaxf(max3f(sc[h][0], sc[h][1], sc[h][2]), sc[h][3]);
#pragma unroll
      for (int off = 4; off < 32; off <<= 1) mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, off));
      // the running maximum is rounded (up): the same number enters every weight, so its rounding cancels
      const float mf = fmaxf(m[h], __fmaf_ru(mt, f2[h], -(float)kQ4PBias));
      alpha[h] = ex2_ftz(m[h] - mf);
      m[h] = mf;
      float ps = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        sc[h][i] = ex2_ftz(fmaf(sc[h][i], f2[h], -mf));
        ps += sc[h][i];
      }
      l[h] = fmaf(l[h], alpha[h], ps);
    }
    // as B operands: token row g, columns (2 t, 2 t + 1), transposed into tokens 2 t, 2 t + 1 of column g
    uint32_t pb[HL][4];  // wide: high, low; narrow: both in one
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (WIDE) {
        const uint32_t hi = pack_f16(sc[0][i], sc[HL - 1][i]);
        pb[0][i] = movmatrix_trans(hi);
        pb[HL - 1][i] = movmatrix_trans(pack_f16(sc[0][i] - h_lo(hi), sc[HL - 1][i] - h_hi(hi)));
      } else {
        pb[0][i] = movmatrix_trans(pack_f16(sc[0][i], sc[0][i] - h_lo(pack_f16(sc[0][i], 0.f))));
      }
    }
    // ---- O = O * alpha + V^T P
    {
      float d[4];
#pragma unroll
      for (int pg = 0; pg < 2; ++pg) {
        // offsets as A operand: row g is group 2 (g % 2), row g + 8 the one after
        const uint8_t* vo = st + pg * kQ4Pair + kQ4Chunk + kQ4VOffsets + t * 16 + (g & 1) * 8;
        const uint2 o0 = *reinterpret_cast<const uint2*>(vo), o1 = *reinterpret_cast<const uint2*>(vo + 64);
        const uint32_t ao[4] = {o0.x, o0.y, o1.x, o1.y};
        if (pg == 0) mma_f16_16816_z(d, ao, pb[0][0], pb[0][1]);
        else mma_f16_16816(d, ao, pb[0][2], pb[0][3]);
        if (WIDE) mma_f16_16816(d, ao, pb[HL - 1][2 * pg], pb[HL - 1][2 * pg + 1]);
      }
      if (WIDE) {
        oo[0][0] = fmaf(oo[0][0], alpha[0], d[0]);
        oo[HL - 1][0] = fmaf(oo[HL - 1][0], alpha[HL - 1], d[1]);
        oo[0][1] = fmaf(oo[0][1], alpha[0], d[2]);
        oo[HL - 1][1] = fmaf(oo[HL - 1][1], alpha[HL - 1], d[3]);
      } else {
        oo[0][0] = fmaf(oo[0][0], alpha[0], d[0] + d[1]);
        oo[0][1] = fmaf(oo[0][1], alpha[0], d[2] + d[3]);
      }
    }
    const uint64_t al2 = f2_pack(alpha[0], alpha[HL - 1]);
#pragma unroll
    for (int wp = 0; wp < 2; ++wp) {
      uint2 vw[4], vs[4];  // [page, half]: two groups' codes and scales of the lane's token pair
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint8_t* vc = st + (i >> 1) * kQ4Pair + kQ4Chunk;
        vw[i] = *reinterpret_cast<const uint2*>(vc + wp * 512 + (i & 1) * 256 + lane * 8);
        vs[i] = *reinterpret_cast<const uint2*>(vc + kQ4Meta + (i & 1) * 64 + t * 16 + wp * 8);
      }
#pragma unroll
      for (int wl = 0; wl < 2; ++wl) {
        const int w = 2 * wp + wl;
        float e[2][4];
#pragma unroll
        for (int pg = 0; pg < 2; ++pg) {
          uint32_t b[2][4];  // [half][n]
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint32_t x = wl ? vw[2 * pg + h].y : vw[2 * pg + h].x;
            const uint32_t s2 = wl ? vs[2 * pg + h].y : vs[2 * pg + h].x;
            q4_centered(x, magic, b[h]);
#pragma unroll
            for (int n = 0; n < 4; ++n) b[h][n] = h2_mul(b[h][n], s2);  // exact: 4 bits times 8
          }
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const uint32_t av[4] = {b[0][2 * i], b[0][2 * i + 1], b[1][2 * i], b[1][2 * i + 1]};
            if (pg == 0) mma_f16_16816_z(e[i], av, pb[HL - 1][0], pb[HL - 1][1]);
            else mma_f16_16816(e[i], av, pb[HL - 1][2], pb[HL - 1][3]);
            if (WIDE) mma_f16_16816(e[i], av, pb[0][2 * pg], pb[0][2 * pg + 1]);
          }
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          if (WIDE) {
            o[w][2 * i] = f2_fma(o[w][2 * i], al2, f2_pack(e[i][0], e[i][1]));
            o[w][2 * i + HL - 1] = f2_fma(o[w][2 * i + HL - 1], al2, f2_pack(e[i][2], e[i][3]));
          } else {
            o[w][i] = f2_fma(o[w][i], al2, f2_pack(e[i][0] + e[i][1], e[i][2] + e[i][3]));
          }
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
  for (int h = 0; h < HL; ++h)
#pragma unroll
    for (int off = 4; off < 32; off <<= 1) l[h] += __shfl_xor_sync(0xffffffffu, l[h], off);
  consumer_bar();  // every warp is done with its ring
  MergeSmem& ms = *reinterpret_cast<MergeSmem*>(smem_q4);
#pragma unroll
  for (int h = 0; h < HL; ++h) {
    const int head = HL * t + h;
    if (g == 0) {
      ms.m[warp][head] = m[h];
      ms.l[warp][head] = l[h];
    }
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float off = __shfl_sync(0xffffffffu, oo[h][w & 1], 4 * (w >> 1) + t);
      float x[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint64_t v = WIDE ? o[w][i & (2 * HL - 1)] : o[w][i >> 1];
        x[i] = ((WIDE ? h : i & 1) ? f2_hi(v) : f2_lo(v)) + off;
      }
      *reinterpret_cast<float4*>(&ms.o[warp][head][32 * w + 4 * g]) = make_float4(x[0], x[1], x[2], x[3]);
    }
  }
  consumer_bar();
  combine_and_store<OUT16, true, kQ4PBias>(ms, a, z, g_kv, item.split, item.nsplit, pool.n_kv, threadIdx.x, s_last,
                          reinterpret_cast<float*>(smem_q4), kRing / 4, s_w);
}

// The merge of a launch whose rows do not fill the GPU, with up to kMaxSplitsQ4
// splits: a kernel of its own, one CTA per (row, q head, 32 dims).  A warp takes
// four splits at a time, eight lanes with four dims each; weights 2^(lse - max)
// and the sums as in merge_splits_staged, in a fixed order.  Rows with a single
// split were written by the decode kernel.
constexpr int kMergeWarps = 16;
template <bool OUT16>
__global__ void __launch_bounds__(kMergeWarps * 32)
    merge_splits_kernel(const DecodeArgs a, const __grid_constant__ SeqBatch sb, const __grid_constant__ DecodeSched sched) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  __shared__ float s_wt[kMaxSplitsQ4];
  __shared__ float s_red[2][kMergeWarps];
  __shared__ float4 s_acc[kMergeWarps][8];
  const int r = blockIdx.x / a.n_heads, h = blockIdx.x - r * a.n_heads;
  const int z = sched.order[r];
  const int n_pages = (sb.len[z] + kPageSize - 1) / kPageSize;
  const int pps = n_pages > 0 ? (n_pages + sched.nsplit[r] - 1) / sched.nsplit[r] : 0;
  const int ns = pps > 0 ? (n_pages + pps - 1) / pps : 1;  // as decode_item
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (ns <= 1) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const size_t zh = (size_t)z * a.n_heads + h, p0 = zh * a.max_splits;
  static_assert(kMaxSplitsQ4 <= kMergeWarps * 32, "one split weight per thread");
  const float ls = (int)threadIdx.x < ns ? __ldcg(a.part_lse + p0 + threadIdx.x) : -INFINITY;
  float M = ls;
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, off));
  if (lane == 0) s_red[0][warp] = M;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kMergeWarps; ++w) M = fmaxf(M, s_red[0][w]);
  const float wt = ls == -INFINITY ? 0.f : exp2f(ls - M);
  s_wt[threadIdx.x] = wt;
  float sum = wt;
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
  if (lane == 0) s_red[1][warp] = sum;
  __syncthreads();
  sum = 0.f;
#pragma unroll
  for (int w = 0; w < kMergeWarps; ++w) sum += s_red[1][w];
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  const int sub = lane >> 3, d = blockIdx.y * 32 + (lane & 7) * 4;
#pragma unroll 8
  for (int s = warp * 4 + sub; s < ns; s += kMergeWarps * 4) {
    const float4 v = __ldcg(reinterpret_cast<const float4*>(a.part_o + (p0 + s) * kHeadDim + d));
    const float w = s_wt[s];
    acc.x += w * v.x; acc.y += w * v.y; acc.z += w * v.z; acc.w += w * v.w;
  }
#pragma unroll
  for (int off = 8; off < 32; off <<= 1) {
    acc.x += __shfl_xor_sync(0xffffffffu, acc.x, off);
    acc.y += __shfl_xor_sync(0xffffffffu, acc.y, off);
    acc.z += __shfl_xor_sync(0xffffffffu, acc.z, off);
    acc.w += __shfl_xor_sync(0xffffffffu, acc.w, off);
  }
  if (sub == 0) s_acc[warp][lane] = acc;
  __syncthreads();
  if (warp != 0 || sub != 0) return;
#pragma unroll
  for (int w = 1; w < kMergeWarps; ++w) {
    const float4 v = s_acc[w][lane];
    acc.x += v.x; acc.y += v.y; acc.z += v.z; acc.w += v.w;
  }
  const float inv = 1.f / sum;
  store_out4<OUT16>(a, zh, d, acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
  if (a.lse && blockIdx.y == 0 && lane == 0) a.lse[zh * a.lse_stride] = (M + log2f(sum)) * 0.69314718055994531f;
}

}  // namespace oomattn
