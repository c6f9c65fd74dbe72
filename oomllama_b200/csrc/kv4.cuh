// The 4-bit KV cache: its format, the quantiser, and the kernel that reads
// cached rows back as values (of any cache type).
//
// A page of 16 tokens of one kv head is a chunk of 1280 bytes of K and, right
// behind it (one copy brings both), one of V.  The 128 values of a token are four groups of 32; with x
// the group,
//   s = f16(bf16((max x - min x) * (1/15)))  (f32; 8 significant bits)
//   o = f16(min x + 8 s)
//   c = clamp(rint((x - o) / s) + 8, 0, 15)  (8 where s = 0)
// and the group stands for o + (c - 8) s.  The roundings: codes are taken against
// the rounded o and s, so a value in their range is off by at most half a step s.
// s is off by 2^-8 of itself (bf16) or 2^-25 (where it is an f16 subnormal), which
// moves the range's end by 15 times that, o by 2^-11 |o|: the least and greatest
// value may lie outside by 0.06 s + 2^-11 |o| + 15 * 2^-25.  Together at most
// 0.53 s + 2^-11 |o| + 5e-7.  s has 8 bits so that (c - 8) s, a 4-bit number times
// an 8-bit one, is exact in f16.  A group that holds a NaN reads back as NaN;
// values saturate at +-60000, which keeps s <= 8000 and (c - 8) s <= 64000 finite
// in f16; s rounds to 0 below a range of 15 * 2^-25, and the group reads back as
// its least value.  5 bits per value, against 16: 160 bytes instead of 512 for a
// token's K and V of one kv head.
//
// The codes lie in the order in which the decode kernel's lanes want them as
// tensor-core operands, so that a lane's 64-bit load is its operand and no
// shuffle is needed (lane = 4 g + t, g = lane / 4 = 0..7, t = lane % 4):
//   K: token r (0..15), dims 32 w + 8 t + n (w = group, n = 0..7): nibble n of
//      the 32-bit word at (w / 2) * 512 + r * 32 + t * 8 + (w % 2) * 4;
//      then at 1024 + r * 16 the token's f16 o[0..3], s[0..3].
//   V: token r = 8 h + 2 t + p (p = 0, 1), dims 32 w + 4 g + n (n = 0..3):
//      nibble n of the 16-bit piece at
//      (w / 2) * 512 + h * 256 + g * 32 + t * 8 + (w % 2) * 4 + p * 2;
//      then f16 s at 1024 and o at 1152, each at + h * 64 + t * 16 + w * 4 + p * 2.
#pragma once
#include <cuda_fp16.h>

#include "common.cuh"
#include "params.cuh"
#include "rope_append.cuh"

namespace oomattn {

constexpr int kQ4Chunk = 1280;        // bytes of a (page, kv head) chunk of K or of V
constexpr int kQ4Pair = 2 * kQ4Chunk; // K and V: the step from one (page, kv head) to the next
constexpr int kQ4Meta = 1024;         // its scales and offsets
constexpr int kQ4VOffsets = 1152;     // V: the offsets, behind the scales
constexpr float kQ4Sat = 60000.f;
static_assert(kPageSize == 16 && kHeadDim == 128, "the chunk layout");

enum : int { kKvF32 = 0, kKvBf16 = 1, kKvQ4 = 2 };  // cache types, as OOMATTN_DTYPE_*

__device__ __forceinline__ float min_nan(float a, float b) {
  float y;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}

// Scale and offset of a group from its least and greatest value (NaN in both
// where the group holds one).
__device__ __forceinline__ void q4_params(float lo, float hi, __half& s, __half& o) {
  if (!(lo <= hi)) {  // a NaN
    s = __ushort_as_half(0);
    o = __ushort_as_half(0x7fff);
    return;
  }
  lo = fminf(fmaxf(lo, -kQ4Sat), kQ4Sat);
  hi = fminf(fmaxf(hi, -kQ4Sat), kQ4Sat);
  s = __float2half_rn(__bfloat162float(__float2bfloat16_rn(__fmul_rn(__fsub_rn(hi, lo), 1.f / 15.f))));
  o = __float2half_rn(__fadd_rn(lo, __fmul_rn(8.f, __half2float(s))));
}

// Codes of N values, nibble n = value n.  rint((x - o) / s) by one reciprocal for
// all of them: the product is within 9 * 2^-23 of the quotient, clamped to 9, so it
// rounds to the same integer unless it lies that close to a half; those few
// groups are divided.
template <int N>
__device__ __forceinline__ uint32_t q4_codes(const float* x, float s, float o) {
  uint32_t w = 0;
  if (!(s > 0.f)) {
#pragma unroll
    for (int i = 0; i < N; ++i) w |= 8u << (4 * i);
    return w;
  }
  const float r = __frcp_rn(s);
  bool near = false;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float q = fminf(fmaxf(__fsub_rn(x[i], o) * r, -9.f), 8.f);  // an infinite x gives an end of the range
    const float c = rintf(q);
    near |= fabsf(q - c) > 0.49999f;
    w |= (uint32_t)(int)(fminf(fmaxf(c, -8.f), 7.f) + 8.f) << (4 * i);
  }
  if (near) {
    w = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float c = rintf(__fdiv_rn(__fsub_rn(x[i], o), s));
      w |= (uint32_t)(int)(fminf(fmaxf(c, -8.f), 7.f) + 8.f) << (4 * i);
    }
  }
  return w;
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
// Nonzero where a half of the pair is a NaN (its magnitude's bits above 0x7c00).
__device__ __forceinline__ uint32_t h2_nan(uint32_t a) { return ((a & 0x7fff7fffu) + 0x03ff03ffu) & 0x80008000u; }
// (x & mask) | magic in one instruction (with both as immediates it takes two).
__device__ __forceinline__ uint32_t and_or(uint32_t x, uint32_t mask, uint32_t magic) {
  uint32_t d;
  asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(d) : "r"(x), "r"(mask), "r"(magic));
  return d;
}
// The four pairs of codes of a word that lie 16 bits apart, nibble n of either
// half, as f16 pairs c - 8: 1024 + c or 1024 + 16 c by the bits, then one exact
// step.  magic: 1024.0 in both halves.
__device__ __forceinline__ void q4_centered(uint32_t x, uint32_t magic, uint32_t* h) {
  const uint32_t y = x >> 8;
  h[0] = h2_add(and_or(x, 0x000f000fu, magic), 0xe408e408u);
  h[1] = h2_fma(and_or(x, 0x00f000f0u, magic), 0x2c002c00u, 0xd480d480u);
  h[2] = h2_add(and_or(y, 0x000f000fu, magic), 0xe408e408u);
  h[3] = h2_fma(and_or(y, 0x00f000f0u, magic), 0x2c002c00u, 0xd480d480u);
}

__device__ __forceinline__ float q4_value(uint32_t code, float s, float o) {
  return __fadd_rn(o, __fmul_rn((float)((int)code - 8), s));
}

// Chunk of (layer, page, kv head) in a 4-bit pool, from pool.k or pool.v.
__device__ __forceinline__ size_t q4_chunk_off(const KVPool& pool, int layer, int page, int g) {
  return ((size_t)((size_t)layer * pool.n_pool_pages + page) * pool.n_kv + g) * kQ4Pair;
}

// Byte offsets inside a chunk.
__host__ __device__ __forceinline__ int q4_k_word(int tok, int block) {  // the 8 dims [8 block, 8 block + 8)
  return (block >> 3) * 512 + tok * 32 + (block & 3) * 8 + ((block >> 2) & 1) * 4;
}
__host__ __device__ __forceinline__ int q4_v_pair(int tok, int g, int wp) {  // 8 bytes: tok's pair (tok & ~1, tok | 1), piece g of groups 2 wp, 2 wp + 1
  return wp * 512 + (tok >> 3) * 256 + g * 32 + ((tok >> 1) & 3) * 8;
}
__host__ __device__ __forceinline__ int q4_v_meta(int tok) {  // the pair's 4 x 2 scales (or, at kQ4VOffsets, offsets)
  return (tok >> 3) * 64 + ((tok >> 1) & 3) * 16;
}

// ---------------------------------------------------------------- rows read back
struct GatherArgs {
  void* k_out;
  void* v_out;
  int layer;
  int n;          // tokens per row: slots sb.len[z] .. sb.len[z] + n - 1
  int pages;      // pages a row's range can touch
  int head_rows;  // not 0: out as [n_kv][head_rows][128] from slot 0, zeros at and past slot n
  int* status;
};

enum : int { kOutF32 = 0, kOutBf16 = 1, kOutF16 = 2 };  // f16: by heads, of a 4-bit cache only
template <int OUT>
__device__ __forceinline__ void store4(void* p, size_t i, const float* x) {
  if (OUT == kOutBf16) {
    *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(p) + i) = make_uint2(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]));
  } else {
    *reinterpret_cast<float4*>(reinterpret_cast<float*>(p) + i) = make_float4(x[0], x[1], x[2], x[3]);
  }
}

// LayerKVCache::get (oomllama_turbo.rs:57-63) on the device: the cached rows as
// values.  One CTA of 128 threads per (row, page, kv head): 64 threads read the
// K chunk, 64 the V chunk; a thread's 128-bit load is 32 codes (4-bit cache).
// A 4-bit page is 2.5 KB read for 8 KB (16-bit) written; for the prefill's rows
// the arithmetic is in f16 pairs (9334 tokens of 8 kv heads 14.8 us in f32).
template <int KV, int OUT>
__global__ void __launch_bounds__(128)
    kv_gather_kernel(const GatherArgs a, const KVPool pool, const __grid_constant__ SeqBatch sb) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int g = blockIdx.x % pool.n_kv;
  const int rest = blockIdx.x / pool.n_kv;
  const int z = rest / a.pages;
  const int first = sb.len[z], last = first + a.n;  // slots wanted
  const int lp = first / kPageSize + (rest - z * a.pages);
  const int s0 = lp * kPageSize;
  if (!a.head_rows && s0 >= last) return;
  const bool held = s0 < last;
  int page = pool.n_pool_pages - 1;
  if (held) {
    const int id = lp < pool.max_pages_per_seq ? __ldg(pool.block_table + (size_t)sb.seq[z] * pool.max_pages_per_seq + lp) : -1;
    if ((unsigned)id < (unsigned)pool.n_pool_pages)
      page = id;
    else if (threadIdx.x == 0)
      report_error(a.status, kDevErrBounds);
  }
  const int u = threadIdx.x & 63;
  const bool is_v = threadIdx.x >= 64;
  void* out = is_v ? a.v_out : a.k_out;
  // element offset of (slot, dim) in the output
  auto at = [&](int slot, int d) -> size_t {
    return a.head_rows ? ((size_t)g * a.head_rows + slot) * kHeadDim + d
                       : (((size_t)z * a.n + (slot - first)) * pool.n_kv + g) * kHeadDim + d;
  };
  auto wanted = [&](int slot) { return slot >= first && slot < last; };
  if (KV == kKvQ4) {
    const uint8_t* c = static_cast<const uint8_t*>(is_v ? pool.v : pool.k) + q4_chunk_off(pool, a.layer, page, g);
    const uint4 w4 = *reinterpret_cast<const uint4*>(c + u * 16);
    const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
    const int wp = u >> 5;  // groups 2 wp and 2 wp + 1; the 16 bytes hold t and t + 1 of each
    if (OUT == kOutF16) {
      // in f16 pairs: (c - 8) s is exact, the sum with o rounded once
      uint32_t magic;
      asm volatile("mov.b32 %0, 0x64006400;" : "=r"(magic));
      uint16_t* dst = reinterpret_cast<uint16_t*>(out);
      if (!is_v) {
        const int tok = (u & 31) >> 1, t = (u & 1) * 2, slot = s0 + tok;
        const uint32_t o2 = *reinterpret_cast<const uint32_t*>(c + kQ4Meta + tok * 16 + wp * 4);
        const uint32_t s2 = *reinterpret_cast<const uint32_t*>(c + kQ4Meta + tok * 16 + 8 + wp * 4);
        const uint32_t keep = wanted(slot) ? ~0u : 0u;
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          const uint32_t s = __byte_perm(s2, 0, q ? 0x3232 : 0x1010), o = __byte_perm(o2, 0, q ? 0x3232 : 0x1010);
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            uint32_t h[4];  // dims (0, 4), (1, 5), (2, 6), (3, 7)
            q4_centered(w[2 * e + q], magic, h);
#pragma unroll
            for (int n = 0; n < 4; ++n) h[n] = h2_add(h2_mul(h[n], s), o) & keep;
            *reinterpret_cast<uint4*>(dst + at(slot, 32 * (2 * wp + q) + 8 * (t + e))) =
                make_uint4(__byte_perm(h[0], h[1], 0x5410), __byte_perm(h[2], h[3], 0x5410),
                           __byte_perm(h[0], h[1], 0x7632), __byte_perm(h[2], h[3], 0x7632));
          }
        }
      } else {
        const int h8 = (u >> 4) & 1, gg = (u >> 1) & 7;
#pragma unroll
        for (int tt = 0; tt < 2; ++tt) {
          const int t = (u & 1) * 2 + tt, slot = s0 + 8 * h8 + 2 * t;
          const uint2 s4 = *reinterpret_cast<const uint2*>(c + kQ4Meta + h8 * 64 + t * 16 + wp * 8);
          const uint2 o4 = *reinterpret_cast<const uint2*>(c + kQ4VOffsets + h8 * 64 + t * 16 + wp * 8);
          const uint32_t keep = (wanted(slot) ? 0xffffu : 0u) | (wanted(slot + 1) ? 0xffff0000u : 0u);
          // a NaN group would reach queries that do not see its token, as 0 * NaN
          if ((h2_nan(o4.x & keep) | h2_nan(o4.y & keep)) != 0) report_error(a.status, kDevErrRange);
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            uint32_t h[4];  // dim n of both tokens
            q4_centered(w[2 * tt + q], magic, h);
#pragma unroll
            for (int n = 0; n < 4; ++n) h[n] = h2_add(h2_mul(h[n], q ? s4.y : s4.x), q ? o4.y : o4.x) & keep;
            const int d = 32 * (2 * wp + q) + 4 * gg;
            *reinterpret_cast<uint2*>(dst + at(slot, d)) = make_uint2(__byte_perm(h[0], h[1], 0x5410), __byte_perm(h[2], h[3], 0x5410));
            *reinterpret_cast<uint2*>(dst + at(slot + 1, d)) = make_uint2(__byte_perm(h[0], h[1], 0x7632), __byte_perm(h[2], h[3], 0x7632));
          }
        }
      }
    } else if (!is_v) {
      const int tok = (u & 31) >> 1, t = (u & 1) * 2, slot = s0 + tok;
      const uint32_t o2 = *reinterpret_cast<const uint32_t*>(c + kQ4Meta + tok * 16 + wp * 4);
      const uint32_t s2 = *reinterpret_cast<const uint32_t*>(c + kQ4Meta + tok * 16 + 8 + wp * 4);
      if (!wanted(slot)) return;
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const float o = __half2float(__ushort_as_half((uint16_t)(o2 >> (16 * q))));
        const float s = __half2float(__ushort_as_half((uint16_t)(s2 >> (16 * q))));
#pragma unroll
        for (int e = 0; e < 2; ++e) {  // t and t + 1 of this group: 16 dims in a row
          float x[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) x[i] = q4_value((w[2 * e + q] >> (4 * i)) & 15u, s, o);
          store8<OUT == kOutBf16>(out, at(slot, 32 * (2 * wp + q) + 8 * (t + e)), x);
        }
      }
    } else {
      const int h = (u >> 4) & 1, gg = (u >> 1) & 7;
#pragma unroll
      for (int tt = 0; tt < 2; ++tt) {
        const int t = (u & 1) * 2 + tt;
        const uint2 s4 = *reinterpret_cast<const uint2*>(c + kQ4Meta + h * 64 + t * 16 + wp * 8);
        const uint2 o4 = *reinterpret_cast<const uint2*>(c + kQ4VOffsets + h * 64 + t * 16 + wp * 8);
#pragma unroll
        for (int p = 0; p < 2; ++p) {
          const int slot = s0 + 8 * h + 2 * t + p;
          if (!wanted(slot)) continue;
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            const float o = __half2float(__ushort_as_half((uint16_t)((q ? o4.y : o4.x) >> (16 * p))));
            const float s = __half2float(__ushort_as_half((uint16_t)((q ? s4.y : s4.x) >> (16 * p))));
            float x[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = q4_value((w[2 * tt + q] >> (16 * p + 4 * i)) & 15u, s, o);
            store4<OUT>(out, at(slot, 32 * (2 * wp + q) + 4 * gg), x);
          }
        }
      }
    }
  } else {
    constexpr int es = KV == kKvBf16 ? 2 : 4;
    const uint8_t* c = static_cast<const uint8_t*>(is_v ? pool.v : pool.k) +
                       (((size_t)a.layer * pool.n_pool_pages + page) * pool.n_kv + g) * (size_t)(kPageSize * kHeadDim * es);
    for (int i = u; i < kPageSize * kHeadDim / 4; i += 64) {
      const int slot = s0 + i / (kHeadDim / 4), d = (i % (kHeadDim / 4)) * 4;
      if (!wanted(slot)) continue;
      float x[4];
      if (KV == kKvBf16) {
        const uint2 v = *reinterpret_cast<const uint2*>(c + (size_t)i * 8);
        x[0] = bf16_lo_f32(v.x); x[1] = bf16_hi_f32(v.x); x[2] = bf16_lo_f32(v.y); x[3] = bf16_hi_f32(v.y);
      } else {
        const float4 v = *reinterpret_cast<const float4*>(c + (size_t)i * 16);
        x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
      }
      store4<OUT>(out, at(slot, d), x);
    }
  }
}

}  // namespace oomattn
