// K-A with a norm of every q and k head and any cache type, in one pass over
// the projected rows:
//   y = x + b;  q, k: y = y / sqrt(mean(y^2) + eps) * w  (over the head's 128
//   values, f32), then the rotation of rope_append.cuh;  k, v: the paged append
//   (f32, bf16 or 4-bit).
// The norm is the one that models with normalised heads put between the
// projection's bias and RoPE; a kernel of its own would read and write q and k
// once more (for a 4096-token prompt of 28 + 4 heads in bf16, 67 MB more).
// Measured on that prompt (70 MB, floor 10.6 us): 23.2 us into the 4-bit cache,
// 18.0 us into a bf16 one (76 MB, 11.5); without a norm rope_append_kernel takes
// 14.0.  Bound by the latency of its loads (ncu: long scoreboard 3.5 of 9 stall
// cycles, issue 2.6 of 4, DRAM 17 %): four CTAs per SM at 64 registers (4 bytes
// spilled into a 4-bit cache) were the best of three to six.  64 tokens of 32q/8kv take 7.3 us with the gather of
// their rows, launch latency.
#pragma once
#include "common.cuh"
#include "kv4.cuh"
#include "params.cuh"
#include "rope_append.cuh"

namespace oomattn {

constexpr int kQkNormWarps = 8;      // per CTA
constexpr int kQkNormCtasPerSm = 4;

struct NormArgs {
  const float* qw;  // [128] or null: no norm
  const float* kw;
  float eps;
};

// The norm of one head, its 128 values spread over 8 lanes with 16 each (in a, b).
__device__ __forceinline__ void head_norm(float* a, float* b, const float* w, int e0, int e1, float eps) {
  float ss = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) ss += a[i] * a[i] + b[i] * b[i];
#pragma unroll
  for (int off = 1; off < 8; off <<= 1) ss += __shfl_xor_sync(0xffffffffu, ss, off);
  const float inv = __fdiv_rn(1.f, sqrtf(ss * (1.f / kHeadDim) + eps));
  float wa[8], wb[8];
  load8<false>(w, e0, wa);
  load8<false>(w, e1, wb);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    a[i] = a[i] * inv * wa[i];
    b[i] = b[i] * inv * wb[i];
  }
}

// K of two heads of a token into a 4-bit cache: sixteen lanes per head, lane l
// (of the sixteen) with elements 4l.. and 64 + 4l.., which close under either
// rotation and lie in groups l / 8 and 2 + l / 8.  In f64 up to the codes: a code
// hangs on which side of a border a value lies, and with f32 roundings on the way
// about one in a million lands on the other.  (f64 runs at half the f32 rate
// here; with a lane's 16 values of the other sections it would take 196
// registers.)
template <bool IN_BF16>
__device__ __forceinline__ void append_k_q4(const AppendArgs& ap, const NormArgs& na, const KVPool& pool, int t,
                                            int head0, int pos, int page, int tok, int lane) {
  const int l = lane & 15, head = min(head0, pool.n_kv - 1);
  const int e0 = 4 * l, e1 = 64 + 4 * l;
  const size_t base = ((size_t)t * pool.n_kv + head) * kHeadDim;
  auto four = [&](const float* p, float* y) {
    const float4 v = *reinterpret_cast<const float4*>(p);
    y[0] = v.x; y[1] = v.y; y[2] = v.z; y[3] = v.w;
  };
  float y[8];
  if (IN_BF16) {
    const uint16_t* p = reinterpret_cast<const uint16_t*>(ap.k) + base;
    const uint2 u = *reinterpret_cast<const uint2*>(p + e0), v = *reinterpret_cast<const uint2*>(p + e1);
    y[0] = bf16_lo_f32(u.x); y[1] = bf16_hi_f32(u.x); y[2] = bf16_lo_f32(u.y); y[3] = bf16_hi_f32(u.y);
    y[4] = bf16_lo_f32(v.x); y[5] = bf16_hi_f32(v.x); y[6] = bf16_lo_f32(v.y); y[7] = bf16_hi_f32(v.y);
  } else {
    four(reinterpret_cast<const float*>(ap.k) + base + e0, y);
    four(reinterpret_cast<const float*>(ap.k) + base + e1, y + 4);
  }
  if (ap.bk || na.kw || ap.rope_k) {
    double x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = y[i];
    float f[8];
    if (ap.bk) {
      four(ap.bk + head * kHeadDim + e0, f);
      four(ap.bk + head * kHeadDim + e1, f + 4);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] += f[i];
    }
    if (na.kw) {
      double ss = 0.;
#pragma unroll
      for (int i = 0; i < 8; ++i) ss += x[i] * x[i];
#pragma unroll
      for (int off = 1; off < 16; off <<= 1) ss += __shfl_xor_sync(0xffffffffu, ss, off);
      const double inv = rsqrt(ss * (1. / kHeadDim) + (double)na.eps);
      four(na.kw + e0, f);
      four(na.kw + e1, f + 4);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] *= inv * f[i];
    }
    if (ap.rope_k) {
      const bool split = ap.variant == 0;
      auto turn = [](double& a, double& b, double c, double s) {
        const double z = a * c - b * s;
        b = a * s + b * c;
        a = z;
      };
      // split-half: pairs (k, 4 + k) are 4l + k; interleaved: (2k, 2k + 1) are 2l + k, of the upper half 32 + 2l + k
      const size_t p0 = (size_t)pos * 64 + (split ? 4 * l : 2 * l), p1 = p0 + (split ? 2 : 32);
      const float2 c0 = *reinterpret_cast<const float2*>(ap.cos_t + p0), c1 = *reinterpret_cast<const float2*>(ap.cos_t + p1);
      const float2 s0 = *reinterpret_cast<const float2*>(ap.sin_t + p0), s1 = *reinterpret_cast<const float2*>(ap.sin_t + p1);
      if (split) {
        turn(x[0], x[4], c0.x, s0.x);
        turn(x[1], x[5], c0.y, s0.y);
        turn(x[2], x[6], c1.x, s1.x);
        turn(x[3], x[7], c1.y, s1.y);
      } else {
        turn(x[0], x[1], c0.x, s0.x);
        turn(x[2], x[3], c0.y, s0.y);
        turn(x[4], x[5], c1.x, s1.x);
        turn(x[6], x[7], c1.y, s1.y);
      }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = (float)x[i];
  }
  // least and greatest of both groups over their eight lanes: even lanes go on with the lower group, odd ones with
  // the upper, and the numbers are exchanged at the end
  float la = min_nan(min_nan(y[0], y[1]), min_nan(y[2], y[3])), ha = max_nan(max_nan(y[0], y[1]), max_nan(y[2], y[3]));
  float lb = min_nan(min_nan(y[4], y[5]), min_nan(y[6], y[7])), hb = max_nan(max_nan(y[4], y[5]), max_nan(y[6], y[7]));
  const bool odd = l & 1;
  float lo = min_nan(odd ? lb : la, __shfl_xor_sync(0xffffffffu, odd ? la : lb, 1));
  float hi = max_nan(odd ? hb : ha, __shfl_xor_sync(0xffffffffu, odd ? ha : hb, 1));
#pragma unroll
  for (int off = 2; off < 8; off <<= 1) {
    lo = min_nan(lo, __shfl_xor_sync(0xffffffffu, lo, off));
    hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, off));
  }
  __half s, o;
  q4_params(lo, hi, s, o);
  const uint32_t mine = (uint32_t)__half_as_ushort(o) | (uint32_t)__half_as_ushort(s) << 16;
  const uint32_t other = __shfl_xor_sync(0xffffffffu, mine, 1);
  const uint32_t ma = odd ? other : mine, mb = odd ? mine : other;
  auto half = [](uint32_t v) { return __half2float(__ushort_as_half((uint16_t)v)); };
  // a word's eight codes lie in two lanes
  uint32_t wa = q4_codes<4>(y, half(ma >> 16), half(ma)) << (16 * (l & 1));
  uint32_t wb = q4_codes<4>(y + 4, half(mb >> 16), half(mb)) << (16 * (l & 1));
  wa |= __shfl_xor_sync(0xffffffffu, wa, 1);
  wb |= __shfl_xor_sync(0xffffffffu, wb, 1);
  if (head0 >= pool.n_kv) return;
  uint8_t* ch = static_cast<uint8_t*>(pool.k) + q4_chunk_off(pool, ap.layer, page, head);
  *reinterpret_cast<uint32_t*>(ch + q4_k_word(tok, (odd ? 8 : 0) + (l >> 1))) = odd ? wb : wa;
  if ((l & 7) < 2) {
    const int grp = (odd ? 2 : 0) + (l >> 3);
    uint16_t* meta = reinterpret_cast<uint16_t*>(ch + kQ4Meta + tok * 16);
    meta[grp] = (uint16_t)mine;
    meta[4 + grp] = (uint16_t)(mine >> 16);
  }
}

// A warp's task is four heads of one token (q, and k and v of f32 and bf16
// caches), eight lanes per head: lane c holds elements 8c.. and 64 + 8c.., which
// close under either rotation.  Lanes of heads past the last repeat it and store
// nothing; every lane stays with its warp through the shuffles.  A 4-bit cache's
// K goes two heads at a time (append_k_q4) and its V as four heads of a pair of
// adjacent slots, whose codes lie pairwise: with both slots new the pair is
// written as 8-byte pieces.  Tasks run v, k, q: the longest first.
// (A token per warp, with its cos / sin and weights kept over the heads, took 122
// registers and 20.0 to 25.1 us for 4096 tokens of 28q/4kv in bf16, against 17.8.)
template <bool IN_BF16, bool Q_BF16, int KV>
__global__ void __launch_bounds__(kQkNormWarps * 32, kQkNormCtasPerSm)
    qk_norm_append_kernel(const AppendArgs ap, const NormArgs na, const KVPool pool,
                          const __grid_constant__ SeqBatch sb, int T) {
  // a programmatic dependent of the projection before it, as rope_append_kernel
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int hq = ap.n_heads, hkv = pool.n_kv;
  const int qw = ap.q ? (hq + 3) / 4 : 0, kw = ap.k ? (hkv + 3) / 4 : 0;
  const int n_v = KV == kKvQ4 ? sb.n * (ap.n_new / 2 + 1) * kw : T * kw;
  const int kw2 = KV == kKvQ4 ? (hkv + 1) / 2 : kw;  // tasks of a token's k
  const int n_k = ap.k ? T * kw2 : 0;
  const int total = n_v + n_k + T * qw;  // < 2^31: checked on the host
  const int lane = threadIdx.x & 31, sub = lane >> 3, c = lane & 7;
  for (int w = (blockIdx.x * blockDim.x + threadIdx.x) >> 5; w < total; w += (gridDim.x * blockDim.x) >> 5) {
    if (KV == kKvQ4 && w < n_v) {
      // ---- V into a 4-bit cache: lane c holds dims 32 q + 4 c .. + 3 of both slots
      const int i = w, pu = i / kw;
      const int per_row = ap.n_new / 2 + 1;
      const int z = pu / per_row;
      const int head0 = (i - pu * kw) * 4 + sub, head = min(head0, hkv - 1);
      const int first = sb.len[z], last = first + ap.n_new;
      const int slot = (first / 2 + pu - z * per_row) * 2;  // the pair's even slot
      const bool in0 = slot >= first && slot < last, in1 = slot + 1 >= first && slot + 1 < last;
      if (!in0 && !in1) continue;
      float x[2][4][4];
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        const int t = z * ap.n_new + min(max(slot + p, first), last - 1) - first;
        const size_t base = ((size_t)t * hkv + head) * kHeadDim + 4 * c;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          if (IN_BF16) {
            const uint2 v = *reinterpret_cast<const uint2*>(reinterpret_cast<const uint16_t*>(ap.v) + base + 32 * q);
            x[p][q][0] = bf16_lo_f32(v.x); x[p][q][1] = bf16_hi_f32(v.x);
            x[p][q][2] = bf16_lo_f32(v.y); x[p][q][3] = bf16_hi_f32(v.y);
          } else {
            const float4 v = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(ap.v) + base + 32 * q);
            x[p][q][0] = v.x; x[p][q][1] = v.y; x[p][q][2] = v.z; x[p][q][3] = v.w;
          }
          if (ap.bv) {
            const float4 b = *reinterpret_cast<const float4*>(ap.bv + head * kHeadDim + 32 * q + 4 * c);
            x[p][q][0] = __fadd_rn(x[p][q][0], b.x); x[p][q][1] = __fadd_rn(x[p][q][1], b.y);
            x[p][q][2] = __fadd_rn(x[p][q][2], b.z); x[p][q][3] = __fadd_rn(x[p][q][3], b.w);
          }
        }
      }
      // least and greatest value of the eight (slot, group) sets over the eight lanes: at each step a lane hands on the
      // half of the sets that it does not keep, so that lane c ends with set c = 4 p + q, whose numbers all then get
      float lo[8], hi[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float* y = x[k >> 2][k & 3];
        lo[k] = min_nan(min_nan(y[0], y[1]), min_nan(y[2], y[3]));
        hi[k] = max_nan(max_nan(y[0], y[1]), max_nan(y[2], y[3]));
      }
#pragma unroll
      for (int off = 4; off > 0; off >>= 1) {
        const bool up = c & off;
#pragma unroll
        for (int k = 0; k < off; ++k) {
          lo[k] = min_nan(up ? lo[k + off] : lo[k], __shfl_xor_sync(0xffffffffu, up ? lo[k] : lo[k + off], off));
          hi[k] = max_nan(up ? hi[k + off] : hi[k], __shfl_xor_sync(0xffffffffu, up ? hi[k] : hi[k + off], off));
        }
      }
      __half s_own, o_own;
      q4_params(lo[0], hi[0], s_own, o_own);
      const uint32_t own = (uint32_t)__half_as_ushort(o_own) | (uint32_t)__half_as_ushort(s_own) << 16;
      uint32_t codes[4], sw[4], ow[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const uint32_t m0 = __shfl_sync(0xffffffffu, own, (lane & 24) + q), m1 = __shfl_sync(0xffffffffu, own, (lane & 24) + 4 + q);
        ow[q] = (m0 & 0xffffu) | m1 << 16;
        sw[q] = m0 >> 16 | (m1 & 0xffff0000u);
        codes[q] = q4_codes<4>(x[0][q], __half2float(__ushort_as_half((uint16_t)sw[q])), __half2float(__ushort_as_half((uint16_t)ow[q]))) |
                   q4_codes<4>(x[1][q], __half2float(__ushort_as_half((uint16_t)(sw[q] >> 16))), __half2float(__ushort_as_half((uint16_t)(ow[q] >> 16)))) << 16;
      }
      const int lp = slot / kPageSize, tok = slot % kPageSize;
      int page = -1;
      if ((unsigned)lp < (unsigned)pool.max_pages_per_seq)
        page = pool.block_table[(size_t)sb.seq[z] * pool.max_pages_per_seq + lp];
      if ((unsigned)page >= (unsigned)(pool.n_pool_pages - 1)) {  // the null page is never written
        report_error(ap.status, kDevErrBounds);
        continue;
      }
      if (head0 >= hkv) continue;
      uint8_t* ch = static_cast<uint8_t*>(pool.v) + q4_chunk_off(pool, ap.layer, page, head);
      uint8_t* cp = ch + q4_v_pair(tok, c, 0);
      uint8_t* mp = ch + kQ4Meta + q4_v_meta(tok);
      if (in0 && in1) {
        *reinterpret_cast<uint2*>(cp) = make_uint2(codes[0], codes[1]);
        *reinterpret_cast<uint2*>(cp + 512) = make_uint2(codes[2], codes[3]);
        if (c == 0) *reinterpret_cast<uint4*>(mp) = make_uint4(sw[0], sw[1], sw[2], sw[3]);
        if (c == 1) *reinterpret_cast<uint4*>(mp + kQ4VOffsets - kQ4Meta) = make_uint4(ow[0], ow[1], ow[2], ow[3]);
      } else {
        // one slot of the pair: the other's 16-bit pieces stay as they are
        const int p = in0 ? 0 : 1;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          *reinterpret_cast<uint16_t*>(cp + (q >> 1) * 512 + (q & 1) * 4 + 2 * p) = (uint16_t)(codes[q] >> (16 * p));
          if (c == 0) *reinterpret_cast<uint16_t*>(mp + 4 * q + 2 * p) = (uint16_t)(sw[q] >> (16 * p));
          if (c == 1)
            *reinterpret_cast<uint16_t*>(mp + kQ4VOffsets - kQ4Meta + 4 * q + 2 * p) = (uint16_t)(ow[q] >> (16 * p));
        }
      }
      continue;
    }
    const int sec = w < n_v ? 2 : (w < n_v + n_k ? 1 : 0);
    const int i = sec == 2 ? w : (sec == 1 ? w - n_v : w - n_v - n_k);
    const int heads = sec == 0 ? hq : hkv;
    const int per = sec == 0 ? qw : (sec == 1 ? kw2 : kw);  // tasks of a token
    const int t = i / per;
    const int row = t / ap.n_new, s = t - row * ap.n_new;
    const int pos = sb.pos[row] + s;
    const bool rope = sec == 0 || (sec == 1 && ap.rope_k);
    if (rope && (unsigned)pos >= (unsigned)ap.max_pos) {
      report_error(ap.status, kDevErrBounds);
      continue;
    }
    int page = -1, tok = 0;
    if (sec > 0) {
      const int slot = sb.len[row] + s, lp = slot / kPageSize;
      tok = slot % kPageSize;
      if ((unsigned)lp < (unsigned)pool.max_pages_per_seq)
        page = pool.block_table[(size_t)sb.seq[row] * pool.max_pages_per_seq + lp];
      if ((unsigned)page >= (unsigned)(pool.n_pool_pages - 1)) {  // the null page is never written
        report_error(ap.status, kDevErrBounds);
        continue;
      }
    }
    if (KV == kKvQ4 && sec == 1) {
      append_k_q4<IN_BF16>(ap, na, pool, t, (i - t * per) * 2 + (lane >> 4), pos, page, tok, lane);
      continue;
    }
    const int head0 = (i - t * per) * 4 + sub, head = min(head0, heads - 1);
    const int e0 = 8 * c, e1 = 64 + 8 * c;
    const void* src = sec == 0 ? ap.q : (sec == 1 ? ap.k : ap.v);
    const size_t base = ((size_t)t * heads + head) * kHeadDim;
    float a[8], b[8];
    load8<IN_BF16>(src, base + e0, a);
    load8<IN_BF16>(src, base + e1, b);
    const float* bias = sec == 0 ? ap.bq : (sec == 1 ? ap.bk : ap.bv);
    if (bias) {
      add_bias8(a, bias + head * kHeadDim + e0);
      add_bias8(b, bias + head * kHeadDim + e1);
    }
    const float* nw = sec == 0 ? na.qw : (sec == 1 ? na.kw : nullptr);
    if (nw) head_norm(a, b, nw, e0, e1, na.eps);
    if (rope) {
      const bool split = ap.variant == 0;
      // split-half: pairs (a[k], b[k]) are 8c + k; interleaved: (a[2k], a[2k + 1]) are 4c + k, of b 32 + 4c + k
      const size_t p0 = (size_t)pos * 64 + (split ? 8 * c : 4 * c), p1 = p0 + (split ? 4 : 32);
      const float4 c0 = *reinterpret_cast<const float4*>(ap.cos_t + p0), c1 = *reinterpret_cast<const float4*>(ap.cos_t + p1);
      const float4 s0 = *reinterpret_cast<const float4*>(ap.sin_t + p0), s1 = *reinterpret_cast<const float4*>(ap.sin_t + p1);
      const float cs[8] = {c0.x, c0.y, c0.z, c0.w, c1.x, c1.y, c1.z, c1.w};
      const float sn[8] = {s0.x, s0.y, s0.z, s0.w, s1.x, s1.y, s1.z, s1.w};
      if (split) {
#pragma unroll
        for (int k = 0; k < 8; ++k) rope_pair(a[k], b[k], cs[k], sn[k], a[k], b[k]);
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          rope_pair(a[2 * k], a[2 * k + 1], cs[k], sn[k], a[2 * k], a[2 * k + 1]);
          rope_pair(b[2 * k], b[2 * k + 1], cs[k + 4], sn[k + 4], b[2 * k], b[2 * k + 1]);
        }
      }
    }
    if (head0 >= heads) continue;
    if (sec == 0) {
      store8<Q_BF16>(ap.q_out, base + e0, a);
      store8<Q_BF16>(ap.q_out, base + e1, b);
    } else {
      const size_t off = (((size_t)ap.layer * pool.n_pool_pages + page) * hkv + head) * (size_t)(kPageSize * kHeadDim) + tok * kHeadDim;
      void* dst = sec == 1 ? pool.k : pool.v;
      store8<KV == kKvBf16>(dst, off + e0, a);
      store8<KV == kKvBf16>(dst, off + e1, b);
    }
  }
}

}  // namespace oomattn
