// K-A with a norm of every q and k head and any cache type, in one pass over
// the projected rows:
//   y = x + b;  q, k: y = y / sqrt(mean(y^2) + eps) * w  (over the head's 128
//   values, f32), then the rotation of rope_append.cuh;  k, v: the paged append
//   (f32, bf16 or 4-bit).
// The norm is the one that models with normalised heads put between the
// projection's bias and RoPE; a kernel of its own would read and write q and k
// once more (for a 4096-token prompt of 28 + 4 heads in bf16, 67 MB more).
#pragma once
#include "common.cuh"
#include "kv4.cuh"
#include "params.cuh"
#include "rope_append.cuh"

namespace oomattn {

constexpr int kQkNormCtasPerSm = 4;  // CTAs of 8 warps

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

// Codes of 8 values, nibble n = value n.
__device__ __forceinline__ uint32_t q4_codes8(const float* x, float s, float o) {
  uint32_t w = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) w |= q4_code(x[i], s, o) << (4 * i);
  return w;
}

// A warp's task is four heads of one token (q, k, and v of f32 / bf16 caches)
// or four heads of one pair of adjacent slots (v of a 4-bit cache, whose codes
// lie pairwise: with both slots new the pair is written as 8-byte pieces).
// Eight lanes per head; every lane stays with its warp through the shuffles,
// lanes of heads past the last repeat it and store nothing.  Tasks run q, k, v.
template <bool IN_BF16, bool Q_BF16, int KV>
__global__ void __launch_bounds__(256)
    qk_norm_append_kernel(const AppendArgs ap, const NormArgs na, const KVPool pool,
                          const __grid_constant__ SeqBatch sb, int T) {
  // a programmatic dependent of the projection before it, as rope_append_kernel
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int hq = ap.n_heads, hkv = pool.n_kv;
  const int qw = ap.q ? (hq + 3) / 4 : 0, kw = ap.k ? (hkv + 3) / 4 : 0;
  const int v_units = KV == kKvQ4 ? sb.n * (ap.n_new / 2 + 1) : T;  // slots pairs, or tokens
  const int n_q = T * qw, n_k = T * kw;
  const int total = n_q + n_k + v_units * kw;  // < 2^31: checked on the host
  const int lane = threadIdx.x & 31, sub = lane >> 3, c = lane & 7;
  for (int w = (blockIdx.x * blockDim.x + threadIdx.x) >> 5; w < total; w += (gridDim.x * blockDim.x) >> 5) {
    if (KV == kKvQ4 && w >= n_q + n_k) {
      // ---- V into a 4-bit cache: lane c holds dims 32 q + 4 c .. + 3 of both slots
      const int i = w - n_q - n_k, pu = i / kw;
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
      uint32_t codes[4], sw[4], ow[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        codes[q] = sw[q] = ow[q] = 0;
#pragma unroll
        for (int p = 0; p < 2; ++p) {
          float lo = min_nan(min_nan(x[p][q][0], x[p][q][1]), min_nan(x[p][q][2], x[p][q][3]));
          float hi = max_nan(max_nan(x[p][q][0], x[p][q][1]), max_nan(x[p][q][2], x[p][q][3]));
#pragma unroll
          for (int off = 1; off < 8; off <<= 1) {
            lo = min_nan(lo, __shfl_xor_sync(0xffffffffu, lo, off));
            hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, off));
          }
          __half s, o;
          q4_params(lo, hi, s, o);
          const float sf = __half2float(s), of = __half2float(o);
#pragma unroll
          for (int e = 0; e < 4; ++e) codes[q] |= q4_code(x[p][q][e], sf, of) << (16 * p + 4 * e);
          sw[q] |= (uint32_t)__half_as_ushort(s) << (16 * p);
          ow[q] |= (uint32_t)__half_as_ushort(o) << (16 * p);
        }
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
    // ---- one token's q, k (or v) heads, 16 values per lane that close under the rotation
    const int sec = w < n_q ? 0 : (w < n_q + n_k ? 1 : 2);
    const int i = sec == 0 ? w : (sec == 1 ? w - n_q : w - n_q - n_k);
    const int per = sec == 0 ? qw : kw, heads = sec == 0 ? hq : hkv;
    const int t = i / per;
    const int head0 = (i - t * per) * 4 + sub, head = min(head0, heads - 1);
    const bool split = ap.variant == 0 && sec < 2;
    const int e0 = split ? 8 * c : 16 * c, e1 = split ? 64 + 8 * c : 16 * c + 8;
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
    const int row = t / ap.n_new, s = t - row * ap.n_new;
    if (sec == 0 || (sec == 1 && ap.rope_k)) {
      const int pos = sb.pos[row] + s;
      if ((unsigned)pos >= (unsigned)ap.max_pos) {
        report_error(ap.status, kDevErrBounds);
        continue;
      }
      float cs[8], sn[8];
      load8<false>(ap.cos_t, (size_t)pos * 64 + 8 * c, cs);
      load8<false>(ap.sin_t, (size_t)pos * 64 + 8 * c, sn);
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
    if (sec == 0) {
      if (head0 < heads) {
        store8<Q_BF16>(ap.q_out, base + e0, a);
        store8<Q_BF16>(ap.q_out, base + e1, b);
      }
      continue;
    }
    const int slot = sb.len[row] + s, lp = slot / kPageSize, tok = slot % kPageSize;
    int page = -1;
    if ((unsigned)lp < (unsigned)pool.max_pages_per_seq)
      page = pool.block_table[(size_t)sb.seq[row] * pool.max_pages_per_seq + lp];
    if ((unsigned)page >= (unsigned)(pool.n_pool_pages - 1)) {
      report_error(ap.status, kDevErrBounds);
      continue;
    }
    if (KV != kKvQ4) {
      if (head0 < heads) {
        const size_t off = (((size_t)ap.layer * pool.n_pool_pages + page) * hkv + head) * (size_t)(kPageSize * kHeadDim) + tok * kHeadDim;
        void* dst = sec == 1 ? pool.k : pool.v;
        store8<KV == kKvBf16>(dst, off + e0, a);
        store8<KV == kKvBf16>(dst, off + e1, b);
      }
      continue;
    }
    // ---- K into a 4-bit cache.  The groups of a and b: e0 / 32 and e1 / 32 --
    // split-half: two groups, each over four lanes; interleaved: one over two.
    float la = a[0], ha = a[0], lb = b[0], hb = b[0];
#pragma unroll
    for (int k = 1; k < 8; ++k) {
      la = min_nan(la, a[k]); ha = max_nan(ha, a[k]);
      lb = min_nan(lb, b[k]); hb = max_nan(hb, b[k]);
    }
    if (!split) {
      la = lb = min_nan(la, lb);
      ha = hb = max_nan(ha, hb);
    }
    la = min_nan(la, __shfl_xor_sync(0xffffffffu, la, 1));
    ha = max_nan(ha, __shfl_xor_sync(0xffffffffu, ha, 1));
    lb = min_nan(lb, __shfl_xor_sync(0xffffffffu, lb, 1));
    hb = max_nan(hb, __shfl_xor_sync(0xffffffffu, hb, 1));
    if (split) {
      la = min_nan(la, __shfl_xor_sync(0xffffffffu, la, 2));
      ha = max_nan(ha, __shfl_xor_sync(0xffffffffu, ha, 2));
      lb = min_nan(lb, __shfl_xor_sync(0xffffffffu, lb, 2));
      hb = max_nan(hb, __shfl_xor_sync(0xffffffffu, hb, 2));
    }
    __half sa, oa, s_b, ob;
    q4_params(la, ha, sa, oa);
    q4_params(lb, hb, s_b, ob);
    const uint32_t wa = q4_codes8(a, __half2float(sa), __half2float(oa));
    const uint32_t wb = q4_codes8(b, __half2float(s_b), __half2float(ob));
    if (head0 >= heads) continue;
    uint8_t* ch = static_cast<uint8_t*>(pool.k) + q4_chunk_off(pool, ap.layer, page, head);
    *reinterpret_cast<uint32_t*>(ch + q4_k_word(tok, e0 >> 3)) = wa;
    *reinterpret_cast<uint32_t*>(ch + q4_k_word(tok, e1 >> 3)) = wb;
    __half* meta = reinterpret_cast<__half*>(ch + kQ4Meta + tok * 16);
    if ((c & (split ? 3 : 1)) == 0) {
      meta[e0 >> 5] = oa;
      meta[4 + (e0 >> 5)] = sa;
      if (split) {
        meta[e1 >> 5] = ob;
        meta[4 + (e1 >> 5)] = s_b;
      }
    }
  }
}

}  // namespace oomattn
