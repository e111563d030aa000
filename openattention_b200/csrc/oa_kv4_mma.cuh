// One warp's attention over tiles of 32 cache records (oa_kv4.cuh), on mma.sync.m16n8k16 (fp16 in, fp32
// accumulated).  The warp attends for up to eight query columns (query heads, query tokens) that read the
// same records.
//
// Mathematics.  With K = s c + z per half h of the head, q . K = sum_h s_h (q_h . c_h) + z_h (sum q_h): the
// tensor cores multiply the bare codes, the scales and offsets enter after, in fp32, once per token and half.
// The value side folds the scale into the weight: o = sum_t (p_t s_t) c_t + sum_t p_t z_t, the second sum in
// fp32 outside the tensor cores.
//
// Codes cost one AND each pair: a nibble left in place in a 16-bit word is an fp16 subnormal, code * 2^-24 (low
// nibble) or 16 * code * 2^-24 (high nibble), exact.  Low and high nibbles are the two halves, so the factor 16
// belongs to a whole half.  q is scaled by a power of two per column (largest element in [2^13, 2^14)), exact
// unless an element is 2^-37 of the largest; p s by a power of two per half, raised so that the largest scale
// seen gives [2^14, 2^15): p s is rounded to fp16 (11 bits) over 28 octaves below the largest.
//
// Layout.  Scores are computed transposed, S^T = codes (16 tokens) x q (8 columns), so that columns lie along
// the accumulator's lanes the same way as in O^T = V^T (16 dims) x P (8 columns): running maxima and sums need
// no exchange, only P turns (movmatrix).  The contraction's order is free, so a lane's operand words are its
// 16 contiguous bytes of a K row and 8 bytes of a V row.  Rows of an MMA are assigned to tokens so that both
// loads touch every bank once although records lie 36 words apart.
#pragma once
#include <cuda_fp16.h>

#include "oa_kv4.cuh"

namespace oa {

constexpr int kTile = 32;                   // records per tile
constexpr int kTileBytes = kTile * kRec;
constexpr uint32_t kLoMask = 0x000f000fu, kHiMask = 0x00f000f0u;

__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}
__device__ __forceinline__ float ex2(float x) {  // 2^x, results under 2^-126 are 0
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float pow2i(int e) { return __int_as_float((e + 127) << 23); }  // -126 <= e <= 127
__device__ __forceinline__ float biased(float m) { return m == -INFINITY ? 0.f : m; }

// shared-space loads
__device__ __forceinline__ uint4 lds128(uint32_t at, int imm) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at + imm));
  return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t at, int imm) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(at + imm));
  return v;
}
__device__ __forceinline__ uint32_t shr8(uint32_t x) { return x >> 8; }

// Token (0..15 of a 16-token block) of MMA row r (0..7); row r + 8 holds the next token.
__device__ __forceinline__ int row_token(int r) { return (r & 1) ? 8 + ((r + 3) & 7) : r; }

struct WarpAttention {
  uint32_t qf[16];           // q operand: half h, word i -> qf[8 h + 2 i], +1
  float scale[2];            // per column (2t, 2t + 1): sm_scale log2(e) 2^(24 - exponent of q)
  float q0[2], q1[2];        // sm_scale log2(e) times the sum of q over each half
  float acc[8][4];           // O^T: half h, tile i -> acc[4 h + i]
  float m[2], bm[2], l[2];   // running maximum (log2 units; bm: 0 while it is -inf), this lane's share of the sum
  float z0[2], z1[2];        // this lane's share of sum p z, per half
  float r0, r1, cap0, cap1;  // power-of-two factors of p s per half, and the largest scale they hold

  // q_col: this lane's column's row (column = lane / 4), NULL for an unused column
  __device__ __forceinline__ void load_q(const __nv_bfloat16* q_col, float qk_scale) {
    const int t = threadIdx.x & 3;
    float lo[16], hi[16], amax = 0.f, s0 = 0.f, s1 = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      uint4 v = make_uint4(0u, 0u, 0u, 0u);
      if (q_col) v = *reinterpret_cast<const uint4*>(q_col + (w >= 2 ? 64 : 0) + 16 * t + 8 * (w & 1));
      float* f = (w >= 2 ? hi : lo) + 8 * (w & 1);
      f[0] = bf_lo(v.x); f[1] = bf_hi(v.x); f[2] = bf_lo(v.y); f[3] = bf_hi(v.y);
      f[4] = bf_lo(v.z); f[5] = bf_hi(v.z); f[6] = bf_lo(v.w); f[7] = bf_hi(v.w);
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      amax = fmaxf(amax, fmaxf(fabsf(lo[i]), fabsf(hi[i])));
      s0 += lo[i];
      s1 += hi[i];
    }
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
      s0 += __shfl_xor_sync(0xffffffffu, s0, o);
      s1 += __shfl_xor_sync(0xffffffffu, s1, o);
    }
    // clamped so that 2^(24 - e) stays finite: |q| up to 2^105 is held
    const int e = amax > 0.f ? min(120, max(-90, 13 - ((__float_as_int(amax) >> 23) - 127))) : 0;
    const float f0 = pow2i(e), f1 = pow2i(e - 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      qf[2 * i] = pack_half2(lo[4 * i] * f0, lo[4 * i + 2] * f0);
      qf[2 * i + 1] = pack_half2(lo[4 * i + 1] * f0, lo[4 * i + 3] * f0);
      qf[8 + 2 * i] = pack_half2(hi[4 * i] * f1, hi[4 * i + 2] * f1);
      qf[8 + 2 * i + 1] = pack_half2(hi[4 * i + 1] * f1, hi[4 * i + 3] * f1);
    }
    const float sc = qk_scale * pow2i(24 - e);
#pragma unroll
    for (int j = 0; j < 2; ++j) {  // column 2t + j lives in the lanes 4 (2t + j) ..
      const int src = 8 * t + 4 * j;
      scale[j] = __shfl_sync(0xffffffffu, sc, src);
      q0[j] = __shfl_sync(0xffffffffu, s0, src) * qk_scale;
      q1[j] = __shfl_sync(0xffffffffu, s1, src) * qk_scale;
    }
  }

  __device__ __forceinline__ void reset() {
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[i][j] = 0.f;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      m[j] = -INFINITY;
      bm[j] = l[j] = z0[j] = z1[j] = 0.f;
    }
    r0 = r1 = pow2i(126);
    cap0 = cap1 = pow2i(15 - 126);
  }

  // A scale above the cap: choose the factor anew for the largest scale of this tile.
  __device__ __forceinline__ void raise_cap(float s, float& r, float& cap, int half) {
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) s = fmaxf(s, __shfl_xor_sync(0xffffffffu, s, o));
    if (!(s > cap)) return;
    const int es = max(-112, (__float_as_int(s) >> 23) - 127);
    const float next = pow2i(14 - es);
    // next / r as a power of two; one under 2^-126 drops what is there, which is that much smaller
    const int d = (__float_as_int(next) >> 23) - (__float_as_int(r) >> 23);
    const float f = d < -126 ? 0.f : pow2i(d);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[4 * half + i][j] *= f;
    r = next;
    cap = pow2i(15) / next;
  }

  // This lane's addresses in a tile (shared-space bytes from the tile's start).
  uint32_t at_k, at_m, at_v0, at_v1;
  __device__ __forceinline__ void lane_addresses() {
    const uint32_t lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const uint32_t tok = row_token(g);
    at_k = tok * kRec + 16 * t;                                // K codes of MMA row g; row g + 8 is the next record
    at_m = tok * kRec + kRecMeta;
    at_v0 = 2 * t * kRec + kRecV + 8 * g;                      // V dims 8g .. 8g + 7 (and + 64) of MMA row 2t
    at_v1 = (8 + ((2 * t + 4) & 7)) * kRec + kRecV + 8 * g;    // and of row 2t + 1
  }

  // One tile of 32 records at shared address `sm`.  MASK: column 2t + j sees only the tokens below lim[j] of the
  // tile; what masked records hold (stale bytes, NaN scales) does not enter.
  template <bool MASK>
  __device__ __forceinline__ void tile(uint32_t sm, const int (&lim)[2]) {
    const int tok = MASK ? row_token((threadIdx.x & 31) >> 2) : 0;
    float x[2][4];
    uint2 vm[2][2];  // value scales and offsets of this lane's four tokens
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      const uint4 ka = lds128(sm + at_k, 16 * b * kRec), kb = lds128(sm + at_k, (16 * b + 1) * kRec);
      const uint4 ma = lds128(sm + at_m, 16 * b * kRec), mb = lds128(sm + at_m, (16 * b + 1) * kRec);
      float c0[4] = {0.f, 0.f, 0.f, 0.f}, c1[4] = {0.f, 0.f, 0.f, 0.f};
      const uint32_t wa[4] = {ka.x, ka.y, ka.z, ka.w}, wb[4] = {kb.x, kb.y, kb.z, kb.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t a = wa[i], c = wb[i], a8 = shr8(a), c8 = shr8(c);
        mma_f16(c0, a & kLoMask, c & kLoMask, a8 & kLoMask, c8 & kLoMask, qf[2 * i], qf[2 * i + 1]);
        mma_f16(c1, a & kHiMask, c & kHiMask, a8 & kHiMask, c8 & kHiMask, qf[8 + 2 * i], qf[8 + 2 * i + 1]);
      }
      vm[b][0] = make_uint2(ma.z, ma.w);
      vm[b][1] = make_uint2(mb.z, mb.w);
      const float sa0 = bf_lo(ma.x), za0 = bf_hi(ma.x), sa1 = bf_lo(ma.y), za1 = bf_hi(ma.y);
      const float sb0 = bf_lo(mb.x), zb0 = bf_hi(mb.x), sb1 = bf_lo(mb.y), zb1 = bf_hi(mb.y);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        x[b][j] = fmaf(fmaf(sa1, c1[j], sa0 * c0[j]), scale[j], fmaf(za1, q1[j], za0 * q0[j]));
        x[b][2 + j] = fmaf(fmaf(sb1, c1[2 + j], sb0 * c0[2 + j]), scale[j], fmaf(zb1, q1[j], zb0 * q0[j]));
        if (MASK) {
          if (16 * b + tok >= lim[j]) x[b][j] = -INFINITY;
          if (16 * b + tok + 1 >= lim[j]) x[b][2 + j] = -INFINITY;
        }
      }
    }
    // m is the same in all lanes of a column, so nothing moves until some lane sees a larger score (or scale)
    float mx[2], s0 = 0.f, s1 = 0.f;
#pragma unroll
    for (int j = 0; j < 2; ++j) mx[j] = fmaxf(fmaxf(x[0][j], x[0][2 + j]), fmaxf(x[1][j], x[1][2 + j]));
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const bool in = !MASK || 16 * b + tok + k < max(lim[0], lim[1]);
        s0 = fmaxf(s0, in ? bf_lo(vm[b][k].x) : 0.f);
        s1 = fmaxf(s1, in ? bf_lo(vm[b][k].y) : 0.f);
      }
    if (__any_sync(0xffffffffu, mx[0] > m[0] || mx[1] > m[1] || s0 > cap0 || s1 > cap1)) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) mx[j] = fmaxf(mx[j], __shfl_xor_sync(0xffffffffu, mx[j], o));
        const float nm = fmaxf(m[j], mx[j]);
        const float al = ex2(m[j] - biased(nm));
        m[j] = nm;
        bm[j] = biased(nm);
        l[j] *= al;
        z0[j] *= al;
        z1[j] *= al;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          acc[i][j] *= al;
          acc[i][2 + j] *= al;
        }
      }
      raise_cap(s0, r0, cap0, 0);
      raise_cap(s1, r1, cap1, 1);
    }
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      uint32_t pl[2], ph[2];  // weights of the two halves, turned: tokens of rows 0..7, of rows 8..15
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const float p0 = ex2(x[b][2 * k] - bm[0]), p1 = ex2(x[b][2 * k + 1] - bm[1]);
        l[0] += p0;
        l[1] += p1;
        const float sa = bf_lo(vm[b][k].x) * r0, za = bf_hi(vm[b][k].x);
        const float sb = bf_lo(vm[b][k].y) * r1, zb = bf_hi(vm[b][k].y);
        float wa0 = p0 * sa, wa1 = p1 * sa, wb0 = p0 * sb, wb1 = p1 * sb;
        if (MASK) {
          const int tk = 16 * b + tok + k;
          const bool in0 = tk < lim[0], in1 = tk < lim[1];
          wa0 = in0 ? wa0 : 0.f;
          wb0 = in0 ? wb0 : 0.f;
          wa1 = in1 ? wa1 : 0.f;
          wb1 = in1 ? wb1 : 0.f;
          z0[0] += in0 ? p0 * za : 0.f;
          z1[0] += in0 ? p0 * zb : 0.f;
          z0[1] += in1 ? p1 * za : 0.f;
          z1[1] += in1 ? p1 * zb : 0.f;
        } else {
          z0[0] = fmaf(p0, za, z0[0]);
          z1[0] = fmaf(p0, zb, z1[0]);
          z0[1] = fmaf(p1, za, z0[1]);
          z1[1] = fmaf(p1, zb, z1[1]);
        }
        pl[k] = transpose8x8(pack_half2(wa0, wa1));
        ph[k] = transpose8x8(pack_half2(wb0, wb1));
      }
      const uint2 a0 = lds64(sm + at_v0, 16 * b * kRec), a1 = lds64(sm + at_v1, 16 * b * kRec);
      const uint2 n0 = lds64(sm + at_v0, (16 * b + 1) * kRec), n1 = lds64(sm + at_v1, (16 * b + 1) * kRec);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t sel = (i & 1) ? 0x7632u : 0x5410u;
        const uint32_t u = __byte_perm(i < 2 ? a0.x : a0.y, i < 2 ? a1.x : a1.y, sel);
        const uint32_t w = __byte_perm(i < 2 ? n0.x : n0.y, i < 2 ? n1.x : n1.y, sel);
        const uint32_t u8 = shr8(u), w8 = shr8(w);
        mma_f16(acc[i], u & kLoMask, u8 & kLoMask, w & kLoMask, w8 & kLoMask, pl[0], pl[1]);
        mma_f16(acc[4 + i], u & kHiMask, u8 & kHiMask, w & kHiMask, w8 & kHiMask, ph[0], ph[1]);
      }
    }
  }

  // The warp's unnormalised result of each column c < ncol: part[c * kD + d], ml[2 c] = m, ml[2 c + 1] = l.
  __device__ __forceinline__ void finish(float* part, float* ml, int ncol) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const float u0 = 1.f / r0, u1 = 1.f / r1;  // powers of two: exact
#pragma unroll
    for (int j = 0; j < 2; ++j) {
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) {
        l[j] += __shfl_xor_sync(0xffffffffu, l[j], o);
        z0[j] += __shfl_xor_sync(0xffffffffu, z0[j], o);
        z1[j] += __shfl_xor_sync(0xffffffffu, z1[j], o);
      }
      const int c = 2 * t + j;
      if (c >= ncol) continue;
      float* dst = part + c * kD + 8 * g;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        dst[2 * i] = fmaf(acc[i][j] * pow2i(24), u0, z0[j]);
        dst[2 * i + 1] = fmaf(acc[i][2 + j] * pow2i(24), u0, z0[j]);
        dst[64 + 2 * i] = fmaf(acc[4 + i][j] * pow2i(20), u1, z1[j]);
        dst[64 + 2 * i + 1] = fmaf(acc[4 + i][2 + j] * pow2i(20), u1, z1[j]);
      }
      if (g == 0) {
        ml[2 * c] = m[j];
        ml[2 * c + 1] = l[j];
      }
    }
  }
};

}  // namespace oa
