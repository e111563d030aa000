// One warp's attention over tiles of 32 cache records (oa_kv4.cuh), on mma.sync.m16n8k16 (fp16 in, fp32
// accumulated).  The warp attends for up to eight query columns (query heads, query tokens) that read the
// same records.
//
// Mathematics.  With K = s c + z per half h of the head, q . K = sum_h s_h (q_h . c_h) + z_h (sum q_h): the
// tensor cores multiply the bare codes, the scales and offsets enter after, in fp32, once per token and half.
// The value side folds the scale into the weight: o = sum_t (p_t s_t) c_t + sum_t p_t z_t, the second sum in
// fp32 outside the tensor cores.
//
// Tensor cores truncate their running sums.  Codes are all positive, so sums of p s c would grow with the context
// and with them the truncation, while the offsets' part cancels most of them (1.1e-2 of the result was seen at
// 131072 tokens in one CTA).  So half of the tokens enter complemented, s c + z = -s (15 - c) + (z + 15 s), at no
// cost (the complement is part of the AND): the sums stay of the result's size.
//
// Codes cost one AND each pair: a nibble left in place in a 16-bit word is an fp16 subnormal, code * 2^-24 (low
// nibble) or 16 * code * 2^-24 (high nibble), exact.  Low and high nibbles are the two halves, so the factor 16
// belongs to a whole half.  q is scaled by a power of two per column (largest element in [2^13, 2^14)), exact
// unless an element is 2^-37 of the largest; p s by a power of two per half, chosen so that the largest scale
// seen gives [2^6, 2^7): p s is rounded to fp16 (11 bits) over 20 octaves below the largest, beneath them it is
// off by 2^-32 of the largest.
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
constexpr float kSlack = 8.f;  // log2
constexpr int kTop = 7;        // scales times r stay at most 2^kTop, weights at most 2^(kTop + kSlack) < fp16's 65504
constexpr uint32_t kLoMask = 0x000f000fu, kHiMask = 0x00f000f0u;

__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_bf16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_bf16_k8(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t b0) {
  asm volatile(
      "mma.sync.aligned.m16n8k8.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5}, {%6}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(b0));
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
__device__ __forceinline__ uint32_t lds32(uint32_t at, int imm) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(at + imm));
  return v;
}

// Token (0..15 of a 16-token block) of MMA row r (0..7); row r + 8 holds the next token.
__device__ __forceinline__ int row_token(int r) { return (r & 1) ? 8 + ((r + 3) & 7) : r; }

// PAIR: at most four columns, and the MMA's eight columns hold each twice: columns 0..3 are the four query rows
// against half 0 of the head, columns 4..7 against half 1.  A lane then serves one half: half the scales to read,
// weights to form and turn; the halves' scores meet through one shuffle.  Otherwise eight columns, each lane
// both halves.  J: accumulator columns of a lane that are in use (1 where there is one query row).
template <bool PAIR, int J = 2>
struct WarpAttention {
  static constexpr int kHalves = PAIR ? 1 : 2;  // halves a lane serves
  uint32_t qf[16];            // q operand: half h, word i -> qf[8 h + 2 i], +1
  float scale[2];             // per column: sm_scale log2(e) 2^(24 - exponent of q)
  float qs[2][kHalves];       // sm_scale log2(e) times the sum of q over the half
  float acc[8][4];            // O^T: half h, tile i -> acc[4 h + i]; PAIR: valid where h is the lane's half
  float m[2], bm[2], l[2];    // running maximum (log2 units; bm: 0 while it is -inf), this lane's share of the sum
  float zs[2][kHalves];       // this lane's share of sum p z
  float r[kHalves], cap[kHalves];  // power-of-two factor of p s, and the largest scale it holds
  uint32_t at_k, at_m, at_v0, at_v1;  // this lane's addresses in a tile

  static __device__ __forceinline__ int lane() { return threadIdx.x & 31; }
  // the query columns of this lane's accumulator columns 0, 1, and of its operand column
  static __device__ __forceinline__ int acc_col(int j) { return 2 * (lane() & (PAIR ? 1 : 3)) + j; }
  static __device__ __forceinline__ int op_col() { return (lane() >> 2) & (PAIR ? 3 : 7); }
  static __device__ __forceinline__ int half() { return PAIR ? (lane() >> 1) & 1 : 0; }

  __device__ __forceinline__ void lane_addresses() {
    const uint32_t g = lane() >> 2, t = lane() & 3;
    const uint32_t tok = row_token(g);
    at_k = tok * kRec + 16 * t;                              // K codes of MMA row g; row g + 8 is the next record
    at_m = tok * kRec + kRecMeta + 4 * half();
    at_v0 = 2 * t * kRec + kRecV + 8 * g;                    // V dims 8g .. 8g + 7 (and + 64) of MMA row 2t
    at_v1 = (8 + ((2 * t + 4) & 7)) * kRec + kRecV + 8 * g;  // and of row 2t + 1
  }

  // q_col: the row of column op_col(), NULL for an unused column
  uint4 q_raw[4];
  __device__ __forceinline__ void load_q(const __nv_bfloat16* q_col) {
    const int t = lane() & 3;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      q_raw[w] = make_uint4(0u, 0u, 0u, 0u);
      if (q_col) q_raw[w] = *reinterpret_cast<const uint4*>(q_col + (w >= 2 ? 64 : 0) + 16 * t + 8 * (w & 1));
    }
  }
  __device__ __forceinline__ void begin(float qk_scale) {
    const int t = lane() & 3;
    float lo[16], hi[16], amax = 0.f, s0 = 0.f, s1 = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const uint4 v = q_raw[w];
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
    float f0 = pow2i(e), f1 = pow2i(e - 4);
    if (PAIR) (lane() < 16 ? f1 : f0) = 0.f;  // columns 0..3 take half 0 only, 4..7 half 1
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      qf[2 * i] = pack_half2(lo[4 * i] * f0, lo[4 * i + 2] * f0);
      qf[2 * i + 1] = pack_half2(lo[4 * i + 1] * f0, lo[4 * i + 3] * f0);
      qf[8 + 2 * i] = pack_half2(hi[4 * i] * f1, hi[4 * i + 2] * f1);
      qf[8 + 2 * i + 1] = pack_half2(hi[4 * i + 1] * f1, hi[4 * i + 3] * f1);
    }
    const float sc = qk_scale * pow2i(24 - e);
#pragma unroll
    for (int j = 0; j < 2; ++j) {  // accumulator column 2t + j is the operand column of the lanes 4 (2t + j) ..
      const int src = 8 * t + 4 * j;
      scale[j] = __shfl_sync(0xffffffffu, sc, src);
      const float a = __shfl_sync(0xffffffffu, s0, src) * qk_scale, b = __shfl_sync(0xffffffffu, s1, src) * qk_scale;
      if (PAIR) {
        qs[j][0] = half() ? b : a;
      } else {
        qs[j][0] = a;
        qs[j][kHalves - 1] = b;
      }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[i][j] = 0.f;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      m[j] = -INFINITY;
      bm[j] = l[j] = 0.f;
#pragma unroll
      for (int h = 0; h < kHalves; ++h) zs[j][h] = 0.f;
    }
#pragma unroll
    for (int h = 0; h < kHalves; ++h) {
      r[h] = pow2i(126);
      cap[h] = pow2i(kTop - 126);
    }
  }

  // A scale above the cap: choose the factor anew for the largest scale of this tile.
  __device__ __forceinline__ void raise_cap(float s, int h) {
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) s = fmaxf(s, __shfl_xor_sync(0xffffffffu, s, o));
    if (!(s > cap[h])) return;
    const int es = max(kTop - 127, (__float_as_int(s) >> 23) - 127);
    const float next = pow2i(kTop - 1 - es);
    // next / r as a power of two; one under 2^-126 drops what is there, which is that much smaller
    const int d = (__float_as_int(next) >> 23) - (__float_as_int(r[h]) >> 23);
    const float f = d < -126 ? 0.f : pow2i(d);
#pragma unroll
    for (int i = 0; i < (PAIR ? 8 : 4); ++i)  // PAIR: the other half's tiles are not read in this lane
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[4 * h + i][j] *= f;
    r[h] = next;
    cap[h] = pow2i(kTop) / next;
  }

  // One tile of 32 records at shared address `sm`.  MASK: the lane's accumulator column j sees only the tokens whose
  // bit is set in sees[j]; what the others' records hold (stale bytes, NaN scales) does not enter.
  template <bool MASK>
  __device__ __forceinline__ void tile(uint32_t sm, const uint32_t (&sees)[2]) {
    uint32_t in[2];  // bit 16 b + k: this lane's token k of block b
#pragma unroll
    for (int j = 0; j < 2; ++j) in[j] = MASK ? sees[j] >> row_token(lane() >> 2) : 0u;
    float x[2][4];
    uint32_t vm[2][2][kHalves];  // value scale and offset of this lane's four tokens
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      const uint4 ka = lds128(sm + at_k, 16 * b * kRec), kb = lds128(sm + at_k, (16 * b + 1) * kRec);
      uint32_t km[2][kHalves];
      if (PAIR) {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          km[k][0] = lds32(sm + at_m, (16 * b + k) * kRec);
          vm[b][k][0] = lds32(sm + at_m, (16 * b + k) * kRec + 8);
        }
      } else {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const uint4 w = lds128(sm + at_m, (16 * b + k) * kRec);
          km[k][0] = w.x;
          km[k][kHalves - 1] = w.y;
          vm[b][k][0] = w.z;
          vm[b][k][kHalves - 1] = w.w;
        }
      }
      float c[kHalves][4];
#pragma unroll
      for (int h = 0; h < kHalves; ++h)
#pragma unroll
        for (int i = 0; i < 4; ++i) c[h][i] = 0.f;
      const uint32_t wa[4] = {ka.x, ka.y, ka.z, ka.w}, wb[4] = {kb.x, kb.y, kb.z, kb.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t a = wa[i], d = wb[i], a8 = a >> 8, d8 = d >> 8;
        mma_f16(c[0], a & kLoMask, d & kLoMask, a8 & kLoMask, d8 & kLoMask, qf[2 * i], qf[2 * i + 1]);
        mma_f16(c[kHalves - 1], a & kHiMask, d & kHiMask, a8 & kHiMask, d8 & kHiMask, qf[8 + 2 * i], qf[8 + 2 * i + 1]);
      }
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int j = 0; j < J; ++j) {
          float y = bf_lo(km[k][0]) * c[0][2 * k + j], z = bf_hi(km[k][0]) * qs[j][0];
          if (!PAIR) {
            y = fmaf(bf_lo(km[k][kHalves - 1]), c[kHalves - 1][2 * k + j], y);
            z = fmaf(bf_hi(km[k][kHalves - 1]), qs[j][kHalves - 1], z);
          }
          float v = fmaf(y, scale[j], z);
          if (PAIR) v += __shfl_xor_sync(0xffffffffu, v, 2);
          if (MASK && !(in[j] >> (16 * b + k) & 1u)) v = -INFINITY;
          x[b][2 * k + j] = v;
        }
    }
    // m is the same in all lanes of a column and nothing moves until some lane sees a score kSlack above it (or
    // a scale above the cap): weights up to 2^kSlack are as good as weights up to 1, and new maxima are common
    float mx[2], s[kHalves];
#pragma unroll
    for (int j = 0; j < J; ++j) mx[j] = fmaxf(fmaxf(x[0][j], x[0][2 + j]), fmaxf(x[1][j], x[1][2 + j]));
#pragma unroll
    for (int h = 0; h < kHalves; ++h) {
      s[h] = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const bool used = !MASK || ((in[0] | in[J - 1]) >> (16 * (i >> 1) + (i & 1)) & 1u);
        s[h] = fmaxf(s[h], used ? bf_lo(vm[i >> 1][i & 1][h]) : 0.f);
      }
    }
    if (__any_sync(0xffffffffu, mx[0] > m[0] + kSlack || mx[J - 1] > m[J - 1] + kSlack || s[0] > cap[0] || s[kHalves - 1] > cap[kHalves - 1])) {
#pragma unroll
      for (int j = 0; j < J; ++j) {
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) mx[j] = fmaxf(mx[j], __shfl_xor_sync(0xffffffffu, mx[j], o));
        const float nm = fmaxf(m[j], mx[j]);
        const float al = ex2(m[j] - biased(nm));
        m[j] = nm;
        bm[j] = biased(nm);
        l[j] *= al;
#pragma unroll
        for (int h = 0; h < kHalves; ++h) zs[j][h] *= al;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          acc[i][j] *= al;
          acc[i][2 + j] *= al;
        }
      }
#pragma unroll
      for (int h = 0; h < kHalves; ++h) raise_cap(s[h], h);
    }
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      uint32_t pw[2][kHalves];  // weights, turned: tokens of MMA rows 0..7, of rows 8..15
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const float p0 = ex2(x[b][2 * k] - bm[0]), p1 = J > 1 ? ex2(x[b][2 * k + 1] - bm[1]) : 0.f;
        l[0] += p0;
        if (J > 1) l[1] += p1;
#pragma unroll
        for (int h = 0; h < kHalves; ++h) {
          // second tokens enter as -s (15 - c) + (z + 15 s): the codes' sums then stay near zero (below)
          const float s1 = bf_lo(vm[b][k][h]), sv = s1 * (k ? -r[h] : r[h]);
          const float zv = k ? fmaf(15.f, s1, bf_hi(vm[b][k][h])) : bf_hi(vm[b][k][h]);
          float w0 = p0 * sv, w1 = J > 1 ? p1 * sv : 0.f;
          if (MASK) {
            const bool in0 = in[0] >> (16 * b + k) & 1u, in1 = J > 1 && (in[1] >> (16 * b + k) & 1u);
            w0 = in0 ? w0 : 0.f;
            w1 = in1 ? w1 : 0.f;
            zs[0][h] += in0 ? p0 * zv : 0.f;
            if (J > 1) zs[1][h] += in1 ? p1 * zv : 0.f;
          } else {
            zs[0][h] = fmaf(p0, zv, zs[0][h]);
            if (J > 1) zs[1][h] = fmaf(p1, zv, zs[1][h]);
          }
          pw[k][h] = transpose8x8(pack_half2(w0, w1));
        }
      }
      const uint2 a0 = lds64(sm + at_v0, 16 * b * kRec), a1 = lds64(sm + at_v1, 16 * b * kRec);
      const uint2 n0 = lds64(sm + at_v0, (16 * b + 1) * kRec), n1 = lds64(sm + at_v1, (16 * b + 1) * kRec);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t sel = (i & 1) ? 0x7632u : 0x5410u;
        const uint32_t u = __byte_perm(i < 2 ? a0.x : a0.y, i < 2 ? a1.x : a1.y, sel);
        const uint32_t w = __byte_perm(i < 2 ? n0.x : n0.y, i < 2 ? n1.x : n1.y, sel);
        const uint32_t u8 = u >> 8, w8 = w >> 8;
        mma_f16(acc[i], u & kLoMask, u8 & kLoMask, ~w & kLoMask, ~w8 & kLoMask, pw[0][0], pw[1][0]);
        mma_f16(acc[4 + i], u & kHiMask, u8 & kHiMask, ~w & kHiMask, ~w8 & kHiMask, pw[0][kHalves - 1], pw[1][kHalves - 1]);
      }
    }
  }

  // ---- bf16 rows among the records (PAIR, J = 1: one query row, in columns 0 and 4): tiles of 8 rows of K, then 8
  // of V, 256 bytes each, 16-byte chunk c of row i at chunk c ^ i.  Scores: MMA rows g and g + 8 are the two halves
  // of K row g, columns 0 and 1 the halves of q; the score is their diagonal's sum.  Values go into the records'
  // accumulators: weights carry the factors that those carry, as two bf16 terms (16 bits) in columns 0, 1 (half 0)
  // and 4, 5 (half 1).
  __device__ __forceinline__ void begin_rows(const __nv_bfloat16* q) {
    const int g = lane() >> 2, t = lane() & 3;
#pragma unroll
    for (int i = 0; i < 8; ++i) qf[i] = 0u;
    if (g < 2) {  // step i: dims 64 g + 16 i + 2t, + 1 and + 8, + 9
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        qf[2 * i] = *reinterpret_cast<const uint32_t*>(q + 64 * g + 16 * i + 2 * t);
        qf[2 * i + 1] = *reinterpret_cast<const uint32_t*>(q + 64 * g + 16 * i + 2 * t + 8);
      }
    }
    // scales of records may have left a factor that would carry a large row past fp32
    if (r[0] > pow2i(60)) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] *= pow2i(60) / r[0];
      cap[0] = pow2i(kTop - 60);
      r[0] = pow2i(60);
    }
  }
  // sm: the tile; in: its live rows (others are zero in memory); bias: this lane's row's (lane < 8) log2 weight
  __device__ __forceinline__ void rows(uint32_t sm, uint32_t in, float bias, float qk_scale) {
    const int g = lane() >> 2, t = lane() & 3;
    // ldmatrix: lane 8 x + i gives row i of matrix x: half x & 1 of K, 8 dims x >> 1 of the 16 of a step
    const uint32_t i8 = lane() & 7, x = lane() >> 3;
    float c[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t k[4];
      const uint32_t chunk = 8 * (x & 1) + 2 * i + (x >> 1);
      asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                   : "=r"(k[0]), "=r"(k[1]), "=r"(k[2]), "=r"(k[3])
                   : "r"(sm + i8 * 256 + ((chunk ^ i8) << 4)));
      mma_bf16(c, k[0], k[1], k[2], k[3], qf[2 * i], qf[2 * i + 1]);
    }
    float v = __shfl_sync(0xffffffffu, c[0] + c[3], lane() & 28);  // lane t = 0 of the row has it
    const float b = __shfl_sync(0xffffffffu, bias, g);
    v = (in >> g & 1u) && !(t & 1) ? fmaf(v, qk_scale, b) : -INFINITY;
    if (__any_sync(0xffffffffu, v > m[0] + kSlack)) {
      float mx = v;
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
      mx = fmaxf(m[0], mx);
      const float al = ex2(m[0] - biased(mx));
      m[0] = mx;
      bm[0] = biased(mx);
      l[0] *= al;
      zs[0][0] *= al;
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] *= al;
    }
    const float p = ex2(v - bm[0]);
    l[0] += p;
    const float w = p * (r[0] * pow2i(half() ? -20 : -24)), hi = bf_round(w);
    const uint32_t pw = transpose8x8((uint32_t)f2bf_bits(hi) | ((uint32_t)f2bf_bits(w - hi) << 16));
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t r0 = 2 * t, r1 = 2 * t + 1, ch = 8 * h + g;
      const uint4 a = lds128(sm + 2048 + r0 * 256 + ((ch ^ r0) << 4), 0), d = lds128(sm + 2048 + r1 * 256 + ((ch ^ r1) << 4), 0);
      mma_bf16_k8(acc[4 * h], __byte_perm(a.x, d.x, 0x5410), __byte_perm(a.x, d.x, 0x7632), pw);
      mma_bf16_k8(acc[4 * h + 1], __byte_perm(a.y, d.y, 0x5410), __byte_perm(a.y, d.y, 0x7632), pw);
      mma_bf16_k8(acc[4 * h + 2], __byte_perm(a.z, d.z, 0x5410), __byte_perm(a.z, d.z, 0x7632), pw);
      mma_bf16_k8(acc[4 * h + 3], __byte_perm(a.w, d.w, 0x5410), __byte_perm(a.w, d.w, 0x7632), pw);
    }
  }

  // The warp's unnormalised result of each column c < ncol: part[c * kD + d], ml[2 c] = m, ml[2 c + 1] = l.
  __device__ __forceinline__ void finish(float* part, float* ml, int ncol) {
    const int g = lane() >> 2;
#pragma unroll
    for (int j = 0; j < J; ++j) {
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) {
        l[j] += __shfl_xor_sync(0xffffffffu, l[j], o);
#pragma unroll
        for (int h = 0; h < kHalves; ++h) zs[j][h] += __shfl_xor_sync(0xffffffffu, zs[j][h], o);
      }
    }
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const int c = acc_col(j);
      if (c < ncol) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if (PAIR && h != half()) continue;
          const int k = PAIR ? 0 : h;
          // codes were 2^-24 (half 1: 2^-20) and weights r times too large; 1 / r is a power of two, exact
          const float f = 1.f / r[k], u = pow2i(h ? 20 : 24), z = zs[j][k];
          float o[8];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            // J = 1: the second column holds the rows' second weight term
            const float* c2 = acc[4 * h + i];
            o[2 * i] = fmaf((J == 1 ? c2[0] + c2[1] : c2[j]) * u, f, z);
            o[2 * i + 1] = fmaf((J == 1 ? c2[2] + c2[3] : c2[2 + j]) * u, f, z);
          }
          float4* dst = reinterpret_cast<float4*>(part + c * kD + 64 * h + 8 * g);
          dst[0] = make_float4(o[0], o[1], o[2], o[3]);
          dst[1] = make_float4(o[4], o[5], o[6], o[7]);
        }
        if (g == 0 && (!PAIR || half() == 0)) {
          ml[2 * c] = m[j];
          ml[2 * c + 1] = l[j];
        }
      }
    }
  }
};

}  // namespace oa
