// One warp's attention over tiles of 32 cache records (oa_kv4.cuh) on the warp-level tensor cores (mma.sync).  The warp
// attends for up to four or eight query columns (query heads, query tokens) that read the same records.  A decode
// step reads each record once for few columns, so memory bounds it; what the tensor cores are for here is that the
// codes need not be turned into numbers by the other pipes.  (tcgen05 takes its operands from shared or tensor memory
// in whole bytes at least: the unpacked codes would have to be written back there first.)
//
// Scores.  With K = s c + z per half h of the head, q . K = sum_h s_h (q_h . c_h) + z_h (sum q_h): the tensor cores
// multiply the bare codes, the scales and offsets enter after, in fp32, once per token and half.  Codes cost one AND
// each pair: a nibble left in place in a 16-bit word is an fp16 subnormal, code * 2^-24 (low nibble) or 16 code * 2^-24
// (high nibble), exact.  Low and high nibbles are the two halves, so the factor 16 belongs to a whole half.  q is
// scaled by a power of two per column (largest element in [2^13, 2^14), half 1 by 2^-4 more), which holds elements
// down to 2^-30 (half 0) and 2^-26 (half 1) of the largest in full; below, they are off by 2^-25, that is by 2^-38 and
// 2^-34 of the largest at most.  (e4m3 operands would hold a code in a byte, but mma.sync takes them apart into fp16
// here: slower.)
//
// Values.  The scale goes into the weight: o = sum_t (p_t s_t) c_t + sum_t p_t z_t, the second sum in fp32 outside the
// tensor cores.  p s is scaled by a power of two r per column and half and rounded to fp16: 11 bits over 20 octaves below
// the largest p s seen, beneath them off by 2^-31 of that.  r is chosen from weight times scale, not from the scale alone:
// a record of huge scale and no weight (or whose weight the running maximum took away later) must not push what the
// others give beneath fp16.  A column's running maximum is its first tile's, so that a row's only token weighs exactly 1,
// and from there moves by whole octaves (up to the next), so that weights, sums and r move by powers of two and what a
// larger maximum takes from the weights r can give back.
//
// Tensor cores truncate their running sums.  Codes are all positive, so sums of p s c would grow with the context
// and with them the truncation, while the offsets' part cancels most of them (1.1e-2 of the result was seen at
// 131072 tokens in one CTA).  So half of the tokens enter complemented, s c + z = -s (15 - c) + (z + 15 s), at no
// cost (the complement is part of the AND): the sums stay of the result's size.
//
// Layout.  Scores are computed transposed, S^T = codes (16 tokens) x q (columns), so that columns lie along the
// accumulator's lanes the same way as in O^T = V^T (16 dims) x P (columns): running maxima and sums need no exchange,
// only P turns (movmatrix).  The contraction's order is free, so a lane's operand words are its 16 contiguous bytes
// of a K row and 8 bytes of a V row.  Rows of an MMA are assigned to tokens so that both loads touch every bank once
// although records lie 36 words apart.  176 of a tile's instructions unpack codes.
#pragma once
#include <cuda_fp16.h>

#include "oa_kv4.cuh"

namespace oa {

constexpr int kTile = 32;                   // records per tile
constexpr int kTileBytes = kTile * kRec;
constexpr float kSlack = 5.f;        // log2
constexpr int kTop = 7;              // p s r stays under 2^kTop where r is chosen
constexpr float kCap = 32768.f;      // p s r above it (fp16 ends at 65504) has r chosen anew
constexpr uint32_t kWide = 0x4480u;  // 2^10 = kCap / 2^kSlack in bf16
// Where nothing was seen: under every score, and finite, so that its difference from itself is 0 and from -inf is -inf.
constexpr float kNoMax = -3.402823466e38f;
constexpr int kRowTop = 20;  // log2 of the largest r beside bf16 rows: their weights, r 2^-24 and r 2^-20 of p, stay at most p
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
__device__ __forceinline__ float lg2(float x) {  // log2, of a subnormal too
  float r;
  asm("lg2.approx.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ uint32_t max_bf16x2(uint32_t a, uint32_t b) {  // the number, of a number and a NaN
  uint32_t v;
  asm("max.bf16x2 %0, %1, %2;" : "=r"(v) : "r"(a), "r"(b));
  return v;
}
__device__ __forceinline__ uint32_t mul_bf16x2(uint32_t a, uint32_t b) {
  uint32_t v;
  asm("mul.bf16x2 %0, %1, %2;" : "=r"(v) : "r"(a), "r"(b));
  return v;
}
__device__ __forceinline__ float pow2i(int e) { return __int_as_float((e + 127) << 23); }  // -126 <= e <= 127

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

// Token (0..15 of a 16-token block) of MMA row r (0..7); row r + 8 holds the next token.
__device__ __forceinline__ int row_token(int r) { return (r & 1) ? 8 + ((r + 3) & 7) : r; }

// QUAD: at most four columns.  The MMA's eight columns are each query's two halves, side by side in a lane, which
// therefore serves one query: column 2c takes half 0 only (its q operand is zero in the other half's steps), 2c + 1
// half 1, in scores and in weights.  Else eight columns, two queries to a lane, and the halves take sums and weights
// of their own.  (32 requests x 32768 tokens with four queries a KV head: 190 us, 222 with eight columns; 40 x 3000: 37.0
// and 39.6; a tile takes 475 instructions, 630 with eight columns.)
template <bool QUAD>
struct WarpAttention {
  static constexpr int J = QUAD ? 1 : 2;  // columns (queries) of a lane
  uint32_t qf[16];          // q operand: half h, word i of the lane's K chunk -> qf[8 h + 2 i], + 1
  float scale[J];           // per column: sm_scale log2(e) 2^(24 - exponent of q)
  float qs[J][2];           // sm_scale log2(e) times the sum of q over each half
  float acc[8][4];          // O^T: half h, tile i -> acc[4 h + i], QUAD: MMA column h of the lane's two counts
  float m[J], l[J];         // running maximum (log2 units; kNoMax: none yet), this lane's share of the sum
  float zs[J][2];           // this lane's share of sum p z, per half
  uint32_t r2[J];           // power-of-two factor of p s per column: bf16 of half 0 | of half 1 << 16
  uint32_t at_k, at_m, at_v0, at_v1;  // this lane's addresses in a tile

  static __device__ __forceinline__ int lane() { return threadIdx.x & 31; }
  // the query columns of this lane's scores, and of its operand column
  static __device__ __forceinline__ int col(int j) { return QUAD ? lane() & 3 : 2 * (lane() & 3) + j; }
  static __device__ __forceinline__ int op_col() { return QUAD ? lane() >> 3 : lane() >> 2; }

  __device__ __forceinline__ void lane_addresses() {
    const uint32_t g = lane() >> 2, t = lane() & 3;
    const uint32_t tok = row_token(g);
    at_k = tok * kRec + 16 * t;                              // K codes of MMA row g; row g + 8 is the next record
    at_m = tok * kRec + kRecMeta;
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
    float q[2][16], amax = 0.f, s[2] = {0.f, 0.f};
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const uint4 v = q_raw[w];
      float* f = q[w >> 1] + 8 * (w & 1);
      f[0] = bf_lo(v.x); f[1] = bf_hi(v.x); f[2] = bf_lo(v.y); f[3] = bf_hi(v.y);
      f[4] = bf_lo(v.z); f[5] = bf_hi(v.z); f[6] = bf_lo(v.w); f[7] = bf_hi(v.w);
    }
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        amax = fmaxf(amax, fabsf(q[h][i]));
        s[h] += q[h][i];
      }
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
      s[0] += __shfl_xor_sync(0xffffffffu, s[0], o);
      s[1] += __shfl_xor_sync(0xffffffffu, s[1], o);
    }
    // clamped so that 2^(24 - e) stays finite: |q| up to 2^105 is held
    const int e = amax > 0.f ? min(120, max(-90, 13 - ((__float_as_int(amax) >> 23) - 127))) : 0;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      // MMA column lane / 4; QUAD: of query column lane / 8, even ones half 0, odd ones half 1
      const float f = QUAD && ((lane() >> 2) & 1) != h ? 0.f : pow2i(h ? e - 4 : e);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        qf[8 * h + 2 * i] = pack_half2(q[h][4 * i] * f, q[h][4 * i + 2] * f);
        qf[8 * h + 2 * i + 1] = pack_half2(q[h][4 * i + 1] * f, q[h][4 * i + 3] * f);
      }
    }
    const float sc = qk_scale * pow2i(24 - e);
#pragma unroll
    for (int j = 0; j < J; ++j) {  // from a lane whose operand column is the lane's column j
      const int src = QUAD ? 8 * t : 8 * t + 4 * j;
      scale[j] = __shfl_sync(0xffffffffu, sc, src);
      qs[j][0] = __shfl_sync(0xffffffffu, s[0], src) * qk_scale;
      qs[j][1] = __shfl_sync(0xffffffffu, s[1], src) * qk_scale;
      m[j] = kNoMax;
      l[j] = zs[j][0] = zs[j][1] = 0.f;
      r2[j] = 0x7e807e80u;  // 2^126
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[i][j] = 0.f;
  }

  __device__ __forceinline__ float r(int j, int h) const { return h ? bf_hi(r2[j]) : bf_lo(r2[j]); }
  // The largest of a column's lanes.
  static __device__ __forceinline__ float column_max(float x) {
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
    return x;
  }
  // Column j's running maximum takes in mx (the lane's largest score): by how many octaves its weights fall.  Sums of
  // weights follow; the accumulators' part is set_factor's.
  __device__ __forceinline__ int raise_max(float mx, int j) {
    const float to = column_max(mx), up = ceilf(to - m[j]);
    const int d = up > 0.f ? (int)fminf(up, 300.f) : 0;
    const float al = d > 126 ? 0.f : pow2i(-d);
    if (d > 0) m[j] = d == 300 ? to : m[j] + up;  // none before, or nothing left of it
    l[j] *= al;
    zs[j][0] *= al;
    zs[j][1] *= al;
    return d;
  }
  // Column j, half h: its factor becomes 2^e (e <= 126) after weights fell by d octaves, but rises by no more than d:
  // what is in the accumulators never grows.
  __device__ __forceinline__ void set_factor(int j, int h, int e, int d) {
    const int now = (int)(h ? r2[j] >> 23 : r2[j] >> 7 & 0xffu) - 127 + d, to = min(now, max(-126, e));
    const float f = to - now < -126 ? 0.f : pow2i(to - now);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if ((k & 1) == (QUAD ? h : j)) acc[4 * h + i][k] *= f;
    r2[j] = __byte_perm(r2[j], (to + 127) << 7, h ? 0x5410 : 0x3254);
  }

  // One tile of 32 records at shared address `sm`.  MASK: the lane's column j sees only the tokens whose bit is set in
  // sees[j]; what the others' records hold (stale bytes, NaN scales) does not enter.
  template <bool MASK>
  __device__ __forceinline__ void tile(uint32_t sm, const uint32_t (&sees)[J]) {
    uint32_t in[J];  // bit 16 b + k: this lane's token k of block b
#pragma unroll
    for (int j = 0; j < J; ++j) in[j] = MASK ? sees[j] >> row_token(lane() >> 2) : 0u;
    float x[2][2][J];      // scores: block, token, column
    uint32_t vm[2][2][2];  // value scale and offset of this lane's four tokens, per half
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      const uint4 ka = lds128(sm + at_k, 16 * b * kRec), kb = lds128(sm + at_k, (16 * b + 1) * kRec);
      const uint4 ma = lds128(sm + at_m, 16 * b * kRec), mb = lds128(sm + at_m, (16 * b + 1) * kRec);
      float c[2][4];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 4; ++i) c[h][i] = 0.f;
      const uint32_t wa[4] = {ka.x, ka.y, ka.z, ka.w}, wb[4] = {kb.x, kb.y, kb.z, kb.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t a = wa[i], d = wb[i], a8 = a >> 8, d8 = d >> 8;
        mma_f16(c[0], a & kLoMask, d & kLoMask, a8 & kLoMask, d8 & kLoMask, qf[2 * i], qf[2 * i + 1]);
        mma_f16(c[QUAD ? 0 : 1], a & kHiMask, d & kHiMask, a8 & kHiMask, d8 & kHiMask, qf[8 + 2 * i], qf[8 + 2 * i + 1]);
      }
      const uint32_t km[2][2] = {{ma.x, ma.y}, {mb.x, mb.y}};
      vm[b][0][0] = ma.z; vm[b][0][1] = ma.w;
      vm[b][1][0] = mb.z; vm[b][1][1] = mb.w;
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int j = 0; j < J; ++j) {
          const float d0 = c[0][2 * k + j], d1 = QUAD ? c[0][2 * k + 1] : c[1][2 * k + j];
          const float y = fmaf(bf_lo(km[k][1]), d1, bf_lo(km[k][0]) * d0);
          const float z = fmaf(bf_hi(km[k][1]), qs[j][1], bf_hi(km[k][0]) * qs[j][0]);
          float v = fmaf(y, scale[j], z);
          if (MASK && !(in[j] >> (16 * b + k) & 1u)) v = -INFINITY;
          x[b][k][j] = v;
        }
    }
    // m is the same in all lanes of a column and nothing moves until some lane sees a score kSlack above it (weights
    // up to 2^kSlack are as good as weights up to 1, and new maxima are common) or a weight that fp16 may not hold.
    // That takes a scale above kCap / 2^kSlack / r; where there is one, the lane's largest weight times its largest
    // scale is a closer bound.  (32 requests x 32768 tokens 188 us, and 195 where every tile has such scales: an early
    // token that takes most of the weight and whose values are 2^-10 of the others'.)
    float mx[J];
#pragma unroll
    for (int j = 0; j < J; ++j) mx[j] = fmaxf(fmaxf(x[0][0][j], x[0][1][j]), fmaxf(x[1][0][j], x[1][1][j]));
    uint32_t s2 = 0u;  // the lane's largest scales, one bf16 for each half
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const bool used = !MASK || ((in[0] | in[J - 1]) >> (16 * (i >> 1) + (i & 1)) & 1u);
      const uint32_t v = __byte_perm(vm[i >> 1][i & 1][0], vm[i >> 1][i & 1][1], 0x5410);
      s2 = max_bf16x2(s2, used ? v : 0u);
    }
    const uint32_t sr = mul_bf16x2(s2, J == 1 ? r2[0] : max_bf16x2(r2[0], r2[J - 1]));
    bool above = false;
#pragma unroll
    for (int j = 0; j < J; ++j) above = above || mx[j] > m[j] + kSlack;
    if (__any_sync(0xffffffffu, above || sr >= kWide << 16 || sr << 16 >= kWide << 16)) {
#pragma unroll
      for (int j = 0; j < J; ++j) {
        const float e = ex2(mx[j] - m[j]);
        above = above || fmaxf(e * bf_lo(s2) * r(j, 0), e * bf_hi(s2) * r(j, 1)) > kCap;
      }
      if (__any_sync(0xffffffffu, above)) {
        float lg[2][4];  // log2 of the scales
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int i = 0; i < 4; ++i) lg[h][i] = lg2(bf_lo(vm[i >> 1][i & 1][h]));
#pragma unroll
        for (int j = 0; j < J; ++j) {
          float top[2];  // log2 of the tile's largest p s; -inf where the column does not see, a NaN drops
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            top[h] = -INFINITY;
#pragma unroll
            for (int i = 0; i < 4; ++i) top[h] = fmaxf(top[h], x[i >> 1][i & 1][j] + lg[h][i]);
            top[h] = column_max(top[h]);
          }
          const int d = raise_max(mx[j], j);
#pragma unroll
          for (int h = 0; h < 2; ++h) set_factor(j, h, kTop - 1 - max(kTop - 1 - 126, __float2int_rd(top[h] - m[j])), d);
        }
      }
    }
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      uint32_t pw[2][2];  // weights, turned: tokens of MMA rows 0..7, of rows 8..15; per half (QUAD: both in one)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        float w[2][J];
        float p[J];
#pragma unroll
        for (int j = 0; j < J; ++j) {
          p[j] = ex2(x[b][k][j] - m[j]);
          l[j] += p[j];
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          // second tokens enter as -s (15 - c) + (z + 15 s)
          const float s1 = bf_lo(vm[b][k][h]);
          const float zv = k ? fmaf(15.f, s1, bf_hi(vm[b][k][h])) : bf_hi(vm[b][k][h]);
#pragma unroll
          for (int j = 0; j < J; ++j) {
            const bool seen = !MASK || (in[j] >> (16 * b + k) & 1u);
            w[h][j] = seen ? p[j] * s1 * (k ? -r(j, h) : r(j, h)) : 0.f;  // in this order: s r may pass fp32
            if (MASK)
              zs[j][h] += seen ? p[j] * zv : 0.f;
            else
              zs[j][h] = fmaf(p[j], zv, zs[j][h]);
          }
        }
        if (QUAD) {
          pw[k][0] = pw[k][1] = transpose8x8(pack_half2(w[0][0], w[1][0]));
        } else {
          pw[k][0] = transpose8x8(pack_half2(w[0][0], w[0][J - 1]));
          pw[k][1] = transpose8x8(pack_half2(w[1][0], w[1][J - 1]));
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
        mma_f16(acc[4 + i], u & kHiMask, u8 & kHiMask, ~w & kHiMask, ~w8 & kHiMask, pw[0][1], pw[1][1]);
      }
    }
  }

  // ---- bf16 rows among the records (QUAD, one query row, in column 0): tiles of 8 rows of K, then 8 of V, 256 bytes
  // each, 16-byte chunk c of row i at chunk c ^ i.  Scores: MMA rows g and g + 8 are the two halves of K row g, columns
  // 0 and 1 the halves of q; the score is their diagonal's sum.  Values go into the records' accumulators: weights
  // carry the factors that those carry, as two bf16 terms (16 bits), the second in the unused columns of query 1.
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
    const float m0 = __shfl_sync(0xffffffffu, m[0], lane() & 28);
    if (t != 0) {
      m[0] = m0;
      l[0] = zs[0][0] = zs[0][1] = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = 0.f;
    }
    // one factor for a row's two terms, and none that would carry a large row past fp32
    r2[0] = __shfl_sync(0xffffffffu, r2[0], lane() & 28);
#pragma unroll
    for (int h = 0; h < 2; ++h)
      set_factor(0, h, kRowTop, 0);
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
    v = (in >> g & 1u) ? fmaf(v, qk_scale, b) : -INFINITY;
    if (__any_sync(0xffffffffu, v > m[0] + kSlack)) {
      const int d = raise_max(v, 0);
#pragma unroll
      for (int h = 0; h < 2; ++h) set_factor(0, h, kRowTop, d);
    }
    const float p = ex2(v - m[0]);
    l[0] += p;
    float w[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const float full = p * (r(0, h) * pow2i(h ? -20 : -24)), hi = bf_round(full);
      w[h] = t == 0 ? hi : t == 1 ? full - hi : 0.f;
    }
    const uint32_t pw = transpose8x8((uint32_t)f2bf_bits(w[0]) | ((uint32_t)f2bf_bits(w[1]) << 16));
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
  // after the last rows(): the second terms join column 0
  __device__ __forceinline__ void end_rows() {
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const float low = __shfl_down_sync(0xffffffffu, acc[4 * h + i][2 * k + h], 1);
          if ((lane() & 3) == 0) acc[4 * h + i][2 * k + h] += low;
        }
  }

  // Every lane's sums over its column's lanes.
  __device__ __forceinline__ void add_up() {
#pragma unroll
    for (int j = 0; j < J; ++j) {
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) {
        l[j] += __shfl_xor_sync(0xffffffffu, l[j], o);
        zs[j][0] += __shfl_xor_sync(0xffffffffu, zs[j][0], o);
        zs[j][1] += __shfl_xor_sync(0xffffffffu, zs[j][1], o);
      }
    }
  }
  // after add_up(): dims 64 h + 8 (lane / 4) .. + 7 of column j, unnormalised.  Codes were 2^-24 (half 1: 2^-20) and
  // weights r times too large; 1 / r is a power of two, exact.  No step on the way is larger than the result: both
  // factors in one for r >= 1, else first u, which leaves r times the result.
  __device__ __forceinline__ void dims(int j, int h, float (&o)[8]) const {
    const float f = 1.f / r(j, h), u = pow2i(h ? 20 : 24), z = zs[j][h];
    const float first = f > 1.f ? u : 1.f, then = f > 1.f ? f : u * f;
    const int k = QUAD ? h : j;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      o[2 * i] = fmaf(acc[4 * h + i][k] * first, then, z);
      o[2 * i + 1] = fmaf(acc[4 * h + i][2 + k] * first, then, z);
    }
  }

  // The warp's unnormalised result of each column c < ncol: part[c * kD + d], ml[2 c] = m, ml[2 c + 1] = l.
  __device__ __forceinline__ void finish(float* part, float* ml, int ncol) {
    const int g = lane() >> 2;
    add_up();
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const int c = col(j);
      if (c < ncol) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float o[8];
          dims(j, h, o);
          float4* dst = reinterpret_cast<float4*>(part + c * kD + 64 * h + 8 * g);
          dst[0] = make_float4(o[0], o[1], o[2], o[3]);
          dst[1] = make_float4(o[4], o[5], o[6], o[7]);
        }
        if (g == 0) {
          ml[2 * c] = m[j];
          ml[2 * c + 1] = l[j];
        }
      }
    }
  }
};

}  // namespace oa
