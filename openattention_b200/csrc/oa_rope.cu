// Rows on their way into attention: per-head RMS norm and position rotation of queries and keys, and the
// 4-bit cache write of keys and values (layout: oa_kv4.cuh), in one pass over the rows.
//
//   y = x * rsqrt(mean(x^2) + eps) * w            (optional, fp32)
//   o[d] = y[d] * cos[p, d] + rot(y)[d] * sin[p, d]   for d < R;  rot(y) = [-y[R/2 .. R), y[0 .. R/2)]
//   o[d] = y[d]                                       for d >= R
// with p = start[b] + offset + i the position of row i of request b.  Both products and the sum round
// separately in fp32, as the eager expression does, so a caller that moves from it keeps its bits; the
// result is rounded once to the rows' type.
//
// Layout: a half-warp owns one head row at a time, lane l dims 4l .. 4l+3 and 64 + 4l .. + 3: a full rotation (R =
// 128) mixes dims of one lane, a byte of codes is one lane's, and loads and stores are 128-byte runs.  A warp takes a
// token's rows two at a time ("slots": two query rows, or the K and the V row of one head, whose record it writes
// whole), kSlots loads in flight; cos and sin stay in registers for all of them.
//
// What bounds it: memory, for long prompts.  32768 tokens of 32 + 8 heads in bf16: 109 us, 6.5 TB/s (with the norm 119);
// rope_append 129 us, floor 113.  Four loads in flight against one: 112 and 142 us; a warp for a whole token against
// one for every slot: 112 and 242.  A decode step's rows take a launch's time.
#include "oa_kv4.cuh"

namespace oa {
namespace {

constexpr int kRowThreads = 256;

struct RowArgs {
  Rows q, k, v;
  Rows qo, ko;           // outputs (p is written)
  unsigned char* cache;  // records, or NULL
  int64_t c_sb, c_sh, Lmax;
  const float* cos;
  const float* sin;
  int64_t P;
  int R;
  PerRequest start, lens;
  int64_t offset;
  const void* wq;
  const void* wk;
  int w_f32;
  float eps;
  int zero_q, zero_k;  // write zeros into padding rows
  int B, T, HQ, HKV;
  int slots, per;      // slots of a token (append_kernel: pairs of heads), slots a warp takes
};

// The lane's part of a row: dims 4l .. (a) and 64 + 4l .. (b); p at dim 4l.  Held as loaded, so that several rows'
// loads are in flight before the first is used.  Plain loads: rows may be rotated where they stand, and the read-only
// path is for memory that no one writes during the launch.
template <typename E>
struct Quads;
template <>
struct Quads<__nv_bfloat16> {
  uint2 a, b;
  __device__ __forceinline__ void load(const __nv_bfloat16* p) {
    a = *reinterpret_cast<const uint2*>(p);
    b = *reinterpret_cast<const uint2*>(p + 64);
  }
  __device__ __forceinline__ void get(float (&x)[8]) const {
    x[0] = bf_lo(a.x); x[1] = bf_hi(a.x); x[2] = bf_lo(a.y); x[3] = bf_hi(a.y);
    x[4] = bf_lo(b.x); x[5] = bf_hi(b.x); x[6] = bf_lo(b.y); x[7] = bf_hi(b.y);
  }
  // bf16x2 of dims (4l + i, 64 + 4l + i)
  __device__ __forceinline__ void pairs(uint32_t (&v)[4]) const {
    v[0] = __byte_perm(a.x, b.x, 0x5410);
    v[1] = __byte_perm(a.x, b.x, 0x7632);
    v[2] = __byte_perm(a.y, b.y, 0x5410);
    v[3] = __byte_perm(a.y, b.y, 0x7632);
  }
};
template <>
struct Quads<float> {
  float4 a, b;
  __device__ __forceinline__ void load(const float* p) {
    a = *reinterpret_cast<const float4*>(p);
    b = *reinterpret_cast<const float4*>(p + 64);
  }
  __device__ __forceinline__ void get(float (&x)[8]) const {
    x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
    x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
  }
  __device__ __forceinline__ void pairs(uint32_t (&v)[4]) const {}  // caches take bf16 rows
};
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ void store_quads(__nv_bfloat16* p, const float (&x)[8]) {
  *reinterpret_cast<uint2*>(p) = make_uint2(pack2(x[0], x[1]), pack2(x[2], x[3]));
  *reinterpret_cast<uint2*>(p + 64) = make_uint2(pack2(x[4], x[5]), pack2(x[6], x[7]));
}
__device__ __forceinline__ void store_quads(float* p, const float (&x)[8]) {
  *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
  *reinterpret_cast<float4*>(p + 64) = make_float4(x[4], x[5], x[6], x[7]);
}
// cos or sin of the lane's dims (0 beyond R)
__device__ __forceinline__ void load_table(const float* row, int R, int hl, float (&c)[8]) {
  const float4 none = make_float4(0.f, 0.f, 0.f, 0.f);
  const float4 a = 4 * hl < R ? *reinterpret_cast<const float4*>(row + 4 * hl) : none;
  const float4 b = 64 + 4 * hl < R ? *reinterpret_cast<const float4*>(row + 64 + 4 * hl) : none;
  c[0] = a.x; c[1] = a.y; c[2] = a.z; c[3] = a.w;
  c[4] = b.x; c[5] = b.y; c[6] = b.z; c[7] = b.w;
}

// the lane's norm weights
__device__ __forceinline__ void load_weights(const void* w, int w_f32, int hl, float (&wf)[8]) {
  if (w_f32) {
    Quads<float> v;
    v.load(static_cast<const float*>(w) + 4 * hl);
    v.get(wf);
  } else {
    Quads<__nv_bfloat16> v;
    v.load(static_cast<const __nv_bfloat16*>(w) + 4 * hl);
    v.get(wf);
  }
}
__device__ __forceinline__ void norm_row(float (&x)[8], const float (&wf)[8], float eps) {
  float ss = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) ss = fmaf(x[i], x[i], ss);
#pragma unroll
  for (int o = 8; o >= 1; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
  const float inv = rsqrtf(ss * (1.f / kD) + eps);
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = x[i] * inv * wf[i];
}

// FULL: R = 128, a lane's dims d and d + 64 rotate into each other.  Else the partner of quad i (of 32) is quad
// i +- R/8, in another lane.  Called by whole warps.
template <bool FULL>
__device__ __forceinline__ void rotate_row(float (&x)[8], const float (&cs)[8], const float (&sn)[8], int R, int hl) {
  if (FULL) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float a = x[i], b = x[4 + i];
      x[i] = __fsub_rn(__fmul_rn(a, cs[i]), __fmul_rn(b, sn[i]));
      x[4 + i] = __fadd_rn(__fmul_rn(b, cs[4 + i]), __fmul_rn(a, sn[4 + i]));
    }
    return;
  }
  const int h = R >> 3;  // quads in half a rotation
  float y[8];
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    const int quad = 16 * s + hl;
    const bool first = quad < h, any = quad < 2 * h;
    const int from = any ? (first ? quad + h : quad - h) : quad;
    const int src = (threadIdx.x & 16) | (from & 15);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float a = __shfl_sync(0xffffffffu, x[i], src), b = __shfl_sync(0xffffffffu, x[4 + i], src);
      const float other = from < 16 ? a : b;
      y[4 * s + i] = any ? __fadd_rn(__fmul_rn(x[4 * s + i], cs[4 * s + i]), __fmul_rn(first ? -other : other, sn[4 * s + i]))
                         : x[4 * s + i];
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = y[i];
}

__device__ __forceinline__ uint32_t min_bf2(uint32_t a, uint32_t b) {  // NaN if either is
  uint32_t r;
  asm("min.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ uint32_t max_bf2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

// 1 / x in two terms, off by 2^-45 of it: of a normal number with a normal reciprocal
struct Reciprocal {
  float hi, lo;
  explicit __device__ __forceinline__ Reciprocal(float x) {
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(hi) : "f"(x));
    lo = fmaf(-x, hi, 1.f) * hi;
  }
  // a / x, rounded once as far as 45 bits tell: exact where it is a float (a tie between two codes among them)
  __device__ __forceinline__ float times(float a) const { return fmaf(a, hi, a * lo); }
};

// Scale of the group in the low (0) or high (1) halves of the two packed extremes.
__device__ __forceinline__ float group_scale(uint32_t lo2, uint32_t hi2, int g) {
  const float lo = g ? bf_hi(lo2) : bf_lo(lo2), hi = g ? bf_hi(hi2) : bf_lo(hi2);
  const float d = hi - lo, q = d * (1.f / 15.f);
  return bf_round(fmaf(fmaf(-q, 15.f, d), 1.f / 15.f, q));  // a quotient's one correction by its remainder
}
// The lane's codes, dims (i, 64 + i) in a byte, and both groups' (scale, offset) words.  kLift: some scale is near
// fp32's smallest numbers (or zero).
template <bool kLift, int N>
__device__ __forceinline__ void code_groups(const uint32_t (&v)[N], uint32_t lo2, float s0, float s1, uint32_t (&word)[N / 4],
                                            uint32_t (&out)[2]) {
  constexpr float kRound = 12582912.f;  // 0x4b400000: a code is the sum's lowest byte
#pragma unroll
  for (int j = 0; j < N / 4; ++j) word[j] = 0u;
#pragma unroll
  for (int g = 0; g < 2; ++g) {
    const float lo = g ? bf_hi(lo2) : bf_lo(lo2), s = g ? s1 : s0;
    const bool ok = s < INFINITY;  // a NaN, an infinity or a range past fp32 is not
    const float lift = kLift && s < 0x1p-60f ? 0x1p80f : 1.f, ss = kLift ? s * lift : s;
    const Reciprocal inv(kLift && s == 0.f ? 1.f : ss);  // a scale of 0: all differences are 0
#pragma unroll
    for (int j = 0; j < N / 4; ++j) {
      uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float d = (g ? bf_hi(v[4 * j + i]) : bf_lo(v[4 * j + i])) - lo;
        if (kLift) d *= lift;
        float q = inv.times(d);
        if (kLift) q = fminf(q, 15.f);  // a normal scale is off by 2^-8 at most, its quotients stay under 15.06
        w[i] = __float_as_uint(q + kRound);
      }
      const uint32_t codes4 = __byte_perm(__byte_perm(w[0], w[1], 0x0040), __byte_perm(w[2], w[3], 0x0040), 0x5410);
      word[j] |= ok ? codes4 << (4 * g) : 0u;
    }
    out[g] = ok ? pack2(s, lo) : 0x00007fc0u;
  }
}

// A row that 64 / N lanes hold, lane l as bf16x2 of dims (N l + i, 64 + N l + i), into one side of a record.  The halves
// of the head lie side by side, so one bf16x2 minimum and maximum serve both groups; NaN and infinities show in them.
// Adding 3 * 2^22 to a quotient rounds it to the nearest whole number, ties to even, in the low bits.  Scales near
// fp32's smallest are lifted by 2^80 first.  Called by whole warps; live: the row is stored.
template <int N>
__device__ __forceinline__ void quantise_row(const uint32_t (&v)[N], unsigned char* codes, int meta, int l, bool live) {
  uint32_t lo2 = v[0], hi2 = v[0];
#pragma unroll
  for (int i = 1; i < N; ++i) {
    lo2 = min_bf2(lo2, v[i]);
    hi2 = max_bf2(hi2, v[i]);
  }
#pragma unroll
  for (int o = 32 / N; o >= 1; o >>= 1) {
    lo2 = min_bf2(lo2, __shfl_xor_sync(0xffffffffu, lo2, o));
    hi2 = max_bf2(hi2, __shfl_xor_sync(0xffffffffu, hi2, o));
  }
  uint32_t word[N / 4], out[2];
  const float s0 = group_scale(lo2, hi2, 0), s1 = group_scale(lo2, hi2, 1);
  if (__any_sync(0xffffffffu, fminf(s0, s1) < 0x1p-60f))
    code_groups<true>(v, lo2, s0, s1, word, out);
  else
    code_groups<false>(v, lo2, s0, s1, word, out);
  if (!live) return;
#pragma unroll
  for (int j = 0; j < N / 4; ++j) reinterpret_cast<uint32_t*>(codes + N * l)[j] = word[j];
  if (l == 0) *reinterpret_cast<uint2*>(codes + meta) = make_uint2(out[0], out[1]);
}

// One half-warp's rows h0, h0 + step, ... below h1 of one token, kSlots at a time: normalised, rotated, stored.  Rows
// behind h1 are read as row h0 and dropped.  Called by whole warps (their half-warps differ in h0).
template <typename E, bool FULL, int kSlots>
__device__ __forceinline__ void rotate_rows(const E* p, int64_t sh, E* out, int64_t oh, int h0, int h1, int half, const void* weight,
                                            const RowArgs& a, const float (&cs)[8], const float (&sn)[8], int hl) {
  float wf[8];
  if (weight) load_weights(weight, a.w_f32, hl, wf);
  for (int h = h0; h < h1; h += 2 * kSlots) {
    Quads<E> raw[kSlots];
#pragma unroll
    for (int j = 0; j < kSlots; ++j) {
      const int r = h + 2 * j + half;
      raw[j].load(p + (r < h1 ? r : h0) * sh);
    }
#pragma unroll
    for (int j = 0; j < kSlots; ++j) {
      const int r = h + 2 * j + half;
      float x[8];
      raw[j].get(x);
      if (weight) norm_row(x, wf, a.eps);
      rotate_row<FULL>(x, cs, sn, a.R, hl);
      if (r < h1) store_quads(out + r * oh, x);
    }
  }
}

// Slots of a token: with a cache, slot i < HKV is K (first half-warp) and V (second) of head i, then two query rows
// each; else two query rows each, then two key rows each.
template <typename E, bool CACHE, bool FULL, int kSlots>
__global__ void __launch_bounds__(kRowThreads) rows_kernel(const RowArgs a) {
  const int lane = threadIdx.x & 31, hl = lane & 15, half = lane >> 4;
  const unsigned token = blockIdx.x * (kRowThreads / 32) + (threadIdx.x >> 5);
  if (token >= (unsigned)a.B * a.T) return;
  const unsigned b = a.T == 1 ? token : token / a.T, t = token - b * a.T;
  const int64_t pos = per_request(a.start, b) + a.offset + t;
  bool live = a.lens.p == nullptr || (int64_t)t < per_request(a.lens, b);
  live = live && pos >= 0 && pos < a.P;
  const int s0 = blockIdx.y * a.per, s1 = min(s0 + a.per, a.slots);
  const E* q = static_cast<const E*>(a.q.p) + b * a.q.sb + t * a.q.st + 4 * hl;
  E* qo = static_cast<E*>(const_cast<void*>(a.qo.p)) + b * a.qo.sb + t * a.qo.st + 4 * hl;
  // this warp's query rows [q0, q1) and key (or key and value) rows [k0, k1)
  const int nq = (a.HQ + 1) / 2;
  const int q0 = 2 * (CACHE ? max(0, s0 - a.HKV) : min(s0, nq)), q1 = min(a.HQ, 2 * (CACHE ? max(0, s1 - a.HKV) : s1));
  const int k0 = CACHE ? s0 : 2 * max(0, s0 - nq), k1 = min(a.HKV, CACHE ? s1 : 2 * max(0, s1 - nq));
  if (!live) {
    const float zero[8] = {};
    if (a.zero_q)
      for (int h = q0 + half; h < q1; h += 2) store_quads(qo + h * a.qo.sh, zero);
    if (!CACHE && a.zero_k) {
      E* ko = static_cast<E*>(const_cast<void*>(a.ko.p)) + b * a.ko.sb + t * a.ko.st + 4 * hl;
      for (int h = k0 + half; h < k1; h += 2) store_quads(ko + h * a.ko.sh, zero);
    }
    return;
  }
  float cs[8], sn[8];
  load_table(a.cos + pos * a.R, a.R, hl, cs);
  load_table(a.sin + pos * a.R, a.R, hl, sn);
  if (CACHE && k0 < k1 && pos >= 0 && pos < a.Lmax) {
    const Rows& r = half ? a.v : a.k;
    const E* p = static_cast<const E*>(r.p) + b * r.sb + t * r.st + 4 * hl + k0 * r.sh;
    const int64_t sh = r.sh;
    unsigned char* codes = a.cache + b * a.c_sb + k0 * a.c_sh + pos * kRec + (half ? kRecV : 0);
    const int meta = half ? kRecMeta + 8 - kRecV : kRecMeta;
    float wf[8];
    if (a.wk) load_weights(a.wk, a.w_f32, hl, wf);
    auto write = [&](const Quads<E>& raw) {  // one head's K and V row into its record
      uint32_t v[4];
      raw.pairs(v);
      // the V rows of the warp go through the shuffles with the K rows and come out as they were
      float x[8];
      raw.get(x);
      if (a.wk) norm_row(x, wf, a.eps);
      rotate_row<FULL>(x, cs, sn, a.R, hl);
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = half ? v[i] : pack2(x[i], x[4 + i]);  // the cache holds bf16 rows
      quantise_row(v, codes, meta, hl, true);
      codes += a.c_sh;
    };
    int h = k0;
    for (; h + kSlots <= k1; h += kSlots) {
      Quads<E> raw[kSlots];
#pragma unroll
      for (int j = 0; j < kSlots; ++j, p += sh) raw[j].load(p);
#pragma unroll
      for (int j = 0; j < kSlots; ++j) write(raw[j]);
    }
    for (; h < k1; ++h, p += sh) {
      Quads<E> raw;
      raw.load(p);
      write(raw);
    }
  }
  if (!CACHE && k0 < k1) {
    const E* k = static_cast<const E*>(a.k.p) + b * a.k.sb + t * a.k.st + 4 * hl;
    E* ko = static_cast<E*>(const_cast<void*>(a.ko.p)) + b * a.ko.sb + t * a.ko.st + 4 * hl;
    rotate_rows<E, FULL, kSlots>(k, a.k.sh, ko, a.ko.sh, k0, k1, half, a.wk, a, cs, sn, hl);
  }
  if (q0 < q1) rotate_rows<E, FULL, kSlots>(q, a.q.sh, qo, a.qo.sh, q0, q1, half, a.wq, a, cs, sn, hl);
}

// Rows into the cache as they are.  Eight lanes to a row, lane l dims 8l .. 8l + 7 and 64 + 8l .. + 7 (a row's minimum and
// maximum are then three exchanges, and what a group costs once is shared by two heads' rows); a warp takes the K and V
// rows of two heads at a time, kPairs of them in flight.  32768 tokens of 8 heads: 45 us, 3.8 TB/s; bound by issue (114
// instructions a record; sixteen lanes to a row took 147 and 59 us).
template <int kPairs>
__global__ void __launch_bounds__(kRowThreads) append_kernel(const RowArgs a) {
  const int lane = threadIdx.x & 31, l = lane & 7, side = lane >> 3 & 1, sub = lane >> 4;
  const unsigned token = blockIdx.x * (kRowThreads / 32) + (threadIdx.x >> 5);
  if (token >= (unsigned)a.B * a.T) return;
  const unsigned b = a.T == 1 ? token : token / a.T, t = token - b * a.T;
  const int64_t pos = per_request(a.start, b) + a.offset + t;
  if (pos < 0 || pos >= a.Lmax || (a.lens.p && (int64_t)t >= per_request(a.lens, b))) return;
  const Rows& r = side ? a.v : a.k;
  const __nv_bfloat16* p = static_cast<const __nv_bfloat16*>(r.p) + b * r.sb + t * r.st + 8 * l;
  const int64_t sh = r.sh;
  unsigned char* rec = a.cache + b * a.c_sb + pos * kRec + (side ? kRecV : 0);
  const int meta = side ? kRecMeta + 8 - kRecV : kRecMeta;
  const int h1 = min(a.HKV, 2 * (blockIdx.y + 1) * a.per);
  for (int h0 = 2 * blockIdx.y * a.per; h0 < h1; h0 += 2 * kPairs) {
    uint4 x[kPairs][2];
#pragma unroll
    for (int j = 0; j < kPairs; ++j) {  // heads behind the last are read as the first, and dropped
      const int h = h0 + 2 * j + sub;
      const uint4* from = reinterpret_cast<const uint4*>(p + (h < h1 ? h : h0) * sh);
      x[j][0] = __ldg(from);
      x[j][1] = __ldg(from + 8);
    }
#pragma unroll
    for (int j = 0; j < kPairs; ++j) {
      if (h0 + 2 * j >= h1) break;
      const int h = h0 + 2 * j + sub;
      const uint32_t lo[4] = {x[j][0].x, x[j][0].y, x[j][0].z, x[j][0].w}, hi[4] = {x[j][1].x, x[j][1].y, x[j][1].z, x[j][1].w};
      uint32_t v[8];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[2 * i] = __byte_perm(lo[i], hi[i], 0x5410);
        v[2 * i + 1] = __byte_perm(lo[i], hi[i], 0x7632);
      }
      quantise_row(v, rec + h * a.c_sh, meta, l, h < h1);
    }
  }
}

// Records back to rows: a half-warp per record, lane l the code words l (dims 4l.. and 64 + 4l..), kRecords in flight.
// 32768 tokens of 8 heads: 35 us, 4.9 TB/s.
struct UnpackArgs {
  const unsigned char* cache;
  int64_t c_sb, c_sh, Lmax;
  PerRequest start, lens;
  int64_t offset;
  Rows ko, vo;
  int zero_k, zero_v;
  int B, T, HKV;
  unsigned ctas;  // for one head's T records
};

// a word's eight codes as values: bytes 0..3 low nibbles, then high ones.  0x4b000000 + n is the float 2^23 + n.
__device__ __forceinline__ void unpack_word(uint32_t w, uint32_t m0, uint32_t m1, float (&v)[8]) {
  const uint32_t lo = w & 0x0f0f0f0fu, hi = (w >> 4) & 0x0f0f0f0fu;
  const float s0 = bf_lo(m0), z0 = bf_hi(m0), s1 = bf_lo(m1), z1 = bf_hi(m1);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[i] = fmaf(s0, __uint_as_float(__byte_perm(lo, 0x4b000000u, 0x7440 + i)) - 8388608.f, z0);
    v[4 + i] = fmaf(s1, __uint_as_float(__byte_perm(hi, 0x4b000000u, 0x7440 + i)) - 8388608.f, z1);
  }
}

constexpr int kRecords = 2;

template <typename E>
__global__ void __launch_bounds__(kRowThreads) unpack_kernel(const UnpackArgs a) {
  const int hl = threadIdx.x & 15;
  const unsigned head = blockIdx.x / a.ctas, b = head / a.HKV, h = head - b * a.HKV;
  const unsigned hw = ((blockIdx.x - head * a.ctas) * kRowThreads + threadIdx.x) >> 4;
  const int64_t first = per_request(a.start, b) + a.offset;
  const int64_t len = a.lens.p ? per_request(a.lens, b) : a.T;
  const unsigned char* rec = a.cache + b * a.c_sb + h * a.c_sh;
  uint32_t kw[kRecords], vw[kRecords];
  uint4 m[kRecords];
  bool live[kRecords];
#pragma unroll
  for (int i = 0; i < kRecords; ++i) {
    const int64_t t = (int64_t)hw * kRecords + i, pos = first + t;
    live[i] = t < a.T && t < len && pos >= 0 && pos < a.Lmax;
    kw[i] = vw[i] = 0u;
    m[i] = make_uint4(0u, 0u, 0u, 0u);
    if (live[i]) {
      const unsigned char* p = rec + pos * kRec;
      kw[i] = *reinterpret_cast<const uint32_t*>(p + 4 * hl);
      vw[i] = *reinterpret_cast<const uint32_t*>(p + kRecV + 4 * hl);
      m[i] = *reinterpret_cast<const uint4*>(p + kRecMeta);
    }
  }
#pragma unroll
  for (int i = 0; i < kRecords; ++i) {  // what is not live reads as zeros
    const int64_t t = (int64_t)hw * kRecords + i;
    if (t >= a.T) break;
    float v[8];
    if (live[i] || a.zero_k) {
      unpack_word(kw[i], m[i].x, m[i].y, v);
      store_quads(static_cast<E*>(const_cast<void*>(a.ko.p)) + b * a.ko.sb + h * a.ko.sh + t * a.ko.st + 4 * hl, v);
    }
    if (live[i] || a.zero_v) {
      unpack_word(vw[i], m[i].z, m[i].w, v);
      store_quads(static_cast<E*>(const_cast<void*>(a.vo.p)) + b * a.vo.sb + h * a.vo.sh + t * a.vo.st + 4 * hl, v);
    }
  }
}

// ---------------------------------------------------------------- host side
// What a launch over tokens and slots of a token needs: a warp takes as many slots (keeping the token's table entries)
// as still leave 24 warps to each of 148 SMs.  (2048 tokens: 8.2 us with 8 to 24 warps to an SM, 9.8 with 48; 4096:
// 14.3 and, with 96, 16.6.)  With four slots or more, four are in flight; fewer would leave loads unused.
int plan_rows(RowArgs& a, int slots, const char* fn, dim3* grid) {
  const int64_t tokens = (int64_t)a.B * a.T;
  OA_REQUIRE(tokens <= 0x7fffffff, "%s: too many rows", fn);
  a.slots = slots;
  a.per = (int)std::min<int64_t>(slots, std::max<int64_t>(1, tokens * slots / (148 * 24)));
  while ((slots + a.per - 1) / a.per > 65535) a.per *= 2;
  *grid = dim3((unsigned)((tokens + kRowThreads / 32 - 1) / (kRowThreads / 32)), (slots + a.per - 1) / a.per);
  return OA_OK;
}
template <typename E, bool CACHE, bool FULL>
int launch_rows(RowArgs& a, const char* fn, cudaStream_t st) {
  const int slots = (CACHE ? a.HKV : (a.HKV + 1) / 2) + (a.HQ + 1) / 2;
  if (a.B == 0 || a.T == 0 || slots == 0) return OA_OK;
  dim3 grid;
  OA_TRY(plan_rows(a, slots, fn, &grid));
  if (a.per >= 4)
    rows_kernel<E, CACHE, FULL, 4><<<grid, kRowThreads, 0, st>>>(a);
  else
    rows_kernel<E, CACHE, FULL, 1><<<grid, kRowThreads, 0, st>>>(a);
  return oa_check_launch(fn);
}
template <typename E, bool CACHE>
int launch_rows(RowArgs& a, const char* fn, cudaStream_t st) {
  return a.R == kD ? launch_rows<E, CACHE, true>(a, fn, st) : launch_rows<E, CACHE, false>(a, fn, st);
}
int launch_append(RowArgs& a, const char* fn, cudaStream_t st) {
  if (a.B == 0 || a.T == 0 || a.HKV == 0) return OA_OK;
  dim3 grid;
  OA_TRY(plan_rows(a, (a.HKV + 1) / 2, fn, &grid));
  if (a.per >= 4)
    append_kernel<4><<<grid, kRowThreads, 0, st>>>(a);
  else
    append_kernel<1><<<grid, kRowThreads, 0, st>>>(a);
  return oa_check_launch(fn);
}

// The parts of a block that oa_qk_norm_rope and oa_kv4_append share.
template <typename Args>
int take_rope(const char* fn, const Args& g, RowArgs& a) {
  OA_REQUIRE(g.cos && g.sin && oa_aligned16(g.cos) && oa_aligned16(g.sin), "%s: cos/sin must be 16-byte aligned", fn);
  OA_REQUIRE(g.P >= 0 && g.R >= 16 && g.R <= kD && g.R % 16 == 0,
             "%s: the rotated width must be a multiple of 16 in 16..128 (got %lld)", fn, (long long)g.R);
  OA_REQUIRE(g.w_dtype == OA_BF16 || g.w_dtype == OA_F32, "%s: w_dtype must be OA_BF16 or OA_F32", fn);
  OA_REQUIRE(oa_aligned16(g.q_weight) && oa_aligned16(g.k_weight), "%s: weights must be 16-byte aligned", fn);
  a.cos = g.cos;
  a.sin = g.sin;
  a.P = g.P;
  a.R = (int)g.R;
  a.wq = g.q_weight;
  a.wk = g.k_weight;
  a.w_f32 = g.w_dtype == OA_F32;
  a.eps = (float)g.eps;
  a.zero_q = g.zero_q != 0;
  return OA_OK;
}

}  // namespace
}  // namespace oa

extern "C" int oa_qk_norm_rope(const oa_qk_norm_rope_args* args, void* stream) {
  const char* fn = "oa_qk_norm_rope";
  OA_REQUIRE(args != nullptr, "%s: null arguments", fn);
  const oa_qk_norm_rope_args& g = *args;
  OA_REQUIRE(g.dtype == OA_BF16 || g.dtype == OA_F32, "%s: dtype must be OA_BF16 or OA_F32", fn);
  oa::RowArgs a{};
  const int es = g.dtype == OA_F32 ? 4 : 2;
  const int64_t B = g.q.size[0], HQ = g.q.size[1], T = g.q.size[2], HKV = g.k.size[1];
  OA_TRY(oa_take_rows(fn, "q", g.q, es, B, -1, T, false, &a.q));
  OA_TRY(oa_take_rows(fn, "k", g.k, es, B, -1, T, false, &a.k));
  OA_TRY(oa_take_rows(fn, "q_out", g.q_out, es, B, HQ, T, true, &a.qo));
  OA_TRY(oa_take_rows(fn, "k_out", g.k_out, es, B, HKV, T, true, &a.ko));
  OA_TRY(oa::take_rope(fn, g, a));
  OA_TRY(oa_take_index(fn, "start", g.start, B, true, &a.start));
  OA_TRY(oa_take_index(fn, "lens", g.lens, B, false, &a.lens));
  a.zero_k = g.zero_k != 0;
  a.offset = g.offset;
  a.B = (int)B; a.T = (int)T; a.HQ = (int)HQ; a.HKV = (int)HKV;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return g.dtype == OA_F32 ? oa::launch_rows<float, false>(a, fn, st) : oa::launch_rows<__nv_bfloat16, false>(a, fn, st);
}

extern "C" int oa_kv4_append(const oa_kv4_append_args* args, void* stream) {
  const char* fn = "oa_kv4_append";
  OA_REQUIRE(args != nullptr, "%s: null arguments", fn);
  const oa_kv4_append_args& g = *args;
  oa::RowArgs a{};
  const unsigned char* cache;
  OA_TRY(oa_take_cache(fn, g.cache, true, &cache, &a.c_sb, &a.c_sh));
  a.cache = const_cast<unsigned char*>(cache);
  a.Lmax = g.cache.size[2];
  const int64_t B = g.cache.size[0], HKV = g.cache.size[1], T = g.k.size[2];
  OA_TRY(oa_take_rows(fn, "k", g.k, 2, B, HKV, T, false, &a.k));
  OA_TRY(oa_take_rows(fn, "v", g.v, 2, B, HKV, T, false, &a.v));
  int64_t HQ = 0;
  if (g.cos || g.sin || g.q.p || g.q_out.p) {
    HQ = g.q.size[1];
    OA_TRY(oa_take_rows(fn, "q", g.q, 2, B, -1, T, false, &a.q));
    OA_TRY(oa_take_rows(fn, "q_out", g.q_out, 2, B, HQ, T, true, &a.qo));
    OA_TRY(oa::take_rope(fn, g, a));
  } else {
    OA_REQUIRE(!g.q_weight && !g.k_weight, "%s: norm weights need the cos/sin tables", fn);
  }
  OA_TRY(oa_take_index(fn, "start", g.start, B, true, &a.start));
  OA_TRY(oa_take_index(fn, "lens", g.lens, B, false, &a.lens));
  a.offset = g.offset;
  a.B = (int)B; a.T = (int)T; a.HQ = (int)HQ; a.HKV = (int)HKV;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  return a.cos ? oa::launch_rows<__nv_bfloat16, true>(a, fn, st) : oa::launch_append(a, fn, st);
}

extern "C" int oa_kv4_unpack(const oa_kv4_unpack_args* args, void* stream) {
  const char* fn = "oa_kv4_unpack";
  OA_REQUIRE(args != nullptr, "%s: null arguments", fn);
  const oa_kv4_unpack_args& g = *args;
  OA_REQUIRE(g.dtype == OA_BF16 || g.dtype == OA_F32, "%s: dtype must be OA_BF16 or OA_F32", fn);
  oa::UnpackArgs a{};
  OA_TRY(oa_take_cache(fn, g.cache, false, &a.cache, &a.c_sb, &a.c_sh));
  a.Lmax = g.cache.size[2];
  const int64_t B = g.cache.size[0], HKV = g.cache.size[1], T = g.k_out.size[2];
  const int es = g.dtype == OA_F32 ? 4 : 2;
  OA_TRY(oa_take_rows(fn, "k_out", g.k_out, es, B, HKV, T, true, &a.ko));
  OA_TRY(oa_take_rows(fn, "v_out", g.v_out, es, B, HKV, T, true, &a.vo));
  OA_TRY(oa_take_index(fn, "start", g.start, B, true, &a.start));
  OA_TRY(oa_take_index(fn, "lens", g.lens, B, false, &a.lens));
  a.offset = g.offset;
  a.zero_k = g.zero_k != 0;
  a.zero_v = g.zero_v != 0;
  a.B = (int)B; a.T = (int)T; a.HKV = (int)HKV;
  if (B == 0 || T == 0 || HKV == 0) return OA_OK;
  const int64_t per_cta = oa::kRowThreads / 16 * oa::kRecords, ctas = (T + per_cta - 1) / per_cta;
  OA_REQUIRE(B * HKV <= 0x7fffffff / ctas, "%s: too many rows", fn);
  a.ctas = (unsigned)ctas;
  const unsigned grid = (unsigned)(B * HKV * ctas);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (g.dtype == OA_F32)
    oa::unpack_kernel<float><<<grid, oa::kRowThreads, 0, st>>>(a);
  else
    oa::unpack_kernel<__nv_bfloat16><<<grid, oa::kRowThreads, 0, st>>>(a);
  return oa_check_launch(fn);
}
