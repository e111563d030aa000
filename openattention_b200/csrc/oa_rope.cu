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
// Layout: a half-warp owns one head row at a time, lane l dims 8l .. 8l+7 (16 bytes of bf16), so the
// rotation's partner dims are R/16 lanes away and a quantisation group is eight lanes.
#include "oa_kv4.cuh"

namespace oa {
namespace {

constexpr int kRowThreads = 256;

struct RowArgs {
  Rows q, k, v;
  Rows qo, ko;         // outputs (p is written)
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
  int heads;   // head rows per token this call handles: HQ + HKV, + HKV values with a cache
  int chunks;  // half-warps per token
};

__device__ __forceinline__ void load8(const __nv_bfloat16* p, float (&x)[8]) {
  const uint4 w = *reinterpret_cast<const uint4*>(p);
  x[0] = bf_lo(w.x); x[1] = bf_hi(w.x); x[2] = bf_lo(w.y); x[3] = bf_hi(w.y);
  x[4] = bf_lo(w.z); x[5] = bf_hi(w.z); x[6] = bf_lo(w.w); x[7] = bf_hi(w.w);
}
__device__ __forceinline__ void load8(const float* p, float (&x)[8]) {
  const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
  x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
  x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
}
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  return (uint32_t)f2bf_bits(lo) | ((uint32_t)f2bf_bits(hi) << 16);
}
__device__ __forceinline__ void store8(__nv_bfloat16* p, const float (&x)[8]) {
  *reinterpret_cast<uint4*>(p) = make_uint4(pack2(x[0], x[1]), pack2(x[2], x[3]), pack2(x[4], x[5]), pack2(x[6], x[7]));
}
__device__ __forceinline__ void store8(float* p, const float (&x)[8]) {
  reinterpret_cast<float4*>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
}

// The half-warp's row x (bf16 values) quantised into one side of a record: `codes` its 64 code bytes,
// `meta` its two (scale, offset) words.
__device__ __forceinline__ void quantise_row(const float (&x)[8], unsigned char* codes, unsigned char* meta,
                                             unsigned hmask) {
  const int hl = threadIdx.x & 15;
  float lo = x[0], hi = x[0];
  bool finite = true;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    lo = fminf(lo, x[i]);
    hi = fmaxf(hi, x[i]);
    finite = finite && fabsf(x[i]) < INFINITY;
  }
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) {
    lo = fminf(lo, __shfl_xor_sync(hmask, lo, o));
    hi = fmaxf(hi, __shfl_xor_sync(hmask, hi, o));
  }
  const unsigned bad = __ballot_sync(hmask, !finite);
  float s = bf_round(__fdiv_rn(hi - lo, 15.f));
  const bool ok = (bad & (0xffu << (threadIdx.x & 24))) == 0u && s < INFINITY;  // a range past fp32 counts as infinite
  if (!ok) s = __uint_as_float(0x7fc00000u);
  uint32_t w[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    w[h] = 0u;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float c = s > 0.f ? fminf(rintf(__fdiv_rn(x[4 * h + i] - lo, s)), 15.f) : 0.f;
      w[h] |= (uint32_t)c << (8 * i);
    }
  }
  // lane l < 8 holds the low nibbles of bytes 8l .. 8l+7, lane l + 8 their high nibbles: each writes four bytes
  const bool upper = hl >= 8;
  const uint32_t other = __shfl_xor_sync(hmask, upper ? w[0] : w[1], 8);
  const uint32_t word = upper ? (other | (w[1] << 4)) : (w[0] | (other << 4));
  *reinterpret_cast<uint32_t*>(codes + 8 * (hl & 7) + (upper ? 4 : 0)) = word;
  if ((hl & 7) == 0) *reinterpret_cast<uint32_t*>(meta + (upper ? 4 : 0)) = pack2(s, ok ? lo : 0.f);
}

template <typename E, bool CACHE, int HPW>
__global__ void __launch_bounds__(kRowThreads) rows_kernel(const RowArgs a) {
  const int lane = threadIdx.x & 31, hl = lane & 15;
  const unsigned hmask = 0xffffu << (lane & 16);
  const int64_t hw = ((int64_t)blockIdx.x * kRowThreads + threadIdx.x) >> 4;
  const int64_t token = hw / a.chunks;
  if (token >= (int64_t)a.B * a.T) return;
  const int chunk = (int)(hw - token * a.chunks);
  const int64_t b = token / a.T, t = token - b * a.T;
  const int64_t pos = per_request(a.start, b) + a.offset + t;
  bool live = a.lens.p == nullptr || t < per_request(a.lens, b);
  if (a.cos) live = live && pos >= 0 && pos < a.P;
  const int h0 = chunk * HPW, h1 = min(h0 + HPW, a.heads);
  const int d0 = 8 * hl;

  float x[HPW][8];
#pragma unroll
  for (int j = 0; j < HPW; ++j) {
    const int h = h0 + j;
    if (live && h < h1) {
      const bool isq = h < a.HQ, isk = !isq && h < a.HQ + a.HKV;
      const Rows& r = isq ? a.q : isk ? a.k : a.v;
      const int64_t hh = isq ? h : isk ? h - a.HQ : h - a.HQ - a.HKV;
      load8(static_cast<const E*>(r.p) + b * r.sb + hh * r.sh + t * r.st + d0, x[j]);
    }
  }
  float cs[8], sn[8];
  const bool rot = a.cos && d0 < a.R;
  int src = hl;
  float sign = 0.f;
  if (live && rot) {
    load8(a.cos + pos * a.R + d0, cs);
    load8(a.sin + pos * a.R + d0, sn);
    const bool first = d0 < (a.R >> 1);
    src = first ? hl + (a.R >> 4) : hl - (a.R >> 4);
    sign = first ? -1.f : 1.f;
  }
#pragma unroll
  for (int j = 0; j < HPW; ++j) {
    const int h = h0 + j;
    if (h >= h1) continue;
    const bool isq = h < a.HQ, isk = !isq && h < a.HQ + a.HKV;
    const int64_t hh = isq ? h : isk ? h - a.HQ : h - a.HQ - a.HKV;
    if (live && (isq || isk)) {
      const void* w = isq ? a.wq : a.wk;
      if (w != nullptr) {
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) ss = fmaf(x[j][i], x[j][i], ss);
#pragma unroll
        for (int o = 8; o >= 1; o >>= 1) ss += __shfl_xor_sync(hmask, ss, o);
        const float inv = rsqrtf(ss * (1.f / kD) + a.eps);
        float wf[8];
        if (a.w_f32)
          load8(static_cast<const float*>(w) + d0, wf);
        else
          load8(static_cast<const __nv_bfloat16*>(w) + d0, wf);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[j][i] = x[j][i] * inv * wf[i];
      }
      if (a.cos) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float other = __shfl_sync(hmask, x[j][i], (lane & 16) | src);
          if (rot) x[j][i] = __fadd_rn(__fmul_rn(x[j][i], cs[i]), __fmul_rn(sign * other, sn[i]));
        }
      }
    }
    if (isq || (isk && !CACHE)) {
      const Rows& o = isq ? a.qo : a.ko;
      E* dst = static_cast<E*>(const_cast<void*>(o.p)) + b * o.sb + hh * o.sh + t * o.st + d0;
      if (live) {
        store8(dst, x[j]);
      } else if (isq ? a.zero_q : a.zero_k) {
        const float zero[8] = {};
        store8(dst, zero);
      }
    } else if (CACHE && live && pos >= 0 && pos < a.Lmax) {
      unsigned char* rec = a.cache + b * a.c_sb + hh * a.c_sh + pos * kRec;
      if (isk) {  // the cache holds bf16 rows' values: round the rotated key first
#pragma unroll
        for (int i = 0; i < 8; ++i) x[j][i] = bf_round(x[j][i]);
      }
      quantise_row(x[j], rec + (isk ? 0 : kRecV), rec + kRecMeta + (isk ? 0 : 8), hmask);
    }
  }
}

// Records back to rows: a half-warp per record, lane l the code words l (dims 4l.. and 64 + 4l..).
struct UnpackArgs {
  const unsigned char* cache;
  int64_t c_sb, c_sh, Lmax;
  PerRequest start, lens;
  int64_t offset;
  Rows ko, vo;
  int zero_k, zero_v;
  int B, T, HKV;
};

template <typename E>
__device__ __forceinline__ void store4(E* p, float a, float b, float c, float d);
template <>
__device__ __forceinline__ void store4(__nv_bfloat16* p, float a, float b, float c, float d) {
  *reinterpret_cast<uint2*>(p) = make_uint2(pack2(a, b), pack2(c, d));
}
template <>
__device__ __forceinline__ void store4(float* p, float a, float b, float c, float d) {
  *reinterpret_cast<float4*>(p) = make_float4(a, b, c, d);
}

template <typename E>
__device__ __forceinline__ void unpack_row(uint32_t w, uint32_t m0, uint32_t m1, E* dst) {
  const float s0 = bf_lo(m0), z0 = bf_hi(m0), s1 = bf_lo(m1), z1 = bf_hi(m1);
  float v[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[i] = fmaf(s0, (float)((w >> (8 * i)) & 15u), z0);
    v[4 + i] = fmaf(s1, (float)((w >> (8 * i + 4)) & 15u), z1);
  }
  store4(dst, v[0], v[1], v[2], v[3]);
  store4(dst + 64, v[4], v[5], v[6], v[7]);
}

template <typename E>
__global__ void __launch_bounds__(kRowThreads) unpack_kernel(const UnpackArgs a) {
  const int hl = threadIdx.x & 15;
  const int64_t hw = ((int64_t)blockIdx.x * kRowThreads + threadIdx.x) >> 4;
  if (hw >= (int64_t)a.B * a.HKV * a.T) return;
  const int64_t bh = hw / a.T, t = hw - bh * a.T;
  const int64_t b = bh / a.HKV, h = bh - b * a.HKV;
  const int64_t pos = per_request(a.start, b) + a.offset + t;
  const bool live = (a.lens.p == nullptr || t < per_request(a.lens, b)) && pos >= 0 && pos < a.Lmax;
  E* kd = static_cast<E*>(const_cast<void*>(a.ko.p)) + b * a.ko.sb + h * a.ko.sh + t * a.ko.st + 4 * hl;
  E* vd = static_cast<E*>(const_cast<void*>(a.vo.p)) + b * a.vo.sb + h * a.vo.sh + t * a.vo.st + 4 * hl;
  if (live) {
    const unsigned char* rec = a.cache + b * a.c_sb + h * a.c_sh + pos * kRec;
    const uint32_t kw = *reinterpret_cast<const uint32_t*>(rec + 4 * hl);
    const uint32_t vw = *reinterpret_cast<const uint32_t*>(rec + kRecV + 4 * hl);
    const uint4 m = *reinterpret_cast<const uint4*>(rec + kRecMeta);
    unpack_row(kw, m.x, m.y, kd);
    unpack_row(vw, m.z, m.w, vd);
  } else {
    if (a.zero_k) store4(kd, 0.f, 0.f, 0.f, 0.f), store4(kd + 64, 0.f, 0.f, 0.f, 0.f);
    if (a.zero_v) store4(vd, 0.f, 0.f, 0.f, 0.f), store4(vd + 64, 0.f, 0.f, 0.f, 0.f);
  }
}

// ---------------------------------------------------------------- host side
template <typename E, bool CACHE>
int launch_rows(RowArgs& a, const char* fn, cudaStream_t st) {
  if (a.B == 0 || a.T == 0 || a.heads == 0) return OA_OK;
  const int hpw = (int64_t)a.B * a.T * a.heads >= 148 * 512 ? 4 : 1;
  a.chunks = (a.heads + hpw - 1) / hpw;
  const int64_t hws = (int64_t)a.B * a.T * a.chunks;
  const int64_t grid = (hws * 16 + kRowThreads - 1) / kRowThreads;
  OA_REQUIRE(grid <= 0x7fffffff, "%s: too many rows", fn);
  if (hpw == 4)
    rows_kernel<E, CACHE, 4><<<(unsigned)grid, kRowThreads, 0, st>>>(a);
  else
    rows_kernel<E, CACHE, 1><<<(unsigned)grid, kRowThreads, 0, st>>>(a);
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
  a.heads = (int)(HQ + HKV);
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
  a.heads = (int)(HQ + 2 * HKV);
  return oa::launch_rows<__nv_bfloat16, true>(a, fn, static_cast<cudaStream_t>(stream));
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
  const int64_t grid = (B * T * HKV * 16 + oa::kRowThreads - 1) / oa::kRowThreads;
  OA_REQUIRE(grid <= 0x7fffffff, "%s: too many rows", fn);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (g.dtype == OA_F32)
    oa::unpack_kernel<float><<<(unsigned)grid, oa::kRowThreads, 0, st>>>(a);
  else
    oa::unpack_kernel<__nv_bfloat16><<<(unsigned)grid, oa::kRowThreads, 0, st>>>(a);
  return oa_check_launch(fn);
}
