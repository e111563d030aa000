// Attention over the 4-bit K/V cache (record layout: oa_kv4.cuh).
//
//   z_t = sm_scale * q . K_t,   o = sum_t softmax(z)_t V_t,   K_t[d] = scale * code + offset (V alike)
//
// kv4_attention: every position below the request's length; query token i of T (at position n - T + i) sees
// positions <= n - T + i.  kv4_flash: index lists and cluster proxies (as OpenAttention.flash).  Rows with
// nothing to attend give zeros.
#include "oa_kv4.cuh"

#include "../../include/openattention_b200.h"

namespace oa {
namespace {

constexpr int kThreads = 128;
constexpr int kHalfWarps = kThreads / 16;

struct DenseArgs {
  Rows q, o;
  const unsigned char* cache;
  int64_t c_sb, c_sh, Lmax;
  PerRequest n;
  int64_t offset;
  int out_f32;
  int B, HQ, HKV, T;
  float qk_scale;  // sm_scale * log2(e)
};

struct ListArgs {
  const __nv_bfloat16* q;
  int64_t q_stride;
  const unsigned char* cache;
  int64_t c_sh, Lmax;
  const int32_t* sel;
  const int32_t* exp;
  int n_sel, n_exp, NB;
  const __nv_bfloat16* kbar;
  const __nv_bfloat16* vbar;
  int64_t kb_sh, kb_sb;
  int per_qhead;
  const float* logn;
  int64_t ln_stride;
  void* out;
  int64_t out_stride;
  int out_f32;
  int G;
  float qk_scale;
};

// One half-warp's online softmax; lane hl holds dims 4hl..4hl+3 (i < 4) and 64 + 4hl.. (i >= 4).
struct State {
  float q[8], acc[8], m, l;
  __device__ __forceinline__ void init(const __nv_bfloat16* qp, int hl) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      q[i] = __bfloat162float(qp[(i < 4 ? 4 * hl + i : 64 + 4 * hl + i - 4)]);
      acc[i] = 0.f;
    }
    m = -INFINITY;
    l = 0.f;
  }
  __device__ __forceinline__ void add(const float (&k)[8], const float (&v)[8], float scale, float bias, unsigned hmask) {
    float d = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) d = fmaf(q[i], k[i], d);
#pragma unroll
    for (int o = 8; o >= 1; o >>= 1) d += __shfl_xor_sync(hmask, d, o);
    const float z = fmaf(d, scale, bias);
    const float mx = fmaxf(m, z);
    const float base = mx == -INFINITY ? 0.f : mx;
    const float al = exp2f(m - base), p = exp2f(z - base);
    l = fmaf(l, al, p);
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[i] = fmaf(acc[i], al, p * v[i]);
    m = mx;
  }
};

__device__ __forceinline__ void record_side(const unsigned char* rec, int side, int hl, float (&x)[8]) {
  const uint32_t w = *reinterpret_cast<const uint32_t*>(rec + kRecV * side + 4 * hl);
  const uint2 mt = *reinterpret_cast<const uint2*>(rec + kRecMeta + 8 * side);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[i] = fmaf(bf_lo(mt.x), (float)((w >> (8 * i)) & 15u), bf_hi(mt.x));
    x[4 + i] = fmaf(bf_lo(mt.y), (float)((w >> (8 * i + 4)) & 15u), bf_hi(mt.y));
  }
}

__device__ __forceinline__ void merge_store(const State& s, int hw, int hl, void* out, int64_t at, int f32) {
  __shared__ float s_m[kHalfWarps], s_l[kHalfWarps], s_acc[kHalfWarps][kD];
  if (hl == 0) {
    s_m[hw] = s.m;
    s_l[hw] = s.l;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) s_acc[hw][i < 4 ? 4 * hl + i : 64 + 4 * hl + i - 4] = s.acc[i];
  __syncthreads();
  float M = -INFINITY, L = 0.f, A = 0.f;
  for (int h = 0; h < kHalfWarps; ++h) M = fmaxf(M, s_m[h]);
  const float base = M == -INFINITY ? 0.f : M;
  for (int h = 0; h < kHalfWarps; ++h) {
    const float w = exp2f(s_m[h] - base);
    L = fmaf(w, s_l[h], L);
    A = fmaf(w, s_acc[h][threadIdx.x], A);
  }
  const float o = L == 0.f ? 0.f : A / L;
  if (f32)
    static_cast<float*>(out)[at + threadIdx.x] = o;
  else
    static_cast<__nv_bfloat16*>(out)[at + threadIdx.x] = __float2bfloat16_rn(o);
}

__global__ void __launch_bounds__(kThreads) dense_kernel(const DenseArgs a) {
  const int lane = threadIdx.x & 31, hl = lane & 15, hw = threadIdx.x >> 4;
  const unsigned hmask = 0xffffu << (lane & 16);
  const int t = blockIdx.x % a.T;
  const int h = (blockIdx.x / a.T) % a.HQ;
  const int64_t b = blockIdx.x / a.T / a.HQ;
  const int64_t n = min(per_request(a.n, b) + a.offset, a.Lmax) - a.T + 1 + t;
  const unsigned char* base = a.cache + b * a.c_sb + (int64_t)(h / (a.HQ / a.HKV)) * a.c_sh;
  State s;
  s.init(static_cast<const __nv_bfloat16*>(a.q.p) + b * a.q.sb + h * a.q.sh + t * a.q.st, hl);
  for (int64_t j = hw; j < n; j += kHalfWarps) {
    float k[8], v[8];
    record_side(base + j * kRec, 0, hl, k);
    record_side(base + j * kRec, 1, hl, v);
    s.add(k, v, a.qk_scale, 0.f, hmask);
  }
  merge_store(s, hw, hl, const_cast<void*>(a.o.p), b * a.o.sb + h * a.o.sh + t * a.o.st, a.out_f32);
}

__global__ void __launch_bounds__(kThreads) list_kernel(const ListArgs a) {
  const int lane = threadIdx.x & 31, hl = lane & 15, hw = threadIdx.x >> 4;
  const unsigned hmask = 0xffffu << (lane & 16);
  const int64_t r = blockIdx.x;
  const int64_t kvh = r / a.G;
  const unsigned char* base = a.cache + kvh * a.c_sh;
  State s;
  s.init(a.q + r * a.q_stride, hl);
  for (int j = hw; j < a.n_sel + a.n_exp; j += kHalfWarps) {
    const int t = j < a.n_sel ? a.sel[r * a.n_sel + j] : a.exp[r * a.n_exp + (j - a.n_sel)];
    if (t < 0 || (int64_t)t >= a.Lmax) continue;
    float k[8], v[8];
    record_side(base + (int64_t)t * kRec, 0, hl, k);
    record_side(base + (int64_t)t * kRec, 1, hl, v);
    s.add(k, v, a.qk_scale, 0.f, hmask);
  }
  const int64_t pr = a.per_qhead ? r : kvh;
  for (int j = hw; j < a.NB; j += kHalfWarps) {
    const float ln = a.logn[r * a.ln_stride + j];
    if (ln == -INFINITY) continue;
    float k[8], v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int d = i < 4 ? 4 * hl + i : 64 + 4 * hl + i - 4;
      k[i] = __bfloat162float(a.kbar[pr * a.kb_sh + j * a.kb_sb + d]);
      v[i] = __bfloat162float(a.vbar[pr * a.kb_sh + j * a.kb_sb + d]);
    }
    s.add(k, v, a.qk_scale, ln * kLog2e, hmask);
  }
  merge_store(s, hw, hl, a.out, r * a.out_stride, a.out_f32);
}

bool rows_ok(const Rows& r, int esize) {
  const int64_t q = 16 / esize;
  return oa_aligned16(r.p) && r.sb % q == 0 && r.sh % q == 0 && r.st % q == 0;
}

}  // namespace
}  // namespace oa

extern "C" size_t oa_kv4_attention_workspace_bytes(int64_t B, int64_t HQ, int64_t HKV, int64_t T, int64_t Lmax) {
  return 0;
}

extern "C" int oa_kv4_attention(const void* q, int64_t q_sb, int64_t q_sh, int64_t q_st, const void* cache,
                                int64_t c_sb, int64_t c_sh, int64_t Lmax, const void* n, int64_t n_stride, int n_i64,
                                int64_t offset, void* out, int64_t o_sb, int64_t o_sh, int64_t o_st, int out_dtype,
                                int64_t B, int64_t HQ, int64_t HKV, int64_t T, float sm_scale, void* workspace,
                                size_t workspace_bytes, void* stream) {
  const char* fn = "oa_kv4_attention";
  OA_REQUIRE(B >= 0 && T >= 0 && HKV >= 1 && HQ >= HKV && HQ % HKV == 0,
             "%s: need B, T >= 0 and HQ a multiple of HKV (B=%lld T=%lld HQ=%lld HKV=%lld)", fn, (long long)B,
             (long long)T, (long long)HQ, (long long)HKV);
  OA_REQUIRE(B * HQ * T <= 0x7fffffff, "%s: too many rows", fn);
  OA_REQUIRE(out_dtype == OA_BF16 || out_dtype == OA_F32, "%s: out_dtype must be OA_BF16 or OA_F32", fn);
  OA_REQUIRE((cache || Lmax == 0) && oa_aligned16(cache) && c_sb % 16 == 0 && c_sh % 16 == 0 && Lmax >= 0,
             "%s: the cache and its strides must be multiples of 16 bytes", fn);
  if (B == 0 || T == 0) return OA_OK;
  OA_REQUIRE(q && out && n, "%s: null q/out/n", fn);
  oa::DenseArgs a;
  a.q = oa::Rows{q, q_sb, q_sh, q_st};
  a.o = oa::Rows{out, o_sb, o_sh, o_st};
  OA_REQUIRE(oa::rows_ok(a.q, 2) && oa::rows_ok(a.o, out_dtype == OA_F32 ? 4 : 2),
             "%s: q and out rows must start on 16-byte boundaries (base addresses and strides)", fn);
  a.cache = static_cast<const unsigned char*>(cache);
  a.c_sb = c_sb;
  a.c_sh = c_sh;
  a.Lmax = Lmax;
  a.n = oa::PerRequest{n, n_stride, n_i64};
  a.offset = offset;
  a.out_f32 = out_dtype == OA_F32;
  a.B = (int)B; a.HQ = (int)HQ; a.HKV = (int)HKV; a.T = (int)T;
  a.qk_scale = sm_scale * oa::kLog2e;
  oa::dense_kernel<<<(unsigned)(B * HQ * T), oa::kThreads, 0, static_cast<cudaStream_t>(stream)>>>(a);
  return oa_check_launch(fn);
}

extern "C" int oa_kv4_flash(const void* q, int64_t q_stride, const void* cache, int64_t c_sh, int64_t Lmax,
                            const int32_t* sel, int64_t n_sel, const int32_t* exp_idx, int64_t n_exp,
                            const void* kbar, const void* vbar, int64_t kbar_stride_h, int64_t kbar_stride_b,
                            int per_qhead, const float* log_n, int64_t log_n_stride, void* out, int64_t out_stride,
                            int out_dtype, int64_t BQ, int64_t BH, int64_t NB, float sm_scale, void* stream) {
  const char* fn = "oa_kv4_flash";
  OA_REQUIRE(BQ >= 0 && BH >= 1 && BQ % BH == 0 && BQ <= 0x7fffffff, "%s: need BQ a multiple of BH (BQ=%lld BH=%lld)",
             fn, (long long)BQ, (long long)BH);
  OA_REQUIRE(n_sel >= 0 && n_exp >= 0 && NB >= 0 && Lmax >= 0 && n_sel + n_exp + NB < (int64_t)1 << 30,
             "%s: bad list sizes", fn);
  OA_REQUIRE(out_dtype == OA_BF16 || out_dtype == OA_F32, "%s: out_dtype must be OA_BF16 or OA_F32", fn);
  if (BQ == 0) return OA_OK;
  OA_REQUIRE(q && (cache || Lmax == 0) && out, "%s: null q/cache/out", fn);
  OA_REQUIRE((n_sel == 0 || sel) && (n_exp == 0 || exp_idx), "%s: null index list", fn);
  OA_REQUIRE(NB == 0 || (kbar && vbar && log_n), "%s: null kbar/vbar/log_n with NB > 0", fn);
  OA_REQUIRE(oa_aligned16(q) && oa_aligned16(cache) && q_stride % 8 == 0 && c_sh % 16 == 0,
             "%s: q and the cache must start on 16-byte boundaries (base addresses and strides)", fn);
  OA_REQUIRE(NB == 0 || (oa_aligned16(kbar) && oa_aligned16(vbar) && kbar_stride_h % 8 == 0 && kbar_stride_b % 8 == 0),
             "%s: kbar/vbar rows must start on 16-byte boundaries", fn);
  oa::ListArgs a;
  a.q = static_cast<const __nv_bfloat16*>(q);
  a.q_stride = q_stride;
  a.cache = static_cast<const unsigned char*>(cache);
  a.c_sh = c_sh;
  a.Lmax = Lmax;
  a.sel = sel;
  a.exp = exp_idx;
  a.n_sel = (int)n_sel; a.n_exp = (int)n_exp; a.NB = (int)NB;
  a.kbar = static_cast<const __nv_bfloat16*>(kbar);
  a.vbar = static_cast<const __nv_bfloat16*>(vbar);
  a.kb_sh = kbar_stride_h;
  a.kb_sb = kbar_stride_b;
  a.per_qhead = per_qhead;
  a.logn = log_n;
  a.ln_stride = log_n_stride;
  a.out = out;
  a.out_stride = out_stride;
  a.out_f32 = out_dtype == OA_F32;
  a.G = (int)(BQ / BH);
  a.qk_scale = sm_scale * oa::kLog2e;
  oa::list_kernel<<<(unsigned)BQ, oa::kThreads, 0, static_cast<cudaStream_t>(stream)>>>(a);
  return oa_check_launch(fn);
}
