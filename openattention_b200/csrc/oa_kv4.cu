// Attention over the 4-bit K/V cache (record layout: oa_kv4.cuh).
//
//   z_t = sm_scale * q . K_t,   o = sum_t softmax(z)_t V_t,   K_t[d] = scale * code + offset (V alike)
//
// kv4_attention: every position below the request's length; query token i of T (at position n - T + i) sees
// positions <= n - T + i.  kv4_flash: index lists and cluster proxies (as OpenAttention.flash).  Rows with
// nothing to attend give zeros.
#include "oa_kv4_mma.cuh"

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

// ---------------------------------------------------------------- dense
// Work: a row is (request, KV head, block of up to 8 query columns); its tiles of 32 records are spread over
// CTAs of 8 warps, each warp with its own ring of kStages tiles filled by asynchronous copies (the 4608 bytes
// of a tile are contiguous).  Lengths live on the device, so each CTA finds its share itself:
//  - each row its own CTAs, grid / rows of them (no more than one per 8 tiles), where that balances;
//  - else the tiles of all rows in one line, cut into equal parts; a CTA then ends one row and begins the next.
// A row that one CTA covers is written by it.  Otherwise each part leaves (m, l, O) in the workspace and the
// last CTA to arrive (atomic ticket, no waiting) merges the parts in CTA order, so the result does not depend
// on which CTA is last.
constexpr int kWarps = 8;
constexpr int kDenseThreads = 32 * kWarps;
constexpr int kStages = 3;
constexpr int kCols = 8;
constexpr int kRowUnits = 12;  // what a row costs a CTA besides its tiles, in tiles (query, merge, idle pipeline)
constexpr int kPartFloats = kCols * kD + 2 * kCols;  // one part: O of 8 columns, then their (m, l)
constexpr int kRingBytes = kWarps * kStages * kTileBytes;

struct DensePlan {
  int blocks;    // column blocks of a KV head: ceil(G T / 8)
  int64_t rows;  // B * HKV * blocks
  int grid;
};

DensePlan dense_plan(int64_t B, int64_t HQ, int64_t HKV, int64_t T, int64_t Lmax) {
  DensePlan p;
  int dev = 0, sms = 0;
  if (cudaGetDevice(&dev) != cudaSuccess ||
      cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || sms < 1) {
    sms = 148;
    (void)cudaGetLastError();  // a host without a GPU sizes for a B200
  }
  p.blocks = (int)((HQ / HKV * T + kCols - 1) / kCols);
  p.rows = B * HKV * p.blocks;
  const int64_t tiles = (Lmax + kTile - 1) / kTile;
  const int64_t parts = std::max<int64_t>(1, (tiles + kWarps - 1) / kWarps);
  // two CTAs per SM (their rings fill its shared memory); no more than one per row and 8 tiles
  p.grid = p.rows > 2 * sms ? 2 * sms : (int)std::max<int64_t>(1, std::min<int64_t>(2 * sms, p.rows * parts));
  return p;
}

struct DenseWork {
  unsigned blocks, per_req, rows;  // column blocks of a KV head; rows of a request; rows
  unsigned cpr;                    // CTAs a row can have to itself: grid / rows
  float* parts;                    // 2 per CTA: [0] of a row that began in an earlier CTA, [1] of one that begins here
  unsigned* tickets;               // one per row, zero between calls
};

__device__ __forceinline__ int dense_len(const DenseArgs& a, int64_t b) {
  const int64_t n = min(per_request(a.n, b) + a.offset, a.Lmax);
  return n < 0 ? 0 : (int)n;
}
// a row without records still has its zeros to write: one (empty) tile
__device__ __forceinline__ int dense_tiles(int n) { return n <= kTile ? 1 : (int)(((unsigned)n + kTile - 1) / kTile); }

__device__ __forceinline__ void axpy(float4& y, float f, const float4& x) {
  y.x = fmaf(f, x.x, y.x);
  y.y = fmaf(f, x.y, y.y);
  y.z = fmaf(f, x.z, y.z);
  y.w = fmaf(f, x.w, y.w);
}
// dims 4 lane .. 4 lane + 3 of the output row at element `at`
__device__ __forceinline__ void store_out4(void* out, int out_f32, int64_t at, int lane, const float4& A, float L) {
  const float inv = L == 0.f ? 0.f : 1.f / L;
  const float4 o = L == 0.f ? make_float4(0.f, 0.f, 0.f, 0.f) : make_float4(A.x * inv, A.y * inv, A.z * inv, A.w * inv);
  if (out_f32) {
    *reinterpret_cast<float4*>(static_cast<float*>(out) + at + 4 * lane) = o;
  } else {
    uint2 w;
    w.x = (uint32_t)f2bf_bits(o.x) | ((uint32_t)f2bf_bits(o.y) << 16);
    w.y = (uint32_t)f2bf_bits(o.z) | ((uint32_t)f2bf_bits(o.w) << 16);
    *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(out) + at + 4 * lane) = w;
  }
}

// The parts of one row, part v at src (v = 0) or src + (2 v - 1) kPartFloats.  Every thread sums four dims of one
// column over its share of the parts, kAhead loads in flight; the first ones are issued before the weights
// 2^(m_v - M) are known.  The shares are added in a fixed order.  o_at: the output row of column `warp`.
// Inlined, and kAhead no larger: a call, or more loads held, spills the caller's main loop.
template <int kAhead>
__device__ __forceinline__ void merge_parts(const float* src, int parts, int ncol, float* sh, void* out, int out_f32,
                                         int64_t o_at) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  float* s_l = sh;                   // per column
  float* s_f = sh + kCols;           // [part][column]
  float* s_a = s_f + kCols * parts;  // [share][column][128]
  const int quads = ncol * (kD / 4), shares = kDenseThreads / quads;  // ncol <= 8: at least one share
  const int share = tid / quads, qd = tid - share * quads, col = qd / (kD / 4);
  auto at = [&](int v) { return src + (v ? 2 * v - 1 : 0) * (int64_t)kPartFloats; };
  float4 x[kAhead];
  if (share < shares) {
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
      if (share + i * shares < parts) x[i] = __ldcg(reinterpret_cast<const float4*>(at(share + i * shares)) + qd);
  }
  if (warp < ncol) {  // the weights of column `warp`
    float M = -INFINITY, L = 0.f;
    for (int v = lane; v < parts; v += 32) {
      const float m = __ldcg(at(v) + kCols * kD + 2 * warp);
      s_f[v * kCols + warp] = m;
      M = fmaxf(M, m);
    }
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
    M = biased(M);
    for (int v = lane; v < parts; v += 32) {
      const float f = ex2(s_f[v * kCols + warp] - M);
      L = fmaf(f, __ldcg(at(v) + kCols * kD + 2 * warp + 1), L);
      s_f[v * kCols + warp] = f;
    }
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) L += __shfl_xor_sync(0xffffffffu, L, o);
    if (lane == 0) s_l[warp] = L;
  }
  __syncthreads();
  if (share < shares) {
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int v = share; v < parts;) {
#pragma unroll
      for (int i = 0; i < kAhead; ++i, v += shares)
        if (v < parts) axpy(acc, s_f[v * kCols + col], x[i]);
#pragma unroll
      for (int i = 0; i < kAhead; ++i)
        if (v + i * shares < parts) x[i] = __ldcg(reinterpret_cast<const float4*>(at(v + i * shares)) + qd);
    }
    reinterpret_cast<float4*>(s_a)[share * quads + qd] = acc;
  }
  __syncthreads();
  if (warp < ncol) {
    float4 A = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int v = 0; v < shares; ++v) axpy(A, 1.f, reinterpret_cast<const float4*>(s_a)[v * quads + 32 * warp + lane]);
    store_out4(out, out_f32, o_at, lane, A, s_l[warp]);
  }
}

// A CTA's way along the line of rows: the row it is at and its tiles of that row.  Counts of units fit 31 bits
// (checked by the host).
struct DenseShare {
  unsigned b, r;          // request, row within it
  int n, tiles;           // the request's length, a row's tiles
  int tile, share;        // first tile and number of tiles of this CTA's part
  bool own;               // the row's CTAs serve no other row
  unsigned line;          // where the part begins on the line (units)
  int left, off;          // units of this CTA's share from there on; units of the row before the part
  unsigned each, extra;   // the line's cut: `extra` CTAs take each + 1 units, the others `each`
  unsigned first, parts;  // own: the row's CTAs
};
// the CTA that unit u belongs to, and where a CTA's units begin
__device__ __forceinline__ unsigned cta_of(const DenseShare& s, unsigned u) {
  const unsigned big = s.extra * (s.each + 1);
  return u < big ? u / (s.each + 1) : s.extra + (u - big) / s.each;
}
__device__ __forceinline__ unsigned cta_begin(const DenseShare& s, unsigned cta) {
  return cta * s.each + min(cta, s.extra);
}

// False: nothing for this CTA.  Every thread of the CTA finds the same.
__device__ __forceinline__ bool dense_share(const DenseArgs& a, const DenseWork& w, DenseShare& s) {
  __shared__ unsigned s_pre[kDenseThreads];  // units of a row of each request before thread i's requests
  __shared__ unsigned s_sum[kWarps];
  __shared__ int s_most[kWarps];
  const unsigned tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const unsigned grid = gridDim.x, cta = blockIdx.x;
  const unsigned c = ((unsigned)a.B + kDenseThreads - 1) / kDenseThreads;  // requests a thread sums
  const bool same = a.n.stride == 0;
  unsigned units;
  int most;
  if (same) {
    s.n = dense_len(a, 0);
    most = dense_tiles(s.n);
    units = a.B * (unsigned)(most + kRowUnits);
  } else {
    unsigned sum = 0;
    most = 0;
    for (unsigned b = tid * c; b < min((tid + 1) * c, (unsigned)a.B); ++b) {
      const int k = dense_tiles(dense_len(a, b));
      sum += k + kRowUnits;
      most = max(most, k);
    }
    unsigned inc = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned v = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += v;
    }
    most = __reduce_max_sync(0xffffffffu, most);
    if (lane == 31) s_sum[warp] = inc;
    if (lane == 0) s_most[warp] = most;
    __syncthreads();
    unsigned before = 0;
    units = 0;
#pragma unroll
    for (unsigned i = 0; i < kWarps; ++i) {
      if (i < warp) before += s_sum[i];
      units += s_sum[i];
      most = max(most, s_most[i]);
    }
    s_pre[tid] = before + inc - sum;
    __syncthreads();
  }
  const unsigned total = units * w.per_req;
  s.own = w.cpr >= 1 && (kRowUnits + (most + w.cpr - 1) / w.cpr) * (8u * grid) <= max((kRowUnits + kWarps) * 8u * grid, 9u * total);
  if (s.own) {
    const unsigned row = cta / w.cpr, j = cta - row * w.cpr;
    if (row >= w.rows) return false;
    s.b = row / w.per_req;
    s.r = row - s.b * w.per_req;
    if (!same) s.n = dense_len(a, s.b);
    s.tiles = dense_tiles(s.n);
    s.parts = min(w.cpr, (unsigned)(s.tiles + kWarps - 1) / kWarps);
    if (j >= s.parts) return false;
    const unsigned each = s.tiles / s.parts, extra = s.tiles - each * s.parts;
    s.tile = j * each + min(j, extra);
    s.share = each + (j < extra ? 1 : 0);
    s.first = cta - j;
    return true;
  }
  const unsigned active = min(grid, (total + kRowUnits + kWarps - 1) / (kRowUnits + kWarps));
  if (cta >= active) return false;
  s.each = total / active;
  s.extra = total - s.each * active;
  s.line = cta_begin(s, cta);
  s.left = s.each + (cta < s.extra ? 1 : 0);
  const unsigned v = s.line / w.per_req;
  unsigned p;
  if (same) {
    s.tiles = most;
    s.b = v / (most + kRowUnits);
    p = s.b * (most + kRowUnits);
  } else {
    unsigned lo = 0, hi = kDenseThreads;  // the last thread whose requests begin at or before v
    while (hi - lo > 1) {
      const unsigned mid = (lo + hi) >> 1;
      if (s_pre[mid] <= v) lo = mid; else hi = mid;
    }
    s.b = lo * c;
    p = s_pre[lo];
    s.n = dense_len(a, s.b);
    s.tiles = dense_tiles(s.n);
    while (p + s.tiles + kRowUnits <= v) {
      p += s.tiles + kRowUnits;
      s.n = dense_len(a, ++s.b);
      s.tiles = dense_tiles(s.n);
    }
  }
  const unsigned rem = s.line - p * w.per_req;
  s.r = rem / (s.tiles + kRowUnits);
  s.off = rem - s.r * (s.tiles + kRowUnits);
  s.tile = max(0, s.off - kRowUnits);
  s.share = min(s.tiles, s.off + s.left - kRowUnits) - s.tile;
  return true;
}

// The next row on the line, if any of its tiles are this CTA's.
__device__ __forceinline__ bool dense_next(const DenseArgs& a, const DenseWork& w, DenseShare& s) {
  const int step = s.tiles + kRowUnits - s.off;
  s.line += step;
  s.left -= step;
  if (s.left <= kRowUnits) return false;
  if (++s.r == w.per_req) {
    s.r = 0;
    ++s.b;
    if (a.n.stride) {
      s.n = dense_len(a, s.b);
      s.tiles = dense_tiles(s.n);
    }
  }
  s.tile = 0;
  s.off = 0;
  s.share = min(s.tiles, s.left - kRowUnits);
  return true;
}

template <bool PAIR>
__global__ void __launch_bounds__(kDenseThreads, 2) dense_kernel(const DenseArgs a, const DenseWork w) {
  extern __shared__ __align__(16) unsigned char s_ring[];
  __shared__ unsigned s_last;
  __shared__ DenseShare s;  // the same for all threads: kept here, out of the loop's registers
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int G = a.HQ / a.HKV, cols = G * a.T;
  const unsigned cta = blockIdx.x;
  {
    DenseShare mine;
    if (!dense_share(a, w, mine)) return;
    if (tid == 0) s = mine;
  }
  __syncthreads();

  const uint32_t ring = smem_u32(s_ring) + warp * (kStages * kTileBytes);
  float* s_part = reinterpret_cast<float*>(s_ring);  // reused once a row's tiles are done
  WarpAttention<PAIR> at;
  at.lane_addresses();

  for (;;) {
    if (s.share <= 0) return;  // the share ends before the row's first tile
    const int kvh = s.r / w.blocks;
    const int col0 = (s.r - kvh * w.blocks) * kCols, ncol = min(kCols, cols - col0);
    // the query row of column c: head h0 + (col0 + c) / T, query token (col0 + c) % T
    const int64_t q_at = s.b * a.q.sb + (int64_t)(kvh * G) * a.q.sh;
    auto split = [&](int c, int& hh, int& tt) {
      hh = a.T == 1 ? col0 + c : (col0 + c) / a.T;
      tt = col0 + c - hh * a.T;
    };
    {
      int hh, tt;
      split(at.op_col(), hh, tt);
      at.load_q(at.op_col() < ncol ? static_cast<const __nv_bfloat16*>(a.q.p) + q_at + hh * a.q.sh + tt * a.q.st : nullptr);
    }
    const int t0 = s.tile + warp, t1 = s.tile + s.share, n = s.n;  // this warp: t0, t0 + 8, ...
    const unsigned char* src = a.cache + s.b * a.c_sb + kvh * a.c_sh + (int64_t)t0 * kTileBytes + 16 * lane;
    auto fetch = [&](int k, uint32_t slot) {  // tile k, `src` at it
      const uint32_t dst = ring + slot * kTileBytes + 16 * lane;
      const int records = n - k * kTile;
      if (records >= kTile) {
#pragma unroll
        for (int i = 0; i < kTileBytes / 512; ++i) cp_async16(dst + 512 * i, src + 512 * i);
      } else {
#pragma unroll
        for (int i = 0; i < kTileBytes / 512; ++i)
          if (16 * lane + 512 * i < records * kRec) cp_async16(dst + 512 * i, src + 512 * i);
      }
      src += (int64_t)kWarps * kTileBytes;
    };
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) {
      if (t0 + i * kWarps < t1) fetch(t0 + i * kWarps, i);
      cp_async_commit();
    }
    at.begin(a.qk_scale);
    const int whole = n - a.T + 1;  // tokens that every column sees
    int sees[2];                      // tokens that the lane's columns see
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      int hh, tt;
      split(at.acc_col(j), hh, tt);
      sees[j] = whole + tt;
    }
    uint32_t slot = 0;
    for (int k = t0; k < t1; k += kWarps) {
      cp_async_wait<kStages - 2>();
      __syncwarp();
      if ((k + 1) * kTile <= whole) {
        const int none[2] = {kTile, kTile};
        at.template tile<false>(ring + slot * kTileBytes, none);
      } else {
        const int lim[2] = {max(0, min(kTile, sees[0] - k * kTile)), max(0, min(kTile, sees[1] - k * kTile))};
        at.template tile<true>(ring + slot * kTileBytes, lim);
      }
      __syncwarp();
      if (k + (kStages - 1) * kWarps < t1) fetch(k + (kStages - 1) * kWarps, slot == 0 ? kStages - 1 : slot - 1);
      cp_async_commit();
      slot = slot + 1 == kStages ? 0 : slot + 1;
    }
    cp_async_wait<0>();

    // ---- merge the 8 warps: warp c takes column c, a lane four dims
    const bool begins = s.tile == 0, alone = begins && s.share == s.tiles;
    __syncthreads();  // every warp is done with its ring
    at.finish(s_part + warp * kPartFloats, s_part + warp * kPartFloats + kCols * kD, ncol);
    __syncthreads();
    int hh, tt;
    split(warp, hh, tt);
    const int64_t o_at = s.b * a.o.sb + (int64_t)(kvh * G + hh) * a.o.sh + tt * a.o.st;
    if (warp < ncol) {
      float f[kWarps], M = -INFINITY, L = 0.f;
#pragma unroll
      for (int v = 0; v < kWarps; ++v) {
        f[v] = s_part[v * kPartFloats + kCols * kD + 2 * warp];
        M = fmaxf(M, f[v]);
      }
      const float base_m = biased(M);
      float4 A = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int v = 0; v < kWarps; ++v) {
        const float e = ex2(f[v] - base_m);
        L = fmaf(e, s_part[v * kPartFloats + kCols * kD + 2 * warp + 1], L);
        axpy(A, e, reinterpret_cast<const float4*>(s_part + v * kPartFloats)[32 * warp + lane]);
      }
      if (alone) {
        store_out4(const_cast<void*>(a.o.p), a.out_f32, o_at, lane, A, L);
      } else {
        float* part = w.parts + (2 * cta + (begins ? 1 : 0)) * (int64_t)kPartFloats;
        reinterpret_cast<float4*>(part)[32 * warp + lane] = A;
        if (lane == 0) *reinterpret_cast<float2*>(part + kCols * kD + 2 * warp) = make_float2(M, L);
      }
    }
    if (!alone) {
      unsigned first = s.first, parts = s.parts;
      if (!s.own) {  // the CTAs of the row's first and last tile
        const unsigned u = s.line - s.off + kRowUnits;
        first = cta_of(s, u);
        parts = cta_of(s, u + s.tiles - 1) - first + 1;
      }
      unsigned* ticket = w.tickets + s.b * w.per_req + s.r;
      __threadfence();
      __syncthreads();
      if (tid == 0) s_last = atomicAdd(ticket, 1u) == parts - 1 ? 1u : 0u;
      __syncthreads();
      if (s_last) {
        __threadfence();
        merge_parts<PAIR ? 6 : 4>(w.parts + (2 * first + 1) * (int64_t)kPartFloats, (int)parts, ncol, s_part,
                                  const_cast<void*>(a.o.p), a.out_f32, o_at);
        if (tid == 0) *ticket = 0u;
      }
    }
    if (s.own) return;
    __syncthreads();
    if (tid == 0) s_last = dense_next(a, w, s) ? 1u : 0u;
    __syncthreads();  // s_part is the ring again
    if (!s_last) return;
  }
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

size_t ticket_bytes(int64_t rows) { return ((size_t)rows * sizeof(unsigned) + 255) & ~size_t(255); }

bool rows_ok(const Rows& r, int esize) {
  const int64_t q = 16 / esize;
  return oa_aligned16(r.p) && r.sb % q == 0 && r.sh % q == 0 && r.st % q == 0;
}

}  // namespace
}  // namespace oa

extern "C" size_t oa_kv4_attention_workspace_bytes(int64_t B, int64_t HQ, int64_t HKV, int64_t T, int64_t Lmax) {
  if (B <= 0 || T <= 0 || HKV <= 0 || HQ < HKV || Lmax < 0) return 0;
  const oa::DensePlan p = oa::dense_plan(B, HQ, HKV, T, Lmax);
  return oa::ticket_bytes(p.rows) + (size_t)p.grid * 2 * oa::kPartFloats * sizeof(float);
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
  OA_REQUIRE(B <= 0x7fffffff && T <= 0x7fffffff && HQ <= 0x7fffffff && HQ * T <= 0x7fffffff / std::max<int64_t>(B, 1) && Lmax <= 0x7fffffff - 64, "%s: too many rows or positions", fn);
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
  const oa::DensePlan p = oa::dense_plan(B, HQ, HKV, T, Lmax);
  // units on the line (and 9 of them per row of the grid's widest product) are counted in 32 bits
  const int64_t most_units = p.rows * ((Lmax + oa::kTile - 1) / oa::kTile + 1 + oa::kRowUnits);
  OA_REQUIRE(most_units <= 0xffffffffll / 9 && most_units / std::max<int64_t>(p.rows, 1) * 8 * p.grid <= 0xffffffffll,
             "%s: too many records (B * HKV * Lmax) for one call", fn);
  const size_t need = oa::ticket_bytes(p.rows) + (size_t)p.grid * 2 * oa::kPartFloats * sizeof(float);
  OA_REQUIRE(workspace && workspace_bytes >= need && oa_aligned16(workspace),
             "%s: needs a 16-byte aligned workspace of %zu bytes (got %zu)", fn, need, workspace_bytes);
  oa::DenseWork w;
  w.blocks = p.blocks;
  w.per_req = (unsigned)(HKV * p.blocks);
  w.rows = (unsigned)p.rows;
  w.cpr = (unsigned)(p.grid / p.rows);
  w.tickets = static_cast<unsigned*>(workspace);
  w.parts = reinterpret_cast<float*>(static_cast<char*>(workspace) + oa::ticket_bytes(p.rows));
  const auto kernel = HQ / HKV * T <= 4 ? &oa::dense_kernel<true> : &oa::dense_kernel<false>;
  const int rc = oa_smem_opt_in(reinterpret_cast<const void*>(kernel), oa::kRingBytes, fn, true);
  if (rc != OA_OK) return rc;
  kernel<<<(unsigned)p.grid, oa::kDenseThreads, oa::kRingBytes, static_cast<cudaStream_t>(stream)>>>(a, w);
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
