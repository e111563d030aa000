// Attention over the 4-bit K/V cache (record layout: oa_kv4.cuh).
//
//   z_t = sm_scale * q . K_t,   o = sum_t softmax(z)_t V_t,   K_t[d] = scale * code + offset (V alike)
//
// kv4_attention: every position below the request's length; query token i of T (at position n - T + i) sees
// positions <= n - T + i.  kv4_flash: index lists and cluster proxies (as OpenAttention.flash).  Rows with
// nothing to attend give zeros.
#include "oa_kv4_mma.cuh"

namespace oa {
namespace {

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

__device__ __forceinline__ void store_list(const ListArgs& a, int64_t r, int d, float A, float L) {
  const float o = L == 0.f ? 0.f : A / L;
  if (a.out_f32)
    static_cast<float*>(a.out)[r * a.out_stride + d] = o;
  else
    static_cast<__nv_bfloat16*>(a.out)[r * a.out_stride + d] = __float2bfloat16_rn(o);
}

// ---------------------------------------------------------------- dense
// Work: a row is (request, KV head, block of up to 8 query columns); its tiles of 32 records are spread over
// CTAs of 8 warps, each warp with its own ring of kStages tiles filled by asynchronous copies (the 4608 bytes
// of a tile are contiguous).  Lengths live on the device, so each CTA finds its share itself:
//  - each row its own CTAs, grid / rows of them (no more than one per 8 tiles), where that balances;
//  - many short rows: a warp each, nothing to merge;
//  - else the tiles of all rows in one line, cut into equal parts; a CTA then ends one row and begins the next.
// A row that one CTA covers is written by it.  Otherwise each part leaves (m, l, O) in the workspace and the
// last CTA to arrive (atomic ticket, no waiting) merges the parts in CTA order, so the result does not depend
// on which CTA is last.
// What bounds it: memory, once rows are long.  32 requests x 32768 tokens, 32 heads over 8: 188 us, 6.4 TB/s of records
// (98% of a copy's rate), and 212-232 us in long runs, which the power limit slows.  The line reaches that where 256
// rows with a CTA each take 207 us; the 8-column tile takes 222 us there.  Two query tokens (8 columns): 8 requests x
// 32768, 65 us, floor 46, with issue active 45% of the time; the first stall is instruction fetch (the tile stands
// four times in the kernel: masked and not, for single warps and for CTAs).  One request x 32768: 15 us, floor 6: a
// launch, the first loads and the merge through global memory.  64 requests of 1 to 8191 tokens, two query tokens: 62
// us, floor 38: what rows cost besides their tiles.
constexpr int kWarps = 8;
constexpr int kDenseThreads = 32 * kWarps;
constexpr int kStages = 3;
constexpr int kCols = 8;
// What a row costs a CTA besides its tiles (query, merge, idle pipeline), in tiles of four columns and of eight.  64
// ragged requests with two query tokens take 114, 83, 70 us with 6, 12, 20; over 24 uneven batches 20 to 23 are best for
// four columns, 27 for eight (2% quicker than 20).
constexpr int kRowUnits4 = 20, kRowUnits8 = 27;
constexpr int kLineUnits = 35;  // what a second row costs a CTA of the line, in tiles
constexpr int kPartFloats = kCols * kD + 2 * kCols;  // one part: O of 8 columns, then their (m, l)
constexpr int kRingBytes = kWarps * kStages * kTileBytes;

struct DensePlan {
  int blocks;    // column blocks of a KV head: ceil(G T / 8)
  int64_t rows;  // B * HKV * blocks
  int grid, most_parts;  // most_parts: two for each CTA of the largest grid
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
  p.most_parts = 4 * sms;
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
// the lowest n bits (none for n <= 0, all for n >= 32)
__device__ __forceinline__ uint32_t first_bits(int n) { return n >= 32 ? ~0u : n <= 0 ? 0u : (1u << n) - 1u; }
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
// Inlined, and kAhead no larger: a call, or more loads held, spills more than the caller's main loop spills as it is (4
// bytes with four columns, 72 with eight).
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

__device__ __forceinline__ unsigned take_ticket(unsigned* p) {
  unsigned v;
  asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;" : "=r"(v) : "l"(p) : "memory");
  return v;
}

// A CTA's way along the line of rows: the row it is at and its tiles of that row.  Counts of units fit 31 bits
// (checked by the host).
struct DenseShare {
  bool by_warp;           // rows go to single warps: nothing below is set
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
template <int kRowUnits>
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
  // Many short rows: a warp each, if that is quicker.  In units (a CTA's time for a tile when all work, 0.2 us) a warp
  // alone takes 4.4 for a tile and all warps together 1.2 for a CTA's worth, a further round 10; the line its share and
  // some 10 more.  (128 requests of 600 tokens: 22.7 us by warps, 33.1 on the line; 64 of 1000: 33.0 and 27.0.)
  const float warps = (float)(grid * kWarps), work = (float)w.rows * (float)most, rounds = ceilf((float)w.rows / warps);
  s.by_warp = w.cpr == 0 && most < (1 << 16) &&
              fmaxf(1.2f * work, 4.4f * rounds * (float)(most * grid)) + 10.f * (rounds - 2.f) * (float)grid < (float)total;
  if (s.by_warp) return true;
  // (32 requests of 1000 tokens: 13.4 us with their own CTAs, 18.5 on the line; 24 of 2000: 20.5 and 23.4; 16 of 32768:
  // 110 and 101)
  s.own = w.cpr >= 1 && (kRowUnits + (most + w.cpr - 1) / w.cpr) * grid <= total + kLineUnits * grid;
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
template <int kRowUnits>
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

// Rows of a few tiles: each warp takes whole rows, and nothing is merged.
template <bool QUAD>
__device__ __forceinline__ void dense_by_warp(const DenseArgs& a, const DenseWork& w, uint32_t ring) {
  constexpr int J = WarpAttention<QUAD>::J;
  const int lane = threadIdx.x & 31, G = a.HQ / a.HKV, cols = G * a.T;
  WarpAttention<QUAD> at;
  at.lane_addresses();
  for (unsigned row = blockIdx.x + (threadIdx.x >> 5) * gridDim.x; row < w.rows; row += gridDim.x * kWarps) {
    const unsigned b = row / w.per_req, r = row - b * w.per_req;
    const int kvh = r / w.blocks, col0 = (r - kvh * w.blocks) * kCols, ncol = min(kCols, cols - col0);
    const int n = dense_len(a, b), tiles = dense_tiles(n), whole = n - a.T + 1;
    const unsigned char* src = a.cache + b * a.c_sb + kvh * a.c_sh + 16 * lane;
    auto fetch = [&](int k, uint32_t slot) {
#pragma unroll
      for (int i = 0; i < kTileBytes / 512; ++i)
        if (16 * lane + 512 * i < (n - k * kTile) * kRec) cp_async16(ring + slot * kTileBytes + 16 * lane + 512 * i, src + 512 * i);
      src += kTileBytes;
    };
    auto split = [&](int c, int& hh, int& tt) {
      hh = a.T == 1 ? col0 + c : (col0 + c) / a.T;
      tt = col0 + c - hh * a.T;
    };
    int hh, tt;
    split(at.op_col(), hh, tt);
    at.load_q(at.op_col() < ncol ? static_cast<const __nv_bfloat16*>(a.q.p) + b * a.q.sb + (int64_t)(kvh * G + hh) * a.q.sh + tt * a.q.st
                                 : nullptr);
    __syncwarp();  // the last row's tiles are read
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) {
      if (i < tiles) fetch(i, i);
      cp_async_commit();
    }
    at.begin(a.qk_scale);
    int sees[J];
#pragma unroll
    for (int j = 0; j < J; ++j) {
      split(at.col(j), hh, tt);
      sees[j] = whole + tt;
    }
    uint32_t slot = 0;
    for (int k = 0; k < tiles; ++k) {
      cp_async_wait<kStages - 2>();
      __syncwarp();
      uint32_t in[J];
#pragma unroll
      for (int j = 0; j < J; ++j) in[j] = first_bits(sees[j] - k * kTile);
      if ((k + 1) * kTile <= whole)
        at.template tile<false>(ring + slot * kTileBytes, in);
      else
        at.template tile<true>(ring + slot * kTileBytes, in);
      __syncwarp();
      if (k + kStages - 1 < tiles) fetch(k + kStages - 1, slot == 0 ? kStages - 1 : slot - 1);
      cp_async_commit();
      slot = slot + 1 == kStages ? 0 : slot + 1;
    }
    at.add_up();
#pragma unroll
    for (int j = 0; j < J; ++j) {
      if (at.col(j) >= ncol) continue;
      split(at.col(j), hh, tt);
      const int64_t o_at = b * a.o.sb + (int64_t)(kvh * G + hh) * a.o.sh + tt * a.o.st + 8 * (lane >> 2);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float o[8];
        at.dims(j, h, o);
        store_out4(const_cast<void*>(a.o.p), a.out_f32, o_at + 64 * h, 0, make_float4(o[0], o[1], o[2], o[3]), at.l[j]);
        store_out4(const_cast<void*>(a.o.p), a.out_f32, o_at + 64 * h + 4, 0, make_float4(o[4], o[5], o[6], o[7]), at.l[j]);
      }
    }
  }
  cp_async_wait<0>();
}

template <bool QUAD>
__global__ void __launch_bounds__(kDenseThreads, 2) dense_kernel(const DenseArgs a, const DenseWork w) {
  extern __shared__ __align__(16) unsigned char s_ring[];
  constexpr int kRowUnits = QUAD ? kRowUnits4 : kRowUnits8;
  __shared__ unsigned s_last;
  __shared__ DenseShare s;  // the same for all threads: kept here, out of the loop's registers
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int G = a.HQ / a.HKV, cols = G * a.T;
  const unsigned cta = blockIdx.x;
  {
    DenseShare mine;
    if (!dense_share<kRowUnits>(a, w, mine)) return;
    if (mine.by_warp) {
      dense_by_warp<QUAD>(a, w, smem_u32(s_ring) + warp * (kStages * kTileBytes));
      return;
    }
    if (tid == 0) s = mine;
  }
  __syncthreads();

  const uint32_t ring = smem_u32(s_ring) + warp * (kStages * kTileBytes);
  float* s_part = reinterpret_cast<float*>(s_ring);  // reused once a row's tiles are done
  WarpAttention<QUAD> at;
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
    constexpr int J = WarpAttention<QUAD>::J;
    int sees[J];                      // tokens that the lane's columns see
#pragma unroll
    for (int j = 0; j < J; ++j) {
      int hh, tt;
      split(at.col(j), hh, tt);
      sees[j] = whole + tt;
    }
    uint32_t slot = 0;
    for (int k = t0; k < t1; k += kWarps) {
      cp_async_wait<kStages - 2>();
      __syncwarp();
      if ((k + 1) * kTile <= whole) {
        const uint32_t all[J] = {};
        at.template tile<false>(ring + slot * kTileBytes, all);
      } else {
        uint32_t in[J];
#pragma unroll
        for (int j = 0; j < J; ++j) in[j] = first_bits(sees[j] - k * kTile);
        at.template tile<true>(ring + slot * kTileBytes, in);
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
      float4 A = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int v = 0; v < kWarps; ++v) {
        const float e = ex2(f[v] - M);
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
      // the barrier orders the CTA's stores before thread 0's release, and its acquire before the CTA's loads
      __syncthreads();
      if (tid == 0) s_last = take_ticket(ticket) == parts - 1 ? 1u : 0u;
      __syncthreads();
      if (s_last) {
        merge_parts<QUAD ? 6 : 4>(w.parts + (2 * first + 1) * (int64_t)kPartFloats, (int)parts, ncol, s_part,
                                  const_cast<void*>(a.o.p), a.out_f32, o_at);
        if (tid == 0) *ticket = 0u;
      }
    }
    if (s.own) return;
    __syncthreads();
    if (tid == 0) s_last = dense_next<kRowUnits>(a, w, s) ? 1u : 0u;
    __syncthreads();  // s_part is the ring again
    if (!s_last) return;
  }
}

// ---------------------------------------------------------------- index lists and proxies
// A row's work is a line of items of about 4 KB: its entries (sel, then exp) in tiles of 32 records, then its proxies
// in tiles of 8 bf16 row pairs.  The W warps of a CTA or, where rows are few, of a cluster of CTAs take them in
// turn, each with a ring of three: asynchronous copies fetch two items ahead (records three to an instruction,
// nine 16-byte chunks each), the indices and log counts of a third are asked for.  Padding entries and skipped
// proxies are masked by a bit and not fetched.  A list belongs to one query row: one of the MMA's query columns is
// used, which is still less work than unpacking codes to fp32 for plain FMAs (a tile of 32 takes some 350
// instructions, against about 770 on the same pipes).  The warps' states are merged in shared memory, then over the
// cluster.  1024 rows of 231 entries and 64 proxies: 24.6 us for 63 MB.  Latency bounds that (a launch, indices, then records:
// DRAM at 46%, issue at 42%); longer lists add 3.75 TB/s of records, which is 5 TB/s of DRAM accesses: a scattered record
// of 144 bytes takes three or four of 64.
constexpr int kRowsPerTile = 8;

__device__ __forceinline__ uint32_t cluster_addr(const void* p, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_u32(p)), "r"(rank));
  return r;
}
__device__ __forceinline__ float ld_cluster(uint32_t at) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

template <int W>
constexpr size_t list_smem() { return (size_t)W * kStages * kTileBytes; }
// Only CTAs of 8 warps form clusters, and leave their state where the others can read it.  What the rule for W counts on,
// 16 warps on an SM (of 228 KB, 1 KB of it taken for each CTA), leaves two warps' CTAs no room for that.
template <int W>
constexpr int kClusterFloats = W == 8 ? kD + 2 : 1;
template <int W>
constexpr bool kSixteenWarps = 16 / W * (list_smem<W>() + kClusterFloats<W> * sizeof(float) + 1024) <= 228 * 1024;
static_assert(kSixteenWarps<2> && kSixteenWarps<4> && kSixteenWarps<8>, "16 warps of list_kernel must fit an SM's shared memory");

template <int W>
__global__ void __launch_bounds__(32 * W, 16 / W) list_kernel(const ListArgs a, int S) {  // S: CTAs of a row (W < 8: one)
  extern __shared__ __align__(16) unsigned char s_dyn[];  // [warp][stage][item]; a warp's state when it is done
  __shared__ float s_cta[kClusterFloats<W>];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (W < 8) S = 1;
  const int rank = S > 1 ? blockIdx.x % S : 0;
  const int64_t r = blockIdx.x / S, kvh = r / a.G;
  const int nw = W * S, total = a.n_sel + a.n_exp;
  const int tiles = (total + kTile - 1) / kTile, items = tiles + (a.NB + kRowsPerTile - 1) / kRowsPerTile;
  const uint32_t ring = smem_u32(s_dyn) + warp * (kStages * kTileBytes);

  // what an item's copies wait for: the lane's index (-1: none), or its proxy's log count (-inf: none)
  auto ask = [&](int j) {
    int v = -1;
    if (j < tiles) {
      const int e = j * kTile + lane;
      if (e < total) v = e < a.n_sel ? a.sel[r * a.n_sel + e] : a.exp[r * a.n_exp + (e - a.n_sel)];
    } else if (j < items) {
      const int e = (j - tiles) * kRowsPerTile + lane;
      v = __float_as_int(lane < kRowsPerTile && e < a.NB ? a.logn[r * a.ln_stride + e] : -INFINITY);
    }
    return v;
  };
  const int third = lane / 9;  // lanes 27..31 have no part in a record
  const unsigned char* rec = a.cache + kvh * a.c_sh + 16 * (lane - 9 * third);
  const int64_t prow = (a.per_qhead ? r : kvh) * a.kb_sh + 8 * (lane & 15);
  const unsigned limit = (unsigned)min(a.Lmax, (int64_t)0x7fffffff);
  auto fetch = [&](int j, int v, int stage) {  // starts an item's copies; returns its live entries
    const uint32_t dst = ring + stage * kTileBytes + 16 * lane;
    uint32_t in = 0u;
    if (j < tiles) {
      in = __ballot_sync(0xffffffffu, (unsigned)v < limit);
      const uint32_t mine = third < 3 ? in >> third : 0u;  // bit 3 i: entry 3 i + third
#pragma unroll
      for (int i = 0; i < 11; ++i) {
        const int at = __shfl_sync(0xffffffffu, v, third + 3 * i);
        if (mine >> (3 * i) & 1u) cp_async16(dst + 3 * i * kRec, rec + (int64_t)at * kRec);
      }
    } else if (j < items) {
      in = __ballot_sync(0xffffffffu, !(__int_as_float(v) == -INFINITY));
      const int e0 = (j - tiles) * kRowsPerTile;
#pragma unroll
      for (int i = 0; i < kRowsPerTile; i += 2) {
        const int e = i + (lane >> 4);
        const bool live = in >> e & 1u;
        const int64_t at = live ? prow + (int64_t)(e0 + e) * a.kb_sb : prow;
        const uint32_t to = ring + stage * kTileBytes + e * 256 + (((lane & 15) ^ e) << 4);
        cp_async16_or_zero(to, a.kbar + at, live);
        cp_async16_or_zero(to + 2048, a.vbar + at, live);
      }
    }
    cp_async_commit();
    return in;
  };
  int j = rank * W + warp;
  int v0 = ask(j), v1 = ask(j + nw), v2 = ask(j + 2 * nw);
  WarpAttention<true> at;
  at.lane_addresses();
  at.load_q(at.op_col() == 0 ? a.q + r * a.q_stride : nullptr);
  uint32_t in0 = fetch(j, v0, 0), in1 = fetch(j + nw, v1, 1);
  at.begin(a.qk_scale);
  bool rows = false;
  for (int stage = 0; j < items; j += nw) {
    const int before = stage == 0 ? kStages - 1 : stage - 1;
    const uint32_t in2 = fetch(j + 2 * nw, v2, before);
    const int v3 = ask(j + 3 * nw);
    cp_async_wait<kStages - 1>();
    __syncwarp();
    const uint32_t sm = ring + stage * kTileBytes;
    if (j < tiles) {
      const uint32_t sees[1] = {in0};
      if (in0 == ~0u)
        at.template tile<false>(sm, sees);
      else if (in0)
        at.template tile<true>(sm, sees);
    } else {
      if (!rows) at.begin_rows(a.q + r * a.q_stride);
      rows = true;
      if (in0) at.rows(sm, in0, __int_as_float(v0) * kLog2e, a.qk_scale);
    }
    __syncwarp();
    in0 = in1;
    in1 = in2;
    v0 = v1;
    v1 = v2;
    v2 = v3;
    stage = stage + 1 == kStages ? 0 : stage + 1;
  }
  cp_async_wait<0>();
  __syncwarp();
  if (rows) at.end_rows();
  {
    float* state = reinterpret_cast<float*>(s_dyn + warp * (kStages * kTileBytes));
    at.finish(state, state + kD, 1);
  }
  __syncthreads();

  // ---- merge the CTA's states, then the cluster's
  const float* st = reinterpret_cast<const float*>(s_dyn);
  constexpr int kNext = kStages * kTileBytes / 4;  // floats from one warp's state to the next
  float M = -INFINITY, L = 0.f, f[W];
#pragma unroll
  for (int i = 0; i < W; ++i) M = fmaxf(M, st[i * kNext + kD]);
#pragma unroll
  for (int i = 0; i < W; ++i) {
    f[i] = ex2(st[i * kNext + kD] - M);
    L = fmaf(f[i], st[i * kNext + kD + 1], L);
  }
  for (int d = tid; d < kD; d += 32 * W) {
    float A = 0.f;
#pragma unroll
    for (int i = 0; i < W; ++i) A = fmaf(f[i], st[i * kNext + d], A);
    if constexpr (W == 8) {
      if (S > 1) {
        s_cta[d] = A;
        continue;
      }
    }
    store_list(a, r, d, A, L);
  }
  if constexpr (W == 8) {
    if (S == 1) return;
    if (tid == 0) {
      s_cta[kD] = M;
      s_cta[kD + 1] = L;
    }
    cluster_sync();
    if (rank == 0) {
      M = -INFINITY;
      for (int k = 0; k < S; ++k) M = fmaxf(M, ld_cluster(cluster_addr(s_cta + kD, k)));
      L = 0.f;
      for (int k = 0; k < S; ++k)
        L = fmaf(ex2(ld_cluster(cluster_addr(s_cta + kD, k)) - M), ld_cluster(cluster_addr(s_cta + kD + 1, k)), L);
      for (int d = tid; d < kD; d += 32 * W) {
        float A = 0.f;
        for (int k = 0; k < S; ++k)
          A = fmaf(ex2(ld_cluster(cluster_addr(s_cta + kD, k)) - M), ld_cluster(cluster_addr(s_cta + d, k)), A);
        store_list(a, r, d, A, L);
      }
    }
    cluster_sync();  // no CTA leaves while its state is read
  }
}

template <int W>
int launch_list(const ListArgs& a, int64_t rows, int S, const char* fn, cudaStream_t st) {
  const int rc = oa_smem_opt_in(reinterpret_cast<const void*>(&list_kernel<W>), list_smem<W>(), fn, true);
  if (rc != OA_OK) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(rows * S));
  cfg.blockDim = dim3(32 * W);
  cfg.dynamicSmemBytes = list_smem<W>();
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = (unsigned)S;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = S > 1 ? 1 : 0;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, &list_kernel<W>, a, S);
  if (e != cudaSuccess) return oa_fail(OA_ERR_CUDA, "%s: %s", fn, cudaGetErrorString(e));
  return oa_check_launch(fn);
}

// A workspace: the parts of the largest grid, then a ticket per row.  Where the tickets lie does not depend on the
// call, so calls of any sizes can share a workspace that is large enough for each.
size_t workspace_bytes(const DensePlan& p) { return (size_t)p.most_parts * kPartFloats * sizeof(float) + (size_t)p.rows * sizeof(unsigned); }

}  // namespace
}  // namespace oa

extern "C" size_t oa_kv4_attention_workspace_bytes(int64_t B, int64_t HQ, int64_t HKV, int64_t T, int64_t Lmax) {
  if (B <= 0 || T <= 0 || HKV <= 0 || HQ < HKV || Lmax < 0) return 0;
  const oa::DensePlan p = oa::dense_plan(B, HQ, HKV, T, Lmax);
  return oa::workspace_bytes(p);
}

extern "C" int oa_kv4_attention(const oa_kv4_attention_args* args, void* stream) {
  const char* fn = "oa_kv4_attention";
  OA_REQUIRE(args != nullptr, "%s: null arguments", fn);
  const oa_kv4_attention_args& g = *args;
  OA_REQUIRE(g.out_dtype == OA_BF16 || g.out_dtype == OA_F32, "%s: out_dtype must be OA_BF16 or OA_F32", fn);
  oa::DenseArgs a;
  const int64_t B = g.q.size[0], HQ = g.q.size[1], T = g.q.size[2], HKV = g.cache.size[1], Lmax = g.cache.size[2];
  OA_TRY(oa_take_cache(fn, g.cache, false, &a.cache, &a.c_sb, &a.c_sh));
  OA_REQUIRE(g.cache.size[0] == B && HKV >= 1 && HQ >= HKV && HQ % HKV == 0,
             "%s: q holds %lld requests of %lld heads, the cache %lld of %lld: need the same requests and a multiple of the KV "
             "heads",
             fn, (long long)B, (long long)HQ, (long long)g.cache.size[0], (long long)HKV);
  OA_TRY(oa_take_rows(fn, "q", g.q, 2, B, HQ, T, false, &a.q));
  OA_TRY(oa_take_rows(fn, "out", g.out, g.out_dtype == OA_F32 ? 4 : 2, B, HQ, T, true, &a.o));
  OA_TRY(oa_take_index(fn, "n", g.n, B, true, &a.n));
  if (B == 0 || T == 0) return OA_OK;
  OA_REQUIRE(HQ * T <= 0x7fffffff / B, "%s: too many rows", fn);
  a.Lmax = Lmax;
  a.offset = g.offset;
  a.out_f32 = g.out_dtype == OA_F32;
  a.B = (int)B; a.HQ = (int)HQ; a.HKV = (int)HKV; a.T = (int)T;
  a.qk_scale = (float)(g.sm_scale * (double)oa::kLog2e);
  void* const workspace = g.workspace;
  const size_t workspace_bytes = (size_t)std::max<int64_t>(g.workspace_bytes, 0);
  const oa::DensePlan p = oa::dense_plan(B, HQ, HKV, T, Lmax);
  // units on the line (and 9 of them per row of the grid's widest product) are counted in 32 bits
  const int64_t most_units = p.rows * ((Lmax + oa::kTile - 1) / oa::kTile + 1 + oa::kRowUnits8);
  OA_REQUIRE(most_units <= 0xffffffffll / 9 && most_units / std::max<int64_t>(p.rows, 1) * 8 * p.grid <= 0xffffffffll,
             "%s: too many records (B * HKV * Lmax) for one call", fn);
  const size_t need = oa::workspace_bytes(p);
  OA_REQUIRE(workspace && workspace_bytes >= need && oa_aligned16(workspace),
             "%s: needs a 16-byte aligned workspace of %zu bytes (got %zu)", fn, need, workspace_bytes);
  oa::DenseWork w;
  w.blocks = p.blocks;
  w.per_req = (unsigned)(HKV * p.blocks);
  w.rows = (unsigned)p.rows;
  w.cpr = (unsigned)(p.grid / p.rows);
  w.parts = static_cast<float*>(workspace);
  w.tickets = reinterpret_cast<unsigned*>(w.parts + (size_t)p.most_parts * oa::kPartFloats);
  // up to four queries of a KV head fit the tile that holds each one's halves side by side (oa_kv4_mma.cuh)
  const auto kernel = HQ / HKV * T <= 4 ? &oa::dense_kernel<true> : &oa::dense_kernel<false>;
  const int rc = oa_smem_opt_in(reinterpret_cast<const void*>(kernel), oa::kRingBytes, fn, true);
  if (rc != OA_OK) return rc;
  kernel<<<(unsigned)p.grid, oa::kDenseThreads, oa::kRingBytes, static_cast<cudaStream_t>(stream)>>>(a, w);
  return oa_check_launch(fn);
}

extern "C" int oa_kv4_flash(const oa_kv4_flash_args* args, void* stream) {
  const char* fn = "oa_kv4_flash";
  OA_REQUIRE(args != nullptr, "%s: null arguments", fn);
  const oa_kv4_flash_args& g = *args;
  const int64_t BQ = g.q.size[0], BH = g.cache.size[0], NB = g.NB;
  OA_REQUIRE(g.out_dtype == OA_BF16 || g.out_dtype == OA_F32, "%s: out_dtype must be OA_BF16 or OA_F32", fn);
  OA_REQUIRE(BQ >= 0 && BQ <= 0x7fffffff && BH >= 1 && BQ % BH == 0, "%s: q's %lld rows must be a multiple of the cache's %lld",
             fn, (long long)BQ, (long long)BH);
  const oa_tensor4 c4 = {g.cache.p, {1, BH, g.cache.size[1], g.cache.size[2]}, {0, g.cache.stride[0], g.cache.stride[1], g.cache.stride[2]}};
  oa::ListArgs a;
  int64_t none;
  OA_TRY(oa_take_cache(fn, c4, false, &a.cache, &none, &a.c_sh));
  OA_REQUIRE(g.q.size[1] == oa::kD && g.out.size[0] == BQ && g.out.size[1] == oa::kD, "%s: q and out must be (%lld, 128)", fn,
             (long long)BQ);
  OA_REQUIRE(g.sel.size[0] == BQ && g.exp_idx.size[0] == BQ, "%s: sel_idx and exp_idx must have %lld rows", fn, (long long)BQ);
  const int64_t n_sel = g.sel.size[1], n_exp = g.exp_idx.size[1];
  OA_REQUIRE(NB >= 0 && n_sel >= 0 && n_exp >= 0 && n_sel + n_exp + NB < (int64_t)1 << 30, "%s: bad list sizes", fn);
  if (BQ == 0) return OA_OK;
  OA_REQUIRE(g.q.p && g.out.p && g.q.stride[1] == 1 && g.out.stride[1] == 1, "%s: q and out must have a contiguous last dim", fn);
  const int es = g.out_dtype == OA_F32 ? 4 : 2;
  a.q_stride = BQ > 1 ? g.q.stride[0] : 0;
  a.out_stride = BQ > 1 ? g.out.stride[0] : 0;
  OA_REQUIRE(BQ <= 1 || a.out_stride >= oa::kD || a.out_stride <= -oa::kD, "%s: out's rows overlap", fn);
  OA_REQUIRE(oa_aligned16(g.q.p) && oa_aligned16(g.out.p) && a.q_stride % 8 == 0 && a.out_stride * es % 16 == 0,
             "%s: q and out rows must start on 16-byte boundaries (base addresses and strides)", fn);
  OA_REQUIRE((n_sel == 0 || (g.sel.p && g.sel.stride[1] == 1 && (BQ == 1 || g.sel.stride[0] == n_sel))) &&
                 (n_exp == 0 || (g.exp_idx.p && g.exp_idx.stride[1] == 1 && (BQ == 1 || g.exp_idx.stride[0] == n_exp))),
             "%s: sel_idx and exp_idx must be contiguous", fn);
  a.kbar = a.vbar = nullptr;
  a.kb_sh = a.kb_sb = a.ln_stride = 0;
  a.logn = nullptr;
  a.per_qhead = 1;
  if (NB > 0) {
    bool same = true;
    for (int i = 0; i < 3; ++i) same = same && g.kbar.size[i] == g.vbar.size[i] && g.kbar.stride[i] == g.vbar.stride[i];
    OA_REQUIRE(same && (g.kbar.size[0] == BQ || g.kbar.size[0] == BH) && g.kbar.size[1] >= NB && g.kbar.size[2] == oa::kD &&
                   g.kbar.stride[2] == 1,
               "%s: kbar and vbar must be (%lld or %lld, >= %lld, 128) of one shape and strides with a contiguous last dim", fn,
               (long long)BQ, (long long)BH, (long long)NB);
    OA_REQUIRE(g.log_n.size[0] == BQ && g.log_n.size[1] >= NB && g.log_n.stride[1] == 1,
               "%s: log_n must be (%lld, >= %lld) with a contiguous last dim", fn, (long long)BQ, (long long)NB);
    OA_REQUIRE(g.kbar.p && g.vbar.p && g.log_n.p, "%s: null kbar/vbar/log_n with NB > 0", fn);
    a.kb_sh = g.kbar.size[0] > 1 ? g.kbar.stride[0] : 0;
    a.kb_sb = g.kbar.size[1] > 1 ? g.kbar.stride[1] : 0;
    OA_REQUIRE(oa_aligned16(g.kbar.p) && oa_aligned16(g.vbar.p) && a.kb_sh % 8 == 0 && a.kb_sb % 8 == 0,
               "%s: kbar/vbar rows must start on 16-byte boundaries", fn);
    a.kbar = static_cast<const __nv_bfloat16*>(g.kbar.p);
    a.vbar = static_cast<const __nv_bfloat16*>(g.vbar.p);
    a.per_qhead = g.kbar.size[0] == BQ;
    a.logn = static_cast<const float*>(g.log_n.p);
    a.ln_stride = BQ > 1 ? g.log_n.stride[0] : 0;
  }
  a.q = static_cast<const __nv_bfloat16*>(g.q.p);
  a.Lmax = g.cache.size[1];
  a.sel = static_cast<const int32_t*>(g.sel.p);
  a.exp = static_cast<const int32_t*>(g.exp_idx.p);
  a.n_sel = (int)n_sel; a.n_exp = (int)n_exp; a.NB = (int)NB;
  a.out = const_cast<void*>(g.out.p);
  a.out_f32 = g.out_dtype == OA_F32;
  a.G = (int)(BQ / BH);
  a.qk_scale = (float)(g.sm_scale * (double)oa::kLog2e);
  // Warps per row.  Few rows: clusters of 8-warp CTAs, no more CTAs than SMs and an item for each warp (32 rows of 1350
  // entries and 192 proxies 14.4 us on one CTA each, 10.3 on clusters of 4, 11.2 of 8; 128 rows 16.4, and 18.4 on
  // clusters of 2).  Else as many warps as make up 16 on every SM, with two items each (256 rows of 694 entries: 19.7 us
  // with 8, 20.5 with 4; 1024 rows of 231: 29.1 with 8, 26.5 with 4, 24.6 with 2).
  const int64_t items = (n_sel + n_exp + oa::kTile - 1) / oa::kTile + (NB + oa::kRowsPerTile - 1) / oa::kRowsPerTile;
  int S = 1;
  while (S < 8 && BQ * 2 * S <= 148 && 16 * S <= items) S *= 2;
  const int64_t warps = std::min(148 * 16 / BQ, (items + 1) / 2);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (S > 1 || warps >= 8) return oa::launch_list<8>(a, BQ, S, fn, st);
  if (warps >= 4) return oa::launch_list<4>(a, BQ, 1, fn, st);
  return oa::launch_list<2>(a, BQ, 1, fn, st);
}
