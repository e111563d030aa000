// The 4-bit K/V cache record and the arithmetic on it, shared by the kernels that write, read and
// attend to one.
//
// One record = one token of one KV head, 144 bytes (a multiple of 16, so every record starts on a
// 16-byte boundary and a run of records is one contiguous copy):
//   bytes   0.. 63  K codes: byte j = code of dim j | code of dim j + 64 << 4
//   bytes  64..127  V codes, the same way
//   bytes 128..143  eight bf16: K scale, offset of dims 0..63; K scale, offset of dims 64..127; V the same
// A value is scale * code + offset with code in 0..15.  The offset is the group's minimum (bf16, as the
// stored rows are, so exact); the scale is bf16((max - min) / 15); code = min(rint((x - offset) / scale), 15),
// ties to the even code, 0 where the scale is 0.  A group that holds an infinity or a NaN (or whose
// range is past fp32's) gets a NaN scale.
// The halves as groups: the two dims a rotation mixes (j, j + 64) share a byte, one 16-bit mask separates the
// groups (low nibbles against high nibbles), and 72 bytes per row and side = 4.5 bits per value.
#pragma once
#include "oa_common.cuh"
#include "../../include/openattention_b200.h"

namespace oa {

constexpr int kRec = 144;
constexpr int kRecV = 64;
constexpr int kRecMeta = 128;

// A device array of per-request numbers: int32 or int64, one for all requests (stride 0) or one each.
struct PerRequest {
  const void* p;  // NULL: absent
  int64_t stride;
  int is64;
};
__device__ __forceinline__ int64_t per_request(const PerRequest& a, int64_t b) {
  return a.is64 ? static_cast<const int64_t*>(a.p)[b * a.stride] : (int64_t) static_cast<const int32_t*>(a.p)[b * a.stride];
}

// (B, heads, T, 128) rows with strides in elements; the last dim is contiguous.
struct Rows {
  const void* p;
  int64_t sb, sh, st;
};

}  // namespace oa

// ---------------------------------------------------------------- host: checks of the argument blocks
#define OA_TRY(e)                 \
  do {                            \
    const int rc_ = (e);          \
    if (rc_ != OA_OK) return rc_; \
  } while (0)

// Whether runs of `run` elements, one for each index of dims with these sizes and strides, lie apart.  From the smallest
// stride on, each must step over everything the smaller ones span: so it is for every view that slicing, permuting
// and splitting of dims can make of a dense tensor.
template <int N>
static inline bool oa_apart(const int64_t* size, const int64_t* stride, int64_t run) {
  __int128 step[N], span = run;
  int n = 0, order[N];
  for (int i = 0; i < N; ++i) {
    if (size[i] <= 1) continue;
    step[i] = stride[i] < 0 ? -(__int128)stride[i] : (__int128)stride[i];
    int at = n++;
    for (; at > 0 && step[order[at - 1]] > step[i]; --at) order[at] = order[at - 1];
    order[at] = i;
  }
  for (int i = 0; i < n; ++i) {
    if (step[order[i]] < span) return false;
    span += (size[order[i]] - 1) * step[order[i]];
  }
  return true;
}

// Rows (B, H, T, 128) of element size `esize` into out (strides of single-element dims cleared: any number may
// stand there); H, T < 0: any.  Empty rows have no address.  `writes`: rows must not share memory.
static inline int oa_take_rows(const char* fn, const char* name, const oa_tensor4& t, int esize, int64_t B, int64_t H,
                               int64_t T, bool writes, oa::Rows* out) {
  OA_REQUIRE(t.size[0] == B && (H < 0 || t.size[1] == H) && (T < 0 || t.size[2] == T) && t.size[3] == oa::kD,
             "%s: %s must be (%lld, %lld, %lld, 128) rows, got (%lld, %lld, %lld, %lld)", fn, name, (long long)B,
             (long long)(H < 0 ? t.size[1] : H), (long long)(T < 0 ? t.size[2] : T), (long long)t.size[0],
             (long long)t.size[1], (long long)t.size[2], (long long)t.size[3]);
  OA_REQUIRE(t.size[0] >= 0 && t.size[1] >= 0 && t.size[2] >= 0 && t.size[0] <= 0x7fffffff && t.size[1] <= 0xfffff &&
                 t.size[2] <= 0x7fffffff,
             "%s: %s: bad sizes (%lld, %lld, %lld, 128)", fn, name, (long long)t.size[0], (long long)t.size[1],
             (long long)t.size[2]);
  const bool empty = t.size[0] == 0 || t.size[1] == 0 || t.size[2] == 0;
  OA_REQUIRE(t.p != nullptr || empty, "%s: null %s", fn, name);
  OA_REQUIRE(t.stride[3] == 1 || empty, "%s: %s must have a contiguous last dim", fn, name);
  int64_t st[3];
  for (int i = 0; i < 3; ++i) {
    st[i] = t.size[i] > 1 ? t.stride[i] : 0;
    OA_REQUIRE(st[i] * esize % 16 == 0 || empty, "%s: %s rows must start on 16-byte boundaries (strides)", fn, name);
  }
  OA_REQUIRE(!writes || empty || oa_apart<3>(t.size, st, oa::kD),
             "%s: %s must not be an expanded tensor or one of interleaved strides: its rows would overlap", fn, name);
  OA_REQUIRE(oa_aligned16(t.p), "%s: %s rows must start on 16-byte boundaries (base address)", fn, name);
  *out = oa::Rows{t.p, st[0], st[1], st[2]};
  return OA_OK;
}

static inline int oa_take_index(const char* fn, const char* name, const oa_index& x, int64_t B, bool required,
                                oa::PerRequest* out) {
  OA_REQUIRE(x.p != nullptr || !required || B == 0, "%s: %s must be given", fn, name);
  OA_REQUIRE(x.p == nullptr || x.size == 1 || x.size == B, "%s: %s must hold %lld numbers or one, got %lld", fn, name,
             (long long)B, (long long)x.size);
  *out = oa::PerRequest{x.p, x.size == 1 ? 0 : x.stride, (int)x.is_int64};
  return OA_OK;
}

// A cache (B, HKV, Lmax, 144): its strides in bytes (0 for dims of one element).
static inline int oa_take_cache(const char* fn, const oa_tensor4& t, bool writes, const unsigned char** p, int64_t* sb,
                                int64_t* sh) {
  OA_REQUIRE(t.size[3] == oa::kRec && t.stride[3] == 1 && (t.size[2] <= 1 || t.stride[2] == oa::kRec),
             "%s: the cache must be (B, hkv, Lmax, 144) bytes with contiguous records, got (%lld, %lld, %lld, %lld) with strides "
             "(%lld, %lld, %lld, %lld)",
             fn, (long long)t.size[0], (long long)t.size[1], (long long)t.size[2], (long long)t.size[3],
             (long long)t.stride[0], (long long)t.stride[1], (long long)t.stride[2], (long long)t.stride[3]);
  OA_REQUIRE(t.size[0] >= 0 && t.size[1] >= 0 && t.size[2] >= 0 && t.size[2] <= 0x7fffffff - 64,
             "%s: the cache has bad sizes (%lld, %lld, %lld, 144)", fn, (long long)t.size[0], (long long)t.size[1],
             (long long)t.size[2]);
  const bool empty = t.size[0] == 0 || t.size[1] == 0 || t.size[2] == 0;
  OA_REQUIRE((t.p != nullptr || empty) && oa_aligned16(t.p), "%s: the cache must start on a 16-byte boundary", fn);
  *p = static_cast<const unsigned char*>(t.p);
  *sb = t.size[0] > 1 ? t.stride[0] : 0;
  *sh = t.size[1] > 1 ? t.stride[1] : 0;
  OA_REQUIRE(empty || (*sb % 16 == 0 && *sh % 16 == 0), "%s: cache strides must be multiples of 16 bytes", fn);
  const int64_t st[2] = {*sb, *sh};
  OA_REQUIRE(!writes || empty || oa_apart<2>(t.size, st, t.size[2] * oa::kRec),
             "%s: the cache must not be an expanded tensor or one of interleaved strides: its requests would share records", fn);
  return OA_OK;
}
