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
