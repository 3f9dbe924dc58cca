// The microscaled 4-bit format of the token cache on gfx950: scale bytes, and the
// conversions between e2m1 codes and float16 / float32 values.
#ifndef IAK_MX_FORMAT_H
#define IAK_MX_FORMAT_H

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "iak_device.h"

namespace iak {

constexpr int MX_BLOCK = 32;                   // channels per scale
constexpr uint32_t MX_SCALE_NAN = 255u;        // e8m0 NaN
constexpr int MX_E_MIN = -23, MX_E_MAX = 13;   // every value code * 2^e is a float16 number
constexpr uint32_t MX_BYTE_MIN = 127 + MX_E_MIN, MX_BYTE_MAX = 127 + MX_E_MAX;

// 2^(clamp(byte, 104, 140) - 127) as a float: finite for every byte
__device__ __forceinline__ float mx_scale(uint32_t byte) {
  const uint32_t b = byte < MX_BYTE_MIN ? MX_BYTE_MIN : (byte > MX_BYTE_MAX ? MX_BYTE_MAX : byte);
  return u2f(b << 23);
}

// Eight e2m1 codes times a scale -> four f16 pairs, exactly (the format's range).
__device__ __forceinline__ void mx8_to_f16(uint32_t x, float s, uint32_t o[4]) {
  o[0] = bits(__builtin_amdgcn_cvt_scalef32_pk_f16_fp4(x, s, 0));
  o[1] = bits(__builtin_amdgcn_cvt_scalef32_pk_f16_fp4(x, s, 1));
  o[2] = bits(__builtin_amdgcn_cvt_scalef32_pk_f16_fp4(x, s, 2));
  o[3] = bits(__builtin_amdgcn_cvt_scalef32_pk_f16_fp4(x, s, 3));
}

// Page and offset of token `pos` of a row, and whether it has a page.
struct MxSlot {
  int64_t token;   // page * PS + offset
  bool there;
};
__device__ __forceinline__ MxSlot mx_slot(const int32_t* row, int pos, int width, int64_t num_pages) {
  if (pos < 0 || pos >= width * (int64_t)PS) return MxSlot{0, false};
  const int page = row[pos >> 4];
  return MxSlot{(int64_t)page * PS + (pos & (PS - 1)), page >= 0 && page < num_pages};
}

}  // namespace iak

#endif
