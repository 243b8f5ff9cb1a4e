// Microscaled 4-bit rows (MXFP4): layout, host-side block quantiser and the launchers of scn_mx.hip.
#pragma once

#include <cstdint>
#include <cstring>

#include "scn_common.hpp"

namespace scn {

constexpr uint32_t kMxBlock = 32;        // channels per scale
constexpr uint32_t kMxBlockBytes = 16;   // code bytes per block

inline uint32_t mx_blocks(uint32_t c) { return c / kMxBlock + (c % kMxBlock != 0); }
inline uint32_t mx_scale_bytes(uint32_t c) { return (mx_blocks(c) + 3u) & ~3u; }
// one-buffer form: codes, then scales, rounded up to whole 16-byte chunks
inline uint32_t mx_row_bytes(uint32_t c) { return (mx_blocks(c) * kMxBlockBytes + mx_scale_bytes(c) + 15u) & ~15u; }

// Host quantiser of one block of up to 32 finite or non-finite values (weights are laid out on the host).
// codes: 16 bytes, missing values 0.  Returns the scale byte.
inline uint8_t mx_quantize_block(const float* v, int n, uint8_t codes[16]) {
  memset(codes, 0, 16);
  uint32_t top = 0;
  for (int i = 0; i < n; ++i) {
    uint32_t u;
    memcpy(&u, &v[i], 4);
    u &= 0x7FFFFFFFu;
    if (u > top) top = u;
  }
  const uint32_t field = top >> 23;
  if (field == 255) return 255;
  const uint32_t e = field > 2 ? field - 2 : 0;
  const uint32_t up_bits = (254 - e) << 23;   // 2^(127 - e)
  float up;
  memcpy(&up, &up_bits, 4);
  for (int i = 0; i < n; ++i) {
    const float s = v[i] * up;   // exact, or far below half of the smallest code
    uint32_t sb;
    memcpy(&sb, &s, 4);
    const float a = s < 0 ? -s : s;
    // midpoints between neighbouring values; a midpoint goes to the even code
    const int code = (a > 0.25f) + (a >= 0.75f) + (a > 1.25f) + (a >= 1.75f) + (a > 2.5f) + (a >= 3.5f) + (a > 5.f);
    codes[i / 2] |= (uint8_t)((code | (sb >> 31 ? 8 : 0)) << (4 * (i & 1)));
  }
  return (uint8_t)e;
}

// Memory that a call reads or writes: `rows` runs of `width` bytes, `ld` bytes apart.
struct MxSpan {
  const void* at;
  uint64_t rows, width, ld;
};
// Whether two of them share a byte.  Rows of the same stride may lie side by side in one array (codes and scales, columns of a
// wider buffer); of two strides whose ranges meet the answer is yes.
inline bool mx_overlap(const MxSpan& a, const MxSpan& b) {
  if (!a.at || !b.at || !a.rows || !b.rows || !a.width || !b.width) return false;
  const unsigned __int128 pa = (uintptr_t)a.at, pb = (uintptr_t)b.at;   // (no product of 32-bit numbers wraps)
  if (pa + (a.rows - 1) * a.ld + a.width <= pb || pb + (b.rows - 1) * b.ld + b.width <= pa) return false;
  const uint64_t ld = a.rows > 1 ? a.ld : b.ld;   // (a single row has no stride of its own)
  if ((a.rows > 1 && b.rows > 1 && a.ld != b.ld) || (a.rows == 1 && b.rows == 1) || ld == 0) return true;
  const uint64_t gap = (uint64_t)(pb >= pa ? pb - pa : pa - pb) % ld, d = pb >= pa || gap == 0 ? gap : ld - gap;   // where b's rows start behind a's
  return d < a.width || d + b.width > ld;
}

int mx_quantize_rows(const void* in, int in_dtype, uint32_t c, uint32_t in_ld, float in_range, int relu, uint8_t* codes,
                     uint32_t codes_ld, uint8_t* scales, uint32_t scales_ld, uint32_t n, const uint32_t* n_dev,
                     hipStream_t stream);
int mx_dequantize_rows(const uint8_t* codes, uint32_t codes_ld, const uint8_t* scales, uint32_t scales_ld, uint32_t c,
                       void* out, int out_dtype, uint32_t out_ld, uint32_t n, const uint32_t* n_dev, hipStream_t stream);
int mx_product(const scn_mx_product_io& io, hipStream_t stream);

}  // namespace scn
