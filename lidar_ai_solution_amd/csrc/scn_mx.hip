// Microscaled 4-bit rows (MXFP4): quantise, dequantise and product kernels (gfx950), and their C ABI.
#include "scn_mx.hpp"

#include <algorithm>

#include "scn_device.hpp"

namespace scn {

typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef float v2f __attribute__((ext_vector_type(2)));
typedef int v8i __attribute__((ext_vector_type(8)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));

// u / d for u < 2^31 by one high multiplication (d >= 1).
struct FastDiv {
  uint32_t d, mul, shift;
  explicit FastDiv(uint32_t d_) : d(d_), shift(0) {
    while (shift < 32 && (1ull << shift) < d) ++shift;
    mul = (uint32_t)(((1ull << 32) * ((1ull << shift) - d)) / d + 1);
  }
  __device__ __forceinline__ uint32_t div(uint32_t u) const { return (__umulhi(u, mul) + u) >> shift; }
};

// --------------------------------------------------------------------------------------------
// quantise / dequantise
// --------------------------------------------------------------------------------------------
// A thread owns 16 bytes of a row (E = 8 fp16, 4 fp32 or 16 int8 channels), so a wave moves 1 KB of consecutive input
// with one load; a block's largest magnitude is the maximum over 32 / E neighbouring lanes.  Both kernels are bound by
// memory: 2 or 4 bytes per channel on one side, 17 / 32 of a byte on the other.
template <int DT>
struct MxIn;
template <>
struct MxIn<SCN_DTYPE_FP16> {
  typedef _Float16 T;
};
template <>
struct MxIn<SCN_DTYPE_FP32> {
  typedef float T;
};
template <>
struct MxIn<SCN_DTYPE_INT8> {
  typedef signed char T;
};

// max over the lanes whose numbers differ in the lowest log2(W) bits (W = 2, 4 or 8)
template <int W>
__device__ __forceinline__ uint32_t lanes_max(uint32_t v) {
  if (W >= 2) v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0xB1, 0xF, 0xF, true));   // quad_perm 1,0,3,2
  if (W >= 4) v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x4E, 0xF, 0xF, true));   // quad_perm 2,3,0,1
  if (W >= 8) v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x141, 0xF, 0xF, true));  // row_half_mirror
  return v;
}

// Scale byte of a block from the fp32 bits of its largest magnitude (255: not finite).
__device__ __forceinline__ uint32_t mx_scale_byte(uint32_t top_bits) {
  const uint32_t f = top_bits >> 23;
  return f == 255u ? 255u : f > 2u ? f - 2u : 0u;
}

// 8 fp32 values times `up` -> 8 codes (the conversion instruction rounds to nearest even and saturates).
__device__ __forceinline__ uint32_t mx_codes8(const float (&v)[8], float up) {
  uint32_t r = 0;
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[0] * up, v[1] * up, 1.f, 0);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[2] * up, v[3] * up, 1.f, 1);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[4] * up, v[5] * up, 1.f, 2);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[6] * up, v[7] * up, 1.f, 3);
  return r;
}

// Channels [ch, ch + E) of a row -> fp32 (ReLU and int8 scale applied), channels >= c read as 0.
template <int DT, int E>
__device__ __forceinline__ void mx_load(const typename MxIn<DT>::T* row, uint32_t ch, uint32_t c, float in_scale, int relu,
                                        float (&v)[E]) {
  typedef typename MxIn<DT>::T T;
  T raw[E];
  if (ch + E <= c) {
    __builtin_memcpy(raw, row + ch, sizeof(raw));   // one 16-byte load at any alignment
  } else {
#pragma unroll
    for (int i = 0; i < E; ++i) raw[i] = ch + i < c ? row[ch + i] : (T)0;
  }
#pragma unroll
  for (int i = 0; i < E; ++i) {
    v[i] = (float)raw[i];
    if (DT == SCN_DTYPE_INT8) v[i] *= in_scale;
    if (relu) v[i] = v[i] > 0.f ? v[i] : 0.f;
  }
}

template <int DT>
__global__ __launch_bounds__(256) void k_mx_quantize(const typename MxIn<DT>::T* in, uint32_t c, uint32_t in_ld,
                                                     float in_scale, int relu, uint8_t* codes, uint32_t codes_ld,
                                                     uint8_t* scales, uint32_t scales_ld, FastDiv blocks,
                                                     uint32_t rows_per_slice, uint32_t n_bound, const uint32_t* n_dev) {
  constexpr int E = 16 / (int)sizeof(typename MxIn<DT>::T), LPB = 32 / E;
  const uint32_t n = eff_n(n_dev, n_bound);
  const uint32_t u = (blockIdx.x * 256u + threadIdx.x) / LPB;   // block of this slice of rows
  const uint32_t sub = threadIdx.x % LPB;
  const uint32_t r = blocks.div(u), b = u - r * blocks.d;
  const size_t row = (size_t)blockIdx.y * rows_per_slice + r;
  const bool live = r < rows_per_slice && row < n;
  float v[E];
#pragma unroll
  for (int i = 0; i < E; ++i) v[i] = 0.f;
  if (live) mx_load<DT, E>(in + row * in_ld, b * 32 + sub * E, c, in_scale, relu, v);
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < E; ++i) top = max(top, __float_as_uint(v[i]) & 0x7FFFFFFFu);
  top = lanes_max<LPB>(top);
  if (!live) return;
  const uint32_t e = mx_scale_byte(top);
  uint32_t w[E >= 8 ? E / 8 : 1];
  const float up = __uint_as_float((254u - (e == 255u ? 0u : e)) << 23);
  if constexpr (E >= 8) {
#pragma unroll
    for (int q = 0; q < E / 8; ++q) {
      float t[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) t[i] = v[q * 8 + i];
      w[q] = e == 255u ? 0u : mx_codes8(t, up);
    }
  } else {
    w[0] = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, v[0] * up, v[1] * up, 1.f, 0);
    w[0] = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w[0], v[2] * up, v[3] * up, 1.f, 1);
    if (e == 255u) w[0] = 0u;
  }
  uint8_t* dst = codes + row * codes_ld + b * 16 + sub * (E / 2);
  if constexpr (E == 8) *reinterpret_cast<uint32_t*>(dst) = w[0];
  if constexpr (E == 16) *reinterpret_cast<uint2*>(dst) = make_uint2(w[0], w[1]);
  if constexpr (E == 4) *reinterpret_cast<uint16_t*>(dst) = (uint16_t)w[0];
  if (sub == 0) {
    uint8_t* s = scales + row * scales_ld;
    s[b] = (uint8_t)e;
    if (b + 1 == blocks.d)
      for (uint32_t q = blocks.d; q < ((blocks.d + 3u) & ~3u); ++q) s[q] = 0;
  }
}

// Scale of a block as fp32: 2^(e - 127); e = 0 is the subnormal 2^-127, 255 is NaN.
__device__ __forceinline__ float mx_scale_value(uint32_t e) {
  return __uint_as_float(e == 0u ? 0x00400000u : e == 255u ? 0x7FC00000u : e << 23);
}

// The values of 8 (fp16) or 4 (fp32) codes.
__device__ __forceinline__ void mx_values(uint32_t w, float x, _Float16 (&v)[8]) {
  const v2h a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, x, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, x, 1),
            c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, x, 2), d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, x, 3);
  v[0] = a.x, v[1] = a.y, v[2] = b.x, v[3] = b.y, v[4] = c.x, v[5] = c.y, v[6] = d.x, v[7] = d.y;
}
__device__ __forceinline__ void mx_values(uint32_t w, float x, float (&v)[4]) {
  const v2f a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, x, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, x, 1);
  v[0] = a.x, v[1] = a.y, v[2] = b.x, v[3] = b.y;
}

template <typename OT>
__global__ __launch_bounds__(256) void k_mx_dequantize(const uint8_t* codes, uint32_t codes_ld, const uint8_t* scales,
                                                       uint32_t scales_ld, uint32_t c, OT* out, uint32_t out_ld,
                                                       FastDiv blocks, uint32_t rows_per_slice, uint32_t n_bound,
                                                       const uint32_t* n_dev) {
  constexpr int E = 16 / (int)sizeof(OT), LPB = 32 / E;
  const uint32_t n = eff_n(n_dev, n_bound);
  const uint32_t u = (blockIdx.x * 256u + threadIdx.x) / LPB;
  const uint32_t sub = threadIdx.x % LPB;
  const uint32_t r = blocks.div(u), b = u - r * blocks.d;
  const size_t row = (size_t)blockIdx.y * rows_per_slice + r;
  if (r >= rows_per_slice || row >= n) return;
  const uint8_t* src = codes + row * codes_ld + b * 16 + sub * (E / 2);
  const uint32_t w = E == 8 ? *reinterpret_cast<const uint32_t*>(src) : *reinterpret_cast<const uint16_t*>(src);
  const float x = mx_scale_value(scales[row * scales_ld + b]);
  OT v[E];
  mx_values(w, x, v);
  const uint32_t ch = b * 32 + sub * E;
  OT* dst = out + row * out_ld + ch;
  if (ch + E <= c) {
    __builtin_memcpy(dst, v, sizeof(v));
  } else {
#pragma unroll
    for (int i = 0; i < E; ++i)
      if (ch + i < c) dst[i] = v[i];
  }
}

// Rows are cut into slices (grid y) so that the blocks of a slice are counted in 31 bits.
struct MxGrid {
  uint32_t rows_per_slice;
  dim3 grid;
  MxGrid(uint32_t n, uint32_t blocks, uint32_t lanes_per_block) {
    const uint64_t cap = (1ull << 31) / ((uint64_t)blocks * lanes_per_block) - 1;   // threads of a slice stay below 2^31
    rows_per_slice = (uint32_t)std::max<uint64_t>(1, std::min<uint64_t>(n, cap));
    // at most 65535 slices: n < 2^32 rows of at most 2^27 blocks would exceed the GPU's memory long before
    const uint64_t threads = (uint64_t)rows_per_slice * blocks * lanes_per_block;
    grid = dim3((unsigned)((threads + 255) / 256), (unsigned)((n + (uint64_t)rows_per_slice - 1) / rows_per_slice));
  }
};

static int mx_check_rows(const char* what, const void* codes, uint32_t codes_ld, const void* scales, uint32_t scales_ld,
                         uint32_t c) {
  SCN_REQUIRE(c > 0 && c <= (1u << 30), SCN_ERR_INVALID, "%s: %u channels", what, c);
  SCN_REQUIRE(codes && scales, SCN_ERR_INVALID, "%s: null codes or scales", what);
  SCN_REQUIRE(((uintptr_t)codes & 15) == 0 && codes_ld % 16 == 0 && codes_ld >= mx_blocks(c) * kMxBlockBytes, SCN_ERR_INVALID,
              "%s: code rows must be 16-byte aligned and hold %u bytes (stride %u)", what, mx_blocks(c) * kMxBlockBytes, codes_ld);
  SCN_REQUIRE(((uintptr_t)scales & 3) == 0 && scales_ld % 4 == 0 && scales_ld >= mx_scale_bytes(c), SCN_ERR_INVALID,
              "%s: scale rows must be 4-byte aligned and hold %u bytes (stride %u)", what, mx_scale_bytes(c), scales_ld);
  return SCN_OK;
}

int mx_quantize_rows(const void* in, int in_dtype, uint32_t c, uint32_t in_ld, float in_range, int relu, uint8_t* codes,
                     uint32_t codes_ld, uint8_t* scales, uint32_t scales_ld, uint32_t n, const uint32_t* n_dev,
                     hipStream_t stream) {
  SCN_REQUIRE(in_dtype == SCN_DTYPE_FP16 || in_dtype == SCN_DTYPE_FP32 || in_dtype == SCN_DTYPE_INT8, SCN_ERR_INVALID,
              "mx_quantize_rows: rows must be fp16, fp32 or int8 (dtype %d)", in_dtype);
  if (n == 0) return SCN_OK;
  if (int rc = mx_check_rows("mx_quantize_rows", codes, codes_ld, scales, scales_ld, c)) return rc;
  const uint32_t esz = in_dtype == SCN_DTYPE_FP32 ? 4 : in_dtype == SCN_DTYPE_FP16 ? 2 : 1;
  SCN_REQUIRE(in && ((uintptr_t)in & (esz - 1)) == 0 && in_ld >= c, SCN_ERR_INVALID,
              "mx_quantize_rows: null or misaligned rows, or row stride %u < %u channels", in_ld, c);
  SCN_REQUIRE(in_dtype != SCN_DTYPE_INT8 || in_range > 0.f, SCN_ERR_INVALID, "mx_quantize_rows: int8 rows need in_range > 0");
  const FastDiv fd(mx_blocks(c));
  const MxGrid g(n, fd.d, 2 * esz);
#define SCN_MX_QUANTIZE(DT)                                                                                            \
  hipLaunchKernelGGL(k_mx_quantize<DT>, g.grid, dim3(256), 0, stream, reinterpret_cast<const MxIn<DT>::T*>(in), c, in_ld, \
                     in_range / 127.f, relu, codes, codes_ld, scales, scales_ld, fd, g.rows_per_slice, n, n_dev)
  if (in_dtype == SCN_DTYPE_FP16) SCN_MX_QUANTIZE(SCN_DTYPE_FP16);
  else if (in_dtype == SCN_DTYPE_FP32) SCN_MX_QUANTIZE(SCN_DTYPE_FP32);
  else SCN_MX_QUANTIZE(SCN_DTYPE_INT8);
#undef SCN_MX_QUANTIZE
  SCN_HIP(hipGetLastError());
  return SCN_OK;
}

int mx_dequantize_rows(const uint8_t* codes, uint32_t codes_ld, const uint8_t* scales, uint32_t scales_ld, uint32_t c,
                       void* out, int out_dtype, uint32_t out_ld, uint32_t n, const uint32_t* n_dev, hipStream_t stream) {
  SCN_REQUIRE(out_dtype == SCN_DTYPE_FP16 || out_dtype == SCN_DTYPE_FP32, SCN_ERR_INVALID,
              "mx_dequantize_rows: output must be fp16 or fp32 (dtype %d)", out_dtype);
  if (n == 0) return SCN_OK;
  if (int rc = mx_check_rows("mx_dequantize_rows", codes, codes_ld, scales, scales_ld, c)) return rc;
  const uint32_t esz = out_dtype == SCN_DTYPE_FP32 ? 4 : 2;
  SCN_REQUIRE(out && ((uintptr_t)out & (esz - 1)) == 0 && out_ld >= c, SCN_ERR_INVALID,
              "mx_dequantize_rows: null or misaligned output, or row stride %u < %u channels", out_ld, c);
  const FastDiv fd(mx_blocks(c));
  const MxGrid g(n, fd.d, 2 * esz);
  if (out_dtype == SCN_DTYPE_FP16)
    hipLaunchKernelGGL(k_mx_dequantize<_Float16>, g.grid, dim3(256), 0, stream, codes, codes_ld, scales, scales_ld, c,
                       (_Float16*)out, out_ld, fd, g.rows_per_slice, n, n_dev);
  else
    hipLaunchKernelGGL(k_mx_dequantize<float>, g.grid, dim3(256), 0, stream, codes, codes_ld, scales, scales_ld, c,
                       (float*)out, out_ld, fd, g.rows_per_slice, n, n_dev);
  SCN_HIP(hipGetLastError());
  return SCN_OK;
}

// --------------------------------------------------------------------------------------------
// product
// --------------------------------------------------------------------------------------------
// Operands of the scaled matrix instructions (A and B in 4-bit codes, wave64):
//   16x16x128: lane l supplies row / column l % 16 and the 16 code bytes of K-block l / 16, with that block's scale
//   32x32x64:  lane l supplies row / column l % 32 and the 16 code bytes of K-block l / 32, with that block's scale
// A block of a microscaled row is exactly what one lane supplies, so rows need no re-ordering.  The rows of A are the
// rows of the weight matrix (output channels), the columns of B the input rows, as in the convolution kernels: a lane
// ends up with 4 (x 4) consecutive output channels of one row.
struct ProductArgs {
  const void* a;
  uint32_t a_ld;
  const uint8_t* as;
  uint32_t as_ld;
  const uint8_t* b;
  uint32_t b_ld;
  const uint8_t* bs;
  uint32_t bs_ld;
  uint32_t m, n, k, kb;   // kb = blocks of a row
  const uint32_t* m_dev;
  const void* bias;
  int bias_fp32, relu;
  const void* res;
  int res_fp32;
  uint32_t res_ld;
  int relu2;
  void* out;
  int out_fp32;
  uint32_t out_ld;
};

__device__ __forceinline__ v8i mx_operand(const uint4& q) {
  return v8i{(int)q.x, (int)q.y, (int)q.z, (int)q.w, 0, 0, 0, 0};
}
__device__ __forceinline__ v4f mx_mma16(const uint4& a, int sa, const uint4& b, int sb, v4f c) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(mx_operand(a), mx_operand(b), c, 4, 4, 0, sa, 0, sb);
}
__device__ __forceinline__ v16f mx_mma32(const uint4& a, int sa, const uint4& b, int sb, v16f c) {
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(mx_operand(a), mx_operand(b), c, 4, 4, 0, sa, 0, sb);
}

// Bias, ReLU, residual and store of one element.
__device__ __forceinline__ void product_store(const ProductArgs& p, uint32_t i, uint32_t j, float y) {
  if (p.bias) y += p.bias_fp32 ? ((const float*)p.bias)[j] : (float)((const _Float16*)p.bias)[j];
  if (p.relu) y = y > 0.f ? y : 0.f;
  if (p.res) {
    const size_t at = (size_t)i * p.res_ld + j;
    y += p.res_fp32 ? ((const float*)p.res)[at] : (float)((const _Float16*)p.res)[at];
  }
  if (p.relu2) y = y > 0.f ? y : 0.f;
  const size_t at = (size_t)i * p.out_ld + j;
  if (p.out_fp32) ((float*)p.out)[at] = y;
  else ((_Float16*)p.out)[at] = (_Float16)y;
}

// Codes and scale of block `b` of a row that is not quantised yet, by one lane.
template <int DT>
__device__ __forceinline__ uint4 mx_quantize_lane(const typename MxIn<DT>::T* row, uint32_t b, uint32_t c, int* scale) {
  float v[32];
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    float t[8];
    mx_load<DT, 8>(row, b * 32 + q * 8, c, 1.f, 0, t);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[q * 8 + i] = t[i];
  }
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 32; ++i) top = max(top, __float_as_uint(v[i]) & 0x7FFFFFFFu);
  const uint32_t e = mx_scale_byte(top);
  *scale = (int)e;
  if (e == 255u) return make_uint4(0, 0, 0, 0);
  const float up = __uint_as_float((254u - e) << 23);
  uint32_t w[4];
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    float t[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) t[i] = v[q * 8 + i];
    w[q] = mx_codes8(t, up);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// Few rows (m <= 16): bound by reading the weights.  A workgroup owns 16 output channels and all rows; its 8 waves
// split the channels k between them (contiguous runs of 128) and add their sums in LDS, in wave order.  Rows that are
// not quantised are quantised by the lane that supplies them (AT = their dtype; SCN_DTYPE_MXFP4: they are).
template <int AT>
__global__ __launch_bounds__(512) void k_mx_product_few(const ProductArgs p) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int lr = lane & 15, lg = lane >> 4;
  const uint32_t m = eff_n(p.m_dev, p.m);
  if (m == 0) return;
  const uint32_t n0 = blockIdx.x * 16;
  const uint32_t brow = min(n0 + lr, p.n - 1), arow = min((uint32_t)lr, m - 1);
  const uint8_t* bc = p.b + (size_t)brow * p.b_ld;
  const uint8_t* bsc = p.bs + (size_t)brow * p.bs_ld;
  const uint32_t steps = (p.kb + 3) / 4, per = (steps + 7) / 8;
  const uint32_t s0 = wave * per, s1 = min(steps, s0 + per);
  v4f acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (uint32_t s = s0; s < s1; ++s) {
    const uint32_t blk = 4 * s + lg;
    uint4 wq = make_uint4(0, 0, 0, 0), xq = make_uint4(0, 0, 0, 0);
    int ws = 0, xs = 0;
    if (blk < p.kb) {
      wq = *reinterpret_cast<const uint4*>(bc + (size_t)blk * 16);
      ws = bsc[blk];
      if constexpr (AT == SCN_DTYPE_MXFP4) {
        xq = *reinterpret_cast<const uint4*>((const uint8_t*)p.a + (size_t)arow * p.a_ld + (size_t)blk * 16);
        xs = p.as[(size_t)arow * p.as_ld + blk];
      } else if ((uint32_t)lr < m) {
        typedef typename MxIn<AT>::T T;
        xq = mx_quantize_lane<AT>((const T*)p.a + (size_t)arow * p.a_ld, blk, p.k, &xs);
      }
    }
    acc = mx_mma16(wq, ws, xq, xs, acc);
  }
  __shared__ float part[8][64][4];
#pragma unroll
  for (int j = 0; j < 4; ++j) part[wave][lane][j] = acc[j];
  __syncthreads();
  if (threadIdx.x < 256) {
    // thread = (row, channel), channels fastest: channel 4 g + j of row r is element j of lane 16 g + r
    const uint32_t i = threadIdx.x / 16, ch = threadIdx.x % 16;
    float y = 0.f;
#pragma unroll
    for (int w = 0; w < 8; ++w) y += part[w][(ch / 4) * 16 + i][ch % 4];
    if (i < m && n0 + ch < p.n) product_store(p, i, n0 + ch, y);
  }
}

// Any number of rows: a wave owns 32 rows x 32 output channels, both operands straight from memory.
__global__ __launch_bounds__(256) void k_mx_product_tile(const ProductArgs p) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int ln = lane & 31, lh = lane >> 5;
  const uint32_t m = eff_n(p.m_dev, p.m);
  const uint32_t i0 = blockIdx.x * 32, n0 = (blockIdx.y * 4 + wave) * 32;
  if (i0 >= m || n0 >= p.n) return;
  const uint32_t brow = min(n0 + ln, p.n - 1), arow = min(i0 + ln, m - 1);
  const uint8_t* bc = p.b + (size_t)brow * p.b_ld;
  const uint8_t* bsc = p.bs + (size_t)brow * p.bs_ld;
  const uint8_t* ac = (const uint8_t*)p.a + (size_t)arow * p.a_ld;
  const uint8_t* asc = p.as + (size_t)arow * p.as_ld;
  v16f acc;
#pragma unroll
  for (int j = 0; j < 16; ++j) acc[j] = 0.f;
  for (uint32_t s = 0; s < (p.kb + 1) / 2; ++s) {
    const uint32_t blk = 2 * s + lh;
    uint4 wq = make_uint4(0, 0, 0, 0), xq = make_uint4(0, 0, 0, 0);
    int ws = 0, xs = 0;
    if (blk < p.kb) {
      wq = *reinterpret_cast<const uint4*>(bc + (size_t)blk * 16);
      xq = *reinterpret_cast<const uint4*>(ac + (size_t)blk * 16);
      ws = bsc[blk];
      xs = asc[blk];
    }
    acc = mx_mma32(wq, ws, xq, xs, acc);
  }
  if (i0 + ln >= m) return;
#pragma unroll
  for (int j = 0; j < 16; ++j) {
    const uint32_t ch = n0 + 8 * (j / 4) + 4 * lh + j % 4;
    if (ch < p.n) product_store(p, i0 + ln, ch, acc[j]);
  }
}

constexpr uint32_t kDirectRows = 16;

static size_t product_workspace(uint32_t m, uint32_t k) { return (size_t)m * mx_row_bytes(k); }

int mx_product(const scn_mx_product_io& io, hipStream_t stream) {
  SCN_REQUIRE(io.a_dtype == SCN_DTYPE_MXFP4 || io.a_dtype == SCN_DTYPE_FP16 || io.a_dtype == SCN_DTYPE_FP32, SCN_ERR_INVALID,
              "mx_product: rows must be microscaled, fp16 or fp32 (dtype %d)", io.a_dtype);
  SCN_REQUIRE(io.out_dtype == SCN_DTYPE_FP16 || io.out_dtype == SCN_DTYPE_FP32, SCN_ERR_INVALID,
              "mx_product: output must be fp16 or fp32 (dtype %d)", io.out_dtype);
  SCN_REQUIRE(io.n > 0 && io.k > 0, SCN_ERR_INVALID, "mx_product: n = %u, k = %u", io.n, io.k);
  SCN_REQUIRE(!io.bias_dev || io.bias_dtype == SCN_DTYPE_FP16 || io.bias_dtype == SCN_DTYPE_FP32, SCN_ERR_INVALID,
              "mx_product: bias must be fp16 or fp32 (dtype %d)", io.bias_dtype);
  SCN_REQUIRE(!io.res_dev || io.res_dtype == SCN_DTYPE_FP16 || io.res_dtype == SCN_DTYPE_FP32, SCN_ERR_INVALID,
              "mx_product: residual must be fp16 or fp32 (dtype %d)", io.res_dtype);
  if (io.m == 0) return SCN_OK;
  const uint32_t kb = mx_blocks(io.k);
  if (int rc = mx_check_rows("mx_product (b)", io.b_codes_dev, io.b_codes_ld, io.b_scales_dev, io.b_scales_ld, io.k)) return rc;
  auto aligned = [](const void* p, int dtype) { return ((uintptr_t)p & (dtype == SCN_DTYPE_FP32 ? 3 : 1)) == 0; };
  SCN_REQUIRE(io.out_dev && aligned(io.out_dev, io.out_dtype) && io.out_ld >= io.n, SCN_ERR_INVALID,
              "mx_product: null or misaligned output, or row stride %u < %u", io.out_ld, io.n);
  SCN_REQUIRE(aligned(io.bias_dev, io.bias_dtype), SCN_ERR_INVALID, "mx_product: misaligned bias");
  SCN_REQUIRE(!io.res_dev || (aligned(io.res_dev, io.res_dtype) && io.res_ld >= io.n), SCN_ERR_INVALID,
              "mx_product: misaligned residual, or row stride %u < %u", io.res_ld, io.n);
  ProductArgs p;
  p.a = io.a_dev;
  p.a_ld = io.a_ld;
  p.as = io.a_scales_dev;
  p.as_ld = io.a_scales_ld;
  p.b = io.b_codes_dev;
  p.b_ld = io.b_codes_ld;
  p.bs = io.b_scales_dev;
  p.bs_ld = io.b_scales_ld;
  p.m = io.m;
  p.n = io.n;
  p.k = io.k;
  p.kb = kb;
  p.m_dev = io.m_dev;
  p.bias = io.bias_dev;
  p.bias_fp32 = io.bias_dtype == SCN_DTYPE_FP32;
  p.relu = io.relu;
  p.res = io.res_dev;
  p.res_fp32 = io.res_dtype == SCN_DTYPE_FP32;
  p.res_ld = io.res_ld;
  p.relu2 = io.relu_after_add;
  p.out = io.out_dev;
  p.out_fp32 = io.out_dtype == SCN_DTYPE_FP32;
  p.out_ld = io.out_ld;
  int at = io.a_dtype;
  if (at == SCN_DTYPE_MXFP4) {
    if (int rc = mx_check_rows("mx_product (a)", (const uint8_t*)io.a_dev, io.a_ld, io.a_scales_dev, io.a_scales_ld, io.k)) return rc;
  } else {
    SCN_REQUIRE(io.a_dev && aligned(io.a_dev, at) && io.a_ld >= io.k, SCN_ERR_INVALID,
                "mx_product: null or misaligned rows, or row stride %u < %u channels", io.a_ld, io.k);
    if (io.m > kDirectRows) {
      const size_t need = product_workspace(io.m, io.k);
      SCN_REQUIRE(io.workspace_dev && ((uintptr_t)io.workspace_dev & 15) == 0 && io.workspace_bytes >= need, SCN_ERR_INVALID,
                  "mx_product: rows of this type need a 16-byte aligned workspace of %zu bytes (%zu given)", need, io.workspace_bytes);
      uint8_t* ws = (uint8_t*)io.workspace_dev;
      p.a = ws;
      p.a_ld = p.as_ld = mx_row_bytes(io.k);
      p.as = ws + (size_t)kb * kMxBlockBytes;
      if (int rc = mx_quantize_rows(io.a_dev, at, io.k, io.a_ld, 0.f, 0, ws, p.a_ld, const_cast<uint8_t*>(p.as), p.as_ld, io.m,
                                    io.m_dev, stream))
        return rc;
      at = SCN_DTYPE_MXFP4;
    }
  }
  if (io.m <= kDirectRows) {
    const dim3 grid(ceil_div(io.n, 16));
    if (at == SCN_DTYPE_MXFP4) hipLaunchKernelGGL(k_mx_product_few<SCN_DTYPE_MXFP4>, grid, dim3(512), 0, stream, p);
    else if (at == SCN_DTYPE_FP16) hipLaunchKernelGGL(k_mx_product_few<SCN_DTYPE_FP16>, grid, dim3(512), 0, stream, p);
    else hipLaunchKernelGGL(k_mx_product_few<SCN_DTYPE_FP32>, grid, dim3(512), 0, stream, p);
  } else {
    SCN_REQUIRE(ceil_div(io.n, 128) <= 65535u, SCN_ERR_UNSUPPORTED, "mx_product: n = %u is too large", io.n);
    hipLaunchKernelGGL(k_mx_product_tile, dim3(ceil_div(io.m, 32), ceil_div(io.n, 128)), dim3(256), 0, stream, p);
  }
  SCN_HIP(hipGetLastError());
  return SCN_OK;
}

}  // namespace scn

using namespace scn;

extern "C" {

size_t scn_mx_row_bytes(uint32_t c) { return mx_row_bytes(c); }

int scn_mx_quantize_rows(const void* in_dev, int in_dtype, uint32_t c, uint32_t in_ld, float in_range, int relu,
                         uint8_t* codes_dev, uint32_t codes_ld, uint8_t* scales_dev, uint32_t scales_ld, uint32_t n,
                         const uint32_t* n_dev, void* stream) {
  int rc = mx_quantize_rows(in_dev, in_dtype, c, in_ld, in_range, relu, codes_dev, codes_ld, scales_dev, scales_ld, n, n_dev,
                            (hipStream_t)stream);
  if (rc == SCN_OK && debug_sync_enabled()) rc = debug_sync_check((hipStream_t)stream, "scn_mx_quantize_rows");
  return rc;
}

int scn_mx_dequantize_rows(const uint8_t* codes_dev, uint32_t codes_ld, const uint8_t* scales_dev, uint32_t scales_ld,
                           uint32_t c, void* out_dev, int out_dtype, uint32_t out_ld, uint32_t n, const uint32_t* n_dev,
                           void* stream) {
  int rc = mx_dequantize_rows(codes_dev, codes_ld, scales_dev, scales_ld, c, out_dev, out_dtype, out_ld, n, n_dev,
                              (hipStream_t)stream);
  if (rc == SCN_OK && debug_sync_enabled()) rc = debug_sync_check((hipStream_t)stream, "scn_mx_dequantize_rows");
  return rc;
}

uint32_t scn_mx_product_direct_rows(void) { return kDirectRows; }
size_t scn_mx_product_workspace(uint32_t m, uint32_t k) { return m > kDirectRows ? product_workspace(m, k) : 0; }

int scn_mx_product(const scn_mx_product_io* io, void* stream) {
  SCN_REQUIRE(io, SCN_ERR_INVALID, "scn_mx_product: null pointer");
  int rc = mx_product(*io, (hipStream_t)stream);
  if (rc == SCN_OK && debug_sync_enabled()) rc = debug_sync_check((hipStream_t)stream, "scn_mx_product");
  return rc;
}

}  // extern "C"
