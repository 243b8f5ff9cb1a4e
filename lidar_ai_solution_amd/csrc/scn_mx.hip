// Microscaled 4-bit rows (MXFP4): quantise, dequantise and product kernels (gfx950), and their C ABI.
#include "scn_mx.hpp"

#include <algorithm>

#include "scn_mx_device.hpp"

namespace scn {

typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef float v2f __attribute__((ext_vector_type(2)));
typedef int v8i __attribute__((ext_vector_type(8)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));

// 16 bytes to an address of any alignment.  STREAM: past the L2 (results that no workgroup of this launch reads again).  Where a
// wave writes whole lines, or nearly, ordinary stores make the write-back L2 the bottleneck: us streaming | ordinary, dequantising
// 16,384 x 8,192 to fp16 52 | 66, to fp32 88 | 123, 50,000 x 1000 to fp16 21.7 | 27.9, 322,224 x 60 to fp16 16.1 | 20.5.
typedef uint32_t v4u_any __attribute__((ext_vector_type(4), aligned(2)));
template <bool STREAM>
__device__ __forceinline__ void store16(void* dst, const void* src) {
  v4u_any q;
  __builtin_memcpy(&q, src, 16);
  if (STREAM) __builtin_nontemporal_store(q, reinterpret_cast<v4u_any*>(dst));
  else *reinterpret_cast<v4u_any*>(dst) = q;
}

// u / d for u < 2^31 by one high multiplication (d >= 1): the round-up method of Granlund and Montgomery (Division by Invariant
// Integers using Multiplication, 1994).
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

// ONE: rows of one block, whose scale and padding are one word (322,224 rows of 32 channels: 8.8 us by bytes, 8.2 us so; words
// put together across lanes for wider rows gain nothing: 123,646 x 128 9.4 us either way, 16,384 x 4096 fp32 56.8 against 59.1).
template <int DT, bool ONE>
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
  const uint32_t e = mx_scale_byte(top);
  if (live && sub == 0) {
    uint8_t* s = scales + row * scales_ld;
    if constexpr (ONE) {
      *reinterpret_cast<uint32_t*>(s) = e;
    } else {
      s[b] = (uint8_t)e;
      if (b + 1 == blocks.d)
        for (uint32_t q = blocks.d; q % 4 != 0; ++q) s[q] = 0;
    }
  }
  if (!live) return;
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
    store16<true>(dst, v);
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
  const MxSpan rows{in, n, (uint64_t)c * esz, (uint64_t)in_ld * esz}, cs{codes, n, mx_blocks(c) * kMxBlockBytes, codes_ld},
      ss{scales, n, mx_scale_bytes(c), scales_ld};
  SCN_REQUIRE(!mx_overlap(rows, cs) && !mx_overlap(rows, ss) && !mx_overlap(cs, ss), SCN_ERR_INVALID,
              "mx_quantize_rows: the rows, the codes and the scales must not overlap");
  const FastDiv fd(mx_blocks(c));
  const MxGrid g(n, fd.d, 2 * esz);
#define SCN_MX_QUANTIZE(DT, ONE)                                                                                          \
  hipLaunchKernelGGL((k_mx_quantize<DT, ONE>), g.grid, dim3(256), 0, stream, reinterpret_cast<const MxIn<DT>::T*>(in), c, \
                     in_ld, in_range / 127.f, relu, codes, codes_ld, scales, scales_ld, fd, g.rows_per_slice, n, n_dev)
#define SCN_MX_QUANTIZE_DT(DT)                     \
  if (fd.d == 1) SCN_MX_QUANTIZE(DT, true);        \
  else SCN_MX_QUANTIZE(DT, false)
  if (in_dtype == SCN_DTYPE_FP16) {
    SCN_MX_QUANTIZE_DT(SCN_DTYPE_FP16);
  } else if (in_dtype == SCN_DTYPE_FP32) {
    SCN_MX_QUANTIZE_DT(SCN_DTYPE_FP32);
  } else {
    SCN_MX_QUANTIZE_DT(SCN_DTYPE_INT8);
  }
#undef SCN_MX_QUANTIZE_DT
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
  const MxSpan rows{out, n, (uint64_t)c * esz, (uint64_t)out_ld * esz};
  SCN_REQUIRE(!mx_overlap(rows, {codes, n, mx_blocks(c) * kMxBlockBytes, codes_ld}) &&
                  !mx_overlap(rows, {scales, n, mx_scale_bytes(c), scales_ld}),
              SCN_ERR_INVALID, "mx_dequantize_rows: the output must not overlap the codes or the scales");
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

// ReLU of a product: a NaN (of a block that is not finite) stays one.
__device__ __forceinline__ float product_relu(float y) { return y < 0.f ? 0.f : y; }

// Bias, ReLU, residual and store of one element.
__device__ __forceinline__ void product_store(const ProductArgs& p, uint32_t i, uint32_t j, float y) {
  if (p.bias) y += p.bias_fp32 ? ((const float*)p.bias)[j] : (float)((const _Float16*)p.bias)[j];
  if (p.relu) y = product_relu(y);
  if (p.res) {
    const size_t at = (size_t)i * p.res_ld + j;
    y += p.res_fp32 ? ((const float*)p.res)[at] : (float)((const _Float16*)p.res)[at];
  }
  if (p.relu2) y = product_relu(y);
  const size_t at = (size_t)i * p.out_ld + j;
  if (p.out_fp32) ((float*)p.out)[at] = y;
  else ((_Float16*)p.out)[at] = (_Float16)y;
}

// Codes and scale byte of block `b` of a row that is not quantised yet, by one thread.
template <int DT>
__device__ __forceinline__ uint4 mx_quantize_block_dev(const typename MxIn<DT>::T* row, uint32_t b, uint32_t c, uint32_t* scale) {
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
  *scale = e;
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

// Few rows (m <= 16 MT): bound by reading the weights.  A workgroup owns 16 output channels and all rows; its (up to 8) waves
// split the channels k between them (contiguous runs of 128) and add their sums in LDS, in wave order.  The weights of U runs
// are requested before anything waits (U KB per wave in flight), so rows that are not quantised yet (AT = their dtype) are
// quantised into LDS by the whole workgroup while the weights travel.
// (8192 x 8192 weights, one fp16 row: 21.4 us with a dependent load per run and every wave quantising for itself, 11.9 us so.)
constexpr uint32_t kFewBlocks = 1024;   // blocks of quantised rows in LDS

template <int AT, int MT, int U>
__global__ __launch_bounds__(512) void k_mx_product_few(const ProductArgs p) {
  constexpr bool MX = AT == SCN_DTYPE_MXFP4;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
  const int lr = lane & 15, lg = lane >> 4;
  __shared__ uint4 xcodes[MX ? 1 : kFewBlocks];
  __shared__ uint8_t xscales[MX ? 1 : kFewBlocks];
  __shared__ float part[8][MT][64][4];
  const uint32_t m = eff_n(p.m_dev, p.m);
  if (m == 0) return;
  const uint32_t n0 = blockIdx.x * 16;
  const uint32_t brow = min(n0 + lr, p.n - 1);
  const uint8_t* bc = p.b + (size_t)brow * p.b_ld;
  const uint8_t* bsc = p.bs + (size_t)brow * p.bs_ld;
  uint32_t arow[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) arow[t] = min((uint32_t)(16 * t + lr), m - 1);
  v4f acc[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) acc[t] = v4f{0.f, 0.f, 0.f, 0.f};
  const uint32_t runs = (p.kb + 3) / 4, per = (runs + waves - 1) / waves;   // runs of 4 blocks
  const uint32_t s1 = min(runs, (wave + 1) * per);
  bool quantised = MX;
  for (uint32_t s = wave * per; !quantised || s < s1; s += U) {
    uint4 wq[U], xq[U][MT];
    uint32_t ws[U], xs[U][MT];
#pragma unroll
    for (int u = 0; u < U; ++u) {   // (a run or block that does not exist reads the row's first block and is masked below)
      const uint32_t blk = s + u < s1 && 4 * (s + u) + lg < p.kb ? 4 * (s + u) + lg : 0u;
      wq[u] = *reinterpret_cast<const uint4*>(bc + (size_t)blk * 16);
      ws[u] = bsc[blk];
      if constexpr (MX) {
#pragma unroll
        for (int t = 0; t < MT; ++t) {
          xq[u][t] = *reinterpret_cast<const uint4*>((const uint8_t*)p.a + (size_t)arow[t] * p.a_ld + (size_t)blk * 16);
          xs[u][t] = p.as[(size_t)arow[t] * p.as_ld + blk];
        }
      }
    }
    if constexpr (!MX) {
      if (!quantised) {
        typedef typename MxIn<AT>::T T;
        for (uint32_t e = threadIdx.x; e < m * p.kb; e += blockDim.x) {
          const uint32_t row = e / p.kb, b = e - row * p.kb;
          uint32_t sc;
          xcodes[e] = mx_quantize_block_dev<AT>((const T*)p.a + (size_t)row * p.a_ld, b, p.k, &sc);
          xscales[e] = (uint8_t)sc;
        }
        __syncthreads();
        quantised = true;
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const bool in = s + u < s1 && 4 * (s + u) + lg < p.kb;
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        if constexpr (!MX) {
          const uint32_t e = arow[t] * p.kb + (in ? 4 * (s + u) + lg : 0u);
          xq[u][t] = xcodes[e];
          xs[u][t] = xscales[e];
        }
        acc[t] = mx_mma16(wq[u], in ? ws[u] : 0u, xq[u][t], in ? xs[u][t] : 0u, acc[t]);
      }
    }
  }
#pragma unroll
  for (int t = 0; t < MT; ++t)
#pragma unroll
    for (int j = 0; j < 4; ++j) part[wave][t][lane][j] = acc[t][j];
  __syncthreads();
  // element = (row, channel), channels fastest: channel 4 g + j of row 16 t + r is element j of lane 16 g + r of tile t
  for (uint32_t q = threadIdx.x; q < 256u * MT; q += blockDim.x) {
    const uint32_t i = q / 16, ch = q % 16;
    if (i >= m || n0 + ch >= p.n) continue;
    float y = 0.f;
    for (int w = 0; w < waves; ++w) y += part[w][i / 16][(ch / 4) * 16 + i % 16][ch % 4];
    product_store(p, i, n0 + ch, y);
  }
}

// Bias, ReLU, residual and store of 8 consecutive channels of one row, from LDS (one 16-byte store in fp16, two in fp32;
// rows of any alignment).  `pre`: the fp16 residual, if there is one.  STREAM: see whole_lines.
template <bool STREAM>
__device__ __forceinline__ void product_store8(const ProductArgs& p, uint32_t i, uint32_t j, const float* src, const v4u pre) {
  if (j + 8 > p.n) {
#pragma unroll 1
    for (uint32_t q = 0; j + q < p.n; ++q) product_store(p, i, j + q, src[q]);
    return;
  }
  float y[8];
  *reinterpret_cast<v4f*>(y) = *reinterpret_cast<const v4f*>(src);
  *reinterpret_cast<v4f*>(y + 4) = *reinterpret_cast<const v4f*>(src + 4);
  if (p.bias) {
    if (p.bias_fp32) {
      float b[8];
      __builtin_memcpy(b, (const float*)p.bias + j, 32);
#pragma unroll
      for (int q = 0; q < 8; ++q) y[q] += b[q];
    } else {
      _Float16 b[8];
      __builtin_memcpy(b, (const _Float16*)p.bias + j, 16);
#pragma unroll
      for (int q = 0; q < 8; ++q) y[q] += (float)b[q];
    }
  }
  if (p.relu) {
#pragma unroll
    for (int q = 0; q < 8; ++q) y[q] = product_relu(y[q]);
  }
  if (p.res) {
    if (p.res_fp32) {
      float r[8];
      __builtin_memcpy(r, (const float*)p.res + (size_t)i * p.res_ld + j, 32);
#pragma unroll
      for (int q = 0; q < 8; ++q) y[q] += r[q];
    } else {
      _Float16 r[8];
      __builtin_memcpy(r, &pre, 16);
#pragma unroll
      for (int q = 0; q < 8; ++q) y[q] += (float)r[q];
    }
  }
  if (p.relu2) {
#pragma unroll
    for (int q = 0; q < 8; ++q) y[q] = product_relu(y[q]);
  }
  const size_t at = (size_t)i * p.out_ld + j;
  if (p.out_fp32) {
    store16<STREAM>((float*)p.out + at, y);
    store16<STREAM>((float*)p.out + at + 4, y + 4);
  } else {
    _Float16 h[8];
#pragma unroll
    for (int q = 0; q < 8; ++q) h[q] = (_Float16)y[q];
    store16<STREAM>((_Float16*)p.out + at, h);
  }
}

// Any number of rows.  A workgroup owns BN output channels x BM rows, a wave of it TN x TM tiles of 32 x 32; both operands are
// staged through LDS, 256 channels (8 blocks = 128 code bytes) at a time, by loads that go straight to LDS, two stages deep.
//   LDS of a stage: codes of the BN weight rows, then of the BM rows (128 bytes each).  Block c of row r lies at position
//   c ^ (r / 2) % 8 of its row, so that the 16-byte operand reads of 16 neighbouring rows touch all 64 banks once.  The hardware
//   places lane l's bytes at base + 16 l, so the order is obtained by permuting which block a lane fetches.
//   Scales are fetched for 2 stages at once (16 bytes per row), two such spans.
// What bounds it is the memory pipe next to the matrix cores: it counts requests, a line of 128 bytes as much as 4 bytes of one,
// so codes come in whole lines and scales in spans.  (8192 cubed with 64-byte code rows and scales word by word: 350 us;
// 64-byte rows and spans: 291 us.)
// The last operands of a stage are multiplied behind the barrier in front of the next one, while that one's first operands are
// read, so the matrix pipe does not wait for LDS there.
//   Per matrix instruction of 64 channels a wave reads (TN + TM) KB / (TN * TM) from LDS.
// Rows beyond the last are read as the last one and not stored.
typedef __attribute__((address_space(3))) void* mx_lptr;

// 64 x 16 (or 64 x 4) bytes from memory to LDS, lane l's to base + 16 l (4 l).  Written in assembly so that the compiler's
// own LDS reads are not ordered after every load in flight (it would drain them all); the waits are the explicit counts
// in the kernel.  The address is a wave's base with a 32-bit offset per lane.  The instruction takes its LDS address from m0,
// which needs one wait state after it is written.
__device__ __forceinline__ void mx_load16_lds(const uint8_t* src, uint32_t offset, uint32_t base) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(offset), "s"(src), "s"(base) : "m0", "memory");
}
__device__ __forceinline__ void mx_load4_lds(const uint8_t* src, uint32_t offset, uint32_t base) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dword %0, %1" ::"v"(offset), "s"(src), "s"(base) : "m0", "memory");
}

// (the byte of the scale registers is an immediate of the instruction)
template <int SEL>
__device__ __forceinline__ v16f mx_mma32_sel(const v4i& a, uint32_t sa, const v4i& b, uint32_t sb, v16f c) {
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(v8i{a[0], a[1], a[2], a[3], 0, 0, 0, 0}, v8i{b[0], b[1], b[2], b[3], 0, 0, 0, 0},
                                                         c, 4, 4, SEL, (int)sa, SEL, (int)sb);
}

// KS > 1: as many groups of waves share a tile, each with a run of the stages and LDS of its own, and add their sums when the
// tile is stored: a few tiles down a long k are bound by the latency of a stage (0.37 us), of which KS then pass at a time
// (100 x 100 x 8192: 14.1 us with one group, 11.3 us with 2, 10.5 us with 4).  The order of the sums is fixed.
template <int BN, int BM, int TN, int TM, int KS>
struct ProductTile {
  static constexpr int WN = BN / (32 * TN), WM = BM / (32 * TM), WAVES = WN * WM;
  static constexpr int STAGE = (BN + BM) * 128, SPAN = (BN + BM) * 16;   // bytes of LDS per stage of codes, per span of scales
  static constexpr int PAD = 32 * TN + 4;                             // floats per row of the store buffer
  static constexpr int STORE = WAVES * 32 * PAD * 4;
  static_assert(KS == 1 || (TN == 1 && TM == 1), "split sums are added tile by tile");
  // bytes of LDS of a group that runs through `stages` stages
  __host__ __device__ static uint32_t lds(uint32_t stages) {
    const uint32_t need = (stages > 1 ? 2 : 1) * STAGE + (stages > 2 ? 2 : 1) * SPAN;
    return need > (uint32_t)STORE ? need : (uint32_t)STORE;
  }
  // stages of a group (whole spans of scales) when all have `stages`
  __host__ __device__ static uint32_t share(uint32_t stages) { return KS == 1 ? stages : ((stages + KS - 1) / KS + 1) / 2 * 2; }
};

template <int BN, int BM, int TN, int TM, int KS>
constexpr int kProductThreads = 64 * ProductTile<BN, BM, TN, TM, KS>::WAVES * KS;

template <int BN, int BM, int TN, int TM, int KS, bool STREAM>
__global__ __launch_bounds__((kProductThreads<BN, BM, TN, TM, KS>), 2) void k_mx_product_lds(const ProductArgs p, uint32_t tiles_n,
                                                                                              uint32_t tiles_m) {
  using T = ProductTile<BN, BM, TN, TM, KS>;
  constexpr int WAVES = T::WAVES, STAGE = T::STAGE, SPAN = T::SPAN;
  constexpr int LOADS = (BN + BM) / 8 / WAVES;   // wave loads per stage of codes
  static_assert(LOADS * 8 * WAVES == BN + BM && BN % (WAVES * 8) == 0 && WAVES % 2 == 0 && BN % 64 == 0 && BN + BM <= WAVES * 64,
                "a wave's load is all weights or all rows, and one load per wave fetches a span of scales");
  extern __shared__ __align__(16) char lds[];
  const int lane = threadIdx.x & 63, wave_all = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wave = wave_all % WAVES, group = wave_all / WAVES;
  const int ln = lane & 31, lh = lane >> 5;
  const uint32_t m = eff_n(p.m_dev, p.m);
  // XCD x takes the x-th contiguous eighth of the tiles (each XCD has its own L2), in bands of 8 row tiles that are walked
  // channel tile by channel tile, so that the tiles in flight on an XCD form a rectangle and share operands
  const uint32_t total = tiles_n * tiles_m, per = (total + 7) / 8;
  const uint32_t t = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
  if ((blockIdx.x >> 3) >= per || t >= total) return;
  const uint32_t band = t / (8 * tiles_n), in_band = t - band * 8 * tiles_n;
  const uint32_t rows_in_band = min(8u, tiles_m - band * 8);
  const uint32_t tm = band * 8 + in_band % rows_in_band, tn = in_band / rows_in_band;
  const uint32_t i0 = tm * BM, n0 = tn * BN;
  if (i0 >= m) return;

  // What this lane fetches: code load q covers 8 rows (lane / 8), position lane % 8; the scale load 64 rows.  A wave's load is
  // all weights or all rows, so an address is a wave's base, which advances from stage to stage, and a lane's offset.
  uint32_t coff[LOADS];
  // this group's run of blocks: kb of them from `first` on (none, for the last groups, when there are few)
  const uint32_t all = (p.kb + 7) / 8, share = T::share(all), first = min(group * share * 8, p.kb);
  const uint32_t kb = min(p.kb - first, share * 8);
  const uint8_t* wcode = p.b + (size_t)n0 * p.b_ld + (size_t)first * 16;
  const uint8_t* xcode = (const uint8_t*)p.a + (size_t)i0 * p.a_ld + (size_t)first * 16;
  const uint32_t last_w = p.n - 1 - n0, last_x = m - 1 - i0;   // rows of this tile that exist
  const uint32_t cblk = (lane & 7) ^ ((wave * 4 + (lane >> 4)) & 7);   // block of a stage this lane fetches
#pragma unroll
  for (int q = 0; q < LOADS; ++q) {
    const uint32_t r = q * WAVES * 8 + wave * 8 + (lane >> 3);
    coff[q] = (q * WAVES * 8 < BN ? min(r, last_w) * p.b_ld : min(r - BN, last_x) * p.a_ld) + cblk * 16;
  }
  const uint32_t srow = (wave * 64) % (BN + BM);               // (the small tile has fewer rows than lanes: some are loaded twice)
  const bool s_is_w = srow < BN;
  const uint8_t* sbase = (s_is_w ? p.bs + (size_t)n0 * p.bs_ld : p.as + (size_t)i0 * p.as_ld) + first;
  const uint32_t s_ld = s_is_w ? p.bs_ld : p.as_ld, srow0 = s_is_w ? srow : srow - BN, last_s = s_is_w ? last_w : last_x;
  const uint32_t soff = min(srow0 + lane, last_s) * s_ld;
  const uint32_t stages = (kb + 7) / 8, words = (kb + 3) / 4;   // stages of 8 blocks, scale words of 4; the last may be shorter
  const uint32_t most = min(share, all);                        // stages of the first group
  char* const lds_g = lds + (KS > 1 ? group * T::lds(most) : 0);
  const uint32_t base = (uint32_t)(uintptr_t)(mx_lptr)lds_g;
  const uint32_t span0 = (most > 1 ? 2 : 1) * STAGE;            // LDS offset of the scales
  // Loads [from, to) of a wave's LOADS of stage st.  In a stage of fewer than 8 blocks a lane whose block does not exist
  // fetches the first one instead: the masked scales (2^-127 on both sides) take it out of the sums.
  auto load = [&](uint32_t st, int from, int to) {
    const uint32_t buf = __builtin_amdgcn_readfirstlane(base + (st & 1) * STAGE);
    const uint32_t back = st * 8 + cblk < kb ? 0u : cblk * 16;
#pragma unroll
    for (int q = 0; q < LOADS; ++q)
      if (q >= from && q < to)
        mx_load16_lds((q * WAVES * 8 < BN ? wcode : xcode) + (size_t)st * 128, coff[q] - back, buf + (q * WAVES + wave) * 1024);
  };
  // Scales of stages 2 t and 2 t + 1: 16 bytes per row in one load, or word by word (4 loads, 16 rows x 4 words each) when the
  // rows end inside the span; words that do not exist are read as the span's first and never used.
  auto load_scales = [&](uint32_t t) {
    const uint32_t buf = __builtin_amdgcn_readfirstlane(base + span0 + (t & 1) * SPAN + srow * 16);
    if (4 * t + 4 <= words) {
      mx_load16_lds(sbase + (size_t)t * 16, soff, buf);
    } else if (4 * t < words) {
      const uint32_t word = 4 * t + (lane & 3) < words ? (lane & 3) * 4 : 0u;
#pragma unroll
      for (int q = 0; q < 4; ++q)
        mx_load4_lds(sbase + (size_t)t * 16, min(srow0 + q * 16 + (lane >> 2), last_s) * s_ld + word, buf + q * 256);
    }
  };

  v16f acc[TN][TM];
#pragma unroll
  for (int a = 0; a < TN; ++a)
#pragma unroll
    for (int b = 0; b < TM; ++b)
#pragma unroll
      for (int j = 0; j < 16; ++j) acc[a][b][j] = 0.f;

  const int wn = wave % T::WN, wm = wave / T::WN;
  const uint32_t w_row = wn * 32 * TN + ln, x_row = BN + wm * 32 * TM + ln;
  const uint32_t swz = (ln >> 1) & 7;
  v4i w[2][TN], x[2][TM];
  uint2 ws[TN], xs[TM], ws1[TN], xs1[TM];
  // operands of step S (64 channels) of stage st
  auto read = [&](uint32_t st, int S, v4i(&wv)[TN], v4i(&xv)[TM]) {
    const char* sb = lds_g + (st & 1) * STAGE;
    const uint32_t pos = ((2 * S + lh) ^ swz) * 16;
#pragma unroll
    for (int a = 0; a < TN; ++a) wv[a] = *reinterpret_cast<const v4i*>(sb + (w_row + 32 * a) * 128 + pos);
#pragma unroll
    for (int b = 0; b < TM; ++b) xv[b] = *reinterpret_cast<const v4i*>(sb + (x_row + 32 * b) * 128 + pos);
  };
  // the scale words of a stage; take_scales: blocks 2 s + lh of step s are bytes 0 and 2 of the words after a shift by lh bytes
  auto read_scales = [&](uint32_t st) {
    const char* sb = lds_g + span0 + ((st >> 1) & 1) * SPAN + (st & 1) * 8;
#pragma unroll
    for (int a = 0; a < TN; ++a) ws1[a] = *reinterpret_cast<const uint2*>(sb + (w_row + 32 * a) * 16);
#pragma unroll
    for (int b = 0; b < TM; ++b) xs1[b] = *reinterpret_cast<const uint2*>(sb + (x_row + 32 * b) * 16);
  };
  auto take_scales = [&](uint32_t mask0, uint32_t mask1) {
#pragma unroll
    for (int a = 0; a < TN; ++a) ws[a] = make_uint2((ws1[a].x & mask0) >> (8 * lh), (ws1[a].y & mask1) >> (8 * lh));
#pragma unroll
    for (int b = 0; b < TM; ++b) xs[b] = make_uint2((xs1[b].x & mask0) >> (8 * lh), (xs1[b].y & mask1) >> (8 * lh));
  };
#define SCN_MX_MULTIPLY(BUF, SEL, WORD)                                                            \
  _Pragma("unroll") for (int a = 0; a < TN; ++a) _Pragma("unroll") for (int b = 0; b < TM; ++b)    \
      acc[a][b] = mx_mma32_sel<SEL>(w[BUF][a], ws[a].WORD, x[BUF][b], xs[b].WORD, acc[a][b]);
// every load has landed and every wave is done with the other buffer (its operands are in registers)
#define SCN_MX_BARRIER()                                                  \
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");             \
  __builtin_amdgcn_s_barrier();                                           \
  asm volatile("" ::: "memory");
  // Steps 0 .. 3 of every stage but the last; the products of a stage's step 3 come behind the next barrier (none before the
  // first: zeros).
#pragma unroll
  for (int a = 0; a < TN; ++a) w[1][a] = v4i{0, 0, 0, 0}, ws[a] = make_uint2(0, 0);
#pragma unroll
  for (int b = 0; b < TM; ++b) x[1][b] = v4i{0, 0, 0, 0}, xs[b] = make_uint2(0, 0);
  uint32_t st = 0;
  if (KS == 1 || stages > 0) {
    load_scales(0);
    load(0, 0, LOADS);
  }
#pragma unroll 1
  for (; st + 1 < stages; ++st) {
    SCN_MX_BARRIER()
    if (!(st & 1)) load_scales(st / 2 + 1);
    read_scales(st);
    read(st, 0, w[0], x[0]);
    __builtin_amdgcn_sched_barrier(0);
    load(st + 1, 0, LOADS / 2);
    SCN_MX_MULTIPLY(1, 2, y)
    take_scales(~0u, ~0u);
    __builtin_amdgcn_sched_barrier(0);
    read(st, 1, w[1], x[1]);
    __builtin_amdgcn_sched_barrier(0);
    load(st + 1, LOADS / 2, LOADS);
    SCN_MX_MULTIPLY(0, 0, x)
    __builtin_amdgcn_sched_barrier(0);
    read(st, 2, w[0], x[0]);
    __builtin_amdgcn_sched_barrier(0);
    SCN_MX_MULTIPLY(1, 2, x)
    __builtin_amdgcn_sched_barrier(0);
    read(st, 3, w[1], x[1]);
    __builtin_amdgcn_sched_barrier(0);
    SCN_MX_MULTIPLY(0, 0, y)
  }
  SCN_MX_MULTIPLY(1, 2, y)
  // What this lane will store, and the fp16 residual it needs there: fetched while the last stage travels where the
  // accumulators leave registers for it, else 32 rows at a time in front of their stores.
  constexpr int LPR = 4 * TN, RPP = 64 / LPR, PASSES = 32 / RPP;   // lanes per row (8 channels each), rows per pass
  constexpr bool EARLY = TN * TM <= 4;
  const uint32_t row0 = i0 + wm * 32 * TM + lane / LPR, ch = n0 + wn * 32 * TN + (lane % LPR) * 8;
  v4u pre[EARLY ? TM * PASSES : PASSES];
  auto residual = [&](int b, int to) {
    const bool want = p.res && !p.res_fp32 && ch + 8 <= p.n;
#pragma unroll
    for (int r = 0; r < PASSES; ++r) {
      pre[to + r] = v4u{0, 0, 0, 0};
      const uint32_t row = row0 + (b * PASSES + r) * RPP;
      if (want && row < m) __builtin_memcpy(&pre[to + r], (const _Float16*)p.res + (size_t)row * p.res_ld + ch, 16);
    }
  };
  if constexpr (EARLY)
#pragma unroll
    for (int b = 0; b < TM; ++b) residual(b, b * PASSES);
  if (KS == 1 || stages > 0) {   // the last stage, of 1 .. 8 blocks
    SCN_MX_BARRIER()
    const uint32_t left = kb - st * 8;
    read_scales(st);
    take_scales(left >= 4 ? ~0u : (1u << (8 * left)) - 1u, left >= 8 ? ~0u : left > 4 ? (1u << (8 * (left - 4))) - 1u : 0u);
    read(st, 0, w[0], x[0]);
    SCN_MX_MULTIPLY(0, 0, x)
    if (left > 2) {
      read(st, 1, w[0], x[0]);
      SCN_MX_MULTIPLY(0, 2, x)
    }
    if (left > 4) {
      read(st, 2, w[0], x[0]);
      SCN_MX_MULTIPLY(0, 0, y)
    }
    if (left > 6) {
      read(st, 3, w[0], x[0]);
      SCN_MX_MULTIPLY(0, 2, y)
    }
  }
#undef SCN_MX_MULTIPLY
#undef SCN_MX_BARRIER
  if constexpr (KS > 1)
    for (uint32_t i = stages; i < most; ++i) __builtin_amdgcn_s_barrier();   // (one per stage of the first group)
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  // Store through LDS (wave-private, 32 rows at a time): a lane of the accumulators holds 4 consecutive channels of one
  // row, a store wants whole 128-byte lines of a row.
  float* buf = reinterpret_cast<float*>(KS > 1 ? lds_g : lds) + wave * 32 * T::PAD;
#pragma unroll
  for (int b = 0; b < TM; ++b) {
    if constexpr (!EARLY) residual(b, 0);
#pragma unroll
    for (int a = 0; a < TN; ++a)
#pragma unroll
      for (int q = 0; q < 4; ++q)
        *reinterpret_cast<v4f*>(buf + ln * T::PAD + a * 32 + q * 8 + lh * 4) =
            v4f{acc[a][b][4 * q], acc[a][b][4 * q + 1], acc[a][b][4 * q + 2], acc[a][b][4 * q + 3]};
    if constexpr (KS > 1) __syncthreads();
#pragma unroll
    for (int r = 0; r < PASSES; ++r) {
      const uint32_t row = row0 + (b * PASSES + r) * RPP;
      if (row >= m || ch >= p.n || r % KS != group) continue;
      float* src = buf + (r * RPP + lane / LPR) * T::PAD + (lane % LPR) * 8;
      if constexpr (KS > 1) {   // the groups' sums, in their order; each pass is one group's to store
        v4f y[2] = {v4f{0.f, 0.f, 0.f, 0.f}, v4f{0.f, 0.f, 0.f, 0.f}};
        for (int g = 0; g < KS; ++g) {
          const float* part = src + ((int)g - group) * (int)(T::lds(most) / 4);
          y[0] += *reinterpret_cast<const v4f*>(part);
          y[1] += *reinterpret_cast<const v4f*>(part + 4);
        }
        reinterpret_cast<v4f*>(src)[0] = y[0];
        reinterpret_cast<v4f*>(src)[1] = y[1];
      }
      product_store8<STREAM>(p, row, ch, src, pre[(EARLY ? b * PASSES : 0) + r]);
    }
  }
}

static size_t product_workspace(uint32_t m, uint32_t n, uint32_t k);   // 0: rows of fp16 / fp32 need none

// What comes in front of a product's launch, once its kernel has taken the sizes: no operand lies where the call writes, and rows
// that go through the workspace (p.a is that then) are quantised into it.
static int product_start(const ProductArgs& p, const scn_mx_product_io& io, hipStream_t stream) {
  const auto size = [](int dtype) -> uint64_t { return dtype == SCN_DTYPE_FP32 ? 4 : 2; };
  const uint64_t codes = (uint64_t)p.kb * kMxBlockBytes, scales = mx_scale_bytes(p.k);
  const bool mx = io.a_dtype == SCN_DTYPE_MXFP4, quantise = !mx && product_workspace(io.m, io.n, io.k) != 0;
  const MxSpan out{io.out_dev, io.m, io.n * size(io.out_dtype), io.out_ld * size(io.out_dtype)},
      ws{quantise ? p.a : nullptr, 1, (uint64_t)io.m * p.a_ld, 0},
      res{io.res_dev, io.m, io.n * size(io.res_dtype), io.res_ld * size(io.res_dtype)};
  const MxSpan read[] = {{io.a_dev, io.m, mx ? codes : io.k * size(io.a_dtype), mx ? io.a_ld : io.a_ld * size(io.a_dtype)},
                         {mx ? io.a_scales_dev : nullptr, io.m, scales, io.a_scales_ld},
                         {io.b_codes_dev, io.n, codes, io.b_codes_ld},
                         {io.b_scales_dev, io.n, scales, io.b_scales_ld},
                         {io.bias_dev, 1, io.n * size(io.bias_dtype), 0},
                         {io.m_dev, 1, 4, 0}};
  for (const MxSpan& r : read)
    SCN_REQUIRE(!mx_overlap(out, r) && !mx_overlap(ws, r), SCN_ERR_INVALID,
                "mx_product: the output and the workspace must not overlap the rows, the weights, the bias or the count");
  SCN_REQUIRE(io.res_dev == io.out_dev || !mx_overlap(out, res), SCN_ERR_INVALID,
              "mx_product: the output must be the residual or not overlap it");
  SCN_REQUIRE(!mx_overlap(ws, out) && !mx_overlap(ws, res), SCN_ERR_INVALID,
              "mx_product: the workspace must not overlap the output or the residual");
  if (!quantise) return SCN_OK;
  return mx_quantize_rows(io.a_dev, io.a_dtype, io.k, io.a_ld, 0.f, 0, static_cast<uint8_t*>(io.workspace_dev), p.a_ld,
                          const_cast<uint8_t*>(p.as), p.as_ld, io.m, io.m_dev, stream);
}

// Rows of a tile lie at 32-bit offsets from its first one.
static bool product_near(const ProductArgs& p) {
  return (uint64_t)std::max(std::max(p.a_ld, p.b_ld), std::max(p.as_ld, p.bs_ld)) * 256 < (1ull << 32);
}

// Streaming or ordinary stores of a product's output.  Streaming ones keep the write-back L2 out of the way, but an L2 that they pass
// cannot join parts of a 128-byte line: an fp32 store of 8 channels is two halves of 16 of every 32 bytes, and rows that are not whole
// lines begin and end inside one.  us streaming | ordinary:
//   fp16, tiled kernels: 8192 x 8192 x 2048 94 | 111, 8192 x 8190 x 2048 110 | 125, 20000 x 1000 x 1000 33.8 | 34.8, 100000 x 128 x 300
//     14.0 | 19.9, 100000 x 100 x 300 17.2 | 20.3: streaming;
//   fp32, tiles of 128 and 256: 8192 x 8192 x 2048 167 | 129, 20000 x 1024 x 1000 53 | 41, 20000 x 500 x 1000 33.7 | 32.8: ordinary;
//   fp32, tiles of 64: 100000 x 128 x 300 17.9 | 25.5, 2000 x 1024 x 300 5.6 | 6.1, but 2000 x 1000 x 300 8.1 | 6.5: by whole lines;
//   quantised in the same launch, fp16: up to 4 blocks 123646 x 256 x 128 22.6 | 28.5, but 123646 x 250 x 128 46.5 | 34.0 and 20000 x
//     1000 x 100 25.8 | 22.6: by whole lines; more blocks 60000 x 250 x 250 24.9 | 28.3: streaming;
//   quantised in the same launch, fp32: 123646 x 250 x 128 92 | 47, 60000 x 250 x 250 41.8 | 33.8: by whole lines; with them 60000 x 128 x
//     256 17.6 | 21.1, 123646 x 96 x 64 17.9 | 21.5, but in the wide tiles of more than 128 channels 123646 x 256 x 128 53 | 41 and
//     20000 x 512 x 100 20.3 | 17.1 (5000 x 1024 x 128, which the L2 holds, 10.2 | 11.3).
static bool whole_lines(const ProductArgs& p) {
  const size_t size = p.out_fp32 ? 4 : 2;
  return ((uintptr_t)p.out | (size_t)p.out_ld * size | (size_t)p.n * size) % 128 == 0;
}

template <int BN, int BM, int TN, int TM, int KS>
static int launch_product(const ProductArgs& p, const scn_mx_product_io& io, hipStream_t stream) {
  using T = ProductTile<BN, BM, TN, TM, KS>;
  const uint64_t tn = ((uint64_t)p.n + BN - 1) / BN, tm = ((uint64_t)p.m + BM - 1) / BM;
  SCN_REQUIRE(product_near(p), SCN_ERR_UNSUPPORTED, "mx_product: rows more than 16 MB apart");
  constexpr uint64_t threads = 64 * T::WAVES * KS;   // (a launch has fewer than 2^32 threads)
  SCN_REQUIRE((tn * tm + 7) / 8 * 8 * threads < (1ull << 32), SCN_ERR_UNSUPPORTED, "mx_product: %u x %u outputs are too many for one call",
              p.m, p.n);
  if (int rc = product_start(p, io, stream)) return rc;
  const uint32_t stages = (p.kb + 7) / 8;
  const auto launch = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3((unsigned)((tn * tm + 7) / 8 * 8)), dim3((unsigned)threads),
                       KS * T::lds(std::min(T::share(stages), stages)), stream, p, (uint32_t)tn, (uint32_t)tm);
  };
  if (!p.out_fp32 || (BN == 64 && whole_lines(p))) launch(k_mx_product_lds<BN, BM, TN, TM, KS, true>);
  else launch(k_mx_product_lds<BN, BM, TN, TM, KS, false>);
  return SCN_OK;
}

// Rows that are not quantised yet, of up to P blocks (P = 2, 4 or 8), times up to a few hundred channels: bound by the rows, the
// residual and the output.  A workgroup owns BM rows x 64 WN channels, a wave TM tiles of 32 rows x 64 channels.  Everything it
// reads is requested at the start: the weights straight to LDS (see above for the order of their blocks), the rows and the
// residual to registers; the rows are quantised into LDS in the operands' order, and one barrier later multiplied.
// (123,646 x 256 x 128, fp16 rows and residual: 34.9 us, 4.5 TB/s of what it cannot do without.)
template <int AT, int WN, int P>
struct FusedTile {
  // 8 waves share the quantisation of long rows; where the tile has fewer outputs than waves, the others do no more
  static constexpr int NW = P == 8 ? 8 : 4, WM = P == 8 ? 2 : 4 / WN, TM = P == 8 || WN < 4 ? 1 : 2, BM = 32 * TM * WM;
  static constexpr int XS = BM * P * 16, WC = XS + BM * 8;           // LDS offsets: codes of the rows, their scales, weights
  static constexpr int PAD = 68, STORE = WN * WM * 32 * PAD * 4;       // floats per row of the store buffer, its bytes
  static constexpr int LDS = WC + WN * 64 * P * 16 > STORE ? WC + WN * 64 * P * 16 : STORE;
};

template <int AT, int WN, int P, bool STREAM>
__global__ __launch_bounds__((64 * FusedTile<AT, WN, P>::NW)) void k_mx_product_fused(const ProductArgs p) {
  using F = FusedTile<AT, WN, P>;
  typedef typename MxIn<AT>::T T;
  constexpr int TM = F::TM, BM = F::BM, NW = F::NW, E = 16 / (int)sizeof(T), LPB = 32 / E, WORDS = (P + 3) / 4;
  __shared__ __align__(16) char lds[F::LDS];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), ln = lane & 31, lh = lane >> 5;
  const int wn = wave % WN, wm = wave / WN;
  const uint32_t m = eff_n(p.m_dev, p.m);
  const uint32_t i0 = blockIdx.x * BM, n0 = blockIdx.y * 64 * WN;
  if (i0 >= m) return;
  const uint32_t last_w = p.n - 1 - n0;
  auto swizzle = [](uint32_t row) { return row / (16 / P) % P; };

  const uint32_t base = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(mx_lptr)lds);
  const uint8_t* wcode = p.b + (size_t)n0 * p.b_ld;
#pragma unroll
  for (int u = 0; u < (WN * P + NW - 1) / NW; ++u) {
    const int unit = u * NW + wave;
    if (unit < WN * P) {   // 64 of the P * 64 * WN chunks of weights
      const uint32_t e = unit * 64 + lane, r = e / P, blk = (e % P) ^ swizzle(r);
      mx_load16_lds(wcode, min(r, last_w) * p.b_ld + (blk < p.kb ? blk * 16 : 0u), base + F::WC + unit * 1024);
    }
  }
  uint32_t ws[2][WORDS];
#pragma unroll
  for (int a = 0; a < 2; ++a)
#pragma unroll
    for (int q = 0; q < WORDS; ++q) {
      const uint8_t* row = p.bs + (size_t)(n0 + min((uint32_t)(wn * 64 + a * 32 + ln), last_w)) * p.bs_ld;
      const uint32_t left = p.kb > 4u * q ? p.kb - 4 * q : 0u;
      ws[a][q] = left ? *reinterpret_cast<const uint32_t*>(row + 4 * q) & (left >= 4 ? ~0u : (1u << (8 * left)) - 1u) : 0u;
    }
  constexpr int LPR = 8, RPP = 8, PASSES = 4;   // lanes per row (8 channels each), rows per pass, passes per 32 rows
  const uint32_t row0 = i0 + wm * 32 * TM + lane / LPR, ch = n0 + wn * 64 + (lane % LPR) * 8;
  v4u pre[TM * PASSES];
  const bool works = wave < WN * F::WM, want = works && p.res && !p.res_fp32 && ch + 8 <= p.n;
#pragma unroll
  for (int q = 0; q < TM * PASSES; ++q) {
    pre[q] = v4u{0, 0, 0, 0};
    const uint32_t row = row0 + q * RPP;
    if (want && row < m) __builtin_memcpy(&pre[q], (const _Float16*)p.res + (size_t)row * p.res_ld + ch, 16);
  }

  constexpr int PIECES = BM * P * LPB / (64 * NW), BATCH = PIECES < 16 ? PIECES : 16;   // pieces of 16 bytes per thread
#pragma unroll 1
  for (int i = 0; i < PIECES; i += BATCH) {
    // whole pieces are requested all at once (other lanes read the tile's first one); a row's last one, if it is short, later
    T raw[BATCH][E];
    if (p.k >= (uint32_t)E) {
#pragma unroll
      for (int z = 0; z < BATCH; ++z) {
        const uint32_t e = (i + z) * 64 * NW + threadIdx.x, at = e / LPB % P * 32 + e % LPB * E, row = i0 + e / (LPB * P);
        const bool whole = at + E <= p.k && row < m;
        __builtin_memcpy(raw[z], (const T*)p.a + (whole ? (size_t)row * p.a_ld + at : (size_t)i0 * p.a_ld), 16);
      }
    }
#pragma unroll
    for (int z = 0; z < BATCH; ++z) {
      const uint32_t e = (i + z) * 64 * NW + threadIdx.x, sub = e % LPB, blk = e / LPB % P, row = e / (LPB * P), at = blk * 32 + sub * E;
      const bool whole = at + E <= p.k && i0 + row < m;
      float v[E];
#pragma unroll
      for (int j = 0; j < E; ++j) v[j] = whole ? (float)raw[z][j] : 0.f;
      if (!whole && at < p.k && i0 + row < m) mx_load<AT, E>((const T*)p.a + (size_t)(i0 + row) * p.a_ld, at, p.k, 1.f, 0, v);
      uint32_t top = 0;
#pragma unroll
      for (int j = 0; j < E; ++j) top = max(top, __float_as_uint(v[j]) & 0x7FFFFFFFu);
      top = lanes_max<LPB>(top);
      const uint32_t sc = mx_scale_byte(top);
      const float up = __uint_as_float((254u - (sc == 255u ? 0u : sc)) << 23);
      char* dst = lds + (row * P + (blk ^ swizzle(row))) * 16 + sub * (E / 2);
      if constexpr (E == 8) {
        *reinterpret_cast<uint32_t*>(dst) = sc == 255u ? 0u : mx_codes8(v, up);
      } else {
        uint32_t w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, v[0] * up, v[1] * up, 1.f, 0);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[2] * up, v[3] * up, 1.f, 1);
        *reinterpret_cast<uint16_t*>(dst) = sc == 255u ? (uint16_t)0 : (uint16_t)w;
      }
      if (sub == 0) *reinterpret_cast<uint8_t*>(lds + F::XS + row * 8 + blk) = blk < p.kb ? (uint8_t)sc : (uint8_t)0;
    }
  }
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");   // (the weights too)
  __syncthreads();

  v16f acc[2][TM];
  if (works) {
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
      for (int b = 0; b < TM; ++b)
#pragma unroll
        for (int j = 0; j < 16; ++j) acc[a][b][j] = 0.f;
#pragma unroll
    for (int s = 0; s < P / 2; ++s) {   // 64 channels; blocks that do not exist have scales of 2^-127 on both sides
      const uint32_t pos = ((2 * s + lh) ^ swizzle(ln)) * 16;
      v4i w[2], x[TM];
      uint32_t xs[TM];
#pragma unroll
      for (int a = 0; a < 2; ++a) w[a] = *reinterpret_cast<const v4i*>(lds + F::WC + (wn * 64 + a * 32 + ln) * P * 16 + pos);
#pragma unroll
      for (int b = 0; b < TM; ++b) {
        const uint32_t row = (wm * TM + b) * 32 + ln;
        x[b] = *reinterpret_cast<const v4i*>(lds + row * P * 16 + pos);
        xs[b] = *reinterpret_cast<const uint32_t*>(lds + F::XS + row * 8 + s / 2 * 4) >> (8 * lh);
      }
#pragma unroll
      for (int a = 0; a < 2; ++a)
#pragma unroll
        for (int b = 0; b < TM; ++b)
          acc[a][b] = s & 1 ? mx_mma32_sel<2>(w[a], ws[a][s / 2] >> (8 * lh), x[b], xs[b], acc[a][b])
                            : mx_mma32_sel<0>(w[a], ws[a][s / 2] >> (8 * lh), x[b], xs[b], acc[a][b]);
    }
  }
  __syncthreads();
  if (!works) return;
  // store through LDS as above
  float* buf = reinterpret_cast<float*>(lds) + wave * 32 * F::PAD;
#pragma unroll
  for (int b = 0; b < TM; ++b) {
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
      for (int q = 0; q < 4; ++q)
        *reinterpret_cast<v4f*>(buf + ln * F::PAD + a * 32 + q * 8 + lh * 4) =
            v4f{acc[a][b][4 * q], acc[a][b][4 * q + 1], acc[a][b][4 * q + 2], acc[a][b][4 * q + 3]};
#pragma unroll
    for (int r = 0; r < PASSES; ++r) {
      const uint32_t row = row0 + (b * PASSES + r) * RPP;
      if (row < m && ch < p.n)
        product_store8<STREAM>(p, row, ch, buf + (r * RPP + lane / LPR) * F::PAD + (lane % LPR) * 8, pre[b * PASSES + r]);
    }
  }
}

template <int AT, int WN, bool STREAM>
static void launch_fused(const ProductArgs& p, hipStream_t stream) {
  const auto launch = [&](auto kernel, uint32_t rows, uint32_t waves) {
    hipLaunchKernelGGL(kernel, dim3(ceil_div(p.m, rows), ceil_div(p.n, 64u * WN)), dim3(64 * waves), 0, stream, p);
  };
  if (p.kb <= 2) launch(k_mx_product_fused<AT, WN, 2, STREAM>, FusedTile<AT, WN, 2>::BM, FusedTile<AT, WN, 2>::NW);
  else if (p.kb <= 4) launch(k_mx_product_fused<AT, WN, 4, STREAM>, FusedTile<AT, WN, 4>::BM, FusedTile<AT, WN, 4>::NW);
  else launch(k_mx_product_fused<AT, WN, 8, STREAM>, FusedTile<AT, WN, 8>::BM, FusedTile<AT, WN, 8>::NW);
}
template <int AT, bool STREAM>
static void launch_fused(const ProductArgs& p, hipStream_t stream) {
  if (p.n <= 64) launch_fused<AT, 1, STREAM>(p, stream);
  else if (p.n <= 128) launch_fused<AT, 2, STREAM>(p, stream);
  else launch_fused<AT, 4, STREAM>(p, stream);
}
template <int AT>
static int launch_fused(const ProductArgs& p, const scn_mx_product_io& io, hipStream_t stream) {
  SCN_REQUIRE((uint64_t)p.b_ld * 256 < (1ull << 32), SCN_ERR_UNSUPPORTED, "mx_product: rows more than 16 MB apart");
  if (int rc = product_start(p, io, stream)) return rc;
  const bool wide = p.n > 128 && p.kb <= 4 && (uint64_t)p.m * p.n > (8u << 20);
  if (p.out_fp32 ? whole_lines(p) && !wide : whole_lines(p) || p.kb > 4) launch_fused<AT, true>(p, stream);
  else launch_fused<AT, false>(p, stream);
  return SCN_OK;
}

// Rows that are not quantised yet are quantised by every workgroup that reads them up to this many blocks; beyond it (and
// beyond 16 rows) a launch of its own is cheaper: 8192 x 8192 weights, 4 fp16 rows (1024 blocks): 15.4 us against 15.8 us,
// 8 rows 19.9 us against 17.3 us.
static bool product_direct(uint32_t m, uint32_t k) { return m <= 16 && (uint64_t)m * mx_blocks(k) <= kFewBlocks; }
// More of them are quantised in the product's own launch while their channels are few: every workgroup of a row quantises it, one
// for 256 channels.  us with the two launches | one, fp16 rows: 123646 x 256 x 128 with residual 41.5 | 34.9, 123646 x 64 x 64 14.1 |
// 8.7, 50000 x 1024 x 64 29.5 | 27.8, 20000 x 1000 x 100 27.6 | 24.6, 50000 x 256 x 256 19.6 | 19.7 (fp32 30.5 | 25.0), 500 x 64 x 256
// 5.4 | 5.2; but 50000 x 512 x 256 23.6 | 25.7, 5000 x 1024 x 256 8.0 | 9.4.  One launch is 6 us less on the host.
// (its longest rows take 8 threads each, and a launch has fewer than 2^32)
static bool product_fused(uint32_t m, uint32_t n, uint32_t k) {
  return m < (1u << 29) - 64 && (k <= 128 ? n <= 1024 : k <= 256 && n <= 256);
}
static size_t product_workspace(uint32_t m, uint32_t n, uint32_t k) {
  return product_direct(m, k) || product_fused(m, n, k) ? 0 : (size_t)m * mx_row_bytes(k);
}

// U = runs a wave requests at once: what it has to do in all, up to 8 (4 for two row tiles).
template <int AT, int MT>
static int launch_few(const ProductArgs& p, const scn_mx_product_io& io, hipStream_t stream) {
  const uint32_t runs = (p.kb + 3) / 4, waves = std::min(8u, runs), per = ceil_div(runs, waves);
  SCN_REQUIRE(p.n < (1u << 27), SCN_ERR_UNSUPPORTED, "mx_product: %u x %u outputs are too many for one call", p.m, p.n);
  if (int rc = product_start(p, io, stream)) return rc;
  const dim3 grid(ceil_div(p.n, 16)), block(64 * waves);
  if (per == 1) hipLaunchKernelGGL((k_mx_product_few<AT, MT, 1>), grid, block, 0, stream, p);
  else if (per == 2) hipLaunchKernelGGL((k_mx_product_few<AT, MT, 2>), grid, block, 0, stream, p);
  else if (per <= 4 || MT > 1) hipLaunchKernelGGL((k_mx_product_few<AT, MT, 4>), grid, block, 0, stream, p);
  else hipLaunchKernelGGL((k_mx_product_few<AT, 1, 8>), grid, block, 0, stream, p);
  return SCN_OK;
}

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
  SCN_REQUIRE(io.res_dev != io.out_dev || (io.res_dtype == io.out_dtype && (io.res_ld == io.out_ld || io.m == 1)), SCN_ERR_INVALID,
              "mx_product: an output that is the residual must have its type and row stride");
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
    if (!product_direct(io.m, io.k) && !product_fused(io.m, io.n, io.k)) {
      const size_t need = product_workspace(io.m, io.n, io.k);
      SCN_REQUIRE(io.workspace_dev && ((uintptr_t)io.workspace_dev & 15) == 0 && io.workspace_bytes >= need, SCN_ERR_INVALID,
                  "mx_product: rows of this type need a 16-byte aligned workspace of %zu bytes (%zu given)", need, io.workspace_bytes);
      uint8_t* ws = (uint8_t*)io.workspace_dev;
      p.a = ws;
      p.a_ld = p.as_ld = mx_row_bytes(io.k);
      p.as = ws + (size_t)kb * kMxBlockBytes;   // (product_start quantises the rows into it)
      at = SCN_DTYPE_MXFP4;
    }
  }
  const auto tiles = [&](uint32_t t) { return (uint64_t)ceil_div(io.n, t) * ceil_div(io.m, t); };
  // Up to 16 rows of up to 120 blocks go to the few-row kernel, longer ones to whichever kernel is faster: the time of the few-row
  // kernel grows with the weight rows and by 2 to 5 % with every row; the tiled ones take a round of the GPU, or two, for 1 row as
  // for 16.  Up to 256 tiles of 64 weight rows they divide k, beyond they do not.  us few | tiled for 1, 4, 8 and 16 rows of 4096
  // channels, weights not in a cache:
  //   8192 weight rows (128 tiles) 7.8 8.5 9.4 11.0 | 9.7 9.8 10.0 10.4; 12288 9.8 11.0 12.4 14.8 | 10.2 10.4 10.6 10.9;
  //   16384 (256) 11.8 13.5 15.4 18.6 | 11.2 11.2 11.4 11.7; 16448 13.6 16.1 18.0 21.8 | 16.6 16.6 16.8 17.0;
  //   24576 16.9 19.0 21.4 26.6 | 17.9 17.9 18.0 18.2; 32768 21.3 24.2 27.4 34.4 | 19.1 19.1 19.3 19.4.
  // Rows too far apart for the tiled kernels' 32-bit offsets stay with the few-row kernel.
  const uint64_t t64 = tiles(64);
  const bool sooner = t64 <= 256 ? io.m <= 8 && t64 <= (io.m > 1 ? 160u : 192u) : t64 + 20 * io.m < 410;
  const bool few = io.m <= 16 && (kb <= 120 || t64 < 72 || sooner || !product_near(p));
  int rc;
  if (at != SCN_DTYPE_MXFP4 && !product_direct(io.m, io.k))
    rc = at == SCN_DTYPE_FP16 ? launch_fused<SCN_DTYPE_FP16>(p, io, stream) : launch_fused<SCN_DTYPE_FP32>(p, io, stream);
  else if (at == SCN_DTYPE_FP16) rc = launch_few<SCN_DTYPE_FP16, 1>(p, io, stream);
  else if (at == SCN_DTYPE_FP32) rc = launch_few<SCN_DTYPE_FP32, 1>(p, io, stream);
  else if (few) rc = launch_few<SCN_DTYPE_MXFP4, 1>(p, io, stream);
  // two row tiles of 16 while the tiled kernel below does not divide k: 32 rows, 1024 x 1024 weights 3.5 against 4.0 us, 8192 x 2048
  // 7.4 against 7.1
  else if (io.m > 16 && io.m <= 32 && kb >= 32 && kb < 64 && io.n <= 4096) rc = launch_few<SCN_DTYPE_MXFP4, 2>(p, io, stream);
  else {
    // The largest tile of which there are enough for the GPU's 256 CUs, when k is long enough for its reuse to count.  us for
    // 64 | 128 | 256 rows and channels a tile:
    //   4096 x 3584 x 2048 38 | 27 | 22, 3584 x 3584 x 512 13.0 | 13.4 | 11.6, 2560 x 2560 x 2048 (100 tiles of 256) 19 | 14 | 18;
    //   32640 x 128 x 2048 14.5 | 12.2 | 18.7, 32640 x 128 x 512 5.6 | 6.1 | 10.3, 100000 x 64 x 1024 15.5 | 20.8 | 28.8.
    // With a residual whose size is beyond the caches' (16 M numbers) the wider stores of the larger tile count as well:
    //   123646 x 256 x 128 31 | 28 | 31, 50000 x 256 x 128 10.6 | 13.2 | 12.7.
    // The smallest tile with k in 4 parts, when there is a CU for every tile and 16 stages: whole | in 4 parts
    //   4096 x 64 x 8192 13.6 | 10.4, 16384 x 64 x 4096 (256 tiles) 12.8 | 10.0; x 2048 6.4 | 6.5; 24576 x 64 x 4096 14 | 17.
    const bool wide = kb > 16 || (io.res_dev && (uint64_t)io.m * io.n >= (16u << 20));
    // Up to 16 rows take no larger tile: 65536 x 4096 weights 31 | 30 | 39, 32768 x 8192 36 | 40 | 43.
    const bool many = io.m > 16;
    rc = many && tiles(256) >= 144 && io.n > 128 && kb > 8 ? launch_product<256, 256, 4, 2, 1>(p, io, stream)
         : many && tiles(128) >= 256 && io.n > 64 && wide  ? launch_product<128, 128, 2, 2, 1>(p, io, stream)
         : t64 <= 256 && kb > 120                          ? launch_product<64, 64, 1, 1, 4>(p, io, stream)
                                                           : launch_product<64, 64, 1, 1, 1>(p, io, stream);
  }
  if (rc) return rc;
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

size_t scn_mx_product_workspace(uint32_t m, uint32_t n, uint32_t k) { return k ? product_workspace(m, n, k) : 0; }

int scn_mx_product(const scn_mx_product_io* io, void* stream) {
  SCN_REQUIRE(io, SCN_ERR_INVALID, "scn_mx_product: null pointer");
  int rc = mx_product(*io, (hipStream_t)stream);
  if (rc == SCN_OK && debug_sync_enabled()) rc = debug_sync_check((hipStream_t)stream, "scn_mx_product");
  return rc;
}

}  // extern "C"
