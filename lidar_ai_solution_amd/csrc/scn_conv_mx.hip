// Convolution on microscaled 4-bit rows (MXFP4): gathered rows x weights on the scaled matrix instructions.
#include "scn_conv_kernels.hpp"
#include "scn_mx.hpp"

namespace scn {

typedef int v8i __attribute__((ext_vector_type(8)));

// v_mfma_scale_f32_32x32x64_f8f6f4 with 4-bit operands: lane l supplies row / column l % 32, the 16 code bytes of K-block
// l / 32 and that block's scale.  K-step s consumes blocks 2s and 2s + 1 of the sequence (offset 0 block 0, offset 0
// block 1, ..., offset kvol-1 block BPR-1), BPR = blocks of an input row: a lane gathers 16 contiguous code bytes and one
// scale byte of one input row.
//   MT = tiles of 32 output channels a wave owns; wider layers take more workgroups (grid y)
template <int MT>
__global__ __launch_bounds__(256) void k_conv_mx_rows(const ConvArgs a, const uint8_t* __restrict__ wscales, int bpr, int mtiles) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int ln = lane & 31, lh = lane >> 5;
  const uint32_t n = eff_n(a.n_out_dev, a.n_bound);
  uint32_t tile;
  if (!xcd_tile(n, 128u, &tile)) return;
  const uint32_t row0 = (tile * 4 + wave) * 32;
  if (row0 >= n) return;
  const uint32_t row = row0 + ln;
  const int t0 = blockIdx.y * MT;
  v16f acc[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t)
#pragma unroll
    for (int j = 0; j < 16; ++j) acc[t][j] = 0.f;
  const int total = a.kvol * bpr;
  for (int s = 0; s < a.steps; ++s) {
    const int g = 2 * s + lh;
    const int k = g / bpr, b = g - k * bpr;
    int32_t idx = -1;
    if (g < total && row < n) idx = a.nbr[(size_t)k * a.nbr_ld + row];
    if (!__any(idx >= 0)) continue;   // no row of this wave has a neighbour at these blocks
    uint4 xq = make_uint4(0, 0, 0, 0);
    int xs = 0;
    if (idx >= 0) {
      const char* src = a.x + (size_t)(uint32_t)idx * a.x_ld_bytes;
      xq = *reinterpret_cast<const uint4*>(src + b * 16);
      xs = *reinterpret_cast<const uint8_t*>(src + bpr * 16 + b);
    }
    const v8i xv = {(int)xq.x, (int)xq.y, (int)xq.z, (int)xq.w, 0, 0, 0, 0};
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      const size_t f = ((size_t)s * mtiles + min(t0 + t, mtiles - 1)) * 64 + lane;
      const uint4 wq = a.wfrag[f];
      const int ws = wscales[f];
      const v8i wv = {(int)wq.x, (int)wq.y, (int)wq.z, (int)wq.w, 0, 0, 0, 0};
      acc[t] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(wv, xv, acc[t], 4, 4, 0, ws, 0, xs);
    }
  }
  if (row >= n) return;
#pragma unroll
  for (int t = 0; t < MT; ++t)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int co = 32 * (t0 + t) + 8 * q + 4 * lh;
      if (t0 + t >= mtiles || co >= ((a.cout + 15) & ~15)) continue;
      float4 b4, sc4;
      epilogue_consts<1>(a, co, &b4, &sc4);
      epilogue_store<1>(a, row, co, v4f{acc[t][4 * q], acc[t][4 * q + 1], acc[t][4 * q + 2], acc[t][4 * q + 3]}, b4, sc4);
    }
}

bool conv_dispatch_mx(const ConvWeights& w, uint32_t n_hint, ConvArgs& a, hipStream_t stream) {
  (void)n_hint;
  a.wfrag = w.wfrag.as<uint4>();
  const uint8_t* ws = w.wscale.as<uint8_t>();
  const int mtiles = (w.cout + 31) / 32;
  const unsigned tiles = (a.n_bound + 127u) / 128u, blocks = ((tiles + 7u) / 8u) * 8u;
  const int mt = mtiles >= 4 ? 4 : mtiles;
  const dim3 grid(blocks, (unsigned)((mtiles + mt - 1) / mt));
  switch (mt) {
    case 1: hipLaunchKernelGGL(k_conv_mx_rows<1>, grid, dim3(256), 0, stream, a, ws, w.chunks, mtiles); break;
    case 2: hipLaunchKernelGGL(k_conv_mx_rows<2>, grid, dim3(256), 0, stream, a, ws, w.chunks, mtiles); break;
    case 3: hipLaunchKernelGGL(k_conv_mx_rows<3>, grid, dim3(256), 0, stream, a, ws, w.chunks, mtiles); break;
    default: hipLaunchKernelGGL(k_conv_mx_rows<4>, grid, dim3(256), 0, stream, a, ws, w.chunks, mtiles); break;
  }
  return true;
}

}  // namespace scn
