// Convolution on microscaled 4-bit rows (MXFP4): gathered rows x weights on the scaled matrix instructions.
#include "scn_conv_kernels.hpp"
#include "scn_mx.hpp"
#include "scn_mx_device.hpp"

namespace scn {

typedef int v8i __attribute__((ext_vector_type(8)));

// v_mfma_scale_f32_32x32x64_f8f6f4 with 4-bit operands: lane l supplies row / column l % 32, the 16 code bytes of K-block
// l / 32 and that block's scale.  Rows of A are output channels, columns of B voxels (as in the other convolution kernels); a
// K-step takes two blocks.  Weights are laid out in units of one block x 32 output channels: wfrag[block][tile][32] x 16
// bytes; the scale bytes of 4 tiles are one word, wscales[block][tile / 4][32][4]; block g = kernel offset * BPR + block of the
// row (BPR = blocks of an input row).  SEL: the byte of ws.
template <int SEL>
__device__ __forceinline__ v16f conv_mma(const uint4& w, uint32_t ws, const uint4& x, uint32_t xs, v16f c) {
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(v8i{(int)w.x, (int)w.y, (int)w.z, (int)w.w, 0, 0, 0, 0},
                                                         v8i{(int)x.x, (int)x.y, (int)x.z, (int)x.w, 0, 0, 0, 0}, c, 4, 4, SEL,
                                                         (int)ws, 0, (int)xs);
}

// Any width: operands straight from memory, a wave owns 32 rows x MT tiles of 32 output channels.
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
    uint32_t xs = 0;
    if (idx >= 0) {
      const char* src = a.x + (size_t)(uint32_t)idx * a.x_ld_bytes;
      xq = *reinterpret_cast<const uint4*>(src + b * 16);
      xs = *reinterpret_cast<const uint8_t*>(src + bpr * 16 + b);
    }
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      const size_t g0 = (size_t)min(g, total - 1);
      const int tt = min(t0 + t, mtiles - 1);
      acc[t] = conv_mma<0>(a.wfrag[(g0 * mtiles + tt) * 32 + ln], wscales[((g0 * ((mtiles + 3) / 4) + tt / 4) * 32 + ln) * 4 + tt % 4],
                           xq, xs, acc[t]);
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

// Rows of up to 4 blocks (128 channels).  What bounds the kernel above is the memory pipe: 16 code bytes of 32 rows in operand
// order are 32 requests, their scale bytes 32 more.  Here a row is fetched whole -- codes and the scale word behind them are
// BPR + 1 chunks of 16 bytes, taken by as many neighbouring lanes -- straight into LDS, and the operands are read from there.
// A workgroup owns 64 rows and MT tiles of 32 output channels; its W waves share the rows' neighbour indices and deal the
// kernel offsets out between them, so a wave only ever waits for its own loads; the waves' sums are added (in wave order) when
// the rows are stored.
//   a stage = one kernel offset that some row has a neighbour at (two of them for rows of one block): 64 gathered rows in LDS and
//   the weights of its blocks in registers (in LDS they leave room for fewer waves); a wave fetches one stage ahead.  Rows without a
//   neighbour read as zeros (scale 2^-127, codes 0).
// (120,000 rows 64 -> 64, 21.6 us: 4.9 for the launch and the neighbour indices, 4.4 for the store, both near the memory's rate;
// in between 5.9 for the products alone, 4.8 of gathers and 3 of weights on top.  Requesting the rows two stages ahead gains
// 0.6 us here and loses 2 us at 60,000 rows 128 -> 128.)
//   LDS rows of 3 and 5 chunks are read without bank conflicts as they are; rows of 2 and 4 chunks hold chunk c at position
//   c ^ (row / 8) % 2 and c ^ (row / 4) % 4.
template <int BPR, int MT, int W>
struct ConvMxStage {
  static constexpr int OFFS = BPR == 1 ? 2 : 1;                  // kernel offsets of a stage
  static constexpr int SB = BPR * OFFS, KS = (SB + 1) / 2;       // blocks and K-steps
  static constexpr int CH = BPR + 1;                             // 16-byte chunks of a row
  static constexpr int GLOADS = CH * OFFS, BYTES = GLOADS * 1024;   // wave loads: 64 rows
  static constexpr int KMAX = 28;                                // kernel offsets whose indices are held at a time
  static constexpr int RING = KMAX * 256;                        // LDS offset of the rings
  static constexpr int PAD = 32 * MT + 4;                        // floats per row of the store buffer
  static constexpr int WAVE = 2 * BYTES > 32 * PAD * 4 ? 2 * BYTES : 32 * PAD * 4;
  static constexpr int LDS = RING + W * WAVE;
  static constexpr int PER_CU = 160 * 1024 / ((LDS + 1279) / 1280 * 1280);   // workgroups whose LDS a CU holds (handed out in 1,280 bytes)
};

// 64 x 16 bytes to LDS, lane l's to base + 16 l: in assembly, because the compiler would order its own LDS
// reads behind every such load in flight.
__device__ __forceinline__ void conv_load16_lds(const void* src, uint32_t base) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(src), "s"(base) : "m0", "memory");
}

// The same of a buffer: bytes [at, at + 16) of it, zeros beyond its size.
__device__ __forceinline__ void conv_load16_lds(const v4i& buffer, uint32_t at, uint32_t base) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds" ::"v"(at), "s"(buffer), "s"(base) : "m0", "memory");
}

// MODE: the epilogue (see epilogue_values): 2 and 4 are fp16 output without and with an fp16 residual, 0 everything.
template <int BPR, int MT, int W, int MODE>
__global__ __launch_bounds__(64 * W, 2) void k_conv_mx_gather(const ConvArgs a, const uint8_t* __restrict__ wscales, int mtiles) {
  using S = ConvMxStage<BPR, MT, W>;
  __shared__ __align__(16) char lds[S::LDS];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), ln = lane & 31, lh = lane >> 5;
  const uint32_t n = eff_n(a.n_out_dev, a.n_bound);
  uint32_t tile;
  if (!xcd_tile(n, 64u, &tile)) return;
  const uint32_t row0 = tile * 64;
  const int t0 = blockIdx.y * MT;
  typedef __attribute__((address_space(3))) char* lptr;
  const uint32_t base = (uint32_t)(uintptr_t)(lptr)lds;
  const int32_t* idx = reinterpret_cast<const int32_t*>(lds);
  const int ring = S::RING + wave * S::WAVE;

  v16f acc[MT][2];
#pragma unroll
  for (int t = 0; t < MT; ++t)
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int j = 0; j < 16; ++j) acc[t][u][j] = 0.f;

  // what this lane fetches of a stage: the row and the chunk of gather load q (of one offset); its weights are those of K-block
  // 2 s + lh of step s
  int grow[S::CH], gchunk[S::CH];
#pragma unroll
  for (int q = 0; q < S::CH; ++q) {
    const int e = q * 64 + lane, r = e / S::CH, p = e - r * S::CH;
    grow[q] = r;
    gchunk[q] = (S::CH == 2 ? p ^ ((r >> 3) & 1) : S::CH == 4 ? p ^ ((r >> 2) & 3) : p) * 16;
  }
  // weights of one kernel offset: uint4 and scale words; this lane's of step s start at woff, soff (a block that does not exist
  // takes another one's codes, and scales of 0)
  const uint32_t wstride = BPR * mtiles * 32, sstride = BPR * ((mtiles + 3) / 4) * 32;
  uint32_t woff[S::KS], soff[S::KS];
#pragma unroll
  for (int s = 0; s < S::KS; ++s) {
    const int b = BPR == 1 || (S::SB % 2 && 2 * s + lh >= S::SB) ? 0 : 2 * s + lh;
    woff[s] = (b * mtiles + t0) * 32 + ln;
    soff[s] = (b * ((mtiles + 3) / 4) + t0 / 4) * 32 + ln;
  }
  // The input rows as a buffer of 2^24 - 1 of them, where the table can name no more and they fit 32 bits: "no neighbour" (-1,
  // 2^24 - 1 in the 24 bits that the multiplication takes) lies behind its end, where loads return 0.  An address is one
  // instruction then (120,000 rows 64 -> 64: 22.9 us with 64-bit addresses and a row of zeros, 21.5 us so).
  const bool near = a.nbr_ld < (1u << 24) && a.x_ld_bytes < 256;
  const uint64_t xbase = (uint64_t)(uintptr_t)a.x;
  const v4i xbuf = {__builtin_amdgcn_readfirstlane((int)(uint32_t)xbase), __builtin_amdgcn_readfirstlane((int)(uint32_t)(xbase >> 32) & 0xFFFF),
                    (int)(0xFFFFFFu * a.x_ld_bytes), 0x00027000};
  uint4 w[S::KS][MT], w1[S::KS][MT];
  uint32_t ws[S::KS], ws1[S::KS];

  for (int k0 = 0; k0 < a.kvol; k0 += S::KMAX) {
    // neighbour rows of up to KMAX offsets; rows beyond the count have none
    const int nk = min(S::KMAX, a.kvol - k0);
    const int32_t* minus1 = reinterpret_cast<const int32_t*>(a.zrow + 512);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    if (W > 1 && k0) __syncthreads();   // (the indices before these have been read)
    // one load: 4 offsets x 64 rows, 4 rows per lane (the table holds -1 from the count up to the next multiple of 32 rows)
    for (int k4 = wave * 4; k4 < nk; k4 += W * 4) {
      const int k = k0 + k4 + (lane >> 4);
      const uint32_t row = row0 + (lane & 15) * 4;
      conv_load16_lds(k4 + (lane >> 4) < nk && row < n ? a.nbr + (size_t)k * a.nbr_ld + row : minus1 + lane * 4,
                      __builtin_amdgcn_readfirstlane(base + k4 * 256));
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    if (W > 1) __syncthreads();
    uint32_t todo = 0;   // offsets at which some row has a neighbour
#pragma unroll
    for (int k4 = 0; k4 < S::KMAX; k4 += 4) {
      if (k4 >= nk) break;
      const int4 v = reinterpret_cast<const int4*>(idx)[k4 * 16 + lane];
      const uint64_t some = __ballot((v.x & v.y & v.z & v.w) >= 0);   // (indices are -1 or not negative: the sign of their AND)
      todo |= ((some & 0xFFFFull ? 1u : 0u) | (some & 0xFFFF0000ull ? 2u : 0u) | (some & 0xFFFF00000000ull ? 4u : 0u) |
               (some >> 48 ? 8u : 0u)) << k4;
    }
    todo = __builtin_amdgcn_readfirstlane(todo);
    // this wave's share: every W-th stage
    const int all = (__popc(todo) + S::OFFS - 1) / S::OFFS, stages = (all - wave + W - 1) / W;
    auto drop = [&](int n_offsets) {
      for (int i = 0; i < n_offsets; ++i) todo &= todo - 1;
    };
    drop(wave * S::OFFS);

    // issues the loads of the next stage in `todo`: rows into ring slot `slot`, weights into w1 and ws1
    auto issue = [&](int slot) {
      const uint32_t buf = __builtin_amdgcn_readfirstlane(base + ring + slot * S::BYTES);
      const int ka = __ffs(todo) - 1;
      todo &= todo - 1;
      int kb = ka;
      bool second = true;
      if constexpr (S::OFFS == 2) {   // (a second offset may not exist: zeros)
        second = todo != 0;
        if (second) kb = __ffs(todo) - 1;
        todo &= todo - 1;
      }
      drop((W - 1) * S::OFFS);
      int i[S::GLOADS];
#pragma unroll
      for (int q = 0; q < S::GLOADS; ++q) i[q] = idx[(q < S::CH ? ka : kb) * 64 + grow[q % S::CH]];
      // (uniform bases, 32-bit offsets per lane)
      const char* wp = reinterpret_cast<const char*>(a.wfrag) + (size_t)(k0 + ka) * wstride * 16;
      const char* sp = reinterpret_cast<const char*>(wscales) + (size_t)(k0 + ka) * sstride * 4;
      const uint32_t other = S::OFFS == 2 && lh ? (uint32_t)(kb - ka) : 0u;
#pragma unroll
      for (int s = 0; s < S::KS; ++s) {
#pragma unroll
        for (int t = 0; t < MT; ++t)
          w1[s][t] = *reinterpret_cast<const uint4*>(wp + (woff[s] + other * wstride + min(t, mtiles - 1 - t0) * 32) * 16);
        ws1[s] = *reinterpret_cast<const uint32_t*>(sp + (soff[s] + other * sstride) * 4);
      }
      if (near) {
#pragma unroll
        for (int q = 0; q < S::GLOADS; ++q) {
          const uint32_t at = ((uint32_t)i[q] & 0xFFFFFFu) * (a.x_ld_bytes & 0xFFFFFFu) + gchunk[q % S::CH];
          conv_load16_lds(xbuf, q < S::CH || second ? at : 0xFFFFFFF0u, buf + q * 1024);
        }
      } else {
#pragma unroll
        for (int q = 0; q < S::GLOADS; ++q) {
          const char* row = a.x + (size_t)(uint32_t)max(i[q], 0) * a.x_ld_bytes;
          row = i[q] >= 0 && (q < S::CH || second) ? row : a.zrow;
          conv_load16_lds(row + gchunk[q % S::CH], buf + q * 1024);
        }
      }
    };
    if (stages > 0) issue(0);
    int slot = 0;
    for (int j = 0; j < stages; ++j) {
      // everything of this stage has landed, and the reads of the slot that is refilled now have returned (the wait is one the
      // compiler knows, so that it adds none for the weights)
      __builtin_amdgcn_s_waitcnt(0x0070);   // vmcnt(0) lgkmcnt(0)
      asm volatile("" ::: "memory");
#pragma unroll
      for (int s = 0; s < S::KS; ++s) {
        ws[s] = ws1[s];
#pragma unroll
        for (int t = 0; t < MT; ++t) w[s][t] = w1[s][t];
      }
      if (j + 1 < stages) issue(slot ^ 1);
      __builtin_amdgcn_sched_barrier(0);
      const char* sb = lds + ring + slot * S::BYTES;
#pragma unroll
      for (int s = 0; s < S::KS; ++s) {
        const int blk = 2 * s + lh;
        const bool in = S::SB % 2 == 0 || blk < S::SB;
        const int b = in ? blk : 0;
        uint4 x[2];
        uint32_t xs[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int r = 32 * u + ln;
          const int cc = BPR == 1 ? 0 : b, sc = BPR;   // chunks of the codes and of the scales
          const int cp = S::CH == 2 ? cc ^ ((r >> 3) & 1) : S::CH == 4 ? cc ^ ((r >> 2) & 3) : cc;
          const int sp = S::CH == 2 ? sc ^ ((r >> 3) & 1) : S::CH == 4 ? sc ^ ((r >> 2) & 3) : sc;
          const char* row = sb + (BPR == 1 ? b * S::CH * 1024 : 0) + r * S::CH * 16;
          x[u] = *reinterpret_cast<const uint4*>(row + cp * 16);
          xs[u] = *reinterpret_cast<const uint8_t*>(row + sp * 16 + (BPR == 1 ? 0 : b));
          if (!in) xs[u] = 0;
        }
        const uint32_t wsv = in ? ws[s] : 0u;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          acc[0][u] = conv_mma<0>(w[s][0], wsv, x[u], xs[u], acc[0][u]);
          if constexpr (MT > 1) acc[1][u] = conv_mma<1>(w[s][1], wsv, x[u], xs[u], acc[1][u]);
          if constexpr (MT > 2) {
            acc[2][u] = conv_mma<2>(w[s][2], wsv, x[u], xs[u], acc[2][u]);
            acc[3][u] = conv_mma<3>(w[s][3], wsv, x[u], xs[u], acc[3][u]);
          }
        }
      }
      slot ^= 1;
    }
  }
  // Store through LDS, 32 rows at a time: a lane of the accumulators holds 4 channels of a row, a store takes 8 of one row
  // and adds the waves' sums.  (Every load has been waited for; the rings are free.)
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
  float* mine = reinterpret_cast<float*>(lds + ring);
  constexpr int LPR = 4 * MT, RPP = 64 * W / LPR;   // threads per row, rows per pass
  const int part = threadIdx.x % LPR, co = 32 * t0 + part * 8;
  const bool wide = co < ((a.cout + 15) & ~15);
  float4 b4[2], sc4;
  if (wide) {
    epilogue_consts<1>(a, co, &b4[0], &sc4);
    epilogue_consts<1>(a, co + 4, &b4[1], &sc4);
  }
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    if (W > 1 && u) __syncthreads();
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int q = 0; q < 4; ++q)
        *reinterpret_cast<v4f*>(mine + ln * S::PAD + t * 32 + q * 8 + lh * 4) =
            v4f{acc[t][u][4 * q], acc[t][u][4 * q + 1], acc[t][u][4 * q + 2], acc[t][u][4 * q + 3]};
    if (W > 1) __syncthreads();
    for (int r = threadIdx.x / LPR; r < 32; r += RPP) {
      const uint32_t row = row0 + 32 * u + r;
      if (row >= n) continue;
      float y[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if (!wide) break;
        const float* src = reinterpret_cast<const float*>(lds + S::RING) + r * S::PAD + part * 8 + 4 * h;
        v4f sum = *reinterpret_cast<const v4f*>(src);
#pragma unroll
        for (int w = 1; w < W; ++w) {
          const v4f other = *reinterpret_cast<const v4f*>(src + w * (S::WAVE / 4));
#pragma unroll
          for (int j = 0; j < 4; ++j) sum[j] += other[j];
        }
        float v[4];
        epilogue_values<1, MODE>(a, row, co + 4 * h, sum, b4[h], sc4, a.res ? residual_ptr(a, row, co + 4 * h) : nullptr, v);
#pragma unroll
        for (int j = 0; j < 4; ++j) y[4 * h + j] = v[j];
      }
      if (MODE == 0 && a.out_dtype == SCN_DTYPE_INT8) {
        const char4 q[2] = {pack_int8(a, y), pack_int8(a, y + 4)};
        if (wide) __builtin_memcpy(a.out + (size_t)row * a.out_ld + co, q, 8);
        continue;
      }
      const v4h q[2] = {pack_fp16(y), pack_fp16(y + 4)};
      if (wide && a.out) __builtin_memcpy(reinterpret_cast<_Float16*>(a.out) + (size_t)row * a.out_ld + co, q, 16);
      if (a.mx_out) {   // microscaled rows of the fp16 values: 4 lanes hold a block
        const int blocks = (a.cout + 31) / 32, b = co / 32;
        float v[8];
        uint32_t top = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          v[j] = co + j < a.cout ? (float)q[j / 4][j % 4] : 0.f;
          top = max(top, __float_as_uint(v[j]) & 0x7FFFFFFFu);
        }
        top = lanes_max<4>(top);
        const uint32_t e = mx_scale_byte(top);
        const float up = __uint_as_float((254u - (e == 255u ? 0u : e)) << 23);
        if (b < blocks) {
          char* dst = a.mx_out + (size_t)row * a.mx_ld;
          *reinterpret_cast<uint32_t*>(dst + b * 16 + (part & 3) * 4) = e == 255u ? 0u : mx_codes8(v, up);
          if ((part & 3) == 0) {
            uint8_t* sc = reinterpret_cast<uint8_t*>(dst + blocks * 16);
            sc[b] = (uint8_t)e;
            if (b + 1 == blocks)
              for (int z = blocks; z % 4 != 0; ++z) sc[z] = 0;
          }
        }
      }
    }
  }
}

template <int BPR, int MT, int W, int MODE>
static void launch_gather(ConvArgs& a, const uint8_t* ws, int mtiles, hipStream_t stream) {
  const unsigned tiles = (a.n_bound + 63u) / 64u;
  hipLaunchKernelGGL((k_conv_mx_gather<BPR, MT, W, MODE>), dim3(((tiles + 7u) / 8u) * 8u, (unsigned)(mtiles + MT - 1) / MT),
                     dim3(64 * W), 0, stream, a, ws, mtiles);
}

// Waves per 64 rows.  Few tiles are bound by the latency of a wave's chain of stages, which more waves shorten.  More of them take
// two waves while all tiles run at once, then one wave while those do, then two again, which balance better over several rounds.
// LDS limits how many run: 9 one-wave or 6 two-wave workgroups a CU at 32 and 64 -> 64 channels (147,456 and 98,304 rows; registers
// would allow 16 waves), 10 or 6 at 16 -> 16, 9 or 5 at 128 -> 64.  us with 1 / 2 / 4 waves, 64 -> 64: 20,000 rows 14.6 / 10.6 / 8.4, 50,000
// 17.1 / 12.6 / 14.5, 80,000 21.4 / 16.2 / 18.4, 95,000 22.2 / 17.6 / 20.0, 110,000 23.3 / 25.6 / 24.1, 142,000 26.2 / 27.1 / 27.1, 163,000 37.9 /
// 28.3 / 31.3, 196,000 39.5 / 34.8 / 34.5, 260,000 43.7 / 39.4 / 44.9; 16 -> 16: 95,000 13.6 / 10.3 / 13.1, 163,000 16.2 / 17.8 / 19.5, 190,000
// 25.0 / 18.6 / 21.7; 128 -> 64: 80,000 25.1 / 20.9 / 22.9, 95,000 26.5 / 29.2 / 25.0; with 128 output channels (twice the work per wave)
// with 2 / 4: 20,000 rows 128 -> 128 18.7 / 15.7, 48,460 rows 64 -> 128 17.2 / 20.1, 150,000 rows 128 -> 128 57.0 / 60.9.
// The choice follows the bound of the row count, never the count or what an earlier forward had: the order of the sums, and
// so their last bit, depends on it.
template <int BPR, int MT, int MODE>
static void launch_waves(ConvArgs& a, const uint8_t* ws, int mtiles, hipStream_t stream) {
  const uint64_t tiles = ((uint64_t)a.n_bound + 63) / 64;
  if (a.n_bound <= 32768) return launch_gather<BPR, MT, 4, MODE>(a, ws, mtiles, stream);
  if constexpr (MT <= 2)
    if (tiles > 256u * ConvMxStage<BPR, MT, 2>::PER_CU && tiles <= 256u * ConvMxStage<BPR, MT, 1>::PER_CU)
      return launch_gather<BPR, MT, 1, MODE>(a, ws, mtiles, stream);
  launch_gather<BPR, MT, 2, MODE>(a, ws, mtiles, stream);
}
template <int BPR, int MODE>
static void launch_gather(ConvArgs& a, const uint8_t* ws, int mtiles, hipStream_t stream) {
  if (mtiles > 2) launch_waves<BPR, 4, MODE>(a, ws, mtiles, stream);
  else if (mtiles == 2) launch_waves<BPR, 2, MODE>(a, ws, mtiles, stream);
  else launch_waves<BPR, 1, MODE>(a, ws, mtiles, stream);
}

template <int BPR>
static bool dispatch_gather(ConvArgs& a, const uint8_t* ws, int mtiles, hipStream_t stream) {
  const bool half = !a.acc && a.out_dtype == SCN_DTYPE_FP16;
  if (half && !a.res) launch_gather<BPR, 2>(a, ws, mtiles, stream);
  else if (half && a.res_dtype == SCN_DTYPE_FP16 && a.mid_dtype == SCN_DTYPE_FP16 && a.a_rq_r == 0.f && a.b_rq_r == 0.f)
    launch_gather<BPR, 4>(a, ws, mtiles, stream);
  else launch_gather<BPR, 0>(a, ws, mtiles, stream);
  return true;
}

bool conv_dispatch_mx(const ConvWeights& w, uint32_t n_hint, ConvArgs& a, hipStream_t stream) {
  (void)n_hint;
  a.wfrag = w.wfrag.as<uint4>();
  const uint8_t* ws = w.wscale.as<uint8_t>();
  const int mtiles = (w.cout + 31) / 32;
  switch (w.chunks) {
    case 1: return dispatch_gather<1>(a, ws, mtiles, stream);
    case 2: return dispatch_gather<2>(a, ws, mtiles, stream);
    case 3: return dispatch_gather<3>(a, ws, mtiles, stream);
    case 4: return dispatch_gather<4>(a, ws, mtiles, stream);
    default: break;
  }
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
