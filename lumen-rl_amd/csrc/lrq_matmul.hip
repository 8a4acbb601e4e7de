// FP8 products on weights in 128x128 tiles (the layout lrq_fp8_block_quant
// writes with 128 x 128 blocks): y = a w^T + bias with a e4m3 in 1x128 blocks,
// given as codes or quantized on the way in.  lrq_mma8.hpp has the mathematics.
#include "lrq.h"
#include "lrq_device.hpp"
#include "lrq_internal.hpp"
#include "lrq_mma8.hpp"

namespace lrq {

__device__ __forceinline__ void store_y(const MatmulArgs& a, int64_t at, float v) {
  if (a.out_dtype == kF32) gst<float>(static_cast<float*>(a.y) + at, v);
  else gst<uint16_t>(static_cast<uint16_t*>(a.y) + at, a.out_dtype == kBF16 ? bits16<kBF16>(v) : bits16<kF16>(v));
}

// ---------------------------------------------------------------------------
// Few tokens
// ---------------------------------------------------------------------------
// A work-group of KW waves makes 16 NT weight rows x 16 MT tokens; each wave
// takes a run of K blocks, and their sums meet in LDS.
struct RowsFromCodes {
  const MatmulArgs& a;
  int n0, m0, c;
  __device__ int row(int i) const { const int n = n0 + 16 * i + c; return n < a.n ? n : (int)a.n - 1; }
  __device__ int64_t token(int j) const { const int64_t m = (int64_t)m0 + 16 * j + c; return m < a.m ? m : a.m - 1; }
  __device__ const uint8_t* w(int i) const { return a.w + (int64_t)row(i) * a.k; }
  __device__ const float* sw(int i) const {
    const int n = n0 + 16 * i;
    return a.sw + (int64_t)((n < a.n ? n : (int)a.n - 1) / kBlk) * a.kb;
  }
  __device__ const uint8_t* x(int j) const { return static_cast<const uint8_t*>(a.x) + token(j) * a.ldx; }
  __device__ const float* sx(int j) const { return a.sx + token(j) * a.kb; }
};

// Tokens quantized by the work-group itself into LDS: rows of `pitch` bytes,
// their scales behind them.
struct RowsFromLds : RowsFromCodes {
  const uint8_t* codes;
  const float* scales;
  int pitch;
  __device__ int mine(int j) const { const int m = 16 * j + c; return m < a.m ? m : (int)a.m - 1; }
  __device__ Codes32 block(int j, int kb) const {
    const uint8_t* p = codes + mine(j) * pitch + kb * kBlk + 16 * ((threadIdx.x & 63) >> 4);
    return {*reinterpret_cast<const v4u*>(p), *reinterpret_cast<const v4u*>(p + 64)};
  }
  __device__ float scale(int j, int kb) const { return scales[mine(j) * (int)a.kb + kb]; }
};

template <int DT, int T>
__device__ __forceinline__ void quant_to_lds(const MatmulArgs& a, uint8_t* codes, float* scales, int pitch) {
  const int groups = (int)(a.m * a.kb);  // 16 lanes each
  for (int e = threadIdx.x >> 4; e < groups; e += T / 16) {
    const int m = e / (int)a.kb, kb = e % (int)a.kb, at = kb * kBlk + 8 * (threadIdx.x & 15);
    float v[8], s;
    load_acts<DT>(static_cast<const uint8_t*>(a.x) + (int64_t)m * a.ldx * (DT == kF32 ? 4 : 2), at, (int)a.k, v);
    *reinterpret_cast<v2u*>(codes + m * pitch + at) = quant8(v, s);
    if ((threadIdx.x & 15) == 0) scales[e] = s;
  }
}

constexpr int kRowWaves = 8;
// XDT: the type of x, or -1: codes and scales
template <int XDT, int NT, int MT, int D>
__global__ __launch_bounds__(64 * kRowWaves) void k_mm8_rows(MatmulArgs a) {
  constexpr int KW = kRowWaves, CELLS = 256 * NT * MT;
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c = lane & 15, g = lane >> 4;
  const int n0 = blockIdx.x * 16 * NT, m0 = blockIdx.y * 16 * MT;
  const int steps = (int)((a.kb + KW - 1) / KW);
  const int kb0 = wave * steps, kb1 = kb0 + steps < a.kb ? kb0 + steps : (int)a.kb;
  f32x4 acc[NT][MT];
  if constexpr (XDT >= 0) {
    const int pitch = (int)a.kb * kBlk + 16;
    float* const scales = reinterpret_cast<float*>(lds + a.m * pitch);
    const RowsFromLds src{{a, n0, m0, c}, lds, scales, pitch};
    row_sums<NT, MT, D, true, true>(src, kb0, kb1, (int)a.k, acc, [&] {
      quant_to_lds<XDT, 64 * KW>(a, lds, scales, pitch);
      lds_barrier8();
    });
    lds_barrier8();
  } else {
    const RowsFromCodes src{a, n0, m0, c};
    row_sums<NT, MT, D, false, true>(src, kb0, kb1, (int)a.k, acc, [] {});
  }
  float* const red = reinterpret_cast<float*>(lds);  // [wave][token][row]
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int j = 0; j < MT; ++j)
      *reinterpret_cast<f32x4*>(red + wave * CELLS + (16 * j + c) * 16 * NT + 16 * i + 4 * g) = acc[i][j];
  lds_barrier8();
  for (int e = tid; e < CELLS; e += 64 * KW) {
    const int64_t m = (int64_t)m0 + e / (16 * NT);
    const int n = n0 + e % (16 * NT);
    if (m >= a.m || n >= a.n) continue;
    float sum = red[e];
#pragma unroll
    for (int w = 1; w < KW; ++w) sum += red[w * CELLS + e];
    if (a.bias != nullptr) sum += load_as_f32(a.bias, a.bias_dtype, n);
    store_y(a, m * a.n + n, sum);
  }
}

// ---------------------------------------------------------------------------
// Many tokens
// ---------------------------------------------------------------------------
struct DenseTile {
  static constexpr bool kCut = true;
  const MatmulArgs& a;
  int n0, m0, n_last, m_last;  // n_last, m_last: within the tile
  bool dma;
  __device__ const uint8_t* w() const { return a.w + (int64_t)n0 * a.k; }
  __device__ const uint8_t* x() const { return static_cast<const uint8_t*>(a.x) + (int64_t)m0 * a.ldx; }
  __device__ uint32_t w_bytes() const { return (uint32_t)((n_last < 255 ? n_last + 1 : 256) * a.k); }
  __device__ uint32_t x_bytes() const { return (uint32_t)((m_last < 255 ? m_last : 255) * a.ldx + a.k); }
  __device__ uint32_t w_off(int r) const { return r <= n_last ? (uint32_t)(r * a.k) : dma ? kNoRow : (uint32_t)(n_last * a.k); }
  __device__ uint32_t x_off(int r) const { return r <= m_last ? (uint32_t)(r * a.ldx) : dma ? kNoRow : (uint32_t)(m_last * a.ldx); }
  __device__ const float* sx() const { return a.sx + (int64_t)m0 * a.kb; }
  __device__ const float* sw() const { return a.sw + (int64_t)(n0 / kBlk) * a.kb; }
  __device__ uint32_t sx_bytes() const { return (uint32_t)(4 * ((m_last < 255 ? m_last : 255) + 1) * a.kb); }
  __device__ uint32_t sw_bytes() const { return (uint32_t)(4 * ((n_last < 255 ? n_last : 255) / kBlk + 1) * a.kb); }
  __device__ uint32_t sx_off(int r) const { return (uint32_t)(4 * (r < m_last ? r : m_last) * a.kb); }
  __device__ uint32_t sw_off(int s) const {
    const int r = (n0 & (kBlk - 1)) + (16 * s < n_last ? 16 * s : n_last);
    return (uint32_t)(4 * (r / kBlk) * a.kb);
  }
};

template <int ODT, int FN, int FM>
__device__ __forceinline__ void store_tile(const MatmulArgs& a, f32x4 (&acc)[FN][FM], int n0, int m0, uint8_t* lds) {
  // 16 tokens at a time through the wave's own piece of LDS, so that rows leave
  // in 16-byte stores
  constexpr int ES = ODT == kF32 ? 4 : 2, COLS = 16 * FN, PITCH = COLS * ES + 16, PER = 16 / ES, PIECES = COLS / PER;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = lane & 15, g = lane >> 4;
  uint8_t* const out = lds + wave * 16 * PITCH;
#pragma unroll
  for (int j = 0; j < FM; ++j) {
    wave_fence8();
#pragma unroll
    for (int i = 0; i < FN; ++i) {
      f32x4 v = acc[i][j];
      if (a.bias != nullptr) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int n = n0 + 16 * i + 4 * g + r;
          v[r] += n < a.n ? load_as_f32(a.bias, a.bias_dtype, n) : 0.0f;
        }
      }
      uint8_t* const at = out + c * PITCH + (16 * i + 4 * g) * ES;
      if constexpr (ODT == kF32) {
        *reinterpret_cast<f32x4*>(at) = v;
      } else {
        *reinterpret_cast<v2u*>(at) = v2u{bits16<ODT>(v[0]) | (uint32_t)bits16<ODT>(v[1]) << 16,
                                          bits16<ODT>(v[2]) | (uint32_t)bits16<ODT>(v[3]) << 16};
      }
    }
    wave_fence8();
#pragma unroll 4
    for (int e = lane; e < 16 * PIECES; e += 64) {
      const int m = m0 + 16 * j + e / PIECES, n = n0 + e % PIECES * PER;
      if (m >= a.m || n >= a.n) continue;
      const uint8_t* const from = out + (e / PIECES) * PITCH + 16 * (e % PIECES);
      uint8_t* const to = static_cast<uint8_t*>(a.y) + ((int64_t)m * a.n + n) * ES;
      if (n + PER <= a.n) {
        *(LRQ_GLOBAL v4u_any*)to = *reinterpret_cast<const v4u*>(from);
      } else {
        for (int i = 0; n + i < a.n; ++i) {
          if constexpr (ODT == kF32) gst<float>(to + 4 * i, reinterpret_cast<const float*>(from)[i]);
          else gst<uint16_t>(to + 2 * i, reinterpret_cast<const uint16_t*>(from)[i]);
        }
      }
    }
  }
}

template <int FN, int FM, int WN, int WM, int STAGES, bool DMA, bool EXACT>
__global__ __launch_bounds__(64 * WN * WM, 1) void k_mm8_tiles(MatmulArgs a, int tiles_m, int tiles_n) {
  constexpr int BN = 16 * FN * WN, BM = 16 * FM * WM, kLds = kTileLds<FN, FM, WN, WM, STAGES>;
  static_assert(WN * WM * 16 * (64 * FN + 16) <= kLds, "results pass through the stages");
  __shared__ __attribute__((aligned(16))) uint8_t lds[kLds];
  int tm, tn;
  tile_of(blockIdx.x, tiles_m, tiles_n, tm, tn);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wn = (wave / WM) * 16 * FN, wm = (wave % WM) * 16 * FM;
  const DenseTile src{a, tn * BN, tm * BM, (int)a.n - 1 - tn * BN, (int)a.m - 1 - tm * BM, DMA};
  f32x4 acc[FN][FM];
  tile_sums<FN, FM, WN, WM, STAGES, DMA, false, EXACT>(src, (int)a.k, lds, acc);
  if constexpr (EXACT) return store_tile<kF32>(a, acc, src.n0 + wn, src.m0 + wm, lds);
  else if (a.out_dtype == kBF16) return store_tile<kBF16>(a, acc, src.n0 + wn, src.m0 + wm, lds);
  else return store_tile<kF16>(a, acc, src.n0 + wn, src.m0 + wm, lds);
}

// ---------------------------------------------------------------------------
// Which kernel
// ---------------------------------------------------------------------------
static int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
static bool dma_ok(const MatmulArgs& a) {
  return a.k % 4 == 0 && a.ldx % 4 == 0 && reinterpret_cast<uintptr_t>(a.x) % 4 == 0 && reinterpret_cast<uintptr_t>(a.w) % 4 == 0;
}

template <int FN, int FM, int WN, int WM, int STAGES, bool DMA, bool EXACT>
static void launch_tiles(const MatmulArgs& a, hipStream_t stream) {
  const int tiles_m = (int)ceil_div(a.m, 16 * FM * WM), tiles_n = (int)ceil_div(a.n, 16 * FN * WN);
  hipLaunchKernelGGL((k_mm8_tiles<FN, FM, WN, WM, STAGES, DMA, EXACT>), dim3((unsigned)(tiles_m * tiles_n)), dim3(64 * WN * WM), 0, stream, a,
                     tiles_m, tiles_n);
}
template <int XDT, int NT, int MT, int D>
static void launch_rows(const MatmulArgs& a, int64_t x_lds, hipStream_t stream) {
  const int64_t sums = 4 * 256 * NT * MT * kRowWaves;
  const dim3 grid((unsigned)ceil_div(a.n, 16 * NT), (unsigned)ceil_div(a.m, 16 * MT));
  hipLaunchKernelGGL((k_mm8_rows<XDT, NT, MT, D>), grid, dim3(64 * kRowWaves), (unsigned)(sums > x_lds ? sums : x_lds), stream, a);
}

template <bool DMA, bool EXACT>
static void launch_tiles_of(const MatmulArgs& a, hipStream_t stream) {
  if constexpr (DMA && !EXACT)
    if (ceil_div(a.m, 256) * ceil_div(a.n, 256) >= 200) return launch_tiles<8, 4, 2, 4, 2, DMA, EXACT>(a, stream);
  if (ceil_div(a.m, 128) * ceil_div(a.n, 128) >= 200) return launch_tiles<4, 4, 2, 2, DMA ? 4 : 2, DMA, EXACT>(a, stream);
  launch_tiles<2, 2, 2, 2, DMA ? 4 : 2, DMA, EXACT>(a, stream);
}

bool matmul_quantizes(int64_t m, int64_t k) {
  return m <= 16 && m * (ceil_div(k, kBlk) * kBlk + 16 + 4 * ceil_div(k, kBlk)) <= 32768;
}

hipError_t launch_matmul(const MatmulArgs& a, int x_dtype, hipStream_t stream) {
  if (x_dtype >= 0) {
    const int64_t x_lds = a.m * (a.kb * kBlk + 16 + 4 * a.kb);
    if (x_dtype == kBF16) launch_rows<kBF16, 1, 1, 4>(a, x_lds, stream);
    else if (x_dtype == kF16) launch_rows<kF16, 1, 1, 4>(a, x_lds, stream);
    else launch_rows<kF32, 1, 1, 4>(a, x_lds, stream);
  } else if (a.m <= 16) {
    launch_rows<-1, 1, 1, 4>(a, 0, stream);
  } else if (a.m <= 32) {
    launch_rows<-1, 1, 2, 2>(a, 0, stream);
  } else if (a.m <= 64) {
    launch_rows<-1, 1, 4, 2>(a, 0, stream);
  } else if (a.out_dtype == kF32) {
    if (dma_ok(a)) launch_tiles_of<true, true>(a, stream);
    else launch_tiles_of<false, true>(a, stream);
  } else {
    if (dma_ok(a)) launch_tiles_of<true, false>(a, stream);
    else launch_tiles_of<false, false>(a, stream);
  }
  return hipGetLastError();
}

}  // namespace lrq
