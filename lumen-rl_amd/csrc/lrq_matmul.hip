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
// Up to four tokens
// ---------------------------------------------------------------------------
// A wave makes R rows of up to M tokens, 1024 k at a time.  XDT: the type of x,
// which the work-group quantizes into LDS while the first weights are on their
// way, or -1: codes and scales.
template <int XDT, int M, int R>
__global__ __launch_bounds__(512) void k_mm8_dot(MatmulArgs a) {
  constexpr int D = 8 / R;  // chunks ahead
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int k = (int)a.k, kb_n = (int)a.kb, m_n = (int)a.m, chunks = (k + 1023) / 1024;
  const int64_t n0 = ((int64_t)blockIdx.x * 8 + wave) * R;
  const int64_t first = n0 < a.n ? n0 : a.n - 1;
  GlobalCodes w[R], x[M];
#pragma unroll
  for (int r = 0; r < R; ++r) w[r] = (GlobalCodes)a.w + (n0 + r < a.n ? n0 + r : a.n - 1) * a.k;
#pragma unroll
  for (int m = 0; m < M; ++m) x[m] = (GlobalCodes)a.x + (m < m_n ? m : m_n - 1) * a.ldx;
  const float* const sw = a.sw + first / kBlk * a.kb;
  const int pitch = kb_n * kBlk;
  const float* const sx = XDT >= 0 ? reinterpret_cast<const float*>(lds + m_n * pitch) : a.sx;
  struct Chunk {
    v4u w[R], x[XDT >= 0 ? 1 : M];
    float s;
  } st[D];
  auto load = [&](Chunk& c, int i) {
    if (i >= chunks) return;
    const int at = 1024 * i + 16 * lane;
    if (1024 * i + 1024 <= k) {
#pragma unroll
      for (int r = 0; r < R; ++r) c.w[r] = load_codes_nt(w[r] + at);
      if constexpr (XDT < 0)
#pragma unroll
        for (int m = 0; m < M; ++m) c.x[m] = load_codes(x[m] + at);
    } else {
#pragma unroll
      for (int r = 0; r < R; ++r) c.w[r] = load_codes_cut(w[r], at, k);
      if constexpr (XDT < 0)
#pragma unroll
        for (int m = 0; m < M; ++m) c.x[m] = load_codes_cut(x[m], at, k);
    }
    c.s = gld<float>(sw + (at / kBlk < kb_n ? at / kBlk : kb_n - 1));
  };
#pragma unroll
  for (int d = 0; d < D; ++d) load(st[d], d);
  if constexpr (XDT >= 0) {
    for (int m = 0; m < m_n; ++m)
      quant_row<XDT, 512>(static_cast<const uint8_t*>(a.x) + m * a.ldx * (XDT == kF32 ? 4 : 2), k, kb_n, lds + m * pitch,
                          const_cast<float*>(sx) + m * kb_n);
    lds_barrier8();
  }
  float acc[R][M];
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int m = 0; m < M; ++m) acc[r][m] = 0.0f;
  for (int i0 = 0; i0 < chunks; i0 += D) {
#pragma unroll
    for (int d = 0; d < D; ++d) {
      if (i0 + d >= chunks) break;
      const int at = 1024 * (i0 + d) + 16 * lane, kb = at / kBlk < kb_n ? at / kBlk : kb_n - 1;
      Floats16 wf[R];
#pragma unroll
      for (int r = 0; r < R; ++r) wf[r] = codes_to_f32(st[d].w[r]);
#pragma unroll
      for (int m = 0; m < M; ++m) {
        const int mm = m < m_n ? m : m_n - 1;
        Floats16 xf;  // past the row's end w is 0 and x any
        if constexpr (XDT >= 0) xf = codes_to_f32(*reinterpret_cast<const v4u*>(lds + mm * pitch + (at < pitch ? at : pitch - 16)));
        else xf = codes_to_f32(st[d].x[m]);
        const float s = (XDT >= 0 ? sx[mm * kb_n + kb] : gld<float>(sx + mm * a.kb + kb)) * st[d].s;
#pragma unroll
        for (int r = 0; r < R; ++r) acc[r][m] = __builtin_fmaf(dot16(wf[r], xf), s, acc[r][m]);
      }
      load(st[d], i0 + d + D);
    }
  }
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int m = 0; m < M; ++m) {
      float sum = lanes_sum(acc[r][m]);
      const int64_t n = n0 + r;
      if (lane != 0 || m >= m_n || n >= a.n) continue;
      if (a.bias != nullptr) sum += load_as_f32(a.bias, a.bias_dtype, n);
      store_y(a, m * a.n + n, sum);
    }
}

// ---------------------------------------------------------------------------
// More: tiles
// ---------------------------------------------------------------------------
struct DenseTile {
  static constexpr bool kCut = true, kSkip = false;  // (the branch costs 256 x 256 tiles their registers)
  const MatmulArgs& a;
  int n0, m0, n_last, m_last;  // n_last, m_last: within the tile
  bool dma;
  __device__ const uint8_t* w() const { return a.w + (int64_t)n0 * a.k; }
  __device__ const uint8_t* x() const { return static_cast<const uint8_t*>(a.x) + (int64_t)m0 * a.ldx; }
  __device__ uint32_t w_bytes() const { return (uint32_t)((n_last < 255 ? n_last + 1 : 256) * a.k); }
  __device__ uint32_t x_bytes() const { return (uint32_t)((m_last < 255 ? m_last : 255) * a.ldx + a.k); }
  __device__ uint32_t w_off(int r) const { return r <= n_last ? (uint32_t)(r * a.k) : dma ? kNoRow : (uint32_t)(n_last * a.k); }
  __device__ uint32_t x_off(int r) const { return r <= m_last ? (uint32_t)(r * a.ldx) : dma ? kNoRow : (uint32_t)(m_last * a.ldx); }
  __device__ int tokens() const { return m_last + 1; }
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

// SPLIT: K in gridDim.y parts, whose sums go to `parts` [part][token][row] in float32.
template <int FN, int FM, int WN, int WM, int STAGES, bool DMA, bool EXACT, bool SPLIT>
__global__ __launch_bounds__(64 * WN * WM, 1) void k_mm8_tiles(MatmulArgs a, int tiles_m, int tiles_n, float* parts) {
  constexpr int BN = 16 * FN * WN, BM = 16 * FM * WM, kLds = kTileLds<FN, FM, WN, WM, STAGES>;
  static_assert(WN * WM * 16 * (64 * FN + 16) <= kLds, "results pass through the stages");
  __shared__ __attribute__((aligned(16))) uint8_t lds[kLds];
  int tm, tn;
  tile_of(blockIdx.x, tiles_m, tiles_n, tm, tn);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wn = (wave / WM) * 16 * FN, wm = (wave % WM) * 16 * FM;
  const DenseTile src{a, tn * BN, tm * BM, (int)a.n - 1 - tn * BN, (int)a.m - 1 - tm * BM, DMA};
  f32x4 acc[FN][FM];
  if constexpr (SPLIT) {
    const int steps = ((int)a.kb + gridDim.y - 1) / gridDim.y, kb0 = steps * blockIdx.y;
    tile_sums<FN, FM, WN, WM, STAGES, DMA, false, EXACT>(src, (int)a.k, kb0, kb0 + steps < a.kb ? kb0 + steps : (int)a.kb, lds, acc);
    MatmulArgs part = a;
    part.bias = nullptr, part.y = parts + blockIdx.y * a.m * a.n;
    store_tile<kF32>(part, acc, src.n0 + wn, src.m0 + wm, lds);
  } else {
    tile_sums<FN, FM, WN, WM, STAGES, DMA, false, EXACT>(src, (int)a.k, 0, (int)a.kb, lds, acc);
    if constexpr (EXACT) return store_tile<kF32>(a, acc, src.n0 + wn, src.m0 + wm, lds);
    else if (a.out_dtype == kBF16) return store_tile<kBF16>(a, acc, src.n0 + wn, src.m0 + wm, lds);
    else return store_tile<kF16>(a, acc, src.n0 + wn, src.m0 + wm, lds);
  }
}

// The parts' sum, in their order.
__global__ __launch_bounds__(256) void k_mm8_join(MatmulArgs a, const float* parts, int count) {
  const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x, cells = a.m * a.n;
  if (at >= cells) return;
  float sum = gld<float>(parts + at);
  for (int p = 1; p < count; ++p) sum += gld<float>(parts + p * cells + at);
  if (a.bias != nullptr) sum += load_as_f32(a.bias, a.bias_dtype, at % a.n);
  store_y(a, at, sum);
}

// ---------------------------------------------------------------------------
// Rows at a pitch of 16 bytes
// ---------------------------------------------------------------------------
// Codes whose rows are not 4-byte aligned go through registers, at less than half the
// speed; with many tokens they are copied to rows of kp = 16 ceil(k / 16) first, zeros
// at the end (8192 tokens x [12288, 4097] 448 us, 1000 as they are; 4096 x [4096, 4097]
// 89 and 192; 1024 tokens 51 and 54, 512 36 and 31).  Codes at odd addresses, or rows at
// an odd pitch, of a k that 4 divides are left as they are.
//
// fp8_block_linear quantizes x into rows at such a pitch anyway, through the caches, where
// the product finds them: with weights from memory, all launches of a call together, 48
// tokens x [4096, 12288] 21.0 us and 8192 x [4096, 4096] 149, by k_row, which stores past
// the caches, 21.9 and 151; 1024 x [4096, 4096] 36 by both.
__global__ __launch_bounds__(256) void k_mm8_pad(const uint8_t* from, int64_t ld, uint32_t pieces, int k, uint32_t per, uint8_t* to) {
  const uint32_t i = blockIdx.x * 256u + threadIdx.x;
  if (i >= pieces) return;
  const uint32_t row = i / per, at = 16 * (i - row * per);
  *(LRQ_GLOBAL v4u*)(to + 16 * (int64_t)i) = load_codes_cut((GlobalCodes)from + row * ld, (int)at, k);
}
template <int DT>
__global__ __launch_bounds__(256) void k_mm8_quant(const void* x, int64_t ld, uint32_t blocks, int k, uint32_t kb, int64_t kp, uint8_t* codes,
                                                   float* scales) {
  const uint32_t b = blockIdx.x * 16u + (threadIdx.x >> 4);
  if (b >= blocks) return;  // 16 lanes at once
  const uint32_t row = b / kb, at = (b - row * kb) * kBlk + 8 * (threadIdx.x & 15);
  float v[8], s;
  load_acts<DT>(static_cast<const uint8_t*>(x) + row * ld * (DT == kF32 ? 4 : 2), (int)at, k, v);
  const v2u q = quant8(v, s);
  if (at < kp) *(LRQ_GLOBAL v2u*)(codes + row * kp + at) = q;
  if ((threadIdx.x & 15) == 0) gst<float>(scales + b, s);
}

// ---------------------------------------------------------------------------
// Which kernel
// ---------------------------------------------------------------------------
static int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
static bool dma_ok(const MatmulArgs& a) {
  return a.k % 4 == 0 && a.ldx % 4 == 0 && reinterpret_cast<uintptr_t>(a.x) % 4 == 0 && reinterpret_cast<uintptr_t>(a.w) % 4 == 0;
}

template <int FN, int FM, int WN, int WM, int STAGES, bool DMA, bool EXACT, bool SPLIT = false>
static void launch_tiles(const MatmulArgs& a, hipStream_t stream, float* parts = nullptr, int count = 1) {
  const int tiles_m = (int)ceil_div(a.m, 16 * FM * WM), tiles_n = (int)ceil_div(a.n, 16 * FN * WN);
  hipLaunchKernelGGL((k_mm8_tiles<FN, FM, WN, WM, STAGES, DMA, EXACT, SPLIT>), dim3((unsigned)(tiles_m * tiles_n), (unsigned)count),
                     dim3(64 * WN * WM), 0, stream, a, tiles_m, tiles_n, parts);
}
template <int XDT, int M, int R>
static void launch_dot(const MatmulArgs& a, hipStream_t stream) {
  const unsigned lds = XDT >= 0 ? (unsigned)(a.m * a.kb * (kBlk + 4)) : 0;
  hipLaunchKernelGGL((k_mm8_dot<XDT, M, R>), dim3((unsigned)ceil_div(a.n, 8 * R)), dim3(512), lds, stream, a);
}
// Two rows a wave from 4096 rows on, so that a token's codes are widened for both; with
// fewer rows, twice the waves.  us by one and by two, weights from memory: one token x
// [2048, 4096] 5.0 and 5.8, [4096, 4096] 7.1 and 6.9, [12288, 4096] 13.6 and 13.2; four
// tokens 9.0 and 11.2, 12.7 and 12.3, 32 and 25.  (Of a K of 1024 one row stays ahead
// up to 6144 rows, by 0.6 us at most; of 12288 two are ahead from 3000 on.)
template <int XDT>
static void launch_dots(const MatmulArgs& a, hipStream_t stream) {
  if (a.m == 1) a.n >= 4096 ? launch_dot<XDT, 1, 2>(a, stream) : launch_dot<XDT, 1, 1>(a, stream);
  else if (a.m == 2) a.n >= 4096 ? launch_dot<XDT, 2, 2>(a, stream) : launch_dot<XDT, 2, 1>(a, stream);
  else a.n >= 4096 ? launch_dot<XDT, 4, 2>(a, stream) : launch_dot<XDT, 4, 1>(a, stream);
}

// Tiles, by what a round of them over the chip takes (us for K = 4096, measured one
// shape at a time): `one` with at most a work-group on each CU, `full` with as many
// as LDS allows (one of 256 x 256 and of 128 tokens x 256, two of the others).
// bf16: 1024 tokens x [12288, 4096] 56 us in 256 x 256, 64 in 128 x 256, 92 in 64 x
// 64; 1536 x [4096, 4096] 51, 34 and 46; 256 x [12288, 4096] 49, 32, 23 in 64 x 128,
// 29.  128 x 128 wins nowhere (1024 x [4096, 4096] 25, as 64 x 128), but for float32
// results, whose conversions take the registers of the larger ones: 3000 x [4096,
// 4096] 91 us, 105 in 64 x 128, 110 in 128 x 256.  So do loads by way of registers.
template <bool DMA, bool EXACT>
static void launch_tiles_of(const MatmulArgs& a, hipStream_t stream) {
  auto whole = [&](int64_t bm, int64_t bn, double full) { return (double)ceil_div(ceil_div(a.m, bm) * ceil_div(a.n, bn), 256) * full; };
  auto pairs = [&](int64_t bm, int64_t bn, double one, double full) {
    const int64_t tiles = ceil_div(a.m, bm) * ceil_div(a.n, bn);
    return tiles <= 256 ? one : tiles <= 512 ? one + (full - one) * (double)(tiles - 256) / 256 : full * (double)tiles / 512;
  };
  const double s = EXACT ? pairs(64, 64, 18, 26.5) : pairs(64, 64, 14.5, 18);
  const double u = EXACT ? pairs(64, 128, 26, 40) : pairs(64, 128, 16, 24.5);
  if constexpr (DMA && EXACT) {
    if (const double d = pairs(128, 128, 36, 62); d <= s && d <= u) return launch_tiles<4, 4, 2, 2, 2, DMA, EXACT>(a, stream);
  } else if constexpr (DMA) {
    const double b = whole(128, 256, 31), l = whole(256, 256, 49);
    if (l <= s && l <= u && l <= b) return launch_tiles<8, 4, 2, 4, 2, DMA, EXACT>(a, stream);
    if (b <= s && b <= u) return launch_tiles<4, 4, 4, 2, 3, DMA, EXACT>(a, stream);
  }
  if (u <= s) return launch_tiles<4, 2, 2, 2, DMA ? 3 : 2, DMA, EXACT>(a, stream);
  launch_tiles<2, 2, 2, 2, DMA && !EXACT ? 4 : 2, DMA, EXACT>(a, stream);
}

constexpr int64_t kDots = 4, kSplitRows = 64;
bool matmul_quantizes(int64_t m, int64_t k) { return m <= kDots && m * ceil_div(k, kBlk) * (kBlk + 4) <= 65536; }

// Parts of K: a work-group for every CU, of 3 blocks at least.  48 tokens x [4096,
// 12288], the product and its join with weights from memory: in 4 parts of 24 blocks
// 16.8 us, 18.5 in 8, 23 in 2, 36 in one; 64-row tiles, as 128-row ones are two times
// fewer.
static int64_t split_parts(int64_t m, int64_t n, int64_t k) {
  if (m <= kDots || m > kSplitRows) return 1;
  const int64_t tiles = ceil_div(n, 64), kb = ceil_div(k, kBlk);
  int64_t parts = 256 / tiles < kb / 3 ? 256 / tiles : kb / 3;
  if (parts < 2) return 1;
  return ceil_div(kb, ceil_div(kb, parts));  // none of them empty
}
static int64_t pitch16(int64_t k) { return (k + 15) / 16 * 16; }
static int64_t up256(int64_t v) { return (v + 255) / 256 * 256; }
bool matmul_repacks(int64_t m, int64_t n, int64_t k) {
  return k % 4 != 0 && m >= 1536 && n * pitch16(k) < int64_t(1) << 31 && m * pitch16(k) < int64_t(1) << 35;
}
int64_t matmul_workspace(int64_t m, int64_t n, int64_t k, bool x_packed) {
  if (matmul_repacks(m, n, k)) return up256(n * pitch16(k)) + (x_packed ? 0 : up256(m * pitch16(k)));
  const int64_t parts = split_parts(m, n, k);
  return parts > 1 ? 4 * parts * m * n : 0;
}

hipError_t launch_matmul_quant(const void* x, int dtype, int64_t ld, int64_t m, int64_t k, uint8_t* codes, float* scales, hipStream_t stream) {
  const int64_t kb = ceil_div(k, kBlk), kp = pitch16(k), es = dtype == kF32 ? 4 : 2;
  const int64_t most = (int64_t(1) << 27) / kb;  // rows of a launch, which has fewer than 2^32 threads, 16 of them a block
  for (int64_t r0 = 0; r0 < m; r0 += most) {
    const int64_t rows = m - r0 < most ? m - r0 : most;
    const dim3 grid((unsigned)ceil_div(rows * kb, 16)), block(256);
    const uint32_t blocks = (uint32_t)(rows * kb);
    const void* const from = static_cast<const uint8_t*>(x) + r0 * ld * es;
    uint8_t* const to = codes + r0 * kp;
    float* const s = scales + r0 * kb;
    if (dtype == kBF16) hipLaunchKernelGGL((k_mm8_quant<kBF16>), grid, block, 0, stream, from, ld, blocks, (int)k, (uint32_t)kb, kp, to, s);
    else if (dtype == kF16) hipLaunchKernelGGL((k_mm8_quant<kF16>), grid, block, 0, stream, from, ld, blocks, (int)k, (uint32_t)kb, kp, to, s);
    else hipLaunchKernelGGL((k_mm8_quant<kF32>), grid, block, 0, stream, from, ld, blocks, (int)k, (uint32_t)kb, kp, to, s);
    if (hipError_t e = hipGetLastError()) return e;
  }
  return hipSuccess;
}

static void pad_rows(const uint8_t* from, int64_t ld, int64_t rows, int64_t k, uint8_t* to, hipStream_t stream) {
  const int64_t per = pitch16(k) / 16, pieces = rows * per;
  hipLaunchKernelGGL(k_mm8_pad, dim3((unsigned)ceil_div(pieces, 256)), dim3(256), 0, stream, from, ld, (uint32_t)pieces, (int)k, (uint32_t)per, to);
}

template <bool EXACT>
static void launch_few(const MatmulArgs& a, float* sums, hipStream_t stream) {
  const int64_t parts = split_parts(a.m, a.n, a.k);
  if (parts > 1) {
    if (dma_ok(a)) launch_tiles<1, 4, 4, 1, 4, true, EXACT, true>(a, stream, sums, (int)parts);
    else launch_tiles<1, 4, 4, 1, 2, false, EXACT, true>(a, stream, sums, (int)parts);
    hipLaunchKernelGGL(k_mm8_join, dim3((unsigned)ceil_div(a.m * a.n, 256)), dim3(256), 0, stream, a, sums, (int)parts);
  } else if (dma_ok(a)) {
    launch_tiles<1, 4, 4, 1, 4, true, EXACT>(a, stream);
  } else {
    launch_tiles<1, 4, 4, 1, 2, false, EXACT>(a, stream);
  }
}

hipError_t launch_matmul(MatmulArgs a, int x_dtype, void* workspace, bool x_packed, hipStream_t stream) {
  if (matmul_repacks(a.m, a.n, a.k)) {
    const int64_t kp = pitch16(a.k);
    uint8_t* const w = static_cast<uint8_t*>(workspace);
    pad_rows(a.w, a.k, a.n, a.k, w, stream);
    if (!x_packed) {
      uint8_t* const x = w + up256(a.n * kp);
      pad_rows(static_cast<const uint8_t*>(a.x), a.ldx, a.m, a.k, x, stream);
      a.x = x, a.ldx = kp;
    }
    a.w = w, a.k = kp;
  }
  if (a.m <= kDots) {
    if (x_dtype == kBF16) launch_dots<kBF16>(a, stream);
    else if (x_dtype == kF16) launch_dots<kF16>(a, stream);
    else if (x_dtype == kF32) launch_dots<kF32>(a, stream);
    else launch_dots<-1>(a, stream);
  } else if (a.m <= kSplitRows) {
    if (a.out_dtype == kF32) launch_few<true>(a, static_cast<float*>(workspace), stream);
    else launch_few<false>(a, static_cast<float*>(workspace), stream);
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
