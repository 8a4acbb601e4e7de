// Building blocks of the FP8 products on 128x128-tile weights (gfx950 only):
// matrix instructions on e4m3 codes, moves of codes into LDS, and the 1x128
// quantization of activations on the way into LDS.
//
// The product of two block-scaled matrices is a sum over K blocks of 128,
//   y[m][n] = sum_b (sa[m][b] sw[n / 128][b]) sum_{k in b} a[m][k] w[n][k].
// The outer sum is a float32 fma per block, with sa sw rounded to float32 first.
// The weight is the matrix instructions' first operand, so that a lane's four
// results belong to one token: one scale, four fmas.  The inner sum comes from
//   * one f8f6f4 instruction (K = 128) per 16 x 16 results.  Its products are
//     exact, but it aligns them to the largest one's exponent and drops what is
//     2^-13 below it, whichever shape is taken (measured: 1.5e-5 of the result's
//     norm with normal codes, where float32 sums have 1e-8).  A 16-bit result's
//     own rounding is a hundred times that; or
//   * EXACT: four bf16 instructions on the same codes, which are exact in bf16, as
//     are their products; sums are float32.  Half the rate, and conversions: 48 tokens
//     x [4096, 12288], the product and its join with weights from memory, 20.2 us
//     instead of 17.0.  Taken for float32 results and for what experts quantize
//     again; or
//   * for up to four tokens, float32 multiply-adds.
#pragma once

#include "lrq_device.hpp"

namespace lrq {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef unsigned int v4u_any __attribute__((ext_vector_type(4), aligned(1)));
typedef const LRQ_GLOBAL uint8_t* GlobalCodes;

constexpr int kBlk = 128;  // K of a block: of a scale and of a matrix instruction

// D[n][m] = sum over 128 k of W[n][k] A[m][k].  Lane l holds 32 codes of row
// n = l % 16 of W and of token m = l % 16 of A, any 32 of the block that W and A
// share: here 16-byte pieces l / 16 and l / 16 + 4 of the row's eight.  It gets
// rows n = 4 (l / 16) .. + 3 of token m = l % 16.
struct Codes32 {
  v4u lo, hi;
};
__device__ __forceinline__ f32x4 mma8(const Codes32& w, const Codes32& a) {
  const i32x8 x = {(int)w.lo.x, (int)w.lo.y, (int)w.lo.z, (int)w.lo.w, (int)w.hi.x, (int)w.hi.y, (int)w.hi.z, (int)w.hi.w};
  const i32x8 y = {(int)a.lo.x, (int)a.lo.y, (int)a.lo.z, (int)a.lo.w, (int)a.hi.x, (int)a.hi.y, (int)a.hi.z, (int)a.hi.w};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(x, y, f32x4{0.0f, 0.0f, 0.0f, 0.0f}, 0, 0, 0, 0, 0, 0);
}


// The same as bf16: piece q holds the codes of word pair q (lo.xy, lo.zw, hi.xy, hi.zw).
typedef __bf16 bf16x8v __attribute__((ext_vector_type(8)));
struct Wide32 {
  v4u q[4];
};
template <bool HI>
__device__ __forceinline__ uint32_t codes2_to_bf16(uint32_t w) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, HI));
}
__device__ __forceinline__ v4u widen_piece(const Codes32& a, int q) {
  const uint32_t w[8] = {a.lo.x, a.lo.y, a.lo.z, a.lo.w, a.hi.x, a.hi.y, a.hi.z, a.hi.w};
  return v4u{codes2_to_bf16<false>(w[2 * q]), codes2_to_bf16<true>(w[2 * q]), codes2_to_bf16<false>(w[2 * q + 1]),
             codes2_to_bf16<true>(w[2 * q + 1])};
}
__device__ __forceinline__ Wide32 widen(const Codes32& a) {
  return Wide32{{widen_piece(a, 0), widen_piece(a, 1), widen_piece(a, 2), widen_piece(a, 3)}};
}
__device__ __forceinline__ f32x4 mma16(v4u w, v4u a, f32x4 d) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8v, w), __builtin_bit_cast(bf16x8v, a), d, 0, 0, 0);
}
template <bool EXACT>
__device__ __forceinline__ auto operand(const Codes32& a) {
  if constexpr (EXACT) return widen(a);
  else return a;
}

// 16 codes from any address.
__device__ __forceinline__ v4u load_codes(GlobalCodes p) { return *(const LRQ_GLOBAL v4u_any*)p; }
__device__ __forceinline__ v4u load_codes_nt(GlobalCodes p) { return __builtin_nontemporal_load((const LRQ_GLOBAL v4u_any*)p); }
// Codes [at, at + 16) of a row of k, zeros past its end, none of them read.
__device__ inline v4u load_codes_cut(GlobalCodes row, int at, int k) {
  if (at + 16 <= k) return load_codes(row + at);
  if (at >= k) return v4u{0, 0, 0, 0};
  uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < 16; ++i)
    if (at + i < k) w[i >> 2] |= (uint32_t)row[at + i] << (8 * (i & 3));
  return v4u{w[0], w[1], w[2], w[3]};
}

// Orders a wave's LDS accesses for the compiler; the hardware keeps one wave's
// in order by itself.
__device__ __forceinline__ void wave_fence8() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}
// Barrier of the work-group for its LDS accesses only: loads into registers
// stay in flight across it.
__device__ __forceinline__ void lds_barrier8() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// ---------------------------------------------------------------------------
// Memory straight into LDS
// ---------------------------------------------------------------------------
// 16 bytes a lane, at `off` from the descriptor's base (words past its
// size read as zeros), to 16 l + `lds`.  In assembly because the compiler, which cannot
// tell a tile's stages apart, waits for every such load before the
// next read of LDS; dma_wait() is the wait, before the barrier that hands the
// stage over.  The instruction has no register output.
typedef uint32_t Rsrc __attribute__((ext_vector_type(4)));
__device__ __forceinline__ Rsrc make_rsrc(const void* base, uint32_t bytes) {
  const uint64_t p = reinterpret_cast<uint64_t>(base);
  return Rsrc{(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)p),
              (uint32_t)__builtin_amdgcn_readfirstlane((int)((uint32_t)(p >> 32) & 0xFFFFu)),
              (uint32_t)__builtin_amdgcn_readfirstlane((int)bytes), 0x00020000u};
}
__device__ __forceinline__ void dma16(Rsrc r, uint32_t off, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
               :: "s"(lds), "v"(off), "s"(r) : "memory", "m0");
}
// Until at most N of the wave's loads are on their way: they arrive in order.
template <int N>
__device__ __forceinline__ void dma_wait() { asm volatile("s_waitcnt vmcnt(%0)" :: "n"(N) : "memory"); }
constexpr uint32_t kNoRow = 0x80000000u;  // an offset past every descriptor's size (below 2^31)

// ---------------------------------------------------------------------------
// Quantizing activations (1 x 128 blocks, weight_quantizer.py:59-71 in float32)
// ---------------------------------------------------------------------------
// 8 elements [at, at + 8) of a row of k, zeros past its end.
template <int DT>
__device__ __forceinline__ void load_acts(const void* row, int at, int k, float* v) {
  if constexpr (DT == kF32) {
    const float* p = static_cast<const float*>(row) + at;
    if (at + 8 <= k) {
      const v4u a = load_live(p), b = load_live(p + 4);
      const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = u2f(w[i]);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = at + i < k ? gld<float>(p + i) : 0.0f;
    }
  } else {
    const uint16_t* p = static_cast<const uint16_t*>(row) + at;
    uint32_t h[8];
    if (at + 8 <= k) {
      const v4u a = load_live(p);
      const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
      for (int i = 0; i < 8; ++i) h[i] = (w[i >> 1] >> (16 * (i & 1))) & 0xFFFFu;
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) h[i] = at + i < k ? gld<uint16_t>(p + i) : 0u;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = DT == kBF16 ? u2f(h[i] << 16) : f16_to_f32(h[i]);
  }
}

// The codes of 8 elements of a block that 16 neighbouring lanes hold, and its scale.
__device__ __forceinline__ v2u quant8(const float* v, float& scale) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t a = f2u(v[i]) & 0x7FFFFFFFu;
    m = a > m ? a : m;
  }
  const BlockScale b = block_scale<kF32>(group_max<16>(m), false);
  scale = b.s;
  if (b.kind >= kScaleInf) {
    uint32_t w[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i >> 2] |= special_code<kF32>(v[i], b) << (8 * (i & 3));
    return v2u{w[0], w[1]};
  }
  float q[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) q[i] = block_quot<kF32>(v[i], b);
  return v2u{cvt_e4m3x4(q[0], q[1], q[2], q[3]), cvt_e4m3x4(q[4], q[5], q[6], q[7])};
}

// ---------------------------------------------------------------------------
// Many tokens: tiles through LDS
// ---------------------------------------------------------------------------
// The sums of a tile of BM = 16 FM WM tokens and BN = 16 FN WN weight rows by
// WN x WM waves, each its 16 FN x 16 FM of it.  K goes block by block through a
// ring of STAGES in LDS: codes of both operands in rows of 128 bytes whose
// 16-byte pieces stand at places (piece ^ row / 2), so that reads of one piece
// from 16 rows fall into all 64 banks.  Behind the ring stand the scales of four
// blocks at a time, and of the next four.  A wave keeps the block of its tokens in
// registers and takes the weight 16 rows at a time; a result is scaled into the
// sums three matrix instructions after its own, which the compiler, left to
// itself, does at once, and waits (8192^3 without any loads 374 us, 334 as here).
//
// DMA (rows are 4-byte aligned): codes and scales go from memory straight into
// LDS, STAGES - 1 blocks ahead, each wave waiting only for its own part of the
// oldest.  Otherwise (any address): through registers, kTileSets blocks ahead.
//
// Src gives: w_bytes(), x_bytes(), sw_bytes(), sx_bytes() and the operands'
// bases w(), x(), sw(), sx();
//   w_off(r), x_off(r): the byte offset of a tile row, kNoRow for none (its sums
//   are not stored; without DMA some row that is there instead);
//   sx_off(r): of the scales of tile row r of the tokens, sw_off(s) of those of
//   weight rows 16 s .. (one scale for 16 rows); of some row that is there, if none.
//   kSkip: waves without a token, of the tokens() that are there, multiply nothing;
//   kCut: k may be no multiple of 16.
// EACH: the scales of a wave's weight rows differ; otherwise the first is for all.
constexpr int kTileSets = 2;
template <int FN, int FM, int WN, int WM>
constexpr int kTileStage = 16 * (FN * WN + FM * WM) * kBlk;
template <int FN, int FM, int WN, int WM>
constexpr int kTileScaleWaves = (16 * FM * WM + 63) / 64 + (FN * WN + 63) / 64;  // a thread for every 16 bytes of scales
template <int FN, int FM, int WN, int WM>
constexpr int kTileScales = 1024 * kTileScaleWaves<FN, FM, WN, WM>;  // of four blocks
template <int FN, int FM, int WN, int WM, int STAGES>
constexpr int kTileLds = STAGES * kTileStage<FN, FM, WN, WM> + 2 * kTileScales<FN, FM, WN, WM>;

// Blocks [kb0, kb1) of K.
template <int FN, int FM, int WN, int WM, int STAGES, bool DMA, bool EACH, bool EXACT, class Src>
__device__ __forceinline__ void tile_sums(const Src& src, int k, int kb0, int kb1, uint8_t* lds, f32x4 (&acc)[FN][FM]) {
  constexpr int T = 64 * WN * WM, BN = 16 * FN * WN, BM = 16 * FM * WM, TILES = FN * FM, LAG = TILES > 4 ? 3 : TILES > 1 ? 1 : 0;
  // 16-byte pieces a thread moves per block; of few tokens the first waves' threads alone
  constexpr int PW = BN * 8 / T, PX = BM * 8 / T > 0 ? BM * 8 / T : 1, XWAVES = BM * 8 / 64 / PX;
  constexpr int SW = (BM + 63) / 64 * 64, SWAVES = kTileScaleWaves<FN, FM, WN, WM>;  // scales: tokens' threads, then weights'
  constexpr int kStage = kTileStage<FN, FM, WN, WM>, kScales = kTileScales<FN, FM, WN, WM>;
  static_assert(PW * T == BN * 8 && PX * XWAVES * 64 == BM * 8 && T % 128 == 0 && SWAVES <= WN * WM, "");
  static_assert(XWAVES == WN * WM || DMA, "");
  static_assert(STAGES >= 2 && STAGES <= 5, "the next four blocks' scales arrive before them");
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c = lane & 15, g = lane >> 4;
  const int wn = (wave / WM) * 16 * FN, wm = (wave % WM) * 16 * FM;
  const int kb_n = kb1 - kb0;
  const int piece = (tid & 7) ^ ((tid >> 4) & 7);  // of tile rows (T / 8) p + tid / 8
  const bool moves_x = XWAVES == WN * WM || wave < XWAVES, moves_s = SWAVES == WN * WM || wave < SWAVES;
  uint32_t wo[PW], xo[PX];
#pragma unroll
  for (int p = 0; p < PW; ++p) wo[p] = src.w_off((T / 8) * p + (tid >> 3)) + 16 * piece;
#pragma unroll
  for (int p = 0; p < PX; ++p) xo[p] = (moves_x ? src.x_off((T / 8) * p + (tid >> 3)) : 0) + 16 * piece;
  // the thread's scales: of a token, or of 16 weight rows
  const bool tokens = wave < SW / 64;
  const uint32_t so = (tokens ? tid < BM ? src.sx_off(tid) : kNoRow : tid < SW + BN / 16 ? src.sw_off(tid - SW) : kNoRow) + 4 * kb0;
  uint8_t* const scales = lds + STAGES * kStage;
#pragma unroll
  for (int i = 0; i < FN; ++i)
#pragma unroll
    for (int j = 0; j < FM; ++j) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

  const int at0 = 16 * (g ^ (c >> 1)), at1 = 16 * ((g + 4) ^ (c >> 1));
  // `between(t)` runs after the block's matrix instruction t
  auto multiply = [&](const uint8_t* stage, int kb, auto between) {
    const uint8_t* const cw = stage + 128 * (wn + c);
    const uint8_t* const cx = stage + 128 * (BN + wm + c);
    const float* const sc = reinterpret_cast<const float*>(scales + (kb >> 2 & 1) * kScales) + (kb & 3);
    float s[FM], si[EACH ? FN : 1];
#pragma unroll
    for (int j = 0; j < FM; ++j) s[j] = sc[4 * (wm + 16 * j + c)];
#pragma unroll
    for (int i = 0; i < (EACH ? FN : 1); ++i) si[i] = sc[4 * (SW + wn / 16 + i)];
    decltype(operand<EXACT>(Codes32{})) x[FM];
    Codes32 w[2];
    w[0] = {*reinterpret_cast<const v4u*>(cw + at0), *reinterpret_cast<const v4u*>(cw + at1)};
#pragma unroll
    for (int j = 0; j < FM; ++j)
      x[j] = operand<EXACT>({*reinterpret_cast<const v4u*>(cx + 2048 * j + at0), *reinterpret_cast<const v4u*>(cx + 2048 * j + at1)});
    if constexpr (!EACH) {
#pragma unroll
      for (int j = 0; j < FM; ++j) s[j] *= si[0];
    }
    auto scale = [&](int i, int j, const f32x4& p) {
      const float f = EACH ? s[j] * si[EACH ? i : 0] : s[j];
#pragma unroll
      for (int r = 0; r < 4; ++r) acc[i][j][r] = __builtin_fmaf(p[r], f, acc[i][j][r]);
    };
    if constexpr (EXACT) {
      // a strip's FM chains of four instructions side by side; between them the strip
      // before is scaled and the next one's codes widened
      f32x4 p[2][FM];
      Wide32 wide[2];
      wide[0] = widen(w[0]);
#pragma unroll
      for (int i = 0; i < FN; ++i) {
        if (i + 1 < FN)
          w[(i + 1) & 1] = {*reinterpret_cast<const v4u*>(cw + 2048 * (i + 1) + at0),
                            *reinterpret_cast<const v4u*>(cw + 2048 * (i + 1) + at1)};
#pragma unroll
        for (int q = 0; q < 4; ++q) {
#pragma unroll
          for (int j = 0; j < FM; ++j)
            p[i & 1][j] = mma16(wide[i & 1].q[q], x[j].q[q], q == 0 ? f32x4{0.0f, 0.0f, 0.0f, 0.0f} : p[i & 1][j]);
#pragma unroll
          for (int j = q * FM / 4; j < (q + 1) * FM / 4; ++j) {
            if (i > 0) scale(i - 1, j, p[(i + 1) & 1][j]);
            between(i * FM + j);
          }
          if (i + 1 < FN) wide[(i + 1) & 1].q[q] = widen_piece(w[(i + 1) & 1], q);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
#pragma unroll
      for (int j = 0; j < FM; ++j) scale(FN - 1, j, p[(FN - 1) & 1][j]);
    } else {
      f32x4 p[LAG + 1];
#pragma unroll
      for (int i = 0; i < FN; ++i) {
        if (i + 1 < FN)
          w[(i + 1) & 1] = {*reinterpret_cast<const v4u*>(cw + 2048 * (i + 1) + at0),
                            *reinterpret_cast<const v4u*>(cw + 2048 * (i + 1) + at1)};
#pragma unroll
        for (int j = 0; j < FM; ++j) {
          const int t = i * FM + j;
          p[t % (LAG + 1)] = mma8(w[i & 1], x[j]);
          if (t >= LAG) scale((t - LAG) / FM, (t - LAG) % FM, p[(t - LAG) % (LAG + 1)]);
          between(t);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
#pragma unroll
      for (int t = TILES - LAG; t < TILES; ++t) scale(t / FM, t % FM, p[t % (LAG + 1)]);
    }
  };

  if constexpr (DMA) {
    const Rsrc rw = make_rsrc(src.w(), src.w_bytes()), rx = make_rsrc(src.x(), src.x_bytes());
    const Rsrc rs = tokens ? make_rsrc(src.sx(), src.sx_bytes()) : make_rsrc(src.sw(), src.sw_bytes());
    const uint32_t to = (uint32_t)reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) uint8_t*)lds) + 1024 * wave;
    // pieces [p0, p1) of a block; blocks past the last are asked for too, so that every
    // wait counts the same, and read as zeros
    auto fetch = [&](int kb, int stage, int p0, int p1) {
      const uint32_t at = (uint32_t)((kb0 + kb) * kBlk), past = kb < kb_n && (int)at + 16 * piece < k ? 0 : kNoRow;
      const uint32_t here = to + (uint32_t)(stage * kStage);
#pragma unroll
      for (int p = 0; p < PW + PX; ++p) {
        if (p < p0 || p >= p1) continue;
        if (p < PW) dma16(rw, (wo[p < PW ? p : 0] + at) | past, here + 128 * (T / 8) * p);
        else if (moves_x) dma16(rx, (xo[p < PW ? 0 : p - PW] + at) | past, here + 128 * (BN + (T / 8) * (p - PW)));
      }
    };
    auto fetch_scales = [&](int kb) {  // of blocks kb .. kb + 3; those past a row's end are the next row's, and not used
      if (moves_s) dma16(rs, (so + 4 * kb) | (kb < kb_n ? 0 : kNoRow), to + (uint32_t)(STAGES * kStage + (kb >> 2 & 1) * kScales));
    };
    // a row's last codes, where 16 bytes would reach past its end: one row a thread
    const bool cut = Src::kCut && k % 16 != 0 && kb1 * kBlk >= k;
    v4u last = {0, 0, 0, 0};
    if (cut && tid < BN + BM) {
      const uint32_t off = tid < BN ? src.w_off(tid) : src.x_off(tid - BN);
      const GlobalCodes row = (GlobalCodes)(tid < BN ? src.w() : src.x()) + (off + (k & ~15));
      if (off != kNoRow) {
        last.x = gld<uint32_t>((const void*)row);
        if (k % 16 > 4) last.y = gld<uint32_t>((const void*)(row + 4));
        if (k % 16 > 8) last.z = gld<uint32_t>((const void*)(row + 8));
      }
    }
    fetch_scales(0);
#pragma unroll
    for (int s = 0; s + 1 < STAGES; ++s) fetch(s, s, 0, PW + PX);
    int stage = 0, free = STAGES - 1;
    for (int kb = 0; kb < kb_n; kb += 4) {
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        if (kb + r >= kb_n) break;
        // on their way since this block's codes were asked for: the blocks between, and scales
        constexpr int kPer = STAGES - 2;
        const bool more = r >= 1 && r <= STAGES - 2 && moves_s;
        if (moves_x) more ? dma_wait<kPer * (PW + PX) + 1>() : dma_wait<kPer * (PW + PX)>();
        else more ? dma_wait<kPer * PW + 1>() : dma_wait<kPer * PW>();
        lds_barrier8();  // every wave's part of this block is there, and every read of the last is done
        if (cut && kb + r == kb_n - 1) {
          static_assert(BN + BM <= T || !Src::kCut, "");
          if (tid < BN + BM) *reinterpret_cast<v4u*>(lds + stage * kStage + 128 * tid + 16 * ((k % kBlk / 16) ^ (tid >> 1 & 7))) = last;
          lds_barrier8();
        }
        // the next loads go out among the first half of the matrix instructions: all at
        // once they would hold up the wave, whose reads of LDS stand behind them
        constexpr int H = TILES >= 2 ? TILES / 2 : 1, N = PW + PX;
        auto next = [&](int t) {
          if (t == 0 && r == 0) fetch_scales(kb + 4);
          if (t < H) fetch(kb + r + STAGES - 1, free, t * N / H, (t + 1) * N / H);
        };
        if (!Src::kSkip || wm < src.tokens()) {
          multiply(lds + stage * kStage, kb + r, next);
        } else {
#pragma unroll
          for (int t = 0; t < H; ++t) next(t);
        }
        free = stage;
        stage = stage + 1 < STAGES ? stage + 1 : 0;
      }
    }
    dma_wait<0>();
    lds_barrier8();
  } else {
    v4u gw[kTileSets][PW], gx[kTileSets][PX];
    float gs[kTileSets];
    const uint8_t* const sb = reinterpret_cast<const uint8_t*>(tokens ? src.sx() : src.sw());
    auto fetch = [&](int kb, int set) {
      const int at = kb < kb_n ? (kb0 + kb) * kBlk : k;
      if (at + kBlk <= k) {
#pragma unroll
        for (int p = 0; p < PW; ++p) gw[set][p] = load_codes((GlobalCodes)src.w() + (wo[p] + at));
#pragma unroll
        for (int p = 0; p < PX; ++p) gx[set][p] = load_codes((GlobalCodes)src.x() + (xo[p] + at));
      } else {
#pragma unroll
        for (int p = 0; p < PW; ++p) gw[set][p] = load_codes_cut((GlobalCodes)src.w() + (wo[p] - 16 * piece), at + 16 * piece, k);
#pragma unroll
        for (int p = 0; p < PX; ++p) gx[set][p] = load_codes_cut((GlobalCodes)src.x() + (xo[p] - 16 * piece), at + 16 * piece, k);
      }
      gs[set] = so < kNoRow && kb < kb_n ? gld<float>(sb + (so + 4 * kb)) : 0.0f;
    };
    auto put = [&](int set, int kb) {
      uint8_t* const s = lds + (kb & 1) * kStage + 16 * tid;
#pragma unroll
      for (int p = 0; p < PW; ++p) *reinterpret_cast<v4u*>(s + 128 * (T / 8) * p) = gw[set][p];
#pragma unroll
      for (int p = 0; p < PX; ++p) *reinterpret_cast<v4u*>(s + 128 * (BN + (T / 8) * p)) = gx[set][p];
      if (moves_s) reinterpret_cast<float*>(scales + (kb >> 2 & 1) * kScales)[4 * tid + (kb & 3)] = gs[set];
    };
#pragma unroll
    for (int s = 0; s < kTileSets; ++s) fetch(s, s);
    put(0, 0);
    fetch(kTileSets, 0);
    for (int kb = 0; kb < kb_n; kb += 2 * kTileSets) {
#pragma unroll
      for (int r = 0; r < 2 * kTileSets; ++r) {
        if (kb + r >= kb_n) break;
        lds_barrier8();
        put((r + 1) % kTileSets, kb + r + 1);
        fetch(kb + r + 1 + kTileSets, (r + 1) % kTileSets);
        multiply(lds + (r & 1) * kStage, kb + r, [](int) {});
      }
    }
    lds_barrier8();
  }
}

// ---------------------------------------------------------------------------
// A few tokens: dot products
// ---------------------------------------------------------------------------
// Up to four tokens are bound by the weight's bytes and by latency.  A wave takes
// whole rows, 16 codes a lane and 1 KiB an instruction, several of them ahead; 24
// vector instructions for 16 codes of a token keep up with memory, and nothing has
// to be turned round for matrix instructions.
struct Floats16 {
  float v[16];
};
__device__ __forceinline__ Floats16 codes_to_f32(v4u c) {
  const uint32_t w[4] = {c.x, c.y, c.z, c.w};
  Floats16 r;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const f32x2 lo = e4m3x2_to_f32<false>(w[i]), hi = e4m3x2_to_f32<true>(w[i]);
    r.v[4 * i] = lo.x, r.v[4 * i + 1] = lo.y, r.v[4 * i + 2] = hi.x, r.v[4 * i + 3] = hi.y;
  }
  return r;
}
__device__ __forceinline__ float dot16(const Floats16& a, const Floats16& b) {
  float s = a.v[0] * b.v[0];
#pragma unroll
  for (int i = 1; i < 16; ++i) s = __builtin_fmaf(a.v[i], b.v[i], s);
  return s;
}
// Over the wave; every lane is active.
__device__ __forceinline__ float lanes_sum(float v) {
#define LRQ_ADD_DPP(ctrl) v += u2f((uint32_t)__builtin_amdgcn_mov_dpp((int)f2u(v), ctrl, 0xF, 0xF, false))
  LRQ_ADD_DPP(0xB1);
  LRQ_ADD_DPP(0x4E);
  LRQ_ADD_DPP(0x141);
  LRQ_ADD_DPP(0x140);
#undef LRQ_ADD_DPP
  v += __shfl_xor(v, 16, 64);
  return v + __shfl_xor(v, 32, 64);
}
// The codes of `blocks` 1x128 blocks of a row of k values into LDS, and their
// scales: 16 lanes a block, T threads.
template <int DT, int T>
__device__ __forceinline__ void quant_row(const void* row, int k, int blocks, uint8_t* codes, float* scales) {
  const int l = threadIdx.x & 15;
  for (int b = threadIdx.x >> 4; b < blocks; b += T / 16) {
    float v[8], s;
    load_acts<DT>(row, b * kBlk + 8 * l, k, v);
    *reinterpret_cast<v2u*>(codes + b * kBlk + 8 * l) = quant8(v, s);
    if (l == 0) scales[b] = s;
  }
}

// ---------------------------------------------------------------------------
// Results
// ---------------------------------------------------------------------------
template <int DT>
__device__ __forceinline__ uint16_t bits16(float v) {
  if constexpr (DT == kBF16) return (f2u(v) & 0x7FFFFFFFu) > 0x7F800000u ? (uint16_t)0x7FC0u : (uint16_t)bf16_bits(v);
  else return (uint16_t)f16_bits(v);
}
__device__ __forceinline__ float load_as_f32(const void* p, int dtype, int64_t i) {
  if (dtype == kF32) return gld<float>(static_cast<const float*>(p) + i);
  const uint16_t b = gld<uint16_t>(static_cast<const uint16_t*>(p) + i);
  return dtype == kBF16 ? u2f((uint32_t)b << 16) : f16_to_f32(b);
}

// The tile of work-group `wg`.  Work-groups go to the 8 XCDs in turn; each XCD
// takes one run of the tiles, walked 8 tile rows at a time, so that the rows of
// both operands that its work-groups read together stay in its L2.
__device__ __forceinline__ void tile_of(int wg, int tiles_m, int tiles_n, int& tm, int& tn) {
  const int tiles = tiles_m * tiles_n, per = tiles >> 3;
  const int t = wg < 8 * per ? (wg & 7) * per + (wg >> 3) : wg;
  const int group = 8 * tiles_n, first = t / group * 8;
  const int rows = tiles_m - first < 8 ? tiles_m - first : 8;
  tm = first + (t % group) % rows;
  tn = (t % group) / rows;
}

}  // namespace lrq
