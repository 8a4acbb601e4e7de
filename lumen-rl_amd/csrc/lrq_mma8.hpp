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
//     are their products; sums are float32.  Half the rate, and conversions.  Taken
//     for float32 results, and wherever memory is the bound anyway (few tokens).
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
__device__ __forceinline__ Wide32 widen(const Codes32& a) {
  const uint32_t w[8] = {a.lo.x, a.lo.y, a.lo.z, a.lo.w, a.hi.x, a.hi.y, a.hi.z, a.hi.w};
  Wide32 r;
#pragma unroll
  for (int q = 0; q < 4; ++q)
    r.q[q] = v4u{codes2_to_bf16<false>(w[2 * q]), codes2_to_bf16<true>(w[2 * q]), codes2_to_bf16<false>(w[2 * q + 1]),
                 codes2_to_bf16<true>(w[2 * q + 1])};
  return r;
}
__device__ __forceinline__ f32x4 mma8(const Wide32& w, const Wide32& a) {
  f32x4 d = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int q = 0; q < 4; ++q)
    d = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8v, w.q[q]), __builtin_bit_cast(bf16x8v, a.q[q]), d, 0, 0, 0);
  return d;
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
// 16 bytes a lane, at `off` from the descriptor's base (zeros if off + 16 passes
// its size), to 16 l + `lds`.  In assembly because the compiler, which cannot
// tell the two stages of a tile apart, waits for every such load before the
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
               :: "s"(lds), "v"(off), "s"(r) : "memory");
}
__device__ __forceinline__ void dma_wait() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }
constexpr uint32_t kNoRow = 0x80000000u;  // an offset past every descriptor's size
constexpr int64_t kDmaBytes = 0x7FFFFF00ll;  // so a descriptor holds at most this

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
// WN x WM waves, each its 16 FN x 16 FM of it.  K goes block by block through
// two stages of LDS, codes of both operands in rows of 128 bytes whose 16-byte
// pieces stand at places (piece ^ row / 2): reads of one piece from 16 rows
// then fall into all 64 banks.  A wave keeps the block of its tokens in
// registers and takes the weight 16 rows at a time: FM matrix instructions,
// whose results the scales multiply into the sums one step later, between the
// next step's matrix instructions.
//
// DMA: codes go from memory straight into LDS; rows are 16-byte aligned.
// Otherwise any address: through registers, which costs 32 of them.
//
// Src gives: w_bytes(), x_bytes() and the operands' bases w(), x();
//   w_off(r), x_off(r): the byte offset of a tile row, kNoRow for none (its sums
//   are not stored; without DMA some row that is there instead);
//   sx(r): the scales of tile row r of the tokens (of some token, if none);
//   sw(i): the scales of the wave's weight rows 16 i .. (one scale for 16 rows).
// EACH: sw(i) differ; otherwise sw(0) is for all of a wave's rows.
template <int FN, int FM, int WN, int WM>
constexpr int kTileStage = 16 * (FN * WN + FM * WM) * kBlk;

template <int FN, int FM, int WN, int WM, bool DMA, bool EACH, bool EXACT, class Src>
__device__ __forceinline__ void tile_sums(const Src& src, int k, uint8_t* lds, f32x4 (&acc)[FN][FM]) {
  constexpr int T = 64 * WN * WM, BN = 16 * FN * WN, BM = 16 * FM * WM;
  constexpr int PW = BN * 8 / T, PX = BM * 8 / T;  // 16-byte pieces a thread moves per block
  constexpr int kStage = kTileStage<FN, FM, WN, WM>, SW = EACH ? FN : 1;
  static_assert(PW * T == BN * 8 && PX * T == BM * 8 && T % 128 == 0, "");
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c = lane & 15, g = lane >> 4;
  const int wn = (wave / WM) * 16 * FN, wm = (wave % WM) * 16 * FM;
  const int kb_n = (k + kBlk - 1) / kBlk;
  const int piece = (tid & 7) ^ ((tid >> 4) & 7);  // of tile rows (T / 8) p + tid / 8
  uint32_t wo[PW], xo[PX];
#pragma unroll
  for (int p = 0; p < PW; ++p) wo[p] = src.w_off((T / 8) * p + (tid >> 3)) + 16 * piece;
#pragma unroll
  for (int p = 0; p < PX; ++p) xo[p] = src.x_off((T / 8) * p + (tid >> 3)) + 16 * piece;
  // DMA: offsets past the row's end in the last block read as zeros
  Rsrc rw, rx;
  uint32_t to = 0;
  if constexpr (DMA) {
    rw = make_rsrc(src.w(), src.w_bytes());
    rx = make_rsrc(src.x(), src.x_bytes());
    to = (uint32_t)reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) uint8_t*)lds) + 1024 * wave;
  }
  v4u gw[DMA ? 1 : PW], gx[DMA ? 1 : PX];
  auto fetch = [&](int kb, int stage) {
    const uint32_t at = (uint32_t)(kb * kBlk);
    if constexpr (DMA) {
      const uint32_t past = (int)at + 16 * piece < k ? 0 : kNoRow;
#pragma unroll
      for (int p = 0; p < PW; ++p) dma16(rw, (wo[p] + at) | past, to + stage * kStage + 128 * (T / 8) * p);
#pragma unroll
      for (int p = 0; p < PX; ++p) dma16(rx, (xo[p] + at) | past, to + stage * kStage + 128 * (BN + (T / 8) * p));
    } else if ((int)at + kBlk <= k) {
#pragma unroll
      for (int p = 0; p < PW; ++p) gw[p] = load_codes((GlobalCodes)src.w() + (wo[p] + at));
#pragma unroll
      for (int p = 0; p < PX; ++p) gx[p] = load_codes((GlobalCodes)src.x() + (xo[p] + at));
    } else {
#pragma unroll
      for (int p = 0; p < PW; ++p) gw[p] = load_codes_cut((GlobalCodes)src.w() + (wo[p] - 16 * piece), (int)at + 16 * piece, k);
#pragma unroll
      for (int p = 0; p < PX; ++p) gx[p] = load_codes_cut((GlobalCodes)src.x() + (xo[p] - 16 * piece), (int)at + 16 * piece, k);
    }
  };
  auto put = [&](int stage) {
    if constexpr (!DMA) {
      uint8_t* const s = lds + stage * kStage + 16 * tid;
#pragma unroll
      for (int p = 0; p < PW; ++p) *reinterpret_cast<v4u*>(s + 128 * (T / 8) * p) = gw[p];
#pragma unroll
      for (int p = 0; p < PX; ++p) *reinterpret_cast<v4u*>(s + 128 * (BN + (T / 8) * p)) = gx[p];
    } else {
      dma_wait();
    }
  };
  const float* sxp[FM];
#pragma unroll
  for (int j = 0; j < FM; ++j) sxp[j] = src.sx(wm + 16 * j + c);
  const float* swp[SW];
#pragma unroll
  for (int i = 0; i < SW; ++i) swp[i] = src.sw(i);
  float sx[FM], sw[SW];
  auto scales = [&](int kb) {
#pragma unroll
    for (int j = 0; j < FM; ++j) sx[j] = gld<float>(sxp[j] + kb);
#pragma unroll
    for (int i = 0; i < SW; ++i) sw[i] = gld<float>(swp[i] + kb);
  };
  f32x4 p[FM], pp[FM];
  float sp[FM];
#pragma unroll
  for (int j = 0; j < FM; ++j) {
    pp[j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    sp[j] = 0.0f;
#pragma unroll
    for (int i = 0; i < FN; ++i) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  }
  fetch(0, 0);
  scales(0);
  put(0);
  lds_barrier8();
  const int at0 = 16 * (g ^ (c >> 1)), at1 = 16 * ((g + 4) ^ (c >> 1));
  for (int kb = 0; kb < kb_n; ++kb) {
    const uint8_t* const cw = lds + (kb & 1) * kStage + 128 * (wn + c);
    const uint8_t* const cx = lds + (kb & 1) * kStage + 128 * (BN + wm + c);
    if (kb + 1 < kb_n) fetch(kb + 1, (kb + 1) & 1);
    float s[FM], si[SW];
#pragma unroll
    for (int j = 0; j < FM; ++j) s[j] = sx[j];
#pragma unroll
    for (int i = 0; i < SW; ++i) si[i] = sw[i];
    if constexpr (!EACH) {
#pragma unroll
      for (int j = 0; j < FM; ++j) s[j] *= si[0];
    }
    if (kb + 1 < kb_n) scales(kb + 1);
    decltype(operand<EXACT>(Codes32{})) x[FM];
    Codes32 w[2];
#pragma unroll
    for (int j = 0; j < FM; ++j)
      x[j] = operand<EXACT>({*reinterpret_cast<const v4u*>(cx + 2048 * j + at0), *reinterpret_cast<const v4u*>(cx + 2048 * j + at1)});
    w[0] = {*reinterpret_cast<const v4u*>(cw + at0), *reinterpret_cast<const v4u*>(cw + at1)};
#pragma unroll
    for (int i = 0; i < FN; ++i) {
      if (i + 1 < FN)
        w[(i + 1) & 1] = {*reinterpret_cast<const v4u*>(cw + 2048 * (i + 1) + at0),
                          *reinterpret_cast<const v4u*>(cw + 2048 * (i + 1) + at1)};
      const auto wi = operand<EXACT>(w[i & 1]);
#pragma unroll
      for (int j = 0; j < FM; ++j) {
        p[j] = mma8(wi, x[j]);
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[(i + FN - 1) % FN][j][r] = __builtin_fmaf(pp[j][r], sp[j], acc[(i + FN - 1) % FN][j][r]);
      }
#pragma unroll
      for (int j = 0; j < FM; ++j) {
        pp[j] = p[j];
        sp[j] = EACH ? s[j] * si[EACH ? i : 0] : s[j];
      }
      __builtin_amdgcn_sched_barrier(0);  // or every strip's codes are read at once, into registers there are not
    }
    if (kb + 1 < kb_n) put((kb + 1) & 1);
    lds_barrier8();  // every read of this stage is done, and the next is whole
  }
#pragma unroll
  for (int j = 0; j < FM; ++j)
#pragma unroll
    for (int r = 0; r < 4; ++r) acc[FN - 1][j][r] = __builtin_fmaf(pp[j][r], sp[j], acc[FN - 1][j][r]);
}

// ---------------------------------------------------------------------------
// Few tokens: weights from memory into registers
// ---------------------------------------------------------------------------
// A wave's sums of 16 NT weight rows and 16 MT tokens over blocks [kb0, kb1).
// Bound by the weight's bytes, each read once: a lane loads its own 32 codes of
// a row, D blocks ahead, and nothing passes through LDS.
// Src gives: w(i), x(j): the lane's row (l % 16) of weight rows 16 i .. and of
// tokens 16 j ..; sx(j): its token's scales; sw(i): the weight rows' scales;
// block(j, kb): the lane's codes of its token, where XOWN.
// XOWN: tokens come from block(), and their scales from scale(j, kb).
// `between` runs once the first loads are on their way.
template <int NT, int MT>
struct RowStage {
  Codes32 w[NT], x[MT];
  float sw[NT], sx[MT];
};

template <int NT, int MT, int D, bool XOWN, bool ONCE, class Src, class Between>
__device__ __forceinline__ void row_sums(const Src& src, int kb0, int kb1, int k, f32x4 (&acc)[NT][MT], Between between) {
  const int g = (threadIdx.x & 63) >> 4;
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int j = 0; j < MT; ++j) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  GlobalCodes wp[NT], xp[MT];
  const float *swp[NT], *sxp[MT];
#pragma unroll
  for (int i = 0; i < NT; ++i) wp[i] = (GlobalCodes)src.w(i), swp[i] = src.sw(i);
#pragma unroll
  for (int j = 0; j < MT; ++j)
    if constexpr (!XOWN) xp[j] = (GlobalCodes)src.x(j), sxp[j] = src.sx(j);
  const int whole = k / kBlk < kb1 ? k / kBlk : kb1;  // blocks before a cut one
  RowStage<NT, MT> st[D];
  auto load = [&](RowStage<NT, MT>& a, int kb) {
    kb = kb < whole ? kb : whole - 1;
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      const GlobalCodes q = wp[i] + (kb * kBlk + 16 * g);
      a.w[i] = ONCE ? Codes32{load_codes_nt(q), load_codes_nt(q + 64)} : Codes32{load_codes(q), load_codes(q + 64)};
      a.sw[i] = gld<float>(swp[i] + kb);
    }
    if constexpr (!XOWN) {
#pragma unroll
      for (int j = 0; j < MT; ++j) {
        const GlobalCodes q = xp[j] + (kb * kBlk + 16 * g);
        a.x[j] = {load_codes(q), load_codes(q + 64)};
        a.sx[j] = gld<float>(sxp[j] + kb);
      }
    }
  };
  auto multiply = [&](RowStage<NT, MT>& a, int kb) {
    if constexpr (XOWN) {
#pragma unroll
      for (int j = 0; j < MT; ++j) a.x[j] = src.block(j, kb), a.sx[j] = src.scale(j, kb);
    }
    Wide32 x[MT];
#pragma unroll
    for (int j = 0; j < MT; ++j) x[j] = widen(a.x[j]);
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      const Wide32 w = widen(a.w[i]);
#pragma unroll
      for (int j = 0; j < MT; ++j) {
        const f32x4 p = mma8(w, x[j]);
        const float s = a.sx[j] * a.sw[i];
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[i][j][r] = __builtin_fmaf(p[r], s, acc[i][j][r]);
      }
    }
  };
  if (kb0 < whole) {
#pragma unroll
    for (int d = 0; d < D; ++d) load(st[d], kb0 + d);
  }
  between();
  int kb = kb0;
  for (; kb + D <= whole; kb += D) {
#pragma unroll
    for (int d = 0; d < D; ++d) {
      multiply(st[d], kb + d);
      load(st[d], kb + d + D);
    }
  }
#pragma unroll
  for (int d = 0; d < D; ++d)
    if (kb + d < whole) multiply(st[d], kb + d);
  if (kb0 < kb1 && whole < kb1) {  // the last block of K, cut
    RowStage<NT, MT>& a = st[0];
    const int at = whole * kBlk + 16 * g;
#pragma unroll
    for (int i = 0; i < NT; ++i) a.w[i] = {load_codes_cut(wp[i], at, k), load_codes_cut(wp[i], at + 64, k)}, a.sw[i] = gld<float>(swp[i] + whole);
    if constexpr (!XOWN) {
#pragma unroll
      for (int j = 0; j < MT; ++j) a.x[j] = {load_codes_cut(xp[j], at, k), load_codes_cut(xp[j], at + 64, k)}, a.sx[j] = gld<float>(sxp[j] + whole);
    }
    multiply(a, whole);
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
