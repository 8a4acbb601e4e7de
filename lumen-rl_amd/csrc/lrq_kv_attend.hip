// Attention of each sequence's last tokens over all of its own, on an FP8 KV cache.
//
//   o = sum_j p_j v_j / sum_j p_j,   p_j = 2^(c (q . k_j) - m),   c = scale log2(e),
// with m the running maximum of a row, in one pass over the keys.  A row is a new token
// and one of its query heads; the rows that share a KV head are taken together, 16 or 32 a
// wave, so that each code is read once for all of them.  Bound by the codes' bytes:
// 256 sequences of up to 8100 keys on 8 heads of 128 (2.1 GB) take 392 us, 5.4 TB/s, where a
// read of as much and nothing else reaches 6.2; one of 1500 keys 13 us, two launches' latency.
//
// Both products run on bf16 or fp16 matrix instructions (float32 sums): e4m3 codes are
// exact in both types, and the keys' scale is applied to the sums.  The first product
// takes the queries' own type.  The second takes p in fp16 and V's codes without their
// scale, which is folded into p: with e_j = log2 of the scale of v_j's page,
//   o 2^M = sum_j 2^(s_j + e_j - M) code_j,   l 2^M = sum_j 2^(s_j + e_j - M) 2^-e_j,
// M the running maximum of s + e.  So p has 11 bits and a range of 2^-34 below the
// largest term (it is taken 2^10 times as large, and fp16's subnormals count), where bf16
// would have 8 bits: its rounding is then far below that of a 16-bit result.  l takes p before
// that rounding: a key of a page whose V is far smaller than others' has a p far below fp16's
// range, and yet its part of l.  That part is in float32's range as long as V's scales are no
// further than 2^96 apart: they are taken within 2^-48 .. 2^48.
//
// Layout: both products are taken transposed, S^T = K Q^T and O^T = V^T P^T, on 16x16x32
// instructions.  Lane l holds of every result the column l % 16, a row of queries, and so
// one maximum and one sum.  Keys are taken 64 at a time; key 16 (l / 16) + 4 t + i is
// result i of tile t in lane l, so that a lane's 16 probabilities are those of the 16
// keys whose V codes it loads with one 16-byte load, in its order, and P never leaves the
// registers.
//
// This kernel is for few rows a sequence, where the codes' bytes are all there is.  The four
// waves of a work-group look for their pieces of work together, by sums over the work-group; then
// each works for itself: its loop over the keys has no barrier and no LDS, the next 64 keys
// are on their way into registers while it works on the present ones.  LDS (16 KiB for each 64
// channels of 16 rows, up to 64 KiB a work-group) holds the sums where NaN codes that only
// some rows see are worked on; registers, not it, bound the waves of a compute unit.
#include "lrq_kv.hpp"
#include "lrq_kv_attend.hpp"

namespace lrq {

namespace {

constexpr int kWaves = 4;  // of a work-group, which share the search for where they begin
static_assert(64 * kWaves == kOwnSearch, "a thread looks at one sequence");

template <int DT>
__device__ __forceinline__ f32x4 mma(v4u a, v4u b, f32x4 d) {
  if constexpr (DT == kBF16)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), d, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), d, 0, 0, 0);
}
// The largest of the lanes l, l ^ 16, l ^ 32 and l ^ 48.
__device__ __forceinline__ float column_max(float v) {
  auto a = __builtin_amdgcn_permlane32_swap(f2u(v), f2u(v), false, false);
  v = fmaxf(u2f(a[0]), u2f(a[1]));
  auto b = __builtin_amdgcn_permlane16_swap(f2u(v), f2u(v), false, false);
  return fmaxf(u2f(b[0]), u2f(b[1]));
}
__device__ __forceinline__ float column_sum(float v) {
  auto a = __builtin_amdgcn_permlane32_swap(f2u(v), f2u(v), false, false);
  v = u2f(a[0]) + u2f(a[1]);
  auto b = __builtin_amdgcn_permlane16_swap(f2u(v), f2u(v), false, false);
  return u2f(b[0]) + u2f(b[1]);
}

// The units of keys that a sequence's rows see: [first, first + count), one at least.
struct Span {
  int first, count;
};
__device__ __forceinline__ Span span_of(const KvSeq& q, int window) {
  int64_t lo = 0;
  if (window > 0) lo = (int64_t)q.len - q.n + 1 - window;
  Span s;
  s.first = lo > 0 ? (int)(lo / kUnit) : 0;
  const int end = (int)(((int64_t)q.len + kUnit - 1) / kUnit);
  s.count = end - s.first;
  if (s.count < 1) s.count = 1;
  return s;
}
// Tiles of a sequence's rows; none where it has so many that k_kv_prefill takes them.
template <int ROWS>
__device__ __forceinline__ int row_tiles(const KvSeq& q, int group, int few) {
  const int64_t rows = (int64_t)q.n * group;
  return rows > few ? 0 : (int)((rows + ROWS - 1) / ROWS);
}

// ---------------------------------------------------------------------------
// Work: an item is a sequence, a KV head and a tile of rows; its units are cut into pieces
// of about the same number, so that all items together make a few pieces for each wave
// that the chip holds.  A wave takes one piece.  Pieces are numbered sequence by sequence,
// then piece by piece, heads and tiles last: waves that run side by side read the heads
// of the same pages.  The pieces of an item that was cut leave unnormalized sums, which
// k_kv_join puts together.
// ---------------------------------------------------------------------------
struct Work {
  int lines, count;  // items, units of each
};
template <int ROWS>
__device__ __forceinline__ Work work_of(const KvAttendArgs& a, const KvSeq& q) {
  Work w;
  w.lines = row_tiles<ROWS>(q, a.group, a.few) * a.cache.heads;
  w.count = span_of(q, a.window).count;
  return w;
}
// For k_kv_join, from the wave that has an item's first piece.
struct PartHead {
  int64_t first;    // the item's first row's token
  int slot, rows;   // its place, rows of the tile
  int tile, h;
  int parts, step;  // its pieces, and from each one's place to the next one's
};
static_assert(sizeof(PartHead) == 32, "the join's heads are 32 bytes apart");

// Waves of a SIMD, by the registers they need.
template <int NC, int MT>
constexpr int kPerSimd = MT * NC > 2 ? 1 : 2;
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ int64_t uniform(int64_t v) {
  return (int64_t)(((uint64_t)(uint32_t)uniform((int)(v >> 32)) << 32) | (uint32_t)uniform((int)v));
}
// Where piece i of n begins in a line of `count`: pieces differ by one at most.
__device__ __forceinline__ int piece_at(int count, int i, int n) {
  const int each = (int)((uint32_t)count / (uint32_t)n), rest = count - each * n;
  return i * each + (i < rest ? i : rest);
}
// Pieces that all work is cut into: three for each SIMD of the chip, of which two run at a
// time (256 sequences of up to 8100 keys: 2, 3, 4, 6 and 8 a SIMD take 428, 403, 408, 411 and
// 423 us; one wave a SIMD 411, three 461).
constexpr int kParts = 256 * 4 * 3;
// Units of a piece at least, if the item has as many; a piece of two tiles leaves twice the sums
// (8000 keys, one row of 16 on each head: 1, 2 and 4 units 15.4, 15.9 and 17.4 us; 128 tokens of
// 4 rows on 2000 keys: 2 units 48.8, 4 units 39.3 us, 48 of up to 5 tokens 23.0 and 21.9).
template <int MT>
constexpr uint32_t kLeast = 2 * MT;
// Units of a piece, where a line has less than 2^25.
template <int MT>
__device__ __forceinline__ uint32_t units_of_piece(int64_t total) {
  const int64_t share = (total + kParts - 1) / kParts;
  return share < kLeast<MT> ? kLeast<MT> : share < 1 << 25 ? (uint32_t)share : 1u << 25;
}
// A sequence's pieces; and those of items that are cut, with (times 2^16) these items: at most
// 2 kParts of each in a call.  Offsets that go back would make rows of several sequences', and
// more pieces than there are waves: sequences whose pieces have not all one are left out.
struct Pieces {
  uint32_t pieces, cut;
};
__device__ __forceinline__ Pieces pieces_of(const Work& w, uint32_t per) {
  const uint32_t cuts = ((uint32_t)w.count + per - 1) / per, pieces = cuts * (uint32_t)w.lines;
  return Pieces{pieces, cuts > 1 ? pieces + ((uint32_t)w.lines << 16) : 0};
}

// An address that is the same in all lanes, kept in scalar registers: loads add a lane's
// 32-bit offset and a constant to it by themselves, up to 4095.
__device__ __forceinline__ const uint8_t* in_scalars(const uint8_t* p) {
  asm("" : "+s"(p));
  return p;
}

// One tile of rows a sequence: each code is read once, past the caches (256 sequences of up to
// 8100 keys 410 -> 393 us).  More tiles find them in the caches, which heads of more than 128
// channels have with 17 rows already (32 sequences of 32 rows and 4000 keys of 192 channels:
// past the caches 152, else 108 us).
template <int NC, int MT>
__device__ __forceinline__ v4u codes_at(const uint8_t* p) {
  return MT == 1 && NC <= 2 ? gld_nt<v4u>(p) : gld<v4u>(p);
}

// With more than kOwnSearch sequences, one work-group before: pieces up to each of them.
template <int MT>
__global__ __launch_bounds__(1024) void k_kv_count(KvAttendArgs a, uint32_t limit) {
  __shared__ int64_t scan[16];
  __shared__ uint32_t scan32[16], carry[2], most;
  const int tid = threadIdx.x, seqs = a.seqs.seqs;
  if (tid == 0) most = 0;
  int64_t units = 0;
  for (int b = tid; b < seqs; b += 1024) {
    const Work w = work_of<16 * MT>(a, kv_seq(a.seqs, b));
    units += (int64_t)w.lines * w.count;
  }
  const uint32_t per = units_of_piece<MT>(block_sum<16>(units, scan));
  uint32_t before = 0, before_cut = 0;
  for (int b0 = 0; b0 < seqs; b0 += 1024) {
    const int b = b0 + tid;
    Work w{};
    if (b < seqs) w = work_of<16 * MT>(a, kv_seq(a.seqs, b));
    const Pieces p = pieces_of(w, per);
    const uint32_t upto = before + block_scan<1024, uint32_t>(p.pieces, scan32);
    const bool in = upto <= limit;
    const uint32_t upto_cut = before_cut + block_scan<1024, uint32_t>(in ? p.cut : 0, scan32);
    if (b < seqs) gst<int32_t>(a.upto + b, (int32_t)(in ? upto : limit + 1)), gst<int32_t>(a.upto_cut + b, (int32_t)upto_cut);
    if (in) atomicMax(&most, upto);
    if (tid == 1023) carry[0] = in ? upto : limit + 1, carry[1] = upto_cut;
    __syncthreads();
    before = carry[0], before_cut = carry[1];
    __syncthreads();
  }
  if (tid == 0) gst<int32_t>(a.counts, (int32_t)per), gst<int32_t>(a.counts + 1, (int32_t)most), gst<int32_t>(a.cut_count, (int32_t)(before_cut >> 16));
}

// FAST: heads of 64 NC channels and pages of 64 keys, which are the constants of the
// addresses then, and a page is one for the whole wave (16, 32 and 64 rows on 4000 keys, 32
// times, 66, 82 and 104 us; without it 78, 102 and 152, and spills of 26 to 117 scalar registers and
// up to 4 vector ones).
template <int DT, int NC, int MT, bool FAST>
__global__ __launch_bounds__(64 * kWaves, (kPerSimd<NC, MT>)) void k_kv_attend(KvAttendArgs a) {
  constexpr int NT = 4 * NC;       // tiles of 16 channels
  constexpr int ROWS = 16 * MT;
  __shared__ int64_t scan[kWaves];
  __shared__ uint32_t scan32[kWaves];
  __shared__ int found[kWaves][4];
  __shared__ f32x4 aside[kWaves * MT * NT * 64];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r = lane & 15, g = lane >> 4;
  const int shift = FAST ? 6 : a.seqs.shift, S = 1 << shift, dim = FAST ? 64 * NC : a.cache.dim, group = a.group;

  // rows of the result that are no sequence's
  if (a.zero_rest) {
    int64_t lead = 0, lo = a.seqs.seqs;  // rows before the first sequence, and where those behind the last begin
    if (a.seqs.offsets != nullptr) lead = gld<int32_t>(a.seqs.offsets), lo = gld<int32_t>(a.seqs.offsets + a.seqs.seqs);
    lead = lead < 0 ? 0 : lead < a.seqs.tokens ? lead : a.seqs.tokens, lo = lo < lead ? lead : lo;
    const int64_t words = (int64_t)a.heads * dim / 2;
    for (int64_t i = blockIdx.x;; i += gridDim.x) {
      const int64_t t = i < lead ? i : lo + (i - lead);
      if (t >= a.seqs.tokens) break;
      for (int64_t w = tid; w < words; w += 64 * kWaves) gst<uint32_t>(static_cast<uint32_t*>(a.out) + t * words + w, 0u);
      if (a.lse != nullptr)
        for (int w = tid; w < a.heads; w += 64 * kWaves) gst<float>(a.lse + t * a.heads + w, -INFINITY);
    }
  }

  // the sequences that the four waves' pieces are of
  int b, place, slot;
  uint32_t per;
  if (a.counts != nullptr) {
    const uint32_t at = blockIdx.x * kWaves + wave;
    per = (uint32_t)sld(a.counts);
    if (at >= (uint32_t)sld(a.counts + 1)) return;
    b = kv_find(a.upto, a.seqs.seqs, at);
    const uint32_t first = b > 0 ? (uint32_t)sld(a.upto_cut + b - 1) : 0;
    place = (int)at - (b > 0 ? sld(a.upto + b - 1) : 0);
    slot = (int)(first & 0xFFFF) + place;
    if (lane == 0) found[wave][3] = (int)(first >> 16);
  } else {
    Work mine{};
    if (tid < a.seqs.seqs) mine = work_of<ROWS>(a, kv_seq(a.seqs, tid));
    const int64_t total = uniform(block_sum<kWaves>((int64_t)mine.lines * mine.count, scan));
    if (total == 0) {  // all sequences are k_kv_prefill's
      if (blockIdx.x == 0 && tid == 0) gst<int32_t>(a.cut_count, 0);
      return;
    }
    per = units_of_piece<MT>(total);
    if (tid < kWaves) found[tid][0] = -1;
    __syncthreads();
    const Pieces p = pieces_of(mine, per);
    const uint32_t upto = block_scan<64 * kWaves, uint32_t>(p.pieces, scan32);
    const bool in = upto <= gridDim.x * kWaves;
    const uint32_t cut = in ? p.cut : 0, upto_cut = block_scan<64 * kWaves, uint32_t>(cut, scan32);
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const uint32_t at = blockIdx.x * kWaves + w - (upto - p.pieces);  // wraps below 0
      if (at < p.pieces && in) {
        const uint32_t first = upto_cut - cut;
        found[w][0] = tid, found[w][1] = (int)at, found[w][2] = (int)((first & 0xFFFF) + at), found[w][3] = (int)(first >> 16);
      }
    }
    if (blockIdx.x == 0 && tid == 64 * kWaves - 1) gst<int32_t>(a.cut_count, (int32_t)(upto_cut >> 16));
    __syncthreads();
    b = uniform(found[wave][0]), place = uniform(found[wave][1]), slot = uniform(found[wave][2]);
    if (b < 0) return;
  }
  const KvSeq q = kv_seq_uniform(a.seqs, b);
  const Work work = work_of<ROWS>(a, q);
  const int cuts = (int)(((uint32_t)work.count + per - 1) / per);
  const int piece = place / work.lines, line = place - piece * work.lines;
  const int tiles = work.lines / a.cache.heads;
  const int h = line / tiles, tile = line - h * tiles;
  const int u0 = span_of(q, a.window).first + piece_at(work.count, piece, cuts);
  const int u1 = span_of(q, a.window).first + piece_at(work.count, piece + 1, cuts);

  // What a lane loads of a unit: K, a row of each of four tiles of 16 keys, key 16 (r / 4) +
  // 4 t + r % 4; V, keys 16 g .. of every 16th channel.  V's codes are asked for before K's
  // are worked on, the next unit's K before V's.
  v4u kc[4][NC], vc[NT];
  int kp, vp;  // the page of this lane's key of K, and of its keys of V (16 keys are of one page)
  auto pages_at = [&](int u, int& kpage, int& vpage) {
    if constexpr (FAST) {
      kpage = vpage = kv_page_uniform(a.seqs, a.cache.pages, b, u);
    } else {
      int p[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) p[i] = kv_page_uniform(a.seqs, a.cache.pages, b, (u * kUnit + 16 * i) >> shift);
      kpage = (r & 8) ? ((r & 4) ? p[3] : p[2]) : ((r & 4) ? p[1] : p[0]);
      vpage = (g & 2) ? ((g & 1) ? p[3] : p[2]) : ((g & 1) ? p[1] : p[0]);
    }
  };
  const uint32_t k_lane = (FAST ? 16 * (r >> 2) + (r & 3) : r & 3) * dim + 16 * g;
  const uint32_t v_lane = FAST ? r * S + 16 * g : r * S;
  auto load_k = [&](int u, int page) {
    const uint8_t* kb = a.cache.k + (int64_t)(page < 0 ? 0 : page) * a.cache.k_page + (int64_t)h * S * dim;
    if constexpr (FAST) {
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        if (t % 2 == 0) kb = in_scalars(a.cache.k + (int64_t)(page < 0 ? 0 : page) * a.cache.k_page + (int64_t)h * S * dim + 4 * t * dim);
#pragma unroll
        for (int k = 0; k < NC; ++k) kc[t][k] = codes_at<NC, MT>(kb + k_lane + (4 * (t % 2) * dim + 64 * k));
      }
    } else {
      kb += ((u * kUnit + 16 * (r >> 2)) & (S - 1)) * dim;
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int k = 0; k < NC; ++k) {
          kc[t][k] = v4u{0, 0, 0, 0};
          if (64 * k + 16 * g < dim) kc[t][k] = codes_at<NC, MT>(kb + k_lane + (4 * t * dim + 64 * k));
        }
    }
  };
  auto load_v = [&](int u, int page) {
    const uint8_t* vb = a.cache.v + (int64_t)(page < 0 ? 0 : page) * a.cache.v_page + (int64_t)h * S * dim;
    if constexpr (FAST) {
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        if (n % 4 == 0) vb = in_scalars(a.cache.v + (int64_t)(page < 0 ? 0 : page) * a.cache.v_page + (int64_t)h * S * dim + 16 * n * S);
        vc[n] = codes_at<NC, MT>(vb + v_lane + 16 * (n % 4) * S);
      }
    } else {
      vb += (u * kUnit + 16 * g) & (S - 1);
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        vc[n] = v4u{0, 0, 0, 0};
        if (16 * n < dim) vc[n] = codes_at<NC, MT>(vb + v_lane + 16 * n * S);
      }
    }
  };

  // this lane's rows, and the keys below hi that they see
  int hi[MT];
  v4u qf[MT][NC][2];
  float m[MT], l[MT];
  f32x4 acc[MT][NT];
  const int64_t row0 = (int64_t)tile * ROWS, all = (int64_t)q.n * group;
  const int rows = (int)(all - row0 < ROWS ? all - row0 : ROWS);
  const int base = q.len - q.n + 1;  // below 1: the first tokens see nothing
#pragma unroll
  for (int t = 0; t < MT; ++t) {
    const int64_t row = row0 + (16 * t + r < rows ? 16 * t + r : 0);
    const int tok = (int)(row / group), qh = h * group + (int)(row - (int64_t)tok * group);
    hi[t] = base + tok < 0 ? 0 : base + tok;
    const uint16_t* const src = static_cast<const uint16_t*>(a.q) + (q.first + tok) * a.q_token + qh * a.q_head;
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int d = 64 * c + 16 * g + 8 * k;
        qf[t][c][k] = v4u{0, 0, 0, 0};
        if (d < dim && 16 * t + r < rows) qf[t][c][k] = load_live(src + d);
      }
    m[t] = kLow, l[t] = 0.0f;
#pragma unroll
    for (int n = 0; n < NT; ++n) acc[t][n] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  }
  // what the first and the last row see (rows are in the order of their tokens)
  const int hi_a = base + (int)(row0 / group), hi_b = base + (int)((row0 + rows - 1) / group);
  const int lo_a = a.window > 0 && hi_a > a.window ? hi_a - a.window : 0;
  const int lo_b = a.window > 0 && hi_b > a.window ? hi_b - a.window : 0;
  float factor, ev, back;  // of this lane's 16 keys: the scores' factor, V's exponent, its inverse
  auto scales_of = [&](int page) {
    const int64_t at = page < 0 ? 0 : page;
    const float* const ksp = a.cache.ks + at * a.cache.ks_page + h;
    const float* const vsp = a.cache.vs + at * a.cache.vs_page + h;
    factor = (FAST ? sld(ksp) : gld<float>(ksp)) * a.scale;
    ev = __builtin_amdgcn_logf(__builtin_amdgcn_fmed3f(FAST ? sld(vsp) : gld<float>(vsp), 0x1p-48f, 0x1p48f));
    back = __builtin_amdgcn_exp2f(-ev);
  };
  auto scores = [&](f32x4 (&s)[MT][4]) {
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int j = 0; j < 4; ++j) s[t][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int k = 0; k < NC; ++k) {
        if (64 * k >= dim) continue;
        const v4u x = widen8<DT>(kc[j][k].x, kc[j][k].y), y = widen8<DT>(kc[j][k].z, kc[j][k].w);
#pragma unroll
        for (int t = 0; t < MT; ++t) {
          s[t][j] = mma<DT>(x, qf[t][k][0], s[t][j]);
          s[t][j] = mma<DT>(y, qf[t][k][1], s[t][j]);
        }
      }
  };
  v4u p[MT][2];
  auto soften = [&](float (&x)[16], int t) {  // from scores and exponents to p; the sums so far fade as the maximum grows
    float top = m[t];
#pragma unroll
    for (int i = 0; i < 16; ++i) top = fmaxf(top, x[i]);
    top = column_max(top);
    const float fade = __builtin_amdgcn_exp2f(m[t] - top);
    m[t] = top;
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      x[i] = __builtin_amdgcn_exp2f(x[i] - top + kLift);
      sum += x[i];
    }
    l[t] = l[t] * fade + sum * back;
#pragma unroll
    for (int k = 0; k < 2; ++k)
      p[t][k] = v4u{f16_pair(x[8 * k], x[8 * k + 1]), f16_pair(x[8 * k + 2], x[8 * k + 3]), f16_pair(x[8 * k + 4], x[8 * k + 5]),
                    f16_pair(x[8 * k + 6], x[8 * k + 7])};
#pragma unroll
    for (int n = 0; n < NT; ++n) acc[t][n] *= fade;
  };
  auto values = [&]() {
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      if (16 * n >= dim) continue;
      const v4u x = widen8<kF16>(vc[n].x, vc[n].y), y = widen8<kF16>(vc[n].z, vc[n].w);
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        acc[t][n] = mma<kF16>(x, p[t][0], acc[t][n]);
        acc[t][n] = mma<kF16>(y, p[t][1], acc[t][n]);
      }
    }
  };
  // units that some row sees a part of, or whose pages are not all there
  auto is_cut = [&](int u) {
    const bool gone = FAST ? vp < 0 : __ballot(vp < 0) != 0;
    return u * kUnit + kUnit > hi_a || u * kUnit < lo_b || gone;
  };

  int u = u0;
  pages_at(u, kp, vp);
  while (u < u1) {
    if (is_cut(u)) {
      const int v_key = u * kUnit + 16 * g, v_now = vp;
      const bool ok = vp >= 0;
      load_k(u, kp);
      load_v(u, vp);
      scales_of(vp);
      f32x4 s[MT][4];
      scores(s);
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        float x[16];
        const int lo = a.window > 0 && hi[t] > a.window ? hi[t] - a.window : 0;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int key = v_key + i;
          x[i] = key < hi[t] && key >= lo && ok ? __builtin_fmaf(s[t][i >> 2][i & 3], factor, ev) : -INFINITY;
        }
        soften(x, t);
      }
      // keys before the first or behind the last that some row sees have no value
      const int keep_hi = ok ? hi_b - v_key : 0, keep_lo = lo_a - v_key;
      uint32_t keep[4], bad = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) keep[i] = low_bytes(keep_hi - 4 * i) & ~low_bytes(keep_lo - 4 * i);
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        vc[n] = v4u{vc[n].x & keep[0], vc[n].y & keep[1], vc[n].z & keep[2], vc[n].w & keep[3]};
        bad |= nan_bytes(vc[n].x) | nan_bytes(vc[n].y) | nan_bytes(vc[n].z) | nan_bytes(vc[n].w);
      }
      if (__ballot(bad != 0) == 0) {
        values();
      } else {
        // NaN codes that some rows see and others do not: 0 x NaN must not reach the
        // others.  So each token's rows get sums of their own, over what that token sees.
        // (By way of LDS, so that this rare path needs few registers of the others'.)
        f32x4* const mine = aside + wave * (MT * NT * 64) + lane;
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
          for (int n = 0; n < NT; ++n) mine[(t * NT + n) * 64] = acc[t][n];
        const uint8_t* const vb = a.cache.v + (int64_t)(v_now < 0 ? 0 : v_now) * a.cache.v_page + (int64_t)h * S * dim + r * S + (v_key & (S - 1));
#pragma unroll 1
        for (int n = 0; 16 * n < dim; ++n) {
          const v4u w = gld<v4u>(vb + (int64_t)16 * n * S);
#pragma unroll 1
          for (int see = hi_a < 1 ? 1 : hi_a; see <= hi_b; ++see) {
            const int see_hi = ok ? see - v_key : 0, see_lo = (a.window > 0 && see > a.window ? see - a.window : 0) - v_key;
            uint32_t some[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) some[i] = low_bytes(see_hi - 4 * i) & ~low_bytes(see_lo - 4 * i);
            const v4u x = widen8<kF16>(w.x & some[0], w.y & some[1]), y = widen8<kF16>(w.z & some[2], w.w & some[3]);
#pragma unroll
            for (int t = 0; t < MT; ++t) {
              const f32x4 was = mine[(t * NT + n) * 64];
              const f32x4 sums = mma<kF16>(y, p[t][1], mma<kF16>(x, p[t][0], was));
              if (hi[t] == see) mine[(t * NT + n) * 64] = sums;
            }
          }
        }
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
          for (int n = 0; n < NT; ++n) acc[t][n] = mine[(t * NT + n) * 64];
      }
      if (++u < u1) pages_at(u, kp, vp);
      continue;
    }
    // a run of units that all rows see the whole of
    load_k(u, kp);
    bool more = true;
    while (more) {
      load_v(u, vp);
      scales_of(vp);
      more = ++u < u1;
      if (more) pages_at(u, kp, vp), more = !is_cut(u);
      __builtin_amdgcn_sched_barrier(0);
      f32x4 s[MT][4];
      scores(s);
      __builtin_amdgcn_sched_barrier(0);
      if (more) load_k(u, kp);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        float x[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i] = __builtin_fmaf(s[t][i >> 2][i & 3], factor, ev);
        soften(x, t);
      }
      values();
    }
  }

  const bool whole = cuts == 1;
  float* const out = a.sums + slot * ((2 + (int64_t)dim) * ROWS);
  if (lane == 0 && piece == 0 && !whole)
    reinterpret_cast<PartHead*>(a.heads_at)[found[wave][3] + line] = PartHead{q.first, slot, rows, tile, h, cuts, work.lines};
#pragma unroll
  for (int t = 0; t < MT; ++t) {
    const float sum = column_sum(l[t]);
    if (16 * t + r >= rows) continue;
    const int64_t row = row0 + 16 * t + r, tok = row / group;
    const int64_t at_row = (q.first + tok) * a.heads + h * group + (row - tok * group);
    if (whole) {
      const float over = sum != 0.0f ? 1.0f / sum : 0.0f;  // a row that sees nothing is 0
#pragma unroll
      for (int n = 0; n < NT; ++n)
        if (16 * n < dim) store4<DT>(a.out, at_row * dim + 16 * n + 4 * g, acc[t][n] * over);
      if (a.lse != nullptr && g == 0)
        gst<float>(a.lse + at_row, sum != 0.0f ? (m[t] - kLift + __builtin_amdgcn_logf(sum)) * kLn2 : -INFINITY);
    } else {
#pragma unroll
      for (int n = 0; n < NT; ++n)
        if (16 * n < dim) gst<f32x4>(out + 2 * ROWS + ((4 * n + g) * ROWS + 16 * t + r) * 4, acc[t][n]);
      if (g == 0) gst<float>(out + 16 * t + r, m[t]), gst<float>(out + ROWS + 16 * t + r, sum);
    }
  }
}

// Items that were cut: their pieces' sums, brought to one maximum.  A thread has four
// channels of a row, and where there are fewer of these than threads, a share of the pieces.
template <int DT, int MT>
__global__ __launch_bounds__(256) void k_kv_join(KvAttendArgs a) {
  constexpr int ROWS = 16 * MT;
  __shared__ f32x4 vals[256];
  __shared__ float tops[256], sums[256];
  const int tid = threadIdx.x, dim = a.cache.dim;
  const int64_t size = (2 + (int64_t)dim) * ROWS;
  const int quads = dim / 4 / gridDim.y;  // of channels, from c0 on
  const int c0 = blockIdx.y * quads;
  const int count = gld<int32_t>(a.cut_count);
  for (int i = blockIdx.x; i < count; i += gridDim.x) {
    const PartHead head = reinterpret_cast<const PartHead*>(a.heads_at)[i];
    const int all = head.rows * quads, shares = all < 256 ? 256 / all : 1;
    const float* const first = a.sums + head.slot * size;
    const int64_t step = head.step * size;
    for (int o0 = 0; o0 < all; o0 += 256) {
      const int o = all < 256 ? tid % all : o0 + tid, share = all < 256 ? tid / all : 0;
      const int r = o / quads, c = c0 + o - r * quads;
      const bool mine = o < all && share < shares;
      float top = kLow, sum = 0.0f;
      f32x4 v = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
      if (mine) {
#pragma unroll 4
        for (int p = share; p < head.parts; p += shares) {
          const float* const at = first + p * step;
          const float m = gld<float>(at + r), l = gld<float>(at + ROWS + r);
          const f32x4 x = gld<f32x4>(at + 2 * ROWS + (c * ROWS + r) * 4);
          const float more = fmaxf(top, m);
          const float f = __builtin_amdgcn_exp2f(top - more), e = __builtin_amdgcn_exp2f(m - more);
          sum = sum * f + l * e, v = v * f + x * e;
          top = more;
        }
      }
      if (shares > 1) {
        __syncthreads();
        vals[tid] = v, tops[tid] = top, sums[tid] = sum;
        __syncthreads();
        if (share == 0) {
          float more = top;
          for (int k = 1; k < shares; ++k) more = fmaxf(more, tops[tid + k * all]);
          const float f = __builtin_amdgcn_exp2f(top - more);
          sum *= f, v *= f;
          for (int k = 1; k < shares; ++k) {
            const float e = __builtin_amdgcn_exp2f(tops[tid + k * all] - more);
            sum += sums[tid + k * all] * e, v += vals[tid + k * all] * e;
          }
          top = more;
        }
      }
      if (mine && share == 0) {
        const int64_t row = (int64_t)head.tile * ROWS + r, tok = row / a.group;
        const int64_t at = (head.first + tok) * a.heads + head.h * a.group + (row - tok * a.group);
        store4<DT>(a.out, at * dim + 4 * c, v * (sum != 0.0f ? 1.0f / sum : 0.0f));
        if (a.lse != nullptr && c == 0) gst<float>(a.lse + at, sum != 0.0f ? (top - kLift + __builtin_amdgcn_logf(sum)) * kLn2 : -INFINITY);
      }
    }
  }
}

// Sequences of more rows than kMostRows are k_kv_prefill's (32 of 4000 keys: with 64 rows each
// 103 us here and 110 there, with 96 rows 126 and 114; 64 channels, pages of 32: 75 and 87), of more
// than half as many where this kernel holds its registers worst: more than 64 channels, without
// FAST (128 in pages of 16, 48 rows 156 and 124 us; 80 channels 122 and 101) or in tiles of 16 rows
// and not of 32 (192 channels, 64 rows: 216 and 188).  But not in a call whose
// rows are kAllRows together at most: three launches less (one of 2000 keys: 1024 rows 50.6
// and 54.4 us, 4096 rows 124 and 102).
constexpr int kMostRows = 64, kAllRows = 1024;
int most_rows(int64_t dim, int shift) { return dim <= 64 || (dim == 128 && shift == 6) ? kMostRows : kMostRows / 2; }
// Rows of a call; one_each: one token a sequence.
int64_t all_rows(int64_t tokens, int64_t seqs, bool one_each, int64_t group) { return (one_each && seqs < tokens ? seqs : tokens) * group; }
bool all_few(int64_t rows, bool one_each, int64_t group, int most) { return one_each ? group <= most : rows <= kAllRows; }

// Items of a call at most, and its pieces: an item of n units is cut into less than n / per + 1.
int64_t most_items(int64_t rows, int64_t heads, int64_t seqs, bool all) {
  int64_t tiles = rows / 16 + seqs;
  if (!all && tiles > seqs * (kMostRows / 16)) tiles = seqs * (kMostRows / 16);
  return tiles * heads;
}
int64_t most_pieces(int64_t items, int64_t width, int shift) {
  const int64_t units = items * ((width << shift) / kUnit + 1);
  return units < items + kParts ? units : items + kParts;
}
// Those that leave sums are of items of more than per units, twice their share at most.
constexpr int64_t kPlaces = 2 * kParts;

template <int DT, int NC, int MT>
void launch(KvAttendArgs a, hipStream_t stream) {
  const int64_t seqs = a.seqs.seqs < a.seqs.tokens ? a.seqs.seqs : a.seqs.tokens;  // others have no new token
  const bool one_each = a.seqs.offsets == nullptr;
  const int64_t rows = all_rows(a.seqs.tokens, a.seqs.seqs, one_each, a.group);
  const int64_t items = most_items(rows, a.cache.heads, seqs, a.few == INT32_MAX);
  const int64_t pieces = most_pieces(items, a.seqs.width, a.seqs.shift);
  const int64_t groups = pieces > 0 ? (pieces + kWaves - 1) / kWaves : 1;
  // few items: a work-group for 32 channels of each (8000, 120000 and 500000 keys of one token
  // 16, 61 and 182 us; 25, 83 and 204 with one for all channels; 8 channels 17, 58 and 180)
  const int64_t joins = items < 2048 ? items : 2048;
  const int split = items <= 256 && a.cache.dim % 32 == 0 ? a.cache.dim / 32 : 1;
  if (a.counts != nullptr) hipLaunchKernelGGL((k_kv_count<MT>), dim3(1), dim3(1024), 0, stream, a, (uint32_t)groups * kWaves);
  if (a.cache.dim == 64 * NC && a.seqs.shift == 6)
    hipLaunchKernelGGL((k_kv_attend<DT, NC, MT, true>), dim3((unsigned)groups), dim3(64 * kWaves), 0, stream, a);
  else
    hipLaunchKernelGGL((k_kv_attend<DT, NC, MT, false>), dim3((unsigned)groups), dim3(64 * kWaves), 0, stream, a);
  if (joins > 0) hipLaunchKernelGGL((k_kv_join<DT, MT>), dim3((unsigned)joins, split), dim3(256), 0, stream, a);
}
template <int DT, int MT>
void launch_dim(const KvAttendArgs& a, hipStream_t stream) {
  if (a.cache.dim <= 64) launch<DT, 1, MT>(a, stream);
  else if (a.cache.dim <= 128) launch<DT, 2, MT>(a, stream);
  else if (a.cache.dim <= 192) launch<DT, 3, 1>(a, stream);  // the registers of two tiles are not there
  else launch<DT, 4, 1>(a, stream);
}
template <int DT>
void launch_of(const KvAttendArgs& a, hipStream_t stream) {
  // Two tiles of 16 rows a wave where a sequence has more than one: 32 rows on 4000 keys, 32 times,
  // 82 us, 97 by single tiles; 4 rows on up to 8100, 256 times, 400 us, 393 by single tiles.
  const int64_t rows = a.seqs.offsets == nullptr ? a.group : a.seqs.tokens * a.group / (a.seqs.seqs > 0 ? a.seqs.seqs : 1);
  if (rows > 16) launch_dim<DT, 2>(a, stream);
  else launch_dim<DT, 1>(a, stream);
}

int64_t counts_bytes(int64_t seqs) { return (4 * seqs + 255) / 256 * 256; }
int64_t few_workspace(int64_t dim) { return 256 + kPlaces * 32 + 4 * kPlaces * (dim <= 128 ? 32 : 16) * (2 + dim); }

}  // namespace

int64_t kv_attend_workspace(int64_t tokens, int64_t heads, int64_t kv_heads, int64_t dim, int64_t seqs, bool one_each) {
  const int64_t group = heads / kv_heads;
  int64_t need = few_workspace(dim) + (seqs > kOwnSearch ? 2 * counts_bytes(seqs) : 0);
  if (!all_few(all_rows(tokens, seqs, one_each, group), one_each, group, kMostRows / 2)) {  // whatever the pages
    const int64_t many = kv_prefill_workspace(kv_prefill_tiles(tokens, group, seqs), seqs, kv_heads, dim);
    if (many > need) need = many;
  }
  return need;
}

hipError_t launch_kv_attend(KvAttendArgs a, int dtype, void* workspace, hipStream_t stream) {
  const bool one_each = a.seqs.offsets == nullptr;
  const int most = most_rows(a.cache.dim, a.seqs.shift);
  const bool all = all_few(all_rows(a.seqs.tokens, a.seqs.seqs, one_each, a.group), one_each, a.group, most);
  a.few = all ? INT32_MAX : most;
  a.cut_count = static_cast<int32_t*>(workspace);
  a.heads_at = static_cast<uint8_t*>(workspace) + 256;
  a.sums = reinterpret_cast<float*>(a.heads_at + kPlaces * 32);
  a.counts = a.upto = a.upto_cut = nullptr;
  if (a.seqs.seqs > kOwnSearch) {
    a.counts = a.cut_count + 1;
    a.upto = reinterpret_cast<int32_t*>(static_cast<uint8_t*>(workspace) + few_workspace(a.cache.dim));
    a.upto_cut = a.upto + counts_bytes(a.seqs.seqs) / 4;
  }
  if (dtype == kBF16) launch_of<kBF16>(a, stream);
  else launch_of<kF16>(a, stream);
  if (!all) {
    // the workspace is used again: the stream keeps the two in order
    if (hipError_t e = launch_kv_prefill(a, dtype, kv_prefill_tiles(a.seqs.tokens, a.group, a.seqs.seqs), workspace, stream)) return e;
  }
  return hipGetLastError();
}

}  // namespace lrq
