// The experts' MLPs on FP8 weights in 128x128 tiles.  For a pair of a token t and
// one of its experts e,
//   g, u = x_q Wgu[e]^T (two halves), h = g / (1 + exp(-g)) u, y = h_q Wd[e]^T,
//   out[t] = sum over the token's pairs of weight y,
// with x and h quantized to e4m3 in 1x128 blocks.  Everything between is float32, but
// for the second product's sums within a block where it goes by tiles (f8f6f4); out is
// rounded once.  lrq_mma8.hpp has the products' mathematics.
//
// Few pairs: two launches, a pair by itself (its expert's weights are all that
// moves).  More: pairs are sorted by expert, and an expert's rows go through tiles
// whose gate and up rows meet in one wave; h leaves the first product quantized.
#include "lrq.h"
#include "lrq_device.hpp"
#include "lrq_internal.hpp"
#include "lrq_mma8.hpp"

namespace lrq {

// g / (1 + exp(-g)) u within some (|g| + 8) 2^-23 of itself for normal g above -131, and
// 0 below, where silu is under 1e-55.  With t = exp(-|g|), which cannot overflow, it is
// g u / (1 + t), times t for g < 0.  t = 2^hi (1 + lo ln 2), where hi + lo is -|g|
// log2(e) to twice float32's bits, by the hardware's 2^x and 1 / x (1 ulp each).  2^x
// has no results below 2^-126: below g = -70 it makes 2^64 t (hi + 64 is exact), and the
// factor goes out last, so that h leaves float32's range no sooner than it has to.
__device__ __forceinline__ float silu_mul(float g, float u) {
  constexpr float kHi = 1.44269502162933349609375f, kLo = 1.92596299112661746887e-8f;  // log2(e)
  const float a = fminf(__builtin_fabsf(g), 1000.0f), hi = -a * kHi;  // (exp(-1000) is 0; of a NaN, n stays one)
  const float lo = __builtin_fmaf(-a, kLo, __builtin_fmaf(-a, kHi, -hi));
  const bool deep = g < -70.0f;
  const float unit = deep ? 0x1p-64f : 1.0f;
  const float e = __builtin_amdgcn_exp2f(deep ? hi + 64.0f : hi);
  const float t = __builtin_fmaf(e, lo * 0.693147182f, e);
  const float n = g < 0.0f ? g * t : g;
  return n * __builtin_amdgcn_rcpf(__builtin_fmaf(t, unit, 1.0f)) * u * unit;
}

// ---------------------------------------------------------------------------
// Tokens quantized, pairs sorted by expert
// ---------------------------------------------------------------------------
// The first work-groups sort, kSortPairs pairs each (or a kSortMost-th of them): they
// count their pairs of each expert, which gives each pair its rank.  The experts'
// runs, the tiles of `bm` rows and each pair's place follow at once if there is one
// such work-group, in a launch of their own if there are more: atomics on a few
// words are slow, 32768 pairs take 42 us in one work-group, 19 in two launches of four.  Pairs of an
// expert come in any order, which no result depends on.  Ids outside 0 .. experts -
// 1 have no place.  The other work-groups meanwhile quantize x, 64 blocks each.
constexpr int kSortThreads = 1024, kSortAhead = 8, kSortPairs = 8192, kSortMost = 64, kBigRows = 256;

// Sums over the threads before this one, and over all.
template <int N>
__device__ __forceinline__ void sums_before(int (&v)[N], int (&all)[N], int32_t (*part)[kSortThreads / 64]) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int own[N];
#pragma unroll
  for (int i = 0; i < N; ++i) own[i] = v[i];
#pragma unroll
  for (int off = 1; off < 64; off *= 2)
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int o = __shfl_up(v[i], off, 64);
      v[i] += lane >= off ? o : 0;
    }
  if (lane == 63)
#pragma unroll
    for (int i = 0; i < N; ++i) part[i][wave] = v[i];
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) {
    all[i] = 0, v[i] -= own[i];
#pragma unroll
    for (int w = 0; w < kSortThreads / 64; ++w) {
      const int o = part[i][w];
      all[i] += o, v[i] += w < wave ? o : 0;
    }
  }
}

// From the pairs of each expert, one expert a thread: their runs' starts, where
// `before` of them belong to other work-groups, and (by the first) the tiles.  An
// expert's rows are cut into tiles of kBigRows, if `big`, as long as more than bm are
// left, and of bm; big tiles come first in the table.
__device__ __forceinline__ void lay_out(const ExpertArgs& a, int bm, bool big, int mine, int before, bool writes, int32_t* start,
                                        int32_t (*part)[kSortThreads / 64]) {
  const int tid = threadIdx.x;
  const int my_big = big ? (mine + kBigRows - 1 - bm) / kBigRows : 0;
  const int rest = mine - my_big * kBigRows, my_tiles = rest > 0 ? (rest + bm - 1) / bm : 0;
  int v[3] = {mine, my_big, my_tiles}, all[3];
  sums_before(v, all, part);
  const int first = v[0], tile_big = v[1], tile = all[1] + v[2];
  if (tid < a.experts) start[tid] = first + before;
  if (!writes) return;
  if (tid == 0) gst<int32_t>(a.total, all[1]), gst<int32_t>(a.total + 1, all[2]);
  for (int i = 0; i < my_big; ++i) {
    const int rows = mine - i * kBigRows < kBigRows ? mine - i * kBigRows : kBigRows;
    a.tiles[tile_big + i] = ExpertTile{tid, first + i * kBigRows, rows, 0};
  }
  for (int i = 0; i < my_tiles; ++i) {
    const int rows = rest - i * bm < bm ? rest - i * bm : bm;
    a.tiles[tile + i] = ExpertTile{tid, first + my_big * kBigRows + i * bm, rows, 0};
  }
}

template <int DT>
__global__ __launch_bounds__(kSortThreads) void k_ex_prepare(ExpertArgs a, int bm, bool big, int groups, int each) {
  __shared__ int32_t count[kExpertsMax], part[3][kSortThreads / 64];
  const int tid = threadIdx.x;
  if ((int)blockIdx.x >= groups) {
    const int64_t b = (int64_t)(blockIdx.x - groups) * (kSortThreads / 16) + (tid >> 4);
    const int64_t t = b / a.kb;
    if (t >= a.tokens) return;  // 16 lanes at once
    const int kb = (int)(b - t * a.kb), at = kb * kBlk + 8 * (tid & 15);
    float v[8], s;
    load_acts<DT>(static_cast<const uint8_t*>(a.x) + t * a.ldx * 2, at, a.hidden, v);
    const v2u q = quant8(v, s);
    if (at < a.hidden) *(LRQ_GLOBAL v2u_out*)(a.xq + t * a.hidden + at) = q;
    if ((tid & 15) == 0) gst<float>(a.xs + b, s);
    return;
  }
  const int pairs = (int)(a.tokens * a.top_k), group = blockIdx.x;
  const int p0 = group * each, p1 = p0 + each < pairs ? p0 + each : pairs;
  const uint32_t none = (uint32_t)a.experts;
  for (int e = tid; e < a.experts; e += kSortThreads) count[e] = 0;
  __syncthreads();
  uint32_t e[kSortAhead];
  int rank[kSortAhead];
  for (int p = p0 + tid; p < p1; p += kSortThreads * kSortAhead) {
#pragma unroll
    for (int i = 0; i < kSortAhead; ++i) e[i] = p + kSortThreads * i < p1 ? (uint32_t)gld<int32_t>(a.ids + p + kSortThreads * i) : none;
#pragma unroll
    for (int i = 0; i < kSortAhead; ++i) rank[i] = e[i] < none ? atomicAdd(&count[e[i]], 1) : 0;
    if (groups > 1)
#pragma unroll
      for (int i = 0; i < kSortAhead; ++i)
        if (e[i] < none) gst<int32_t>(a.rank + p + kSortThreads * i, rank[i]);
  }
  __syncthreads();
  const int mine = tid < a.experts ? count[tid] : 0;
  if (groups > 1) {
    if (tid < a.experts) gst<int32_t>(a.counts + group * a.experts + tid, mine);
    return;
  }
  // one group has kSortPairs at most: the thread's pairs are still in its registers
  lay_out(a, bm, big, mine, 0, true, count, part);
  __syncthreads();
  if (p0 + tid >= p1) return;
#pragma unroll
  for (int i = 0; i < kSortAhead; ++i)
    if (e[i] < none) gst<int32_t>(a.order + count[e[i]] + rank[i], p0 + tid + kSortThreads * i);
}

__global__ __launch_bounds__(kSortThreads) void k_ex_place(ExpertArgs a, int bm, bool big, int groups, int each) {
  __shared__ int32_t start[kExpertsMax], part[3][kSortThreads / 64];
  const int tid = threadIdx.x, group = blockIdx.x, pairs = (int)(a.tokens * a.top_k);
  const int p0 = group * each, p1 = p0 + each < pairs ? p0 + each : pairs;
  const uint32_t none = (uint32_t)a.experts;
  int mine = 0, before = 0;
  if (tid < a.experts)
    for (int g = 0; g < groups; ++g) {
      const int n = gld<int32_t>(a.counts + g * a.experts + tid);
      mine += n, before += g < group ? n : 0;
    }
  lay_out(a, bm, big, mine, before, group == 0, start, part);
  __syncthreads();
  for (int p = p0 + tid; p < p1; p += kSortThreads * kSortAhead) {
    uint32_t e[kSortAhead];
    int rank[kSortAhead];
#pragma unroll
    for (int i = 0; i < kSortAhead; ++i) {
      const bool has = p + kSortThreads * i < p1;
      const int q = has ? p + kSortThreads * i : p;
      e[i] = (uint32_t)gld<int32_t>(a.ids + q), rank[i] = gld<int32_t>(a.rank + q);
      if (!has) e[i] = none;
    }
#pragma unroll
    for (int i = 0; i < kSortAhead; ++i)
      if (e[i] < none) gst<int32_t>(a.order + start[e[i]] + rank[i], p + kSortThreads * i);
  }
}
static_assert(kSortPairs == kSortThreads * kSortAhead, "");

// Work-group wg's tile and its piece of nb, or of nb_big if the tile is a big one: each
// XCD (wg % 8) takes one run of the big tiles and one of the others, a tile's pieces after
// one another, so that it reads an expert's weights once, and the longest work comes first.
struct ExpertPiece {
  int tile, n;  // tile < 0: none is left
  bool big;
};
__device__ __forceinline__ ExpertPiece expert_piece(const ExpertArgs& a, int wg, int nb_big, int nb) {
  const int big = gld<int32_t>(a.total), rest = gld<int32_t>(a.total + 1);
  const int per_big = (big * nb_big + 7) >> 3, per = (rest * nb + 7) >> 3, i = wg >> 3, x = wg & 7;
  const bool is_big = i < per_big;
  const int t = is_big ? x * per_big + i : x * per + i - per_big, pieces = is_big ? nb_big : nb;
  if (t >= (is_big ? big : rest) * pieces || i - per_big >= per) return {-1, 0, false};
  return {t / pieces + (is_big ? 0 : big), t % pieces, is_big};
}

// h [rows, 128] of a work-group whose WN waves hold 16 NS columns each: lane (c, g)
// has columns 16 i + 4 g .. + 3 of rows 16 j + c.  Quantized and stored.
template <int NS, int FM, int WN>
__device__ __forceinline__ void store_hidden(const ExpertArgs& a, f32x4 (&h)[NS][FM], int first, int row0, int rows, int block, int wn,
                                             uint32_t* amax, int bm) {
  const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
#pragma unroll
  for (int j = 0; j < FM; ++j) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < NS; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const uint32_t v = f2u(h[i][j][r]) & 0x7FFFFFFFu;
        m = v > m ? v : m;
      }
    uint32_t o = (uint32_t)__shfl_xor((int)m, 16, 64);
    m = o > m ? o : m;
    o = (uint32_t)__shfl_xor((int)m, 32, 64);
    m = o > m ? o : m;
    if (g == 0) amax[wn * bm + row0 + 16 * j + c] = m;
  }
  lds_barrier8();
#pragma unroll
  for (int j = 0; j < FM; ++j) {
    const int row = row0 + 16 * j + c;
    uint32_t m = amax[row];
#pragma unroll
    for (int w = 1; w < WN; ++w) {
      const uint32_t o = amax[w * bm + row];
      m = o > m ? o : m;
    }
    const BlockScale b = block_scale<kF32>(m, false);
    if (row >= rows) continue;
    const int64_t at = first + row;
    if (wn == 0 && g == 0) gst<float>(a.hs + at * a.ib + block, b.s);
#pragma unroll
    for (int i = 0; i < NS; ++i) {
      const int n = 128 * block + 16 * (NS * wn + i) + 4 * g;
      if (n >= a.inter) continue;
      uint32_t q;
      if (b.kind >= kScaleInf) {
        q = 0;
#pragma unroll
        for (int r = 0; r < 4; ++r) q |= special_code<kF32>(h[i][j][r], b) << (8 * r);
      } else {
        q = cvt_e4m3x4(block_quot<kF32>(h[i][j][0], b), block_quot<kF32>(h[i][j][1], b), block_quot<kF32>(h[i][j][2], b),
                       block_quot<kF32>(h[i][j][3], b));
      }
      gst<uint32_t>(a.hq + at * a.inter + n, q);
    }
  }
}

// ---------------------------------------------------------------------------
// An expert's rows in tiles
// ---------------------------------------------------------------------------
// Weight rows of a tile: 16 of gate, the same 16 of up, and so on.
struct UpTile {
  static constexpr bool kCut = false, kSkip = true;
  const ExpertArgs& a;
  const ExpertTile& t;
  int block;
  __device__ const uint8_t* w() const { return a.gu + (int64_t)t.expert * 2 * a.inter * a.hidden; }
  __device__ const uint8_t* x() const { return a.xq; }
  __device__ uint32_t w_bytes() const { return (uint32_t)(2 * a.inter * a.hidden); }
  __device__ uint32_t x_bytes() const { return (uint32_t)(a.tokens * a.hidden); }
  __device__ int column(int r) const { return 128 * block + 16 * (r >> 5) + (r & 15); }
  __device__ uint32_t w_off(int r) const {
    const int n = column(r);
    return n < a.inter ? (uint32_t)((r >> 4 & 1 ? a.inter : 0) + n) * (uint32_t)a.hidden : kNoRow;
  }
  __device__ int token(int r) const { return gld<int32_t>(a.order + t.first + (r < t.rows ? r : t.rows - 1)) / a.top_k; }
  __device__ uint32_t x_off(int r) const { return r < t.rows ? (uint32_t)token(r) * (uint32_t)a.hidden : kNoRow; }
  __device__ int tokens() const { return t.rows; }
  __device__ const float* sx() const { return a.xs; }
  __device__ const float* sw() const { return a.gus + (int64_t)t.expert * a.gb * a.kb; }
  __device__ uint32_t sx_bytes() const { return (uint32_t)(4 * a.tokens * a.kb); }
  __device__ uint32_t sw_bytes() const { return (uint32_t)(4 * a.gb * a.kb); }
  __device__ uint32_t sx_off(int r) const { return 4 * (uint32_t)token(r) * (uint32_t)a.kb; }
  __device__ uint32_t sw_off(int s) const {
    const int n = column(16 * s) < a.inter ? column(16 * s) : a.inter - 1;
    return (uint32_t)(4 * (((s & 1 ? a.inter : 0) + n) / kBlk) * a.kb);
  }
};

// h comes from float32 sums (lrq_mma8.hpp), in whatever tile, so that a token's hidden
// codes do not depend on the tokens beside it.  The f8f6f4 instructions' sums are off by
// 1.5e-5 of their norm, which is little beside h's 4 bits, but moves one code in some
// 3000 to its neighbour: 2e-3 of the norm of out, as much as a bf16 result's rounding
// (0.0026 against 64 bits, 0.0018 as here).  4096 tokens of 8 pairs x 768 take 520 us,
// 400 with them; 200 on a quarter, where memory bounds both, 54 and 51.
// Big tiles are taken in parts of BM rows, side by side: conversions to bf16 take the
// registers of 256.
template <int FN, int FM, int WN, int WM, int STAGES>
__global__ __launch_bounds__(64 * WN * WM, 1) void k_ex_up_tiles(ExpertArgs a) {
  static_assert(16 * FN * WN == 256, "128 columns of h");
  constexpr int BM = 16 * FM * WM, PARTS = kBigRows / BM;
  __shared__ __attribute__((aligned(16))) uint8_t lds[kTileLds<FN, FM, WN, WM, STAGES>];
  const ExpertPiece p = expert_piece(a, blockIdx.x, PARTS * a.ib, a.ib);
  if (p.tile < 0) return;
  ExpertTile t = a.tiles[p.tile];
  const int block = p.big ? p.n / PARTS : p.n, part = p.big ? p.n % PARTS : 0;
  t.first += BM * part, t.rows -= BM * part;
  if (t.rows <= 0) return;
  t.rows = t.rows < BM ? t.rows : BM;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  f32x4 acc[FN][FM], h[FN / 2][FM];
  tile_sums<FN, FM, WN, WM, STAGES, true, true, true>(UpTile{a, t, block}, a.hidden, 0, a.kb, lds, acc);
#pragma unroll
  for (int i = 0; i < FN / 2; ++i)
#pragma unroll
    for (int j = 0; j < FM; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r) h[i][j][r] = silu_mul(acc[2 * i][j][r], acc[2 * i + 1][j][r]);
  store_hidden<FN / 2, FM, WN>(a, h, t.first, wave % WM * 16 * FM, t.rows, block, wave / WM, reinterpret_cast<uint32_t*>(lds), BM);
}

template <bool SKIP>
struct DownTile {
  static constexpr bool kCut = false, kSkip = SKIP;
  const ExpertArgs& a;
  const ExpertTile& t;
  int n0;
  __device__ const uint8_t* w() const { return a.dn + (int64_t)t.expert * a.hidden * a.inter; }
  __device__ const uint8_t* x() const { return a.hq + (int64_t)t.first * a.inter; }
  __device__ uint32_t w_bytes() const { return (uint32_t)(a.hidden * a.inter); }
  __device__ uint32_t x_bytes() const { return (uint32_t)(t.rows * a.inter); }
  __device__ uint32_t w_off(int r) const { return n0 + r < a.hidden ? (uint32_t)(n0 + r) * (uint32_t)a.inter : kNoRow; }
  __device__ uint32_t x_off(int r) const { return r < t.rows ? (uint32_t)r * (uint32_t)a.inter : kNoRow; }
  __device__ int tokens() const { return t.rows; }
  __device__ const float* sx() const { return a.hs + (int64_t)t.first * a.ib; }
  __device__ const float* sw() const { return a.dns + (int64_t)t.expert * a.kb * a.ib; }
  __device__ uint32_t sx_bytes() const { return (uint32_t)(4 * t.rows * a.ib); }
  __device__ uint32_t sw_bytes() const { return (uint32_t)(4 * a.kb * a.ib); }
  __device__ uint32_t sx_off(int r) const { return (uint32_t)(4 * (r < t.rows ? r : t.rows - 1) * a.ib); }
  __device__ uint32_t sw_off(int s) const {
    const int n = n0 + 16 * s < a.hidden ? n0 + 16 * s : a.hidden - 1;
    return (uint32_t)(4 * (n / kBlk) * a.ib);
  }
};

template <int FN, int FM, int WN, int WM, int STAGES, bool SKIP = true>
__device__ __forceinline__ void down_tile(const ExpertArgs& a, const ExpertTile& t, int block, uint8_t* lds) {
  static_assert(16 * FN <= kBlk, "one scale for a wave's rows");
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = lane & 15, g = lane >> 4, wn = wave / WM * 16 * FN, wm = wave % WM * 16 * FM;
  const DownTile<SKIP> src{a, t, block * 16 * FN * WN};
  f32x4 acc[FN][FM];
  tile_sums<FN, FM, WN, WM, STAGES, true, false, false>(src, a.inter, 0, a.ib, lds, acc);
#pragma unroll
  for (int j = 0; j < FM; ++j) {
    const int row = wm + 16 * j + c;
    if (row >= t.rows) continue;
    const int pair = gld<int32_t>(a.order + t.first + row);
    const float w = gld<float>(a.weights + pair);
#pragma unroll
    for (int i = 0; i < FN; ++i) {
      const int n = src.n0 + wn + 16 * i + 4 * g;
      if (n < a.hidden)
        gst<f32x4>(a.y + (int64_t)pair * a.hidden + n, f32x4{acc[i][j][0] * w, acc[i][j][1] * w, acc[i][j][2] * w, acc[i][j][3] * w});
    }
  }
}

template <int FN, int FM, int WN, int WM, int STAGES>
__global__ __launch_bounds__(64 * WN * WM, 1) void k_ex_down_tiles(ExpertArgs a) {
  constexpr int BN = 16 * FN * WN;
  __shared__ __attribute__((aligned(16))) uint8_t lds[kTileLds<FN, FM, WN, WM, STAGES>];
  const int nb = (a.hidden + BN - 1) / BN;
  const ExpertPiece p = expert_piece(a, blockIdx.x, nb, nb);
  if (p.tile < 0) return;
  const ExpertTile t = a.tiles[p.tile];
  down_tile<FN, FM, WN, WM, STAGES>(a, t, p.n, lds);
}
// Tiles of 256 and of up to 128 rows in one launch: the large ones take 49 us a round
// over the chip, of 4096 k, and the others 31 (and cut experts' rows with less left
// over: 32768 pairs of 128 experts in 27 % more rows than there are, 256 rows alone in
// 55 %).  4096 tokens of 8 pairs: 144 us, 171 in tiles of 128.
constexpr int kMixedLds = kTileLds<4, 4, 4, 2, 3> > kTileLds<8, 4, 2, 4, 2> ? kTileLds<4, 4, 4, 2, 3> : kTileLds<8, 4, 2, 4, 2>;
__global__ __launch_bounds__(512, 1) void k_ex_down_mixed(ExpertArgs a) {
  __shared__ __attribute__((aligned(16))) uint8_t lds[kMixedLds];
  const int nb = (a.hidden + 255) / 256;
  const ExpertPiece p = expert_piece(a, blockIdx.x, nb, nb);
  if (p.tile < 0) return;
  const ExpertTile t = a.tiles[p.tile];
  if (t.rows > 128) down_tile<8, 4, 2, 4, 2, false>(a, t, p.n, lds);
  else down_tile<4, 4, 4, 2, 3>(a, t, p.n, lds);
}

// out[t] = the sum of the token's rows of y, in the order of its pairs.
template <int DT>
__global__ __launch_bounds__(256) void k_ex_sum(ExpertArgs a) {
  const int64_t at = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 8;
  if (at >= a.tokens * a.hidden) return;
  const int64_t t = at / a.hidden, n = at % a.hidden;
  float s[8] = {0, 0, 0, 0, 0, 0, 0, 0};
  constexpr int AHEAD = 8;
  for (int j0 = 0; j0 < a.top_k; j0 += AHEAD) {
    f32x4 lo[AHEAD], hi[AHEAD];
    bool has[AHEAD];
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      const int64_t pair = t * a.top_k + (j0 + j < a.top_k ? j0 + j : 0);
      has[j] = j0 + j < a.top_k && (uint32_t)gld<int32_t>(a.ids + pair) < (uint32_t)a.experts;
      lo[j] = gld_nt<f32x4>(a.y + pair * a.hidden + n), hi[j] = gld_nt<f32x4>(a.y + pair * a.hidden + n + 4);
    }
#pragma unroll
    for (int j = 0; j < AHEAD; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        s[i] = has[j] ? s[i] + lo[j][i] : s[i];
        s[4 + i] = has[j] ? s[4 + i] + hi[j][i] : s[4 + i];
      }
  }
  uint32_t b[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) b[i] = bits16<DT>(s[i]);
  *(LRQ_GLOBAL v4u_any*)(static_cast<uint16_t*>(a.out) + at) = v4u{b[0] | b[1] << 16, b[2] | b[3] << 16, b[4] | b[5] << 16, b[6] | b[7] << 16};
}

// ---------------------------------------------------------------------------
// Few pairs
// ---------------------------------------------------------------------------
// h of a pair: a wave makes one column, from its rows of gate and up; x is
// quantized by every work-group while the first weights are on their way.
template <int DT>
__global__ __launch_bounds__(512) void k_ex_up_few(ExpertArgs a) {
  constexpr int D = 4;
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  const int pair = blockIdx.y, lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int expert = gld<int32_t>(a.ids + pair);
  if ((uint32_t)expert >= (uint32_t)a.experts) return;
  const int n = 8 * blockIdx.x + wave, chunks = (a.hidden + 1023) / 1024, pitch = a.kb * kBlk;
  float* const scales = reinterpret_cast<float*>(lds + pitch);
  const GlobalCodes w[2] = {(GlobalCodes)a.gu + ((int64_t)expert * 2 * a.inter + n) * a.hidden,
                            (GlobalCodes)a.gu + ((int64_t)expert * 2 * a.inter + a.inter + n) * a.hidden};
  const float* const sw[2] = {a.gus + ((int64_t)expert * a.gb + n / kBlk) * a.kb,
                              a.gus + ((int64_t)expert * a.gb + (a.inter + n) / kBlk) * a.kb};
  struct Chunk {
    v4u w[2];
    float s[2];
  } st[D];
  auto load = [&](Chunk& c, int i) {
    if (i >= chunks) return;
    const int at = 1024 * i + 16 * lane, kb = at < a.hidden ? at / kBlk : 0;
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      c.w[r] = at < a.hidden ? load_codes_nt(w[r] + at) : v4u{0, 0, 0, 0};
      c.s[r] = gld<float>(sw[r] + kb);
    }
  };
#pragma unroll
  for (int d = 0; d < D; ++d) load(st[d], d);
  quant_row<DT, 512>(static_cast<const uint8_t*>(a.x) + (int64_t)(pair / a.top_k) * a.ldx * 2, a.hidden, a.kb, lds, scales);
  lds_barrier8();
  float acc[2] = {0.0f, 0.0f};
  for (int i0 = 0; i0 < chunks; i0 += D) {
#pragma unroll
    for (int d = 0; d < D; ++d) {
      if (i0 + d >= chunks) break;
      const int at = 1024 * (i0 + d) + 16 * lane, x_at = at < a.hidden ? at : 0;
      const Floats16 x = codes_to_f32(*reinterpret_cast<const v4u*>(lds + x_at));
      const float s = scales[x_at / kBlk];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const float p = dot16(codes_to_f32(st[d].w[r]), x);
        acc[r] = at < a.hidden ? __builtin_fmaf(p, s * st[d].s[r], acc[r]) : acc[r];
      }
      load(st[d], i0 + d + D);
    }
  }
  const float g = lanes_sum(acc[0]), u = lanes_sum(acc[1]);
  if (lane == 0) gst<float>(a.y + (int64_t)pair * a.inter + n, silu_mul(g, u));
}

// A token's output: a wave makes one column of all its pairs, whose h every
// work-group quantizes; the pairs' K stand one after another.
template <int DT>
__global__ __launch_bounds__(512) void k_ex_down_few(ExpertArgs a) {
  constexpr int D = 6;
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  const int t = blockIdx.y, lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = 8 * blockIdx.x + wave, each = a.inter / 16, pieces = a.top_k * each, chunks = (pieces + 63) / 64;
  const int pitch = a.ib * kBlk;
  float* const scales = reinterpret_cast<float*>(lds + a.top_k * pitch);
  // lane j holds pair j's expert and weight
  const int64_t first = (int64_t)t * a.top_k;
  const int id = lane < a.top_k ? gld<int32_t>(a.ids + first + lane) : -1;
  const float weight = lane < a.top_k ? gld<float>(a.weights + first + lane) : 0.0f;
  struct Chunk {
    v4u w;
    float s;
    int at;  // of the piece in LDS, -1: none
  } st[D];
  auto load = [&](Chunk& c, int i) {
    if (i >= chunks) return;
    const int p = 64 * i + lane, j = p < pieces ? p / each : 0, k = 16 * (p - j * each);
    const int expert = __shfl(id, j, 64);
    const float f = __shfl(weight, j, 64);
    c.at = p < pieces && (uint32_t)expert < (uint32_t)a.experts ? j * pitch + k : -1;
    c.w = v4u{0, 0, 0, 0}, c.s = 0.0f;
    if (c.at < 0) return;
    c.w = load_codes_nt((GlobalCodes)a.dn + (((int64_t)expert * a.hidden + n) * a.inter + k));
    c.s = f * gld<float>(a.dns + ((int64_t)expert * a.kb + n / kBlk) * a.ib + k / kBlk);
  };
#pragma unroll
  for (int d = 0; d < D; ++d) load(st[d], d);
  for (int b = threadIdx.x >> 4; b < a.top_k * a.ib; b += 32) {
    const int j = b / a.ib, at = (b - j * a.ib) * kBlk + 8 * (threadIdx.x & 15);
    float v[8], q;
    load_acts<kF32>(a.y + (first + j) * a.inter, at, a.inter, v);
    *reinterpret_cast<v2u*>(lds + j * pitch + at) = quant8(v, q);
    if ((threadIdx.x & 15) == 0) scales[b] = q;
  }
  lds_barrier8();
  float acc = 0.0f;
  for (int i0 = 0; i0 < chunks; i0 += D) {
#pragma unroll
    for (int d = 0; d < D; ++d) {
      if (i0 + d >= chunks) break;
      const int at = st[d].at < 0 ? 0 : st[d].at;
      const float p = dot16(codes_to_f32(st[d].w), codes_to_f32(*reinterpret_cast<const v4u*>(lds + at)));
      acc = st[d].at < 0 ? acc : __builtin_fmaf(p, scales[at / kBlk] * st[d].s, acc);
      load(st[d], i0 + d + D);
    }
  }
  acc = lanes_sum(acc);
  if (lane == 0) gst<uint16_t>(static_cast<uint16_t*>(a.out) + (int64_t)t * a.hidden + n, bits16<DT>(acc));
}

// ---------------------------------------------------------------------------
// Which kernels, and their memory
// ---------------------------------------------------------------------------
static int64_t up256(int64_t v) { return (v + 255) / 256 * 256; }

// Rows of a tile, by the pairs an expert has on average; 0 for few pairs.  us in tiles
// of 16, 64 and 128 rows (256 and 128 in the second product): with 128 experts of 2048 x
// 192, 100 tokens of 8 pairs 49, 51, 67; 200 tokens 57, 55, 72; 800 tokens 110, 95, 127;
// 2048 tokens -, 168, 173; 4096 tokens -, 281, 267.  Of 2048 x 768: 200 tokens 130, 137,
// 164; 512 tokens 192, 164, 190; 2048 tokens -, 330, 322; 4096 tokens -, 551, 511.  32
// rows win nowhere.
static int expert_rows(int64_t tokens, const ExpertArgs& a) {
  const int64_t pairs = tokens * a.top_k, few_lds = (int64_t)a.top_k * a.ib * (kBlk + 4);
  if (pairs <= 64 && pairs <= a.experts && few_lds <= 48 * 1024 && a.kb * (kBlk + 4) <= 48 * 1024) return 0;
  const int64_t each = pairs / a.experts;
  return each < 16 ? 16 : each < 128 ? 64 : 128;
}
// Tokens of a pass: 32-bit offsets into the codes of x, 1 GiB of y and 1 GiB of h's codes.
static int64_t expert_pass(int64_t tokens, const ExpertArgs& a) {
  const int64_t y = (int64_t(1) << 28) / ((int64_t)a.top_k * a.hidden), h = (int64_t(1) << 30) / ((int64_t)a.top_k * a.inter);
  int64_t most = y < h ? y : h;
  most = most < 1 ? 1 : most;
  return tokens < most ? tokens : most;
}
static int64_t tile_bound(int64_t pairs, int bm, int experts) {
  return (pairs + bm - 1) / bm + (pairs < experts ? pairs : experts);
}

static int64_t expert_layout(int64_t tokens, int bm, ExpertArgs& a, uint8_t* base) {
  const int64_t pairs = tokens * a.top_k;
  int64_t at = 0;
  auto take = [&](int64_t bytes) { uint8_t* p = base + at; at += up256(bytes); return p; };
  if (bm == 0) {
    a.y = reinterpret_cast<float*>(take(4 * pairs * a.inter));
    return at;
  }
  a.xq = take(tokens * a.hidden);
  a.xs = reinterpret_cast<float*>(take(4 * tokens * a.kb));
  a.order = reinterpret_cast<int32_t*>(take(4 * pairs));
  a.rank = reinterpret_cast<int32_t*>(take(4 * pairs));
  a.counts = reinterpret_cast<int32_t*>(take(4 * kSortMost * (int64_t)a.experts));
  a.total = reinterpret_cast<int32_t*>(take(8));
  a.tiles = reinterpret_cast<ExpertTile*>(take((int64_t)sizeof(ExpertTile) * tile_bound(pairs, bm, a.experts)));
  a.hq = take(pairs * a.inter);
  a.hs = reinterpret_cast<float*>(take(4 * pairs * a.ib));
  a.y = reinterpret_cast<float*>(take(4 * pairs * a.hidden));
  return at;
}

int64_t experts_workspace(int64_t tokens, ExpertArgs a) {
  const int64_t pass = expert_pass(tokens, a);
  int64_t most = expert_layout(pass, expert_rows(pass, a), a, nullptr);
  if (tokens % pass) {  // the last pass can be laid out otherwise
    const int64_t last = expert_layout(tokens % pass, expert_rows(tokens % pass, a), a, nullptr);
    most = last > most ? last : most;
  }
  return most;
}

template <int DT>
static hipError_t few(const ExpertArgs& a, hipStream_t stream) {
  const unsigned up = (unsigned)(a.kb * (kBlk + 4)), down = (unsigned)(a.top_k * a.ib * (kBlk + 4));
  hipLaunchKernelGGL((k_ex_up_few<DT>), dim3((unsigned)(a.inter / 8), (unsigned)(a.tokens * a.top_k)), dim3(512), up, stream, a);
  hipLaunchKernelGGL((k_ex_down_few<DT>), dim3((unsigned)(a.hidden / 8), (unsigned)a.tokens), dim3(512), down, stream, a);
  return hipGetLastError();
}

template <int FN, int FM, int WN, int WM, int STAGES>
static void up(const ExpertArgs& a, int64_t tiles, hipStream_t stream) {
  hipLaunchKernelGGL((k_ex_up_tiles<FN, FM, WN, WM, STAGES>), dim3((unsigned)((tiles * a.ib + 7) / 8 * 8)), dim3(64 * WN * WM), 0,
                     stream, a);
}
template <int FN, int FM, int WN, int WM, int STAGES>
static void down(const ExpertArgs& a, int64_t tiles, hipStream_t stream) {
  constexpr int BN = 16 * FN * WN;
  hipLaunchKernelGGL((k_ex_down_tiles<FN, FM, WN, WM, STAGES>), dim3((unsigned)((tiles * ((a.hidden + BN - 1) / BN) + 7) / 8 * 8)),
                     dim3(64 * WN * WM), 0, stream, a);
}

hipError_t launch_experts(ExpertArgs a, int dtype, int64_t tokens, void* workspace, hipStream_t stream) {
  const int64_t pass = expert_pass(tokens, a);
  const uint8_t* const x = static_cast<const uint8_t*>(a.x);
  const int32_t* const ids = a.ids;
  const float* const weights = a.weights;
  uint8_t* const out = static_cast<uint8_t*>(a.out);
  for (int64_t t0 = 0; t0 < tokens; t0 += pass) {
    a.tokens = tokens - t0 < pass ? tokens - t0 : pass;
    a.x = x + 2 * t0 * a.ldx, a.ids = ids + t0 * a.top_k, a.weights = weights + t0 * a.top_k, a.out = out + 2 * t0 * a.hidden;
    const int bm = expert_rows(a.tokens, a);
    expert_layout(a.tokens, bm, a, static_cast<uint8_t*>(workspace));
    if (bm == 0) {
      if (hipError_t e = dtype == kBF16 ? few<kBF16>(a, stream) : few<kF16>(a, stream)) return e;
      continue;
    }
    const int64_t pairs = a.tokens * a.top_k, tiles = tile_bound(pairs, bm, a.experts);
    const bool big = bm == 128;
    int64_t each = (pairs + kSortMost - 1) / kSortMost;
    each = each < kSortPairs ? kSortPairs : each;
    const int groups = (int)((pairs + each - 1) / each);
    const dim3 prepare((unsigned)(groups + (a.tokens * a.kb + kSortThreads / 16 - 1) / (kSortThreads / 16)));
    if (dtype == kBF16) hipLaunchKernelGGL((k_ex_prepare<kBF16>), prepare, dim3(kSortThreads), 0, stream, a, bm, big, groups, (int)each);
    else hipLaunchKernelGGL((k_ex_prepare<kF16>), prepare, dim3(kSortThreads), 0, stream, a, bm, big, groups, (int)each);
    if (groups > 1) hipLaunchKernelGGL(k_ex_place, dim3((unsigned)groups), dim3(kSortThreads), 0, stream, a, bm, big, groups, (int)each);
    if (bm == 16) {
      up<2, 1, 8, 1, 2>(a, tiles, stream);
      down<1, 1, 4, 1, 2>(a, tiles, stream);
    } else if (bm == 64) {
      up<4, 2, 4, 2, 3>(a, tiles, stream);
      down<4, 2, 2, 2, 2>(a, tiles, stream);
    } else {
      // each kind's runs are rounded up to 8 pieces: 16 tiles more hold them
      up<4, 4, 4, 2, 3>(a, tiles + 16, stream);
      hipLaunchKernelGGL(k_ex_down_mixed, dim3((unsigned)(tiles + 16) * (unsigned)((a.hidden + 255) / 256)), dim3(512), 0, stream, a);
    }
    const dim3 sum((unsigned)((a.tokens * a.hidden / 8 + 255) / 256));
    if (dtype == kBF16) hipLaunchKernelGGL((k_ex_sum<kBF16>), sum, dim3(256), 0, stream, a);
    else hipLaunchKernelGGL((k_ex_sum<kF16>), sum, dim3(256), 0, stream, a);
    if (hipError_t e = hipGetLastError()) return e;
  }
  return hipSuccess;
}

}  // namespace lrq
