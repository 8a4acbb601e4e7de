// Attention of each sequence's last tokens over all of its own, on an FP8 KV cache.
//
//   o = sum_j p_j v_j / sum_j p_j,   p_j = 2^(c (q . k_j) - m),   c = scale log2(e),
// with m the running maximum of a row, in one pass over the keys.  A row is a new token
// and one of its query heads; the rows that share a KV head are taken together, 16 a
// work-group, so that each code is read once for all of them.
//
// Both products run on bf16 or fp16 matrix instructions (float32 sums): e4m3 codes are
// exact in both types, and the keys' scale is applied to the sums.  The first product
// takes the queries' own type.  The second takes p in fp16 and V's codes without their
// scale, which is folded into p: with e_j = log2 of the scale of v_j's page,
//   o 2^M = sum_j 2^(s_j + e_j - M) code_j,   l 2^M = sum_j 2^(s_j + e_j - M) 2^-e_j,
// M the running maximum of s + e.  So p has 11 bits and a range of 2^-34 below the
// largest term (it is taken 2^10 times as large, and fp16's subnormals count), where bf16
// would have 8 bits: its rounding is then far below that of a 16-bit result.
//
// Layout: both products are taken transposed, S^T = K Q^T and O^T = V^T P^T, on 16x16x32
// instructions.  Lane l holds of every result the column l % 16, a row of queries, and so
// one maximum and one sum.  Keys are taken 64 at a time; key 16 (l / 16) + 4 t + i is
// result i of tile t in lane l, so that a lane's 16 probabilities are those of the 16
// keys whose V codes it loads with one 16-byte load, in its order, and P never leaves the
// registers.
#include "lrq_kv.hpp"
#include "lrq_kv_attend.hpp"

namespace lrq {

namespace {

constexpr int kRows = 16;    // rows of a work-group
constexpr int kWaves = 4;
constexpr int kJoinTiles = 8;  // tiles of 16 channels that the waves' sums go through LDS with
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
__device__ __forceinline__ int64_t row_tiles(const KvSeq& q, int group, int few) {
  const int64_t rows = (int64_t)q.n * group;
  return rows > few ? 0 : (rows + kRows - 1) / kRows;
}

// ---------------------------------------------------------------------------
// Work: the units of all items (sequence, KV head, 16 rows) stand in one line, which is
// cut into equal parts, one a work-group, whatever lengths the sequences have.  Where a
// cut falls inside an item, its parts leave unnormalized sums, which k_kv_join puts
// together.  Part w has two places for them: 2 w for an item that an earlier part
// began, 2 w + 1 for one that it begins and a later part ends.
// ---------------------------------------------------------------------------
constexpr int kPlaceWords = kRows * 2;  // maxima and sums; then kRows x dim
struct Item {
  int b, h, tile, unit;  // unit: where in the item
  int64_t left;          // units of the item from `unit` on
};

struct PartHead {
  int64_t first;  // the item's first row's token
  int rows;       // rows of the tile, 0: no such item
  int tile, h;
  int parts;      // parts that hold pieces of it, the first included
};
static_assert(sizeof(PartHead) <= 32, "the join's heads are 32 bytes apart");

template <int DT, int NC>
__global__ __launch_bounds__(64 * kWaves) void k_kv_attend(KvAttendArgs a) {
  constexpr int NT = 4 * NC;  // tiles of 16 channels
  extern __shared__ float lds[];  // waves' maxima and sums, then their sums of values
  __shared__ int64_t scan[kWaves];
  __shared__ int64_t found[4];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r = lane & 15, g = lane >> 4;
  const int shift = a.seqs.shift, S = 1 << shift, dim = a.cache.dim, group = a.group;
  const int64_t part = blockIdx.x;

  // rows of the result that are no sequence's
  if (a.zero_rest) {
    int64_t lo = a.seqs.seqs, hi = a.seqs.tokens;
    if (a.seqs.offsets != nullptr) lo = gld<int32_t>(a.seqs.offsets + a.seqs.seqs);
    lo = lo < 0 ? 0 : lo;
    const int64_t words = (int64_t)a.heads * dim / 2;
    for (int64_t t = lo + part; t < hi; t += gridDim.x) {
      for (int64_t i = tid; i < words; i += 64 * kWaves) gst<uint32_t>(static_cast<uint32_t*>(a.out) + t * words + i, 0u);
      if (a.lse != nullptr)
        for (int i = tid; i < a.heads; i += 64 * kWaves) gst<float>(a.lse + t * a.heads + i, -INFINITY);
    }
  }

  auto work_of = [&](int b) -> int64_t {
    const KvSeq q = kv_seq(a.seqs, b);
    return row_tiles(q, group, a.few) * a.cache.heads * span_of(q, a.window).count;
  };
  // all work, then the sequence in which this part begins
  int64_t total = 0;
  for (int b0 = 0; b0 < a.seqs.seqs; b0 += 64 * kWaves) {
    const int64_t upto = block_scan<64 * kWaves, int64_t>(b0 + tid < a.seqs.seqs ? work_of(b0 + tid) : 0, scan);
    if (tid == 64 * kWaves - 1) found[3] = upto;
    __syncthreads();
    total += found[3];
    __syncthreads();
  }
  int64_t per = (total + gridDim.x - 1) / gridDim.x;
  if (per < a.least) per = a.least;
  const int64_t begin = part * per;
  int64_t end = begin + per < total ? begin + per : total;
  PartHead* const head = reinterpret_cast<PartHead*>(a.heads_at + 32 * part);
  if (tid == 0) head->rows = 0;
  if (begin >= end) return;
  {
    int64_t before = 0;
    for (int b0 = 0; b0 < a.seqs.seqs; b0 += 64 * kWaves) {
      const int64_t mine = b0 + tid < a.seqs.seqs ? work_of(b0 + tid) : 0;
      const int64_t upto = before + block_scan<64 * kWaves, int64_t>(mine, scan);
      if (begin >= upto - mine && begin < upto) found[0] = b0 + tid, found[1] = begin - (upto - mine);
      if (tid == 64 * kWaves - 1) found[3] = upto;
      __syncthreads();
      before = found[3];
      __syncthreads();
      if (begin < before) break;
    }
  }
  int b = __builtin_amdgcn_readfirstlane((int)found[0]);
  int64_t inside = found[1];
  __syncthreads();

  for (int64_t at = begin; at < end && b < a.seqs.seqs;) {
    const KvSeq q = kv_seq(a.seqs, b);
    const Span span = span_of(q, a.window);
    const int64_t tiles = row_tiles(q, group, a.few);
    if (inside >= tiles * a.cache.heads * span.count) {  // the next sequence
      ++b, inside = 0;
      continue;
    }
    const int64_t item = inside / span.count;
    const int from = (int)(inside - item * span.count);
    const int64_t most = end - at;
    const int to = span.count - from < most ? span.count : from + (int)most;
    const int h = (int)(item / tiles);
    const int64_t tile = item - h * tiles;
    const int64_t row0 = tile * kRows;
    const int rows = (int)((int64_t)q.n * group - row0 < kRows ? (int64_t)q.n * group - row0 : kRows);

    // this lane's row: token and head, and the keys [lo, hi) that it sees
    const int64_t mine = row0 + (r < rows ? r : 0);
    const int tok = (int)(mine / group), qh = h * group + (int)(mine - (int64_t)tok * group);
    const int pos = q.len - q.n + tok;  // below 0: it sees none
    const int hi = pos + 1 < 0 ? 0 : pos + 1;
    const int lo = a.window > 0 && pos + 1 > a.window ? pos + 1 - a.window : 0;
    // what the first and the last row see (rows are in the order of their tokens)
    const int tok_a = (int)(row0 / group), tok_b = (int)((row0 + rows - 1) / group);
    const int hi_a = q.len - q.n + tok_a + 1, hi_b = q.len - q.n + tok_b + 1;
    const int lo_a = a.window > 0 && hi_a > a.window ? hi_a - a.window : 0;
    const int lo_b = a.window > 0 && hi_b > a.window ? hi_b - a.window : 0;

    v4u qf[NC][2];
    {
      const uint16_t* const src = static_cast<const uint16_t*>(a.q) + (q.first + tok) * a.q_token + qh * a.q_head;
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const int d = 64 * c + 16 * g + 8 * k;
          qf[c][k] = v4u{0, 0, 0, 0};
          if (d < dim && r < rows) qf[c][k] = load_live(src + d);
        }
    }
    float m = kLow, l = 0.0f;
    f32x4 acc[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) acc[n] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

    for (int u = from + wave; u < to; u += kWaves) {
      const int key0 = (span.first + u) * kUnit;
      if (key0 >= hi_b || key0 + kUnit <= lo_a) continue;  // none of the rows sees any
      // K: this lane's row of a tile is key 16 (r / 4) + 4 t + r % 4; V: keys 16 g ..
      const int k_key = key0 + 16 * (r >> 2), v_key = key0 + 16 * g;
      const int k_place = k_key >> shift, v_place = v_key >> shift;
      const int kp = k_place < a.seqs.width ? kv_page(a.seqs, a.cache.pages, b, k_place) : -1;
      const int vp = v_place < a.seqs.width ? kv_page(a.seqs, a.cache.pages, b, v_place) : -1;
      const uint8_t* const kb = a.cache.k + (int64_t)(kp < 0 ? 0 : kp) * a.cache.k_page +
                                ((int64_t)h * S + (k_key & (S - 1)) + (r & 3)) * dim + 16 * g;
      const uint8_t* const vb = a.cache.v + (int64_t)(vp < 0 ? 0 : vp) * a.cache.v_page + (int64_t)h * S * dim + r * S + (v_key & (S - 1));
      const float ks = gld<float>(a.cache.ks + (int64_t)(vp < 0 ? 0 : vp) * a.cache.ks_page + h);
      const float vs = gld<float>(a.cache.vs + (int64_t)(vp < 0 ? 0 : vp) * a.cache.vs_page + h);
      v4u kr[4][NC], vr[NT];
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          kr[t][c] = v4u{0, 0, 0, 0};
          if (64 * c + 16 * g < dim) kr[t][c] = gld<v4u>(kb + 4 * t * dim + 64 * c);
        }
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        vr[n] = v4u{0, 0, 0, 0};
        if (16 * n < dim) vr[n] = gld<v4u>(vb + (int64_t)16 * n * S);
      }

      f32x4 s[4];
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        s[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          if (64 * c >= dim) continue;
          s[t] = mma<DT>(widen8<DT>(kr[t][c].x, kr[t][c].y), qf[c][0], s[t]);
          s[t] = mma<DT>(widen8<DT>(kr[t][c].z, kr[t][c].w), qf[c][1], s[t]);
        }
      }
      const float factor = ks * a.scale;
      const float ev = __builtin_amdgcn_logf(__builtin_amdgcn_fmed3f(vs, 0x1p-48f, 0x1p48f));
      const float back = __builtin_amdgcn_exp2f(-ev);
      const bool cut = key0 + kUnit > hi_a || key0 < lo_b || __ballot(vp < 0 || kp < 0) != 0;
      float x[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) x[i] = __builtin_fmaf(s[i >> 2][i & 3], factor, ev);
      uint32_t bad = 0;
      if (cut) {
        // keys before the first or behind the last that some row sees have no value
        const int keep_hi = vp < 0 ? 0 : hi_b - v_key, keep_lo = lo_a - v_key;
        uint32_t keep[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) keep[i] = low_bytes(keep_hi - 4 * i) & ~low_bytes(keep_lo - 4 * i);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          vr[n] = v4u{vr[n].x & keep[0], vr[n].y & keep[1], vr[n].z & keep[2], vr[n].w & keep[3]};
          bad |= nan_bytes(vr[n].x) | nan_bytes(vr[n].y) | nan_bytes(vr[n].z) | nan_bytes(vr[n].w);
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int key = v_key + i;
          x[i] = key < hi && key >= lo && vp >= 0 ? x[i] : -INFINITY;
        }
      }
      float top = m;
#pragma unroll
      for (int i = 0; i < 16; ++i) top = fmaxf(top, x[i]);
      top = column_max(top);
      const float fade = __builtin_amdgcn_exp2f(m - top);
      m = top;
      float sum = 0.0f;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        x[i] = __builtin_amdgcn_exp2f(x[i] - top + kLift);
        sum += x[i];
      }
      l = l * fade + sum * back;
      v4u p[2];
#pragma unroll
      for (int k = 0; k < 2; ++k)
        p[k] = v4u{f16_pair(x[8 * k], x[8 * k + 1]), f16_pair(x[8 * k + 2], x[8 * k + 3]), f16_pair(x[8 * k + 4], x[8 * k + 5]),
                   f16_pair(x[8 * k + 6], x[8 * k + 7])};
#pragma unroll
      for (int n = 0; n < NT; ++n) acc[n] *= fade;
      if (__ballot(bad != 0) != 0) {
        // NaN codes that some rows see and others do not: 0 x NaN must not reach the
        // others, so they are counted by a product of their own
        v4u see[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          uint32_t w[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int key = v_key + 8 * k + 2 * i;
            w[i] = (key < hi && key >= lo ? 0x3C00u : 0u) | (key + 1 < hi && key + 1 >= lo ? 0x3C000000u : 0u);
          }
          see[k] = v4u{w[0], w[1], w[2], w[3]};
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          if (16 * n >= dim) continue;
          f32x4 hits = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
          const uint32_t w[4] = {vr[n].x, vr[n].y, vr[n].z, vr[n].w};
          uint32_t is[4], no[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t b80 = nan_bytes(w[i]);
            is[i] = (b80 >> 7) * 0x38u;                       // the code of 1
            no[i] = w[i] & ~((b80 >> 7) * 0xFFu);
          }
          hits = mma<kF16>(widen8<kF16>(is[0], is[1]), see[0], hits);
          hits = mma<kF16>(widen8<kF16>(is[2], is[3]), see[1], hits);
          acc[n] = mma<kF16>(widen8<kF16>(no[0], no[1]), p[0], acc[n]);
          acc[n] = mma<kF16>(widen8<kF16>(no[2], no[3]), p[1], acc[n]);
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[n][i] = hits[i] > 0.0f ? __builtin_nanf("") : acc[n][i];
        }
      } else {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          if (16 * n >= dim) continue;
          acc[n] = mma<kF16>(widen8<kF16>(vr[n].x, vr[n].y), p[0], acc[n]);
          acc[n] = mma<kF16>(widen8<kF16>(vr[n].z, vr[n].w), p[1], acc[n]);
        }
      }
    }
    l = column_sum(l);

    // the waves' sums together, 128 channels at a time: wave w adds up tiles w, w + 4, ..
    float* const tops = lds;                       // [wave][row] maxima, then sums
    float* const vals = lds + 2 * kWaves * kRows;  // [wave][channel / 4][row][4]
    if (g == 0) tops[wave * kRows + r] = m, tops[(kWaves + wave) * kRows + r] = l;
    const bool whole = from == 0 && to == span.count, starts = from == 0;
    const int64_t place = 2 * part + (starts ? 1 : 0);
    float* const out = a.sums + place * (kPlaceWords + (int64_t)kRows * dim);
    float all = kLow, sum = 0.0f;
#pragma unroll
    for (int n0 = 0; n0 < NT; n0 += kJoinTiles) {
      if (16 * n0 >= dim) continue;
      if (n0 > 0) __syncthreads();
#pragma unroll
      for (int n = n0; n < n0 + kJoinTiles && n < NT; ++n)
        if (16 * n < dim) *reinterpret_cast<f32x4*>(vals + ((wave * 4 * kJoinTiles + 4 * (n - n0) + g) * kRows + r) * 4) = acc[n];
      __syncthreads();
      all = tops[r];
#pragma unroll
      for (int w = 1; w < kWaves; ++w) all = fmaxf(all, tops[w * kRows + r]);
      float part_of[kWaves];
      sum = 0.0f;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        part_of[w] = __builtin_amdgcn_exp2f(tops[w * kRows + r] - all);
        sum += part_of[w] * tops[(kWaves + w) * kRows + r];
      }
      const float over = sum != 0.0f ? 1.0f / sum : 0.0f;  // a row that sees nothing is 0
#pragma unroll
      for (int n = 0; n < kJoinTiles / kWaves; ++n) {
        const int t = wave + kWaves * n, ch = 16 * (n0 + t) + 4 * g;
        if (16 * (n0 + t) >= dim) continue;
        f32x4 v = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int w = 0; w < kWaves; ++w)
          v += part_of[w] * *reinterpret_cast<const f32x4*>(vals + ((w * 4 * kJoinTiles + 4 * t + g) * kRows + r) * 4);
        if (!whole) gst<f32x4>(out + kPlaceWords + (ch / 4 * kRows + r) * 4, v);
        else if (r < rows) store4<DT>(a.out, ((q.first + tok) * a.heads + qh) * dim + ch, v * over);
      }
    }
    if (wave == 0 && g == 0) {
      if (!whole) {
        gst<float>(out + r, all), gst<float>(out + kRows + r, sum);
      } else if (a.lse != nullptr && r < rows) {
        gst<float>(a.lse + (q.first + tok) * a.heads + qh,
                   sum != 0.0f ? (all - kLift + __builtin_amdgcn_logf(sum)) * kLn2 : -INFINITY);
      }
    }
    if (tid == 0 && starts && !whole) {
      head->first = q.first, head->tile = (int)tile, head->h = h;
      // the units behind this part's, over the parts that follow
      head->parts = 1 + (int)((span.count - to + per - 1) / per);
      head->rows = rows;
    }
    __syncthreads();  // before LDS is written again
    at += to - from;
    inside += to - from;
  }
}

// Items that were cut: their parts' sums, brought to one maximum.  Work-group w looks
// after the item that part w began.
template <int DT>
__global__ __launch_bounds__(256) void k_kv_join(KvAttendArgs a) {
  const PartHead head = *reinterpret_cast<const PartHead*>(a.heads_at + 32 * (int64_t)blockIdx.x);
  if (head.rows == 0) return;
  const int dim = a.cache.dim;
  const int64_t step = kPlaceWords + (int64_t)kRows * dim;
  const float* const first = a.sums + (2 * (int64_t)blockIdx.x + 1) * step;
  const float* const rest = a.sums + 2 * (int64_t)blockIdx.x * step;  // part i at 2 i steps
  for (int i = threadIdx.x; i < dim / 4 * kRows; i += 256) {
    const int r = i % kRows, c = i / kRows;
    float top = gld<float>(first + r);
    for (int p = 1; p < head.parts; ++p) top = fmaxf(top, gld<float>(rest + 2 * p * step + r));
    float sum = 0.0f;
    f32x4 v = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    for (int p = 0; p < head.parts; ++p) {
      const float* const at = p == 0 ? first : rest + 2 * p * step;
      const float f = __builtin_amdgcn_exp2f(gld<float>(at + r) - top);
      sum += f * gld<float>(at + kRows + r);
      v += f * gld<f32x4>(at + kPlaceWords + i * 4);
    }
    if (r >= head.rows) continue;
    const int64_t row = (int64_t)head.tile * kRows + r;
    const int64_t tok = row / a.group;
    const int64_t at = (head.first + tok) * a.heads + head.h * a.group + (row - tok * a.group);
    store4<DT>(a.out, at * dim + 4 * c, v * (sum != 0.0f ? 1.0f / sum : 0.0f));
    if (a.lse != nullptr && c == 0)
      gst<float>(a.lse + at, sum != 0.0f ? (top - kLift + __builtin_amdgcn_logf(sum)) * kLn2 : -INFINITY);
  }
}

template <int DT, int NC>
void launch(const KvAttendArgs& a, hipStream_t stream) {
  const unsigned lds = 4 * (2 * kWaves * kRows + kWaves * kRows * 16 * kJoinTiles);
  hipLaunchKernelGGL((k_kv_attend<DT, NC>), dim3(a.parts), dim3(64 * kWaves), lds, stream, a);
  hipLaunchKernelGGL((k_kv_join<DT>), dim3(a.parts), dim3(256), 0, stream, a);
}
template <int DT>
void launch_of(const KvAttendArgs& a, hipStream_t stream) {
  if (a.cache.dim <= 64) launch<DT, 1>(a, stream);
  else if (a.cache.dim <= 128) launch<DT, 2>(a, stream);
  else launch<DT, 4>(a, stream);
}

constexpr unsigned kParts = 512;  // two work-groups a compute unit

// Sequences of more rows than this are k_kv_prefill's, if the call has as many.
constexpr int kFew = 64;

int64_t few_workspace(int64_t dim) { return kParts * 32 + 2 * kParts * 4 * (kPlaceWords + kRows * dim); }

}  // namespace

int64_t kv_attend_workspace(int64_t tokens, int64_t heads, int64_t kv_heads, int64_t dim, int64_t seqs, bool one_each) {
  const int64_t group = heads / kv_heads, rows = (one_each ? 1 : tokens) * group;
  int64_t need = few_workspace(dim);
  if (rows > kFew) {
    const int64_t many = kv_prefill_workspace(kv_prefill_tiles(tokens, group, seqs), seqs, kv_heads, dim);
    if (many > need) need = many;
  }
  return need;
}

hipError_t launch_kv_attend(KvAttendArgs a, int dtype, void* workspace, hipStream_t stream) {
  // no sequence has more rows than the call
  const int64_t most = a.seqs.offsets == nullptr ? a.group : a.seqs.tokens * a.group;
  a.few = most > kFew ? kFew : INT32_MAX;
  a.heads_at = static_cast<uint8_t*>(workspace);
  a.sums = reinterpret_cast<float*>(a.heads_at + kParts * 32);
  a.parts = kParts;
  a.least = kWaves;
  if (dtype == kBF16) launch_of<kBF16>(a, stream);
  else launch_of<kF16>(a, stream);
  if (most > kFew) {
    // the workspace is used again: the stream keeps the two in order
    if (hipError_t e = launch_kv_prefill(a, dtype, kv_prefill_tiles(a.seqs.tokens, a.group, a.seqs.seqs), workspace, stream)) return e;
  }
  return hipGetLastError();
}

}  // namespace lrq
