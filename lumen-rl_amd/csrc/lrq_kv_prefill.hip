// Attention of many new tokens a sequence on an FP8 KV cache (lrq_kv_attend.hip has the
// formulas, and the kernel for few).  Bound by instructions: 4 prompts of 3500 to 4096 tokens, 32
// heads on 4 of 128 channels, take 560 to 575 us (850 TFLOP/s) once the clock has settled (650 us in
// the first twenty calls, 562 from the eightieth on), the matrix units busy for 39 % of the
// cycles and the other vector instructions (exponentials, widening) for 50 %.
//
// A work-group takes 128 rows (tokens times the query heads of one KV head), 32 a wave,
// and 64 keys at a time.  Both products are taken transposed, S^T = K Q^T and O^T = V^T P^T, on
// 32x32x16 instructions, so that lane l holds the column l % 32 of every result: one row
// of queries, of which l and l + 32 have half the keys each.  P goes from the first product's
// result into the second's operand within its lane.
//
// The codes are widened once for all four waves, on their way into LDS: there they lie as the
// instructions' operands, 1 KiB each, 16 bytes a lane in its order.  K, a piece of 16 channels
// of a token: channels 0-7 go to the lower half of an operand, 8-15 to the upper.  V, 16 keys
// of a channel: the lower half takes keys 0-3 and 8-11, the upper 4-7 and 12-15, the keys that
// the halves of a lane pair hold of P.  A row's place in an operand is moved by twice the piece's
// number modulo 4, so that eight lanes that write four pieces of two rows meet eight places.
// While a tile is worked on, the next one's codes are on their way into registers.
//
// In units that some rows see only a part of, NaN codes of V are taken as 0 and a flag is
// left: 0 x NaN must not reach rows that do not see it.  k_kv_join_tiles, the last launch,
// then looks for them again and writes NaN to the rows that do.
#include "lrq_kv.hpp"
#include "lrq_kv_attend.hpp"

namespace lrq {

namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int kTileRows = 128;
// Shares that the work is cut into, at most: a work-group that a compute unit holds each, two of
// them, or one with heads of more than 128 channels (32 prompts of 24 tokens on 4000 keys: 128
// channels, 512 shares 114, 256 shares 129 us; 192 channels, 192 and 166).
constexpr int kSlots = 512;
template <int NC>
constexpr int kShares = NC > 2 ? kSlots / 2 : kSlots;
// Below it a tile is not cut: its pieces' sums cost as much (42 prompts of 40 to 68 tokens on up
// to 1138 keys, 8 units 62 us, 4 units 72; one of 912 tokens on 21, 36 and 33).
constexpr int kLeastUnits = 8;
constexpr float kSlack = 5.0f;  // what a row's maximum may grow by before its sums are scaled (p stays below 2^15)

template <int DT>
__device__ __forceinline__ f32x16 mma32(v4u a, v4u b, f32x16 d) {
  if constexpr (DT == kBF16)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), d, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), d, 0, 0, 0);
}
__device__ __forceinline__ float pair_max(float v) {
  auto a = __builtin_amdgcn_permlane32_swap(f2u(v), f2u(v), false, false);
  return fmaxf(u2f(a[0]), u2f(a[1]));
}
__device__ __forceinline__ float pair_sum(float v) {
  auto a = __builtin_amdgcn_permlane32_swap(f2u(v), f2u(v), false, false);
  return u2f(a[0]) + u2f(a[1]);
}

// The rows of a tile of a sequence: how many, and the units of keys that some of them see.
struct TileSpan {
  int rows, hi, lo, first, end;  // keys [lo, hi), units [first, end)
};
__device__ __forceinline__ TileSpan tile_span(const KvSeq& q, int group, int window, int64_t tile) {
  TileSpan s;
  const int64_t row0 = tile * kTileRows, all = (int64_t)q.n * group;
  s.rows = (int)(all - row0 < kTileRows ? all - row0 : kTileRows);
  const int a = (int)(row0 / group), b = (int)((row0 + s.rows - 1) / group);
  const int base = q.len - q.n + 1;
  s.hi = base + b < 0 ? 0 : base + b;
  s.lo = window > 0 && base + a > window ? base + a - window : 0;
  s.first = s.lo / kUnit;
  s.end = (s.hi + kUnit - 1) / kUnit;
  if (s.end < s.first) s.end = s.first;
  return s;
}
__device__ __forceinline__ int64_t tiles_of(const KvAttendArgs& a, int b) {
  const KvSeq q = kv_seq(a.seqs, b);
  const int64_t rows = (int64_t)q.n * a.group;
  return rows <= a.few ? 0 : (rows + kTileRows - 1) / kTileRows;
}

// ---------------------------------------------------------------------------
// The plan, by one work-group: all tiles of the sequences that have many rows, those with
// more units than a work-group's share cut into pieces, the longest pieces first.
// ---------------------------------------------------------------------------
constexpr int kBuckets = 1024;  // of pieces' lengths; the last one takes all longer ones
__global__ __launch_bounds__(1024) void k_kv_tiles(KvAttendArgs a) {
  __shared__ int64_t scan[16];
  __shared__ int64_t carry;
  __shared__ uint32_t scan32[16];
  __shared__ int ends[1024];  // upto, where it is no longer than that
  __shared__ uint32_t bucket[kBuckets];
  __shared__ uint32_t counts[2];  // places of pieces, and tiles that were cut
  const KvTiles& p = a.tiles;
  const int tid = threadIdx.x, seqs = a.seqs.seqs;
  // upto[b]: tiles of the sequences 0 .. b
  if (tid == 0) carry = 0, counts[0] = counts[1] = 0, gst<int32_t>(p.count + 2, 0);
  bucket[tid] = 0;
  __syncthreads();
  for (int b0 = 0; b0 < seqs; b0 += 1024) {
    const int64_t base = carry;
    const int64_t upto = base + block_scan<1024, int64_t>(b0 + tid < seqs ? tiles_of(a, b0 + tid) : 0, scan);
    // offsets that go back would make rows of several sequences', and more tiles than there is room for
    const int end = upto < p.most ? (int)upto : p.most;
    if (b0 + tid < seqs) gst<int32_t>(p.upto + b0 + tid, end);
    ends[tid] = end;
    if (tid == 1023) carry = upto;
    __syncthreads();
  }
  const int tiles = carry < p.most ? (int)carry : p.most;
  __syncthreads();
  auto end_of = [&](int b) { return seqs <= 1024 ? ends[b] : gld<int32_t>(p.upto + b); };
  auto find = [&](int i, int& tile) {  // the sequence of tile i
    int lo = 0, hi = seqs - 1;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (end_of(mid) > i) hi = mid;
      else lo = mid + 1;
    }
    tile = i - (lo > 0 ? end_of(lo - 1) : 0);
    return lo;
  };
  // a thread's first tile is looked at once, others (in calls of more tiles than threads) three times
  int my_tile = 0;
  const int my_b = tid < tiles ? find(tid, my_tile) : 0;
  TileSpan my_span{};
  if (tid < tiles) my_span = tile_span(kv_seq(a.seqs, my_b), a.group, a.window, my_tile);
  auto look = [&](int i, int& tile, TileSpan& span) {
    if (i == tid) {
      tile = my_tile, span = my_span;
      return my_b;
    }
    const int b = find(i, tile);
    span = tile_span(kv_seq(a.seqs, b), a.group, a.window, tile);
    return b;
  };
  int64_t units = 0;
  for (int i = tid; i < tiles; i += 1024) {
    int tile;
    TileSpan s;
    look(i, tile, s);
    units += s.end - s.first;
  }
  const int64_t sum = block_scan<1024, int64_t>(units, scan);
  if (tid == 1023) carry = sum;
  __syncthreads();
  int64_t most = (carry * a.cache.heads + p.shares - 1) / p.shares;
  if (most < kLeastUnits) most = kLeastUnits;
  auto cuts_of = [&](int n) { return n <= most ? 1 : (int)((n + most - 1) / most); };
  auto bucket_of = [&](int n) { return n >= kBuckets ? 0 : kBuckets - 1 - n; };
  for (int i = tid; i < tiles; i += 1024) {
    int tile;
    TileSpan s;
    look(i, tile, s);
    const int n = s.end - s.first, cuts = cuts_of(n);
    atomicAdd(&bucket[bucket_of(n / cuts)], (uint32_t)cuts);
  }
  __syncthreads();
  const uint32_t mine = bucket[tid];
  const uint32_t before = block_scan<1024, uint32_t>(mine, scan32) - mine;
  bucket[tid] = before;
  if (tid == 1023) gst<int32_t>(p.count, (int32_t)(before + mine));
  __syncthreads();
  for (int i = tid; i < tiles; i += 1024) {
    int tile;
    TileSpan s;
    const int b = look(i, tile, s);
    const int n = s.end - s.first, cuts = cuts_of(n);
    const uint32_t at = atomicAdd(&bucket[bucket_of(n / cuts)], (uint32_t)cuts);
    int slot = -1;
    if (cuts > 1) {
      slot = (int)atomicAdd(&counts[0], (uint32_t)cuts);
      const uint32_t cut = atomicAdd(&counts[1], 1u);
      gst<v4i>(p.cut + cut, v4i{b, tile, slot, cuts});
    }
    for (int j = 0; j < cuts; ++j) {
      const int u0 = s.first + (int)((int64_t)n * j / cuts), u1 = s.first + (int)((int64_t)n * (j + 1) / cuts);
      gst<v4i>(p.piece + 2 * (at + j), v4i{b, tile, u0, u1});
      gst<v4i>(p.piece + 2 * (at + j) + 1, v4i{slot < 0 ? -1 : slot + j, 0, 0, 0});
    }
  }
  __syncthreads();
  if (tid == 0) gst<int32_t>(p.count + 1, (int32_t)counts[1]);
}

// Heads of more than 64 (NC - 1) channels, 64 NC at most: those that are not there are zeros.
// FAST: pages of 64 keys or more, so that a unit is of one page (4 prompts of up to 4000 tokens
// 591 us; 626 without it).
template <int DT, int NC, bool FAST>
__global__ __launch_bounds__(256, NC > 2 ? 1 : 2) void k_kv_prefill(KvAttendArgs a) {
  constexpr int KS = 4 * NC, VT = 2 * NC;       // steps of 16 channels, tiles of 32
  constexpr int kStage = (2 * KS + 4 * VT) * 64;  // 16-byte places of a tile: K's operands, then V's
  __shared__ __attribute__((aligned(16))) v4u stage[2][kStage];
  __shared__ __attribute__((aligned(16))) float page_of[2][12];  // per 16 keys: factor, exponent, its inverse
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r = lane & 31, half = lane >> 5;
  const int heads = a.cache.heads, dim = a.cache.dim, shift = a.seqs.shift, S = 1 << shift, group = a.group;
  const int count = gld<int32_t>(a.tiles.count);
  const int h = blockIdx.x % heads, idx = blockIdx.x / heads;
  if (idx >= count) return;
  const v4i piece = gld<v4i>(a.tiles.piece + 2 * idx);
  const int slot = gld<int32_t>(a.tiles.piece + 2 * idx + 1);
  const int b = __builtin_amdgcn_readfirstlane(piece.x), tile = __builtin_amdgcn_readfirstlane(piece.y);
  const int u0 = __builtin_amdgcn_readfirstlane(piece.z), u1 = __builtin_amdgcn_readfirstlane(piece.w);
  const KvSeq q = kv_seq(a.seqs, b);
  const TileSpan span = tile_span(q, group, a.window, tile);

  // this lane's row, and the keys [lo, hi) that it sees
  const int mine = wave * 32 + r;
  const int64_t row = (int64_t)tile * kTileRows + (mine < span.rows ? mine : 0);
  const int tok = (int)(row / group), qh = h * group + (int)(row - (int64_t)tok * group);
  const int pos1 = q.len - q.n + tok + 1;
  const int hi = pos1 < 0 ? 0 : pos1, lo = a.window > 0 && pos1 > a.window ? pos1 - a.window : 0;
  // what the first and the last row of the tile see
  const int first_hi = q.len - q.n + (int)((int64_t)tile * kTileRows / group) + 1;
  const int last_hi = q.len - q.n + (int)(((int64_t)tile * kTileRows + span.rows - 1) / group) + 1;
  const int last_lo = a.window > 0 && last_hi > a.window ? last_hi - a.window : 0;

  v4u qf[KS];
  {
    const uint16_t* const src = static_cast<const uint16_t*>(a.q) + (q.first + tok) * a.q_token + qh * a.q_head;
    const uint32_t flip = a.scale < 0.0f ? 0x80008000u : 0u;  // the keys' factor is to be positive
#pragma unroll
    for (int k = 0; k < KS; ++k) {
      qf[k] = v4u{0, 0, 0, 0};
      if (16 * k < dim && mine < span.rows) {
        const v4u w = load_live(src + 16 * k + 8 * half);
        qf[k] = v4u{w.x ^ flip, w.y ^ flip, w.z ^ flip, w.w ^ flip};
      }
    }
  }
  const float scale = __builtin_fabsf(a.scale);

  // what this thread brings of a tile: of K token tid / 4, of V keys 16 (tid % 4) .., a piece of each 64 channels
  const int k_tok = tid >> 2, c4 = tid & 3;
  v4u kr[NC], vr[NC];
  int kp = -1, vp = -1;  // the pages of the next load
  auto look_up = [&](int u) {
    if constexpr (FAST) {
      kp = vp = kv_page_uniform(a.seqs, a.cache.pages, b, (u * kUnit) >> shift);
    } else {  // 16 keys are of one page
      int p[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) p[i] = kv_page_uniform(a.seqs, a.cache.pages, b, (u * kUnit + 16 * i) >> shift);
      const int g = k_tok >> 4;
      kp = (g & 2) ? ((g & 1) ? p[3] : p[2]) : ((g & 1) ? p[1] : p[0]);
      vp = (c4 & 2) ? ((c4 & 1) ? p[3] : p[2]) : ((c4 & 1) ? p[1] : p[0]);
    }
  };
  bool k_ok = false, v_ok = false;
  int vp_now = -1;
  float ks = 0.0f, vs = 0.0f;  // of the keys 16 (tid % 4) ..; FAST: of the unit
  auto load = [&](int u) {
    const int key = u * kUnit + k_tok, vkey = u * kUnit + 16 * c4;
    k_ok = kp >= 0, v_ok = vp >= 0, vp_now = vp;
    const int64_t kpage = k_ok ? kp : 0, vpage = v_ok ? vp : 0;
    const uint8_t* const kb = a.cache.k + kpage * a.cache.k_page + ((int64_t)h * S + (key & (S - 1))) * dim + 16 * c4;
    const uint8_t* const vb = a.cache.v + vpage * a.cache.v_page + ((int64_t)h * dim + k_tok) * S + (vkey & (S - 1));
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      if (i == NC - 1) kr[i] = vr[i] = v4u{0, 0, 0, 0};
      if (i < NC - 1 || 64 * i + 16 * c4 < dim) kr[i] = gld<v4u>(kb + 64 * i);
      if (i < NC - 1 || 64 * i + k_tok < dim) vr[i] = gld<v4u>(vb + (int64_t)64 * i * S);
    }
    if constexpr (FAST) {
      ks = sld(a.cache.ks + vpage * a.cache.ks_page + h), vs = sld(a.cache.vs + vpage * a.cache.vs_page + h);
    } else if (tid < 4) {
      ks = gld<float>(a.cache.ks + vpage * a.cache.ks_page + h), vs = gld<float>(a.cache.vs + vpage * a.cache.vs_page + h);
    }
  };
  // units that some row sees a part of
  auto cut_at = [&](int u) { return u * kUnit + kUnit > first_hi || u * kUnit < last_lo; };
  // What was loaded of unit u: nothing where there is no page; where rows see a part of it,
  // keys that none sees are 0, and so are NaN codes of V.
  auto clean = [&](int u) {
    uint32_t keep[4], bad = 0;
    const int v_key = u * kUnit + 16 * c4;
#pragma unroll
    for (int i = 0; i < 4; ++i) keep[i] = v_ok ? low_bytes(span.hi - v_key - 4 * i) & ~low_bytes(span.lo - v_key - 4 * i) : 0u;
    const bool cut = cut_at(u);
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      kr[i] = k_ok ? kr[i] : v4u{0, 0, 0, 0};
      const v4u w = v4u{vr[i].x & keep[0], vr[i].y & keep[1], vr[i].z & keep[2], vr[i].w & keep[3]};
      const v4u nan = v4u{nan_bytes(w.x), nan_bytes(w.y), nan_bytes(w.z), nan_bytes(w.w)} >> 7;
      if (cut) bad |= nan.x | nan.y | nan.z | nan.w;
      vr[i] = cut ? w & ~(nan * 0xFF) : w;
    }
    if (bad != 0) gst<int32_t>(a.tiles.count + 2, 1);
  };
  auto is_odd = [&](int u) { return cut_at(u) || (FAST ? vp_now < 0 : __ballot(!k_ok || !v_ok) != 0); };
  auto put_k = [&](int at, int i) {  // a piece's operands into stage `at`
    v4u* const to = stage[at] + ((k_tok >> 5) * KS + 4 * i + c4) * 64 + ((k_tok & 31) ^ (2 * c4));
    to[0] = widen8<DT>(kr[i].x, kr[i].y);
    to[32] = widen8<DT>(kr[i].z, kr[i].w);
  };
  auto put_v = [&](int at, int i) {
    const int d = 64 * i + k_tok;
    v4u* const to = stage[at] + 2 * KS * 64 + ((d >> 5) * 4 + c4) * 64 + ((d & 31) ^ (2 * c4));
    const v4u x = widen8<kF16>(vr[i].x, vr[i].y), y = widen8<kF16>(vr[i].z, vr[i].w);  // keys 0-7, 8-15
    to[0] = v4u{x.x, x.y, y.x, y.y};
    to[32] = v4u{x.z, x.w, y.z, y.w};
  };
  auto put_page = [&](int at) {
    if (FAST ? tid == 0 : tid < 4) {
      const float ev = __builtin_amdgcn_logf(__builtin_amdgcn_fmed3f(vs, 0x1p-48f, 0x1p48f));
      page_of[at][tid] = fmaxf(ks * scale, 0x1p-120f);  // above 0, so that no key stays no key
      page_of[at][4 + tid] = v_ok ? ev : -INFINITY;
      page_of[at][8 + tid] = v_ok ? __builtin_amdgcn_exp2f(-ev) : 0.0f;
    }
  };

  float m = kLow, l = 0.0f;
  f32x16 acc[VT];
#pragma unroll
  for (int n = 0; n < VT; ++n) acc[n] = f32x16{};
  // Unit u's operands are in LDS, the next one's codes on their way into registers.  They are
  // widened and put there while the matrix units take the scores; then the loads of the one
  // after go out.  The second product's instructions run while the next exponentials are taken.
  const int last = u1 - 1;
  if (u0 < u1) {
    look_up(u0);
    load(u0);
    look_up(u0 < last ? u0 + 1 : last);
    clean(u0);
#pragma unroll
    for (int i = 0; i < NC; ++i) put_k(0, i), put_v(0, i);
    put_page(0);
    load(u0 < last ? u0 + 1 : last);
  }
  __syncthreads();
  for (int u = u0; u < u1; ++u) {
    const int at = (u - u0) & 1;
    const int coming = u + 1 < last ? u + 1 : last;  // (once more the last one, into the stage that no one reads)
    look_up(u + 2 < last ? u + 2 : last);
    if (is_odd(coming)) clean(coming);
    const v4u* const kst = stage[at];
    const v4u* const vst = stage[at] + 2 * KS * 64;
    f32x16 s[2] = {f32x16{}, f32x16{}};
#pragma unroll
    for (int k = 0; k < KS; ++k) {
#pragma unroll
      for (int t = 0; t < 2; ++t)
        s[t] = mma32<DT>(kst[(t * KS + k) * 64 + (lane ^ (2 * (k & 3)))], qf[k], s[t]);
      if (k % 4 == 1) put_k(at ^ 1, k / 4);
      if (k % 4 == 3) put_v(at ^ 1, k / 4);
    }
    put_page(at ^ 1);
    load(u + 2 < last ? u + 2 : last);
    // the scores' factor, V's exponent and its inverse: of every 16 keys, or of them all
    constexpr int E = FAST ? 1 : 4;
    float factor[E], ev[E], back[E];
    bool gone = false;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      factor[e] = page_of[at][e], ev[e] = page_of[at][4 + e], back[e] = page_of[at][8 + e];
      gone |= ev[e] == -INFINITY;
    }
    if (__builtin_amdgcn_readfirstlane(cut_at(u) || gone)) {
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int key = u * kUnit + 32 * t + 8 * (i >> 2) + 4 * half + (i & 3);
          s[t][i] = key < hi && key >= lo && ev[(2 * t + (i >> 3)) % E] != -INFINITY ? s[t][i] : -INFINITY;
        }
    }
    float top = m;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      constexpr int N = 32 / E;
      float x = s[e >> 1][8 * (e & 1)];
#pragma unroll
      for (int i = 1; i < N; ++i) x = fmaxf(x, s[(e >> 1) + (i >> 4)][(8 * (e & 1) + i) & 15]);
      // no key of them: 0 x -inf and -inf + -inf are kept out of it
      top = x == -INFINITY ? top : fmaxf(top, __builtin_fmaf(x, factor[e], ev[e]));
    }
    top = pair_max(top);
    if (__ballot(top > m + kSlack) != 0) {
      const float fade = __builtin_amdgcn_exp2f(m - top);
      m = top;
      l *= fade;
#pragma unroll
      for (int n = 0; n < VT; ++n)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[n][i] *= fade;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float shift_by = ev[e % E] - m + kLift;
      float x[8], sum = 0.0f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        x[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[e >> 1][8 * (e & 1) + i], factor[e % E], shift_by));
        sum += x[i];
      }
      l = __builtin_fmaf(sum, back[e % E], l);
      const v4u p = v4u{f16_pair(x[0], x[1]), f16_pair(x[2], x[3]), f16_pair(x[4], x[5]), f16_pair(x[6], x[7])};
#pragma unroll
      for (int n = 0; n < VT; ++n)
        acc[n] = mma32<kF16>(vst[(n * 4 + e) * 64 + (lane ^ (2 * e))], p, acc[n]);
      __builtin_amdgcn_sched_barrier(0);
    }
    __syncthreads();
  }
  l = pair_sum(l);

  if (slot < 0) {
    if (mine >= span.rows) return;
    const float over = l != 0.0f ? 1.0f / l : 0.0f;  // a row that sees nothing is 0
    const int64_t at = (q.first + tok) * a.heads + qh;
#pragma unroll
    for (int n = 0; n < VT; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int d = 32 * n + 8 * i + 4 * half;
        if (d < dim) store4<DT>(a.out, at * dim + d, f32x4{acc[n][4 * i], acc[n][4 * i + 1], acc[n][4 * i + 2], acc[n][4 * i + 3]} * over);
      }
    if (a.lse != nullptr && half == 0) gst<float>(a.lse + at, l != 0.0f ? (m - kLift + __builtin_amdgcn_logf(l)) * kLn2 : -INFINITY);
    return;
  }
  float* const out = a.tiles.sums + ((int64_t)slot * heads + h) * (kTileRows * (2 + (int64_t)dim));
  if (half == 0) gst<float>(out + mine, m), gst<float>(out + kTileRows + mine, l);
#pragma unroll
  for (int n = 0; n < VT; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int d = 32 * n + 8 * i + 4 * half;
      if (d < dim)
        gst<f32x4>(out + 2 * kTileRows + ((int64_t)(d / 4) * kTileRows + mine) * 4,
                   f32x4{acc[n][4 * i], acc[n][4 * i + 1], acc[n][4 * i + 2], acc[n][4 * i + 3]});
    }
}

// NaN for the channels of rows of a tile that see a NaN code of V in a unit that others of
// the tile see only a part of.  Work-group y of `of` has every of-th eight channels.
template <int DT>
__device__ void spread_nan(const KvAttendArgs& a, int b, int tile, int h, int y, int of) {
  const int dim = a.cache.dim, S = 1 << a.seqs.shift, group = a.group;
  const KvSeq q = kv_seq(a.seqs, b);
  const TileSpan span = tile_span(q, group, a.window, tile);
  const int64_t row0 = (int64_t)tile * kTileRows;
  const int base = q.len - q.n + 1, first_hi = base + (int)(row0 / group), last_hi = base + (int)((row0 + span.rows - 1) / group);
  const int last_lo = a.window > 0 && last_hi > a.window ? last_hi - a.window : 0;
  for (int u = span.first; u < span.end; ++u) {
    if (u * kUnit + kUnit <= first_hi && u * kUnit >= last_lo) continue;
    for (int i = threadIdx.x; i < kUnit * dim; i += 256) {
      const int key = u * kUnit + i % kUnit, d = i / kUnit;
      if (key < span.lo || key >= span.hi || d / 8 % of != y) continue;
      const int page = kv_page(a.seqs, a.cache.pages, b, key >> a.seqs.shift);
      if (page < 0) continue;
      const uint8_t code = gld<uint8_t>(a.cache.v + (int64_t)page * a.cache.v_page + ((int64_t)h * dim + d) * S + (key & (S - 1)));
      if ((code & 0x7F) != 0x7F) continue;
      for (int r = 0; r < span.rows; ++r) {
        const int64_t tok = (row0 + r) / group;
        const int hi = base + (int)tok;
        if (key >= hi || (a.window > 0 && key < hi - a.window)) continue;
        const int64_t at = (q.first + tok) * a.heads + h * group + (row0 + r - tok * group);
        gst<uint16_t>(static_cast<uint16_t*>(a.out) + at * dim + d, DT == kBF16 ? 0x7FC0 : 0x7E00);
      }
    }
  }
}

// Last: tiles that were cut get their pieces' sums, brought to one maximum; and if there were
// NaN codes that k_kv_prefill took as 0, every tile gets those.  blockIdx.y has every fourth
// eight channels of a cut tile, in both.
template <int DT>
__global__ __launch_bounds__(256) void k_kv_join_tiles(KvAttendArgs a) {
  const int heads = a.cache.heads, dim = a.cache.dim, step_all = gridDim.x / heads;
  const int h = blockIdx.x % heads, idx = blockIdx.x / heads;
  const v4i count = gld<v4i>(a.tiles.count);  // pieces, cut tiles, NaN codes
  if (idx < count.y) {  // (the grid has a work-group for each)
    const v4i cut = gld<v4i>(a.tiles.cut + idx);
    const int b = cut.x, tile = cut.y, slot = cut.z, pieces = cut.w;
    const KvSeq q = kv_seq(a.seqs, b);
    const int64_t all = (int64_t)q.n * a.group, row0 = (int64_t)tile * kTileRows;
    const int64_t step = (int64_t)heads * kTileRows * (2 + dim);
    const float* const first = a.tiles.sums + ((int64_t)slot * heads + h) * (kTileRows * (2 + (int64_t)dim));
    const int r = threadIdx.x % kTileRows;
    if (row0 + r < all) {
      float top = gld<float>(first + r);
      for (int p = 1; p < pieces; ++p) top = fmaxf(top, gld<float>(first + p * step + r));
      float sum = 0.0f;
      for (int p = 0; p < pieces; ++p) sum += __builtin_amdgcn_exp2f(gld<float>(first + p * step + r) - top) * gld<float>(first + p * step + kTileRows + r);
      const float over = sum != 0.0f ? 1.0f / sum : 0.0f;
      const int64_t tok = (row0 + r) / a.group;
      const int64_t at = (q.first + tok) * a.heads + h * a.group + (row0 + r - tok * a.group);
      for (int c = blockIdx.y * 2 + threadIdx.x / kTileRows; c < dim / 4; c += 2 * gridDim.y) {
        f32x4 v = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        for (int p = 0; p < pieces; ++p)
          v += __builtin_amdgcn_exp2f(gld<float>(first + p * step + r) - top) * gld<f32x4>(first + p * step + 2 * kTileRows + ((int64_t)c * kTileRows + r) * 4);
        store4<DT>(a.out, at * dim + 4 * c, v * over);
        if (a.lse != nullptr && c == 0) gst<float>(a.lse + at, sum != 0.0f ? (top - kLift + __builtin_amdgcn_logf(sum)) * kLn2 : -INFINITY);
      }
    }
    if (count.z != 0) {
      __syncthreads();  // the results above are written before
      spread_nan<DT>(a, b, tile, h, blockIdx.y, gridDim.y);
    }
  }
  if (count.z == 0 || blockIdx.y != 0) return;
  for (int i = idx; i < count.x; i += step_all) {
    const v4i piece = gld<v4i>(a.tiles.piece + 2 * i);
    if (gld<int32_t>(a.tiles.piece + 2 * i + 1) < 0) spread_nan<DT>(a, piece.x, piece.y, h, 0, 1);
  }
}

template <int DT, int NC>
void launch(KvAttendArgs a, int64_t tiles, hipStream_t stream) {
  const int64_t heads = a.cache.heads;
  a.tiles.shares = kShares<NC>;
  hipLaunchKernelGGL(k_kv_tiles, dim3(1), dim3(1024), 0, stream, a);
  const dim3 grid((unsigned)((tiles + 2 * kSlots / heads + 1) * heads));
  if (a.seqs.shift >= 6) hipLaunchKernelGGL((k_kv_prefill<DT, NC, true>), grid, dim3(256), 0, stream, a);
  else hipLaunchKernelGGL((k_kv_prefill<DT, NC, false>), grid, dim3(256), 0, stream, a);
  hipLaunchKernelGGL((k_kv_join_tiles<DT>), dim3((unsigned)((kSlots / heads + 1) * heads), 4), dim3(256), 0, stream, a);
}
template <int DT>
void launch_of(const KvAttendArgs& a, int64_t tiles, hipStream_t stream) {
  if (a.cache.dim <= 64) launch<DT, 1>(a, tiles, stream);
  else if (a.cache.dim <= 128) launch<DT, 2>(a, tiles, stream);
  else if (a.cache.dim <= 192) launch<DT, 3>(a, tiles, stream);
  else launch<DT, 4>(a, tiles, stream);
}

int64_t pad256(int64_t n) { return (n + 255) / 256 * 256; }

}  // namespace

// Tiles that the call's rows can come to; one that is cut is at most twice its share in pieces.
int64_t kv_prefill_tiles(int64_t tokens, int64_t group, int64_t seqs) {
  return tokens * group / kTileRows + (seqs < tokens ? seqs : tokens);
}
static int64_t most_pieces(int64_t tiles, int64_t heads) { return tiles + 2 * kSlots / heads + 1; }
int64_t kv_prefill_workspace(int64_t tiles, int64_t seqs, int64_t heads, int64_t dim) {
  return 256 + pad256(4 * seqs) + pad256(32 * most_pieces(tiles, heads)) + pad256(16 * (kSlots / heads + 1)) +
         4 * (2 * kSlots / heads + 1) * heads * kTileRows * (2 + dim);
}
hipError_t launch_kv_prefill(KvAttendArgs a, int dtype, int64_t tiles, void* workspace, hipStream_t stream) {
  uint8_t* w = static_cast<uint8_t*>(workspace);
  const int64_t heads = a.cache.heads;
  a.tiles.count = reinterpret_cast<int32_t*>(w), w += 256;
  a.tiles.upto = reinterpret_cast<int32_t*>(w), w += pad256(4 * (int64_t)a.seqs.seqs);
  a.tiles.piece = reinterpret_cast<v4i*>(w), w += pad256(32 * most_pieces(tiles, heads));
  a.tiles.cut = reinterpret_cast<v4i*>(w), w += pad256(16 * (kSlots / heads + 1));
  a.tiles.sums = reinterpret_cast<float*>(w);
  a.tiles.most = (int)tiles;
  if (dtype == kBF16) launch_of<kBF16>(a, tiles, stream);
  else launch_of<kF16>(a, tiles, stream);
  return hipGetLastError();
}

}  // namespace lrq
