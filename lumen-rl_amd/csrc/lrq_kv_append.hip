// Writing new tokens' keys and values into the pages of an FP8 KV cache.
//
// A page's scale for a head is the least power of two that takes the largest finite
// magnitude it holds to 448 at most.  New tokens join a page behind the slots that are in
// use: where they need a larger scale than the page has, the codes that are there are
// rounded to it again; where they are the page's first, its scale starts anew.  Infinities
// and NaN become NaN codes and leave the scale alone.
//
// A page that more than one row holds is not written.  Its tokens are the other rows' as well, and
// two of them that write to it would round its codes again side by side: a row that could not
// have a page of its own (a full pool) is to lose its new tokens and no one's old ones.
//
// Bound by its bytes: a page and head of 64 tokens reads 32 KiB (bf16) and writes 16.  32 prompts
// of 33 to 1500 tokens on 8 heads of 128 (154 MB) take 35 us, 4.4 TB/s (moved pages: 5.2).  A page's
// values are read once, into registers, where both passes (the maximum, the codes) find them.
// V is turned round on its way: codes go through LDS as words of four channels, and come out
// as eight tokens of four channels, whose bytes are exchanged in registers.
#include "lrq_kv.hpp"

namespace lrq {

namespace {

// Eight values of a row, as they are.
template <int DT>
struct Raw8 {
  v4u w[DT == kF32 ? 2 : 1];
};
template <int DT>
__device__ __forceinline__ Raw8<DT> load_raw(const void* base, int64_t at) {
  Raw8<DT> r;
  if constexpr (DT == kF32) {
    r.w[0] = load_live(static_cast<const float*>(base) + at), r.w[1] = load_live(static_cast<const float*>(base) + at + 4);
  } else {
    r.w[0] = load_live(static_cast<const uint16_t*>(base) + at);
  }
  return r;
}
template <int DT>
__device__ __forceinline__ void values_of(const Raw8<DT>& r, float* v) {
  if constexpr (DT == kF32) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = u2f(r.w[i >> 2][i & 3]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t w = r.w[0][i];
      v[2 * i] = DT == kBF16 ? bf16_lo(w) : f16_to_f32(w & 0xFFFFu);
      v[2 * i + 1] = DT == kBF16 ? bf16_hi(w) : f16_to_f32(w >> 16);
    }
  }
}
// The largest magnitude so far, as bits of the values' own type (two 16-bit ones a word).
template <int DT>
__device__ __forceinline__ uint32_t amax_raw(const Raw8<DT>& r, uint32_t m) {
  if constexpr (DT == kF32) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t u = r.w[i >> 2][i & 3] & 0x7FFFFFFFu;
      m = u > m ? u : m;
    }
    return m;
  } else {
    u16x2 x = __builtin_bit_cast(u16x2, m);
#pragma unroll
    for (int i = 0; i < 4; ++i) x = amax_bf16x2(x, r.w[0][i]);
    return __builtin_bit_cast(uint32_t, x);
  }
}
// The larger of a word's two, or the word.
template <int DT>
__device__ __forceinline__ uint32_t amax_word(uint32_t m) {
  if constexpr (DT == kF32) return m;
  return (m & 0xFFFFu) > (m >> 16) ? m & 0xFFFFu : m >> 16;
}
template <int DT>
constexpr uint32_t kNotFinite = DT == kF32 ? 0x7F800000u : DT == kBF16 ? 0x7F80u : 0x7C00u;
template <int DT>
__device__ __forceinline__ uint32_t amax_f32(uint32_t m) {
  return DT == kF32 ? m : DT == kBF16 ? m << 16 : f2u(f16_to_f32(m));
}
// The same without what is not finite, for rows that have such.
template <int DT>
__device__ __forceinline__ uint32_t amax_finite(const Raw8<DT>& r, uint32_t m) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    uint32_t u;
    if constexpr (DT == kF32) u = r.w[i >> 2][i & 3] & 0x7FFFFFFFu;
    else u = (r.w[0][i >> 1] >> (16 * (i & 1))) & 0x7FFFu;
    m = u < kNotFinite<DT> && u > m ? u : m;
  }
  return m;
}

// What values are multiplied with: the reciprocal of a power of two is exact, and codes are
// the quotients', rounded once.  (A scale that is none, of a caller's own cache, is divided by.)
struct Divisor {
  float scale, by;
  bool exact;
};
__device__ __forceinline__ Divisor divisor(float scale) { return Divisor{scale, 1.0f / scale, (f2u(scale) & 0x7FFFFFu) == 0}; }
// Eight codes; what is not finite, or rounds past 448, is NaN (the instruction's own rule,
// torch's for the unscaled cast).
template <int DT>
__device__ __forceinline__ v2u codes8(const Raw8<DT>& r, const Divisor& d) {
  float v[8];
  values_of<DT>(r, v);
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = d.exact ? v[i] * d.by : v[i] / d.scale;
  return v2u{cvt_e4m3x4(v[0], v[1], v[2], v[3]), cvt_e4m3x4(v[4], v[5], v[6], v[7])};
}
// Four codes rounded to a scale 1 / ratio times theirs.
__device__ __forceinline__ uint32_t recode4(uint32_t w, float ratio) {
  const f32x2 a = e4m3x2_to_f32<false>(w), b = e4m3x2_to_f32<true>(w);
  return cvt_e4m3x4(a.x * ratio, a.y * ratio, b.x * ratio, b.y * ratio);
}
// The first `slots` of a page: K [page, dim], V [dim, page]; `threads` threads share it.
__device__ __forceinline__ void recode_k(uint8_t* kc, int slots, int dim, float ratio, int tid, int threads) {
  for (int i = tid * 4; i < slots * dim; i += threads * 4) {
    uint32_t* const p = reinterpret_cast<uint32_t*>(kc + i);
    *p = recode4(*p, ratio);
  }
}
__device__ __forceinline__ void recode_v(uint8_t* vc, int slots, int page, int dim, float ratio, int tid, int threads) {
  const int words = (slots + 3) / 4;  // the last one's bytes one by one: what is behind them is the new tokens'
  for (int i = tid; i < words * dim; i += threads) {
    const int d = i / words, w = i - d * words;
    uint8_t* const p = vc + (int64_t)d * page + 4 * w;
    const uint32_t was = *reinterpret_cast<const uint32_t*>(p), now = recode4(was, ratio);
    if (4 * w + 4 <= slots) {
      *reinterpret_cast<uint32_t*>(p) = now;
    } else {
      for (int j = 0; 4 * w + j < slots; ++j) p[j] = (uint8_t)(now >> (8 * j));
    }
  }
}

// How many rows hold a page, the same one in all lanes; it is not waited for before it is looked at.
__device__ __forceinline__ int holders(const KvCache& c, int page) { return c.refs != nullptr ? sld(c.refs + page) : 0; }

// ---------------------------------------------------------------------------
// One new token a sequence: a wave for each token and head, K in its lower half, V in the
// upper, eight channels a lane.  Its values do not wait for where they go.
// ---------------------------------------------------------------------------
template <int DT>
__global__ __launch_bounds__(256) void k_kv_append_one(KvAppendArgs a) {
  const int lane = threadIdx.x & 63, S = 1 << a.seqs.shift, dim = a.cache.dim;
  const int64_t item = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int b = (int)(item / a.cache.heads), h = (int)(item - (int64_t)b * a.cache.heads);
  if (b >= a.seqs.seqs || b >= a.seqs.tokens) return;
  const bool is_v = lane >= 32;
  const int d = (lane & 31) * 8;
  const int64_t es = DT == kF32 ? 4 : 2;
  Raw8<DT> x{};
  if (d < dim) {
    const uint8_t* const in = is_v ? static_cast<const uint8_t*>(a.v) + (b * a.v_token + h * a.v_head) * es
                                   : static_cast<const uint8_t*>(a.k) + (b * a.k_token + h * a.k_head) * es;
    x = load_raw<DT>(in, d);
  }
  const KvSeq q = kv_seq_uniform(a.seqs, b);
  if (q.len == 0) return;
  const int j = (q.len - 1) >> a.seqs.shift, slot = (q.len - 1) & (S - 1);
  const int page = kv_page_uniform(a.seqs, a.cache.pages, b, j);
  if (page < 0) return;
  float* const ks = a.cache.ks + (int64_t)page * a.cache.ks_page + h;
  float* const vs = a.cache.vs + (int64_t)page * a.cache.vs_page + h;
  const float was = is_v ? gld<float>(vs) : gld<float>(ks);
  const int held = holders(a.cache, page);
  uint32_t m = group_max<32>(amax_word<DT>(amax_raw<DT>(x, 0)));
  if (__ballot(m >= kNotFinite<DT>) != 0) m = group_max<32>(amax_finite<DT>(x, 0));
  if (held > 1) return;
  float scale = kv_scale(amax_f32<DT>(m));
  if (slot > 0) scale = fmaxf(scale, was);
  uint8_t* const kc = a.cache.k + (int64_t)page * a.cache.k_page + (int64_t)h * S * dim;
  uint8_t* const vc = a.cache.v + (int64_t)page * a.cache.v_page + (int64_t)h * S * dim;
  const float k_was = u2f(__builtin_amdgcn_readlane(f2u(was), 0)), k_now = u2f(__builtin_amdgcn_readlane(f2u(scale), 0));
  const float v_was = u2f(__builtin_amdgcn_readlane(f2u(was), 32)), v_now = u2f(__builtin_amdgcn_readlane(f2u(scale), 32));
  if (slot > 0 && k_now != k_was) recode_k(kc, slot, dim, k_was / k_now, lane, 64);
  if (slot > 0 && v_now != v_was) recode_v(vc, slot, S, dim, v_was / v_now, lane, 64);
  if ((lane & 31) == 0) gst<float>(is_v ? vs : ks, scale);
  if (d >= dim) return;
  const v2u c = codes8<DT>(x, divisor(scale));
  if (is_v) {
#pragma unroll
    for (int i = 0; i < 8; ++i) gst<uint8_t>(vc + (int64_t)(d + i) * S + slot, (uint8_t)(c[i >> 2] >> (8 * (i & 3))));
  } else {
    gst<v2u>(kc + (int64_t)slot * dim + d, c);
  }
}

// ---------------------------------------------------------------------------
// Any number: a work-group for each page that a sequence's new tokens fall into, and head.
// ---------------------------------------------------------------------------
static_assert(kOwnSearch == 256, "a thread looks at one sequence");
__device__ __forceinline__ int pages_written(const KvSeqs& s, int b) {
  const KvSeq q = kv_seq(s, b);
  const int start = q.len - q.n < 0 ? 0 : q.len - q.n;
  return q.n > 0 && q.len > start ? ((q.len - 1) >> s.shift) - (start >> s.shift) + 1 : 0;
}
// With more than kOwnSearch sequences, one work-group before: pages up to each of them, and above
// `limit` no higher.
__global__ __launch_bounds__(1024) void k_kv_append_count(KvSeqs s, int32_t* upto, int limit) {
  __shared__ int scan[16], carry;
  const int tid = threadIdx.x;
  int before = 0;
  for (int b0 = 0; b0 < s.seqs; b0 += 1024) {
    const int b = b0 + tid;
    int end = before + block_scan<1024, int>(b < s.seqs ? pages_written(s, b) : 0, scan);
    end = end > limit ? limit + 1 : end;
    if (b < s.seqs) gst<int32_t>(upto + b, end);
    if (tid == 1023) carry = end;
    __syncthreads();
    before = carry;
    __syncthreads();
  }
}
constexpr int kHeld = 4;                    // pieces of eight values of K, and of V, that a thread holds
constexpr int kSlab = kHeld * 256 * 8;      // values of a work-group: a page of 64 tokens of 128 channels
template <int DT>
__global__ __launch_bounds__(256) void k_kv_append(KvAppendArgs a) {
  __shared__ int lds_scan[4];
  __shared__ int found[2];
  __shared__ uint32_t lds_max[2][2][4];
  extern __shared__ uint8_t turn[];  // codes of V, [token][dim + 4]
  const int tid = threadIdx.x, h = blockIdx.y, S = 1 << a.seqs.shift, dim = a.cache.dim;
  // which sequence, and which of the pages that its new tokens fall into
  int b, tile;
  if (a.upto != nullptr) {
    if (blockIdx.x >= (uint32_t)sld(a.upto + a.seqs.seqs - 1)) return;
    b = kv_find(a.upto, a.seqs.seqs, blockIdx.x);
    tile = (int)blockIdx.x - (b > 0 ? sld(a.upto + b - 1) : 0);
  } else {
    if (tid == 0) found[0] = -1;
    __syncthreads();
    const int tiles = tid < a.seqs.seqs ? pages_written(a.seqs, tid) : 0;
    const int mine = (int)blockIdx.x - (block_scan<256>(tiles, lds_scan) - tiles);
    if (mine >= 0 && mine < tiles) found[0] = tid, found[1] = mine;
    __syncthreads();
    b = __builtin_amdgcn_readfirstlane(found[0]), tile = __builtin_amdgcn_readfirstlane(found[1]);
    if (b < 0) return;
  }
  const KvSeq q = kv_seq_uniform(a.seqs, b);
  // tokens whose place would be before the sequence's start have none
  const int skip = q.len - q.n < 0 ? q.n - q.len : 0, start = q.len - q.n + skip;
  const int j = (start >> a.seqs.shift) + tile;
  const int s0 = tile == 0 ? start & (S - 1) : 0;
  const int s1 = q.len - (j << a.seqs.shift) < S ? q.len - (j << a.seqs.shift) : S;
  const int page = kv_page_uniform(a.seqs, a.cache.pages, b, j);
  if (page < 0) return;
  const int n = s1 - s0, d8 = dim / 8;
  const int64_t row0 = q.first + skip + ((int64_t)(j << a.seqs.shift) + s0 - start);
  const int64_t es = DT == kF32 ? 4 : 2;
  const uint8_t* const kin = static_cast<const uint8_t*>(a.k) + (row0 * a.k_token + h * a.k_head) * es;
  const uint8_t* const vin = static_cast<const uint8_t*>(a.v) + (row0 * a.v_token + h * a.v_head) * es;
  float* const ks = a.cache.ks + (int64_t)page * a.cache.ks_page + h;
  float* const vs = a.cache.vs + (int64_t)page * a.cache.vs_page + h;
  const float k_old = gld<float>(ks), v_old = gld<float>(vs);
  const int held = holders(a.cache, page);

  // slabs of tokens whose values the threads hold: one, but for pages of more than kSlab values
  const int per = kSlab / dim, slabs = (n + per - 1) / per;
  Raw8<DT> kx[kHeld], vx[kHeld];
  auto load = [&](int slab) {
#pragma unroll
    for (int u = 0; u < kHeld; ++u) {
      const int i = u * 256 + tid, t = i / d8, d = (i - t * d8) * 8;
      kx[u] = vx[u] = Raw8<DT>{};
      if (t < per && slab * per + t < n) {
        kx[u] = load_raw<DT>(kin, (slab * per + t) * a.k_token + d);
        vx[u] = load_raw<DT>(vin, (slab * per + t) * a.v_token + d);
      }
    }
  };
  uint32_t km = 0, vm = 0;
  for (int slab = 0; slab < slabs; ++slab) {
    load(slab);
#pragma unroll
    for (int u = 0; u < kHeld; ++u) km = amax_raw<DT>(kx[u], km), vm = amax_raw<DT>(vx[u], vm);
  }
  auto over_all = [&](uint32_t k, uint32_t v, int round) {
    k = wave_max(k), v = wave_max(v);
    if ((tid & 63) == 0) lds_max[round][0][tid >> 6] = k, lds_max[round][1][tid >> 6] = v;
    __syncthreads();
    km = vm = 0;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      km = lds_max[round][0][w] > km ? lds_max[round][0][w] : km;
      vm = lds_max[round][1][w] > vm ? lds_max[round][1][w] : vm;
    }
  };
  over_all(amax_word<DT>(km), amax_word<DT>(vm), 0);
  if (km >= kNotFinite<DT> || vm >= kNotFinite<DT>) {  // the same in all threads
    uint32_t kf = 0, vf = 0;
    for (int slab = 0; slab < slabs; ++slab) {
      if (slabs > 1) load(slab);
#pragma unroll
      for (int u = 0; u < kHeld; ++u) kf = amax_finite<DT>(kx[u], kf), vf = amax_finite<DT>(vx[u], vf);
    }
    over_all(kf, vf, 1);
  }
  float k_new = kv_scale(amax_f32<DT>(km)), v_new = kv_scale(amax_f32<DT>(vm));
  if (s0 > 0) k_new = fmaxf(k_new, k_old), v_new = fmaxf(v_new, v_old);
  if (held > 1) return;  // the same in all threads
  // every thread has the old scales (the barrier above) before one writes the new
  if (tid == 0) gst<float>(ks, k_new), gst<float>(vs, v_new);

  uint8_t* const kc = a.cache.k + (int64_t)page * a.cache.k_page + (int64_t)h * S * dim;
  uint8_t* const vc = a.cache.v + (int64_t)page * a.cache.v_page + (int64_t)h * S * dim;
  if (s0 > 0 && k_new != k_old) recode_k(kc, s0, dim, k_old / k_new, tid, 256);
  if (s0 > 0 && v_new != v_old) recode_v(vc, s0, S, dim, v_old / v_new, tid, 256);
  const Divisor kd = divisor(k_new), vd = divisor(v_new);
  const int pitch = dim + 4;
  for (int slab = 0; slab < slabs; ++slab) {
    if (slabs > 1) load(slab);
    const int t0 = slab * per, m = n - t0 < per ? n - t0 : per;
    __syncthreads();  // the slab before is out of LDS
#pragma unroll
    for (int u = 0; u < kHeld; ++u) {
      const int i = u * 256 + tid, t = i / d8, d = (i - t * d8) * 8;
      if (t >= m) continue;
      gst<v2u>(kc + (int64_t)(s0 + t0 + t) * dim + d, codes8<DT>(kx[u], kd));
      const v2u c = codes8<DT>(vx[u], vd);
      uint32_t* const p = reinterpret_cast<uint32_t*>(turn + t * pitch + d);
      p[0] = c.x, p[1] = c.y;
    }
    __syncthreads();
    // eight slots of four channels a thread
    const int first = (s0 + t0) >> 3, groups = ((s0 + t0 + m - 1) >> 3) - first + 1;
    for (int i = tid; i < groups * (dim / 4); i += 256) {
      const int d = i / groups, g = i - d * groups, slot = (first + g) * 8, t = slot - s0 - t0;  // t: in the slab, may begin before it
      uint32_t w[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) w[e] = t + e >= 0 && t + e < m ? *reinterpret_cast<const uint32_t*>(turn + (t + e) * pitch + 4 * d) : 0u;
      // a 4 x 4 exchange of bytes, twice: channel c of four tokens
      uint32_t c[4][2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const uint32_t lo = __builtin_amdgcn_perm(w[4 * e + 1], w[4 * e], 0x05010400), hi = __builtin_amdgcn_perm(w[4 * e + 3], w[4 * e + 2], 0x05010400);
        const uint32_t lo2 = __builtin_amdgcn_perm(w[4 * e + 1], w[4 * e], 0x07030602), hi2 = __builtin_amdgcn_perm(w[4 * e + 3], w[4 * e + 2], 0x07030602);
        c[0][e] = __builtin_amdgcn_perm(hi, lo, 0x05040100), c[1][e] = __builtin_amdgcn_perm(hi, lo, 0x07060302);
        c[2][e] = __builtin_amdgcn_perm(hi2, lo2, 0x05040100), c[3][e] = __builtin_amdgcn_perm(hi2, lo2, 0x07060302);
      }
      uint8_t* const to = vc + (int64_t)(4 * d) * S + slot;
      if (t >= 0 && t + 8 <= m) {
#pragma unroll
        for (int r = 0; r < 4; ++r) gst<v2u>(to + r * S, v2u{c[r][0], c[r][1]});
      } else {
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (t + e >= 0 && t + e < m) gst<uint8_t>(to + r * S + e, (uint8_t)(c[r][e >> 2] >> (8 * (e & 3))));
      }
    }
  }
}

template <int DT>
void launch(const KvAppendArgs& a, hipStream_t stream) {
  if (a.seqs.offsets == nullptr) {
    const int64_t items = kv_append_tiles(a.seqs) * a.cache.heads;
    hipLaunchKernelGGL((k_kv_append_one<DT>), dim3((unsigned)((items + 3) / 4)), dim3(256), 0, stream, a);
    return;
  }
  const dim3 grid((unsigned)kv_append_tiles(a.seqs), (unsigned)a.cache.heads);
  if (a.upto != nullptr) hipLaunchKernelGGL(k_kv_append_count, dim3(1), dim3(1024), 0, stream, a.seqs, a.upto, (int)grid.x);
  const int most = kSlab / a.cache.dim < 1 << a.seqs.shift ? kSlab / a.cache.dim : 1 << a.seqs.shift;
  hipLaunchKernelGGL((k_kv_append<DT>), grid, dim3(256), most * (a.cache.dim + 4), stream, a);
}

}  // namespace

// n tokens fall into at most n pages, and at most (n - 1) / S + 2
int64_t kv_append_tiles(const KvSeqs& s) {
  const int64_t T = s.tokens, B = s.seqs;
  const int64_t tiles = s.offsets == nullptr ? B : (T >> s.shift) + 2 * B;
  return tiles < T ? tiles : T;
}
int64_t kv_append_workspace(int64_t seqs, bool one_each) { return one_each || seqs <= kOwnSearch ? 0 : (4 * seqs + 255) / 256 * 256; }
hipError_t launch_kv_append(KvAppendArgs a, int dtype, void* workspace, hipStream_t stream) {
  a.upto = kv_append_workspace(a.seqs.seqs, a.seqs.offsets == nullptr) > 0 ? static_cast<int32_t*>(workspace) : nullptr;
  if (dtype == kBF16) launch<kBF16>(a, stream);
  else if (dtype == kF16) launch<kF16>(a, stream);
  else launch<kF32>(a, stream);
  return hipGetLastError();
}

}  // namespace lrq
