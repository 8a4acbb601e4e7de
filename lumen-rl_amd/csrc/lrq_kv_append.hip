// Writing new tokens' keys and values into the pages of an FP8 KV cache.
//
// A page's scale for a head is the least power of two that takes the largest finite
// magnitude it holds to 448 at most.  New tokens join a page behind the slots that are in
// use: where they need a larger scale than the page has, the codes that are there are
// rounded to it again; where they are the page's first, its scale starts anew.  Infinities
// and NaN become NaN codes and leave the scale alone.
#include "lrq_kv.hpp"

namespace lrq {

namespace {

constexpr int kSlab = 64;  // tokens whose V codes are turned round in LDS at a time

// Eight values of a row, zeros past n of them.
template <int DT>
__device__ __forceinline__ void load8(const void* base, int64_t at, float* v) {
  if constexpr (DT == kF32) {
    const v4u a = load_live(static_cast<const float*>(base) + at), b = load_live(static_cast<const float*>(base) + at + 4);
    const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = u2f(w[i]);
  } else {
    const v4u a = load_live(static_cast<const uint16_t*>(base) + at);
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = DT == kBF16 ? bf16_lo(w[i]) : f16_to_f32(w[i] & 0xFFFFu);
      v[2 * i + 1] = DT == kBF16 ? bf16_hi(w[i]) : f16_to_f32(w[i] >> 16);
    }
  }
}

__device__ __forceinline__ uint32_t finite_amax(const float* v, uint32_t m) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t u = f2u(v[i]) & 0x7FFFFFFFu;
    m = u < 0x7F800000u && u > m ? u : m;
  }
  return m;
}

// Four values in a scale's codes; what is not finite, or rounds past 448, is NaN (the
// instruction's own rule, torch's for the unscaled cast).
__device__ __forceinline__ uint32_t codes4(const float* v, float s) {
  return cvt_e4m3x4(v[0] / s, v[1] / s, v[2] / s, v[3] / s);
}
// Four codes of scale `from` rounded to scale `to`.
__device__ __forceinline__ uint32_t recode4(uint32_t w, float ratio) {
  const f32x2 a = e4m3x2_to_f32<false>(w), b = e4m3x2_to_f32<true>(w);
  return cvt_e4m3x4(a.x * ratio, a.y * ratio, b.x * ratio, b.y * ratio);
}

template <int DT>
__global__ __launch_bounds__(256) void k_kv_append(KvAppendArgs a) {
  __shared__ int lds_scan[4];
  __shared__ int found[2];
  __shared__ uint32_t lds_max[2][4];
  extern __shared__ uint8_t turn[];  // [kSlab][dim + 4]
  const int tid = threadIdx.x, h = blockIdx.y, S = 1 << a.seqs.shift, dim = a.cache.dim;
  // which sequence, and which of the pages that its new tokens fall into
  int b = (int)blockIdx.x, tile = 0;
  if (a.seqs.offsets != nullptr) {
    if (tid == 0) found[0] = -1;
    __syncthreads();
    int64_t before = 0;
    for (int b0 = 0; b0 < a.seqs.seqs; b0 += 256) {
      int tiles = 0;
      if (b0 + tid < a.seqs.seqs) {
        const KvSeq q = kv_seq(a.seqs, b0 + tid);
        const int start = q.len - q.n < 0 ? 0 : q.len - q.n;
        if (q.n > 0 && q.len > start) tiles = ((q.len - 1) >> a.seqs.shift) - (start >> a.seqs.shift) + 1;
      }
      const int upto = block_scan<256>(tiles, lds_scan);
      const int64_t mine = (int64_t)blockIdx.x - before - (upto - tiles);
      if (mine >= 0 && mine < tiles) found[0] = b0 + tid, found[1] = (int)mine;
      if (tid == 255) lds_scan[0] = upto;
      __syncthreads();
      before += lds_scan[0];
      const bool done = found[0] >= 0 || before > (int64_t)blockIdx.x;
      __syncthreads();
      if (done) break;
    }
    b = found[0], tile = found[1];
    if (b < 0) return;
  }
  const KvSeq q = kv_seq(a.seqs, b);
  // tokens whose place would be before the sequence's start have none
  const int skip = q.len - q.n < 0 ? q.n - q.len : 0, start = q.len - q.n + skip;
  if (q.n == 0 || q.len <= start) return;
  const int j = (start >> a.seqs.shift) + tile;
  const int s0 = tile == 0 ? start & (S - 1) : 0;
  const int s1 = q.len - (j << a.seqs.shift) < S ? q.len - (j << a.seqs.shift) : S;
  const int page = kv_page(a.seqs, a.cache.pages, b, j);
  if (page < 0) return;
  const int n = s1 - s0, d8 = dim / 8;
  const int64_t row0 = q.first + skip + ((int64_t)(j << a.seqs.shift) + s0 - start);
  const int64_t es = DT == kF32 ? 4 : 2;
  const uint8_t* const kin = static_cast<const uint8_t*>(a.k) + (row0 * a.k_token + h * a.k_head) * es;
  const uint8_t* const vin = static_cast<const uint8_t*>(a.v) + (row0 * a.v_token + h * a.v_head) * es;

  uint32_t km = 0, vm = 0;
  for (int i = tid; i < n * d8; i += 256) {
    const int t = i / d8, d = (i - t * d8) * 8;
    float x[8];
    load8<DT>(kin, t * a.k_token + d, x);
    km = finite_amax(x, km);
    load8<DT>(vin, t * a.v_token + d, x);
    vm = finite_amax(x, vm);
  }
  km = wave_max(km), vm = wave_max(vm);
  if ((tid & 63) == 0) lds_max[0][tid >> 6] = km, lds_max[1][tid >> 6] = vm;
  float* const ks = a.cache.ks + (int64_t)page * a.cache.ks_page + h;
  float* const vs = a.cache.vs + (int64_t)page * a.cache.vs_page + h;
  const float k_old = *ks, v_old = *vs;
  __syncthreads();
  km = vm = 0;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    km = lds_max[0][w] > km ? lds_max[0][w] : km;
    vm = lds_max[1][w] > vm ? lds_max[1][w] : vm;
  }
  float k_new = kv_scale(km), v_new = kv_scale(vm);
  if (s0 > 0) k_new = fmaxf(k_new, k_old), v_new = fmaxf(v_new, v_old);
  // every thread has read the old scales (the barrier above) before one writes the new
  if (tid == 0) *ks = k_new, *vs = v_new;

  uint8_t* const kc = a.cache.k + (int64_t)page * a.cache.k_page + (int64_t)h * S * dim;
  uint8_t* const vc = a.cache.v + (int64_t)page * a.cache.v_page + (int64_t)h * S * dim;
  if (s0 > 0 && k_new != k_old) {
    const float ratio = k_old / k_new;
    for (int i = tid * 4; i < s0 * dim; i += 1024) {
      uint32_t* const p = reinterpret_cast<uint32_t*>(kc + i);
      *p = recode4(*p, ratio);
    }
  }
  if (s0 > 0 && v_new != v_old) {
    const float ratio = v_old / v_new;
    for (int i = tid; i < s0 * dim; i += 256) {
      uint8_t* const p = vc + (i / s0) * S + i % s0;
      *p = (uint8_t)recode4(*p, ratio);
    }
  }
  for (int i = tid; i < n * d8; i += 256) {
    const int t = i / d8, d = (i - t * d8) * 8;
    float x[8];
    load8<DT>(kin, t * a.k_token + d, x);
    *reinterpret_cast<v2u*>(kc + (int64_t)(s0 + t) * dim + d) = v2u{codes4(x, k_new), codes4(x + 4, k_new)};
  }
  const int pitch = dim + 4;
  for (int t0 = 0; t0 < n; t0 += kSlab) {
    const int m = n - t0 < kSlab ? n - t0 : kSlab;
    __syncthreads();
    for (int i = tid; i < m * d8; i += 256) {
      const int t = i / d8, d = (i - t * d8) * 8;
      float x[8];
      load8<DT>(vin, (t0 + t) * a.v_token + d, x);
      uint32_t* const p = reinterpret_cast<uint32_t*>(turn + t * pitch + d);
      p[0] = codes4(x, v_new), p[1] = codes4(x + 4, v_new);
    }
    __syncthreads();
    for (int i = tid; i < m * dim; i += 256) {
      const int d = i / m, t = i - d * m;
      vc[(int64_t)d * S + s0 + t0 + t] = turn[t * pitch + d];
    }
  }
}

}  // namespace

// n tokens fall into at most n pages, and at most (n - 1) / S + 2
int64_t kv_append_tiles(const KvSeqs& s) {
  const int64_t T = s.tokens, B = s.seqs;
  const int64_t tiles = s.offsets == nullptr ? B : (T >> s.shift) + 2 * B;
  return tiles < T ? tiles : T;
}
hipError_t launch_kv_append(const KvAppendArgs& a, int dtype, hipStream_t stream) {
  const dim3 grid((unsigned)kv_append_tiles(a.seqs), (unsigned)a.cache.heads);
  const unsigned lds = kSlab * (a.cache.dim + 4);
  if (dtype == kBF16) hipLaunchKernelGGL((k_kv_append<kBF16>), grid, dim3(256), lds, stream, a);
  else if (dtype == kF16) hipLaunchKernelGGL((k_kv_append<kF16>), grid, dim3(256), lds, stream, a);
  else hipLaunchKernelGGL((k_kv_append<kF32>), grid, dim3(256), lds, stream, a);
  return hipGetLastError();
}

}  // namespace lrq
