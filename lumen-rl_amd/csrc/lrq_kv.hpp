// What the kernels of the FP8 KV cache share (gfx950 only): its layout, and how a
// work-group finds the sequence it works on.
//
// K is [pages, heads, page, dim] and V [pages, heads, dim, page], e4m3 codes, with one
// float32 scale per page and head for each.  V lies with its tokens side by side because
// the second product of attention sums over them: a lane's 16-byte load is an operand of
// a matrix instruction, for K (16 of a token's channels) and for V (16 tokens of a
// channel) alike, and no transposition is left to the reader, who comes a thousand times
// for each write.  A page's scales are powers of two, so that codes can move to a larger
// scale with no rounding but that of the smallest of them.
//
// Page numbers, lengths and offsets are the caller's device data: whatever they hold, no
// access leaves the buffers.  A page number outside the pool stands for no page: nothing
// is written there and its tokens are not seen.
#pragma once

#include "lrq_device.hpp"
#include "lrq_internal.hpp"

namespace lrq {

typedef float f32x4 __attribute__((ext_vector_type(4)));

// A load for the whole wave through the scalar cache, of data that no one writes meanwhile;
// `p` is the same in all lanes.  It does not stand in the line of the vector loads: a page
// number that a lane had to wait for would first wait for all codes asked for before it.
template <class T>
__device__ __forceinline__ T sld(const T* p) {
  return *(const __attribute__((address_space(4))) T*)(uintptr_t)p;
}

// A sequence: its new tokens are rows [first, first + n) of the call's; len counts them in.
struct KvSeq {
  int64_t first;
  int n, len;
};
__device__ __forceinline__ KvSeq kv_seq(const KvSeqs& s, int b) {
  KvSeq q;
  const int64_t most = (int64_t)s.width << s.shift;
  const int64_t len = gld<int32_t>(s.lengths + b);
  q.len = (int)(len < 0 ? 0 : len > most ? most : len);
  if (s.offsets == nullptr) {
    q.first = b;
    q.n = b < s.tokens ? 1 : 0;
    return q;
  }
  const int64_t lo = gld<int32_t>(s.offsets + b), hi = gld<int32_t>(s.offsets + b + 1);
  q.first = lo < 0 ? 0 : lo > s.tokens ? s.tokens : lo;
  const int64_t end = hi < q.first ? q.first : hi > s.tokens ? s.tokens : hi;
  q.n = (int)(end - q.first);
  return q;
}
// The pool's page number at place j of row b, or -1.
__device__ __forceinline__ int kv_page(const KvSeqs& s, int pages, int b, int j) {
  const int p = gld<int32_t>(s.table + (int64_t)b * s.ld + j);
  return (uint32_t)p < (uint32_t)pages ? p : -1;
}

// The same for one b and j in all lanes.
__device__ __forceinline__ KvSeq kv_seq_uniform(const KvSeqs& s, int b) {
  KvSeq q;
  const int64_t most = (int64_t)s.width << s.shift;
  const int64_t len = sld(s.lengths + b);
  q.len = (int)(len < 0 ? 0 : len > most ? most : len);
  if (s.offsets == nullptr) {
    q.first = b;
    q.n = b < s.tokens ? 1 : 0;
    return q;
  }
  const int64_t lo = sld(s.offsets + b), hi = sld(s.offsets + b + 1);
  q.first = lo < 0 ? 0 : lo > s.tokens ? s.tokens : lo;
  const int64_t end = hi < q.first ? q.first : hi > s.tokens ? s.tokens : hi;
  q.n = (int)(end - q.first);
  return q;
}
__device__ __forceinline__ int kv_page_uniform(const KvSeqs& s, int pages, int b, int j) {
  if (j >= s.width) return -1;
  const int p = sld(s.table + (int64_t)b * s.ld + j);
  return (uint32_t)p < (uint32_t)pages ? p : -1;
}

// Work is numbered through all sequences of a call.  Up to so many are looked over by each
// work-group to find where its own is; with more, a launch before leaves the numbers up to each
// sequence, which a wave searches 64 at a time (4096 sequences, one token of each on 100 keys:
// 654 us without that launch, 260 with it; 1024 on 400 keys 204 and 172; two tokens appended to
// each of 4096: 656 and 181).
constexpr int kOwnSearch = 256;
// The first of n places whose number is above `at`; the last one's is.
__device__ __forceinline__ int kv_find(const int32_t* upto, int n, uint32_t at) {
  const int lane = threadIdx.x & 63;
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int step = (hi - lo + 63) >> 6, mine = lo + (lane + 1) * step - 1;
    const uint64_t above = __ballot((uint32_t)gld<int32_t>(upto + (mine < hi ? mine : hi - 1)) > at);
    lo += above != 0 ? __builtin_ctzll(above) * step : hi - 1 - lo;
    hi = lo + step < hi ? lo + step : hi;
  }
  return __builtin_amdgcn_readfirstlane(lo);
}

// Inclusive sum over the work-group's threads (256 or 1024); `waves` is LDS, one word a wave.
template <int THREADS, class T>
__device__ __forceinline__ T block_scan(T v, T* waves) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const T o = __shfl_up(v, off, 64);
    if (lane >= off) v += o;
  }
  if (lane == 63) waves[wave] = v;
  __syncthreads();
  T before = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 64; ++w) before += w < wave ? waves[w] : T(0);
  __syncthreads();
  return v + before;
}

// The sum over the work-group's threads, for each of them.
template <int WAVES, class T>
__device__ __forceinline__ T block_sum(T v, T* waves) {
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) v += __shfl_xor(v, off, 64);
  if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = v;
  __syncthreads();
  T sum = 0;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) sum += waves[w];
  __syncthreads();
  return sum;
}

// The least e in -48 .. 48 whose 448 x 2^e is not below amax (a finite value's bits).
// Values behind that range become NaN codes, as in an unscaled cast.
constexpr int kKvExpMin = -48, kKvExpMax = 48;
__device__ __forceinline__ float kv_scale(uint32_t amax_bits) {
  // 448 = 1.75 x 2^8; a subnormal amax has the exponent field 0 and is clamped
  const int e = (int)(amax_bits >> 23) - 127 - 8 + ((amax_bits & 0x7FFFFFu) > 0x600000u);
  const int c = e < kKvExpMin ? kKvExpMin : e > kKvExpMax ? kKvExpMax : e;
  return u2f((uint32_t)(c + 127) << 23);
}

}  // namespace lrq
