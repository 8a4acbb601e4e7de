// Routing to experts: scores, the choice of top_k of them, their weights, and the
// gradient of the logits.
//
//   score_e = softmax(x)_e or sigmoid(x_e);  pick_e = score_e + bias_e
//   a group's value: the sum of its group_top (1 or 2) highest picks
//   ids: the top_k highest picks of the top_groups best groups, ties to the
//        lowest index; weights: scale score_id, over sum score_id if renormalized.
//
// The choice is that of exact arithmetic, up to 64-bit rounding.  Without a bias
// both scores rise with the logit, so logits are compared.  Picks, and sums of two
// scores, are computed in float32.  What is compared becomes one word of an expert:
// the order of a 16-bit logit above the index, or a fixed-point value (23 to 25 bits
// of the 4 below a token's highest pick, of the 64 below its highest logit) above
// it; so a round of the choice is one maximum, and ties go to the lowest index.  A
// token with two neighbours in that order (or two groups) nearer to each other than
// the words can tell is chosen again by its whole wave in float64, unless the two
// have the same logit and bias and so are a tie.  A tie of the last one chosen with the
// next counts only if all open experts behind them that are as near are their equals.
// With random biases a token in a thousand is chosen again, and costs the rest nothing.
//
// Moves little: 2 or 4 bytes an expert.  What it spends is instructions, 1.5 an
// expert for each of the top_k rounds and some 15 before; so 16 lanes take a token,
// four tokens a wave, whose maxima go through DPP rows without LDS.
#include "lrq.h"
#include "lrq_device.hpp"
#include "lrq_internal.hpp"
#include "lrq_mma8.hpp"

namespace lrq {

constexpr int kRouteTokens = 16;  // a work-group's: 4 waves, 16 lanes a token
constexpr float kLog2e = 1.44269504088896341f;

// ---------------------------------------------------------------------------
// order: unsigned integers that rise with the value, -0 as 0, NaN above all
// ---------------------------------------------------------------------------
__device__ __forceinline__ uint32_t order32(float v) {
  const uint32_t b = f2u(v + 0.0f);
  return v != v ? 0xFFFFFFFFu : b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ uint64_t order64(double v) {
  const uint64_t b = (uint64_t)__double_as_longlong(v + 0.0);
  return v != v ? ~0ull : b ^ ((uint64_t)((int64_t)b >> 63) | 0x8000000000000000ull);
}
__device__ __forceinline__ double order64_value(uint64_t k) {
  return __longlong_as_double((long long)(k ^ (k >> 63 ? 0x8000000000000000ull : ~0ull)));
}

// Over the 16 lanes of a DPP row; every lane of the wave is active.
template <class F>
__device__ __forceinline__ uint32_t row16(uint32_t v, F f) {
  v = f(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0xB1, 0xF, 0xF, false));
  v = f(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x4E, 0xF, 0xF, false));
  v = f(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x141, 0xF, 0xF, false));
  return f(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x140, 0xF, 0xF, false));
}
__device__ __forceinline__ uint32_t row_max(uint32_t v) {
  return row16(v, [](uint32_t a, uint32_t b) { return a > b ? a : b; });
}
__device__ __forceinline__ float row_fmax(float v) {
  return u2f(row16(f2u(v), [](uint32_t a, uint32_t b) { return f2u(fmaxf(u2f(a), u2f(b))); }));
}
__device__ __forceinline__ float row_sum(float v) {
  return u2f(row16(f2u(v), [](uint32_t a, uint32_t b) { return f2u(u2f(a) + u2f(b)); }));
}
// e / size = e group_recip(size) / 2^20, for e and size up to 512
__device__ __forceinline__ uint32_t group_recip(int size) { return ((1u << 20) + (uint32_t)size - 1) / (uint32_t)size; }

// Pairwise, so that the error grows with the logarithm of the count.
template <int N>
__device__ __forceinline__ float tree_sum(const float* v) {
  if constexpr (N == 1) return v[0];
  else return tree_sum<N / 2>(v) + tree_sum<N - N / 2>(v + N / 2);
}

// ---------------------------------------------------------------------------
// a token's logits: lane l of 16 holds experts 128 c + 8 l .. + 7 at 8 c ..
// ---------------------------------------------------------------------------
template <int DT, int CHUNKS>
__device__ __forceinline__ void load_row(const void* row, int experts, int l, float* x) {
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c) load_acts<DT>(row, 128 * c + 8 * l, experts, x + 8 * c);
}
__device__ __forceinline__ int expert_of(int s, int l) { return 128 * (s >> 3) + 8 * l + (s & 7); }

template <int DT, int CHUNKS>
__device__ __forceinline__ void store_row(void* row, int experts, int l, const float* v) {
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c) {
    const int e = 128 * c + 8 * l;
    if (e >= experts) continue;
    if constexpr (DT == kF32) {
      float* const p = static_cast<float*>(row) + e;
      if (e + 8 <= experts) {
        *(LRQ_GLOBAL v4u_any*)p = v4u{f2u(v[8 * c]), f2u(v[8 * c + 1]), f2u(v[8 * c + 2]), f2u(v[8 * c + 3])};
        *(LRQ_GLOBAL v4u_any*)(p + 4) = v4u{f2u(v[8 * c + 4]), f2u(v[8 * c + 5]), f2u(v[8 * c + 6]), f2u(v[8 * c + 7])};
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (e + i < experts) gst<float>(p + i, v[8 * c + i]);
      }
    } else {
      uint16_t* const p = static_cast<uint16_t*>(row) + e;
      uint32_t h[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) h[i] = bits16<DT>(v[8 * c + i]);
      if (e + 8 <= experts) {
        *(LRQ_GLOBAL v4u_any*)p = v4u{h[0] | h[1] << 16, h[2] | h[3] << 16, h[4] | h[5] << 16, h[6] | h[7] << 16};
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (e + i < experts) gst<uint16_t>(p + i, (uint16_t)h[i]);
      }
    }
  }
}

// Scores good to 2^-20 (of 1), for the choice only.
template <int CHUNKS>
__device__ __forceinline__ void quick_scores(const RouteArgs& a, const float* x, int l, bool normalize, float* p) {
  constexpr int S = 8 * CHUNKS;
  if (a.sigmoid) {
#pragma unroll
    for (int s = 0; s < S; ++s) p[s] = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-kLog2e * x[s]));
    return;
  }
  float top = -INFINITY;
#pragma unroll
  for (int s = 0; s < S; ++s) top = expert_of(s, l) < a.experts ? fmaxf(top, x[s]) : top;
  top = row_fmax(top);
#pragma unroll
  for (int s = 0; s < S; ++s) p[s] = expert_of(s, l) < a.experts ? __builtin_amdgcn_exp2f(kLog2e * (x[s] - top)) : 0.0f;
  if (!normalize) return;
  const float inv = __builtin_amdgcn_rcpf(row_sum(tree_sum<S>(p)));
#pragma unroll
  for (int s = 0; s < S; ++s) p[s] *= inv;
}

// ---------------------------------------------------------------------------
// one token's choice in float64, by a whole wave
// ---------------------------------------------------------------------------
template <int CTRL>
__device__ __forceinline__ uint64_t moved64(uint64_t v) {
  const uint32_t lo = (uint32_t)__builtin_amdgcn_mov_dpp((int)(uint32_t)v, CTRL, 0xF, 0xF, false);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_mov_dpp((int)(uint32_t)(v >> 32), CTRL, 0xF, 0xF, false);
  return (uint64_t)hi << 32 | lo;
}
__device__ __forceinline__ uint64_t lane64(uint64_t v, int lane) {
  return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(v >> 32), lane) << 32 |
         (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, lane);
}
// Over the wave, in DPP rows and then from one lane of each.
template <class F>
__device__ __forceinline__ uint64_t wave64(uint64_t v, F f) {
  v = f(v, moved64<0xB1>(v));
  v = f(v, moved64<0x4E>(v));
  v = f(v, moved64<0x141>(v));
  v = f(v, moved64<0x140>(v));
  return f(f(lane64(v, 0), lane64(v, 16)), f(lane64(v, 32), lane64(v, 48)));
}
__device__ __forceinline__ uint64_t wave_max64(uint64_t v) {
  return wave64(v, [](uint64_t a, uint64_t b) { return a > b ? a : b; });
}
__device__ __forceinline__ double wave_sum64(double v) {
  return __longlong_as_double((long long)wave64((uint64_t)__double_as_longlong(v), [](uint64_t a, uint64_t b) {
    return (uint64_t)__double_as_longlong(__longlong_as_double((long long)a) + __longlong_as_double((long long)b));
  }));
}

template <int DT, int CHUNKS>
__device__ __forceinline__ void choose_wide(const RouteArgs& a, int64_t token, uint64_t* stage, uint32_t* ids) {
  constexpr int J = 2 * CHUNKS;
  const int lane = threadIdx.x & 63;
  float x[J];
  double p[J];
#pragma unroll
  for (int j = 0; j < J; ++j) {
    const int e = lane + 64 * j;
    x[j] = e < a.experts ? load_as_f32(a.logits, DT, token * a.ld + e) : -INFINITY;
  }
  if (a.sigmoid) {
#pragma unroll
    for (int j = 0; j < J; ++j) p[j] = 1.0 / (1.0 + exp(-(double)x[j]));
  } else {
    float top = -INFINITY;
#pragma unroll
    for (int j = 0; j < J; ++j) top = fmaxf(top, x[j]);
    top = row_fmax(top);
    auto row = [&](int lane) { return u2f((uint32_t)__builtin_amdgcn_readlane((int)f2u(top), lane)); };
    top = fmaxf(fmaxf(row(0), row(16)), fmaxf(row(32), row(48)));
    double sum = 0.0;
#pragma unroll
    for (int j = 0; j < J; ++j) {
      p[j] = lane + 64 * j < a.experts ? exp((double)x[j] - (double)top) : 0.0;
      sum += p[j];
    }
    sum = wave_sum64(sum);
#pragma unroll
    for (int j = 0; j < J; ++j) p[j] /= sum;
  }
  const bool by_logit = a.bias == nullptr;
#pragma unroll
  for (int j = 0; j < J; ++j)
    if (!by_logit && lane + 64 * j < a.experts) p[j] += (double)gld<float>(a.bias + lane + 64 * j);
  uint64_t allowed = ~0ull;
  const int size = a.experts / a.groups;
  if (a.groups > 1) {
    wave_fence8();
#pragma unroll
    for (int j = 0; j < J; ++j)
      if (lane + 64 * j < a.experts) stage[lane + 64 * j] = order64(by_logit && a.group_top == 1 ? (double)x[j] : p[j]);
    wave_fence8();
    uint64_t value = 0;
    if (lane < a.groups) {
      uint64_t first = 0, second = 0;
#pragma unroll 8
      for (int i = 0; i < size; ++i) {
        const uint64_t k = stage[lane * size + i];
        second = k > first ? first : k > second ? k : second;
        first = k > first ? k : first;
      }
      value = a.group_top == 2 && size > 1 ? order64(order64_value(first) + order64_value(second)) : first;
    }
    int before = 0;
    for (int g = 0; g < a.groups; ++g) {
      const uint64_t o = lane64(value, g);
      before += o > value || (o == value && g < lane) ? 1 : 0;
    }
    allowed = __ballot(lane < a.groups && before < a.top_groups);
  }
  uint64_t key[J];
#pragma unroll
  for (int j = 0; j < J; ++j) {
    const int e = lane + 64 * j;
    key[j] = by_logit ? order32(x[j]) : order64(p[j]);
    const uint32_t g = (uint32_t)e * group_recip(size) >> 20;
    if (e >= a.experts || !(allowed >> (g & 63) & 1)) key[j] = 0;
  }
  for (int i = 0; i < a.top_k; ++i) {
    uint64_t best = 0;
#pragma unroll
    for (int j = 0; j < J; ++j) best = key[j] > best ? key[j] : best;
    best = wave_max64(best);
    uint32_t e = 0;
#pragma unroll
    for (int j = J - 1; j >= 0; --j) {
      const uint64_t has = __ballot(key[j] == best);
      e = has ? 64 * j + (uint32_t)__builtin_ctzll(has) : e;
    }
#pragma unroll
    for (int j = 0; j < J; ++j) key[j] = e == (uint32_t)(lane + 64 * j) ? 0 : key[j];
    if (lane == 0) ids[i] = e;
  }
}

// ---------------------------------------------------------------------------
// the router
// ---------------------------------------------------------------------------
enum RouteKeys { kKeysLogit16, kKeysLogit32, kKeysPick };

__device__ __forceinline__ void top_two(float& first, float& second, float a, float b) {  // a >= b
  second = fmaxf(fmaxf(second, b), fminf(first, a));
  first = fmaxf(first, a);
}

template <int DT, int CHUNKS, int KEYS>
__global__ __launch_bounds__(256) void k_route(RouteArgs a) {
  constexpr int S = 8 * CHUNKS;
  constexpr int BITS = KEYS == kKeysLogit16 ? 16 : CHUNKS == 1 ? 7 : CHUNKS == 2 ? 8 : 9;  // of the index
  constexpr uint32_t kIndex = (1u << BITS) - 1;
  constexpr float kWindow = KEYS == kKeysPick ? 4.0f : 64.0f, kMost = (float)((1ull << (32 - BITS)) - 16);
  // words of LDS: each token's choice and its keys, its groups' values, then (with
  // groups) its picks
  extern __shared__ __attribute__((aligned(16))) uint32_t lds_route[];
  const int tid = threadIdx.x, lane = tid & 63, l = lane & 15, row = tid >> 4;
  const int64_t token = (int64_t)blockIdx.x * kRouteTokens + row;
  const int64_t mine = token < a.tokens ? token : a.tokens - 1;
  const uint8_t* const logits = static_cast<const uint8_t*>(a.logits) + mine * a.ld * (DT == kF32 ? 4 : 2);
  uint32_t* const ids = lds_route + row * kRouteWords;
  uint32_t* const keys = ids + kRoutePitch;
  float* const values = reinterpret_cast<float*>(keys + kRoutePitch);
  uint32_t* const waves = lds_route + kRouteWords * kRouteTokens + (tid >> 6) * 4 * a.experts;  // the wave's stage
  float* const stage = reinterpret_cast<float*>(waves + (row & 3) * a.experts);

  float x[S], v[S];  // v: what orders experts
  load_row<DT, CHUNKS>(logits, a.experts, l, x);
  bool unsure = false;
  float poison = 0.0f;  // NaN where a logit that need not be chosen makes every softmax score NaN
#pragma unroll
  for (int s = 0; s < S; s += 2) unsure |= __builtin_isunordered(x[s], x[s + 1]);  // past the last expert they are 0
  if constexpr (KEYS == kKeysPick) {
    quick_scores<CHUNKS>(a, x, l, true, v);
    if (!a.sigmoid) poison = 0.0f * v[0];
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
      float b[8];
      load_acts<kF32>(a.bias, 128 * c + 8 * l, a.experts, b);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[8 * c + i] += b[i];
    }
#pragma unroll
    for (int s = 0; s < S; s += 2) unsure |= __builtin_isunordered(v[s], v[s + 1]);
  } else {
#pragma unroll
    for (int s = 0; s < S; ++s) v[s] = x[s];
  }

  uint32_t key[S];
  const float tol = a.sigmoid ? kRouteTol : 2.0f * kRouteTol;
  float low = 0.0f;
  if constexpr (KEYS == kKeysLogit16) {
#pragma unroll
    for (int s = 0; s < S; ++s) {
      const uint32_t b = DT == kBF16 ? f2u(x[s] + 0.0f) >> 16 : f16_bits(x[s] + 0.0f);
      const uint32_t order = b & 0x8000u ? 0xFFFFu ^ b : 0x8000u | b;
      key[s] = order << 16 | (kIndex - (uint32_t)expert_of(s, l));
    }
  } else {
    float top = -INFINITY;
#pragma unroll
    for (int s = 0; s < S; ++s) top = fmaxf(top, expert_of(s, l) < a.experts ? v[s] : -INFINITY);
    top = row_fmax(top);
    unsure |= fabsf(top) == INFINITY;
    low = top - kWindow;
#pragma unroll
    for (int s = 0; s < S; ++s) {
      const float q = fmaxf((v[s] - low) * (kMost / kWindow), 1.0f);  // rises with v; NaN and below the window: 1
      key[s] = (uint32_t)q << BITS | (kIndex - (uint32_t)expert_of(s, l));
    }
  }
#pragma unroll
  for (int s = 0; s < S; ++s)
    if (expert_of(s, l) >= a.experts) key[s] = 0;

  if (a.groups > 1) {
    const int size = a.experts / a.groups;
    const bool sums = KEYS == kKeysPick || a.group_top == 2;  // otherwise logits, which are exact
    if (KEYS != kKeysPick && a.group_top == 2) quick_scores<CHUNKS>(a, x, l, false, v);
    float first = -INFINITY, second = -INFINITY;  // lane g: of group g
    if (size % 8 == 0) {  // a lane's 8 experts are in one group
#pragma unroll
      for (int c = 0; c < CHUNKS; ++c) {
        float one = v[8 * c], two = -INFINITY;
#pragma unroll
        for (int i = 1; i < 8; ++i) top_two(one, two, v[8 * c + i], -INFINITY);
        if (128 * c + 8 * l < a.experts) {
          stage[2 * (16 * c + l)] = one;
          stage[2 * (16 * c + l) + 1] = two;
        }
      }
      wave_fence8();
      if (l < a.groups)
        for (int i = 0; i < size / 8; ++i) {
          const float* const p = stage + 2 * (l * (size / 8) + i);
          top_two(first, second, p[0], p[1]);
        }
    } else {
#pragma unroll
      for (int s = 0; s < S; ++s)
        if (expert_of(s, l) < a.experts) stage[expert_of(s, l)] = v[s];
      wave_fence8();
      if (l < a.groups) {
        int at = l % size;  // each lane from another place: no bank conflicts
        for (int i = 0; i < size; ++i) {
          top_two(first, second, stage[l * size + at], -INFINITY);
          at = at + 1 < size ? at + 1 : 0;
        }
      }
    }
    const float value = a.group_top == 2 && size > 1 ? first + second : first;
    values[l] = l < a.groups ? value : -INFINITY;
    wave_fence8();
    int before = 0;
#pragma unroll
    for (int g = 0; g < kRouteGroupsMax; ++g) {
      const float o = values[g];
      before += g < a.groups && (o > value || (o == value && g < l)) ? 1 : 0;
      unsure |= sums && l < a.groups && g < a.groups && g != l && !(fabsf(o - value) > tol * (1.0f + fabsf(value)));
    }
    const uint64_t all = __ballot(l < a.groups && before < a.top_groups);
    const uint32_t allowed = (uint32_t)(all >> (lane & 48)) & 0xFFFFu;
    const uint32_t recip = group_recip(size);
    if (size % 8 == 0) {
#pragma unroll
      for (int c = 0; c < CHUNKS; ++c) {
        const uint32_t g = (uint32_t)(128 * c + 8 * l) * recip >> 20;
        const bool open = allowed >> (g & 31) & 1;
#pragma unroll
        for (int i = 0; i < 8; ++i) key[8 * c + i] = open ? key[8 * c + i] : 0;
      }
    } else {
#pragma unroll
      for (int s = 0; s < S; ++s) {
        const uint32_t g = (uint32_t)expert_of(s, l) * recip >> 20;
        if (!(allowed >> (g & 31) & 1)) key[s] = 0;
      }
    }
  }

  // Rounds: the highest key below the last one.  key - last wraps round for the keys
  // below it, which so come above all others, in their order.
  const int left = a.groups > 1 ? a.experts / a.groups * a.top_groups : a.experts;
  const int rounds = KEYS != kKeysLogit16 && left > a.top_k ? a.top_k + 1 : a.top_k;
  uint32_t last = 0;
  for (int i = 0; i < rounds; ++i) {
    uint32_t best = 0;
#pragma unroll
    for (int s = 0; s < S; ++s) {
      const uint32_t k = key[s] - last;
      best = k > best ? k : best;
    }
    last += row_max(best);
    if (l == 0) ids[i] = kIndex - (last & kIndex), keys[i] = last >> BITS;
  }
  wave_fence8();
  if constexpr (KEYS != kKeysLogit16) {
    // words that cannot tell which is higher, `next` being no higher than `word`
    auto near = [&](uint32_t word, uint32_t next) {
      const float here = (float)word * (kWindow / kMost), there = (float)next * (kWindow / kMost);
      return KEYS == kKeysPick ? !(here - there > tol * (1.0f + fabsf(low + here))) : word == next;
    };
    auto expert = [&](int i) { return ids[i] < (uint32_t)a.experts ? ids[i] : 0u; };
    auto bias_of = [&](uint32_t e) { return KEYS == kKeysPick ? gld<float>(a.bias + e) : 0.0f; };
    auto equal = [&](uint32_t e, uint32_t f) {
      return load_as_f32(logits, DT, e) == load_as_f32(logits, DT, f) && bias_of(e) == bias_of(f);
    };
    for (int i = l; i + 1 < rounds; i += 16)
      if (near(keys[i], keys[i + 1])) unsure |= !equal(expert(i), expert(i + 1));
    // A tie of the last one and the next does not settle the choice: any open expert
    // behind them, as near to them but not their equal, may be higher.
    const int k = a.top_k - 1;
    if (rounds > a.top_k && near(keys[k], keys[k + 1]) && equal(expert(k), expert(k + 1))) {
      const uint32_t e = expert(k), last_key = keys[k] << BITS | (kIndex - ids[k]);
#pragma unroll
      for (int s = 0; s < S; ++s)
        if (key[s] != 0 && key[s] < last_key && near(keys[k], key[s] >> BITS)) {
          if (!equal(e, (uint32_t)expert_of(s, l))) unsure = true;
        }
    }
  }
  uint64_t again = __ballot(unsure);
  while (again) {
    const int r = __builtin_ctzll(again) >> 4;
    again &= ~(0xFFFFull << (16 * r));
    const int64_t t = (int64_t)blockIdx.x * kRouteTokens + (row & ~3) + r;
    wave_fence8();
    choose_wide<DT, CHUNKS>(a, t < a.tokens ? t : a.tokens - 1, reinterpret_cast<uint64_t*>(waves),
                            lds_route + ((row & ~3) + r) * kRouteWords);
  }
  wave_fence8();

  // weights, in float32: softmax over the chosen alone when they are renormalized
  float top = 0.0f, sum = 1.0f;
  if (!a.sigmoid) {
    top = -INFINITY;
    if (a.renormalize) {
      for (int i = l; i < a.top_k; i += 16) top = fmaxf(top, load_as_f32(logits, DT, ids[i]));
    } else {
#pragma unroll
      for (int s = 0; s < S; ++s) top = expert_of(s, l) < a.experts ? fmaxf(top, x[s]) : top;
    }
    top = row_fmax(top);
  }
  float w[kRouteMost / 16];
#pragma unroll
  for (int r = 0; r < kRouteMost / 16; ++r) {
    w[r] = 0.0f;
    if (16 * r >= a.top_k) break;
    const int i = 16 * r + l;
    if (i < a.top_k) {
      const float v = load_as_f32(logits, DT, ids[i]);
      w[r] = a.sigmoid ? 1.0f / (1.0f + expf(-v)) : expf(v - top);
    }
  }
  if (a.renormalize) {
    sum = row_sum(w[0] + w[1] + (w[2] + w[3])) + (a.sigmoid ? 1e-20f : poison);
  } else if (!a.sigmoid) {
#pragma unroll
    for (int s = 0; s < S; ++s) x[s] = expert_of(s, l) < a.experts ? expf(x[s] - top) : 0.0f;
    sum = row_sum(tree_sum<S>(x));
  }
  if (token >= a.tokens) return;
#pragma unroll
  for (int r = 0; r < kRouteMost / 16; ++r) {
    const int i = 16 * r + l;
    if (i >= a.top_k) break;
    gst<float>(a.weights + token * a.top_k + i, w[r] / sum * a.scale);
    gst<int32_t>(a.ids + token * a.top_k + i, (int32_t)ids[i]);
  }
}

// ---------------------------------------------------------------------------
// the gradient of the logits
// ---------------------------------------------------------------------------
// With q = the scores (over their sum if renormalized) and g the weights' gradient:
//   renormalized   dx_i = scale q_i (g_i - sum_j g_j q_j), times 1 - s_i for sigmoid
//   sigmoid alone  dx_i = scale s_i (1 - s_i) g_i
//   softmax alone  dx_e = scale p_e (g_e [e chosen] - sum_j g_j p_j) for every expert
// Only the last reads logits that were not chosen.  The rest of the row is zeros.
template <int DT, int CHUNKS>
__global__ __launch_bounds__(256) void k_route_grad(RouteArgs a, const float* grad, void* out) {
  constexpr int S = 8 * CHUNKS, PITCH = 128 * CHUNKS;
  __shared__ __attribute__((aligned(16))) float lds[kRouteTokens * PITCH];
  const int tid = threadIdx.x, l = tid & 15, row = tid >> 4;
  const int64_t token = (int64_t)blockIdx.x * kRouteTokens + row;
  const int64_t mine = token < a.tokens ? token : a.tokens - 1;
  const uint8_t* const logits = static_cast<const uint8_t*>(a.logits) + mine * a.ld * (DT == kF32 ? 4 : 2);
  float* const dense = lds + row * PITCH;
  const bool all = !a.sigmoid && !a.renormalize;
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c) {
    *reinterpret_cast<f32x4*>(dense + 128 * c + 8 * l) = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    *reinterpret_cast<f32x4*>(dense + 128 * c + 8 * l + 4) = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  }
  float x[S], top = -INFINITY, sum = 1.0f;
  if (all) {
    load_row<DT, CHUNKS>(logits, a.experts, l, x);
#pragma unroll
    for (int s = 0; s < S; ++s) top = expert_of(s, l) < a.experts ? fmaxf(top, x[s]) : top;
    top = row_fmax(top);
#pragma unroll
    for (int s = 0; s < S; ++s) x[s] = expert_of(s, l) < a.experts ? expf(x[s] - top) : 0.0f;
    sum = row_sum(tree_sum<S>(x));
#pragma unroll
    for (int s = 0; s < S; ++s) x[s] /= sum;
  }
  constexpr int R = kRouteMost / 16;
  float q[R], keep[R], g[R];
  int id[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int i = 16 * r + l;
    id[r] = i < a.top_k ? gld<int32_t>(a.ids + mine * a.top_k + i) : -1;
    const bool has = (uint32_t)id[r] < (uint32_t)a.experts;  // any other has no gradient
    id[r] = has ? id[r] : -1;
    g[r] = has ? gld<float>(grad + mine * a.top_k + i) * a.scale : 0.0f;
    q[r] = has ? load_as_f32(logits, DT, id[r]) : -INFINITY;
    if (!all && !a.sigmoid) top = fmaxf(top, q[r]);
  }
  if (!all && !a.sigmoid) top = row_fmax(top);
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const float t = expf(a.sigmoid ? -q[r] : q[r] - top);
    keep[r] = a.sigmoid ? t / (1.0f + t) : 1.0f;  // 1 - s
    if (a.sigmoid && t == INFINITY) keep[r] = 1.0f;
    q[r] = id[r] < 0 ? 0.0f : a.sigmoid ? 1.0f / (1.0f + t) : t / sum;
  }
  if (a.renormalize) {
    const float total = row_sum(q[0] + q[1] + (q[2] + q[3])) + (a.sigmoid ? 1e-20f : 0.0f);
#pragma unroll
    for (int r = 0; r < R; ++r) q[r] /= total;
  }
  const float dot = row_sum(g[0] * q[0] + g[1] * q[1] + (g[2] * q[2] + g[3] * q[3]));
  wave_fence8();
#pragma unroll
  for (int r = 0; r < R; ++r)
    if (id[r] >= 0) dense[id[r]] = all ? g[r] : q[r] * keep[r] * (a.renormalize ? g[r] - dot : g[r]);
  wave_fence8();
  float d[S];
#pragma unroll
  for (int s = 0; s < S; ++s) {
    d[s] = dense[expert_of(s, l)];
    if (all) d[s] = x[s] * (d[s] - dot);
  }
  if (token >= a.tokens) return;
  store_row<DT, CHUNKS>(static_cast<uint8_t*>(out) + token * a.experts * (DT == kF32 ? 4 : 2), a.experts, l, d);
}

// ---------------------------------------------------------------------------
template <int DT, int CHUNKS>
static void launch(const RouteArgs& a, const float* grad, void* out, hipStream_t stream) {
  const dim3 grid((unsigned)((a.tokens + kRouteTokens - 1) / kRouteTokens));
  if (out != nullptr) {
    hipLaunchKernelGGL((k_route_grad<DT, CHUNKS>), grid, dim3(256), 0, stream, a, grad, out);
    return;
  }
  const unsigned lds = 4 * kRouteTokens * (kRouteWords + (a.groups > 1 ? a.experts : 0));
  if (a.bias != nullptr) hipLaunchKernelGGL((k_route<DT, CHUNKS, kKeysPick>), grid, dim3(256), lds, stream, a);
  else hipLaunchKernelGGL((k_route<DT, CHUNKS, DT == kF32 ? kKeysLogit32 : kKeysLogit16>), grid, dim3(256), lds, stream, a);
}
template <int DT>
static void launch_of(const RouteArgs& a, const float* grad, void* out, hipStream_t stream) {
  if (a.experts <= 128) launch<DT, 1>(a, grad, out, stream);
  else if (a.experts <= 256) launch<DT, 2>(a, grad, out, stream);
  else launch<DT, 4>(a, grad, out, stream);
}
// A launch has fewer than 2^32 threads, 16 of them a token.
constexpr int64_t kRouteLaunch = int64_t(1) << 27;
hipError_t launch_route(RouteArgs a, int dtype, const float* grad, void* out, hipStream_t stream) {
  const int64_t es = dtype == kF32 ? 4 : 2, tokens = a.tokens;
  for (int64_t t0 = 0; t0 < tokens; t0 += kRouteLaunch) {
    a.tokens = tokens - t0 < kRouteLaunch ? tokens - t0 : kRouteLaunch;
    if (dtype == kBF16) launch_of<kBF16>(a, grad, out, stream);
    else if (dtype == kF16) launch_of<kF16>(a, grad, out, stream);
    else launch_of<kF32>(a, grad, out, stream);
    if (hipError_t e = hipGetLastError()) return e;
    a.logits = static_cast<const uint8_t*>(a.logits) + kRouteLaunch * a.ld * es;
    a.ids += kRouteLaunch * a.top_k;
    if (out != nullptr) grad += kRouteLaunch * a.top_k, out = static_cast<uint8_t*>(out) + kRouteLaunch * a.experts * es;
    else a.weights += kRouteLaunch * a.top_k;
  }
  return hipSuccess;
}

}  // namespace lrq
