// Upkeep of the pages of an FP8 KV cache: rows of the page table are copied, grown,
// shortened and ended, and the pages in use are moved together.
//
// refs[p] counts the rows that hold page p; a page is free where that is not above 0.
// Counts change by atomic additions, which commute, so results do not depend on their
// order; pages are handed out lowest first, in the order of the rows, by prefix sums.
//
// Without data to move these are launches and little else: a fork 3 us, a resize of 256 rows
// 1.6, 5.3 and 1.8, whose second launch, one work-group, waits for its loads in turn.  Data moves
// at 5.2 TB/s, read and written (271 MB in 103 us).
#include "lrq_kv.hpp"

namespace lrq {

namespace {

__device__ __forceinline__ int pages_of(int64_t len, int shift) { return (int)((len + (1 << shift) - 1) >> shift); }
__device__ __forceinline__ int64_t clamp_len(int64_t len, const KvTable& t) {
  const int64_t most = (int64_t)t.width << t.shift;
  return len < 0 ? 0 : len > most ? most : len;
}
__device__ __forceinline__ int entry(const KvTable& t, int64_t row, int j) { return gld<int32_t>(t.table + row * t.ld + j); }
__device__ __forceinline__ bool in_pool(int p, int pages) { return (uint32_t)p < (uint32_t)pages; }

// ---------------------------------------------------------------------------
// fork
// ---------------------------------------------------------------------------
__global__ __launch_bounds__(256) void k_kv_fork(KvTable t, const int32_t* parents, int32_t* refs, int pages, int32_t* out,
                                                 int32_t* out_len) {
  const int r = blockIdx.x;
  int p = gld<int32_t>(parents + r);
  if ((uint32_t)p >= (uint32_t)t.rows) p = r;
  const int64_t len = clamp_len(gld<int32_t>(t.lengths + p), t);
  const int n = pages_of(len, t.shift), old = pages_of(clamp_len(gld<int32_t>(t.lengths + r), t), t.shift);
  if (threadIdx.x == 0) gst<int32_t>(out_len + r, (int32_t)len);
  for (int j = threadIdx.x; j < t.width; j += 256) {
    const int e = j < n ? entry(t, p, j) : -1;
    gst<int32_t>(out + (int64_t)r * t.width + j, e);
    if (p == r) continue;
    if (in_pool(e, pages)) atomicAdd(refs + e, 1);
    if (j < old) {
      const int was = entry(t, r, j);
      if (in_pool(was, pages)) atomicAdd(refs + was, -1);
    }
  }
}

// ---------------------------------------------------------------------------
// the pages' data
// ---------------------------------------------------------------------------
constexpr int64_t kPart = 16384;  // bytes that a work-group copies before it looks for more

// Pairs (source, target) of pages, in every layer; no target is a source or twice a target.
// Targets are written past the caches (128 copies of 1 MiB of shared pages 58.9 -> 38.7 us);
// sources are read past them where each is read ONCE (271 MB moved 115.8 -> 112.4 us).
template <bool ONCE>
__device__ void copy_pages(const KvPool& c, const int32_t* pairs, int64_t count) {
  const int64_t bytes = ((int64_t)c.heads << c.shift) * c.dim, parts = (bytes + kPart - 1) / kPart;
  const int64_t total = count * c.layers * 2 * parts;
  for (int64_t i = blockIdx.x; i < total; i += gridDim.x) {
    const int64_t part = i % parts, of = i / parts;
    const bool v = of & 1;
    const int64_t layer = (of >> 1) % c.layers, pair = (of >> 1) / c.layers;
    const int64_t src = gld<int32_t>(pairs + 2 * pair), dst = gld<int32_t>(pairs + 2 * pair + 1);
    uint8_t* const base = v ? c.v + layer * c.v_layer : c.k + layer * c.k_layer;
    const int64_t step = v ? c.v_page : c.k_page;
    const uint8_t* const from = base + src * step;
    uint8_t* const to = base + dst * step;
#pragma unroll
    for (int u = 0; u < kPart / 4096; ++u) {
      const int64_t at = part * kPart + u * 4096 + threadIdx.x * 16;
      if (at < bytes) gst_nt<v4u>(to + at, ONCE ? gld_nt<v4u>(from + at) : gld<v4u>(from + at));
    }
    if (part == 0) {
      float* const s = v ? c.vs + layer * c.vs_layer : c.ks + layer * c.ks_layer;
      const int64_t sp = v ? c.vs_page : c.ks_page;
      for (int h = threadIdx.x; h < c.heads; h += 256) gst<float>(s + dst * sp + h, gld<float>(s + src * sp + h));
    }
  }
}

// ---------------------------------------------------------------------------
// resize
// ---------------------------------------------------------------------------
// What a row has and is to have; one that wants more than the table holds keeps what it has.
struct Change {
  int64_t len, want;
  int old_n, new_n;
};
__device__ __forceinline__ Change change_of(const KvTable& t, const int32_t* wanted, int64_t r) {
  Change c;
  c.len = clamp_len(gld<int32_t>(t.lengths + r), t);
  c.want = gld<int32_t>(wanted + r);
  c.want = c.want < 0 ? 0 : c.want;
  if (c.want > (int64_t)t.width << t.shift) c.want = c.len;
  c.old_n = pages_of(c.len, t.shift), c.new_n = pages_of(c.want, t.shift);
  return c;
}

// First: what shrinks is given back, and the table's rows are copied as far as they stay.
__global__ __launch_bounds__(256) void k_kv_release(KvTable t, const int32_t* wanted, int32_t* refs, int pages, int32_t* out) {
  const int r = blockIdx.x;
  const Change c = change_of(t, wanted, r);
  for (int j = threadIdx.x; j < t.width; j += 256) {
    const int e = j < c.old_n ? entry(t, r, j) : -1;
    gst<int32_t>(out + (int64_t)r * t.width + j, j < c.new_n ? e : -1);
    if (j >= c.new_n && in_pool(e, pages)) atomicAdd(refs + e, -1);
  }
}

// Pages p .. p + 3's counts; 1 behind the last page.
__device__ __forceinline__ v4i counts4(const int32_t* refs, int64_t p, int pages) {
  if (p + 4 <= pages) {
    const v4u w = load_live(refs + p);
    return v4i{(int)w.x, (int)w.y, (int)w.z, (int)w.w};
  }
  v4i r;
#pragma unroll
  for (int i = 0; i < 4; ++i) r[i] = p + i < pages ? gld<int32_t>(refs + p + i) : 1;
  return r;
}

// Second, one work-group: how many pages each row takes, which are free, who gets any.
// out_ready (or null): the new length of a row that has what it wants, 0 of one that was refused.
__global__ __launch_bounds__(1024) void k_kv_plan(KvTable t, const int32_t* wanted, const int32_t* refs, int pages, KvPlan plan,
                                                  int32_t* out_len, int32_t* out_ready, int32_t* out_short) {
  __shared__ int64_t scan64[16];
  __shared__ int scan[16];
  __shared__ int64_t carry;
  __shared__ int pairs;
  const int tid = threadIdx.x;
  if (tid == 0) carry = 0, pairs = 0;
  __syncthreads();
  // a row that grows from inside a page that others hold as well takes one to copy it to
  auto need_of = [&](int64_t r, const Change& c, bool& copy) {
    copy = false;
    if (c.want > c.len && (c.len & ((1 << t.shift) - 1)) != 0) {
      const int e = entry(t, r, c.old_n - 1);
      copy = in_pool(e, pages) && gld<int32_t>(refs + e) > 1;
    }
    return (c.new_n > c.old_n ? c.new_n - c.old_n : 0) + (copy ? 1 : 0);
  };
  for (int64_t r0 = 0; r0 < t.rows; r0 += 1024) {
    const int64_t r = r0 + tid;
    int need = 0;
    bool copy = false;
    if (r < t.rows) need = need_of(r, change_of(t, wanted, r), copy);
    const int64_t base = carry;
    const int64_t after = base + block_scan<1024, int64_t>(need, scan64);
    if (r < t.rows) gst<int64_t>(plan.after + r, after), gst<int32_t>(plan.need + r, copy ? -need : need);
    if (tid == 1023) carry = after;
    __syncthreads();
  }
  const int64_t total = carry;
  // the lowest free pages, as many as are wanted: a thread has four next to each other
  int64_t found = 0;
  for (int64_t p0 = 0; p0 < pages && found < total; p0 += 4096) {
    const int64_t p = p0 + 4 * tid;
    const v4i r = counts4(refs, p, pages);
    const int mine = (r.x <= 0) + (r.y <= 0) + (r.z <= 0) + (r.w <= 0);
    int64_t at = found + block_scan<1024, int>(mine, scan) - mine;
    if (tid == 1023) carry = at + mine;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (r[i] <= 0) {
        if (at < total && at < plan.capacity) gst<int32_t>(plan.free + at, (int32_t)(p + i));
        ++at;
      }
    __syncthreads();
    found = carry;
    __syncthreads();
  }
  if (found > plan.capacity) found = plan.capacity;
  if (tid == 0) gst<int32_t>(out_short, (int32_t)(total > found ? total - found : 0));
  // the list is read by other threads than wrote it
  __threadfence_block();
  __syncthreads();
  for (int64_t r = tid; r < t.rows; r += 1024) {
    const Change c = change_of(t, wanted, r);
    const int64_t after = gld<int64_t>(plan.after + r);
    const int signed_need = gld<int32_t>(plan.need + r), need = signed_need < 0 ? -signed_need : signed_need;
    const bool granted = need == 0 || after <= found;
    const int32_t now = (int32_t)(granted || c.want <= c.len ? c.want : c.len);
    gst<int32_t>(out_len + r, now);
    if (out_ready != nullptr) gst<int32_t>(out_ready + r, now == gld<int32_t>(wanted + r) ? now : 0);
    if (!granted) gst<int32_t>(plan.need + r, 0);
    if (granted && signed_need < 0) {
      const int at = atomicAdd(&pairs, 1);
      gst<int32_t>(plan.pairs + 2 * at, entry(t, r, c.old_n - 1));
      gst<int32_t>(plan.pairs + 2 * at + 1, gld<int32_t>(plan.free + after - need));
    }
  }
  __syncthreads();
  if (tid == 0) gst<int32_t>(plan.count, pairs);
}

// Third: rows take their pages, and pages that they must not share are copied.
__global__ __launch_bounds__(256) void k_kv_take(KvTable t, KvPool c, KvPlan plan, int32_t* out) {
  for (int64_t r = blockIdx.x; r < t.rows; r += gridDim.x) {
    const int signed_need = gld<int32_t>(plan.need + r);
    if (signed_need == 0) continue;
    const bool copy = signed_need < 0;
    const int need = copy ? -signed_need : signed_need;
    const int64_t begin = gld<int64_t>(plan.after + r) - need;
    const int old_n = pages_of(clamp_len(gld<int32_t>(t.lengths + r), t), t.shift);
    for (int i = threadIdx.x; i < need; i += 256) {
      const int p = gld<int32_t>(plan.free + begin + i);
      gst<int32_t>(c.refs + p, 1);
      gst<int32_t>(out + r * t.width + old_n + i - (copy ? 1 : 0), p);
    }
    if (copy && threadIdx.x == 0) atomicAdd(c.refs + entry(t, r, old_n - 1), -1);
  }
  const int64_t count = gld<int32_t>(plan.count);
  if (count > 0) copy_pages<false>(c, plan.pairs, count);
}

// ---------------------------------------------------------------------------
// compact
// ---------------------------------------------------------------------------
// First, one work-group: with n pages in use, the k-th of them at or behind n moves to the
// k-th free one before n.  map[p] is the new place of page p, for p at or behind n.
//
// A thread has four pages next to each other at a time; the first kHeldRounds rounds' counts
// stay in registers from the first pass (how many are in use) to the second (which move where),
// whose sums hold strays in their lower half and holes in their upper.
constexpr int kHeldRounds = 4;
__global__ __launch_bounds__(1024) void k_kv_gather(int32_t* refs, int pages, KvPlan plan, int32_t* out_count) {
  __shared__ uint32_t scan[16];
  __shared__ uint32_t carry[2];
  const int tid = threadIdx.x;
  int held[kHeldRounds][4];
  auto look = [&](int64_t p0, int (&r)[4]) {
    const v4i w = counts4(refs, p0 + 4 * tid, pages);
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = p0 + 4 * tid + i < pages ? w[i] : 0;
  };
  uint32_t live = 0;
#pragma unroll
  for (int k = 0; k < kHeldRounds; ++k)
    if (4096 * k < pages) look(4096 * k, held[k]);
#pragma unroll
  for (int k = 0; k < kHeldRounds; ++k)
    if (4096 * k < pages)
#pragma unroll
      for (int i = 0; i < 4; ++i) live += held[k][i] > 0;
  for (int64_t p0 = 4096 * kHeldRounds; p0 < pages; p0 += 4096) {
    int r[4];
    look(p0, r);
#pragma unroll
    for (int i = 0; i < 4; ++i) live += r[i] > 0;
  }
  const int n = (int)block_sum<16>(live, scan);
  if (tid < 2) carry[tid] = 0;
  __syncthreads();
  auto place = [&](int64_t p0, const int (&r)[4]) {
    uint32_t mine = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int64_t p = p0 + 4 * tid + i;
      mine += p < n ? (r[i] > 0 ? 0u : 0x10000u) : (r[i] > 0 ? 1u : 0u);
    }
    const uint32_t upto = block_scan<1024, uint32_t>(mine, scan), first = upto - mine;
    uint32_t stray = carry[0] + (first & 0xFFFF), hole = carry[1] + (first >> 16);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int64_t p = p0 + 4 * tid + i;
      if (p >= pages) continue;
      if (r[i] <= 0) gst<int32_t>(refs + p, 0);
      if (p < n) {
        if (r[i] <= 0) gst<int32_t>(plan.pairs + 2 * (int64_t)hole++ + 1, (int32_t)p);
      } else if (r[i] > 0) {
        gst<int32_t>(plan.pairs + 2 * (int64_t)stray++, (int32_t)p);
      } else {
        gst<int32_t>(plan.free + p, (int32_t)p);
      }
    }
    __syncthreads();
    if (tid == 1023) carry[0] += upto & 0xFFFF, carry[1] += upto >> 16;
    __syncthreads();
  };
#pragma unroll
  for (int k = 0; k < kHeldRounds; ++k)
    if (4096 * k < pages) place(4096 * k, held[k]);
  for (int64_t p0 = 4096 * kHeldRounds; p0 < pages; p0 += 4096) {
    int r[4];
    look(p0, r);
    place(p0, r);
  }
  __threadfence_block();
  __syncthreads();
  const int moves = (int)carry[0];
  for (int i = tid; i < moves; i += 1024) {
    const int from = gld<int32_t>(plan.pairs + 2 * (int64_t)i), to = gld<int32_t>(plan.pairs + 2 * (int64_t)i + 1);
    gst<int32_t>(plan.free + from, to);
    gst<int32_t>(refs + to, gld<int32_t>(refs + from));
    gst<int32_t>(refs + from, 0);
  }
  if (tid == 0) gst<int32_t>(plan.count, moves), gst<int32_t>(plan.count + 1, n), gst<int32_t>(out_count, n);
}

// Second: the table's entries get their pages' new numbers, and the pages' data moves.
__global__ __launch_bounds__(256) void k_kv_move(KvTable t, KvPool c, KvPlan plan, int32_t* out) {
  const int64_t count = gld<int32_t>(plan.count);
  const int n = gld<int32_t>(plan.count + 1);
  const int64_t cells = (int64_t)t.rows * t.width;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < cells; i += (int64_t)gridDim.x * 256) {
    const int64_t r = i / t.width;
    const int e = entry(t, r, (int)(i - r * t.width));
    gst<int32_t>(out + i, in_pool(e, c.pages) && e >= n ? gld<int32_t>(plan.free + e) : e);
  }
  if (count > 0) copy_pages<true>(c, plan.pairs, count);
}

constexpr unsigned kCopyGroups = 2048;

}  // namespace

hipError_t launch_kv_fork(const KvTable& t, const int32_t* parents, int32_t* refs, int pages, int32_t* out, int32_t* out_len,
                          hipStream_t stream) {
  hipLaunchKernelGGL(k_kv_fork, dim3((unsigned)t.rows), dim3(256), 0, stream, t, parents, refs, pages, out, out_len);
  return hipGetLastError();
}

// The plan's workspace: after [rows] int64, need [rows], pairs, free [pages], count [2].
static int64_t pad256(int64_t n) { return (n + 255) / 256 * 256; }
int64_t kv_resize_workspace(int64_t rows, int64_t pages) {
  return pad256(8 * rows) + pad256(4 * rows) + pad256(8 * rows) + pad256(4 * pages) + 256;
}
int64_t kv_compact_workspace(int64_t pages) { return pad256(8 * pages) + pad256(4 * pages) + 256; }

hipError_t launch_kv_resize(const KvTable& t, const KvPool& c, const int32_t* wanted, int32_t* out, int32_t* out_len,
                            int32_t* out_ready, int32_t* out_short, void* workspace, hipStream_t stream) {
  uint8_t* w = static_cast<uint8_t*>(workspace);
  KvPlan plan{};
  plan.after = reinterpret_cast<int64_t*>(w), w += pad256(8 * (int64_t)t.rows);
  plan.need = reinterpret_cast<int32_t*>(w), w += pad256(4 * (int64_t)t.rows);
  plan.pairs = reinterpret_cast<int32_t*>(w), w += pad256(8 * (int64_t)t.rows);
  plan.free = reinterpret_cast<int32_t*>(w), w += pad256(4 * (int64_t)c.pages);
  plan.count = reinterpret_cast<int32_t*>(w);
  plan.capacity = c.pages;
  if (t.rows > 0) hipLaunchKernelGGL(k_kv_release, dim3((unsigned)t.rows), dim3(256), 0, stream, t, wanted, c.refs, c.pages, out);
  hipLaunchKernelGGL(k_kv_plan, dim3(1), dim3(1024), 0, stream, t, wanted, c.refs, c.pages, plan, out_len, out_ready,
                     out_short);
  hipLaunchKernelGGL(k_kv_take, dim3(kCopyGroups), dim3(256), 0, stream, t, c, plan, out);
  return hipGetLastError();
}

hipError_t launch_kv_compact(const KvTable& t, const KvPool& c, int32_t* out, int32_t* out_count, void* workspace,
                             hipStream_t stream) {
  uint8_t* w = static_cast<uint8_t*>(workspace);
  KvPlan plan{};
  plan.pairs = reinterpret_cast<int32_t*>(w), w += pad256(8 * (int64_t)c.pages);
  plan.free = reinterpret_cast<int32_t*>(w), w += pad256(4 * (int64_t)c.pages);
  plan.count = reinterpret_cast<int32_t*>(w);
  plan.capacity = c.pages;
  hipLaunchKernelGGL(k_kv_gather, dim3(1), dim3(1024), 0, stream, c.refs, c.pages, plan, out_count);
  hipLaunchKernelGGL(k_kv_move, dim3(kCopyGroups), dim3(256), 0, stream, t, c, plan, out);
  return hipGetLastError();
}

}  // namespace lrq
