// Eviction from a paged KV cache by accumulated attention weight: per (sequence, KV head) the first n_sink and the last
// n_recent keys stay, and of the others those with the greatest sums of weights, up to n_keep keys in all.
//
// Cannot do without: one read and one write of every row that moves.  Figures here and below are of evictions with new weights each
// time and L2 cold, in which all but the first few rows move.  32 sequences of 2 K to 16 K keys down to 4096, 8 KV heads of 128: 926 MB
// in 237 us, 3.9 TB/s; the selection is 27 us of that, the move 203, 4.5 TB/s: before each step's rows stand two
// latencies, the list's entry and then the table's.  One short sequence is latency (2049 keys down to 1024 17 us, the selection 9, the
// move 8).  Evicting a cache again whose best keys lie in front already moves the recent ones alone: 157 and 15 us.
//
// Two launches:
//   evict_select_kernel : one CTA or cluster of CTAs per (sequence, KV head) finds the weight T of the last key that stays by radix selection
//                         (passes over digits of the weights' order-preserving integers), then one pass in the order
//                         of the positions writes the list of the kept ones and moves their weights.  Of the keys
//                         that weigh exactly T the lower positions stay.
//   evict_move_kernel   : moves the kept K and V rows to the front.  A kept key's new row is at most its old one, so a
//                         CTA that walks the list forward may move in place: every row of a step has been read before the
//                         step's first store, and what a step writes lies below what later steps read.  Different
//                         columns of a row do not meet, so the columns are spread over CTAs.  (evict_move_few_kernel: a launch of few.)
#include <cuda_bf16.h>

#include <algorithm>
#include <atomic>

#include "attn_internal.h"
#include "evict_plan.h"
#include "fast_div.h"
#include "mma_sync.cuh"
#include "ptx_sm100.cuh"

namespace tyr {
namespace {

constexpr int kMoveThreads = 256;

struct EvictParams {
  __nv_bfloat16 *k, *v;
  const int32_t* table;
  int64_t table_stride;
  FastDiv by_page;
  int n_pages;
  const int32_t* kv_lens;
  float* weights;
  int64_t w_stride_b, w_stride_h;
  int32_t *new_lens, *kept;
  int n_kv_head, max_len, n_keep, n_recent, n_sink;
  int64_t ks[3], vs[3];  // page, head, row
  int ranks;             // CTAs of a cluster that share a (sequence, KV head)
  int* status;
};

// Integers in the order of the floats; both zeros are one, a NaN comes before every number.
__device__ __forceinline__ uint32_t ordered(float x) {
  if (x != x) return 0u;
  const uint32_t u = __float_as_uint(x + 0.0f);  // -0 + 0 = +0
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

// Positions a thread holds at once: position k * kThreads + thread as item k.
constexpr int kItems = 16, kAhead = 4;
// kCluster: the CTAs of a cluster share the (sequence, KV head), a segment of kItems * kThreads positions each, so that a
// long sequence's weights stay in registers too; the histograms and counts are added through distributed shared memory.  The launch
// goes by the greatest length there can be; CTAs behind a sequence's last key leave at once (four sequences of 2000 keys
// in a cache of 131072 80 -> 29 us, in one of 2000 23).
// Otherwise one CTA, which reads the weights again in every pass where they are more than a segment.
// kBits: of a digit; the first digit of 11 has the sign, the exponent and two bits of the mantissa, of 8, which weights fill half a
// dozen values of, it has most of the exponent.  Three passes of 11 bits are faster where there are many keys, four of 8, with an
// eighth of the bins to clear and to add up, where there are few (the launch says which).
template <int kThreads, bool kCluster, int kBits>
__global__ void __launch_bounds__(kThreads, 1024 / kThreads) evict_select_kernel(const EvictParams p) {
  constexpr int kSegment = kItems * kThreads, kWarps = kThreads / 32, kBins = 1 << kBits, kPasses = (32 + kBits - 1) / kBits;
  __shared__ __align__(16) uint32_t hist[2][kBins];             // of this CTA, alternating from pass to pass
  __shared__ uint32_t counts[kItems * kWarps];  // per item and warp, in the order of the positions: over, equal << 16
  __shared__ uint32_t warp_sums[kWarps], bin_sums[(kBins / 8 + 31) / 32];
  __shared__ uint32_t sel_digit, sel_left, own_total;
  grid_launch_dependents();
  grid_dependency_wait();
  const int rank = kCluster ? (int)cluster_rank() : 0;
  int ranks = kCluster ? p.ranks : 1;
  const int hkv = kCluster ? blockIdx.x / ranks : blockIdx.x, b = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  float* w = p.weights + b * p.w_stride_b + hkv * p.w_stride_h;
  const int i_own = rank * kSegment;              // the first position of this CTA's (first) segment
  uint32_t u[kItems];
#pragma unroll
  for (int k = 0; k < kAhead; ++k) {  // on their way while the length is fetched (the array has max_len entries)
    const int i = i_own + k * kThreads + tid;
    u[k] = i < p.max_len ? __float_as_uint(w[i]) : 0u;
  }
  for (int q = tid; q < kBins / 4; q += kThreads) reinterpret_cast<uint4*>(hist[0])[q] = make_uint4(0u, 0u, 0u, 0u);
  const int raw = p.kv_lens[b], n = min(max(raw, 0), p.max_len);
  int32_t* kept = p.kept + ((int64_t)b * p.n_kv_head + hkv) * p.n_keep;
  if (hkv == 0 && rank == 0 && tid == 0) {
    if (raw != n) atomicOr(p.status, kStatusOutOfRange);
    p.new_lens[b] = min(n, p.n_keep);
  }
  if (n <= p.n_keep) {  // within the budget (the whole cluster)
    for (int i = rank * kThreads + tid; i < p.n_keep; i += ranks * kThreads) kept[i] = i < n ? i : -1;
    return;
  }
  if (kCluster) {
    ranks = (n + kSegment - 1) / kSegment;
    if (rank >= ranks) return;  // (a cluster's barriers wait for the threads that have not exited)
  }
  // The weights as integers in their order; what always stays is above all of them, and what lies behind the last
  // position is 0 like a NaN, whose equals before it are enough.  A segment's stay in registers over all passes.
  const int lo = p.n_sink, hi = n - p.n_recent;
  auto load = [&](int i0, int k0) {
#pragma unroll
    for (int k = 0; k < kItems; ++k) {
      const int i = i0 + k * kThreads + tid;
      if (k >= k0) u[k] = i < n ? __float_as_uint(w[i]) : 0u;
    }
#pragma unroll
    for (int k = 0; k < kItems; ++k) {
      if (i0 + k * kThreads >= n) break;
      const int i = i0 + k * kThreads + tid;
      u[k] = i >= n ? 0u : i < lo || i >= hi ? 0xffffffffu : ordered(__uint_as_float(u[k]));
    }
  };
  const bool held = kCluster || n <= kSegment;    // every weight is in its thread's registers
  const int i_end = kCluster ? min(n, i_own + kSegment) : n;
  load(i_own, kAhead);
  // T: the n_keep-th greatest; `left`: how many of those equal to it stay
  uint32_t T = 0, left = p.n_keep;
  __syncthreads();
  for (int pass = 0; pass < kPasses; ++pass) {
    const int shift = max(32 - kBits * (pass + 1), 0);  // (the last digit may be shorter)
    const uint32_t above = pass == 0 ? 0u : 0xffffffffu << (32 - kBits * pass), digits = ~above >> shift;
    uint32_t* own = hist[pass & 1];
    for (int i0 = i_own; i0 < i_end; i0 += kSegment) {
      if (!held) load(i0, 0);
#pragma unroll
      for (int k = 0; k < kItems; ++k) {
        if (i0 + k * kThreads >= n) break;
        if ((u[k] & above) == T) atomicAdd(&own[(u[k] >> shift) & digits], 1u);
      }
    }
    // Behind this barrier every CTA has read the other histogram (it belongs to the pass before): it is the next pass's.
    if (kCluster) cluster_sync();
    else __syncthreads();
    // thread t has digits kBins - 1 - 8 t .. kBins - 8 - 8 t: the greatest first
    uint32_t c[8], sum = 0, before = 0;
    if (tid < kBins / 8) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t at = smem_u32(&own[kBins - 8 - 8 * tid + 4 * (1 - h)]);
        uint4 v = make_uint4(0u, 0u, 0u, 0u);
        for (int r = 0; r < ranks; ++r) {
          const uint4 y = kCluster ? cluster_ld_u32x4(cluster_map(at, r)) : *reinterpret_cast<const uint4*>(&own[kBins - 8 - 8 * tid + 4 * (1 - h)]);
          v.x += y.x;
          v.y += y.y;
          v.z += y.z;
          v.w += y.w;
        }
        c[4 * h] = v.w;
        c[4 * h + 1] = v.z;
        c[4 * h + 2] = v.y;
        c[4 * h + 3] = v.x;
      }
#pragma unroll
      for (int d = 0; d < 8; ++d) sum += c[d];
      before = sum;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t y = __shfl_up_sync(0xffffffffu, before, o);
        if (lane >= o) before += y;
      }
      if (lane == 31) bin_sums[warp] = before;
      before -= sum;
    } else {
      for (int q = tid - kBins / 8; q < kBins / 4; q += kThreads - kBins / 8)
        reinterpret_cast<uint4*>(hist[(pass & 1) ^ 1])[q] = make_uint4(0u, 0u, 0u, 0u);
    }
    if (kBins / 8 > 32) __syncthreads();
    if (tid < kBins / 8) {
      for (int v = 0; v < warp; ++v) before += bin_sums[v];
#pragma unroll
      for (int d = 0; d < 8; ++d) {
        if (before < left && before + c[d] >= left) {
          sel_digit = kBins - 1 - 8 * tid - d;
          sel_left = left - before;
        }
        before += c[d];
      }
    }
    __syncthreads();
    T |= sel_digit << shift;
    left = sel_left;
    // (sel_* and bin_sums are written again only behind the next pass's first barrier)
  }
  // in the order of the positions: a key stays if it is above T, or one of the first `left` equal to T
  uint32_t over_before = 0, equal_before = 0;
  for (int i0 = i_own; kCluster ? i0 == i_own : i0 < n; i0 += kSegment) {
    if (!held) load(i0, 0);
    uint32_t over_bits = 0, equal_bits = 0;  // of this thread's items
#pragma unroll
    for (int k = 0; k < kItems; ++k) {
      if (i0 + k * kThreads >= n) {
        if (lane == 0) counts[k * kWarps + warp] = 0u;
        continue;
      }
      const int i = i0 + k * kThreads + tid;
      const bool over = u[k] > T, equal = u[k] == T;
      over_bits |= (uint32_t)over << k;
      equal_bits |= (uint32_t)equal << k;
      const uint32_t c = __popc(__ballot_sync(0xffffffffu, over)) | __popc(__ballot_sync(0xffffffffu, equal)) << 16;
      if (lane == 0) counts[k * kWarps + warp] = c;
      if ((over || equal) && i < n) u[k] = __float_as_uint(w[i]);  // the weight itself, its bits as they are
    }
    __syncthreads();
    // exclusive prefix sums of the counts (at most kSegment of either kind: 16 bits each)
    constexpr int kCounts = kItems * kWarps;
    static_assert(kCounts <= kThreads && kSegment < 65536, "one count per thread");
    const uint32_t mine = tid < kCounts ? counts[tid] : 0u;
    uint32_t sum = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t y = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += y;
    }
    if (lane == 31) warp_sums[warp] = sum;
    __syncthreads();
    uint32_t base = 0, total = 0;
#pragma unroll
    for (int v = 0; v < kCounts / 32; ++v) {
      base += v < warp ? warp_sums[v] : 0u;
      total += warp_sums[v];
    }
    if (tid < kCounts) counts[tid] = base + sum - mine;
    // Behind this barrier every weight of the segment (of the sequence, in a cluster) that stays is in a register: what is
    // written below may be another thread's position.
    if (kCluster) {
      if (tid == 0) own_total = total;
      cluster_sync();
      for (int r = 0; r < rank; ++r) {
        const uint32_t t = cluster_ld_u32(cluster_map(smem_u32(&own_total), r));
        over_before += t & 0xffffu;
        equal_before += t >> 16;
      }
    } else {
      __syncthreads();
    }
#pragma unroll
    for (int k = 0; k < kItems; ++k) {
      if (i0 + k * kThreads >= n) break;
      const bool over = (over_bits >> k) & 1u, equal = (equal_bits >> k) & 1u;
      const uint32_t lower = (1u << lane) - 1u, c = counts[k * kWarps + warp];
      const uint32_t over_at = over_before + (c & 0xffffu) + __popc(__ballot_sync(0xffffffffu, over) & lower);
      const uint32_t equal_at = equal_before + (c >> 16) + __popc(__ballot_sync(0xffffffffu, equal) & lower);
      if (over || (equal && equal_at < left)) {
        const uint32_t to = over_at + min(equal_at, left);
        kept[to] = i0 + k * kThreads + tid;
        w[to] = __uint_as_float(u[k]);  // (at most the key's own position)
      }
    }
    over_before += total & 0xffffu;
    equal_before += total >> 16;
    if (!kCluster) __syncthreads();  // (the counts are the next segment's)
  }
  for (int i = max(i_own, p.n_keep) + tid; i < i_end; i += kThreads) w[i] = 0.f;
  if (kCluster) cluster_sync();  // no CTA's shared memory goes away while another still reads it
}

// The columns of a row that one CTA moves, in lanes of 16 bytes.
constexpr int kLanes = 8, kFewLanes = 2;

// A step's rows come to shared memory asynchronously, two steps ahead of their stores.
struct MoveCfg {
  static constexpr int kRows = 4, kStages = 3;                    // rows of a thread in a step; steps in shared memory
  static constexpr int kGroup = kMoveThreads / kLanes, kStep = kRows * kGroup;  // kStep: rows a step moves
  static constexpr int kBufBytes = kStages * kRows * kMoveThreads * 16;
  static constexpr int kSmemBytes = kBufBytes + kStages * kStep * 8;
};
__global__ void __launch_bounds__(kMoveThreads) evict_move_kernel(const EvictParams p) {
  using C = MoveCfg;
  constexpr int kRows = C::kRows, kStages = C::kStages, kGroup = C::kGroup, kStep = C::kStep;
  extern __shared__ __align__(16) uint8_t smem[];
  uint4* buf = reinterpret_cast<uint4*>(smem);                               // [stage][row of the thread][thread]
  long long* to = reinterpret_cast<long long*>(smem + C::kBufBytes);         // [stage][row of the step]: where it goes, -1: nowhere
  grid_launch_dependents();
  grid_dependency_wait();
  const int hkv = blockIdx.y, b = blockIdx.z, tid = threadIdx.x, group = tid / kLanes, slices = gridDim.x / 2;
  const int n = min(max(p.kv_lens[b], 0), p.max_len);
  if (n <= p.n_keep) return;
  const bool is_v = (int)blockIdx.x >= slices;
  const int col = ((is_v ? blockIdx.x - slices : blockIdx.x) * kLanes + tid % kLanes) * 8;
  const int64_t st0 = is_v ? p.vs[0] : p.ks[0], st2 = is_v ? p.vs[2] : p.ks[2];
  __nv_bfloat16* base = (is_v ? p.v + hkv * p.vs[1] : p.k + hkv * p.ks[1]) + col;
  const int32_t* kept = p.kept + ((int64_t)b * p.n_kv_head + hkv) * p.n_keep;
  const int32_t* table = p.table + b * p.table_stride;
  const int n_steps = (p.n_keep + kStep - 1) / kStep;
  bool bad = false;
  auto fetch = [&](int step) {
    if (step < n_steps) {
      int src[kRows], page_from[kRows], page_to[kRows];
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
        const int i = step * kStep + r * kGroup + group;
        src[r] = i < p.n_keep ? kept[i] : i;
      }
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
        const int i = step * kStep + r * kGroup + group;
        page_from[r] = src[r] == i ? 0 : table[p.by_page.div(src[r])];  // (a row that stays where it is needs none)
        page_to[r] = src[r] == i ? 0 : table[p.by_page.div(i)];
      }
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
        const int i = step * kStep + r * kGroup + group;
        const bool out = (unsigned)page_from[r] >= (unsigned)p.n_pages || (unsigned)page_to[r] >= (unsigned)p.n_pages;  // not followed
        const bool moves = src[r] != i && !out;
        bad = bad || (src[r] != i && out);
        if (moves)
          cp_async16(smem_u32(&buf[(step % kStages * kRows + r) * kMoveThreads + tid]),
                     base + page_from[r] * st0 + (src[r] - p.by_page.div(src[r]) * (int)p.by_page.d) * st2);
        if (tid % kLanes == 0)
          to[step % kStages * kStep + r * kGroup + group] =
              moves ? page_to[r] * st0 + (i - p.by_page.div(i) * (int)p.by_page.d) * st2 : -1;
      }
    }
    cp_async_commit();
  };
#pragma unroll
  for (int step = 0; step < kStages - 1; ++step) fetch(step);
  for (int step = 0; step < n_steps; ++step) {
    cp_async_wait<kStages - 2>();
    __syncthreads();  // every row of the step is in shared memory, and every store of the step before has read its rows there
    fetch(step + kStages - 1);  // (rows at or behind their own new places, which this step and the next do not write)
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      const long long at = to[step % kStages * kStep + r * kGroup + group];
      if (at >= 0) *reinterpret_cast<uint4*>(base + at) = buf[(step % kStages * kRows + r) * kMoveThreads + tid];
    }
  }
  if (bad) atomicOr(p.status, kStatusOutOfRange);
}

// For few (sequence, KV head) pairs: 32 bytes of a row per CTA, up to 1024 rows a step in registers; the next step's addresses (list
// entry, then table entry) are on their way while a step's rows arrive.
__global__ void __launch_bounds__(kMoveThreads) evict_move_few_kernel(const EvictParams p) {
  constexpr int kLanes = kFewLanes, kRows = 8, kGroup = kMoveThreads / kLanes, kStep = kRows * kGroup;  // kStep: rows a step moves
  grid_launch_dependents();
  grid_dependency_wait();
  const int hkv = blockIdx.y, b = blockIdx.z, tid = threadIdx.x, slices = gridDim.x / 2;
  const int n = min(max(p.kv_lens[b], 0), p.max_len);
  if (n <= p.n_keep) return;
  const bool is_v = (int)blockIdx.x >= slices;
  const int col = ((is_v ? blockIdx.x - slices : blockIdx.x) * kLanes + tid % kLanes) * 8;
  const int64_t st0 = is_v ? p.vs[0] : p.ks[0], st2 = is_v ? p.vs[2] : p.ks[2];
  __nv_bfloat16* base = (is_v ? p.v + hkv * p.vs[1] : p.k + hkv * p.ks[1]) + col;
  const int32_t* kept = p.kept + ((int64_t)b * p.n_kv_head + hkv) * p.n_keep;
  const int32_t* table = p.table + b * p.table_stride;
  bool bad = false;
  __nv_bfloat16 *from[kRows], *to[kRows];
  auto addresses = [&](int i0) {
    int src[kRows], page_from[kRows], page_to[kRows];
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      const int i = i0 + r * kGroup + tid / kLanes;
      src[r] = i < p.n_keep ? kept[i] : i;
    }
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      const int i = i0 + r * kGroup + tid / kLanes;
      page_from[r] = src[r] == i ? 0 : table[p.by_page.div(src[r])];  // (a row that stays where it is needs none)
      page_to[r] = src[r] == i ? 0 : table[p.by_page.div(i)];
    }
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      const int i = i0 + r * kGroup + tid / kLanes;
      const bool out = (unsigned)page_from[r] >= (unsigned)p.n_pages || (unsigned)page_to[r] >= (unsigned)p.n_pages;  // not followed
      bad = bad || (src[r] != i && out);
      from[r] = base + page_from[r] * st0 + (src[r] - p.by_page.div(src[r]) * (int)p.by_page.d) * st2;
      to[r] = src[r] == i || out ? nullptr : base + page_to[r] * st0 + (i - p.by_page.div(i) * (int)p.by_page.d) * st2;
    }
  };
  addresses(0);
  for (int i0 = 0; i0 < p.n_keep; i0 += kStep) {
    uint4 x[kRows];
    __nv_bfloat16* here[kRows];
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      here[r] = to[r];
      if (here[r] != nullptr) x[r] = *reinterpret_cast<const uint4*>(from[r]);
    }
    if (i0 + kStep < p.n_keep) addresses(i0 + kStep);
    __syncthreads();  // every row of the step is in registers
#pragma unroll
    for (int r = 0; r < kRows; ++r)
      if (here[r] != nullptr) *reinterpret_cast<uint4*>(here[r]) = x[r];
  }
  if (bad) atomicOr(p.status, kStatusOutOfRange);
}

// 128 bytes of a row per CTA, or 32 where those CTAs would be fewer than two per SM.  Both launches with the former kernel / the latter,
// us, 8 KV heads of 128: one sequence of 2049 keys to 1024 29.7 / 17.4, of 8192 to 4096 76.8 / 33.8, of 100000 to 16384 294 / 120; sequences of
// 4096 to 2048, four 50.0 / 35.8, nine 72.8 / 58.3, ten (the line) 74.8 / 64.5, twelve 74.7 / 74.2, sixteen 74.8 / 89.1;
// of 1000 to 500, ten 25.6 / 27.6, sixteen 27.7 / 37.9, sixty-four 72.7 / 118; 32 of up to 16 K to 4096 238 / 276.
int launch_move(const EvictParams& p, int batch, int head_dim, cudaStream_t st) {
  static std::atomic<bool> set[64] = {};  // per device
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return (int)e;
  if (dev < 0 || dev >= 64) return (int)cudaErrorInvalidDevice;
  if (!set[dev].load(std::memory_order_acquire)) {
    e = cudaFuncSetAttribute(evict_move_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, MoveCfg::kSmemBytes);
    if (e != cudaSuccess) return (int)e;
    set[dev].store(true, std::memory_order_release);
  }
  const int slices = head_dim / (8 * kLanes), few_slices = head_dim / (8 * kFewLanes);
  if (2ll * slices * p.n_kv_head * batch >= 2ll * sm_count())
    e = launch_overlapped(evict_move_kernel, dim3(2 * slices, p.n_kv_head, batch), dim3(kMoveThreads), MoveCfg::kSmemBytes, st, 1, p);
  else
    e = launch_overlapped(evict_move_few_kernel, dim3(2 * few_slices, p.n_kv_head, batch), dim3(kMoveThreads), 0, st, 1, p);
  count_launch();
  return (int)(e != cudaSuccess ? e : cudaGetLastError());
}

// Clusters of 2^k CTAs of the selection that can be resident at once: depends on how the SMs are spread over the GPCs, asked for
// once per device.
int cluster_capacity(int dev, int k) {
  static std::atomic<int> known[64][kMaxEvictLog + 1] = {};  // per device; 0: not asked yet, else capacity + 1
  const int have = known[dev][k].load(std::memory_order_acquire);
  if (have > 0) return have - 1;
  auto* kernel = evict_select_kernel<1024, true, 11>;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = 1u << k;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(1u << k);
  cfg.blockDim = dim3(1024);
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  int n = 0;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess ||
      cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess) {
    cudaGetLastError();  // no clusters of this size then
    n = 0;
  }
  known[dev][k].store(n + 1, std::memory_order_release);
  return n;
}

}  // namespace

int launch_paged_evict(const TyrAttnEvictArgs& a, int* status, cudaStream_t st) {
  EvictParams p;
  p.k = static_cast<__nv_bfloat16*>(a.k);
  p.v = static_cast<__nv_bfloat16*>(a.v);
  p.table = a.pages.table;
  p.table_stride = a.pages.table_stride;
  p.by_page = make_fastdiv(a.pages.page_size);
  p.n_pages = a.pages.n_pages;
  p.kv_lens = a.kv_lens;
  p.weights = a.weights;
  p.w_stride_b = a.weights_stride[0];
  p.w_stride_h = a.weights_stride[1];
  p.new_lens = a.new_lens;
  p.kept = a.kept;
  p.n_kv_head = a.n_kv_head;
  p.max_len = a.max_kv_seq;
  p.n_keep = a.n_keep;
  p.n_recent = a.n_recent;
  p.n_sink = a.n_sink;
  for (int i = 0; i < 3; ++i) { p.ks[i] = a.k_stride[i]; p.vs[i] = a.v_stride[i]; }
  p.status = status;
  // Half as many threads, two CTAs per SM, while they hold a sequence (both launches, every pass with new weights: 64 sequences of 1000
  // keys, 8 KV heads of 128, 85 -> 73 us; for 32 sequences of up to 16 K half as many take 261 for 237), and digits of 8 bits there
  // (64 of 1000 with digits of 11 75).
  const int segment = kItems * 1024;
  const bool few = a.max_kv_seq <= kItems * 512;
  int dev = 0;
  if (cudaError_t got = cudaGetDevice(&dev); got != cudaSuccess) return (int)got;
  if (dev < 0 || dev >= 64) return (int)cudaErrorInvalidDevice;
  p.ranks = evict_ranks(a.max_kv_seq, segment, [&](int k) { return cluster_capacity(dev, k); });
  cudaError_t e;
  if (p.ranks > 1) {
    e = launch_overlapped(evict_select_kernel<1024, true, 11>, dim3(a.n_kv_head * p.ranks, a.batch), dim3(1024), 0, st, p.ranks, p);
  } else {
    e = launch_overlapped(few ? evict_select_kernel<512, false, 8> : evict_select_kernel<1024, false, 11>, dim3(a.n_kv_head, a.batch),
                          dim3(few ? 512 : 1024), 0, st, 1, p);
  }
  count_launch();
  if (e == cudaSuccess) e = cudaGetLastError();
  if (e != cudaSuccess) return (int)e;
  return launch_move(p, a.batch, a.head_dim, st);
}

}  // namespace tyr
