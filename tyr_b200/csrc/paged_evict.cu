// Eviction from a paged KV cache by accumulated attention weight: per (sequence, KV head) the first n_sink and the last
// n_recent keys stay, and of the others those with the greatest sums of weights, up to n_keep keys in all.
//
// Two launches:
//   evict_select_kernel : one CTA per (sequence, KV head) finds the weight T of the last key that stays by radix selection
//                         (four passes over 8 bits of the weights' order-preserving integers), then one pass in the order
//                         of the positions writes the list of the kept ones and moves their weights.  Of the keys
//                         that weigh exactly T the lower positions stay.
//   evict_move_kernel   : moves the kept K and V rows to the front.  A kept key's new row is at most its old one, so a
//                         CTA that walks the list forward may move in place: every row of a step is in registers
//                         before the step's first store, and what a step writes lies below what later steps read.  Different
//                         columns of a row do not meet, so the columns are spread over CTAs.
#include <cuda_bf16.h>

#include <algorithm>

#include "attn_internal.h"
#include "fast_div.h"
#include "ptx_sm100.cuh"

namespace tyr {
namespace {

constexpr int kMoveThreads = 256;

struct EvictParams {
  __nv_bfloat16 *k, *v;
  const int32_t* table;
  int64_t table_stride;
  FastDiv by_page;
  int n_pages, max_pages;
  const int32_t* kv_lens;
  float* weights;
  int64_t w_stride_b, w_stride_h;
  int32_t *new_lens, *kept;
  int n_kv_head, max_len, n_keep, n_recent, n_sink;
  int64_t ks[3], vs[3];  // page, head, row
  int* status;
};

// Integers in the order of the floats; both zeros are one, a NaN comes before every number.
__device__ __forceinline__ uint32_t ordered(float x) {
  if (x != x) return 0u;
  const uint32_t u = __float_as_uint(x + 0.0f);  // -0 + 0 = +0
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

// Positions a thread holds at once: position k * kThreads + thread as item k.  kAhead of them are fetched before the length is known.
constexpr int kItems = 16, kAhead = 4;

template <int kThreads>
__global__ void __launch_bounds__(kThreads, 1024 / kThreads) evict_select_kernel(const EvictParams p) {
  constexpr int kSegment = kItems * kThreads;
  __shared__ uint32_t hist[256];
  __shared__ uint32_t counts[kItems * kThreads / 32];  // per item and warp, in the order of the positions: over, equal << 16
  __shared__ uint32_t warp_sums[kThreads / 32];
  __shared__ uint32_t sel_digit, sel_left;
  grid_launch_dependents();
  grid_dependency_wait();
  const int hkv = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  float* w = p.weights + b * p.w_stride_b + hkv * p.w_stride_h;
  // a segment's weights stay in registers over all passes where there is only one (the array has max_len entries)
  float x[kItems];
#pragma unroll
  for (int k = 0; k < kItems; ++k) {
    const int i = k * kThreads + tid;
    x[k] = k < kAhead && i < p.max_len ? w[i] : 0.f;
  }
  const int raw = p.kv_lens[b], n = min(max(raw, 0), p.max_len);
  int32_t* kept = p.kept + ((int64_t)b * p.n_kv_head + hkv) * p.n_keep;
  if (hkv == 0 && tid == 0) {
    if (raw != n) atomicOr(p.status, kStatusOutOfRange);
    p.new_lens[b] = min(n, p.n_keep);
  }
  if (n <= p.n_keep) {  // within the budget
    for (int i = tid; i < p.n_keep; i += kThreads) kept[i] = i < n ? i : -1;
    return;
  }
  const int lo = p.n_sink, hi = n - p.n_recent;        // the candidates' positions
  const uint32_t m = p.n_keep - p.n_sink - p.n_recent;  // how many of them stay: fewer than there are
  auto load = [&](int i0, int k0) {
#pragma unroll
    for (int k = 0; k < kItems; ++k) {
      if (k < k0) continue;
      const int i = i0 + k * kThreads + tid;
      x[k] = i < n ? w[i] : 0.f;
    }
  };
  const bool one_segment = n <= kSegment;
  load(0, kAhead);
  // T: the m-th greatest; `left`: how many of the keys equal to it stay
  uint32_t T = 0xffffffffu, left = 0;
  if (m > 0) {
    T = 0;
    left = m;
    for (int shift = 24; shift >= 0; shift -= 8) {
      if (tid < 256) hist[tid] = 0;
      __syncthreads();
      const uint32_t above = shift == 24 ? 0u : 0xffffffffu << (shift + 8);
      for (int i0 = 0; i0 < hi; i0 += kSegment) {
        if (!one_segment) load(i0, 0);
#pragma unroll
        for (int k = 0; k < kItems; ++k) {
          const int i = i0 + k * kThreads + tid;
          if (i0 + k * kThreads >= hi) break;
          const uint32_t u = ordered(x[k]);
          if (i >= lo && i < hi && (u & above) == T) atomicAdd(&hist[(u >> shift) & 255u], 1u);
        }
      }
      __syncthreads();
      if (tid < 32) {
        // lane l has digits 255 - 8 l .. 248 - 8 l: the greatest first
        uint32_t c[8], sum = 0;
#pragma unroll
        for (int d = 0; d < 8; ++d) {
          c[d] = hist[255 - 8 * tid - d];
          sum += c[d];
        }
        uint32_t before = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const uint32_t y = __shfl_up_sync(0xffffffffu, before, o);
          if (tid >= o) before += y;
        }
        before -= sum;
#pragma unroll
        for (int d = 0; d < 8; ++d) {
          if (before < left && before + c[d] >= left) {
            sel_digit = 255 - 8 * tid - d;
            sel_left = left - before;
          }
          before += c[d];
        }
      }
      __syncthreads();
      T |= sel_digit << shift;
      left = sel_left;
    }
  }
  // in the order of the positions: a key stays if it always does, weighs more than T, or is one of the first `left` equal to T
  uint32_t over_before = 0, equal_before = 0;
  for (int i0 = 0; i0 < n; i0 += kSegment) {
    if (!one_segment) load(i0, 0);
    uint32_t over_bits = 0, equal_bits = 0;  // of this thread's items
#pragma unroll
    for (int k = 0; k < kItems; ++k) {
      const int i = i0 + k * kThreads + tid;
      if (i0 + k * kThreads >= n) {
        if (lane == 0) counts[k * (kThreads / 32) + warp] = 0u;
        continue;
      }
      const uint32_t u = ordered(x[k]);
      const bool candidate = i >= lo && i < hi;
      const bool over = i < lo || (i >= hi && i < n) || (candidate && u > T), equal = candidate && u == T;
      over_bits |= (uint32_t)over << k;
      equal_bits |= (uint32_t)equal << k;
      const uint32_t c = __popc(__ballot_sync(0xffffffffu, over)) | __popc(__ballot_sync(0xffffffffu, equal)) << 16;
      if (lane == 0) counts[k * (kThreads / 32) + warp] = c;
    }
    __syncthreads();  // every weight of the segment is in a register, every count in shared memory
    // exclusive prefix sums of the counts (at most kSegment of either kind: 16 bits each)
    constexpr int kCounts = kItems * kThreads / 32;
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
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kItems; ++k) {
      if (i0 + k * kThreads >= n) break;
      const bool over = (over_bits >> k) & 1u, equal = (equal_bits >> k) & 1u;
      const uint32_t lower = (1u << lane) - 1u, c = counts[k * (kThreads / 32) + warp];
      const uint32_t over_at = over_before + (c & 0xffffu) + __popc(__ballot_sync(0xffffffffu, over) & lower);
      const uint32_t equal_at = equal_before + (c >> 16) + __popc(__ballot_sync(0xffffffffu, equal) & lower);
      if (over || (equal && equal_at < left)) {
        const uint32_t to = over_at + min(equal_at, left);
        kept[to] = i0 + k * kThreads + tid;
        w[to] = x[k];  // (at most the key's own position)
      }
    }
    over_before += total & 0xffffu;
    equal_before += total >> 16;
    __syncthreads();  // (the counts are the next segment's)
  }
  for (int i = p.n_keep + tid; i < n; i += kThreads) w[i] = 0.f;
}

// kLanes threads of 16 bytes make one row of a CTA's columns; kRows rows of each thread are in flight, and the next step's
// addresses (list entry, then table entry) are on their way while a step's rows arrive.
template <int kLanes>
__global__ void __launch_bounds__(kMoveThreads) evict_move_kernel(const EvictParams p, int slices) {
  constexpr int kRows = 8, kGroup = kMoveThreads / kLanes, kStep = kRows * kGroup;  // kStep: rows a step moves
  grid_launch_dependents();
  grid_dependency_wait();
  const int hkv = blockIdx.y, b = blockIdx.z, tid = threadIdx.x;
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

// The columns of a row that one CTA moves: 128 bytes, or 32 where those CTAs would not fill the SMs.
template <int kLanes>
cudaError_t launch_move(const EvictParams& p, int batch, int head_dim, cudaStream_t st) {
  const int slices = head_dim / (8 * kLanes);
  return launch_overlapped(evict_move_kernel<kLanes>, dim3(2 * slices, p.n_kv_head, batch), dim3(kMoveThreads), 0, st, 1, p, slices);
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
  p.max_pages = a.pages.max_pages;
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
  // Half as many threads, two CTAs per SM, while they hold a sequence: 64 sequences of 1000 keys, 8 KV heads, both launches
  // 56.9 -> 47.1 us, one of 2049 11.1 -> 10.4; with half as many for 32 sequences of up to 16 K 155.8 -> 161.9.
  const bool few = a.max_kv_seq <= kItems * 512;
  cudaError_t e = launch_overlapped(few ? evict_select_kernel<512> : evict_select_kernel<1024>, dim3(a.n_kv_head, a.batch),
                                    dim3(few ? 512 : 1024), 0, st, 1, p);
  count_launch();
  if (e == cudaSuccess) e = cudaGetLastError();
  if (e != cudaSuccess) return (int)e;
  const bool wide = 2ll * (a.head_dim / 64) * a.n_kv_head * a.batch >= 2ll * sm_count();
  e = wide ? launch_move<8>(p, a.batch, a.head_dim, st) : launch_move<2>(p, a.batch, a.head_dim, st);
  count_launch();
  return (int)(e != cudaSuccess ? e : cudaGetLastError());
}

}  // namespace tyr
