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

constexpr int kSelectThreads = 1024;
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

// Exclusive prefix sums of `x` over the CTA's threads, and the total.
__device__ __forceinline__ uint2 block_scan(uint2 x, uint2* warp_sums, uint2& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint2 s = x;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t a = __shfl_up_sync(0xffffffffu, s.x, o), b = __shfl_up_sync(0xffffffffu, s.y, o);
    if (lane >= o) {
      s.x += a;
      s.y += b;
    }
  }
  if (lane == 31) warp_sums[warp] = s;
  __syncthreads();
  uint2 base = make_uint2(0u, 0u);
  total = make_uint2(0u, 0u);
#pragma unroll 8
  for (int w = 0; w < kSelectThreads / 32; ++w) {
    const uint2 y = warp_sums[w];
    if (w < warp) {
      base.x += y.x;
      base.y += y.y;
    }
    total.x += y.x;
    total.y += y.y;
  }
  __syncthreads();  // the sums are the next call's
  return make_uint2(base.x + s.x - x.x, base.y + s.y - x.y);
}

__global__ void __launch_bounds__(kSelectThreads) evict_select_kernel(const EvictParams p) {
  __shared__ uint32_t hist[256];
  __shared__ uint2 warp_sums[kSelectThreads / 32];
  __shared__ uint32_t sel_digit, sel_left;
  grid_launch_dependents();
  grid_dependency_wait();
  const int hkv = blockIdx.x, b = blockIdx.y, tid = threadIdx.x;
  const int raw = p.kv_lens[b], n = min(max(raw, 0), p.max_len);
  int32_t* kept = p.kept + ((int64_t)b * p.n_kv_head + hkv) * p.n_keep;
  if (hkv == 0 && tid == 0) {
    if (raw != n) atomicOr(p.status, kStatusOutOfRange);
    p.new_lens[b] = min(n, p.n_keep);
  }
  if (n <= p.n_keep) {  // within the budget
    for (int i = tid; i < p.n_keep; i += kSelectThreads) kept[i] = i < n ? i : -1;
    return;
  }
  float* w = p.weights + b * p.w_stride_b + hkv * p.w_stride_h;
  const int lo = p.n_sink, hi = n - p.n_recent;        // the candidates' positions
  const uint32_t m = p.n_keep - p.n_sink - p.n_recent;  // how many of them stay: fewer than there are
  // T: the m-th greatest; `left`: how many of the keys equal to it stay
  uint32_t T = 0xffffffffu, left = 0;
  if (m > 0) {
    T = 0;
    left = m;
    for (int shift = 24; shift >= 0; shift -= 8) {
      if (tid < 256) hist[tid] = 0;
      __syncthreads();
      const uint32_t above = shift == 24 ? 0u : 0xffffffffu << (shift + 8);
      for (int i = lo + tid; i < hi; i += kSelectThreads) {
        const uint32_t u = ordered(w[i]);
        if ((u & above) == T) atomicAdd(&hist[(u >> shift) & 255u], 1u);
      }
      __syncthreads();
      if (tid < 32) {
        // lane l has digits 255 - 8 l .. 248 - 8 l: the greatest first
        uint32_t c[8], sum = 0;
#pragma unroll
        for (int x = 0; x < 8; ++x) {
          c[x] = hist[255 - 8 * tid - x];
          sum += c[x];
        }
        uint32_t before = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const uint32_t y = __shfl_up_sync(0xffffffffu, before, o);
          if (tid >= o) before += y;
        }
        before -= sum;
#pragma unroll
        for (int x = 0; x < 8; ++x) {
          if (before < left && before + c[x] >= left) {
            sel_digit = 255 - 8 * tid - x;
            sel_left = left - before;
          }
          before += c[x];
        }
      }
      __syncthreads();
      T |= sel_digit << shift;
      left = sel_left;
    }
  }
  // in the order of the positions: a key stays if it always does, weighs more than T, or is one of the first `left` equal to T
  uint32_t over_before = 0, equal_before = 0;
  for (int i0 = 0; i0 < n; i0 += kSelectThreads) {
    const int i = i0 + tid;
    const float x = i < n ? w[i] : 0.f;
    const uint32_t u = ordered(x);
    const bool always = i < lo || (i >= hi && i < n), candidate = i >= lo && i < hi;
    const bool over = always || (candidate && u > T), equal = candidate && u == T;
    uint2 total;
    const uint2 before = block_scan(make_uint2(over, equal), warp_sums, total);  // (every weight of the step is in a register behind it)
    const uint32_t eq = equal_before + before.y;
    if (over || (equal && eq < left)) {
      const uint32_t to = over_before + before.x + min(eq, left);
      kept[to] = i;
      w[to] = x;
    }
    over_before += total.x;
    equal_before += total.y;
  }
  __syncthreads();
  for (int i = p.n_keep + tid; i < n; i += kSelectThreads) w[i] = 0.f;
}

// kLanes threads of 16 bytes make one row of a CTA's columns; kRows rows of each thread are in flight.
template <int kLanes>
__global__ void __launch_bounds__(kMoveThreads) evict_move_kernel(const EvictParams p, int slices) {
  constexpr int kRows = 8, kGroup = kMoveThreads / kLanes;  // rows a step moves: kRows * kGroup
  grid_launch_dependents();
  grid_dependency_wait();
  const int hkv = blockIdx.y, b = blockIdx.z, tid = threadIdx.x;
  const int n = min(max(p.kv_lens[b], 0), p.max_len);
  if (n <= p.n_keep) return;
  const bool is_v = (int)blockIdx.x >= slices;
  const int col = ((is_v ? blockIdx.x - slices : blockIdx.x) * kLanes + tid % kLanes) * 8;
  const int64_t* st = is_v ? p.vs : p.ks;
  __nv_bfloat16* base = (is_v ? p.v : p.k) + hkv * st[1] + col;
  const int32_t* kept = p.kept + ((int64_t)b * p.n_kv_head + hkv) * p.n_keep;
  const int32_t* table = p.table + b * p.table_stride;
  auto row_of = [&](int r) -> __nv_bfloat16* {
    const int at = p.by_page.div(r), id = table[at];
    if ((unsigned)id >= (unsigned)p.n_pages) return nullptr;  // not followed
    return base + (int64_t)id * st[0] + (int64_t)(r - at * (int)p.by_page.d) * st[2];
  };
  bool bad = false;
  for (int i0 = 0; i0 < p.n_keep; i0 += kRows * kGroup) {
    uint4 x[kRows];
    __nv_bfloat16* to[kRows];
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      const int i = i0 + r * kGroup + tid / kLanes;
      to[r] = nullptr;
      if (i >= p.n_keep) continue;
      const int src = kept[i];
      if (src == i) continue;  // it lies there
      const __nv_bfloat16* from = row_of(src);
      to[r] = row_of(i);
      if (from == nullptr || to[r] == nullptr) {
        to[r] = nullptr;
        bad = true;
        continue;
      }
      x[r] = *reinterpret_cast<const uint4*>(from);
    }
    __syncthreads();  // every row of the step is in registers
#pragma unroll
    for (int r = 0; r < kRows; ++r)
      if (to[r] != nullptr) *reinterpret_cast<uint4*>(to[r]) = x[r];
  }
  if (bad) atomicOr(p.status, kStatusOutOfRange);
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
  cudaError_t e = launch_overlapped(evict_select_kernel, dim3(a.n_kv_head, a.batch), dim3(kSelectThreads), 0, st, 1, p);
  count_launch();
  if (e == cudaSuccess) e = cudaGetLastError();
  if (e != cudaSuccess) return (int)e;
  constexpr int kLanes = 8;  // 128 bytes of a row per CTA
  const int slices = a.head_dim / (8 * kLanes);
  e = launch_overlapped(evict_move_kernel<kLanes>, dim3(2 * slices, a.n_kv_head, a.batch), dim3(kMoveThreads), 0, st, 1, p, slices);
  count_launch();
  return (int)(e != cudaSuccess ? e : cudaGetLastError());
}

}  // namespace tyr
