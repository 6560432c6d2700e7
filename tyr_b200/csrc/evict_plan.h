// How many CTAs share the selection of one (sequence, KV head) in an eviction.  Plain C++ on sizes alone (the cluster capacities
// are an argument), so that the choice can be checked on the host.
#pragma once

namespace tyr {

constexpr int kMaxEvictLog = 4;  // clusters of up to 16 CTAs

// One CTA up to `segment` keys, what it holds in registers.  Past that the smallest cluster that holds all of them (both launches, 8
// KV heads of 128: one sequence of 30000 keys 60 us against one CTA's 83, of 100000 120 against 202, 32 of 30000 542 against 550),
// if the device can place one: `capacity(k)` is how many clusters of 2^k CTAs can be resident at once, 0 where none can (the
// larger ones need that many free SMs in one GPC).  Otherwise, and past the greatest cluster, one CTA does it in segments.
template <class Capacity>
int evict_ranks(long long max_len, int segment, Capacity&& capacity) {
  for (int k = 0; k <= kMaxEvictLog; ++k)
    if (((long long)segment << k) >= max_len) return k > 0 && capacity(k) <= 0 ? 1 : 1 << k;
  return 1;
}

}  // namespace tyr
