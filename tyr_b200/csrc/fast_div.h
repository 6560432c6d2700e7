// Division of a non-negative 32-bit number by a divisor fixed per launch, as a multiply-high and a
// shift: q = umulhi(n, mul) >> shr with mul = ceil(2^(31 + ceil(log2 d)) / d), exact for n < 2^31.
// The hardware has no integer divider.
#pragma once
#include <stdint.h>

namespace tyr {

struct FastDiv {
  uint32_t mul, shr, d;
  __device__ __forceinline__ int div(int n) const {
    return d == 1u ? n : static_cast<int>(__umulhi(static_cast<uint32_t>(n), mul) >> shr);
  }
};
inline FastDiv make_fastdiv(int d) {
  FastDiv f;
  f.d = static_cast<uint32_t>(d > 1 ? d : 1);
  f.mul = 0;
  f.shr = 0;
  if (f.d > 1u) {
    int lg = 0;
    while ((1ull << lg) < f.d) ++lg;  // ceil(log2 d)
    const int pw = 31 + lg;
    f.mul = static_cast<uint32_t>(((1ull << pw) + f.d - 1) / f.d);
    f.shr = static_cast<uint32_t>(pw - 32);
  }
  return f;
}

}  // namespace tyr
