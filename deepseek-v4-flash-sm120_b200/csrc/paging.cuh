// Token positions to cache slots: the device side of block tables.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace dsv4 {

// Division of n < 2^31 by a constant: (umulhi(mul, n) + n) >> shift.
struct FastDiv {
  uint32_t mul, shift, d;
};
inline FastDiv fast_div(uint32_t d) {
  uint32_t l = 0;
  while ((1ull << l) < d) ++l;
  const uint64_t m = ((1ull << 32) * ((1ull << l) - d)) / d + 1;
  return FastDiv{static_cast<uint32_t>(m), l, d};
}
__device__ __forceinline__ uint32_t div_by(uint32_t n, const FastDiv& f) {
  return (__umulhi(f.mul, n) + n) >> f.shift;
}

__device__ __forceinline__ int slot_of(const int32_t* table, int max_pages, const FastDiv& page, int pos) {
  if (pos < 0) return -1;
  const uint32_t col = div_by(static_cast<uint32_t>(pos), page);
  if (col >= static_cast<uint32_t>(max_pages)) return -1;
  const int id = __ldg(table + col);
  if (id < 0) return -1;
  const long long s = static_cast<long long>(id) * page.d + (static_cast<uint32_t>(pos) - col * page.d);
  return s > 0x7fffffff ? -1 : static_cast<int>(s);
}

}  // namespace dsv4
