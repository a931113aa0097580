// Division of small indices by a fixed number, as a multiplication and a shift.
#pragma once
#include <stdint.h>

namespace sfb200 {

struct RowDivider {
  uint64_t mul;
  int shift;
};
// For 1 <= d <= 2^28 and 0 <= i < 2^31: i / d == i * mul >> shift, with l = ceil(log2 d), shift = 31 + l and
// mul = floor(2^shift / d) + 1: 2^shift < mul * d <= 2^shift + 2^l, so the product is above i / d by less than
// i * 2^l / (d * 2^shift) < 1 / d.  mul <= 2^32: the product fits 64 bits.
inline RowDivider row_divider(uint32_t d) {
  int l = 0;
  while ((1ull << l) < d) ++l;
  return RowDivider{(1ull << (31 + l)) / d + 1, 31 + l};
}

}  // namespace sfb200
