// Whether two strided views of memory are apart.  Plain C++: included by torch_binding.cpp and by tests/footprint_check.cpp, which compares it on the
// host with the sets of bytes themselves.
#pragma once

#include <algorithm>
#include <cstdint>

namespace segpt {

// Where a tensor's elements lie: bytes from its first one, by the dimensions that have more than one element, the widest step first
struct Footprint {
  int64_t element, step[8], size[8];
  int dims = 0;
  Footprint(int64_t n, const int64_t* sizes, const int64_t* strides, int64_t element_bytes) : element(element_bytes) {  // n: at most 8
    for (int64_t d = 0; d < n && dims < 8; ++d) {
      if (sizes[d] <= 1) continue;
      const int64_t s = strides[d] * element;
      int i = dims++;
      for (; i > 0 && step[i - 1] < s; --i) { step[i] = step[i - 1]; size[i] = size[i - 1]; }
      step[i] = s; size[i] = sizes[d];
    }
  }
  int64_t span(int from) const {  // of the dimensions from that one on
    int64_t n = element;
    for (int i = from; i < dims; ++i) n += (size[i] - 1) * step[i];
    return n;
  }
};
// Whether no byte of b's is one of a's.  far: from the first byte of a's dimensions i .. to the first of b's j ..  The widest step is taken apart: of the places
// it leads to only those count where the rest may meet, which are one or two for views that lie side by side in every row, page or head of a
// buffer.  Where they are many the answer is no.
inline bool apart(const Footprint& a, int i, const Footprint& b, int j, int64_t far) {
  if (far >= a.span(i) || far + b.span(j) <= 0) return true;
  const int64_t wide_a = i < a.dims ? a.step[i] : 0, wide_b = j < b.dims ? b.step[j] : 0, wide = std::max(wide_a, wide_b);
  if (wide <= 0) return false;
  const bool of_a = wide_a == wide, of_b = wide_b == wide;
  const int ni = i + of_a, nj = j + of_b;
  // far + k * wide for k of b's places less k of a's
  const int64_t first = of_a ? -(a.size[i] - 1) : 0, last = of_b ? b.size[j] - 1 : 0, below = -b.span(nj), above = a.span(ni);
  auto floor_div = [](int64_t x, int64_t y) { return x / y - (x % y < 0); };
  const int64_t from = std::max(first, floor_div(below - far, wide) + 1), to = std::min(last, floor_div(above - far - 1, wide));
  if (to - from >= 4) return false;
  for (int64_t k = from; k <= to; ++k)
    if (!apart(a, ni, b, nj, far + k * wide)) return false;
  return true;
}

}  // namespace segpt
