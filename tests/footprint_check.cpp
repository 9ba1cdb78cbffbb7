// Host check of csrc/footprint.hpp (no GPU), built and run by tests/test_footprint.py: views of a small buffer, drawn at random, against the sets of their
// bytes.  Views that share a byte are never called apart; views that lie side by side in every row, page or head are.
#include <cstdio>
#include <random>
#include <set>
#include <vector>

#include "footprint.hpp"

using segpt::apart;
using segpt::Footprint;

namespace {

struct View {
  int64_t at, element;
  std::vector<int64_t> sizes, strides;
  Footprint footprint() const { return Footprint((int64_t)sizes.size(), sizes.data(), strides.data(), element); }
  std::set<int64_t> bytes() const {
    std::set<int64_t> r;
    std::vector<int64_t> i(sizes.size(), 0);
    while (true) {
      int64_t b = at;
      for (size_t d = 0; d < i.size(); ++d) b += i[d] * strides[d] * element;
      for (int64_t e = 0; e < element; ++e) r.insert(b + e);
      size_t d = 0;
      while (d < i.size() && ++i[d] == sizes[d]) i[d++] = 0;
      if (d == i.size()) return r;
    }
  }
};
bool share(const View& a, const View& b) {
  const auto x = a.bytes();
  for (int64_t y : b.bytes())
    if (x.count(y)) return true;
  return false;
}
bool said_apart(const View& a, const View& b) { return apart(a.footprint(), 0, b.footprint(), 0, b.at - a.at); }

}  // namespace

int main() {
  std::mt19937 rng(1);
  auto pick = [&](int lo, int hi) { return (int64_t)(lo + rng() % (hi - lo + 1)); };
  int n_apart = 0, n_share = 0, unsure = 0;
  for (int trial = 0; trial < 200000; ++trial) {
    View v[2];
    for (View& x : v) {
      x.element = pick(0, 1) ? 2 : 4;
      x.at = pick(0, 150) * 2;
      const int dims = (int)pick(0, 4);
      for (int d = 0; d < dims; ++d) {
        x.sizes.push_back(pick(1, 4));
        x.strides.push_back(pick(0, 9) == 0 ? 0 : pick(1, 24));
      }
    }
    if (pick(0, 2) == 0) v[1].strides = v[0].strides, v[1].sizes = v[0].sizes, v[1].element = v[0].element;  // slices of one buffer
    const bool s = share(v[0], v[1]), a = said_apart(v[0], v[1]);
    if (a != said_apart(v[1], v[0])) { std::printf("VIOLATION: not the same the other way round\n"); return 1; }
    if (s && a) { std::printf("VIOLATION: views that share a byte are called apart (trial %d)\n", trial); return 1; }
    s ? ++n_share : a ? ++n_apart : ++unsure;
  }
  std::printf("apart %d, sharing %d, apart but not seen to be %d\n", n_apart, n_share, unsure);
  if (n_apart < 10000 || n_share < 10000) return 1;
  // side by side in one buffer: two pools, page by page, slot by slot and head by head; slices of a projection, a row of one element a head among them
  const View sides[][2] = {
      {{0, 2, {5, 2, 4, 8}, {128, 32, 8, 1}}, {64 * 2, 2, {5, 2, 4, 8}, {128, 32, 8, 1}}},
      {{0, 2, {5, 2, 4, 8}, {128, 64, 16, 1}}, {8 * 2, 2, {5, 2, 4, 8}, {128, 64, 16, 1}}},
      {{0, 2, {5, 2, 4, 8}, {128, 8, 32, 1}}, {16 * 2, 2, {5, 2, 4, 8}, {128, 8, 32, 1}}},
      {{0, 2, {7, 3, 8}, {60, 8, 1}}, {24 * 2, 2, {7, 3, 8}, {60, 8, 1}}},
      {{0, 2, {7, 3, 8}, {60, 8, 1}}, {57 * 2, 2, {7, 3}, {60, 1}}},
      {{0, 2, {7, 3, 8}, {0, 8, 1}}, {24 * 2, 2, {7, 3, 8}, {24, 8, 1}}},
  };
  for (const auto& s : sides)
    if (share(s[0], s[1]) || !said_apart(s[0], s[1]) || !said_apart(s[1], s[0])) { std::printf("VIOLATION: side by side, but not called apart\n"); return 1; }
  const View shifted[2] = {{0, 2, {7, 6, 8}, {100, 8, 1}}, {24 * 2, 2, {7, 6, 8}, {100, 8, 1}}};
  if (said_apart(shifted[0], shifted[1])) { std::printf("VIOLATION: a slice shifted by three heads\n"); return 1; }
  return 0;
}
