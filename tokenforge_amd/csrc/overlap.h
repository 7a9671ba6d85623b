// Whether strided sets of byte runs share memory.
#pragma once

#include <cstdint>
#include <utility>

namespace tf {

// Runs of `run` bytes from `at` on, in `dims` dimensions of two or more, the largest stride (bytes) first.
struct Runs {
  int64_t at, run;
  int dims = 0;
  std::pair<int64_t, int64_t> dim[3];  // stride, size

  Runs(const void* p, int64_t bytes) : at((int64_t)reinterpret_cast<uintptr_t>(p)), run(bytes) {}

  void add(int64_t stride, int64_t size) {
    if (size < 2) return;
    int i = dims++;
    for (; i > 0 && dim[i - 1].first < stride; --i) dim[i] = dim[i - 1];
    dim[i] = {stride, size};
  }

  // Bytes from the first to the last of what lies within dimension i on.
  int64_t extent(int i) const {
    int64_t e = run;
    for (; i < dims; ++i) e += dim[i].first * (dim[i].second - 1);
    return e;
  }
};

// Whether runs a and, `far` bytes behind where they begin, runs b share a byte, both from their dimension i on. A dimension
// of one stride in both is settled by the (one or two) differences of its indices that bring what lies within it
// together; where the strides differ, ranges that meet count as overlap. Dimensions that are not nested (what lies
// within one reaches over its stride) are not looked into: the operators refuse them before.
inline bool runs_meet(const Runs& a, const Runs& b, int64_t far, int i) {
  const int64_t ea = a.extent(i), eb = b.extent(i);
  if (far >= ea || far <= -eb) return false;
  if (i >= a.dims || i >= b.dims || a.dim[i].first != b.dim[i].first) return true;
  const int64_t s = a.dim[i].first, ia = a.extent(i + 1), ib = b.extent(i + 1);
  if (ia > s || ib > s) return false;
  // far + s t in (-ib, ia), t in (-a's size, b's size)
  const auto floor_div = [](int64_t n, int64_t d) { return n / d - (n % d < 0 ? 1 : 0); };
  int64_t t = floor_div(-ib - far, s) + 1, last = floor_div(ia - 1 - far, s);
  if (t <= -a.dim[i].second) t = 1 - a.dim[i].second;
  if (last >= b.dim[i].second) last = b.dim[i].second - 1;
  for (; t <= last; ++t)
    if (runs_meet(a, b, far + s * t, i + 1)) return true;
  return false;
}

inline bool overlap(const Runs& a, const Runs& b) { return runs_meet(a, b, b.at - a.at, 0); }

}  // namespace tf
