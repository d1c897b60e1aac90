// Whether strided memory overlaps: a pool of pages with itself, two pools, a pool and a dense buffer.
// Host only, no CUDA.
#pragma once

#include <cstdint>

namespace wc {

// size[i] steps of stride[i] bytes in every dimension, a run of bytes at each place; after sort(), the
// dimensions of more than one step, the widest stride first.
struct Strided {
  static constexpr int kDims = 4;
  uintptr_t at = 0;
  long long size[kDims], stride[kDims], run = 0;
  int dims = 0;
  bool nested = false;  // each step passes all that lies below it: no two places overlap

  void add(long long n, long long step) {
    if (n < 2) return;
    int i = dims++;
    for (; i > 0 && stride[i - 1] < step; --i) {
      size[i] = size[i - 1];
      stride[i] = stride[i - 1];
    }
    size[i] = n;
    stride[i] = step;
  }
  // Bytes from the first to behind the last, without the widest `from` dimensions.
  long long extent(int from = 0) const {
    long long e = run;
    for (int i = from; i < dims; ++i) e += (size[i] - 1) * stride[i];
    return e;
  }
  void close() {
    nested = true;
    for (int i = 0; i < dims; ++i) nested = nested && stride[i] >= extent(i + 1);
  }
};

inline long long floor_div(long long a, long long b) { return a / b - (a % b < 0); }  // b > 0

// Whether a[i..] at 0 meets a dense run of bytes [lo, hi). Exact where a is nested; where not, whether
// its extent does.
inline bool meets_run(const Strided& a, long long lo, long long hi, int i = 0) {
  if (lo >= hi || hi <= 0 || lo >= a.extent(i)) return false;
  if (i == a.dims || !a.nested) return true;
  // steps k whose bytes [k s, k s + below) meet the run: from the third on, one lies inside it whole
  const long long s = a.stride[i], below = a.extent(i + 1);
  long long k0 = floor_div(lo - below, s) + 1, k1 = floor_div(hi - 1, s);
  if (k0 < 0) k0 = 0;
  if (k1 > a.size[i] - 1) k1 = a.size[i] - 1;
  if (k1 - k0 >= 2) return true;
  for (long long k = k0; k <= k1; ++k)
    if (meets_run(a, lo - k * s, hi - k * s, i + 1)) return true;
  return false;
}
inline bool meets_run(const Strided& a, const void* p, long long bytes) {
  const long long lo = (long long)(reinterpret_cast<uintptr_t>(p) - a.at);
  return p && meets_run(a, lo, lo + bytes);
}

// Whether a[i..] at 0 meets b[i..] at d. Where both step alike (two pools that are cut from one buffer) only
// the steps at which what lies below can meet are followed, so the answer is exact for nested pools of
// equal strides; where they do not, extents decide.
inline bool meets(const Strided& a, const Strided& b, long long d, int i = 0) {
  const long long ea = a.extent(i), eb = b.extent(i);
  if (d >= ea || d + eb <= 0) return false;
  if (i == a.dims && i == b.dims) return true;
  if (!a.nested || !b.nested || i == a.dims || i == b.dims || a.stride[i] != b.stride[i]) return true;
  const long long s = a.stride[i], ba = a.extent(i + 1), bb = b.extent(i + 1);
  // step k of b against a: -bb < d + k s < ba
  long long k0 = floor_div(-bb - d, s) + 1, k1 = floor_div(ba - d - 1, s);
  if (k0 < 1 - a.size[i]) k0 = 1 - a.size[i];
  if (k1 > b.size[i] - 1) k1 = b.size[i] - 1;
  for (long long k = k0; k <= k1; ++k)
    if (meets(a, b, d + k * s, i + 1)) return true;
  return false;
}
inline bool meets(const Strided& a, const Strided& b) { return meets(a, b, (long long)(b.at - a.at)); }

}  // namespace wc
