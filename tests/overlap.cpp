// overlap.h against sets of bytes, on small pools.
#include "../woodcock_b200/csrc/overlap.h"

#include <cstdio>
#include <random>
#include <vector>

using wc::Strided;

static std::vector<int> bytes(const Strided& s, long long base, long long n) {
  std::vector<int> m(n);
  long long total = 1;
  for (int i = 0; i < s.dims; ++i) total *= s.size[i];
  for (long long x = 0; x < total; ++x) {
    long long at = base, y = x;
    for (int i = 0; i < s.dims; ++i) {
      at += y % s.size[i] * s.stride[i];
      y /= s.size[i];
    }
    for (long long r = 0; r < s.run; ++r) ++m[at + r];
  }
  return m;
}

int main() {
  std::mt19937 rng(1);
  auto pick = [&](int lo, int hi) { return lo + int(rng() % unsigned(hi - lo + 1)); };
  const long long N = 6000, mid = 2500;
  long long seen[2][2] = {}, runs[2] = {}, pairs[2] = {}, loose = 0, bad = 0;
  for (int it = 0; it < 12000; ++it) {
    Strided a;
    a.run = pick(1, 4);
    long long st[4], sz[4], e = a.run;
    for (int i = 0; i < 4; ++i) {  // from the tightest step on, some steps too short
      sz[i] = pick(1, 4);
      st[i] = e + (pick(0, 2) ? 0 : pick(0, 5)) - (pick(0, 11) ? 0 : pick(1, 4));
      if (st[i] < 1) st[i] = 1;
      e = (sz[i] - 1) * st[i] + e;
    }
    const int order = pick(0, 3);
    for (int i = 0; i < 4; ++i) a.add(sz[(i + order) % 4], st[(i + order) % 4]);
    a.close();
    if (a.extent() > 900) continue;
    const std::vector<int> ma = bytes(a, mid, N);
    bool twice = false;
    for (int x : ma) twice = twice || x > 1;
    ++seen[a.nested][twice];
    if (a.nested && twice) ++bad;
    for (int j = 0; j < 6; ++j) {  // dense runs
      const long long lo = pick(-20, int(a.extent()) + 10), len = pick(0, j < 3 ? 6 : 200);
      bool meet = false;
      for (long long x = lo; x < lo + len; ++x) meet = meet || ma[mid + x];
      const bool got = meets_run(a, lo, lo + len);
      ++runs[meet];
      if (a.nested ? got != meet : meet && !got) ++bad;
    }
    for (int j = 0; j < 6; ++j) {  // a second pool: the same steps, or others below the widest
      Strided b = a;
      if (j >= 4 && b.dims) {
        b.run = pick(1, 4);
        b.stride[b.dims - 1] += pick(0, 3);
        b.close();
      }
      const long long d = pick(-int(b.extent()) - 3, int(a.extent()) + 3);
      const std::vector<int> mb = bytes(b, mid + d, N);
      bool meet = false;
      for (long long x = 0; x < N; ++x) meet = meet || (ma[x] && mb[x]);
      const bool got = meets(a, b, d);
      if (meet && !got) ++bad;
      if (j < 4 && a.nested && got != meet) ++bad;
      ++pairs[meet];
      loose += got && !meet;
    }
  }
  // K and V of a page side by side, of a head, of a row; halves of one buffer; shifted by a page
  auto pool = [](long long page, long long head, long long row, uintptr_t at) {
    Strided s;
    s.at = at;
    s.run = 256;
    s.add(50, page);
    s.add(8, head);
    s.add(16, row);
    s.close();
    return s;
  };
  const long long row = 256, head = 16 * row, page = 8 * head;
  bad += meets(pool(2 * page, head, row, 4096), pool(2 * page, head, row, 4096 + page));
  bad += meets(pool(2 * page, 2 * head, row, 4096), pool(2 * page, 2 * head, row, 4096 + head));
  bad += meets(pool(2 * page, 2 * head, 2 * row, 4096), pool(2 * page, 2 * head, 2 * row, 4096 + row));
  bad += meets(pool(page, head, row, 4096), pool(page, head, row, 4096 + 50 * page));
  bad += meets(pool(2 * page, head, row, 4096), pool(2 * page, head, row, 4096 + 5 * page));
  bad += meets(pool(2 * page, head, row, 4096), pool(2 * page, row, 8 * row, 4096 + page));  // V by positions
  bad += !meets(pool(page, head, row, 4096), pool(page, head, row, 4096));
  bad += !meets(pool(page, head, row, 4096), pool(page, head, row, 4096 + 3 * page));
  bad += !meets(pool(2 * page, head, row, 4096), pool(2 * page, head, row, 4096 + page / 2));
  bad += !meets(pool(page, head, row, 4096 + 49 * page + 7 * head), pool(page, head, row, 4096));
  printf("%lld wrong; nested %lld, not %lld + %lld; runs %lld + %lld, pairs %lld + %lld (%lld refused that do not meet)\n",
         bad, seen[1][0], seen[0][0], seen[0][1], runs[0], runs[1], pairs[0], pairs[1], loose);
  const bool all = seen[1][0] && seen[0][1] && runs[0] && runs[1] && pairs[0] && pairs[1];
  return bad || !all;
}
