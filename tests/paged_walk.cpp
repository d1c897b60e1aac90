// A block's walk over the line of key tiles (PagedWalk in paged.cuh) on CPU threads: one thread per
// device thread, barriers for __syncthreads and shuffles, so that a thread sanitizer sees shared-memory
// accesses that no barrier orders. Reads cases from the standard input, prints every block's items.
//
// -DSTORE_ALWAYS: thread 0 keeps the walk whether or not the block has work, as a check that the
// sanitizer reports what it should.
#include <cuda_runtime.h>
#undef __global__
#define __global__ static inline
#undef __launch_bounds__
#define __launch_bounds__(...)
#undef __grid_constant__
#define __grid_constant__

#include <pthread.h>

#include <algorithm>
#include <cmath>
#include <cstdio>
#include <thread>
#include <vector>

using std::max;
using std::min;

thread_local uint3 threadIdx, blockIdx;
thread_local dim3 blockDim, gridDim;

// ---------------------------------------------------------------------------- what the walk calls
struct Barrier {
  pthread_barrier_t b;
  explicit Barrier(int n) { pthread_barrier_init(&b, nullptr, n); }
  void wait() { pthread_barrier_wait(&b); }
};
constexpr int kThreads = 384;
Barrier block_barrier(kThreads);
Barrier* warp_barrier[kThreads / 32];
long long lane_value[kThreads];

void __syncthreads() { block_barrier.wait(); }
template <class T>
T __shfl_up_sync(unsigned, T x, int o) {
  const int t = threadIdx.x, lane = t % 32;
  lane_value[t] = x;
  warp_barrier[t / 32]->wait();
  const T y = T(lane_value[lane >= o ? t - o : t]);
  warp_barrier[t / 32]->wait();
  return y;
}
int errors = 0;
int atomicOr(int* at, int bits) { return __atomic_fetch_or(at, bits, __ATOMIC_RELAXED); }

// ---------------------------------------------------------------------------- what it does not
#define NOT_HERE(type, name) \
  template <class... A>      \
  type name(A...);
NOT_HERE(float, __uint_as_float)
NOT_HERE(unsigned, __float_as_uint)
NOT_HERE(unsigned, __umulhi)
NOT_HERE(unsigned, __cvta_generic_to_shared)
NOT_HERE(void, __nanosleep)
NOT_HERE(void, __syncwarp)
NOT_HERE(int, __any_sync)
NOT_HERE(int, __syncthreads_or)
NOT_HERE(int, __syncthreads_count)
template <class T>
T __shfl_xor_sync(unsigned, T, int);
template <class T>
T __shfl_sync(unsigned, T, int);

#include "../woodcock_b200/csrc/paged.cuh"

using namespace wc;

struct Item {
  int prefix, idx, head, qt, kt0, kt1, ktn, first, count;
};

int main() {
  for (int i = 0; i < kThreads / 32; ++i) warp_barrier[i] = new Barrier(32);
  int cases = 0;
  if (scanf("%d", &cases) != 1) return 2;
  for (int c = 0; c < cases; ++c) {
    int B, G, H, Hk, page_log2, tree, grid, least, kinds;
    if (scanf("%d %d %d %d %d %d %d %d %d", &B, &G, &H, &Hk, &page_log2, &tree, &grid, &least, &kinds) != 9) return 2;
    auto read = [](int n) {
      std::vector<int> v(n);
      for (int& x : v)
        if (scanf("%d", &x) != 1) exit(2);
      return v;
    };
    std::vector<int> lens = read(B), offsets = read(B + 1), plens = read(G), groups = read(G ? G + 1 : 0);
    PagedAttnParams p = {};
    p.lens = lens.data();
    p.offsets = offsets.data();
    p.prefix_lens = plens.data();
    p.groups = groups.data();
    p.T = offsets[B];
    p.B = B;
    p.G = G;
    p.H = H;
    p.Hk = Hk;
    p.rep = H / Hk;
    p.page_log2 = page_log2;
    p.table_cols = p.prefix_cols = 1 << 12;
    p.err = &errors;
    const long long bits = 0;
    p.tree = tree ? &bits : nullptr;  // looked at for being there
    using Walk = PagedWalk<128, 128, 3>;
    std::vector<std::vector<Item>> items(grid);
    std::vector<char> same(grid, 1);
    std::vector<std::vector<long long>> sh(grid, std::vector<long long>(kWalkShared));
    auto thread = [&](int t) {
      threadIdx = {unsigned(t), 0, 0};
      blockDim = dim3(kThreads);
      gridDim = dim3(grid);
      for (int b = 0; b < grid; ++b) {
        blockIdx = {unsigned(b), 0, 0};
        Walk w;
#ifdef STORE_ALWAYS
        bool work = w.begin(p, kinds, least, sh[b].data());
        if (t == 0) *reinterpret_cast<Walk*>(sh[b].data()) = w;
#else
        bool work = w.begin_kept(p, kinds, least, sh[b].data());
#endif
        __syncthreads();  // the kernel's last one
        if (t == 0 && work) {
          Walk again = *reinterpret_cast<Walk*>(sh[b].data());
          do items[b].push_back({w.g.prefix, w.g.idx, w.head, w.qt, w.kt0, w.kt1, w.ktn, w.first, w.count});
          while (w.next(p, kinds));
          size_t n = 0;
          do {
            const Item& x = items[b][min(n, items[b].size() - 1)];
            if (again.g.idx != x.idx || again.head != x.head || again.qt != x.qt || again.kt0 != x.kt0) same[b] = 0;
          } while (++n, again.next(p, kinds));
          if (n != items[b].size()) same[b] = 0;
        }
      }
    };
    std::vector<std::thread> pool;
    for (int t = 0; t < kThreads; ++t) pool.emplace_back(thread, t);
    for (auto& t : pool) t.join();
    printf("case %d\n", c);
    for (int b = 0; b < grid; ++b) {
      printf("block %d %d\n", b, int(same[b]));
      for (const Item& x : items[b])
        printf("%d %d %d %d %d %d %d %d %d\n", x.prefix, x.idx, x.head, x.qt, x.kt0, x.kt1, x.ktn, x.first, x.count);
    }
  }
  return errors ? 3 : 0;
}
