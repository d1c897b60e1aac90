// Failures and launches of several threads that share a context (host.h), for the thread sanitizer.
#include "../woodcock_b200/csrc/host.h"

#include <cstdio>
#include <cstring>

int main() {
  wc_ctx ctx;
  int bad = 0;
  auto run = [&](int n, int* wrong) {
    // messages longer than a string holds in place, of different lengths
    const std::string mine = std::string(40 + 60 * n, char('a' + n));
    for (int i = 0; i < 2000; ++i) {
      const wc_status st = guard(&ctx, [&] { fail(n ? WC_ERR_INVALID : WC_ERR_CAPACITY, mine); });
      if (st != (n ? WC_ERR_INVALID : WC_ERR_CAPACITY) || mine != ctx.err.get()) ++*wrong;
      count_launch(&ctx, reinterpret_cast<cudaStream_t>(1));
    }
  };
  int wrong[4] = {};
  std::vector<std::thread> pool;
  for (int n = 0; n < 4; ++n) pool.emplace_back(run, n, &wrong[n]);
  for (auto& t : pool) t.join();
  for (int w : wrong) bad += w;
  if (!std::strlen(ctx.err.get())) ++bad;  // a thread without a failure is told the latest
  if (ctx.launches != 8000) ++bad;
  ctx.capturing = true;  // what the context's own stream records; other streams' launches run now
  count_launch(&ctx, ctx.stream);
  count_launch(&ctx, reinterpret_cast<cudaStream_t>(1));
  if (ctx.launches != 8001 || ctx.capture_launches != 1) ++bad;
  printf("%d\n", bad);
  return bad != 0;
}
