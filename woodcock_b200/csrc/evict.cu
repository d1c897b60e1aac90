// Entry points of the gathered attention weight and of the eviction by it: argument checks, workspace layout
// and launches of the kernels in evict.cuh.
#include <cmath>
#include <cstring>

#include "evict.cuh"
#include "paged_host.h"

using namespace wc;

namespace {

// The mass of one layer's keys (layer >= 0), or of all layers'.
Strided mass_places(const wc_pages& g, const wc_mass& m, int layer) {
  Strided s;
  s.at = reinterpret_cast<uintptr_t>(m.p) + (layer > 0 ? m.stride[0] * layer * 4 : 0);
  s.run = g.page_size * 4ll;
  if (layer < 0) s.add(g.layers, m.stride[0] * 4);
  s.add(g.pages, m.stride[1] * 4);
  s.add(g.kv_heads, m.stride[2] * 4);
  s.close();
  return s;
}

void check_mass(const wc_pages& g, const wc_mass& m) {
  need(m.p != nullptr && reinterpret_cast<uintptr_t>(m.p) % 4 == 0, "paged: null or misaligned mass");
  const int sizes[3] = {g.layers, g.pages, g.kv_heads};
  for (int i = 0; i < 3; ++i) need(sizes[i] == 1 || m.stride[i] > 0, "paged: mass pages must not overlap");
}

wc_pages keys_only(wc_pages g) {
  g.v = g.k;
  std::memcpy(g.v_stride, g.k_stride, sizeof(g.v_stride));
  return g;
}

// Which kernels a call may need: the number of a request's rows is device data where offsets are given.
struct MassLayout {
  bool few, many;        // requests of at most 16 rows a KV head, of more
  int blocks, few_blocks, per, width, most;
  MassModes rows, keys;
  size_t row_ml, part_ml, rec, tiles, few_ml, few_part, scores, pieces, part_sum, keys_rec, rows_q, rows_l, bytes;
  int ids;
};

MassLayout mass_layout(const wc_ctx* ctx, const wc_paged_mass_args& a) {
  const wc_paged_batch& b = a.batch;
  MassLayout l;
  std::memset(&l, 0, sizeof(l));
  size_t at = 0;
  const wc_pages& g = a.pages;
  const long long rep = b.heads / g.kv_heads, each = rep * (b.q_offsets ? b.rows : b.rows / b.requests);
  l.few = g.dtype == WC_BF16 && (b.q_offsets || each <= 16);
  l.many = g.dtype != WC_BF16 || each > 16;
  if (l.few) {
    l.few_blocks = ctx->num_sms;
    l.width = int(std::min(16ll, each));
    // what the pool holds, or the tables, and each item's units beside its tiles
    const long long in_table = ((long long)b.table_cols * g.page_size + MF_KT - 1) / MF_KT + 1, heads = (long long)b.requests * g.kv_heads;
    const long long units = std::min(mass_most_tiles(g.pages, log2i(g.page_size), b.requests, g.kv_heads, MF_KT), heads * in_table) +
                            heads * MF_OVER;
    l.per = int((units + l.few_blocks - 1) / l.few_blocks);
    l.most = l.per / (1 + MF_OVER) + 4;  // an item's units but at both ends, and the list's end
    l.pieces = take(at, size_t(l.few_blocks) * l.most * sizeof(MassPiece));
    l.few_ml = take(at, size_t(b.rows) * b.heads * MF_CONSUMERS * sizeof(float2));
    l.few_part = take(at, size_t(l.few_blocks) * 2 * MF_M * MF_CONSUMERS * sizeof(float2));
    l.scores = take(at, size_t(l.few_blocks) * l.per * MF_KT * l.width * sizeof(float));
  }
  if (g.dtype != WC_BF16) l.row_ml = take(at, size_t(b.rows) * b.heads * sizeof(float2));
  if (l.many && g.dtype == WC_BF16) {
    const long long mean = (rep * b.rows + b.requests - 1) / b.requests;
    l.blocks = ctx->num_sms;
    // 8 requests of 8192 keys, 32 query and 8 KV heads: 68 rows a head 82 us in the windows' modes and 88 in the
    // prompts', 128 rows 83 and 89, 192 rows 129 and 124, 256 rows 129 and 124; 2 prompts of 1000 rows 193 and 174.
    // Which requests have how many rows is device data: the mean counts those that these kernels do not see, so
    // that a prompt beside many steps may get the windows' modes.
    l.rows = mean <= 128 ? kRows128 : kRows256;
    l.keys = mean <= 128 ? kKeysWindow : kKeysPrompt;
    l.ids = int(rep * b.rows / 128) + b.requests + 1;
    l.rows_q = take(at, size_t(g.kv_heads) * l.ids * 128 * g.head_dim * 2);
    l.rows_l = take(at, size_t(g.kv_heads) * l.ids * 128 * sizeof(float));
    l.part_sum = take(at, size_t(l.blocks) * 2 * MK_KEYS * sizeof(float));
    l.keys_rec = take(at, l.blocks * sizeof(MassRec));
  } else {
    l.blocks = ctx->num_sms * 2;
    l.tiles = take(at, (size_t(b.requests) + 1) * sizeof(long long));
  }
  const int M = g.dtype != WC_BF16 ? MS_M : l.rows == kRows128 ? 128 : 256;
  l.part_ml = take(at, size_t(l.blocks) * 2 * M * sizeof(float2));
  l.rec = take(at, l.blocks * sizeof(PagedRec));
  l.bytes = at;
  return l;
}

void check_mass_args(const wc_paged_mass_args& a) {
  check_pages(keys_only(a.pages));
  check_batch(a.pages, a.batch);
  need(a.layer >= 0 && a.layer < a.pages.layers, "paged_mass: layer out of range");
  need(std::isfinite(a.scale) && a.scale > 0, "paged_mass: scale must be positive");
}

template <int D, int NT>
void launch_few_rows(wc_ctx* ctx, cudaStream_t st, const MassParams& p, int blocks) {
  constexpr size_t smem = MfLayout<D>::bytes();
  static_assert(smem <= kSmemOptinBytes, "shared memory");
  opt_in(ctx, mass_few_rows_kernel<D, NT>, smem);
  launch_on(ctx, st, "mass_few_rows", mass_few_rows_kernel<D, NT>, dim3(blocks), dim3(MF_THREADS), smem, true, 1,
            p);
}

template <int D>
void gather_few(wc_ctx* ctx, cudaStream_t st, const wc_pages& g, MassParams p, const MassLayout& l, char* ws) {
  p.kinds = kOwnRows | kFewRows;
  p.row_ml = reinterpret_cast<float2*>(ws + l.few_ml);
  p.part_ml = reinterpret_cast<float2*>(ws + l.few_part);
  p.scores = reinterpret_cast<float*>(ws + l.scores);
  p.per = l.per;
  p.width = l.width;
  p.pieces = reinterpret_cast<MassPiece*>(ws + l.pieces);
  p.most = l.most;
  if (l.width <= 8) launch_few_rows<D, 1>(ctx, st, p, l.few_blocks);
  else launch_few_rows<D, 2>(ctx, st, p, l.few_blocks);
  // four sums at a time where they lie on 16 bytes
  const bool wide = reinterpret_cast<uintptr_t>(p.mass.ptr) % 16 == 0 && (g.pages == 1 || p.mass.page % 4 == 0) &&
                    (g.kv_heads == 1 || p.mass.head % 4 == 0);
  launch_on(ctx, st, "mass_few_keys", mass_few_keys_kernel, dim3(l.few_blocks, MF_SPREAD), dim3(MF_KEYS_THREADS), 0, true, 1, p,
            wide);
}

template <int D, int kMode>
void launch_many(wc_ctx* ctx, cudaStream_t st, const wc_pages& g, const MassParams& p) {
  constexpr size_t smem = MmLayout<D, kMode>::bytes();
  static_assert(smem <= kSmemOptinBytes, "shared memory");
  opt_in(ctx, mass_many_kernel<D, kMode>, smem);
  launch_on(ctx, st, "mass_many", mass_many_kernel<D, kMode>, dim3(p.blocks), dim3(MM_THREADS), smem, true, 1,
            page_map(g, p.a.K, 128, 1), p);
}

template <int D>
void gather_many(wc_ctx* ctx, cudaStream_t st, const wc_pages& g, MassParams p, const MassLayout& l, char* ws) {
  p.part_sum = reinterpret_cast<float*>(ws + l.part_sum);
  p.rows_q = reinterpret_cast<unsigned char*>(ws + l.rows_q);
  p.rows_l = reinterpret_cast<float*>(ws + l.rows_l);
  p.ids = l.ids;
  p.keys_rec = reinterpret_cast<MassRec*>(ws + l.keys_rec);
  if (l.rows == kRows128) launch_many<D, kRows128>(ctx, st, g, p);
  else launch_many<D, kRows256>(ctx, st, g, p);
  launch_on(ctx, st, "mass_join", l.rows == kRows128 ? mass_join_kernel<128, 128> : mass_join_kernel<256, 128>, dim3(p.blocks),
            dim3(256), 0, true, 1, p);
  if (l.keys == kKeysWindow) launch_many<D, kKeysWindow>(ctx, st, g, p);
  else launch_many<D, kKeysPrompt>(ctx, st, g, p);
  launch_on(ctx, st, "mass_fold", mass_fold_kernel, dim3(p.blocks), dim3(MK_KEYS), 0, true, 1, p);
}

template <typename S, int D>
void gather_mass(wc_ctx* ctx, cudaStream_t st, const wc_pages& g, MassParams p, const MassLayout& l, char* ws) {
  if constexpr (sizeof(S) == 2) {
    if (l.few) gather_few<D>(ctx, st, g, p, l, ws);
    p.kinds = kOwnRows | (l.few ? kManyRows : 0);
    if (l.many) gather_many<D>(ctx, st, g, p, l, ws);
  } else {
    p.kinds = kOwnRows;
    opt_in(ctx, mass_rows_kernel<D>, mass_simt_smem<D>());
    opt_in(ctx, mass_keys_kernel<D>, mass_simt_smem<D>());
    launch_on(ctx, st, "mass_rows", mass_rows_kernel<D>, dim3(p.blocks), dim3(MS_THREADS), mass_simt_smem<D>(), true, 1, p);
    launch_on(ctx, st, "mass_join", mass_join_kernel<MS_M, MS_KT>, dim3(p.blocks + 1), dim3(256), 0, true, 1, p);
    launch_on(ctx, st, "mass_keys", mass_keys_kernel<D>, dim3(ctx->num_sms * 2), dim3(MS_THREADS), mass_simt_smem<D>(),
              true, 1, p);
  }
}

}  // namespace

extern "C" wc_status wc_paged_mass_workspace(wc_ctx* ctx, const wc_paged_mass_args* a, uint64_t* bytes) {
  if (!ctx || !a || !bytes) return WC_ERR_INVALID;
  return guard(ctx, [&] {
    check_mass_args(*a);
    *bytes = mass_layout(ctx, *a).bytes;
  });
}

extern "C" wc_status wc_paged_mass(wc_ctx* ctx, void* stream, const wc_paged_mass_args* a) {
  if (!ctx || !a) return WC_ERR_INVALID;
  return guard(ctx, [&] {
    check_mass_args(*a);
    const wc_pages g = keys_only(a->pages);
    const wc_paged_batch& b = a->batch;
    check_mass(g, a->mass);
    const Run table = table_run(b.page_table, b.table_stride, b.table_cols, b.requests), lens = ints_run(b.kv_lens, b.requests),
              offsets = ints_run(b.q_offsets, b.requests + 1ll);
    const Strided K = places(g, g.k, g.k_stride, a->layer), mass = mass_places(g, a->mass, a->layer);
    need(mass.nested, "paged: mass pages must not overlap");
    need(!meets(K, mass), "paged_mass: mass must not overlap the pages");
    for (const Run& x : {table, lens, offsets})
      need(!meets_run(mass, x.p, x.bytes), "paged_mass: mass must not overlap the workspace or an input");
    MassParams p;
    std::memset(&p, 0, sizeof(p));
    p.a.K = pool(g, g.k, g.k_stride, a->layer);
    p.a.pages = g.pages;
    p.a.page_log2 = log2i(g.page_size);
    p.a.table = b.page_table;
    p.a.table_ld = int(b.table_stride);
    p.a.table_cols = b.table_cols;
    p.a.lens = b.kv_lens;
    p.a.offsets = b.q_offsets;
    p.a.T = b.rows;
    p.a.B = b.requests;
    p.a.H = b.heads;
    p.a.Hk = g.kv_heads;
    p.a.rep = b.heads / g.kv_heads;
    p.a.scale_log2 = a->scale * kLog2e;
    p.a.err = ctx->d_err;
    p.mass = {a->mass.p + a->mass.stride[0] * a->layer, a->mass.stride[0], a->mass.stride[1], a->mass.stride[2]};
    p.add = a->add;
    const cudaStream_t st = stream_of(ctx, stream);
    if (b.rows == 0) {
      DeviceScope scope(ctx->device);
      const long long heads = (long long)b.requests * g.kv_heads;
      if (!a->add)
        launch_on(ctx, st, "mass_clear", mass_clear_kernel, dim3(unsigned(std::min(heads, ctx->num_sms * 8ll))), dim3(256), 0, true, 1,
                  p);
      return;
    }
    check_rows(a->q, a->q_stride, g.dtype, "paged_mass: q must be 16-byte aligned, rows contiguous");
    const MassLayout l = mass_layout(ctx, *a);
    if (!a->workspace || reinterpret_cast<uintptr_t>(a->workspace) % 256 || a->workspace_bytes < l.bytes)
      fail(WC_ERR_CAPACITY, "paged_mass: workspace missing, misaligned or too small");
    const Run scratch{a->workspace, (long long)l.bytes},
        q = rows_run(a->q, a->q_stride, g.dtype, b.rows, b.heads, g.head_dim);
    check_apart(scratch, {q, table, lens, offsets}, "paged_mass: the workspace must not overlap an input");
    need(!meets_run(K, scratch.p, scratch.bytes), "paged_mass: the workspace must not overlap the pages");
    for (const Run& x : {scratch, q})
      need(!meets_run(mass, x.p, x.bytes), "paged_mass: mass must not overlap the workspace or an input");
    DeviceScope scope(ctx->device);
    char* ws = static_cast<char*>(a->workspace);
    p.a.q = a->q;
    p.a.q_row = a->q_stride[0];
    p.a.q_head = a->q_stride[1];
    p.a.rec = reinterpret_cast<PagedRec*>(ws + l.rec);
    p.row_ml = reinterpret_cast<float2*>(ws + l.row_ml);
    p.part_ml = reinterpret_cast<float2*>(ws + l.part_ml);
    p.tiles = reinterpret_cast<long long*>(ws + l.tiles);
    p.blocks = l.blocks;
    if (g.dtype == WC_BF16) {
      if (g.head_dim == 64) gather_mass<uint16_t, 64>(ctx, st, g, p, l, ws);
      else gather_mass<uint16_t, 128>(ctx, st, g, p, l, ws);
    } else {
      if (g.head_dim == 64) gather_mass<float, 64>(ctx, st, g, p, l, ws);
      else gather_mass<float, 128>(ctx, st, g, p, l, ws);
    }
  });
}

// ============================================================================ eviction

namespace {

void check_evict_args(const wc_paged_evict_args& a) {
  check_pages(a.pages);
  check_table(a.page_table, a.table_stride, a.table_cols, a.pages.page_size, "paged_evict: bad page table");
  need(a.requests > 0 && a.requests < (1 << 24), "paged_evict: bad request count");
  need(a.sinks >= 0 && a.recent >= 0 && a.sinks < (1 << 30) && a.recent < (1 << 30), "paged_evict: negative sinks or recent");
  need(a.budgets || a.budget >= a.sinks + a.recent, "paged_evict: budget below sinks + recent");
  need((long long)a.pages.layers * a.requests * a.pages.kv_heads < (1ll << 31), "paged_evict: batch too large");
  if ((long long)a.pages.pages * a.pages.page_size >= (1ll << 31)) fail(WC_ERR_UNSUPPORTED, "paged_evict: a pool of 2^31 keys");
}

int evict_most(const wc_paged_evict_args& a) {
  const int cap = a.table_cols * a.pages.page_size;
  return a.budgets ? cap : std::min(cap, a.budget);
}

}  // namespace

extern "C" wc_status wc_paged_evict_workspace(wc_ctx* ctx, const wc_paged_evict_args* a, uint64_t* bytes) {
  if (!ctx || !a || !bytes) return WC_ERR_INVALID;
  return guard(ctx, [&] {
    check_evict_args(*a);
    *bytes = uint64_t(a->pages.layers) * a->requests * a->pages.kv_heads * (evict_most(*a) + 1) * sizeof(int);
  });
}

extern "C" wc_status wc_paged_evict(wc_ctx* ctx, void* stream, const wc_paged_evict_args* a) {
  if (!ctx || !a) return WC_ERR_INVALID;
  return guard(ctx, [&] {
    const wc_pages& g = a->pages;
    check_evict_args(*a);
    check_mass(g, a->mass);
    need(a->kv_lens && a->lens_out, "paged_evict: null kv_lens or lens_out");
    const int most = evict_most(*a);
    const long long lists = (long long)g.layers * a->requests * g.kv_heads;
    const long long bytes = lists * (most + 1) * (long long)sizeof(int);
    if (!a->workspace || reinterpret_cast<uintptr_t>(a->workspace) % 256 || a->workspace_bytes < uint64_t(bytes))
      fail(WC_ERR_CAPACITY, "paged_evict: workspace missing, misaligned or too small");
    const Strided K = places(g, g.k, g.k_stride, -1), V = places(g, g.v, g.v_stride, -1), mass = mass_places(g, a->mass, -1);
    check_written(K, V);
    need(mass.nested, "paged: mass pages must not overlap");
    need(!meets(K, mass) && !meets(V, mass), "paged_evict: mass must not overlap the pages");
    const Run scratch{a->workspace, bytes}, out = ints_run(a->lens_out, a->requests),
              table = table_run(a->page_table, a->table_stride, a->table_cols, a->requests),
              lens = ints_run(a->kv_lens, a->requests), budgets = ints_run(a->budgets, a->requests);
    check_apart(out, {table, lens, budgets, scratch}, "paged_evict: lens_out must not overlap an input or the workspace");
    check_apart(scratch, {table, lens, budgets}, "paged_evict: the workspace must not overlap an input");
    check_pages_apart(K, V, {out, table, lens, budgets, scratch},
                      "paged_evict: the pages must not overlap lens_out, the workspace or an input");
    for (const Run& x : {out, table, lens, budgets, scratch})
      need(!meets_run(mass, x.p, x.bytes), "paged_evict: mass must not overlap lens_out, the workspace or an input");
    DeviceScope scope(ctx->device);
    EvictParams p;
    std::memset(&p, 0, sizeof(p));
    p.K = pool(g, g.k, g.k_stride, 0);
    p.V = pool(g, g.v, g.v_stride, 0);
    p.k_layer = g.k_stride[0];
    p.v_layer = g.v_stride[0];
    p.mass = {a->mass.p, a->mass.stride[0], a->mass.stride[1], a->mass.stride[2]};
    p.pages = g.pages;
    p.page_log2 = log2i(g.page_size);
    p.B = a->requests;
    p.Hk = g.kv_heads;
    p.layers = g.layers;
    p.esize_log2 = g.dtype == WC_BF16 ? 1 : 2;
    p.row_chunks = (g.head_dim << p.esize_log2) / 16;
    p.table = a->page_table;
    p.table_ld = int(a->table_stride);
    p.table_cols = a->table_cols;
    p.lens = a->kv_lens;
    p.budgets = a->budgets;
    p.budget = a->budget;
    p.sinks = a->sinks;
    p.recent = a->recent;
    p.lens_out = a->lens_out;
    p.list = static_cast<int*>(a->workspace);
    p.most = most;
    p.cache = std::min(a->table_cols * g.page_size, EV_CACHE);
    // One kernel where blocks of lists fill most of the device, else two, with rows in parts of 64 bytes or more. 8192
    // keys to 2048: 8 lists 33 us in two kernels and 66 in one, 64 lists 55 and 72, 112 lists 94 and 82, 224 lists
    // 188 and 113.
    p.splits = lists * 3 >= ctx->num_sms * 2 ? 0 : std::min(p.row_chunks / 4, 4);
    p.err = ctx->d_err;
    const cudaStream_t st = stream_of(ctx, stream);
    opt_in(ctx, evict_kernel, EV_CACHE * sizeof(float));
    launch_on(ctx, st, "evict", evict_kernel, dim3(unsigned(lists)), dim3(EV_THREADS), p.cache * sizeof(float), true, 1, p);
    if (p.splits)
      launch_on(ctx, st, "evict_move", evict_move_kernel, dim3(unsigned(lists), 2 * p.splits), dim3(EV_THREADS), 0, true, 1, p);
  });
}
