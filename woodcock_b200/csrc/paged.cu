// The paged-cache entry points of include/woodcock_b200.h: argument checks, workspace layout and
// launches of the kernels in paged.cuh.
#include <cmath>
#include <cstring>

#include "paged.cuh"
#include "paged_host.h"

using namespace wc;

namespace {

// base^(-2i/D) of the calling thread's last base and head dim: the powers cost 3 us of a call, and
// Python threads share a device's context.
const double* turn_frequencies(double base, int head_dim) {
  thread_local double freq[kPagedMaxHeadDim / 2], of_base = 0;
  thread_local int of_dim = 0;
  if (of_base != base || of_dim != head_dim) {
    for (int i = 0; i < head_dim / 2; ++i) freq[i] = std::pow(base, -2.0 * i / head_dim);
    of_base = base;
    of_dim = head_dim;
  }
  return freq;
}

template <typename S, typename P, int D>
void launch_append(wc_ctx* ctx, cudaStream_t st, const PagedAppendParams& p) {
  launch_on(ctx, st, "paged_append", paged_append_kernel<S, P, D>, dim3(p.T), dim3(PA_THREADS), 0, true, 1, p);
}

template <typename S, typename P>
void launch_append(wc_ctx* ctx, cudaStream_t st, const PagedAppendParams& p, int D) {
  if (D == 64) launch_append<S, P, 64>(ctx, st, p);
  else launch_append<S, P, 128>(ctx, st, p);
}

}  // namespace

extern "C" wc_status wc_paged_append(wc_ctx* ctx, void* stream, const wc_paged_append_args* a) {
  if (!ctx || !a) return WC_ERR_INVALID;
  return guard(ctx, [&] {
    const wc_pages& g = a->pages;
    const wc_paged_batch& b = a->batch;
    check_pages(g);
    check_batch(g, b);
    need(a->layer >= 0 && a->layer < g.layers, "paged_append: layer out of range");
    need(a->src_dtype == WC_F32 || a->src_dtype == WC_BF16, "paged_append: rows must be fp32 or bf16");
    if (b.rows == 0) return;
    check_rows(a->q, a->q_stride, a->src_dtype, "paged_append: q must be 16-byte aligned, rows contiguous");
    check_rows(a->k, a->k_stride, a->src_dtype, "paged_append: k must be 16-byte aligned, rows contiguous");
    check_rows(a->v, a->v_stride, a->src_dtype, "paged_append: v must be 16-byte aligned, rows contiguous");
    need(a->q_out && aligned16(a->q_out), "paged_append: q_out must be 16-byte aligned");
    const Strided K = places(g, g.k, g.k_stride, a->layer), V = places(g, g.v, g.v_stride, a->layer);
    check_written(K, V);
    const Run out{a->q_out, (long long)b.rows * b.heads * g.head_dim * element(g.dtype)};
    const Run q = rows_run(a->q, a->q_stride, a->src_dtype, b.rows, b.heads, g.head_dim),
              k = rows_run(a->k, a->k_stride, a->src_dtype, b.rows, g.kv_heads, g.head_dim),
              v = rows_run(a->v, a->v_stride, a->src_dtype, b.rows, g.kv_heads, g.head_dim),
              table = table_run(b.page_table, b.table_stride, b.table_cols, b.requests),
              lens = ints_run(b.kv_lens, b.requests), offsets = ints_run(b.q_offsets, b.requests + 1ll),
              positions = ints_run(a->positions, b.rows), qn{a->q_norm, g.head_dim * 4ll}, kn{a->k_norm, g.head_dim * 4ll};
    check_apart(out, {q, k, v, table, lens, offsets, positions, qn, kn}, "paged_append: q_out must not overlap an input");
    check_pages_apart(K, V, {out, q, k, v, table, lens, offsets, positions, qn, kn},
                      "paged_append: the pages must not overlap q_out or an input");
    need(!a->q_norm || aligned16(a->q_norm), "paged_append: q_norm must be 16-byte aligned");
    need(!a->k_norm || aligned16(a->k_norm), "paged_append: k_norm must be 16-byte aligned");
    need(a->base > 0 && std::isfinite(a->base), "paged_append: base must be positive");
    need(a->eps >= 0 && std::isfinite(a->eps), "paged_append: eps must not be negative");
    DeviceScope scope(ctx->device);
    PagedAppendParams p;
    std::memset(&p, 0, sizeof(p));
    p.q = a->q;
    p.k = a->k;
    p.v = a->v;
    p.q_row = a->q_stride[0];
    p.q_head = a->q_stride[1];
    p.k_row = a->k_stride[0];
    p.k_head = a->k_stride[1];
    p.v_row = a->v_stride[0];
    p.v_head = a->v_stride[1];
    p.q_norm = a->q_norm;
    p.k_norm = a->k_norm;
    p.eps = a->eps;
    p.q_out = a->q_out;
    p.K = pool(g, g.k, g.k_stride, a->layer);
    p.V = pool(g, g.v, g.v_stride, a->layer);
    p.pages = g.pages;
    p.page_log2 = log2i(g.page_size);
    p.table = b.page_table;
    p.table_ld = int(b.table_stride);
    p.table_cols = b.table_cols;
    p.lens = b.kv_lens;
    p.offsets = b.q_offsets;
    p.positions = a->positions;
    p.T = b.rows;
    p.B = b.requests;
    p.H = b.heads;
    p.Hk = g.kv_heads;
    p.err = ctx->d_err;
    std::memcpy(p.freq, turn_frequencies(a->base, g.head_dim), sizeof(p.freq));
    const cudaStream_t st = stream_of(ctx, stream);
    const bool sb = a->src_dtype == WC_BF16, pb = g.dtype == WC_BF16;
    if (sb && pb) launch_append<uint16_t, uint16_t>(ctx, st, p, g.head_dim);
    else if (sb) launch_append<uint16_t, float>(ctx, st, p, g.head_dim);
    else if (pb) launch_append<float, uint16_t>(ctx, st, p, g.head_dim);
    else launch_append<float, float>(ctx, st, p, g.head_dim);
  });
}

extern "C" wc_status wc_paged_compact(wc_ctx* ctx, void* stream, const wc_paged_compact_args* a) {
  if (!ctx || !a) return WC_ERR_INVALID;
  return guard(ctx, [&] {
    const wc_pages& g = a->pages;
    check_pages(g);
    check_table(a->page_table, a->table_stride, a->table_cols, g.page_size, "paged_compact: bad page table");
    need(a->requests > 0 && a->starts && a->keep && a->n_keep && a->lens_out, "paged_compact: null argument");
    need(a->max_keep > 0 && a->keep_stride >= a->max_keep && a->keep_stride < (1ll << 31), "paged_compact: bad keep list");
    if (a->max_keep > PC_MAXKEEP) fail(WC_ERR_UNSUPPORTED, "paged_compact: keep list longer than 64");
    const Strided K = places(g, g.k, g.k_stride, -1), V = places(g, g.v, g.v_stride, -1);
    check_written(K, V);
    const Run lens = ints_run(a->lens_out, a->requests), starts = ints_run(a->starts, a->requests),
              n_keep = ints_run(a->n_keep, a->requests),
              keep = table_run(a->keep, a->keep_stride, a->max_keep, a->requests),
              table = table_run(a->page_table, a->table_stride, a->table_cols, a->requests);
    check_apart(lens, {starts, keep, n_keep, table}, "paged_compact: lens_out must not overlap an input");
    check_pages_apart(K, V, {lens, starts, keep, n_keep, table},
                      "paged_compact: the pages must not overlap lens_out or an input");
    if (g.layers > 65535) fail(WC_ERR_UNSUPPORTED, "paged_compact: more than 65535 layers");
    DeviceScope scope(ctx->device);
    PagedCompactParams p;
    std::memset(&p, 0, sizeof(p));
    p.K = pool(g, g.k, g.k_stride, 0);
    p.V = pool(g, g.v, g.v_stride, 0);
    p.k_layer = g.k_stride[0];
    p.v_layer = g.v_stride[0];
    p.pages = g.pages;
    p.page_log2 = log2i(g.page_size);
    p.Hk = g.kv_heads;
    p.esize_log2 = g.dtype == WC_BF16 ? 1 : 2;
    p.row_chunks = (g.head_dim << p.esize_log2) / 16;
    p.table = a->page_table;
    p.table_ld = int(a->table_stride);
    p.table_cols = a->table_cols;
    p.starts = a->starts;
    p.keep = a->keep;
    p.keep_ld = int(a->keep_stride);
    p.max_keep = a->max_keep;
    p.n_keep = a->n_keep;
    p.lens_out = a->lens_out;
    p.err = ctx->d_err;
    launch_on(ctx, stream_of(ctx, stream), "paged_compact", paged_compact_kernel, dim3(a->requests, g.layers),
              dim3(PC_THREADS), 0, true, 1, p);
  });
}

// ============================================================================ attention

namespace {

enum Variant { kSimt, kFew, kMany128, kMany256 };

struct Launch {
  Variant variant;
  int M, blocks, least;
};

// One launch: its row tile, the blocks that share its key tiles and the units that a block takes at
// least. `rows`: query rows per segment and KV head, on average; `prefixes`: beside shared prefixes,
// where each part costs a row more states to join (eight chains of five rows under 1001 keys: 31.6 us
// with parts of one tile, 24.8 with least 4, 29.0 with 8; one decoding step alone: 12.8, 13.2, 15.3).
// bf16, 64 requests: 16 rows 168 us on the streamed kernel and 184 on tensor memory at 4000 keys, 35
// and 50 at 300; 18 rows 211 and 172 at 4000 keys, 77 and 70 at 1000, 42 and 48 at 300 (the streamed
// kernel then in a 32-row form, since removed). All of these are uniform batches; the mean tells little of
// one that mixes: 255 steps over 2000 keys 343 us, one chunk of 1024 rows over 8192 keys 89 us (256-row
// tiles), both in one call (mean 10 a head) 868 us, the chunk among 255 idle slots 489 us; 63 steps 97 us,
// with the chunk (mean 34, 128-row tiles) 165 us.
Launch plan_launch(const wc_ctx* ctx, const wc_pages& g, long long rows, bool prefixes) {
  Launch l;
  l.least = 1;
  if (g.dtype == WC_F32) {
    l.variant = kSimt;
    l.M = PS_M;
    l.blocks = ctx->num_sms * 2;
  } else {
    l.variant = rows <= 16 ? kFew : rows <= 128 ? kMany128 : kMany256;
    l.M = rows <= 16 ? 16 : rows <= 128 ? 128 : 256;
    l.blocks = ctx->num_sms;
    if (prefixes || l.variant != kFew) l.least = 4;
  }
  return l;
}

struct Layout {
  Launch own, prefix;
  size_t part_o[2], part_ml[2], rec, desc[2], whole_o[2], whole_ml[2], bytes;
};

Layout layout(const wc_ctx* ctx, const wc_paged_attention_args& a) {
  const wc_pages& g = a.pages;
  const wc_paged_batch& b = a.batch;
  const int rep = b.heads / g.kv_heads;
  Layout l;
  std::memset(&l, 0, sizeof(l));
  const long long rows = (long long)b.rows * rep;
  l.own = plan_launch(ctx, g, (rows + b.requests - 1) / b.requests, a.groups > 0);
  l.prefix = plan_launch(ctx, g, a.groups ? (rows + a.groups - 1) / a.groups : 0, true);
  size_t at = 0;
  for (int kind = 0; kind < (a.groups ? 2 : 1); ++kind) {
    const Launch& x = kind ? l.prefix : l.own;
    const size_t slots = size_t(x.blocks) * 2 * x.M;
    const size_t items = size_t((long long)b.rows * rep / x.M) + (kind ? a.groups : b.requests) + 2;
    l.part_o[kind] = take(at, slots * g.head_dim * sizeof(float));
    l.part_ml[kind] = take(at, slots * sizeof(float2));
    if (!a.groups) {
      l.rec = take(at, x.blocks * sizeof(PagedRec));
    } else {
      l.desc[kind] = take(at, items * g.kv_heads * sizeof(int2));
      l.whole_o[kind] = take(at, size_t(b.rows) * b.heads * g.head_dim * sizeof(float));
      l.whole_ml[kind] = take(at, size_t(b.rows) * b.heads * sizeof(float2));
    }
  }
  l.bytes = at;
  return l;
}

void check_attention(const wc_paged_attention_args& a) {
  check_pages(a.pages);
  check_batch(a.pages, a.batch);
  need(a.layer >= 0 && a.layer < a.pages.layers, "paged_attention: layer out of range");
  need(a.groups >= 0 && a.groups < (1 << 24), "paged_attention: bad group count");
  need(std::isfinite(a.scale) && a.scale > 0, "paged_attention: scale must be positive");
}

template <int D>
void launch_few(wc_ctx* ctx, cudaStream_t st, const wc_pages& g, const PagedAttnParams& p, int kinds, const Launch& l,
                 bool late) {
  const size_t smem = PfLayout<D>::bytes();
  static_assert(PfLayout<D>::bytes() <= kSmemOptinBytes, "shared memory");
  opt_in(ctx, paged_few_kernel<D>, smem);
  launch_on(ctx, st, "paged_few", paged_few_kernel<D>, dim3(l.blocks), dim3(PF_THREADS), smem, true, 1,
            page_map(g, p.K, PF_KT, D / 64), page_map(g, p.V, PF_KT, D / 64), p, kinds, l.least, late);
}

template <int D, bool kTwo>
void launch_many(wc_ctx* ctx, cudaStream_t st, const wc_pages& g, const PagedAttnParams& p, int kinds, const Launch& l,
                 bool late) {
  const size_t smem = PmLayout<D, kTwo>::bytes();
  static_assert(PmLayout<D, kTwo>::bytes() <= kSmemOptinBytes, "shared memory");
  opt_in(ctx, paged_many_kernel<D, kTwo>, smem);
  launch_on(ctx, st, "paged_many", paged_many_kernel<D, kTwo>, dim3(l.blocks), dim3(PM_THREADS), smem, true, 1,
            page_map(g, p.K, PM_KT, 1), page_map(g, p.V, PM_KT, D / 64), p, kinds, l.least, late);
}

template <typename S, int D>
void launch_attention(wc_ctx* ctx, cudaStream_t st, const wc_pages& g, const PagedAttnParams& p, int kinds,
                      const Launch& l, bool late) {
  if constexpr (sizeof(S) == 4) {
    opt_in(ctx, paged_simt_kernel<S, D>, paged_simt_smem<D>());
    launch_on(ctx, st, "paged_simt", paged_simt_kernel<S, D>, dim3(l.blocks), dim3(PS_THREADS), paged_simt_smem<D>(),
              true, 1, p, kinds, l.least, late);
  } else if (l.variant == kFew) {
    launch_few<D>(ctx, st, g, p, kinds, l, late);
  } else if (l.variant == kMany128) {
    launch_many<D, false>(ctx, st, g, p, kinds, l, late);
  } else {
    launch_many<D, true>(ctx, st, g, p, kinds, l, late);
  }
}

template <typename S, int D>
void attend(wc_ctx* ctx, cudaStream_t st, const wc_pages& g, PagedAttnParams p, const Layout& l, char* ws) {
  PagedCombineParams c;
  std::memset(&c, 0, sizeof(c));
  for (int kind = p.G ? 1 : 0; kind >= 0; --kind) {
    const Launch& x = kind ? l.prefix : l.own;
    p.part_o = reinterpret_cast<float*>(ws + l.part_o[kind]);
    p.part_ml = reinterpret_cast<float2*>(ws + l.part_ml[kind]);
    // The own rows' kernel needs nothing of the prefixes': it may start beside it, and waits for it at
    // its end, so that the joining kernel comes after both.
    launch_attention<S, D>(ctx, st, g, p, kind ? kPrefixRows : kOwnRows, x, p.G && !kind && ctx->pdl);
    c.part_o[kind] = p.part_o;
    c.part_ml[kind] = p.part_ml;
    c.M[kind] = x.M;
    c.blocks[kind] = x.blocks;
  }
  if (!p.G) {
    launch_on(ctx, st, "paged_join", paged_join_kernel<S, D>, dim3(l.own.blocks, l.own.M / PJ_ROWS),
              dim3(PJ_ROWS * D / 4), 0, true, 1, p, l.own.M);
  } else {
    c.a = p;
    const int heads = PC_JOIN / (D / 4);  // a block's
    launch_on(ctx, st, "paged_combine", paged_combine_kernel<S, D>, dim3(p.T, (p.H + heads - 1) / heads),
              dim3(PC_JOIN), 0, true, 1, c);
  }
}

}  // namespace

extern "C" wc_status wc_paged_attention_workspace(wc_ctx* ctx, const wc_paged_attention_args* a, uint64_t* bytes) {
  if (!ctx || !a || !bytes) return WC_ERR_INVALID;
  return guard(ctx, [&] {
    check_attention(*a);
    *bytes = layout(ctx, *a).bytes;
  });
}

extern "C" wc_status wc_paged_attention(wc_ctx* ctx, void* stream, const wc_paged_attention_args* a) {
  if (!ctx || !a) return WC_ERR_INVALID;
  return guard(ctx, [&] {
    check_attention(*a);
    const wc_pages& g = a->pages;
    const wc_paged_batch& b = a->batch;
    if (b.rows == 0) return;
    check_rows(a->q, a->q_stride, g.dtype, "paged_attention: q must be 16-byte aligned, rows contiguous");
    need(a->out && aligned16(a->out), "paged_attention: out must be 16-byte aligned");
    if (a->groups) {
      check_table(a->prefix_table, a->prefix_stride, a->prefix_cols, g.page_size, "paged_attention: bad prefix table");
      need(a->prefix_lens && a->group_offsets, "paged_attention: null prefix_lens or group_offsets");
    }
    const Layout l = layout(ctx, *a);
    if (!a->workspace || reinterpret_cast<uintptr_t>(a->workspace) % 256 || a->workspace_bytes < l.bytes)
      fail(WC_ERR_CAPACITY, "paged_attention: workspace missing, misaligned or too small");
    const Run out{a->out, (long long)b.rows * b.heads * g.head_dim * element(g.dtype)},
        scratch{a->workspace, (long long)l.bytes}, q = rows_run(a->q, a->q_stride, g.dtype, b.rows, b.heads, g.head_dim),
        table = table_run(b.page_table, b.table_stride, b.table_cols, b.requests), lens = ints_run(b.kv_lens, b.requests),
        offsets = ints_run(b.q_offsets, b.requests + 1ll), tree{a->tree_mask, a->tree_mask ? b.rows * 8ll : 0},
        ptable = table_run(a->prefix_table, a->prefix_stride, a->prefix_cols, a->groups),
        plens = ints_run(a->prefix_lens, a->groups), ends = ints_run(a->group_offsets, a->groups ? a->groups + 1ll : 0);
    check_apart(out, {q, table, lens, offsets, tree, ptable, plens, ends}, "paged_attention: out must not overlap an input");
    check_apart(scratch, {out, q, table, lens, offsets, tree, ptable, plens, ends},
                "paged_attention: the workspace must not overlap out or an input");
    check_pages_apart(places(g, g.k, g.k_stride, a->layer), places(g, g.v, g.v_stride, a->layer), {out, scratch},
                      "paged_attention: out and the workspace must not overlap the pages");
    DeviceScope scope(ctx->device);
    char* ws = static_cast<char*>(a->workspace);
    PagedAttnParams p;
    std::memset(&p, 0, sizeof(p));
    p.q = a->q;
    p.q_row = a->q_stride[0];
    p.q_head = a->q_stride[1];
    p.K = pool(g, g.k, g.k_stride, a->layer);
    p.V = pool(g, g.v, g.v_stride, a->layer);
    p.pages = g.pages;
    p.page_log2 = log2i(g.page_size);
    p.table = b.page_table;
    p.table_ld = int(b.table_stride);
    p.table_cols = b.table_cols;
    p.lens = b.kv_lens;
    p.offsets = b.q_offsets;
    p.tree = reinterpret_cast<const long long*>(a->tree_mask);
    p.prefix_table = a->prefix_table;
    p.prefix_ld = int(a->prefix_stride);
    p.prefix_cols = a->prefix_cols;
    p.prefix_lens = a->prefix_lens;
    p.groups = a->group_offsets;
    p.T = b.rows;
    p.B = b.requests;
    p.G = a->groups;
    p.H = b.heads;
    p.Hk = g.kv_heads;
    p.rep = b.heads / g.kv_heads;
    p.scale_log2 = a->scale * kLog2e;
    p.out = a->out;
    p.rec = reinterpret_cast<PagedRec*>(ws + l.rec);
    for (int i = 0; i < 2; ++i) {
      p.desc[i] = reinterpret_cast<int2*>(ws + l.desc[i]);
      p.whole_o[i] = reinterpret_cast<float*>(ws + l.whole_o[i]);
      p.whole_ml[i] = reinterpret_cast<float2*>(ws + l.whole_ml[i]);
    }
    p.err = ctx->d_err;
    const cudaStream_t st = stream_of(ctx, stream);
    if (g.dtype == WC_BF16) {
      if (g.head_dim == 64) attend<uint16_t, 64>(ctx, st, g, p, l, ws);
      else attend<uint16_t, 128>(ctx, st, g, p, l, ws);
    } else {
      if (g.head_dim == 64) attend<float, 64>(ctx, st, g, p, l, ws);
      else attend<float, 128>(ctx, st, g, p, l, ws);
    }
  });
}
