// Entry points of the beam search operators: argument checks, workspace layout and launches of the kernels in
// beams.cuh.
#include <cstring>

#include "beams.cuh"
#include "paged_host.h"

using namespace wc;

namespace {

struct SelectLayout {
  int pieces, rounds;
  size_t stat, cand, counts, bytes;
};

SelectLayout select_layout(const wc_ctx* ctx, const wc_beam_select_args& a) {
  SelectLayout l;
  std::memset(&l, 0, sizeof(l));
  const size_t rows = size_t(a.requests) * a.beams;
  // A piece's first round costs more than later ones, and a piece of many leaves blocks idle at the end: as many rounds
  // as leave three pieces for each place on the device (64 x 8 beams over 151,936 tokens: 68 us, one piece 74,
  // two 71, four 69, eight 75).
  const long long in_row = (a.vocab + BS_ROUND - 1) / BS_ROUND, places = ctx->num_sms * 4ll;
  l.rounds = int(std::min(in_row, std::max(1ll, (long long)rows * in_row / (3 * places))));
  l.pieces = int((in_row + l.rounds - 1) / l.rounds);
  l.rounds = int((in_row + l.pieces - 1) / l.pieces);
  size_t at = 0;
  l.stat = take(at, rows * l.pieces * sizeof(double2));
  l.cand = take(at, rows * l.pieces * 2 * a.n * sizeof(unsigned long long));
  l.counts = take(at, rows * l.pieces * sizeof(int));
  l.bytes = at;
  return l;
}

void check_select(const wc_beam_select_args& a) {
  need(a.dtype == WC_F32 || a.dtype == WC_BF16, "beam_select: logits must be fp32 or bf16");
  need(a.requests > 0 && a.beams > 0 && a.vocab > 0, "beam_select: empty batch");
  if (a.beams > BS_MAX_W) fail(WC_ERR_UNSUPPORTED, "beam_select: more than 64 beams");
  need(a.n > 0, "beam_select: n must be positive");
  if (a.n > BS_MAX_N) fail(WC_ERR_UNSUPPORTED, "beam_select: n above 64");
  if ((long long)a.beams * a.vocab >= (1ll << 31) || (long long)a.requests * a.beams >= (1ll << 24) || a.vocab >= (1 << 30))
    fail(WC_ERR_UNSUPPORTED, "beam_select: too many logits");
  need(a.pad >= 0 && a.pad < a.vocab, "beam_select: pad must be a token");
}

}  // namespace

extern "C" wc_status wc_beam_select_workspace(wc_ctx* ctx, const wc_beam_select_args* a, uint64_t* bytes) {
  if (!ctx || !a || !bytes) return WC_ERR_INVALID;
  return guard(ctx, [&] {
    check_select(*a);
    *bytes = select_layout(ctx, *a).bytes;
  });
}

extern "C" wc_status wc_beam_select(wc_ctx* ctx, void* stream, const wc_beam_select_args* a) {
  if (!ctx || !a) return WC_ERR_INVALID;
  return guard(ctx, [&] {
    check_select(*a);
    const int e = int(element(a->dtype));
    need(a->logits && reinterpret_cast<uintptr_t>(a->logits) % e == 0, "beam_select: null or misaligned logits");
    need(a->request_stride >= 0 && a->beam_stride >= 0, "beam_select: negative stride");
    need(a->scores && a->out_scores && a->out_parents && a->out_tokens, "beam_select: null argument");
    const SelectLayout l = select_layout(ctx, *a);
    if (!a->workspace || reinterpret_cast<uintptr_t>(a->workspace) % 256 || a->workspace_bytes < l.bytes)
      fail(WC_ERR_CAPACITY, "beam_select: workspace missing, misaligned or too small");
    const long long rows = (long long)a->requests * a->beams, places = (long long)a->requests * a->n;
    const Run logits{a->logits, ((a->requests - 1) * a->request_stride + (a->beams - 1) * a->beam_stride + a->vocab) * e},
        scores{a->scores, rows * 4}, finished{a->finished, a->finished ? rows : 0}, scratch{a->workspace, (long long)l.bytes},
        os{a->out_scores, places * 4}, op{a->out_parents, places * 4}, ot{a->out_tokens, places * 4};
    check_apart(scratch, {logits, scores, finished, os, op, ot}, "beam_select: the workspace must not overlap another argument");
    check_apart(os, {logits, scores, finished, op, ot}, "beam_select: an output must not overlap another argument");
    check_apart(op, {logits, scores, finished, ot}, "beam_select: an output must not overlap another argument");
    check_apart(ot, {logits, scores, finished}, "beam_select: an output must not overlap another argument");
    const long long blocks = rows * l.pieces;
    if (blocks >= (1ll << 31)) fail(WC_ERR_UNSUPPORTED, "beam_select: too many logits");
    DeviceScope scope(ctx->device);
    char* ws = static_cast<char*>(a->workspace);
    BeamSelectParams p;
    std::memset(&p, 0, sizeof(p));
    p.logits = a->logits;
    p.request = a->request_stride;
    p.beam = a->beam_stride;
    p.scores = a->scores;
    p.finished = a->finished;
    p.B = a->requests;
    p.W = a->beams;
    p.V = a->vocab;
    p.n = a->n;
    p.pieces = l.pieces;
    p.rounds = l.rounds;
    p.pad = a->pad;
    p.stat = reinterpret_cast<double2*>(ws + l.stat);
    p.cand = reinterpret_cast<unsigned long long*>(ws + l.cand);
    p.counts = reinterpret_cast<int*>(ws + l.counts);
    p.out_scores = a->out_scores;
    p.out_parents = a->out_parents;
    p.out_tokens = a->out_tokens;
    p.err = ctx->d_err;
    const cudaStream_t st = stream_of(ctx, stream);
    launch_on(ctx, st, "beam_pieces", a->dtype == WC_BF16 ? beam_pieces_kernel<uint16_t> : beam_pieces_kernel<float>,
              dim3(unsigned(blocks)), dim3(BS_THREADS), 0, true, 1, p);
    launch_on(ctx, st, "beam_join", beam_join_kernel, dim3(a->requests), dim3(BJ_THREADS), 0, true, 1, p);
  });
}

extern "C" wc_status wc_beam_reorder(wc_ctx* ctx, void* stream, const wc_beam_reorder_args* a) {
  if (!ctx || !a) return WC_ERR_INVALID;
  return guard(ctx, [&] {
    const wc_pages& g = a->pages;
    check_pages(g);
    need(a->requests > 0 && a->beams > 0 && a->requests < (1 << 24), "beam_reorder: empty batch");
    if (a->beams > BS_MAX_W) fail(WC_ERR_UNSUPPORTED, "beam_reorder: more than 64 beams");
    check_table(a->page_table, a->table_stride, a->table_cols, g.page_size, "beam_reorder: bad page table");
    need(a->kv_lens && a->parents, "beam_reorder: null argument");
    need(a->table_cols == 0 || (a->table_out && a->out_stride >= a->table_cols && a->out_stride < (1ll << 31)),
         "beam_reorder: bad table_out");
    need((long long)a->beams * a->table_cols < (1ll << 31), "beam_reorder: a table of 2^31 entries or more");
    if (g.layers > 65535) fail(WC_ERR_UNSUPPORTED, "beam_reorder: more than 65535 layers");
    const int rows = a->requests * a->beams;
    const Strided K = places(g, g.k, g.k_stride, -1), V = places(g, g.v, g.v_stride, -1);
    check_written(K, V);
    const Run out = table_run(a->table_out, a->out_stride, a->table_cols, rows),
              table = table_run(a->page_table, a->table_stride, a->table_cols, rows), lens = ints_run(a->kv_lens, rows),
              parents = ints_run(a->parents, rows);
    check_apart(out, {table, lens, parents}, "beam_reorder: table_out must not overlap an input");
    check_pages_apart(K, V, {out, table, lens, parents}, "beam_reorder: the pages must not overlap table_out or an input");
    DeviceScope scope(ctx->device);
    BeamReorderParams p;
    std::memset(&p, 0, sizeof(p));
    p.K = pool(g, g.k, g.k_stride, 0);
    p.V = pool(g, g.v, g.v_stride, 0);
    p.k_layer = g.k_stride[0];
    p.v_layer = g.v_stride[0];
    p.pages = g.pages;
    p.page_log2 = log2i(g.page_size);
    p.Hk = g.kv_heads;
    p.layers = g.layers;
    p.esize_log2 = g.dtype == WC_BF16 ? 1 : 2;
    p.row_chunks = (g.head_dim << p.esize_log2) / 16;
    p.table = a->page_table;
    p.table_ld = int(a->table_stride);
    p.cols = a->table_cols;
    p.lens = a->kv_lens;
    p.parents = a->parents;
    p.table_out = a->table_out;
    p.out_ld = int(a->out_stride);
    p.W = a->beams;
    p.parts = BR_PARTS;
    p.err = ctx->d_err;
    launch_on(ctx, stream_of(ctx, stream), "beam_reorder", beam_reorder_kernel, dim3(a->requests, g.layers, p.parts),
              dim3(BR_THREADS), 0, true, 1, p);
  });
}
