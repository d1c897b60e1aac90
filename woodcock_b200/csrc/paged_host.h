// Host side of the operators over a paged cache: argument checks, workspace layout, tensor maps. Included
// by the translation units that offer them.
#pragma once

#include <algorithm>
#include <initializer_list>

#include "host.h"
#include "overlap.h"
#include "paged_walk.cuh"
#include "tcgen05.cuh"

namespace {

using wc::meets;
using wc::meets_run;
using wc::PagePool;
using wc::Strided;

void need(bool ok, const char* what) {
  if (!ok) fail(WC_ERR_INVALID, what);
}

long long element(int dtype) { return dtype == WC_BF16 ? 2 : 4; }

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

int log2i(int n) {
  int l = 0;
  while ((1 << l) < n) ++l;
  return l;
}

void check_pages(const wc_pages& g) {
  need(g.k && g.v, "paged: null pages");
  need(g.dtype == WC_F32 || g.dtype == WC_BF16, "paged: pages must be fp32 or bf16");
  if (g.head_dim != 64 && g.head_dim != 128) fail(WC_ERR_UNSUPPORTED, "paged: head_dim must be 64 or 128");
  if (g.page_size < 16 || g.page_size > 256 || (g.page_size & (g.page_size - 1)))
    fail(WC_ERR_UNSUPPORTED, "paged: page_size must be a power of two from 16 to 256");
  need(g.pages > 0 && g.kv_heads > 0 && g.layers > 0, "paged: empty pool");
  need(aligned16(g.k) && aligned16(g.v), "paged: pages must be 16-byte aligned");
  const int unit = g.dtype == WC_BF16 ? 8 : 4;
  const int sizes[4] = {g.layers, g.pages, g.kv_heads, g.page_size};
  for (int i = 0; i < 4; ++i) {
    if (sizes[i] == 1) continue;  // never stepped over
    need(g.k_stride[i] % unit == 0 && g.v_stride[i] % unit == 0, "paged: page strides must be multiples of 16 bytes");
    need(g.k_stride[i] > 0 && g.v_stride[i] > 0, "paged: pages must not overlap");
  }
}

void check_table(const int* table, long long stride, int cols, int page_size, const char* what) {
  need(cols >= 0 && (table || cols == 0) && stride >= cols && stride < (1ll << 31), what);
  need((long long)cols * page_size < (1ll << 30), "paged: a table of 2^30 keys or more");
}

PagePool pool(const wc_pages& g, const void* base, const int64_t* st, int layer) {
  PagePool r;
  r.ptr = static_cast<char*>(const_cast<void*>(base)) + st[0] * layer * element(g.dtype);
  r.page = st[1];
  r.head = st[2];
  r.row = st[3];
  return r;
}

void check_batch(const wc_pages& g, const wc_paged_batch& b) {
  need(b.requests > 0 && b.rows >= 0 && b.heads > 0, "paged: bad batch sizes");
  need(b.heads % g.kv_heads == 0, "paged: heads must be a multiple of kv_heads");
  need(b.kv_lens != nullptr, "paged: null kv_lens");
  need(b.q_offsets || b.rows % b.requests == 0, "paged: rows must be a multiple of requests without q_offsets");
  need((long long)b.rows * b.heads < (1ll << 30) && b.requests < (1 << 24), "paged: batch too large");
  check_table(b.page_table, b.table_stride, b.table_cols, g.page_size, "paged: bad page table");
}

void check_rows(const void* p, const int64_t* st, int dtype, const char* what) {
  const int unit = dtype == WC_BF16 ? 8 : 4;
  need(p != nullptr, what);
  need(aligned16(p) && st[0] % unit == 0 && st[1] % unit == 0 && st[0] >= 0 && st[1] >= 0, what);
}

// What a call writes must lie apart from what its blocks read, and from itself: nothing orders them.
struct Run {
  const void* p;
  long long bytes;
};

// Strided rows [rows][heads][head_dim] as the range from their first byte to their last.
Run rows_run(const void* p, const int64_t* st, int dtype, int rows, int heads, int head_dim) {
  return {p, ((rows - 1) * st[0] + (heads - 1) * st[1] + head_dim) * element(dtype)};
}

Run ints_run(const int* p, long long n) { return {p, p ? n * 4 : 0}; }
Run table_run(const int* p, long long stride, int cols, int n) { return ints_run(p, n > 0 ? (n - 1) * stride + cols : 0); }

void check_apart(const Run& out, std::initializer_list<Run> in, const char* what) {
  const uintptr_t o = reinterpret_cast<uintptr_t>(out.p);
  for (const Run& x : in) {
    const uintptr_t b = reinterpret_cast<uintptr_t>(x.p);
    need(!b || x.bytes <= 0 || o + out.bytes <= b || b + x.bytes <= o, what);
  }
}

// The places of one layer's pages (layer >= 0), or of all layers'.
Strided places(const wc_pages& g, const void* base, const int64_t* st, int layer) {
  const long long e = element(g.dtype);
  Strided s;
  s.at = reinterpret_cast<uintptr_t>(base) + (layer > 0 ? st[0] * layer * e : 0);
  s.run = g.head_dim * e;
  if (layer < 0) s.add(g.layers, st[0] * e);
  s.add(g.pages, st[1] * e);
  s.add(g.kv_heads, st[2] * e);
  s.add(g.page_size, st[3] * e);
  s.close();
  return s;
}

// Pages that a call writes.
void check_written(const Strided& K, const Strided& V) {
  need(K.nested && V.nested, "paged: pages must not overlap");
  need(!meets(K, V), "paged: k and v must not share their pages");
}

void check_pages_apart(const Strided& K, const Strided& V, std::initializer_list<Run> runs, const char* what) {
  for (const Run& x : runs) need(!meets_run(K, x.p, x.bytes) && !meets_run(V, x.p, x.bytes), what);
}

cudaStream_t stream_of(wc_ctx* ctx, void* s) { return s ? static_cast<cudaStream_t>(s) : ctx->stream; }

size_t take(size_t& at, size_t bytes) {
  const size_t here = at;
  at += (bytes + 255) / 256 * 256;
  return here;
}

// Dynamic shared memory above 48 KB is opted into once per kernel and device.
template <typename K>
void opt_in(const wc_ctx* ctx, K kernel, size_t bytes) {
  static std::mutex mu;
  static std::map<std::pair<int, const void*>, bool> done;
  std::lock_guard<std::mutex> lock(mu);
  bool& d = done[{ctx->device, reinterpret_cast<const void*>(kernel)}];
  if (d) return;
  CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(bytes)));
  d = true;
}

// K or V pages as a 5-D tensor (64 dims, row, half row, head, page); a copy takes `rows` rows of one page,
// and `halves` of the half rows of head_dim 128 (128 bytes, the swizzle's width), one after the other.
CUtensorMap page_map(const wc_pages& g, const PagePool& pool, int rows, int halves) {
  CUtensorMap m;
  const cuuint64_t dims[5] = {64, cuuint64_t(g.page_size), cuuint64_t(g.head_dim / 64), cuuint64_t(g.kv_heads),
                              cuuint64_t(g.pages)};
  const long long st[4] = {pool.row, 64, g.kv_heads > 1 ? pool.head : 64, g.pages > 1 ? pool.page : 64};
  const cuuint64_t strides[4] = {cuuint64_t(st[0]) * 2, cuuint64_t(st[1]) * 2, cuuint64_t(st[2]) * 2,
                                 cuuint64_t(st[3]) * 2};
  const cuuint32_t box[5] = {64, cuuint32_t(std::min(rows, g.page_size)), cuuint32_t(halves), 1, 1};
  const cuuint32_t es[5] = {1, 1, 1, 1, 1};
  const CUresult r = encode_tiled()(&m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 5, pool.ptr, dims, strides, box, es,
                                    CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                                    CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) fail(WC_ERR_INVALID, "paged: the pages' strides cannot be described to the copy engine");
  return m;
}

}  // namespace
