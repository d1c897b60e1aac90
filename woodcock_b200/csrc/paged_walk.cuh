// Which blocks of an attention launch do what over a paged cache: segments, the line of key tiles and its
// equal shares, the rows' sight of the keys, page numbers. Shared by the kernels of paged.cuh and
// evict.cuh.
#pragma once

#include "common.cuh"

namespace wc {

// One pool (K or V) and its strides in elements; rows are contiguous.
struct PagePool {
  void* ptr;
  long long page, head, row;
};

// Eight consecutive elements as fp32.
__device__ __forceinline__ void load8(const float* p, float (&x)[8]) {
  const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
  x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
}
__device__ __forceinline__ void load8(const uint16_t* p, float (&x)[8]) {
  const uint4 a = *reinterpret_cast<const uint4*>(p);
  const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = __uint_as_float(w[i] << 16);
    x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}
__device__ __forceinline__ void store8(float* p, const float (&x)[8]) {
  reinterpret_cast<float4*>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;\n" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ void store8(uint16_t* p, const float (&x)[8]) {
  *reinterpret_cast<uint4*>(p) =
      make_uint4(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]), pack_bf16(x[4], x[5]), pack_bf16(x[6], x[7]));
}

// ---------------------------------------------------------------------------- attention: the work
// o = softmax(scale q K^T) V for every query row, over the keys it sees. A segment is a set of rows
// that share keys: a request's rows and its own pages, or a group's rows and the group's prefix
// pages (seen whole). Query rows of a segment and KV head are numbered rho = token * rep + j (the
// rep query heads of one KV head), cut into tiles of M rows; keys into tiles of KT. An item is
// (segment, KV head, row tile); its key tiles, in one line over all items, are cut into equal
// ranges, one per block, so blocks carry equal work whatever the lengths. An item that crosses a
// cut leaves partial states (running maximum in log2 units, sum, unnormalised output), joined in
// block order by the combine kernel: no atomics, the same result every time.
enum PagedKinds : int {
  kOwnRows = 1,
  kPrefixRows = 2,
  kFewRows = 4,   // requests of at most 16 query rows a KV head alone
  kManyRows = 8,  // requests of more
};

// A divided item as the joining kernel needs it; count 0: none.
struct PagedRec {
  int tok0, rows, qt, head, count, idx, pad[2];  // rows: the segment's, times rep
};

struct PagedAttnParams {
  const void* q;
  long long q_row, q_head;
  PagePool K, V;
  int pages, page_log2;
  const int* table;
  int table_ld, table_cols;
  const int* lens;
  const int* offsets;           // [B + 1] or null: T / B rows each
  const long long* tree;        // [T] visible new rows as bits, or null: causal
  const int* prefix_table;
  int prefix_ld, prefix_cols;
  const int* prefix_lens;
  const int* groups;            // [G + 1] first request of each group
  int T, B, G, H, Hk, rep;
  float scale_log2;             // scale * log2(e)
  void* out;                    // [T][H][D]
  // workspace
  float* part_o;                // [blocks][2][M][D]
  float2* part_ml;              // [blocks][2][M]
  PagedRec* rec;                // [blocks], without prefixes: the divided item that begins in the block
  int2* desc[2];                // with prefixes, per item (own, prefix): {first block, number of blocks}
  float* whole_o[2];            // with prefixes: items of one block, [T][H][D]
  float2* whole_ml[2];          // [T][H]
  int* err;
};

struct PagedSeg {
  int prefix, idx;   // group or request
  int tok0, n, klen; // rows and keys
};

__device__ __forceinline__ int paged_row0(const PagedAttnParams& p, int b) {
  return p.offsets ? min(max(p.offsets[b], 0), p.T) : b * (p.T / p.B);
}

__device__ __forceinline__ PagedSeg paged_seg(const PagedAttnParams& p, int kinds, int s) {
  PagedSeg g;
  const int ng = (kinds & kPrefixRows) ? p.G : 0;
  g.prefix = s < ng;
  g.idx = g.prefix ? s : s - ng;
  int cap;
  if (g.prefix) {
    const int r0 = min(max(p.groups[s], 0), p.B), r1 = min(max(p.groups[s + 1], r0), p.B);
    g.tok0 = paged_row0(p, r0);
    g.n = max(0, paged_row0(p, r1) - g.tok0);
    g.klen = p.prefix_lens[s];
    cap = p.prefix_cols << p.page_log2;
  } else {
    g.tok0 = paged_row0(p, g.idx);
    g.n = max(0, paged_row0(p, g.idx + 1) - g.tok0);
    if ((kinds & kFewRows) && g.n * p.rep > 16) g.n = 0;
    if ((kinds & kManyRows) && g.n * p.rep <= 16) g.n = 0;
    g.klen = p.lens[g.idx];
    cap = p.table_cols << p.page_log2;
    if (p.tree && g.n > 64) raise_error(p.err, kErrRows);
  }
  if (g.klen < 0 || g.klen > cap) raise_error(p.err, kErrCapacity);
  g.klen = min(max(g.klen, 0), cap);
  return g;
}

// Key tiles of one row tile: at least one, so that rows without keys are answered too.
template <int M, int KT>
__device__ __forceinline__ int paged_item_tiles(const PagedAttnParams& p, const PagedSeg& g, int qt) {
  int seen = g.klen;
  if (!g.prefix && !p.tree) {
    const int last = min(g.n - 1, ((qt + 1) * M - 1) / p.rep);
    seen = min(max(g.klen - g.n + last + 1, 0), g.klen);
  }
  return max(1, (seen + KT - 1) / KT);
}

template <int M, int KT>
__device__ __forceinline__ long long paged_head_tiles(const PagedAttnParams& p, const PagedSeg& g) {
  const int qts = (g.n * p.rep + M - 1) / M;
  if (g.prefix || p.tree) return (long long)qts * paged_item_tiles<M, KT>(p, g, 0);
  // the last row of tile qt is ((qt + 1) M - 1) / rep: its quotient and remainder step from tile to tile
  const int base = g.klen - g.n + 1, dq = M / p.rep, dr = M - dq * p.rep;
  int q = (M - 1) / p.rep, r = (M - 1) - q * p.rep;
  long long n = 0;
  for (int qt = 0; qt < qts; ++qt) {
    const int seen = min(max(base + min(g.n - 1, q), 0), g.klen);
    n += max(1, (seen + KT - 1) / KT);
    q += dq;
    r += dr;
    if (r >= p.rep) {
      r -= p.rep;
      ++q;
    }
  }
  return n;
}

// a / b for a >= 0, b > 0: almost always of 32-bit values, whose division is several times shorter
__device__ __forceinline__ long long paged_div(long long a, long long b) {
  return ((a | b) >> 32) ? a / b : (long long)(uint32_t(a) / uint32_t(b));
}

// One block's walk over its range of the line, item by item. An item counts kOver units beyond its key
// tiles, for what it costs whatever its length (its queries, its result, the way there); a block whose
// range holds only such units of an item passes it over. A block takes `least` units at least, where
// more parts would cost the joining kernel more than they save.
template <int M, int KT, int kOver>
struct PagedWalk {
  PagedSeg g;
  int head, qt, qts;    // the item
  int kt0, kt1, ktn;    // this block's key tiles [kt0, kt1) of the item's ktn
  int first, count;     // the blocks that share the item
  int seg, nseg, per;
  long long pos, end;   // units of the line: the item's first one here, the block's end

  __device__ static long long units(const PagedAttnParams& p, const PagedSeg& g) {
    const int qts = (g.n * p.rep + M - 1) / M;
    return paged_head_tiles<M, KT>(p, g) + (long long)qts * kOver;
  }

  // Block-collective; `sh` holds kWalkShared words. False: the block has no work, and other warps may
  // still be reading `sh`.
  __device__ bool begin(const PagedAttnParams& p, int kinds, int least, long long* sh) {
    nseg = ((kinds & kPrefixRows) ? p.G : 0) + ((kinds & kOwnRows) ? p.B : 0);
    const int tid = threadIdx.x, nt = blockDim.x, lane = tid & 31, warp = tid >> 5, nw = (nt + 31) >> 5;
    long long total = 0, w = 0, x = 0;
    pos = 0;
    for (int pass = 0; pass < 2; ++pass) {
      if (pass) {
        per = max(least, int(paged_div(total + gridDim.x - 1, gridDim.x)));
        pos = (long long)blockIdx.x * per;
        end = min(pos + per, total);
        if (pos >= end) return false;
      }
      long long base = 0;
      for (int s0 = 0; s0 < nseg; s0 += nt) {
        const int s = s0 + tid;
        if (!pass || nseg > nt) {  // one round of segments: the first pass has it all
          w = 0;
          if (s < nseg) w = units(p, paged_seg(p, kinds, s)) * p.Hk;
          x = w;
#pragma unroll
          for (int o = 1; o < 32; o *= 2) {
            const long long y = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= o) x += y;
          }
          if (lane == 31) sh[warp] = x;
          __syncthreads();
        }
        long long before = base, all = 0;
        for (int i = 0; i < nw; ++i) {
          if (i < warp) before += sh[i];
          all += sh[i];
        }
        const long long a = before + x - w;  // the segment's first unit
        if (pass && a <= pos && pos < a + w) {
          sh[32] = s;
          sh[33] = pos - a;
          sh[34] = w;
        }
        base += all;
        if (pass || nseg > nt) __syncthreads();
      }
      total = base;
    }
    seg = int(sh[32]);
    long long off = sh[33];
    g = paged_seg(p, kinds, seg);
    qts = (g.n * p.rep + M - 1) / M;
    const long long ph = paged_div(sh[34], p.Hk);
    head = int(paged_div(off, ph));
    off -= head * ph;
    qt = 0;
    while (off >= (ktn = paged_item_tiles<M, KT>(p, g, qt)) + kOver) {
      off -= ktn + kOver;
      ++qt;
    }
    return place(int(off)) || next(p, kinds);
  }
  // begin(), and the line's beginning kept in sh for a second walk. Only where there is work: there the
  // search has ended in a barrier, while a block without work leaves between its reads of sh.
  __device__ bool begin_kept(const PagedAttnParams& p, int kinds, int least, long long* sh) {
    static_assert(sizeof(PagedWalk) <= 8 * 32, "kept where the search has been");
    if (!begin(p, kinds, least, sh)) return false;
    if (threadIdx.x == 0) *reinterpret_cast<PagedWalk*>(sh) = *this;
    return true;
  }
  // The item's tiles in this block's range; false: only units that hold no tiles.
  __device__ bool place(int off) {
    const long long item = pos - off;  // the item's first unit
    kt0 = max(0, off - kOver);
    kt1 = int(min((long long)ktn, end - item - kOver));
    first = int(paged_div(item + kOver, per));
    count = int(paged_div(item + kOver + ktn - 1, per)) - first + 1;
    pos = min(end, item + kOver + ktn);
    return kt1 > kt0;
  }
  __device__ bool next(const PagedAttnParams& p, int kinds) {
    do {
      if (pos >= end) return false;
      if (++qt == qts) {
        qt = 0;
        if (++head == p.Hk) {
          head = 0;
          do {
            g = paged_seg(p, kinds, ++seg);
          } while (g.n == 0);
          qts = (g.n * p.rep + M - 1) / M;
        }
      }
      ktn = paged_item_tiles<M, KT>(p, g, qt);
    } while (!place(0));
    return true;
  }
  // Number of the item among those of its kind and head: distinct, below T rep / M + segments + 1.
  __device__ int item(const PagedAttnParams& p) const {
    return g.tok0 * p.rep / M + g.idx + qt;  // rows x heads is below 2^30
  }
  // Where this block's share of a divided item goes: slot 0 when the item began in an earlier block.
  __device__ int slot() const { return kt0 > 0 ? 0 : 1; }
  // One thread, once per item: what the joining kernel needs to know of it.
  __device__ void report(const PagedAttnParams& p) const {
    if (kt0 > 0) return;
    if (p.G > 0) p.desc[g.prefix][item(p) * p.Hk + head] = make_int2(first, count);
    else if (count > 1) p.rec[blockIdx.x] = PagedRec{g.tok0, g.n * p.rep, qt, head, count, g.idx, {}};
  }
};
// Before the first report of a block.
__device__ __forceinline__ void paged_no_rec(const PagedAttnParams& p) {
  if (p.G == 0 && threadIdx.x == 0) p.rec[blockIdx.x] = PagedRec{};
}
constexpr int kWalkShared = 36;

// An item as the warp that walks hands it to the others; count 0: the line's end.
struct __align__(16) PagedItem {
  PagedSeg g;
  int head, qt, kt0, kt1, count, slot, pad[5];
};
static_assert(sizeof(PagedItem) == 64, "item queue");

// What one query row sees: keys below `lim`, and with a tree the new rows in `bits`.
struct PagedRow {
  bool valid;
  int tok, h;  // row and query head
  int lim;
  int base, klen;
  unsigned long long bits;
  __device__ bool sees(int key) const {
    if (key < lim) return true;
    const int i = key - base;
    return key < klen && unsigned(i) < 64u && ((bits >> i) & 1ull);
  }
};

__device__ __forceinline__ PagedRow paged_row(const PagedAttnParams& p, const PagedSeg& g, int head, int rho) {
  PagedRow r;
  r.valid = rho < g.n * p.rep;
  const int i = r.valid ? rho / p.rep : 0;
  r.tok = g.tok0 + i;
  r.h = head * p.rep + (r.valid ? rho - i * p.rep : 0);
  r.klen = g.klen;
  r.base = g.klen - g.n;
  r.bits = 0ull;
  if (g.prefix) {
    r.lim = g.klen;
  } else if (p.tree) {
    r.lim = r.base;
    if (r.valid) r.bits = (unsigned long long)p.tree[r.tok];
  } else {
    r.lim = min(r.base + i + 1, g.klen);
  }
  if (!r.valid) r.lim = 0;
  return r;
}

// Page of a segment's key, or -1 (an entry outside the pool raises the error bit).
__device__ __forceinline__ int paged_page(const PagedAttnParams& p, const PagedSeg& g, int pi) {
  if (pi >= (g.prefix ? p.prefix_cols : p.table_cols)) return -1;
  const int page = g.prefix ? p.prefix_table[(long long)g.idx * p.prefix_ld + pi]
                            : p.table[(long long)g.idx * p.table_ld + pi];
  if (page < 0 || page >= p.pages) {
    raise_error(p.err, kErrPage);
    return -1;
  }
  return page;
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;\n" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

__device__ __forceinline__ void store4(float* p, const float (&x)[4]) {
  *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
}
__device__ __forceinline__ void store4(uint16_t* p, const float (&x)[4]) {
  *reinterpret_cast<uint2*>(p) = make_uint2(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]));
}

// Waits give up after a bound; then `dead` lets the block's other waits pass, so that it ends.
__device__ __forceinline__ void paged_wait(uint64_t* bar, uint32_t parity, volatile int* dead, int* err) {
  if (mbar_wait(bar, parity, 1) || *dead) return;
  if (!mbar_wait(bar, parity)) {
    *dead = 1;
    raise_error(err, kErrTimeout);
  }
}

// The page numbers of a segment, 32 at a time over the warp's lanes and 32 more on their way.
struct PageWindow {
  int base, cur, nxt, npages, cols;
  const int* row;
  __device__ int fetch(const PagedAttnParams& p, int i) const {
    if (i >= npages || i >= cols) return p.pages;  // behind the last key: the copy fills zeros
    const int page = row[i];
    if (page < 0 || page >= p.pages) {
      raise_error(p.err, kErrPage);
      return p.pages;
    }
    return page;
  }
  __device__ void start(const PagedAttnParams& p, const PagedSeg& g, int first, int lane) {
    row = g.prefix ? p.prefix_table + (long long)g.idx * p.prefix_ld : p.table + (long long)g.idx * p.table_ld;
    cols = g.prefix ? p.prefix_cols : p.table_cols;
    npages = (g.klen + (1 << p.page_log2) - 1) >> p.page_log2;
    base = first;
    cur = fetch(p, base + lane);
    nxt = fetch(p, base + 32 + lane);
  }
  // Warp-collective: page of index i (not before the last call's window) for each lane.
  __device__ void seek(const PagedAttnParams& p, int first, int lane) {
    if (first >= base + 32) {
      base += 32;
      cur = nxt;
      nxt = fetch(p, base + 32 + lane);
    }
  }
};

}  // namespace wc
