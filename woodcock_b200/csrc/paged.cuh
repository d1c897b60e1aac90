// Operators over a paged KV cache: append with rotation, ragged attention (causal or tree-masked),
// attention under shared prefixes, compaction. Pages are [pages][kv_heads][page_size][head_dim],
// any strides with contiguous rows; a request's key j lives in page table[b][j / page_size], row
// j % page_size. The device checks every page number and length it reads before it uses them.
#pragma once

#include "common.cuh"
#include "tcgen05.cuh"

namespace wc {

constexpr int kPagedMaxHeadDim = 128;

// One pool (K or V) and its strides in elements; rows are contiguous.
struct PagePool {
  void* ptr;
  long long page, head, row;
};

// ---------------------------------------------------------------------------- append
// y = x rsqrt(mean x^2 + eps) w per head (q and k, when gains are given), the rotation
// (a, b) -> (a cos - b sin, b cos + a sin) of the halves' pairs at theta_i = position * base^(-2i/D),
// then q to a dense tensor and k, v to the row's page slot.
struct PagedAppendParams {
  const void *q, *k, *v;
  long long q_row, q_head, k_row, k_head, v_row, v_head;  // strides in elements
  const float *q_norm, *k_norm;
  float eps;
  void* q_out;  // [T][H][D]
  PagePool K, V;
  int pages, page_log2;
  const int* table;
  int table_ld, table_cols;
  const int* lens;       // keys per request, the new rows included
  const int* offsets;    // [B + 1] first row of each request, or null: T / B rows each
  const int* positions;  // [T] or null: the row's slot
  int T, B, H, Hk;
  int* err;
  double freq[kPagedMaxHeadDim / 2];  // base^(-2i/D)
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

// Which request row t belongs to: the number of requests that end at or before it (block-collective;
// B when the row lies behind the last request).
__device__ __forceinline__ int request_of_row(const int* offsets, int t, int T, int B) {
  if (!offsets) return t / (T / B);
  int n = 0;
  for (int b0 = 0; b0 < B; b0 += int(blockDim.x)) {
    const int b = b0 + int(threadIdx.x);
    n += __syncthreads_count(b < B && offsets[b + 1] <= t);
  }
  return n;
}

constexpr int PA_THREADS = 128;

// Eight elements as they lie in memory.
template <typename S>
struct __align__(16) Raw8 {
  uint4 w[sizeof(S) / 2];
};
__device__ __forceinline__ void unpack8(const Raw8<float>& r, float (&x)[8]) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    x[4 * i] = __uint_as_float(r.w[i].x);
    x[4 * i + 1] = __uint_as_float(r.w[i].y);
    x[4 * i + 2] = __uint_as_float(r.w[i].z);
    x[4 * i + 3] = __uint_as_float(r.w[i].w);
  }
}
__device__ __forceinline__ void unpack8(const Raw8<uint16_t>& r, float (&x)[8]) {
  const uint32_t w[4] = {r.w[0].x, r.w[0].y, r.w[0].z, r.w[0].w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = __uint_as_float(w[i] << 16);
    x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}

// One block per row; D / 16 lanes share a head, eight pairs each. Bound by HBM on prompts (each value is
// read once and written once), by the chain request -> length -> page -> store on single rows: the
// first heads' values are on their way before that chain begins, and the next heads' while one step's
// are turned. 13.0 thousand prompt rows of 48 heads: 65 us, 4.9 TB/s, the issue slots 64% used (77 us
// without the early loads; 256 threads a block 105 us); 64 single rows: 3.9 us.
template <typename S, typename P, int D>
__global__ void __launch_bounds__(PA_THREADS) paged_append_kernel(const __grid_constant__ PagedAppendParams p) {
  constexpr int LPH = D / 16, HPB = PA_THREADS / LPH;  // lanes per head, heads per step
  __shared__ __align__(16) float cs[2][D / 2];
  pdl_launch_dependents();
  pdl_wait();
  const int t = blockIdx.x, sub = threadIdx.x % LPH;  // pairs [8 sub, 8 sub + 8)
  const int nh = p.H + 2 * p.Hk;
  auto fetch = [&](int h, Raw8<S>& lo, Raw8<S>& hi) {
    if (h >= nh) return;
    const S* x = h < p.H ? static_cast<const S*>(p.q) + t * p.q_row + h * p.q_head
                         : (h < p.H + p.Hk ? static_cast<const S*>(p.k) + t * p.k_row + (h - p.H) * p.k_head
                                           : static_cast<const S*>(p.v) + t * p.v_row + (h - p.H - p.Hk) * p.v_head);
    lo = *reinterpret_cast<const Raw8<S>*>(x + 8 * sub);
    hi = *reinterpret_cast<const Raw8<S>*>(x + D / 2 + 8 * sub);
  };
  Raw8<S> lo = {}, hi = {};
  int h = int(threadIdx.x) / LPH;
  fetch(h, lo, hi);
  const int b = request_of_row(p.offsets, t, p.T, p.B);
  if (b >= p.B) return;  // a row behind the last request
  const int row0 = p.offsets ? p.offsets[b] : b * (p.T / p.B);
  const int n = p.offsets ? p.offsets[b + 1] - row0 : p.T / p.B;
  const int slot = p.lens[b] - n + (t - row0);
  const int pi = slot >> p.page_log2;
  int page = -1;
  if (slot >= 0 && t >= row0 && pi < p.table_cols) page = p.table[(long long)b * p.table_ld + pi];
  if (page < 0 || page >= p.pages) {
    if (threadIdx.x == 0) raise_error(p.err, page < 0 && (slot < 0 || pi >= p.table_cols) ? kErrCapacity : kErrPage);
    page = -1;  // k and v are not written
  }
  if (threadIdx.x < D / 2) {
    // The angle in 64 bits: at position 10^6 a 32-bit product would be off by 0.06. Reduced to
    // [-pi, pi] before it is rounded, so the cosine is within 2^-22 of the exact one.
    constexpr double kTwoPi = 6.283185307179586476925287;
    const double a = double(p.positions ? p.positions[t] : slot) * p.freq[threadIdx.x];
    const float r = float(a - kTwoPi * rint(a * (1.0 / kTwoPi)));
    float s, c;
    sincosf(r, &s, &c);
    cs[0][threadIdx.x] = c;
    cs[1][threadIdx.x] = s;
  }
  __syncthreads();
  float c8[8], s8[8];
  load8(cs[0] + 8 * sub, c8);
  load8(cs[1] + 8 * sub, s8);
  const int r = slot & ((1 << p.page_log2) - 1);
  for (int h0 = 0; h0 < nh; h0 += HPB, h += HPB) {
    float a[8], c[8];
    unpack8(lo, a);
    unpack8(hi, c);
    fetch(h + HPB, lo, hi);
    const bool isq = h < p.H, isk = !isq && h < p.H + p.Hk;
    const float* w = isq ? p.q_norm : (isk ? p.k_norm : nullptr);
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) ss += a[i] * a[i] + c[i] * c[i];
#pragma unroll
    for (int o = 1; o < LPH; o *= 2) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    if (h >= nh) continue;
    if (w) {
      const float inv = 1.f / sqrtf(ss / float(D) + p.eps);
      float g[8];
      load8(w + 8 * sub, g);
#pragma unroll
      for (int i = 0; i < 8; ++i) a[i] *= inv * g[i];
      load8(w + D / 2 + 8 * sub, g);
#pragma unroll
      for (int i = 0; i < 8; ++i) c[i] *= inv * g[i];
    }
    if (isq || isk) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float x0 = a[i] * c8[i] - c[i] * s8[i], x1 = c[i] * c8[i] + a[i] * s8[i];
        a[i] = x0;
        c[i] = x1;
      }
    }
    P* dst;
    if (isq) {
      dst = static_cast<P*>(p.q_out) + ((long long)t * p.H + h) * D;
    } else {
      if (page < 0) continue;
      const PagePool& pool = isk ? p.K : p.V;
      dst = static_cast<P*>(pool.ptr) + page * pool.page + (isk ? h - p.H : h - p.H - p.Hk) * pool.head + r * pool.row;
    }
    store8(dst + 8 * sub, a);
    store8(dst + D / 2 + 8 * sub, c);
  }
}

// ---------------------------------------------------------------------------- compaction
// Rows start + keep[i] -> start + i of every layer, new length start + n_keep. keep is strictly
// increasing from keep[0] >= 0 (checked), so keep[i] >= i: each thread moves one 16-byte column
// chunk of all rows in order, up to eight rows read before they are written, and a row is read
// before any later step overwrites it. 64 paths of 5 over 28 layers: 13.8 us, 4.3 TB/s:
// 1792 blocks of 54 registers a thread are three waves, and each walks the chain start -> list -> page
// -> row anew (profile: DRAM at 23% of nominal, 43% of the warps; stalls on that chain, the barrier and
// the lists in shared memory).
constexpr int PC_THREADS = 256;
constexpr int PC_MAXKEEP = 64;

struct PagedCompactParams {
  PagePool K, V;
  long long k_layer, v_layer;  // layer strides in elements
  int pages, page_log2, Hk, row_chunks;  // 16-byte pieces of a row
  int esize_log2;
  const int* table;
  int table_ld, table_cols;
  const int* starts;
  const int* keep;  // [B][keep_ld]
  int keep_ld, max_keep;
  const int* n_keep;
  int* lens_out;
  int* err;
};

__global__ void __launch_bounds__(PC_THREADS) paged_compact_kernel(const __grid_constant__ PagedCompactParams p) {
  __shared__ int s_src[PC_MAXKEEP], s_dst[PC_MAXKEEP], s_sr[PC_MAXKEEP], s_dr[PC_MAXKEEP];
  pdl_launch_dependents();
  pdl_wait();
  const int b = blockIdx.x, layer = blockIdx.y;
  const int start = p.starts[b], nk = p.n_keep[b];
  const int mask = (1 << p.page_log2) - 1;
  bool bad = nk < 0 || nk > p.max_keep || start < 0;
  if (!bad && int(threadIdx.x) < nk) {
    const int i = threadIdx.x;
    const int* keep = p.keep + (long long)b * p.keep_ld;
    const int k = keep[i];
    const long long from = (long long)start + k;
    bad = k < 0 || (i > 0 && k <= keep[i - 1]) || (from >> p.page_log2) >= p.table_cols;
    if (!bad) {
      const int to = start + i;
      const int ps = p.table[(long long)b * p.table_ld + int(from >> p.page_log2)];
      const int pd = p.table[(long long)b * p.table_ld + (to >> p.page_log2)];
      bad = ps < 0 || ps >= p.pages || pd < 0 || pd >= p.pages;
      s_src[i] = ps;
      s_sr[i] = int(from) & mask;
      s_dst[i] = pd;
      s_dr[i] = to & mask;
    }
  }
  if (__syncthreads_or(bad)) {
    if (threadIdx.x == 0) raise_error(p.err, kErrTree);
    if (layer == 0 && threadIdx.x == 0) p.lens_out[b] = start;
    return;
  }
  if (layer == 0 && threadIdx.x == 0) p.lens_out[b] = start + nk;
  int first = 0;  // the rows before the first gap stay where they are
  while (first < nk && s_src[first] == s_dst[first] && s_sr[first] == s_dr[first]) ++first;
  const int units = 2 * p.Hk * p.row_chunks;
  for (int u = threadIdx.x; u < units; u += PC_THREADS) {
    const int chunk = u % p.row_chunks, hv = u / p.row_chunks, head = hv >> 1;
    const PagePool& pool = (hv & 1) ? p.V : p.K;
    char* base = static_cast<char*>(pool.ptr) +
                 ((((hv & 1) ? p.v_layer : p.k_layer) * layer + head * pool.head) << p.esize_log2) + chunk * 16;
    for (int i0 = first; i0 < nk; i0 += 8) {
      uint4 x[8];
      const int m = min(8, nk - i0);
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (j < m)
          x[j] = *reinterpret_cast<const uint4*>(
              base + ((s_src[i0 + j] * pool.page + s_sr[i0 + j] * pool.row) << p.esize_log2));
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (j < m && (s_src[i0 + j] != s_dst[i0 + j] || s_sr[i0 + j] != s_dr[i0 + j]))
          *reinterpret_cast<uint4*>(base + ((s_dst[i0 + j] * pool.page + s_dr[i0 + j] * pool.row) << p.esize_log2)) = x[j];
    }
  }
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
enum PagedKinds : int { kOwnRows = 1, kPrefixRows = 2 };

// A divided item as the joining kernel needs it; count 0: none.
struct PagedRec {
  int tok0, rows, qt, head, count, pad[3];  // rows: the segment's, times rep
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
    else if (count > 1) p.rec[blockIdx.x] = PagedRec{g.tok0, g.n * p.rep, qt, head, count, {}};
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

__device__ __forceinline__ void store4(float* p, const float (&x)[4]) {
  *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
}
__device__ __forceinline__ void store4(uint16_t* p, const float (&x)[4]) {
  *reinterpret_cast<uint2*>(p) = make_uint2(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]));
}

// ---------------------------------------------------------------------------- attention on the CUDA cores
// 16 query rows x 64 keys per tile, 8 warps: scores with one key and four rows per thread, the
// softmax of two rows per warp, then the same warp's rows of P V with four columns per thread. For fp32
// pages; 8 requests of 5 rows over 600 keys, 4 heads of 64: 13 us, bound by latency.
constexpr int PS_THREADS = 256, PS_M = 16, PS_KT = 64;

template <int D>
constexpr size_t paged_simt_smem() {
  return sizeof(float) * (size_t(2) * PS_KT * (D + 4) + PS_M * D + PS_M * (PS_KT + 4)) + 8 * kWalkShared;
}

template <typename S, int D>
__global__ void __launch_bounds__(PS_THREADS)
    paged_simt_kernel(const __grid_constant__ PagedAttnParams p, int kinds, int least, bool late) {
  constexpr int M = PS_M, KT = PS_KT, LD = D + 4, LS = KT + 4;
  constexpr int RPT = D / 64;  // rows per thread of P V: two (D 128), one (D 64)
  extern __shared__ __align__(16) float ps_smem[];
  float* ks = ps_smem;
  float* vs = ks + KT * LD;
  float* qs = vs + KT * LD;
  float* ss = qs + M * D;
  long long* sh = reinterpret_cast<long long*>(ss + M * LS);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (!late) pdl_wait();
  pdl_launch_dependents();
  PagedWalk<M, KT, 1> w;
  paged_no_rec(p);
  if (!w.begin(p, kinds, least, sh)) {
    if (late) pdl_wait();
    return;
  }
  do {
    __syncthreads();
    for (int c = tid; c < M * (D / 8); c += PS_THREADS) {
      const int m = c / (D / 8), col = (c % (D / 8)) * 8;
      const PagedRow r = paged_row(p, w.g, w.head, w.qt * M + m);
      float x[8] = {};
      if (r.valid) load8(static_cast<const S*>(p.q) + r.tok * p.q_row + r.h * p.q_head + col, x);
      store8(qs + m * D + col, x);
    }
    const int sk = tid & 63, sr = (tid >> 6) * 4;
    PagedRow rows[2];  // the warp's rows
#pragma unroll
    for (int i = 0; i < 2; ++i) rows[i] = paged_row(p, w.g, w.head, w.qt * M + 2 * warp + i);
    float m2[2] = {-INFINITY, -INFINITY}, l2[2] = {0.f, 0.f};
    float o[RPT][4] = {};
    const int col = (lane % (D / 4)) * 4, prow = 2 * warp + (D == 64 ? lane / 16 : 0);
    for (int kt = w.kt0; kt < w.kt1; ++kt) {
      __syncthreads();
      for (int c = tid; c < KT * (D / 8); c += PS_THREADS) {
        const int kr = c / (D / 8), cc = (c % (D / 8)) * 8, key = kt * KT + kr;
        float x[8] = {}, y[8] = {};
        const int page = key < w.g.klen ? paged_page(p, w.g, key >> p.page_log2) : -1;
        if (page >= 0) {
          const int r = key & ((1 << p.page_log2) - 1);
          load8(static_cast<const S*>(p.K.ptr) + page * p.K.page + w.head * p.K.head + r * p.K.row + cc, x);
          load8(static_cast<const S*>(p.V.ptr) + page * p.V.page + w.head * p.V.head + r * p.V.row + cc, y);
        }
        store8(ks + kr * LD + cc, x);
        store8(vs + kr * LD + cc, y);
      }
      __syncthreads();
      float s[4] = {};
#pragma unroll 8
      for (int d = 0; d < D; d += 4) {
        const float4 k4 = *reinterpret_cast<const float4*>(ks + sk * LD + d);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float4 q4 = *reinterpret_cast<const float4*>(qs + (sr + i) * D + d);
          s[i] = fmaf(q4.x, k4.x, fmaf(q4.y, k4.y, fmaf(q4.z, k4.z, fmaf(q4.w, k4.w, s[i]))));
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) ss[(sr + i) * LS + sk] = s[i];
      __syncthreads();
      float alpha[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float z[2], mx = -INFINITY;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          z[h] = ss[(2 * warp + i) * LS + lane + 32 * h] * p.scale_log2;
          if (!rows[i].sees(kt * KT + lane + 32 * h)) z[h] = -INFINITY;
          mx = fmaxf(mx, z[h]);
        }
        mx = fmaxf(warp_max(mx), m2[i]);
        const float mg = mx == -INFINITY ? 0.f : mx;
        alpha[i] = exp2f(m2[i] - mg);
        const float e0 = exp2f(z[0] - mg), e1 = exp2f(z[1] - mg);
        l2[i] = l2[i] * alpha[i] + warp_sum(e0 + e1);
        m2[i] = mx;
        ss[(2 * warp + i) * LS + lane] = e0;
        ss[(2 * warp + i) * LS + lane + 32] = e1;
      }
      __syncwarp();
#pragma unroll
      for (int i = 0; i < RPT; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[i][e] *= D == 64 ? (lane < 16 ? alpha[0] : alpha[1]) : alpha[i];
      // a key of weight zero adds nothing, whatever its value holds
      for (int k = 0; k < KT; ++k) {
        const float4 v = *reinterpret_cast<const float4*>(vs + k * LD + col);
#pragma unroll
        for (int i = 0; i < RPT; ++i) {
          const float e = ss[(prow + i) * LS + k];
          if (e != 0.f) {
            o[i][0] = fmaf(e, v.x, o[i][0]);
            o[i][1] = fmaf(e, v.y, o[i][1]);
            o[i][2] = fmaf(e, v.z, o[i][2]);
            o[i][3] = fmaf(e, v.w, o[i][3]);
          }
        }
      }
    }
    if (tid == 0) w.report(p);
#pragma unroll
    for (int i = 0; i < RPT; ++i) {
      const int ri = D == 64 ? lane / 16 : i;
      const PagedRow& r = rows[ri];
      if (!r.valid) continue;
      const float m = ri ? m2[1] : m2[0], l = ri ? l2[1] : l2[0];
      if (w.count == 1 && p.G == 0) {
        const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
        float y[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = o[i][e] * inv;
        store4(static_cast<S*>(p.out) + ((long long)r.tok * p.H + r.h) * D + col, y);
      } else {
        float* po;
        float2* pm;
        if (w.count == 1) {
          const long long at = (long long)r.tok * p.H + r.h;
          po = p.whole_o[w.g.prefix] + at * D;
          pm = p.whole_ml[w.g.prefix] + at;
        } else {
          const long long at = ((long long)blockIdx.x * 2 + w.slot()) * M + prow + i;
          po = p.part_o + at * D;
          pm = p.part_ml + at;
        }
        store4(po + col, o[i]);
        if (col == 0) *pm = make_float2(m, l);
      }
    }
  } while (w.next(p, kinds));
  if (late) pdl_wait();
}

// A row's state over keys [k0, k1), key by key and without those that it does not see: the slow way,
// warp-collective, for rows beside a value that is not finite.
template <int D>
__device__ __forceinline__ void paged_redo_row(const PagedAttnParams& p, const PagedSeg& g, const PagedRow& r, int head,
                                               int k0, int k1, int lane, float& M, float& L, float (&o)[D / 32]) {
  constexpr int E = D / 32;
  M = -INFINITY;
  L = 0.f;
  float q[E];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    o[e] = 0.f;
    q[e] = bf16_bits_to_f32(static_cast<const uint16_t*>(p.q)[r.tok * p.q_row + r.h * p.q_head + lane * E + e]);
  }
#pragma unroll 1
  for (int key = k0; key < min(k1, g.klen); ++key) {
    if (!r.sees(key)) continue;
    const int page = paged_page(p, g, key >> p.page_log2), pr = key & ((1 << p.page_log2) - 1);
    float v[E] = {}, z = 0.f;
    if (page >= 0) {
      const uint16_t* kp = static_cast<const uint16_t*>(p.K.ptr) + page * p.K.page + head * p.K.head + pr * p.K.row + lane * E;
      const uint16_t* vp = static_cast<const uint16_t*>(p.V.ptr) + page * p.V.page + head * p.V.head + pr * p.V.row + lane * E;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        z = fmaf(q[e], bf16_bits_to_f32(kp[e]), z);
        v[e] = bf16_bits_to_f32(vp[e]);
      }
    }
    z = warp_sum(z) * p.scale_log2;
    const float mn = fmaxf(M, z), mg = mn == -INFINITY ? 0.f : mn;
    const float wa = exp2f(M - mg), wb = exp2f(z - mg);
    M = mn;
    L = L * wa + wb;
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = o[e] * wa + wb * v[e];
  }
}

// ---------------------------------------------------------------------------- few rows: streamed pages
// Decoding steps and short chains: at most 16 rows against each key, so the pages' bytes bound the
// time. One producer warp streams 64-key tiles of K and V (TMA, 128-byte swizzle, a page's rows per
// copy) through a ring that fills most of shared memory; two sets of four consumer warps take the
// tiles in turn, a 16-key slice per warp, so that no two warps wait for one another before the item's
// end: each keeps its own running maximum, sum and 16 x D output (mma m16n8k16), joined in shared
// memory once per item. The producer also walks the line and hands the items over with their query
// rows, one item ahead. 64 requests of 6000 keys, pages of 64: 239 us, 6.6 TB/s; pages of 16 263 us
// (4 KB copies).
constexpr int PF_CONSUMERS = 8;
constexpr int PF_THREADS = 32 * (PF_CONSUMERS + 1);
constexpr int PF_KT = 64, PF_M = 16;
constexpr int PF_OVER = 4;  // own parts under 4 prefixes: with 1 145 us, with 4 133

template <int D>
struct PfLayout {
  static constexpr int M = PF_M;
  static constexpr int kTile = PF_KT * D * 2;          // K or V of one tile
  static constexpr int kStage = 2 * kTile;
  static constexpr int kJoin = 4 * 16 * D * 4;         // four 16-row partial outputs
  static constexpr int kQRow = (D + 8) * 2;            // a query row, padded against bank conflicts
  static constexpr int kQ = 2 * M * kQRow;             // two items' queries
  static constexpr int kTail = 8 * kWalkShared + 256 + 8 * 16 * 8 + M * 8 + 2 * 64;
  static constexpr int kStages = (int(kSmemOptinBytes) - 1024 - kJoin - kQ - kTail) / kStage;
  static constexpr size_t bytes() { return 1024 + size_t(kStages) * kStage + kJoin + kQ + kTail; }
};

// Waits give up after a bound; then `dead` lets the block's other waits pass, so that it ends.
__device__ __forceinline__ void paged_wait(uint64_t* bar, uint32_t parity, volatile int* dead, int* err) {
  if (*dead) return;
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

template <int D>
__global__ void __launch_bounds__(PF_THREADS, 1)
    paged_few_kernel(const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv,
                     const __grid_constant__ PagedAttnParams p, int kinds, int least, bool late) {
  constexpr int M = PF_M, KT = PF_KT, NK = D / 16, ND = D / 8;
  using L = PfLayout<D>;
  constexpr int NST = L::kStages;
  extern __shared__ unsigned char pf_raw[];
  unsigned char* sm = pf_raw + ((1024u - (smem_addr(pf_raw) & 1023u)) & 1023u);
  float* join = reinterpret_cast<float*>(sm + size_t(NST) * L::kStage);
  unsigned char* qbuf = reinterpret_cast<unsigned char*>(join) + L::kJoin;
  unsigned char* tail = qbuf + L::kQ;
  long long* sh = reinterpret_cast<long long*>(tail);
  uint64_t* it_full = reinterpret_cast<uint64_t*>(tail + 8 * kWalkShared);  // [2] items handed over
  uint64_t* it_empty = it_full + 2;
  uint64_t* full = it_full + 4;
  uint64_t* empty = full + NST;
  volatile int* dead = reinterpret_cast<volatile int*>(tail + 8 * kWalkShared + 248);
  volatile int* stop = dead + 1;
  float2* wml = reinterpret_cast<float2*>(tail + 8 * kWalkShared + 256);  // [8 warps][16 rows]
  float2* rml = wml + 8 * 16;                                            // [M]
  PagedItem* items = reinterpret_cast<PagedItem*>(rml + M);              // [2]
  static_assert(32 + 16 * NST <= 248, "barriers");
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    for (int s = 0; s < NST; ++s) {
      mbar_init(full + s, 1);
      mbar_init(empty + s, PF_CONSUMERS);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(it_full + s, 1);
      mbar_init(it_empty + s, PF_CONSUMERS);
    }
    mbar_fence_init();
    *dead = 0;
  }
  if (!late) pdl_wait();
  pdl_launch_dependents();
  PagedWalk<M, KT, PF_OVER> w;
  paged_no_rec(p);
  __syncthreads();
  if (!w.begin(p, kinds, least, sh)) {
    if (late) pdl_wait();
    return;
  }

  if (warp == PF_CONSUMERS) {  // ---- producer
    const int psize = 1 << p.page_log2;
    const int box = min(psize, KT), parts = KT / box;  // copies of K and of V per tile
    const int part = lane >> 1;
    const bool isv = lane & 1, issue = part < parts;
    int cnt = 0, nitem = 0;
    bool more = true;
    do {
      // the item and its query rows (those past the segment's keep what the buffer holds: nobody reads them)
      const int b = nitem & 1;
      PageWindow win;
      win.start(p, w.g, (w.kt0 * KT) >> p.page_log2, lane);
      if (lane == 0) {
        w.report(p);
        if (nitem >= 2) paged_wait(it_empty + b, ((nitem >> 1) - 1) & 1, dead, p.err);
        items[b] = PagedItem{w.g, w.head, w.qt, w.kt0, w.kt1, w.count, w.slot(), {}};
        const int rows = min(M, w.g.n * p.rep - w.qt * M);
        if (!*dead) mbar_arrive_expect_tx(it_full + b, rows * D * 2);
      }
      __syncwarp();
      if (*dead) break;
      {
        const PagedRow r = paged_row(p, w.g, w.head, w.qt * M + lane);
        if (lane < M && r.valid)
          bulk_g2s(qbuf + (b * M + lane) * L::kQRow,
                   static_cast<const uint16_t*>(p.q) + r.tok * p.q_row + r.h * p.q_head, D * 2, it_full + b);
      }
      ++nitem;
      for (int kt = w.kt0; kt < w.kt1; ++kt, ++cnt) {
        const int s = cnt % NST;
        const int first = (kt * KT) >> p.page_log2;
        win.seek(p, first, lane);
        const int page = __shfl_sync(0xffffffffu, win.cur, (first - win.base + part) & 31);
        if (lane == 0) {
          if (cnt >= NST) paged_wait(empty + s, ((cnt / NST) - 1) & 1, dead, p.err);
          if (!*dead) mbar_arrive_expect_tx(full + s, L::kStage);
        }
        __syncwarp();
        if (*dead) break;
        if (issue)
          tma_load_5d(sm + size_t(s) * L::kStage + (isv ? L::kTile : 0) + part * box * (D * 2), isv ? &tv : &tk, 0,
                      (kt * KT) & (psize - 1), 0, w.head, page, full + s);
        __syncwarp();
      }
      more = !*dead && w.next(p, kinds);
    } while (more);
    if (lane == 0) {
      const int b = nitem & 1;
      if (nitem >= 2) paged_wait(it_empty + b, ((nitem >> 1) - 1) & 1, dead, p.err);
      const bool closed = !*dead;
      if (closed) {  // an item without blocks ends the line
        items[b].count = 0;
        mbar_arrive(it_full + b);
      }
      // shared memory must outlive the copies
      for (int q = max(0, cnt - NST); q < cnt; ++q)
        if (!mbar_wait(full + q % NST, (q / NST) & 1)) raise_error(p.err, kErrTimeout);
      for (int q = max(0, nitem - (closed ? 1 : 2)); q < nitem; ++q)  // the closing item's buffer was empty
        if (!mbar_wait(it_full + (q & 1), (q >> 1) & 1)) raise_error(p.err, kErrTimeout);
    }
    __syncwarp();
    if (late) pdl_wait();
    return;
  }

  // ---- consumers
  const int g = lane >> 2, t = lane & 3;
  const int slice = warp & 3;
  const float sl2 = p.scale_log2;
  // a copy's rows lie together, half rows of 128 bytes one after the other
  const int box = min(1 << p.page_log2, KT), hstride = box * 128;
  const int slice_at = (slice * 16 / box) * box * (D * 2) + (slice * 16 % box) * 128;
  int cnt = 0;
  for (int nitem = 0;; ++nitem) {
    // One thread says for all of them whether the line goes on: the warps meet at the item's end, so
    // none may leave alone. The barrier also frees the joining space of the item before.
    const int b = nitem & 1;
    paged_wait(it_full + b, (nitem >> 1) & 1, dead, p.err);
    if (tid == 0) *stop = *dead || items[b].count == 0;
    named_sync(1, 32 * PF_CONSUMERS);
    if (*stop) break;
    const PagedItem it = items[b];
    const PagedRow ra = paged_row(p, it.g, it.head, it.qt * M + g);
    const PagedRow rb = paged_row(p, it.g, it.head, it.qt * M + g + 8);
    uint32_t qa[NK][4];
#pragma unroll
    for (int kk = 0; kk < NK; ++kk)
      ldsm_x4(qa[kk], qbuf + (b * M + (lane & 15)) * L::kQRow + kk * 32 + (lane >> 4) * 16);
    __syncwarp();
    if (lane == 0) mbar_arrive(it_empty + b);
    // rows that pad the tile count as seeing everything: their results go nowhere
    const int lim0 = ra.valid ? ra.lim : 0x7fffffff, lim1 = rb.valid ? rb.lim : 0x7fffffff;
    const int lim = min(lim0, lim1);
    float o[ND][4];
#pragma unroll
    for (int j = 0; j < ND; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[j][e] = 0.f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};

    for (int kt = it.kt0; kt < it.kt1; ++kt, ++cnt) {
      const int s = cnt % NST;
      paged_wait(full + s, (cnt / NST) & 1, dead, p.err);
      if ((cnt & 1) != (warp >> 2)) {
        // The other set's tile. Its phases are waited for and passed on all the same: a set that met a
        // stage only every other use could take an earlier use, which a wait by parity does not tell
        // apart, for its own.
        if (lane == 0) mbar_arrive(empty + s);
        continue;
      }
      const unsigned char* kb = sm + size_t(s) * L::kStage + slice_at;  // the slice's first key
      const unsigned char* vb = kb + L::kTile;
      // ---- S = Q K^T, 16 keys: the dims in two chains of each n-tile
      float sc[2][4], sx[2][4];
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) sc[j][e] = sx[j][e] = 0.f;
#pragma unroll
      for (int i = 0; i < D / 32; ++i) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          uint32_t b[4];
          const int chunk = (i & 1) * 4 + (lane >> 3);
          ldsm_x4(b, kb + (i >> 1) * hstride + (j * 8 + (lane & 7)) * 128 + ((chunk ^ (lane & 7)) << 4));
          mma_bf16_16816r(sc[j], qa[2 * i], b[0], b[1]);
          mma_bf16_16816r(sx[j], qa[2 * i + 1], b[2], b[3]);
        }
      }
      // ---- visibility, scale, running maximum
      const int key0 = kt * KT + slice * 16;
      const bool masked = key0 + 16 > lim;
      float tm[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float v = (sc[j][e] + sx[j][e]) * sl2;
          if (masked) {
            const int key = key0 + j * 8 + 2 * t + (e & 1);
            if ((e & 2) ? (rb.valid && !rb.sees(key)) : (ra.valid && !ra.sees(key))) v = -INFINITY;
          }
          sc[j][e] = v;
          tm[e >> 1] = fmaxf(tm[e >> 1], v);
        }
      float alpha[2], mg[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        tm[h] = fmaxf(tm[h], __shfl_xor_sync(0xffffffffu, tm[h], 1));
        tm[h] = fmaxf(tm[h], __shfl_xor_sync(0xffffffffu, tm[h], 2));
        const float mn = fmaxf(m[h], tm[h]);
        mg[h] = mn == -INFINITY ? 0.f : mn;
        alpha[h] = ex2_approx(m[h] - mg[h]);
        m[h] = mn;
      }
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) sc[j][e] = ex2_approx(sc[j][e] - mg[e >> 1]);
      l[0] = l[0] * alpha[0] + (sc[0][0] + sc[0][1]) + (sc[1][0] + sc[1][1]);
      l[1] = l[1] * alpha[1] + (sc[0][2] + sc[0][3]) + (sc[1][2] + sc[1][3]);
      if (__any_sync(0xffffffffu, alpha[0] != 1.f || alpha[1] != 1.f)) {
#pragma unroll
        for (int j = 0; j < ND; ++j) {
          o[j][0] *= alpha[0];
          o[j][1] *= alpha[0];
          o[j][2] *= alpha[1];
          o[j][3] *= alpha[1];
        }
      }
      // A masked place may hold anything: where the slice's values are not all finite, the product
      // is summed without the keys of weight zero (0 x NaN would reach every row).
      bool clean = true;
      if (__any_sync(0xffffffffu, masked)) {
        const unsigned char* vr = vb + (lane & 15) * 128 + (lane >> 4) * 64;
        uint32_t worst = 0;
#pragma unroll
        for (int h = 0; h < D / 64; ++h)
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const uint4 x = *reinterpret_cast<const uint4*>(vr + h * hstride + c * 16);
            const uint32_t xs[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              worst = max(worst, xs[q] & 0x7f800000u);
              worst = max(worst, (xs[q] << 16) & 0x7f800000u);
            }
          }
        clean = !__any_sync(0xffffffffu, worst == 0x7f800000u);
      }
      if (clean) {
        // ---- O += P V; the weights are rounded to bf16, as the values are: at most 2^-8 of each, as much
        // as the output's own rounding. The row's sum takes them unrounded. Two bf16 terms, as the
        // contiguous kernels keep, would double this product.
        const uint32_t a[4] = {pack_bf16(sc[0][0], sc[0][1]), pack_bf16(sc[0][2], sc[0][3]),
                               pack_bf16(sc[1][0], sc[1][1]), pack_bf16(sc[1][2], sc[1][3])};
#pragma unroll
        for (int dj = 0; dj < ND; dj += 2) {
          uint32_t b[4];
          const int key = lane & 15, chunk = dj + (lane >> 4);
          ldsm_x4_trans(b, vb + (chunk >> 3) * hstride + key * 128 + (((chunk & 7) ^ (key & 7)) << 4));
          mma_bf16_16816r(o[dj], a, b[0], b[1]);
          mma_bf16_16816r(o[dj + 1], a, b[2], b[3]);
        }
      } else {
#pragma unroll 1
        for (int c = 0; c < 16; ++c) {
          const int from = (lane & ~3) | ((c & 7) >> 1);
          const float x0 = c < 8 ? ((c & 1) ? sc[0][1] : sc[0][0]) : ((c & 1) ? sc[1][1] : sc[1][0]);
          const float x1 = c < 8 ? ((c & 1) ? sc[0][3] : sc[0][2]) : ((c & 1) ? sc[1][3] : sc[1][2]);
          const float p0 = __shfl_sync(0xffffffffu, x0, from), p1 = __shfl_sync(0xffffffffu, x1, from);
#pragma unroll
          for (int dj = 0; dj < ND; ++dj) {
            const uint32_t v = *reinterpret_cast<const uint32_t*>(vb + (dj >> 3) * hstride + c * 128 +
                                                                  (((dj & 7) ^ (c & 7)) << 4) + 4 * t);
            const float v0 = __uint_as_float(v << 16), v1 = __uint_as_float(v & 0xffff0000u);
            if (p0 != 0.f) {
              o[dj][0] = fmaf(p0, v0, o[dj][0]);
              o[dj][1] = fmaf(p0, v1, o[dj][1]);
            }
            if (p1 != 0.f) {
              o[dj][2] = fmaf(p1, v0, o[dj][2]);
              o[dj][3] = fmaf(p1, v1, o[dj][3]);
            }
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(empty + s);
    }

    // ---- the warps' states of this item joined: rows' maxima and sums, then the outputs in two steps
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
      l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
      if (t == 0) wml[warp * 16 + g + 8 * h] = make_float2(m[h], l[h]);
    }
    named_sync(1, 32 * PF_CONSUMERS);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float mx = -INFINITY, sum = 0.f;
#pragma unroll
      for (int q = 0; q < PF_CONSUMERS; ++q) mx = fmaxf(mx, wml[q * 16 + g + 8 * h].x);
      const float mgx = mx == -INFINITY ? 0.f : mx;
#pragma unroll
      for (int q = 0; q < PF_CONSUMERS; ++q) {
        const float2 x = wml[q * 16 + g + 8 * h];
        sum += x.y * ex2_approx(x.x - mgx);
      }
      const float f = ex2_approx(m[h] - mgx);
#pragma unroll
      for (int j = 0; j < ND; ++j) {
        o[j][2 * h] *= f;
        o[j][2 * h + 1] *= f;
      }
      if (warp == 0 && t == 0) rml[g + 8 * h] = make_float2(mx, sum);
    }
    float* mine = join + (warp & 3) * 16 * D;
    auto at = [&](int row, int col) { return row * D + (col ^ ((row & 3) << 3)); };  // spreads rows over the banks
    if (warp >= 4) {
#pragma unroll
      for (int j = 0; j < ND; ++j) {
        *reinterpret_cast<float2*>(mine + at(g, j * 8 + 2 * t)) = make_float2(o[j][0], o[j][1]);
        *reinterpret_cast<float2*>(mine + at(g + 8, j * 8 + 2 * t)) = make_float2(o[j][2], o[j][3]);
      }
    }
    named_sync(1, 32 * PF_CONSUMERS);
    if (warp < 4) {
#pragma unroll
      for (int j = 0; j < ND; ++j) {
        float2* x0 = reinterpret_cast<float2*>(mine + at(g, j * 8 + 2 * t));
        float2* x1 = reinterpret_cast<float2*>(mine + at(g + 8, j * 8 + 2 * t));
        *x0 = make_float2(x0->x + o[j][0], x0->y + o[j][1]);
        *x1 = make_float2(x1->x + o[j][2], x1->y + o[j][3]);
      }
    }
    named_sync(1, 32 * PF_CONSUMERS);
    for (int c = tid; c < M * (D / 4); c += 32 * PF_CONSUMERS) {
      const int row = c / (D / 4), col = (c % (D / 4)) * 4;
      const int rho = it.qt * M + row;
      if (rho >= it.g.n * p.rep) continue;
      float y[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const float4 x = *reinterpret_cast<const float4*>(join + q * 16 * D + at(row, col));
        y[0] += x.x;
        y[1] += x.y;
        y[2] += x.z;
        y[3] += x.w;
      }
      const float2 ml = rml[row];
      const int i = rho / p.rep;
      const long long to = (long long)(it.g.tok0 + i) * p.H + it.head * p.rep + (rho - i * p.rep);
      if (it.count == 1 && p.G == 0) {
        const float inv = ml.y > 0.f ? 1.f / ml.y : (ml.y == 0.f ? 0.f : ml.y);
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] *= inv;
        store4(static_cast<uint16_t*>(p.out) + to * D + col, y);
      } else if (it.count == 1) {
        store4(p.whole_o[it.g.prefix] + to * D + col, y);
        if (col == 0) p.whole_ml[it.g.prefix][to] = ml;
      } else {
        const long long pt = ((long long)blockIdx.x * 2 + it.slot) * M + row;
        store4(p.part_o + pt * D + col, y);
        if (col == 0) p.part_ml[pt] = ml;
      }
    }
  }
  if (late) pdl_wait();
}

// 32 bytes to a 32-byte aligned address in one store
__device__ __forceinline__ void store32(float* dst, const float* y) {
  asm volatile("st.global.v8.f32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};\n" ::"l"(dst), "f"(y[0]), "f"(y[1]), "f"(y[2]),
               "f"(y[3]), "f"(y[4]), "f"(y[5]), "f"(y[6]), "f"(y[7])
               : "memory");
}

// ---------------------------------------------------------------------------- many rows: tensor memory
// Prompts, draft trees and shared prefixes: tiles of 128 rows x 128 keys, both products on tcgen05.
// Warp 0 walks the line and streams K tiles (TMA), warp 2 V tiles, warp 1 issues the products, two groups
// of four warps each own a slot of tensor memory: scores S (128 columns; the weights P overwrite them as bf16) and output O
// (head_dim columns), one row per thread. While one slot's warps take the softmax of their scores,
// the tensor core works for the other slot. The slots are two row tiles that share every K and V tile
// (kTwo: an item has 256 rows), or alternate key tiles of one row tile, joined at the item's end
// (128 rows). A row's output is rescaled only when its running maximum grows by more than 2^8: P is
// then at most 2^8 instead of 1, and the final division by the sum takes the same factor out.
// Measured: 64 trees of 32 nodes over 4128 keys 186 us (HBM: 5.9 TB/s); a 2048-row chunk over 8192 keys,
// 32 heads, 247-255 us (960 TFLOP/s: softmax about 2500 cycles a tile and slot, then 1460 for the slot's
// products, tensor pipe and exponential unit 41% busy each).
constexpr int PM_THREADS = 384;  // K, products, V, one idle warp; 2 x 4 softmax warps
constexpr int PM_KT = 128;
constexpr int PM_OVER = 3;  // ragged prompts: 0 508, 1 474, 2 445, 3 429 us

constexpr int kRedo = 16;  // words: 512 items are told apart

template <int D, bool kTwo>
struct PmLayout {
  static constexpr int kTile = PM_KT * D * 2;  // a K or V tile
  static constexpr int kQ = (kTwo ? 2 : 1) * 128 * D * 2;
  static constexpr int kTail = 8 * kWalkShared + 384 + 4 * 64 + 2 * kRedo * 4 + (kTwo ? 0 : 4 * 128 * 8);
  static constexpr int kStages = (int(kSmemOptinBytes) - 1024 - kQ - kTail) / kTile > 12
                                     ? 12
                                     : (int(kSmemOptinBytes) - 1024 - kQ - kTail) / kTile;
  static constexpr size_t bytes() { return 1024 + size_t(kQ) + size_t(kStages) * kTile + kTail; }
};

__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;\n" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// Bits of the 32 keys from k0 on that a row sees.
__device__ __forceinline__ uint32_t low_bits(int n) { return n >= 32 ? 0xffffffffu : (n <= 0 ? 0u : (1u << n) - 1u); }
__device__ __forceinline__ uint32_t seen_bits(const PagedRow& r, int k0) {
  uint32_t w = low_bits(r.lim - k0);
  if (r.bits) {
    const int sh = k0 - r.base;
    const uint32_t x = sh >= 64 ? 0u : (sh >= 0 ? uint32_t(r.bits >> sh) : (sh > -32 ? uint32_t(r.bits << -sh) : 0u));
    w |= x & low_bits(r.klen - k0);
  }
  return w;
}

template <int D, bool kTwo>
__global__ void __launch_bounds__(PM_THREADS, 1)
    paged_many_kernel(const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv,
                      const __grid_constant__ PagedAttnParams p, int kinds, int least, bool late) {
  using L = PmLayout<D, kTwo>;
  constexpr int M = kTwo ? 256 : 128, KT = PM_KT, NST = L::kStages, HALVES = D / 64;
  constexpr uint32_t kColO = 256;
  extern __shared__ unsigned char pm_raw[];
  unsigned char* sm = pm_raw + ((1024u - (smem_addr(pm_raw) & 1023u)) & 1023u);
  unsigned char* qs = sm;                    // [slot][half][128 rows][128 B], swizzled
  unsigned char* ring = sm + L::kQ;          // [stage][half][128 keys][128 B]
  unsigned char* tail = ring + size_t(NST) * L::kTile;
  long long* sh = reinterpret_cast<long long*>(tail);
  uint64_t* bars = reinterpret_cast<uint64_t*>(tail + 8 * kWalkShared);
  uint64_t* kv_full = bars;                  // [12]
  uint64_t* kv_empty = bars + 12;            // [12]
  uint64_t* q_full = bars + 24;              // [2]: the slot's queries are in shared memory
  uint64_t* s_full = bars + 26;              // [2]: scores complete (and every product issued before)
  uint64_t* p_full = bars + 28;              // [2]: weights written, output rescaled
  uint64_t* o_full = bars + 30;              // [2]: the item's output complete
  uint64_t* o_empty = bars + 32;             // [2]: and read
  uint64_t* drain = bars + 34;
  uint64_t* x_full = bars + 35;              // the slots' states are in shared memory
  uint64_t* it_full = bars + 36;             // [4]: an item handed over
  uint64_t* it_empty = bars + 40;            // [4]: and read by all
  volatile int* dead = reinterpret_cast<volatile int*>(bars + 44);
  uint32_t* tslot = reinterpret_cast<uint32_t*>(bars + 45);
  PagedItem* queue = reinterpret_cast<PagedItem*>(tail + 8 * kWalkShared + 384);  // [4]
  uint32_t* redo = reinterpret_cast<uint32_t*>(queue + 4);  // [slot][kRedo]: items to be summed again, by number
  float2* xml = reinterpret_cast<float2*>(redo + 2 * kRedo);  // [item & 1][slot][row]
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    for (int s = 0; s < NST; ++s) {
      mbar_init(kv_full + s, 1);
      mbar_init(kv_empty + s, 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(q_full + s, 4);
      mbar_init(s_full + s, 1);
      mbar_init(p_full + s, 4);
      mbar_init(o_full + s, 1);
      mbar_init(o_empty + s, kTwo ? 4 : 8);
    }
    for (int s = 0; s < 4; ++s) {
      mbar_init(it_full + s, 1);
      mbar_init(it_empty + s, 10);  // V copies, products, 8 softmax warps
    }
    mbar_init(x_full, 8);
    mbar_init(drain, 1);
    mbar_fence_init();
    *dead = 0;
  }
  if (tid < 2 * kRedo) redo[tid] = 0;
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(smem_addr(tslot)),
                 "r"(512u)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
  }
  if (!late) pdl_wait();
  pdl_launch_dependents();
  paged_no_rec(p);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tslot;
  using Walk = PagedWalk<M, KT, PM_OVER>;
  Walk w;
  const bool work = w.begin_kept(p, kinds, least, sh);

  // The next item of the line, as the walking warp left it.
  auto take_item = [&](int n) {
    paged_wait(it_full + (n & 3), (n >> 2) & 1, dead, p.err);
    PagedItem it = queue[n & 3];
    if (*dead) it.count = 0;
    return it;
  };
  auto release_item = [&](int n) {
    __syncwarp();
    if (lane == 0) mbar_arrive(it_empty + (n & 3));
  };

  if ((warp == 0 || warp == 2) && work) {  // ---- K tiles (warp 0, which also walks) and V tiles (warp 2)
    const bool isv = warp == 2;
    const int psize = 1 << p.page_log2;
    const int box = min(psize, KT), parts = KT / box;
    // K: half rows apart, so that the tile's 128 keys have one stride as the product wants it; V: a
    // copy's rows together
    const int part = isv ? lane : lane / HALVES, half = isv ? 0 : lane % HALVES;
    const int at = isv ? part * box * (D * 2) : half * (KT * 128) + part * box * 128;
    int base = 0, last = -1;
    bool more = true;
    for (int n = 0; more; ++n) {
      PagedItem it;
      if (!isv) {
        if (n >= 4) paged_wait(it_empty + (n & 3), ((n >> 2) - 1) & 1, dead, p.err);
        it = PagedItem{w.g, w.head, w.qt, w.kt0, w.kt1, w.count, w.slot(), {}};
        if (lane == 0) {
          w.report(p);
          queue[n & 3] = it;
          mbar_arrive(it_full + (n & 3));
        }
      } else {
        it = take_item(n);
        release_item(n);
        if (it.count == 0) break;
      }
      const int nt = it.kt1 - it.kt0;
      PageWindow win;
      win.start(p, it.g, (it.kt0 * KT) >> p.page_log2, lane);
      for (int t = 0; t < nt; ++t) {
        // The tile's place in the ring, in the order that the products take the tiles: K0 V0 K1 V1 ...,
        // or with alternating slots K0 K1 V0 K2 V1 ... The two warps meet at a stage in turns; since the
        // products free the stages in order, the use before last is over when this warp's last one was.
        const int pos = base + (kTwo ? 2 * t + isv : isv ? t + min(t + 2, nt) : t < 2 ? t : 2 * t - 1);
        const int s = pos % NST;
        const int first = ((it.kt0 + t) * KT) >> p.page_log2;
        win.seek(p, first, lane);
        const int page = __shfl_sync(0xffffffffu, win.cur, (first - win.base + part) & 31);
        if (lane == 0) {
          if (pos >= NST) paged_wait(kv_empty + s, ((pos / NST) - 1) & 1, dead, p.err);
          if (!*dead) mbar_arrive_expect_tx(kv_full + s, L::kTile);
        }
        __syncwarp();
        if (*dead) break;
        if (part < parts)
          tma_load_5d(ring + size_t(s) * L::kTile + at, isv ? &tv : &tk, 0, ((it.kt0 + t) * KT) & (psize - 1), half,
                      it.head, page, kv_full + s);
        __syncwarp();
        last = pos;
      }
      base += 2 * nt;
      if (*dead) break;
      if (!isv && !(more = w.next(p, kinds))) {
        const int e = n + 1;
        if (e >= 4) paged_wait(it_empty + (e & 3), ((e >> 2) - 1) & 1, dead, p.err);
        if (lane == 0) {
          queue[e & 3].count = 0;
          mbar_arrive(it_full + (e & 3));
        }
      }
    }
    // shared memory must outlive the copies: the last one is waited for here, those before it by the
    // products that the block waits for, unless the block has given up
    if (lane == 0)
      for (int q = max(0, last - (*dead ? NST - 1 : 0)); q <= last; ++q)
        if (!mbar_wait(kv_full + q % NST, (q / NST) & 1)) raise_error(p.err, kErrTimeout);
  } else if (warp == 1 && work) {  // ---- products: the warp walks together, one lane issues
    constexpr uint32_t id_s = umma_idesc_bf16_m128(KT, 0), id_o = umma_idesc_bf16_m128(D, 1);
    const bool issuer = elect_one();
    const uint32_t q_lo = umma_lo(smem_addr(qs), 1), k_lo = umma_lo(smem_addr(ring), 1);
    const int vlog = min(p.page_log2, 7);  // keys of one copy of V
    const uint32_t v_lo = umma_lo(smem_addr(ring), (128u << vlog) >> 4);
    const uint32_t v_more = (((D - 64) * 2) << vlog) / 16;  // from a copy's last key to the next one's first
    int st = 0;               // ring stage of the next tile taken
    uint32_t ring_ph = 0;     // and its phase
    uint32_t p_ph = 0, o_ph = 0, q_ph = 0;  // phases by slot, as bits
    uint32_t used = 0;        // slots with an item before
    auto take = [&]() {
      const int s = st;
      paged_wait(kv_full + s, ring_ph, dead, p.err);
      if (++st == NST) {
        st = 0;
        ring_ph ^= 1;
      }
      return s;
    };
    auto queries = [&](int slot) {
      paged_wait(q_full + slot, (q_ph >> slot) & 1, dead, p.err);
      q_ph ^= 1u << slot;
    };
    auto scores = [&](int slot, int qslot, int s) {
      tc_fence_after();
      if (issuer) {
        const uint32_t a = q_lo + qslot * (128 * D * 2 / 16), b = k_lo + s * (L::kTile / 16), d = tmem + slot * 128;
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk)
          umma_ss(d, a + (kk / 4) * (128 * 128 / 16) + (kk % 4) * 2, b + (kk / 4) * (KT * 128 / 16) + (kk % 4) * 2, id_s,
                  kk != 0);
        umma_commit(s_full + slot);
      }
    };
    auto output = [&](int slot, int s, bool first) {
      paged_wait(p_full + slot, (p_ph >> slot) & 1, dead, p.err);
      p_ph ^= 1u << slot;
      if (first) {
        if ((used >> slot) & 1) {
          paged_wait(o_empty + slot, (o_ph >> slot) & 1, dead, p.err);
          o_ph ^= 1u << slot;
        }
        used |= 1u << slot;
      }
      tc_fence_after();
      if (issuer) {
        const uint32_t b = v_lo + s * (L::kTile / 16), d = tmem + kColO + slot * D, a = tmem + slot * 128;
#pragma unroll
        for (int kk = 0; kk < KT / 16; ++kk)
          umma_ts(d, a + kk * 8, b + kk * (16 * 128 / 16) + uint32_t((kk * 16) >> vlog) * v_more, id_o, !first || kk != 0);
      }
    };
    auto done = [&](uint64_t* bar) {
      if (issuer) umma_commit(bar);
    };
    for (int n = 0;; ++n) {
      const PagedItem it = take_item(n);
      release_item(n);
      if (it.count == 0) break;
      const int nt = it.kt1 - it.kt0;
      if constexpr (kTwo) {
        const bool two = it.g.n * p.rep - it.qt * M > 128;
        int ks = take();
        queries(0);
        scores(0, 0, ks);
        if (two) {
          queries(1);
          scores(1, 1, ks);
        }
        done(kv_empty + ks);
        for (int t = 0; t < nt && !*dead; ++t) {
          const int vs = take();
          const bool more = t + 1 < nt;
          output(0, vs, t == 0);
          if (!two) done(kv_empty + vs);
          if (more) {
            ks = take();
            scores(0, 0, ks);
          } else {
            done(o_full);
          }
          if (two) {
            output(1, vs, t == 0);
            done(kv_empty + vs);
            if (more) scores(1, 1, ks);
            else done(o_full + 1);
          }
          if (more) done(kv_empty + ks);
        }
      } else {
        int ks = take();
        queries(0);
        scores(0, 0, ks);
        done(kv_empty + ks);
        if (nt > 1) {
          ks = take();
          scores(1, 0, ks);
          done(kv_empty + ks);
        }
        for (int t = 0; t < nt && !*dead; ++t) {
          const int vs = take(), slot = t & 1;
          output(slot, vs, t < 2);
          done(kv_empty + vs);
          if (t + 2 < nt) {
            ks = take();
            scores(slot, 0, ks);
            done(kv_empty + ks);
          } else {
            done(o_full + slot);
          }
        }
      }
    }
    done(drain);  // tensor memory is given back only when nothing writes it any more
    if (!mbar_wait(drain, 0)) raise_error(p.err, kErrTimeout);
    __syncwarp();
  } else if (warp >= 4 && work) {  // ---- softmax: thread = row of its slot
    const int slot = (warp - 4) >> 2, qd = warp & 3, r128 = qd * 32 + lane;
    const uint32_t lanes = tmem + (uint32_t(qd * 32) << 16);
    const uint32_t ts = lanes + slot * 128, to = lanes + kColO + slot * D;
    const float sl2 = p.scale_log2;
    const bool wide_out = (reinterpret_cast<unsigned long long>(p.out) & 31) == 0;
    int ns = 0, no[2] = {0, 0};  // scores and outputs waited for
    int vcnt = 0;                // ring position of the item's first K tile
    int nitem = 0;

    // Query rows of an item into the slot's swizzled tile, asynchronously: 16 or 8 lanes copy a row, whose
    // place the lane that owns it knows.
    auto copy_q = [&](const PagedItem& x) {
      constexpr int CH = D / 8, RPI = 32 / CH;  // 16-byte pieces of a row, rows per step
      const PagedRow r = paged_row(p, x.g, x.head, x.qt * M + (kTwo ? slot * 128 : 0) + r128);
      const long long mine = r.valid ? r.tok * p.q_row + r.h * p.q_head : -1;
      const int c = lane % CH;
      unsigned char* dst = qs + (kTwo ? slot : 0) * (128 * D * 2) + (c / 8) * (128 * 128) + qd * 32 * 128;
#pragma unroll 4
      for (int k = 0; k < 32; k += RPI) {
        const int row = k + lane / CH;
        const long long from = __shfl_sync(0xffffffffu, mine, row);
        cp_async16(dst + row * 128 + (((c & 7) ^ (row & 7)) << 4),
                   static_cast<const uint16_t*>(p.q) + (from < 0 ? 0 : from) + c * 8, from < 0 ? 0 : 16);
      }
      cp_async_commit();
    };
    auto copied_q = [&]() {
      cp_async_wait<0>();
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(q_full + (kTwo ? slot : 0));
    };
    // whether an item's rows reach the second slot's tile; only then are its queries copied and waited for
    auto both = [&](const PagedItem& x) { return x.g.n * p.rep - x.qt * M > 128; };
    PagedItem w = take_item(0);
    if (w.count && (slot == 0 || (kTwo && both(w)))) {
      copy_q(w);
      copied_q();
    }
    for (; w.count; ++nitem) {
      const int nt = w.kt1 - w.kt0;
      const bool two = kTwo ? both(w) : nt > 1;  // the second slot has work
      const bool active = slot == 0 || two;
      const PagedRow r = paged_row(p, w.g, w.head, w.qt * M + (kTwo ? slot * 128 : 0) + r128);
      const int lim = r.valid ? r.lim : 0x7fffffff;  // rows that pad the tile see everything, for nobody
      // keys that every row of the slot's tile sees
      const int edge = min(w.g.klen, w.g.prefix ? w.g.klen
                                                : w.g.klen - w.g.n + (p.tree ? 0 : (w.qt * M + (kTwo ? slot * 128 : 0)) / p.rep + 1));
      float m = -INFINITY, l = 0.f;
      const int step = kTwo ? 1 : 2;
      const bool rows = __any_sync(0xffffffffu, r.valid);
      for (int t = kTwo ? 0 : slot; t < nt && active; t += step) {
        paged_wait(s_full + slot, ns & 1, dead, p.err);
        ++ns;
        tc_fence_after();
        const int key0 = (w.kt0 + t) * KT;
        const bool masked = key0 + KT > lim;
        // Values in masked places may be anything, and 0 x NaN would reach every row. Behind the last
        // key they are cleared; between keys (a later row, another branch) they mark the slot's rows,
        // which are summed again over the seen keys alone when the line is done.
        if (key0 + KT > edge) {
          const int vpos = vcnt + (kTwo ? 2 * t + 1 : min(2 * t + 2, nt + t));
          const int vs = vpos % NST;
          paged_wait(kv_full + vs, (vpos / NST) & 1, dead, p.err);
          const int vbox = min(1 << p.page_log2, KT), hstride = vbox * 128;
          unsigned char* vrow = ring + size_t(vs) * L::kTile + r128 * 128 + (r128 / vbox) * (vbox * (D - 64) * 2);
          if (key0 + r128 >= w.g.klen) {
            if (slot == 0 || !kTwo) {  // slot 1 of a shared tile multiplies after slot 0
#pragma unroll
              for (int h = 0; h < HALVES; ++h)
#pragma unroll
                for (int c = 0; c < 8; ++c)
                  *reinterpret_cast<uint4*>(vrow + h * hstride + c * 16) = make_uint4(0, 0, 0, 0);
            }
          } else {
            uint32_t worst = 0;
#pragma unroll
            for (int h = 0; h < HALVES; ++h)
#pragma unroll
              for (int c = 0; c < 8; ++c) {
                const uint4 x = *reinterpret_cast<const uint4*>(vrow + h * hstride + c * 16);
                const uint32_t xs[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  worst = max(worst, xs[e] & 0x7f800000u);
                  worst = max(worst, (xs[e] << 16) & 0x7f800000u);
                }
              }
            if (worst == 0x7f800000u) atomicOr(redo + slot * kRedo + (nitem >> 5) % kRedo, 1u << (nitem & 31));
          }
          fence_proxy_async_smem();
        }
        if (rows) {  // a warp whose rows only pad the tile passes on
          // The scores are read from tensor memory twice, 32 columns at a time: for the maximum and for
          // the weights. The loops stay rolled: the tile's code is small enough to stay in the instruction
          // caches beside the other warps', which is worth more than the loads it would save (unrolled,
          // or with the next load under way: 6 to 20% more time).
          if (__any_sync(0xffffffffu, masked)) {  // tensor memory is read and written by whole warps
#pragma unroll 1
            for (int c = 0; c < KT; c += 32) {
              uint32_t v[32];
              tmem_ld32(ts + c, v);
              const uint32_t see = masked ? seen_bits(r, key0 + c) : 0xffffffffu;
#pragma unroll
              for (int j = 0; j < 32; ++j)
                if (!((see >> j) & 1u)) v[j] = 0xff800000u;
              tmem_st32(ts + c, v);
            }
            tmem_st_wait();
          }
          float mt = -INFINITY;
#pragma unroll 1
          for (int c = 0; c < KT; c += 32) {
            uint32_t v[32];
            tmem_ld32(ts + c, v);
            float x[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = fmaxf(__uint_as_float(v[e]), __uint_as_float(v[e + 4]));
#pragma unroll
            for (int j = 8; j < 32; j += 8)
#pragma unroll
              for (int e = 0; e < 4; ++e) x[e] = max3(x[e], __uint_as_float(v[j + e]), __uint_as_float(v[j + e + 4]));
            mt = max3(mt, fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
          }
          mt *= sl2;
          if (t < step) {
            m = mt;
          } else if (__any_sync(0xffffffffu, mt > m + 8.f)) {
            const float mn = mt > m + 8.f ? mt : m;
            const float f = m == mn ? 1.f : ex2_approx(m - mn);
            m = mn;
            l *= f;
#pragma unroll 1
            for (int c = 0; c < D; c += 32) {
              uint32_t v[32];
              tmem_ld32(to + c, v);
#pragma unroll
              for (int j = 0; j < 32; ++j) v[j] = __float_as_uint(__uint_as_float(v[j]) * f);
              tmem_st32(to + c, v);
            }
          }
          const float mg = m == -INFINITY ? 0.f : m;
          float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
          for (int c = 0; c < KT; c += 32) {
            uint32_t v[32], pk[16];
            tmem_ld32(ts + c, v);
#pragma unroll
            for (int j = 0; j < 16; ++j) {
              const float x = ex2_approx(fmaf(__uint_as_float(v[2 * j]), sl2, -mg));
              const float y = ex2_approx(fmaf(__uint_as_float(v[2 * j + 1]), sl2, -mg));
              sum[(j & 1) * 2] += x;
              sum[(j & 1) * 2 + 1] += y;
              pk[j] = pack_bf16(x, y);  // rounded to bf16, as the values are: at most 2^-8 of each, whatever m
            }
            tmem_st16u(ts + c / 2, pk);  // over scores that both passes have read
          }
          l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
        }
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(p_full + slot);
      }
      vcnt += 2 * nt;
      // The item's queries have been used for the last time where the last scores were waited for (with
      // alternating slots, by the slot of the last tile): the next item's take their place while the
      // last product runs.
      const PagedItem nx = take_item(nitem + 1);
      const bool load = nx.count && (kTwo ? slot == 0 || both(nx) : ((nt - 1) & 1) == slot);
      if (load) copy_q(nx);
      // ---- the item's result
      float f0 = 1.f, f1 = 0.f;
      if constexpr (!kTwo) {  // the slots' states joined; each group of warps takes half of the columns
        float2* x = xml + (nitem & 1) * 256;  // by turns: the item before last has been read by all
        x[slot * 128 + r128] = make_float2(m, l);
        __syncwarp();
        if (lane == 0) mbar_arrive(x_full);
        paged_wait(x_full, nitem & 1, dead, p.err);
        const float2 a = x[r128], b = x[128 + r128];
        m = fmaxf(a.x, b.x);
        const float mg = m == -INFINITY ? 0.f : m;
        f0 = ex2_approx(a.x - mg);
        f1 = ex2_approx(b.x - mg);
        l = a.y * f0 + b.y * f1;
        paged_wait(o_full, no[0] & 1, dead, p.err);
        ++no[0];
        if (two) {
          paged_wait(o_full + 1, no[1] & 1, dead, p.err);
          ++no[1];
        }
      } else if (active) {
        paged_wait(o_full + slot, no[0] & 1, dead, p.err);
        ++no[0];
      }
      if (load) copied_q();
      if (active || !kTwo) {
        tc_fence_after();
        const bool direct = w.count == 1 && p.G == 0;
        const float inv = direct ? (l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l)) : 1.f;
        const long long at = (long long)r.tok * p.H + r.h;
        const long long pt = ((long long)blockIdx.x * 2 + w.slot) * M + (kTwo ? slot * 128 : 0) + r128;
        float* po = w.count == 1 ? p.whole_o[w.g.prefix] + at * D : p.part_o + pt * D;
        const int c0 = kTwo ? 0 : slot * (D / 2), c1 = kTwo ? D : c0 + D / 2;
#pragma unroll 1
        for (int c = c0; c < c1; c += 32) {
          uint32_t v[32];
          tmem_ld32(lanes + kColO + (kTwo ? slot * D : 0) + c, v);
          float y[32];
          if constexpr (kTwo) {
#pragma unroll
            for (int j = 0; j < 32; ++j) y[j] = __uint_as_float(v[j]) * inv;
          } else {
            const float g0 = f0 * inv, g1 = f1 * inv;
#pragma unroll
            for (int j = 0; j < 32; ++j) y[j] = __uint_as_float(v[j]) * g0;
            if (two) {
              tmem_ld32(lanes + kColO + D + c, v);
#pragma unroll
              for (int j = 0; j < 32; ++j) y[j] = fmaf(__uint_as_float(v[j]), g1, y[j]);
            }
          }
          if (r.valid) {
            if (direct) {
              uint16_t* dst = static_cast<uint16_t*>(p.out) + at * D + c;
              float v8[16];
#pragma unroll
              for (int j = 0; j < 16; ++j) v8[j] = __uint_as_float(pack_bf16(y[2 * j], y[2 * j + 1]));
              if (wide_out) {
                store32(reinterpret_cast<float*>(dst), v8);
                store32(reinterpret_cast<float*>(dst) + 8, v8 + 8);
              } else {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                  reinterpret_cast<float4*>(dst)[j] = make_float4(v8[4 * j], v8[4 * j + 1], v8[4 * j + 2], v8[4 * j + 3]);
              }
            } else {  // scratch: 256-byte aligned rows
#pragma unroll
              for (int j = 0; j < 4; ++j) store32(po + c + 8 * j, y + 8 * j);
            }
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          if (kTwo) {
            mbar_arrive(o_empty + slot);
          } else {
            mbar_arrive(o_empty);
            if (two) mbar_arrive(o_empty + 1);
          }
        }
        if (r.valid && !direct && (kTwo || slot == 0)) {
          if (w.count == 1) p.whole_ml[w.g.prefix][at] = make_float2(m, l);
          else p.part_ml[pt] = make_float2(m, l);
        }
      }
      release_item(nitem);
      w = nx;
    }
    // Rows beside values that are not finite, once more from the line's beginning (nobody waits for these
    // warps now, however long it takes); with alternating slots each takes every other row.
    named_sync(1, 256);
    uint32_t any = 0;
    for (int i = 0; i < kRedo; ++i) any |= kTwo ? redo[slot * kRedo + i] : redo[i] | redo[kRedo + i];
    if (any) {
      Walk again = *reinterpret_cast<const Walk*>(sh);
      int n = 0;
      do {
        const int word = (n >> 5) % kRedo;
        if (!(((kTwo ? redo[slot * kRedo + word] : redo[word] | redo[kRedo + word]) >> (n & 31)) & 1u)) continue;
        const bool direct = again.count == 1 && p.G == 0;
#pragma unroll 1
        for (int i = kTwo ? 0 : slot; i < 32; i += kTwo ? 1 : 2) {
          const int row = (kTwo ? slot * 128 : 0) + qd * 32 + i;
          const PagedRow r = paged_row(p, again.g, again.head, again.qt * M + row);
          if (!r.valid) break;
          float m, l, o[D / 32];
          paged_redo_row<D>(p, again.g, r, again.head, again.kt0 * KT, again.kt1 * KT, lane, m, l, o);
          const long long to = (long long)r.tok * p.H + r.h;
          const long long pt = ((long long)blockIdx.x * 2 + again.slot()) * M + row;
          const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
#pragma unroll
          for (int e = 0; e < D / 32; ++e) {
            const int c = lane * (D / 32) + e;
            if (direct) static_cast<uint16_t*>(p.out)[to * D + c] = f32_to_bf16_bits(o[e] * inv);
            else (again.count == 1 ? p.whole_o[again.g.prefix] + to * D : p.part_o + pt * D)[c] = o[e];
          }
          if (!direct && lane == 0)
            (again.count == 1 ? p.whole_ml[again.g.prefix] + to : p.part_ml + pt)[0] = make_float2(m, l);
        }
      } while (++n, again.next(p, kinds));
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(512u) : "memory");
  }
  if (late) pdl_wait();
}

// ---------------------------------------------------------------------------- joining
// States (m, l, o) of one row over different keys: with M = max m_i, o = sum 2^(m_i - M) o_i /
// sum 2^(m_i - M) l_i, taken in the order of the keys. Both kernels read a few states that are still
// in L2; they are bound by the latency of the loads that depend on one another, so each thread first
// finds where its states are, then has all of their loads in flight.
template <typename S>
__device__ __forceinline__ void paged_store_out(void* out, long long at, const float (&o)[4], float L) {
  const float inv = L > 0.f ? 1.f / L : (L == 0.f ? 0.f : L);
  const float y[4] = {o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv};
  store4(static_cast<S*>(out) + at, y);
}

// Without prefixes: block (x, y) joins rows [8 y, 8 y + 8) of the divided item that began in block x
// of the attention; D / 4 threads a row.
constexpr int PJ_ROWS = 8;
template <typename S, int D>
__global__ void __launch_bounds__(PJ_ROWS* D / 4)
    paged_join_kernel(const __grid_constant__ PagedAttnParams p, int M) {
  pdl_launch_dependents();
  pdl_wait();
  const PagedRec rec = p.rec[blockIdx.x];
  const int row = blockIdx.y * PJ_ROWS + int(threadIdx.x) / (D / 4), col = (threadIdx.x % (D / 4)) * 4;
  const int rho = rec.qt * M + row;
  if (rec.count < 2 || rho >= rec.rows) return;
  const long long at = ((long long)blockIdx.x * 2 + 1) * M + row;  // later parts: the next blocks' first slots
  const float2* pm = p.part_ml + at;
  const float* po = p.part_o + at * D + col;
  float top = pm[0].x;
#pragma unroll 8
  for (int i = 1; i < rec.count; ++i) top = fmaxf(top, pm[(long long)i * 2 * M - M].x);
  const float mg = top == -INFINITY ? 0.f : top;
  float L = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int i = 0; i < rec.count; ++i) {
    const long long r = i ? (long long)i * 2 * M - M : 0;
    const float2 ml = pm[r];
    const float4 x = *reinterpret_cast<const float4*>(po + r * D);
    const float f = exp2f(ml.x - mg);
    L += ml.y * f;
    o[0] += x.x * f;
    o[1] += x.y * f;
    o[2] += x.z * f;
    o[3] += x.w * f;
  }
  const int i = rho / p.rep;
  paged_store_out<S>(p.out, ((long long)(rec.tok0 + i) * p.H + rec.head * p.rep + (rho - i * p.rep)) * D + col, o, L);
}

// With prefixes: a row and query head per D / 4 threads; its prefix item's states, then its own.
struct PagedCombineParams {
  PagedAttnParams a;
  const float* part_o[2];  // own, prefix
  const float2* part_ml[2];
  int M[2];
  int blocks[2];           // blocks of the launch that wrote them
};

constexpr int PC_JOIN = 256;
template <typename S, int D>
__global__ void __launch_bounds__(PC_JOIN) paged_combine_kernel(const __grid_constant__ PagedCombineParams c) {
  const PagedAttnParams& p = c.a;
  pdl_launch_dependents();
  pdl_wait();
  const int t = blockIdx.x, col = (threadIdx.x % (D / 4)) * 4;
  const int b = request_of_row(p.offsets, t, p.T, p.B);
  if (b >= p.B) return;
  int grp = 0;
  for (int g0 = 0; g0 < p.G; g0 += PC_JOIN) {
    const int g = g0 + int(threadIdx.x);
    grp += __syncthreads_count(g < p.G && p.groups[g + 1] <= b);
  }
  if (grp >= p.G || p.groups[grp] > b) grp = -1;
  const int h = blockIdx.y * (PC_JOIN / (D / 4)) + int(threadIdx.x) / (D / 4);
  if (h >= p.H) return;
  const float2* pm[2];
  const float* po[2];
  long long step[2], less[2];
  int count[2] = {0, 0};
#pragma unroll
  for (int kind = 0; kind < 2; ++kind) {
    if (kind && grp < 0) continue;
    const int tok0 = paged_row0(p, kind ? min(max(p.groups[grp], 0), p.B) : b);
    const int rho = (t - tok0) * p.rep + h % p.rep, m = c.M[kind], qt = rho / m;
    if (rho < 0) continue;  // offsets that do not increase
    const int2 d = p.desc[kind][(tok0 * p.rep / m + (kind ? grp : b) + qt) * p.Hk + h / p.rep];
    if (d.x < 0 || d.y < 1 || d.y > c.blocks[kind] || d.x > c.blocks[kind] - d.y) continue;  // never written
    count[kind] = d.y;
    const bool one = d.y == 1;
    const long long at = one ? (long long)t * p.H + h : ((long long)d.x * 2 + 1) * m + (rho - qt * m);
    pm[kind] = (one ? p.whole_ml[kind] : c.part_ml[kind]) + at;
    po[kind] = (one ? p.whole_o[kind] : c.part_o[kind]) + at * D + col;
    step[kind] = 2 * m;
    less[kind] = m;
  }
  float top = -INFINITY;
#pragma unroll
  for (int kind = 1; kind >= 0; --kind)
#pragma unroll 4
    for (int i = 0; i < count[kind]; ++i) top = fmaxf(top, pm[kind][i ? i * step[kind] - less[kind] : 0].x);
  const float mg = top == -INFINITY ? 0.f : top;
  float L = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int kind = 1; kind >= 0; --kind)
#pragma unroll 4
    for (int i = 0; i < count[kind]; ++i) {
      const long long r = i ? i * step[kind] - less[kind] : 0;
      const float2 ml = pm[kind][r];
      const float4 x = *reinterpret_cast<const float4*>(po[kind] + r * D);
      const float f = exp2f(ml.x - mg);
      L += ml.y * f;
      o[0] += x.x * f;
      o[1] += x.y * f;
      o[2] += x.z * f;
      o[3] += x.w * f;
    }
  paged_store_out<S>(p.out, ((long long)t * p.H + h) * D + col, o, L);
}

}  // namespace wc
