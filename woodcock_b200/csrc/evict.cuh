// Keys that a long session keeps: the attention weight that each key gathers, and the eviction of those
// that gather least.
#pragma once

#include <type_traits>

#include "common.cuh"
#include "paged_walk.cuh"
#include "tcgen05.cuh"

namespace wc {

// The gathered weight of each key, fp32 [pages][kv_heads][page_size] beside the pages, rows contiguous.
struct MassPool {
  float* ptr;
  long long layer, page, head;
};

// ---------------------------------------------------------------------------- the weight a key gathers
// mass_j (+)= sum over new rows i and query heads h of the key's head of p_ih(j),
// p_ih(j) = 2^(s_ih(j) - M_ih) / L_ih over the keys that row i sees. A weight needs its row's maximum and sum
// over all keys first, so the scores are needed twice.
struct MassRec {
  int request, head, kt, count;  // count 0: none
};

// What one block of the few rows' first kernel had of an item, for the second; tiles 0: the list's end.
struct MassPiece {
  int request, head, key0, tiles;
  int klen, old, rows;  // keys, those before the new ones, rows of the head
  int at;               // of the item's first row, whole_ml's
  int first, count;     // the blocks that share the item
  int pad[2];
};

struct MassParams {
  PagedAttnParams a;     // q, K pages, batch
  MassPool mass;
  int add;               // 0: the sums of all keys start anew
  // workspace
  float2* row_ml;        // [T][H]: maximum (log2 units) and 1 / sum
  float2* part_ml;       // [blocks][2][16]: of divided items
  long long* tiles;      // [B + 1]: key tiles before each request (all of its heads')
  int blocks;            // of the statistics' launch
  int kinds;             // which requests' rows
  float* scores;         // few rows: [blocks][per tiles][width rows][64 keys], log2 units
  int per, width;        // key tiles of a block at most, rows of a tile at most
  MassPiece* pieces;     // [blocks][most]
  int most;
  unsigned char* rows_q; // many rows: [Hk][ids] tiles of 128 query rows as shared memory has them
  float* rows_l;         // [Hk][ids][128]: -(M + log2(sum)) of their rows; -inf: a row that weighs nothing
  int ids;
  float* part_sum;       // many rows: [blocks][2][256], of divided key tiles
  MassRec* keys_rec;     // [blocks]: the divided key tile that begins in the block
  int key_blocks;
};

// What a weight is before the sums are joined: rows that see nothing keep 0.
__device__ __forceinline__ float2 mass_row(float m, float l) {
  return make_float2(m == -INFINITY ? 0.f : m, l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l));
}

// The same as one number: 2^(s - M) / sum = 2^(s + it). Its rounding, 2^-24 of M + log2(sum), is the weights' own;
// with M and 1 / sum apart an exponential would take an instruction more, and they are what bounds the many rows.
__device__ __forceinline__ float mass_minus_l(float m, float l) {
  const float2 y = mass_row(m, l);
  return log2f(y.y) - y.x;
}

// Pages of a request whose sums the call writes.
__device__ __forceinline__ int mass_pages(const MassParams& mp, const PagedSeg& g) {
  return g.n > 0 || !mp.add ? (g.klen + (1 << mp.a.page_log2) - 1) >> mp.a.page_log2 : 0;
}

// Requests that share no pages have no more of them than the pool: raises the error bit where the call's have, whose
// sums several blocks write. For kThreads threads of one block, t their numbers, while they would wait for their
// first tiles anyway (in a kernel's last block, or before its search, it costs 1 us); `pages` is 0 before.
template <int kThreads>
__device__ __forceinline__ void mass_check_pool(const MassParams& mp, int t, unsigned long long* pages) {
  const PagedAttnParams& p = mp.a;
  unsigned long long mine = 0;
  for (int b = t; b < p.B; b += kThreads) mine += mass_pages(mp, paged_seg(p, kOwnRows, b));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
  if (t % 32 == 0 && mine) atomicAdd(pages, mine);
  named_sync(1, kThreads);
  if (t == 0 && *pages > (unsigned long long)p.pages) raise_error(p.err, kErrPage);
}

// A call that starts the sums anew does so for requests without rows too. Each block takes its share of their heads.
__device__ __forceinline__ void mass_clear(const MassParams& mp, int block, int blocks) {
  const PagedAttnParams& p = mp.a;
  for (long long at = block; at < (long long)p.B * p.Hk; at += blocks) {
    const int b = int(at / p.Hk), head = int(at - (long long)b * p.Hk);
    const PagedSeg g = paged_seg(p, kOwnRows, b);
    if (g.n > 0) continue;
    for (int key = threadIdx.x; key < g.klen; key += blockDim.x) {
      const int page = paged_page(p, g, key >> p.page_log2);
      if (page >= 0) mp.mass.ptr[page * mp.mass.page + head * mp.mass.head + (key & ((1 << p.page_log2) - 1))] = 0.f;
    }
  }
}

// A call in which no request has a row.
__global__ void __launch_bounds__(256) mass_clear_kernel(const __grid_constant__ MassParams mp) {
  pdl_wait();
  pdl_launch_dependents();
  mass_clear(mp, blockIdx.x, gridDim.x);
}

// The first kernel's scores, one row tile against one key tile: 16 rows x 64 keys, a key and four rows a
// thread. qs [16][D], ks [64][D + 4].
template <int D>
__device__ __forceinline__ void mass_scores(const float* qs, const float* ks, int sk, int sr, float (&s)[4]) {
#pragma unroll 8
  for (int d = 0; d < D; d += 4) {
    const float4 k4 = *reinterpret_cast<const float4*>(ks + sk * (D + 4) + d);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float4 q4 = *reinterpret_cast<const float4*>(qs + (sr + i) * D + d);
      s[i] = fmaf(q4.x, k4.x, fmaf(q4.y, k4.y, fmaf(q4.z, k4.z, fmaf(q4.w, k4.w, s[i]))));
    }
  }
}

constexpr int MS_THREADS = 256, MS_M = 16, MS_KT = 64;

template <int D>
__device__ __forceinline__ void mass_load_q(const PagedAttnParams& p, const PagedSeg& g, int head, int rho0, float* qs) {
  for (int c = threadIdx.x; c < MS_M * (D / 8); c += MS_THREADS) {
    const int m = c / (D / 8), col = (c % (D / 8)) * 8;
    const PagedRow r = paged_row(p, g, head, rho0 + m);
    float x[8] = {};
    if (r.valid) load8(static_cast<const float*>(p.q) + r.tok * p.q_row + r.h * p.q_head + col, x);
    store8(qs + m * D + col, x);
  }
}
template <int D>
__device__ __forceinline__ void mass_load_k(const PagedAttnParams& p, const PagedSeg& g, int head, int kt, float* ks) {
  for (int c = threadIdx.x; c < MS_KT * (D / 8); c += MS_THREADS) {
    const int kr = c / (D / 8), cc = (c % (D / 8)) * 8, key = kt * MS_KT + kr;
    float x[8] = {};
    const int page = key < g.klen ? paged_page(p, g, key >> p.page_log2) : -1;
    if (page >= 0)
      load8(static_cast<const float*>(p.K.ptr) + page * p.K.page + head * p.K.head +
                (key & ((1 << p.page_log2) - 1)) * p.K.row + cc, x);
    store8(ks + kr * (D + 4) + cc, x);
  }
}

template <int D>
constexpr size_t mass_simt_smem() {
  return sizeof(float) * (size_t(MS_KT) * (D + 4) + MS_M * D + MS_M * (MS_KT + 4)) + 8 * kWalkShared;
}

// Every row's maximum and sum, for fp32 pages on the CUDA cores. Items as in paged attention; a divided one leaves its parts.
template <int D>
__global__ void __launch_bounds__(MS_THREADS) mass_rows_kernel(const __grid_constant__ MassParams mp) {
  const PagedAttnParams& p = mp.a;
  constexpr int M = MS_M, KT = MS_KT, LS = KT + 4;
  extern __shared__ __align__(16) float ms_smem[];
  float* ks = ms_smem;
  float* qs = ks + KT * (D + 4);
  float* ss = qs + M * D;
  long long* sh = reinterpret_cast<long long*>(ss + M * LS);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  pdl_wait();
  pdl_launch_dependents();
  PagedWalk<M, KT, 1> w;
  paged_no_rec(p);
  if (!w.begin(p, mp.kinds, 1, sh)) return;
  do {
    __syncthreads();
    mass_load_q<D>(p, w.g, w.head, w.qt * M, qs);
    const int sk = tid & 63, sr = (tid >> 6) * 4;
    PagedRow rows[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) rows[i] = paged_row(p, w.g, w.head, w.qt * M + 2 * warp + i);
    float m2[2] = {-INFINITY, -INFINITY}, l2[2] = {0.f, 0.f};
    for (int kt = w.kt0; kt < w.kt1; ++kt) {
      __syncthreads();
      mass_load_k<D>(p, w.g, w.head, kt, ks);
      __syncthreads();
      float s[4] = {};
      mass_scores<D>(qs, ks, sk, sr, s);
#pragma unroll
      for (int i = 0; i < 4; ++i) ss[(sr + i) * LS + sk] = s[i];
      __syncthreads();
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
        l2[i] = l2[i] * exp2f(m2[i] - mg) + warp_sum(exp2f(z[0] - mg) + exp2f(z[1] - mg));
        m2[i] = mx;
      }
    }
    if (tid == 0) w.report(p);
    if (lane == 0) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (!rows[i].valid) continue;
        if (w.count == 1) mp.row_ml[(long long)rows[i].tok * p.H + rows[i].h] = mass_row(m2[i], l2[i]);
        else mp.part_ml[((long long)blockIdx.x * 2 + w.slot()) * M + 2 * warp + i] = make_float2(m2[i], l2[i]);
      }
    }
  } while (w.next(p, mp.kinds));
}

// A row tile's number among those of its head: distinct, below T rep / 128 + requests + 1.
__device__ __forceinline__ int mass_tile(const PagedAttnParams& p, int tok0, int request, int qt) {
  return tok0 * p.rep / 128 + request + qt;  // rows x heads is below 2^30
}

// Key tiles of requests that share no pages, at most.
inline long long mass_most_tiles(int pages, int page_log2, int B, int Hk, int KT) {
  return (((long long)pages << page_log2) / KT + B) * Hk;
}

// Joins the parts of divided items, one block an item; where `tiles` is asked for, a last block counts the key
// tiles before each request, and the pages of all.
template <int M, int KT>
__global__ void __launch_bounds__(256) mass_join_kernel(const __grid_constant__ MassParams mp) {
  constexpr int LANES = 256 / M;  // lanes a row
  const PagedAttnParams& p = mp.a;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  pdl_wait();
  pdl_launch_dependents();
  if (int(blockIdx.x) == mp.blocks) {
    __shared__ long long sums[8];
    long long base = 0, pages = 0;
    for (int b0 = 0; b0 < p.B; b0 += 256) {
      const int b = b0 + tid;
      long long w = 0;
      if (b < p.B) {
        const PagedSeg g = paged_seg(p, mp.kinds, b);
        if (g.n > 0) w = (long long)((g.klen + KT - 1) / KT) * p.Hk;
        pages += mass_pages(mp, g);
      }
      long long x = w;
#pragma unroll
      for (int o = 1; o < 32; o *= 2) {
        const long long y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
      }
      if (lane == 31) sums[warp] = x;
      __syncthreads();
      long long before = base;
      for (int i = 0; i < 8; ++i) {
        if (i < warp) before += sums[i];
        base += sums[i];
      }
      if (b < p.B) mp.tiles[b] = before + x - w;
      __syncthreads();
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) pages += __shfl_xor_sync(0xffffffffu, pages, o);
    if (lane == 0) sums[warp] = pages;
    __syncthreads();
    if (tid == 0) {
      for (int i = 1; i < 8; ++i) pages += sums[i];
      const bool shared = pages > p.pages;  // requests share pages, whose sums two blocks would write
      if (shared) raise_error(p.err, kErrPage);
      mp.tiles[p.B] = shared ? 0 : base;
    }
    return;
  }
  const PagedRec rec = p.rec[blockIdx.x];
  if (rec.count == 0) return;
  const int r = tid / LANES, rho = rec.qt * M + r;
  float m = -INFINITY, l = 0.f;
  if (rho < rec.rows)
    for (int i = tid % LANES; i < rec.count; i += LANES) {
      const float2 y = mp.part_ml[((long long)(blockIdx.x + i) * 2 + (i == 0 ? 1 : 0)) * M + r];
      const float mn = fmaxf(m, y.x), mg = mn == -INFINITY ? 0.f : mn;
      l = l * exp2f(m - mg) + y.y * exp2f(y.x - mg);
      m = mn;
    }
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) {
    const float m2 = __shfl_xor_sync(0xffffffffu, m, o), l2 = __shfl_xor_sync(0xffffffffu, l, o);
    const float mn = fmaxf(m, m2), mg = mn == -INFINITY ? 0.f : mn;
    l = l * exp2f(m - mg) + l2 * exp2f(m2 - mg);
    m = mn;
  }
  if constexpr (M > MS_M) {
    if (tid % LANES == 0 && rho / 128 * 128 < rec.rows)
      mp.rows_l[(size_t)(rec.head * mp.ids + mass_tile(p, rec.tok0, rec.idx, rho / 128)) * 128 + rho % 128] =
          rho < rec.rows ? mass_minus_l(m, l) : -INFINITY;
  } else if (rho < rec.rows && tid % LANES == 0) {
    const int i = rho / p.rep;
    mp.row_ml[(long long)(rec.tok0 + i) * p.H + rec.head * p.rep + rho - i * p.rep] = mass_row(m, l);
  }
}

// The request whose tiles hold tile `at` (warp-collective; tiles[] ascends, tiles[B] is above `at`).
__device__ __forceinline__ int mass_request(const long long* tiles, int B, long long at, int lane) {
  int lo = 0, hi = B;  // tiles[lo] <= at < tiles[hi]
  while (hi - lo > 1) {
    const int step = (hi - lo + 31) / 32, i = min(lo + (lane + 1) * step, hi);
    const uint32_t above = __ballot_sync(0xffffffffu, tiles[i] > at);
    const int f = __ffs(above) - 1;  // lane 31's is hi at the latest
    const int nhi = min(lo + (f + 1) * step, hi);
    lo = lo + f * step;
    hi = nhi;
  }
  return lo;
}

// Sums over the rows, a key tile and head at a time: every row tile that sees the keys, in order.
template <int D>
__global__ void __launch_bounds__(MS_THREADS) mass_keys_kernel(const __grid_constant__ MassParams mp) {
  const PagedAttnParams& p = mp.a;
  constexpr int M = MS_M, KT = MS_KT;
  extern __shared__ __align__(16) float ms_smem[];
  float* ks = ms_smem;
  float* qs = ks + KT * (D + 4);
  float* ss = qs + M * D;  // [4][KT]
  __shared__ float2 ml[M];
  __shared__ int lim[M];
  const int tid = threadIdx.x, lane = tid & 31;
  pdl_wait();
  pdl_launch_dependents();
  const long long total = mp.tiles[p.B];
  const int sk = tid & 63, sr = (tid >> 6) * 4;
  for (long long at = blockIdx.x; at < total; at += gridDim.x) {
    const int b = mass_request(mp.tiles, p.B, at, lane);
    const PagedSeg g = paged_seg(p, mp.kinds, b);
    const int nt = (g.klen + KT - 1) / KT;
    const int head = int((at - mp.tiles[b]) / nt), kt = int((at - mp.tiles[b]) - (long long)head * nt);
    __syncthreads();
    mass_load_k<D>(p, g, head, kt, ks);
    const int key = kt * KT + sk, rows = g.n * p.rep;
    // the first row that sees the tile's first key
    const int first = max(0, kt * KT - (g.klen - g.n)) * p.rep / M * M;
    float sum = 0.f;
    for (int rho0 = first; rho0 < rows; rho0 += M) {
      __syncthreads();
      mass_load_q<D>(p, g, head, rho0, qs);
      if (tid < M) {
        const PagedRow r = paged_row(p, g, head, rho0 + tid);
        ml[tid] = r.valid ? mp.row_ml[(long long)r.tok * p.H + r.h] : make_float2(0.f, 0.f);
        lim[tid] = r.lim;
      }
      __syncthreads();
      float s[4] = {};
      mass_scores<D>(qs, ks, sk, sr, s);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (key < lim[sr + i]) sum += exp2f(s[i] * p.scale_log2 - ml[sr + i].x) * ml[sr + i].y;
    }
    ss[(tid >> 6) * KT + sk] = sum;
    __syncthreads();
    if (tid < KT && key < g.klen) {
      const int page = paged_page(p, g, key >> p.page_log2);
      if (page >= 0) {
        float* to = mp.mass.ptr + page * mp.mass.page + head * mp.mass.head + (key & ((1 << p.page_log2) - 1));
        const float was = mp.add && key < g.klen - g.n ? *to : 0.f;
        *to = was + ((ss[tid] + ss[KT + tid]) + (ss[2 * KT + tid] + ss[3 * KT + tid]));
      }
    }
    __syncthreads();
  }
  if (!mp.add && p.offsets) mass_clear(mp, blockIdx.x, gridDim.x);
}

// ---- few rows (bf16 pages, at most 16 a KV head: steps and accepted chains)
// K's bytes bound the time, so it is read once. The first kernel takes scores (keys as the products' rows, mma
// m16n8k16) and keeps them, 4 bytes a key and row beside the key's 2 head_dim; the second, on the same
// shares, turns them into weights and adds them up. Four producer warps stream tiles of 64 keys
// (cp.async, 16 bytes a lane) through a ring that fills shared memory: the bytes on their way do not depend
// on how an SM happens to be split between L1 and shared memory, nor on the pages' size. Two sets of four warps take the tiles in turn, 16 keys a
// warp; each warp keeps its own maximum and sum. 64 steps of up to 12289 keys, pages of 16: 137 us, 5.7 TB/s of
// K; with TMA copies, 4 KB each at that page size, 152 us. A product sums over head_dim in any order, so a lane's
// 16 consecutive bytes of a key serve as the places that the operand's layout gives it, if the query's are
// taken alike: no operand is rearranged.
constexpr int MF_CONSUMERS = 8, MF_PRODUCERS = 4, MF_THREADS = 32 * (MF_CONSUMERS + MF_PRODUCERS), MF_M = 16, MF_KT = 64;
constexpr int MF_OVER = 4;  // 64 ragged steps: 0, 1 and 2 185 to 187 us, 4 182
constexpr int MF_SPREAD = 4, MF_KEYS_THREADS = 256;  // blocks of the second kernel for one of the first

template <int D>
struct MfLayout {
  static constexpr int kStage = MF_KT * D * 2;
  static constexpr int kTail = 8 * kWalkShared + 16 + 24 * 16;
  static constexpr int kFit = (int(kSmemOptinBytes) - 1024 - kTail) / kStage;
  // a multiple of the sets and of the producers: a stage is always of the same ones, which then see each phase
  static constexpr int kStages = (kFit < 24 ? kFit : 24) / MF_PRODUCERS * MF_PRODUCERS;
  static constexpr size_t bytes() { return 1024 + size_t(kStages) * kStage + kTail; }
};

// Where the warps' states of an item's rows lie that one block has whole: rows of 8, an item's in a row.
__device__ __forceinline__ int mass_whole_at(const PagedAttnParams& p, const PagedSeg& g, int head) {
  return g.tok0 * p.H + head * g.n * p.rep;
}

template <int D, int NT>
__global__ void __launch_bounds__(MF_THREADS, 1)
    mass_few_rows_kernel(const __grid_constant__ MassParams mp) {
  const PagedAttnParams& p = mp.a;
  using L = MfLayout<D>;
  constexpr int NV = D / 32, NST = L::kStages;  // 16-byte pieces of a key in a lane
  extern __shared__ unsigned char mf_raw[];
  unsigned char* ring = mf_raw + ((1024u - (smem_addr(mf_raw) & 1023u)) & 1023u);
  unsigned char* tail = ring + size_t(NST) * L::kStage;
  long long* sh = reinterpret_cast<long long*>(tail);
  volatile int* dead = reinterpret_cast<volatile int*>(tail + 8 * kWalkShared);
  uint64_t* full = reinterpret_cast<uint64_t*>(tail + 8 * kWalkShared + 16);
  uint64_t* empty = full + NST;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid < NST) {
    mbar_init(full + tid, 32);
    mbar_init(empty + tid, MF_CONSUMERS / 2);
    mbar_fence_init();
  }
  if (tid == 0) {
    *dead = 0;
    sh[35] = 0;
  }
  pdl_wait();
  pdl_launch_dependents();
  __syncthreads();
  PagedWalk<MF_M, MF_KT, MF_OVER> w;
  MassPiece* piece = mp.pieces + (long long)blockIdx.x * mp.most;
  if (!w.begin(p, mp.kinds, 1, sh)) {
    if (tid == 0) piece->tiles = 0;
    return;
  }
  if (w.per > mp.per) {  // more keys than the pool holds: requests share pages
    if (tid == 0) {
      raise_error(p.err, kErrPage);
      piece->tiles = 0;
    }
    return;
  }
  int pos = 0;  // tiles of the block before the item's
  if (warp >= MF_CONSUMERS) {  // ---- producers: every fourth tile
    constexpr int CH = D / 8, RPI = 32 / CH;  // 16-byte pieces of a row, rows a step
    const int c = lane % CH, r0 = lane / CH;
    unsigned char* mine = ring + (c / 8) * (MF_KT * 128);
    do {
      PageWindow win;
      win.start(p, w.g, (w.kt0 * MF_KT) >> p.page_log2, lane);
      const int nt = (min(w.kt1 * MF_KT, w.g.klen) - w.kt0 * MF_KT + MF_KT - 1) / MF_KT;
      const uint16_t* head = static_cast<const uint16_t*>(p.K.ptr) + w.head * p.K.head + c * 8;
      for (int t = (warp - pos) & (MF_PRODUCERS - 1); t < nt && !*dead; t += MF_PRODUCERS) {
        const int at = pos + t, s = at % NST, key0 = (w.kt0 + t) * MF_KT, first = key0 >> p.page_log2;
        win.seek(p, first, lane);
        if (at >= NST) paged_wait(empty + s, ((at / NST) - 1) & 1, dead, p.err);
        unsigned char* dst = mine + size_t(s) * L::kStage;
#pragma unroll
        for (int k = 0; k < MF_KT; k += 16) {  // 16 rows lie in one page
          const int key = key0 + k, page = __shfl_sync(0xffffffffu, win.cur, ((key >> p.page_log2) - win.base) & 31);
          const bool there = page < p.pages;
          const uint16_t* src = head + (there ? page : 0) * p.K.page + ((key & ((1 << p.page_log2) - 1)) + r0) * p.K.row;
#pragma unroll
          for (int i = 0; i < 16; i += RPI) {
            const int row = k + i + r0;
            cp_async16(dst + row * 128 + (((c & 7) ^ (row & 7)) << 4), src + i * p.K.row, there ? 16 : 0);
          }
        }
        cp_async_arrive(full + s);
      }
      pos += nt;
    } while (!*dead && w.next(p, mp.kinds));
    cp_async_commit();
    cp_async_wait<0>();  // shared memory must outlive the copies
    return;
  }
  // ---- scores: lane (g8, t4) has keys of a slice and 16-byte pieces t4, t4 + 4, ... of them. Which keys is free:
  // neighbours in g8 are four rows apart, where the swizzle has them in different banks.
  const int g8 = lane >> 2, t4 = lane & 3, kr = (g8 >> 1) | ((g8 & 1) << 2);
  const int set = warp >> 2, slice = (warp & 3) * 16;
  float* buf = mp.scores + (long long)blockIdx.x * mp.per * MF_KT * mp.width;
  if (blockIdx.x == MF_OVER / w.per)  // it has the line's first tile
    mass_check_pool<32 * MF_CONSUMERS>(mp, tid, reinterpret_cast<unsigned long long*>(sh + 35));
  do {
    const int R = min(w.g.n * p.rep, 8 * NT);
    uint4 q[NT][NV];
    int lim[NT][2];
    float m[NT][2], l[NT][2];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const PagedRow r = paged_row(p, w.g, w.head, t * 8 + g8);
#pragma unroll
      for (int i = 0; i < NV; ++i)
        q[t][i] = r.valid ? *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.q) + r.tok * p.q_row +
                                                            r.h * p.q_head + i * 32 + t4 * 8)
                          : make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        lim[t][e] = paged_row(p, w.g, w.head, t * 8 + 2 * t4 + e).lim;
        m[t][e] = -INFINITY;
        l[t][e] = 0.f;
      }
    }
    const int nt = (min(w.kt1 * MF_KT, w.g.klen) - w.kt0 * MF_KT + MF_KT - 1) / MF_KT;
    if (tid == 0 && nt > 0)
      *piece++ = MassPiece{w.g.idx, w.head, w.kt0 * MF_KT, nt, w.g.klen, w.g.klen - w.g.n, R, mass_whole_at(p, w.g, w.head),
                           w.first, w.count, {}};
    for (int t = (pos ^ set) & 1; t < nt; t += 2) {
      const int s = (pos + t) % NST;
      paged_wait(full + s, ((pos + t) / NST) & 1, dead, p.err);
      const unsigned char* k = ring + size_t(s) * L::kStage + (slice + kr) * 128;
      uint4 a[NV], b[NV];
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = (i / 2) * (MF_KT * 128) + ((((i & 1) * 4 + t4) ^ kr) << 4);
        a[i] = *reinterpret_cast<const uint4*>(k + c);
        b[i] = *reinterpret_cast<const uint4*>(k + 8 * 128 + c);
      }
      float c[NT][4];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        c[n][0] = c[n][1] = c[n][2] = c[n][3] = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          mma_bf16_16816(c[n], make_uint4(a[i].x, b[i].x, a[i].y, b[i].y), q[n][i].x, q[n][i].y);
          mma_bf16_16816(c[n], make_uint4(a[i].z, b[i].z, a[i].w, b[i].w), q[n][i].z, q[n][i].w);
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(empty + s);
      const int key = (w.kt0 + t) * MF_KT + slice + kr;
      float* to = buf + (size_t)t * MF_KT * mp.width + slice + kr;
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float z0 = key < lim[n][e] ? c[n][e] * p.scale_log2 : -INFINITY;
          const float z1 = key + 8 < lim[n][e] ? c[n][2 + e] * p.scale_log2 : -INFINITY;
          const int row = n * 8 + 2 * t4 + e;
          if (row < R) {
            to[row * MF_KT] = z0;
            to[row * MF_KT + 8] = z1;
          }
          const float mn = fmaxf(m[n][e], fmaxf(z0, z1)), mg = mn == -INFINITY ? 0.f : mn;
          l[n][e] = l[n][e] * ex2_approx(m[n][e] - mg) + (ex2_approx(z0 - mg) + ex2_approx(z1 - mg));
          m[n][e] = mn;
        }
    }
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
#pragma unroll
        for (int o = 4; o < 32; o *= 2) {
          const float m2 = __shfl_xor_sync(0xffffffffu, m[n][e], o), l2 = __shfl_xor_sync(0xffffffffu, l[n][e], o);
          const float mn = fmaxf(m[n][e], m2), mg = mn == -INFINITY ? 0.f : mn;
          l[n][e] = l[n][e] * ex2_approx(m[n][e] - mg) + l2 * ex2_approx(m2 - mg);
          m[n][e] = mn;
        }
        const int row = n * 8 + 2 * t4 + e;
        if (g8 == 0 && row < R) {
          float2* at = w.count == 1 ? mp.row_ml + (mass_whole_at(p, w.g, w.head) + (long long)row) * MF_CONSUMERS
                                    : mp.part_ml + (((long long)blockIdx.x * 2 + w.slot()) * MF_M + row) * MF_CONSUMERS;
          at[warp] = make_float2(m[n][e], l[n][e]);
        }
      }
    buf += (size_t)nt * MF_KT * mp.width;
    pos += nt;
  } while (w.next(p, mp.kinds));
  if (tid == 0) piece->tiles = 0;
}

// The scores' weights, added up: a thread has four keys, MF_SPREAD blocks share what one block before had. Bound
// by latency: piece -> states -> weights, a few pieces a block (28 us where the kernel before takes 137; with 2
// blocks for one 193 us together, with 4 or 8 185).
__global__ void __launch_bounds__(MF_KEYS_THREADS, 4) mass_few_keys_kernel(const __grid_constant__ MassParams mp, bool wide) {
  const PagedAttnParams& p = mp.a;
  __shared__ float2 ml[2][MF_M];
  const int tid = threadIdx.x, row = tid >> 4, part = tid & 15;
  pdl_wait();
  pdl_launch_dependents();
  const float* buf = mp.scores + (long long)blockIdx.x * mp.per * MF_KT * mp.width;
  const MassPiece* pieces = mp.pieces + (long long)blockIdx.x * mp.most;
  MassPiece g = pieces[0];
  for (int n = 1; g.tiles > 0; ++n) {
    const MassPiece next = pieces[n];
    const int* table = p.table + (long long)g.request * p.table_ld;
    const int keys = min(g.tiles * MF_KT, g.klen - g.key0), old = mp.add ? g.old : 0;
    int k = (blockIdx.y * MF_KEYS_THREADS + tid) * 4;
    // the page of all four (pages begin at multiples of 16); one outside the pool is written nothing
    int page = k < keys ? table[(g.key0 + k) >> p.page_log2] : -1;
    float M = -INFINITY, L = 0.f;
    if (row < g.rows) {
      if (g.count == 1) {
        if (part < MF_CONSUMERS) {
          const float2 y = mp.row_ml[(g.at + (long long)row) * MF_CONSUMERS + part];
          M = y.x;
          L = y.y;
        }
      } else {
        for (int i = part; i < g.count * MF_CONSUMERS; i += 16) {
          const int block = i / MF_CONSUMERS;
          const float2 y = mp.part_ml[((((long long)g.first + block) * 2 + (block == 0 ? 1 : 0)) * MF_M + row) * MF_CONSUMERS + i % MF_CONSUMERS];
          const float mn = fmaxf(M, y.x), mg = mn == -INFINITY ? 0.f : mn;
          L = L * ex2_approx(M - mg) + y.y * ex2_approx(y.x - mg);
          M = mn;
        }
      }
    }
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) {
      const float m2 = __shfl_xor_sync(0xffffffffu, M, o), l2 = __shfl_xor_sync(0xffffffffu, L, o);
      const float mn = fmaxf(M, m2), mg = mn == -INFINITY ? 0.f : mn;
      L = L * ex2_approx(M - mg) + l2 * ex2_approx(m2 - mg);
      M = mn;
    }
    if (part == 0) ml[n & 1][row] = mass_row(M, L);
    __syncthreads();  // and the other buffer's readers have passed the one before
    while (k < keys) {
      const float* z = buf + (size_t)(k / MF_KT) * MF_KT * mp.width + k % MF_KT;
      const int key = g.key0 + k;
      float* to = nullptr;
      float was[4] = {0.f, 0.f, 0.f, 0.f};
      const bool four = wide && k + 4 <= keys;
      if (page >= 0 && page < p.pages) {
        to = mp.mass.ptr + page * mp.mass.page + g.head * mp.mass.head + (key & ((1 << p.page_log2) - 1));
        if (four && key + 4 <= old) {
          const float4 y = *reinterpret_cast<const float4*>(to);
          was[0] = y.x, was[1] = y.y, was[2] = y.z, was[3] = y.w;
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (key + e < old && k + e < keys) was[e] = to[e];
        }
      }
      float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
      for (int r = 0; r < g.rows; ++r) {
        const float4 y = *reinterpret_cast<const float4*>(z + r * MF_KT);
        const float2 s = ml[n & 1][r];
        sum[0] += ex2_approx(y.x - s.x) * s.y;
        sum[1] += ex2_approx(y.y - s.x) * s.y;
        sum[2] += ex2_approx(y.z - s.x) * s.y;
        sum[3] += ex2_approx(y.w - s.x) * s.y;
      }
      // The score that a row has for a new key it does not see, -inf, gives a weight of 0 unless the row's sum is no
      // number: then without such rows.
      if (key + 3 > g.old && !(fabsf((sum[0] + sum[1]) + (sum[2] + sum[3])) < INFINITY)) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          sum[e] = 0.f;
#pragma unroll 1
          for (int r = max(0, key + e - g.old) * p.rep; r < g.rows; ++r)
            sum[e] += ex2_approx(z[r * MF_KT + e] - ml[n & 1][r].x) * ml[n & 1][r].y;
        }
      }
      if (to) {
        if (four) {
          *reinterpret_cast<float4*>(to) = make_float4(was[0] + sum[0], was[1] + sum[1], was[2] + sum[2], was[3] + sum[3]);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (k + e < keys) to[e] = was[e] + sum[e];
        }
      }
      k += MF_SPREAD * MF_KEYS_THREADS * 4;
      if (k < keys) page = table[(g.key0 + k) >> p.page_log2];
    }
    buf += (size_t)g.tiles * MF_KT * mp.width;
    g = next;
  }
  if (!mp.add && p.offsets) mass_clear(mp, blockIdx.y * gridDim.x + blockIdx.x, gridDim.x * gridDim.y);
}

// ---- many rows (bf16 pages, more than 16 a KV head: windows and prompts)
// Scores on tensor memory, twice. First with the rows as the product's lanes, 128 keys as its columns: a
// thread has a row and needs its maximum and sum alone. Then turned round: a thread has a key, the columns
// are 128 rows, and the key's weights are added up where they are, without an exchange between threads.
// Weights are 2^(s - L), L = M + log2(sum).
//
// Both kernels are one code: a lane operand A that stays for an item, a column operand B that streams, four
// groups of four warps that read the products from tensor memory, a buffer each. kMode: rows of at most
// 128 a request (the groups take the B tiles in turn); rows of more (two groups for each half of 256 lanes);
// keys (the same, 256 keys), with rings for prompts (Q streams) or for windows (K streams). The first kernel
// leaves the query tiles as it had them in shared memory, so that the second has each of them by one copy:
// gathered row by row again, they took 3600 clocks a tile. Prompts of up to 4096 rows, 32 heads: 467 us, the
// exponential unit 69 and 73% busy in the two; windows of 32 rows over 8 x 16384 keys: 125 us, 4.4 TB/s of K in the
// first.
// Bound by the exponential unit: 16 a clock, 1024 clocks for a product of 512. With two groups of two
// buffers the unit was 48 to 60% busy, two warps a scheduler being too few to cover the loads' latency.
enum MassModes : int { kRows128 = 0, kRows256 = 1, kKeysPrompt = 2, kKeysWindow = 3 };
constexpr int MM_THREADS = 640;  // 3 warps of copies (K and Q), products; 4 x 4 warps of sums
constexpr int MM_OVER = 2, MK_OVER = 2, MK_KEYS = 256;

template <int D, int kMode>
struct MmLayout {
  // tiles of 128 rows: the operand that streams has the deeper ring (windows: K from memory, at 44 GB/s an SM)
  static constexpr int KS = kMode == kRows128 ? 5 : kMode == kRows256 ? 3 : kMode == kKeysPrompt ? 2 : 4, QS = 6 - KS;
  static constexpr int kTile = 128 * D * 2;
  static constexpr int kTail = 8 * kWalkShared + 256 + QS * 128 * 4 + 2 * 3 * 128 * 8;
  static constexpr size_t bytes() { return 1024 + size_t(KS + QS) * kTile + kTail; }
};

// The line of key tiles (256 keys), each with the row tiles that see it: a block's share begins and ends anywhere.
struct MassWalk {
  PagedSeg g;
  int seg, head, kt, nkt;
  int QT, qf;         // row tiles of the request, the first that sees the key tile
  int qt0, qt1;       // this block's
  int first, count;   // the blocks that share the tile
  int per;
  long long pos, lo, hi;

  __device__ __forceinline__ int first_row_tile(const PagedAttnParams& p, int k) const {
    const int i = k * MK_KEYS - (g.klen - g.n);  // the first row that sees the tile's first key
    return i <= 0 ? 0 : int((long long)i * p.rep / 128);
  }
  __device__ __forceinline__ void enter(const PagedAttnParams& p) {  // a segment
    nkt = (g.klen + MK_KEYS - 1) / MK_KEYS;
    QT = (g.n * p.rep + 127) / 128;
  }
  __device__ __forceinline__ int plain_tiles() const {  // key tiles that every row tile sees
    return g.klen < g.n ? 0 : min(nkt, (g.klen - g.n) / MK_KEYS + 1);
  }
  __device__ long long units(const PagedAttnParams& p) {  // of one head
    if (g.n <= 0 || g.klen <= 0) return 0;
    enter(p);
    const int plain = plain_tiles();
    long long u = (long long)plain * (QT + MK_OVER);
    for (int k = plain; k < nkt; ++k) u += QT - first_row_tile(p, k) + MK_OVER;
    return u;
  }
  // Block-collective; false: no work.
  __device__ bool begin(const PagedAttnParams& p, int kinds, long long* sh) {
    const int tid = threadIdx.x, nt = blockDim.x, lane = tid & 31, warp = tid >> 5, nw = nt >> 5;
    long long total = 0;
    for (int pass = 0; pass < 2; ++pass) {
      if (pass) {
        per = int(max(1ll, (total + gridDim.x - 1) / gridDim.x));
        lo = (long long)blockIdx.x * per;
        hi = min(lo + per, total);
        if (lo >= hi) return false;
      }
      long long base = 0;
      for (int s0 = 0; s0 < p.B; s0 += nt) {
        const int s = s0 + tid;
        long long w = 0;
        if (s < p.B) {
          g = paged_seg(p, kinds, s);
          w = units(p) * p.Hk;
        }
        long long x = w;
#pragma unroll
        for (int o = 1; o < 32; o *= 2) {
          const long long y = __shfl_up_sync(0xffffffffu, x, o);
          if (lane >= o) x += y;
        }
        if (lane == 31) sh[warp] = x;
        __syncthreads();
        long long before = base;
        for (int i = 0; i < nw; ++i) {
          if (i < warp) before += sh[i];
          base += sh[i];
        }
        const long long a = before + x - w;
        if (pass && a <= lo && lo < a + w) {
          sh[32] = s;
          sh[33] = a;
          sh[34] = w;
        }
        __syncthreads();
      }
      total = base;
    }
    seg = int(sh[32]);
    const long long ph = sh[34] / p.Hk;
    g = paged_seg(p, kinds, seg);
    enter(p);
    head = int((lo - sh[33]) / ph);
    pos = sh[33] + head * ph;
    kt = int(min((long long)plain_tiles(), (lo - pos) / (QT + MK_OVER)));
    pos += (long long)kt * (QT + MK_OVER);
    for (;;) {
      qf = first_row_tile(p, kt);
      if (pos + QT - qf + MK_OVER > lo) break;
      pos += QT - qf + MK_OVER;
      ++kt;
    }
    return place() || next(p, kinds);
  }
  __device__ bool place() {
    const long long at = pos + MK_OVER;
    if (at >= lo && at + QT - qf <= hi) {  // whole, without a division
      qt0 = qf;
      qt1 = QT;
      first = blockIdx.x;
      count = 1;
      return true;
    }
    qt0 = qf + int(max(0ll, lo - at));
    qt1 = int(min((long long)QT, qf + hi - at));
    first = int(paged_div(at, per));
    count = int(paged_div(at + QT - qf - 1, per)) - first + 1;
    return qt1 > qt0;
  }
  __device__ bool next(const PagedAttnParams& p, int kinds) {
    do {
      pos += QT - qf + MK_OVER;
      if (pos >= hi) return false;
      if (++kt == nkt) {
        kt = 0;
        if (++head == p.Hk) {
          head = 0;
          do {
            g = paged_seg(p, kinds, ++seg);
          } while (g.n <= 0 || g.klen <= 0);
          enter(p);
        }
      }
      qf = first_row_tile(p, kt);
    } while (!place());
    return true;
  }
  __device__ int slot() const { return qt0 > qf ? 0 : 1; }
};

template <int D, int kMode>
__global__ void __launch_bounds__(MM_THREADS, 1)
    mass_many_kernel(const __grid_constant__ CUtensorMap tk, const __grid_constant__ MassParams mp) {
  constexpr bool kKeys = kMode >= kKeysPrompt, kTwo = kMode != kRows128;
  using L = MmLayout<D, kMode>;
  using Walk = std::conditional_t<kKeys, MassWalk, PagedWalk<kTwo ? 256 : 128, 128, MM_OVER>>;
  // Warps that copy K and Q. Where two take K's tiles in turn the ring is even: a stage stays with one of them.
  constexpr int KW = kKeys ? 2 : 1, QW = 3 - KW;
  constexpr int M = kTwo ? 256 : 128, KS = L::KS, QS = L::QS, HALVES = D / 64;
  static_assert(KS % KW == 0, "stages");
  const PagedAttnParams& p = mp.a;
  extern __shared__ unsigned char mm_raw[];
  unsigned char* sm = mm_raw + ((1024u - (smem_addr(mm_raw) & 1023u)) & 1023u);
  unsigned char* ks = sm;                             // [KS][half][128 keys][128 B], swizzled
  unsigned char* qs = sm + size_t(KS) * L::kTile;     // [QS][half][128 rows][128 B]
  unsigned char* tail = qs + size_t(QS) * L::kTile;
  long long* sh = reinterpret_cast<long long*>(tail);
  uint64_t* bars = reinterpret_cast<uint64_t*>(tail + 8 * kWalkShared);
  uint64_t* k_full = bars;        // [KS]
  uint64_t* k_empty = bars + 5;   // [KS]
  uint64_t* q_full = bars + 10;   // [QS]
  uint64_t* q_empty = bars + 14;  // [QS]
  uint64_t* s_full = bars + 18;   // [4]: a group's product is complete
  uint64_t* s_empty = bars + 22;  // [4]: and read
  uint64_t* x_full = bars + 26;   // [2]: the other groups' states are in shared memory
  uint64_t* x_empty = bars + 28;  // [2]: and read
  uint64_t* drain = bars + 30;
  volatile int* dead = reinterpret_cast<volatile int*>(bars + 31);
  uint32_t* tslot = reinterpret_cast<uint32_t*>(bars + 31) + 1;
  static_assert(KS <= 5 && QS <= 4, "barriers");
  float* nl = reinterpret_cast<float*>(tail + 8 * kWalkShared + 256);  // [QS][128]: -L of the tile's rows
  float2* xml = reinterpret_cast<float2*>(nl + QS * 128);              // [item & 1][group - 1][lane]
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    for (int i = 0; i < KS; ++i) {
      mbar_init(k_full + i, 1);
      mbar_init(k_empty + i, 1);
    }
    for (int i = 0; i < QS; ++i) {
      mbar_init(q_full + i, kKeys ? 1 : QW);
      mbar_init(q_empty + i, kKeys ? 9 : 1);  // two groups read a tile's L
    }
    for (int i = 0; i < 4; ++i) {
      mbar_init(s_full + i, 1);
      mbar_init(s_empty + i, 4);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(x_full + i, kTwo ? 8 : 12);
      mbar_init(x_empty + i, kTwo ? 8 : 4);
    }
    mbar_init(drain, 1);
    mbar_fence_init();
    *dead = 0;
    sh[35] = 0;
  }
  pdl_wait();
  pdl_launch_dependents();
  if constexpr (!kKeys) paged_no_rec(p);
  else if (tid == 0) mp.keys_rec[blockIdx.x] = MassRec{0, 0, 0, 0};
  Walk w;
  bool work;
  if constexpr (kKeys) work = w.begin(p, mp.kinds, sh);
  else work = w.begin(p, mp.kinds, 1, sh);
  if (!work) return;
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(smem_addr(tslot)),
                 "r"(512u)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tslot;

  // An item: its A tiles (one or two in use), its B tiles, the K tiles' first key
  struct Item {
    int nb, key0, rho0, tile;  // tile: the first row tile's number
    bool two, first;           // first: this block has the item's first key tile
  };
  auto item_of = [&](const Walk& x) {
    Item it;
    if constexpr (kKeys) {
      it.nb = x.qt1 - x.qt0;
      it.key0 = x.kt * MK_KEYS;
      it.rho0 = x.qt0 * 128;
      it.two = x.g.klen - it.key0 > 128;
      it.tile = mass_tile(p, x.g.tok0, x.g.idx, x.qt0);
      it.first = false;
    } else {
      it.nb = x.kt1 - x.kt0;
      it.key0 = x.kt0 * 128;
      it.rho0 = x.qt * M;
      it.two = kTwo && x.g.n * p.rep - it.rho0 > 128;
      it.tile = mass_tile(p, x.g.tok0, x.g.idx, x.qt * (M / 128));
      it.first = x.kt0 == 0;
    }
    return it;
  };

  if (warp < KW) {  // ---- K tiles, in turn
    const int psize = 1 << p.page_log2, box = min(psize, 128), parts = 128 / box;
    const int part = lane / HALVES, half = lane % HALVES, at = half * (128 * 128) + part * box * 128;
    int pos = 0, last = -1;
    do {
      const Item it = item_of(w);
      const int nt = kKeys ? 2 : it.nb;
      const int* row = p.table + (long long)w.g.idx * p.table_ld;
      const int npages = min((w.g.klen + psize - 1) >> p.page_log2, p.table_cols);
      auto fetch = [&](int t) {  // the page of this lane's copy of tile t; one outside the pool reads as zeros
        const int i = ((it.key0 + t * 128) >> p.page_log2) + part;
        if (part >= parts || t >= nt || i >= npages) return p.pages;
        const int page = row[i];
        if (page >= 0 && page < p.pages) return page;
        raise_error(p.err, kErrPage);
        return p.pages;
      };
      int t = (warp + pos) % KW;
      int page = fetch(t);
      for (; t < nt; t += KW) {
        const int q = pos + t, s = q % KS, next = fetch(t + KW);
        if (q >= KS) paged_wait(k_empty + s, ((q / KS) - 1) & 1, dead, p.err);
        if (__any_sync(0xffffffffu, *dead)) break;
        if (lane == 0) mbar_arrive_expect_tx(k_full + s, L::kTile);
        __syncwarp();
        if (part < parts)
          tma_load_5d(ks + size_t(s) * L::kTile + at, &tk, 0, (it.key0 + t * 128) & (psize - 1), half, w.head, page, k_full + s);
        page = next;
        last = q;
      }
      pos += nt;
    } while (!*dead && w.next(p, mp.kinds));
    // shared memory must outlive the copies: the last one of this warp's, and those before it where nobody waited
    if (lane == 0)
      for (int q = max(warp, last - KS + KW); q <= last; q += KW)
        if (!mbar_wait(k_full + q % KS, (q / KS) & 1)) raise_error(p.err, kErrTimeout);
  } else if (warp == 3) {  // ---- products: the warp walks together, one lane issues
    constexpr uint32_t id = umma_idesc_bf16_m128(128, 0);
    const bool issuer = elect_one();
    const uint32_t k_lo = umma_lo(smem_addr(ks), 1), q_lo = umma_lo(smem_addr(qs), 1);
    int kpos = 0, qpos = 0;
    uint32_t used = 0, phase = 0;  // by group, as bits
    auto product = [&](int group, int kslot, int qslot) {
      if ((used >> group) & 1) {
        paged_wait(s_empty + group, (phase >> group) & 1, dead, p.err);
        phase ^= 1u << group;
      }
      used |= 1u << group;
      tc_fence_after();
      if (issuer) {
        const uint32_t kt = k_lo + kslot * (L::kTile / 16), qt = q_lo + qslot * (L::kTile / 16);
        const uint32_t a = kKeys ? kt : qt, b = kKeys ? qt : kt;
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk)
          umma_ss(tmem + group * 128, a + (kk / 4) * (128 * 128 / 16) + (kk % 4) * 2, b + (kk / 4) * (128 * 128 / 16) + (kk % 4) * 2,
                  id, kk != 0);
        umma_commit(s_full + group);
      }
    };
    auto done = [&](uint64_t* bar) {
      if (issuer) umma_commit(bar);
    };
    do {
      const Item it = item_of(w);
      const int ka = kpos, qa = qpos;  // the item's A tiles
      if constexpr (kKeys) {
        for (int a = 0; a < 2; ++a, ++kpos) paged_wait(k_full + kpos % KS, (kpos / KS) & 1, dead, p.err);
      } else {
        qpos += kTwo ? 2 : 1;
      }
      auto query = [&](int a) { paged_wait(q_full + (qa + a) % QS, ((qa + a) / QS) & 1, dead, p.err); };
      for (int t = 0; t < it.nb && !*dead; ++t) {
        if constexpr (kKeys) {
          const int s = qpos % QS;
          paged_wait(q_full + s, (qpos / QS) & 1, dead, p.err);
          ++qpos;
          const int turn = (qpos - 1) & 1;
          product(turn, ka % KS, s);
          if (it.two) product(2 + turn, (ka + 1) % KS, s);
          done(q_empty + s);
        } else {
          const int s = kpos % KS;
          paged_wait(k_full + s, (kpos / KS) & 1, dead, p.err);
          ++kpos;
          if (t == 0) query(0);
          if constexpr (kTwo) {
            product(t & 1, s, qa % QS);
            if (t == 0) query(1);
            if (it.two) product(2 + (t & 1), s, (qa + 1) % QS);
          } else {
            product(t & 3, s, qa % QS);
          }
          done(k_empty + s);
        }
      }
      if constexpr (kKeys) {
        for (int a = 0; a < 2; ++a) done(k_empty + (ka + a) % KS);
      } else {
        for (int a = 0; a < (kTwo ? 2 : 1); ++a) done(q_empty + (qa + a) % QS);
      }
    } while (!*dead && w.next(p, mp.kinds));
    done(drain);  // tensor memory is given back only when nothing writes it any more
    if (!mbar_wait(drain, 0)) raise_error(p.err, kErrTimeout);
    __syncwarp();
  } else if (kKeys && warp < 3) {  // ---- Q tiles with their rows' L, as the first kernel left them
    if (lane == 0) {
      int pos = 0;
      do {
        const Item it = item_of(w);
        const int tile = w.head * mp.ids + it.tile;
        for (int t = 0; t < it.nb; ++t, ++pos) {
          const int s = pos % QS;
          if (pos >= QS) paged_wait(q_empty + s, ((pos / QS) - 1) & 1, dead, p.err);
          if (*dead) break;
          mbar_arrive_expect_tx(q_full + s, L::kTile + 512);
          bulk_g2s(qs + size_t(s) * L::kTile, mp.rows_q + (size_t)(tile + t) * L::kTile, L::kTile, q_full + s);
          bulk_g2s(nl + s * 128, mp.rows_l + (size_t)(tile + t) * 128, 512, q_full + s);
        }
      } while (!*dead && w.next(p, mp.kinds));
      for (int q = max(0, pos - QS); q < pos; ++q)
        if (!mbar_wait(q_full + q % QS, (q / QS) & 1)) raise_error(p.err, kErrTimeout);
    }
  } else if (warp < 3) {  // ---- Q tiles: 64 or 128 rows a warp, 16 or 8 lanes a row
    constexpr int CH = D / 8, RPI = 32 / CH, QR = 128 / QW;
    const int r0 = (warp - KW) * QR, c = lane % CH;
    int pos = 0;
    do {
      const Item it = item_of(w);
      const int nt = kTwo ? 2 : 1;
      for (int t = 0; t < nt && !*dead; ++t, ++pos) {
        const int s = pos % QS;
        long long from[QR / 32];
#pragma unroll
        for (int e = 0; e < QR / 32; ++e) {
          // A tile is filled up with the request's last row, for nobody: it sees every key, so that where its product is
          // no number nor is the key's sum, as 0 times an infinite key would make it. Tiles of no rows are zeros.
          const int rho = it.rho0 + t * 128 + r0 + e * 32 + lane;
          const PagedRow r = paged_row(p, w.g, w.head, t == 0 || it.two ? min(rho, w.g.n * p.rep - 1) : rho);
          from[e] = r.valid ? r.tok * p.q_row + r.h * p.q_head : -1;
        }
        if (pos >= QS) paged_wait(q_empty + s, ((pos / QS) - 1) & 1, dead, p.err);
        if (*dead) break;
        if (lane == 0) bulk_wait_read();  // the slot's tile has left it
        __syncwarp();
        unsigned char* slot = qs + size_t(s) * L::kTile + r0 * 128;
        unsigned char* dst = slot + (c / 8) * (128 * 128);
#pragma unroll
        for (int e = 0; e < QR / 32; ++e)
#pragma unroll 4
          for (int k = 0; k < 32; k += RPI) {
            const int row = k + lane / CH;
            const long long at = __shfl_sync(0xffffffffu, from[e], row);
            cp_async16(dst + (e * 32 + row) * 128 + (((c & 7) ^ (row & 7)) << 4),
                       static_cast<const uint16_t*>(p.q) + (at < 0 ? 0 : at) + c * 8, at < 0 ? 0 : 16);
          }
        cp_async_commit();
        cp_async_wait<0>();
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(q_full + s);
          if (it.first && (t == 0 || it.two)) {
            unsigned char* to = mp.rows_q + (size_t)(w.head * mp.ids + it.tile + t) * L::kTile + r0 * 128;
#pragma unroll
            for (int h = 0; h < HALVES; ++h) bulk_s2g(to + h * (128 * 128), slot + h * (128 * 128), QR * 128);
            bulk_commit();
          }
        }
      }
    } while (!*dead && w.next(p, mp.kinds));
    if (lane == 0) bulk_wait();
  } else {  // ---- sums: a thread has a lane of its group's products
    const int group = (warp - 4) >> 2, qd = warp & 3, r128 = qd * 32 + lane;
    const int half = kTwo ? group >> 1 : 0;                    // of the item's lanes
    const int t0 = kTwo ? group & 1 : group, dt = kTwo ? 2 : 4;  // the B tiles
    const uint32_t ts = tmem + (uint32_t(qd * 32) << 16) + group * 128;
    const float sl2 = p.scale_log2;
    int ns = 0, qpos = 0, nitem = 0;
    auto scores = [&]() {  // waits for the group's next product
      paged_wait(s_full + group, ns & 1, dead, p.err);
      ++ns;
      tc_fence_after();
    };
    auto scores_read = [&]() {
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(s_empty + group);
    };
    // the states of the groups with the same lanes meet in the first of them: f(another's), in order
    auto meet = [&](float2 mine, auto f) {
      const int xb = nitem & 1, xn = nitem >> 1;
      ++nitem;
      if (t0 > 0) {
        if (xn > 0) paged_wait(x_empty + xb, (xn - 1) & 1, dead, p.err);
        xml[(xb * 3 + group - 1) * 128 + r128] = mine;
        __syncwarp();
        if (lane == 0) mbar_arrive(x_full + xb);
      } else {
        paged_wait(x_full + xb, xn & 1, dead, p.err);
#pragma unroll
        for (int i = 1; i < (kTwo ? 2 : 4); ++i) f(xml[(xb * 3 + group + i - 1) * 128 + r128]);
        __syncwarp();
        if (lane == 0) mbar_arrive(x_empty + xb);
      }
    };
    if constexpr (kKeys) {
      do {
        const Item it = item_of(w);
        const bool active = half == 0 || it.two;
        const int key = it.key0 + half * 128 + r128;
        // one tile: its group has the item alone, and the other goes on to the next; several: the first group adds up
        const bool adds = it.nb > 1 ? t0 == 0 : (qpos & 1) == t0, mine = adds && key < w.g.klen && w.count == 1;
        int page = -1;
        float* to = nullptr;
        float was = 0.f;
        if (mine) page = paged_page(p, w.g, key >> p.page_log2);
        auto sum_before = [&]() {  // once the page's number is here, on its way beside the sums
          if (page < 0) return;
          to = mp.mass.ptr + page * mp.mass.page + w.head * mp.mass.head + (key & ((1 << p.page_log2) - 1));
          if (mp.add && key < w.g.klen - w.g.n) was = *to;
          page = -1;
        };
        // rows from this one on see the key
        const long long see = (long long)max(0, key - (w.g.klen - w.g.n)) * p.rep;
        float sum[4] = {0.f, 0.f, 0.f, 0.f};
        for (int t = (t0 ^ qpos) & 1; t < it.nb; t += 2) {
          const int q = qpos + t, s = q % QS;
          paged_wait(q_full + s, (q / QS) & 1, dead, p.err);
          if (active && !__any_sync(0xffffffffu, *dead)) {  // tensor memory is read by whole warps
            scores();
            const float* row = nl + s * 128;
            const int hide = int(min(see - (it.rho0 + t * 128), 128ll));  // columns before this one do not see the key
            if (__any_sync(0xffffffffu, hide > 0)) {
#pragma unroll 1
              for (int c = 0; c < 128; c += 32) {
                uint32_t v[32];
                tmem_ld32(ts + c, v);
#pragma unroll
                for (int i = 0; i < 32; i += 4) {
                  const float4 l4 = *reinterpret_cast<const float4*>(row + c + i);
                  const float x[4] = {l4.x, l4.y, l4.z, l4.w};
#pragma unroll
                  for (int e = 0; e < 4; ++e) {
                    const float y = ex2_approx(fmaf(__uint_as_float(v[i + e]), sl2, x[e]));
                    sum[e] += c + i + e >= hide ? y : 0.f;
                  }
                }
              }
            } else {
#pragma unroll 1
              for (int c = 0; c < 128; c += 32) {
                uint32_t v[32];
                tmem_ld32(ts + c, v);
                if (c == 32) sum_before();
#pragma unroll
                for (int i = 0; i < 32; i += 4) {
                  const float4 l4 = *reinterpret_cast<const float4*>(row + c + i);
                  sum[0] += ex2_approx(fmaf(__uint_as_float(v[i]), sl2, l4.x));
                  sum[1] += ex2_approx(fmaf(__uint_as_float(v[i + 1]), sl2, l4.y));
                  sum[2] += ex2_approx(fmaf(__uint_as_float(v[i + 2]), sl2, l4.z));
                  sum[3] += ex2_approx(fmaf(__uint_as_float(v[i + 3]), sl2, l4.w));
                }
              }
            }
            scores_read();
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(q_empty + s);
        }
        qpos += it.nb;
        if (*dead) break;
        if (it.nb == 1 && !adds) continue;
        float total = (sum[0] + sum[1]) + (sum[2] + sum[3]);
        if (it.nb > 1) meet(make_float2(total, 0.f), [&](float2 y) { total += y.x; });
        if (w.count == 1) {
          sum_before();
          if (to) *to = was + total;
        } else if (adds) {
          mp.part_sum[((long long)blockIdx.x * 2 + w.slot()) * MK_KEYS + half * 128 + r128] = total;
          if (half == 0 && qd == 0 && lane == 0 && w.slot() == 1)
            mp.keys_rec[blockIdx.x] = MassRec{w.seg, w.head, w.kt, w.count};
        }
      } while (w.next(p, mp.kinds));
    } else {
      if (blockIdx.x == MM_OVER / w.per)  // it has the line's first tile
        mass_check_pool<512>(mp, tid - 128, reinterpret_cast<unsigned long long*>(sh + 35));
      do {
        const Item it = item_of(w);
        const PagedRow r = paged_row(p, w.g, w.head, it.rho0 + half * 128 + r128);
        const int lim = r.valid ? r.lim : 0x7fffffff;  // rows that fill the tile up see everything, for nobody
        float m = -INFINITY, l = 0.f;
        if (half == 0 || it.two) {
          for (int t = t0; t < it.nb; t += dt) {
            scores();
            if (__any_sync(0xffffffffu, *dead)) break;
            const int key0 = it.key0 + t * 128;
            const bool masked = __any_sync(0xffffffffu, key0 + 128 > lim);
#pragma unroll 1
            for (int c = 0; c < 128; c += 32) {
              uint32_t v[32];
              tmem_ld32(ts + c, v);
              if (masked) {
#pragma unroll
                for (int i = 0; i < 32; ++i)
                  if (key0 + c + i >= lim) v[i] = 0xff800000u;
              }
              float mx = max3(__uint_as_float(v[0]), __uint_as_float(v[1]), __uint_as_float(v[2]));
#pragma unroll
              for (int i = 3; i < 31; i += 2) mx = max3(mx, __uint_as_float(v[i]), __uint_as_float(v[i + 1]));
              mx = fmaxf(mx, __uint_as_float(v[31]));
              const float mn = fmaxf(m, mx * sl2), mg = mn == -INFINITY ? 0.f : mn;
              float sum[4] = {l * ex2_approx(m - mg), 0.f, 0.f, 0.f};
#pragma unroll
              for (int i = 0; i < 32; ++i) sum[i & 3] += ex2_approx(fmaf(__uint_as_float(v[i]), sl2, -mg));
              l = (sum[0] + sum[1]) + (sum[2] + sum[3]);
              m = mn;
            }
            scores_read();
          }
        }
        if (*dead) break;
        meet(make_float2(m, l), [&](float2 y) {
          const float mn = fmaxf(m, y.x), mg = mn == -INFINITY ? 0.f : mn;
          l = l * ex2_approx(m - mg) + y.y * ex2_approx(y.x - mg);
          m = mn;
        });
        if (group == 0 && qd == 0 && lane == 0) w.report(p);
        if (t0 == 0 && (half == 0 || it.two)) {
          if (w.count == 1) mp.rows_l[(size_t)(w.head * mp.ids + it.tile + half) * 128 + r128] = r.valid ? mass_minus_l(m, l) : -INFINITY;
          else mp.part_ml[((long long)blockIdx.x * 2 + w.slot()) * M + half * 128 + r128] = make_float2(m, l);
        }
      } while (w.next(p, mp.kinds));
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(512u) : "memory");
  }
}

// Adds up the parts of divided key tiles, in order: one block a tile, a thread a key.
__global__ void __launch_bounds__(MK_KEYS) mass_fold_kernel(const __grid_constant__ MassParams mp) {
  const PagedAttnParams& p = mp.a;
  pdl_wait();
  pdl_launch_dependents();
  const MassRec rec = mp.keys_rec[blockIdx.x];
  if (rec.count == 0) return;
  const PagedSeg g = paged_seg(p, mp.kinds, rec.request);
  const int key = rec.kt * MK_KEYS + threadIdx.x;
  if (key >= g.klen) return;
  const int page = paged_page(p, g, key >> p.page_log2);
  if (page < 0) return;
  float sum = 0.f;
  for (int i = 0; i < rec.count; ++i)
    sum += mp.part_sum[((long long)(blockIdx.x + i) * 2 + (i == 0 ? 1 : 0)) * MK_KEYS + threadIdx.x];
  float* to = mp.mass.ptr + page * mp.mass.page + rec.head * mp.mass.head + (key & ((1 << p.page_log2) - 1));
  *to = (mp.add && key < g.klen - g.n ? *to : 0.f) + sum;
}

// ---------------------------------------------------------------------------- eviction
// Of n keys the first `sinks` and the last `recent` stay, and of those between the ones of the largest mass,
// ties to the lower key, until m are left; they move together in order. A block selects for one list (layer,
// request, head), writes down where the kept rows lie and moves their sums. Where there are lists enough it
// moves the rows as well: its selection, bound by latency, runs beside other blocks' copies, bound by HBM.
// Where there are few, a second kernel moves them, several blocks a list. 32 requests, 4 layers, 1024 lists: 305 us
// (5.3 TB/s; in two kernels 331); one request, 28 layers, 224 lists: 33 us (in two kernels 40). Lists beyond EV_CACHE
// read their sums from memory in four passes.
constexpr int EV_THREADS = 512;
constexpr int EV_CACHE = 16384;  // sums held in shared memory; those behind are read again in every pass
constexpr int EM_ROWS = 4;       // rows a thread has on their way, twice

struct EvictParams {
  PagePool K, V;
  long long k_layer, v_layer;
  MassPool mass;
  int pages, page_log2, B, Hk, layers, row_chunks, esize_log2;
  const int* table;
  int table_ld, table_cols;
  const int* lens;
  const int* budgets;  // [B] or null: `budget`
  int budget, sinks, recent;
  int* lens_out;
  int* list;           // [layers][B][Hk][1 + most]: how many rows stay in place, then the kept keys' rows in the pool
  int most;
  int cache;           // sums in shared memory
  int splits;          // of the second kernel: blocks of a list and pool, each with a part of every row; 0: no second kernel
  int* err;
};

struct EvictJob {
  int n, m;  // keys, and how many stay; n <= m: nothing to do
};
__device__ __forceinline__ EvictJob evict_job(const EvictParams& p, int b, int& bad) {
  EvictJob j;
  j.n = p.lens[b];
  j.m = p.budgets ? p.budgets[b] : p.budget;
  if (j.n < 0 || j.n > (p.table_cols << p.page_log2)) bad |= kErrCapacity;
  if (j.m < p.sinks + p.recent || j.m < 0) bad |= kErrBudget;
  if (bad) j.m = j.n = max(j.n, 0);
  return j;
}

// Larger mass, larger key; no number is below all others.
__device__ __forceinline__ uint32_t mass_key(float x) {
  return x != x ? 0u : uint32_t(argmax_key(x + 0.f, 0) >> 32);
}

// Moves the kept rows of one list together, in one pool, or a part of every row's columns: kept row i comes from
// key s_i >= i, so a step's rows are read before any is written, and no later step reads a row that an earlier
// one wrote: the next step's may be on their way before this one's are stored. Block-collective.
__device__ __forceinline__ void evict_rows(const EvictParams& p, const PagePool& pool, long long layer_stride, int layer, int b,
                                           int h, int m, const int* list, int split, int splits) {
  const int mask = (1 << p.page_log2) - 1, chunks = p.row_chunks / splits, step = EV_THREADS / chunks;
  const int* row = p.table + (long long)b * p.table_ld;
  char* base = static_cast<char*>(pool.ptr) + ((layer_stride * layer + h * pool.head) << p.esize_log2) +
               (split * chunks + int(threadIdx.x) % chunks) * 16;
  auto at = [&](int page, int r) {
    return reinterpret_cast<uint4*>(base + ((page * pool.page + r * pool.row) << p.esize_log2));
  };
  uint4 x[EM_ROWS], y[EM_ROWS];
  auto read = [&](uint4(&to)[EM_ROWS], int i0) {
    int from[EM_ROWS];
#pragma unroll
    for (int u = 0; u < EM_ROWS; ++u) from[u] = i0 + u * step < m ? list[i0 + u * step] : -1;
#pragma unroll
    for (int u = 0; u < EM_ROWS; ++u)
      if (from[u] >= 0) to[u] = *at(from[u] >> p.page_log2, from[u] & mask);
  };
  auto write = [&](const uint4(&from)[EM_ROWS], int i0) {
#pragma unroll
    for (int u = 0; u < EM_ROWS; ++u) {
      const int i = i0 + u * step;
      if (i < m) *at(row[i >> p.page_log2], i & mask) = from[u];
    }
  };
  const int tile = EM_ROWS * step;
  int i = list[-1], mine = i + int(threadIdx.x) / chunks;
  if (i >= m) return;
  read(x, mine);
  for (;;) {
    if (i + tile < m) read(y, mine + tile);
    __syncthreads();  // this step's rows are read
    write(x, mine);
    i += tile;
    mine += tile;
    if (i >= m) break;
    if (i + tile < m) read(x, mine + tile);
    __syncthreads();
    write(y, mine);
    i += tile;
    mine += tile;
    if (i >= m) break;
  }
}

__global__ void __launch_bounds__(EV_THREADS, 2) evict_kernel(const __grid_constant__ EvictParams p) {
  constexpr int BINS = 2048, WARPS = EV_THREADS / 32;
  extern __shared__ float ev_cache[];
  __shared__ int hist[BINS];
  __shared__ int s_warp[2][WARPS];
  __shared__ int s_bin, s_left;
  __shared__ int s_bad, s_still;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int h = blockIdx.x % p.Hk, lb = blockIdx.x / p.Hk, b = lb % p.B, layer = lb / p.B;
  pdl_wait();
  pdl_launch_dependents();
  int bad = 0;
  const EvictJob job = evict_job(p, b, bad);
  const int n = job.n, m = job.m, mask = (1 << p.page_log2) - 1;
  const int* row = p.table + (long long)b * p.table_ld;
  if (tid == 0) s_bad = s_still = 0;
  __syncthreads();
  if (!bad && n > m)  // a page outside the pool: the request stays as it is
    for (int c = tid; c < (n + mask) >> p.page_log2; c += EV_THREADS)
      if (row[c] < 0 || row[c] >= p.pages) s_bad = kErrPage;
  __syncthreads();
  bad |= s_bad;
  if (layer == 0 && h == 0 && tid == 0) {
    if (bad) raise_error(p.err, bad);
    p.lens_out[b] = bad ? p.lens[b] : min(n, m);
  }
  if (bad || n <= m) return;
  float* base = p.mass.ptr + layer * p.mass.layer + h * p.mass.head;
  auto at = [&](int j) { return base + row[j >> p.page_log2] * p.mass.page + (j & mask); };
  const int lo = p.sinks, hi = n - p.recent;
  int left = m - p.sinks - p.recent;  // to be taken of [lo, hi), fewer than there are
  const bool held = n <= p.cache;     // all sums in shared memory
  for (int j0 = tid; j0 < min(n, p.cache); j0 += 8 * EV_THREADS) {
    float x[8];
#pragma unroll
    for (int u = 0; u < 8; ++u)
      if (j0 + u * EV_THREADS < min(n, p.cache)) x[u] = *at(j0 + u * EV_THREADS);
#pragma unroll
    for (int u = 0; u < 8; ++u)
      if (j0 + u * EV_THREADS < min(n, p.cache)) ev_cache[j0 + u * EV_THREADS] = x[u];
  }
  auto value = [&](int j) { return j < p.cache ? ev_cache[j] : *at(j); };
  // The key of the last one taken, from its upper bits down: 11, 11, 10
  uint32_t prefix = 0;
  int shift = 32;
  for (int pass = 0; pass < 3; ++pass) {
    const int bits = pass < 2 ? 11 : 10;
    shift -= bits;
    __syncthreads();
    for (int i = tid; i < BINS; i += EV_THREADS) hist[i] = 0;
    __syncthreads();
    for (int j = lo + tid; j < hi; j += EV_THREADS) {
      const uint32_t k = mass_key(value(j));
      if (pass == 0 || (k >> (shift + bits)) == prefix) atomicAdd(hist + ((k >> shift) & ((1 << bits) - 1)), 1);
    }
    __syncthreads();
    // counts from the top: thread t has bins [4 t', 4 t' + 4) of the reversed order
    int c[4], sum = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      c[i] = hist[BINS - 1 - (4 * tid + i)];
      sum += c[i];
    }
    int x = sum;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
      const int y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    if (lane == 31) s_warp[0][warp] = x;
    __syncthreads();
    int above = x - sum;
    for (int i = 0; i < warp; ++i) above += s_warp[0][i];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (above < left && above + c[i] >= left) {
        s_bin = BINS - 1 - (4 * tid + i);
        s_left = left - above;
      }
      above += c[i];
    }
    __syncthreads();
    if (left > 0) {
      prefix = (prefix << bits) | uint32_t(s_bin);
      left = s_left;
    }
  }
  // `left` of those equal to the key, the lowest first, and all above it, in order
  const bool any = m > p.sinks + p.recent;
  int* list = p.list + (long long)blockIdx.x * (p.most + 1);
  int kept = 0, equal = 0, still = 0;
  auto keep = [&](int j, int to, float x) {
    list[1 + to] = (row[j >> p.page_log2] << p.page_log2) + (j & mask);
    if (to != j) *at(to) = x;
    else ++still;  // keys before the first gap
  };
  if (held) {
    // a warp has a run of keys: counts first, then places; sums are written to where no block reads them any more
    const int run = ((n + WARPS - 1) / WARPS + 31) & ~31, j0 = warp * run, j1 = min(j0 + run, n);
    auto look = [&](int j, bool& in, bool& tie) {
      in = tie = false;
      if (j >= j1) return;
      if (j < lo || j >= hi) {
        in = true;
      } else if (any) {
        const uint32_t k = mass_key(ev_cache[j]);
        in = k > prefix;
        tie = k == prefix;
      }
    };
    int ties = 0, ins = 0;
    for (int j = j0 + lane; j - lane < j1; j += 32) {
      bool in, tie;
      look(j, in, tie);
      ins += __popc(__ballot_sync(0xffffffffu, in));
      ties += __popc(__ballot_sync(0xffffffffu, tie));
    }
    if (lane == 0) {
      s_warp[0][warp] = ties;
      s_warp[1][warp] = ins;
    }
    __syncthreads();
    for (int i = 0; i < warp; ++i) {
      equal += s_warp[0][i];
      kept += s_warp[1][i];
    }
    for (int j = j0 + lane; j - lane < j1; j += 32) {
      bool in, tie;
      look(j, in, tie);
      const uint32_t bi = __ballot_sync(0xffffffffu, in), bt = __ballot_sync(0xffffffffu, tie), below = (1u << lane) - 1;
      const int te = equal + __popc(bt & below);
      if (in || (tie && te < left)) keep(j, kept + __popc(bi & below) + min(te, left), ev_cache[j]);
      kept += __popc(bi);
      equal += __popc(bt);
    }
  } else {
    for (int j0 = 0; j0 < n; j0 += EV_THREADS) {
      const int j = j0 + tid;
      float x = 0.f;
      bool in = false, tie = false;
      if (j < n) {
        x = *at(j);
        if (j < lo || j >= hi) {
          in = true;
        } else if (any) {
          const uint32_t k = mass_key(x);
          in = k > prefix;
          tie = k == prefix;
        }
      }
      const uint32_t ties = __ballot_sync(0xffffffffu, tie);
      const uint32_t ins = __ballot_sync(0xffffffffu, in);
      if (lane == 0) {
        s_warp[0][warp] = __popc(ties);
        s_warp[1][warp] = __popc(ins);
      }
      __syncthreads();  // all of this step's sums are read, and none of a later one's is written to
      int te = equal, ki = kept, tie_all = 0, in_all = 0;
      for (int i = 0; i < WARPS; ++i) {
        if (i < warp) {
          te += s_warp[0][i];
          ki += s_warp[1][i];
        }
        tie_all += s_warp[0][i];
        in_all += s_warp[1][i];
      }
      const uint32_t below = (1u << lane) - 1;
      te += __popc(ties & below);                        // equal ones before
      ki += __popc(ins & below) + min(te, left) - min(equal, left);
      // of the ties before this one, those of earlier steps are in `kept` already
      if (in || (tie && te < left)) keep(j, ki, x);
      kept += in_all + min(equal + tie_all, left) - min(equal, left);
      equal += tie_all;
      __syncthreads();
    }
  }
  still = __reduce_add_sync(0xffffffffu, still);
  if (lane == 0) atomicAdd(&s_still, still);
  __syncthreads();
  if (tid == 0) list[0] = s_still;
  if (p.splits) return;
  __syncthreads();
  evict_rows(p, p.K, p.k_layer, layer, b, h, m, list + 1, 0, 1);
  evict_rows(p, p.V, p.v_layer, layer, b, h, m, list + 1, 0, 1);
}

__global__ void __launch_bounds__(EV_THREADS, 2) evict_move_kernel(const __grid_constant__ EvictParams p) {
  const int tid = threadIdx.x;
  const int h = blockIdx.x % p.Hk, lb = blockIdx.x / p.Hk, b = lb % p.B, layer = lb / p.B;
  pdl_wait();
  pdl_launch_dependents();
  int bad = 0;
  const EvictJob job = evict_job(p, b, bad);
  if (bad || job.n <= job.m) return;
  const int mask = (1 << p.page_log2) - 1;
  const int* row = p.table + (long long)b * p.table_ld;
  for (int c = tid; c < (job.n + mask) >> p.page_log2; c += EV_THREADS) bad |= row[c] < 0 || row[c] >= p.pages;
  if (__syncthreads_or(bad)) return;
  const bool isv = blockIdx.y & 1;
  evict_rows(p, isv ? p.V : p.K, isv ? p.v_layer : p.k_layer, layer, b, h, job.m, p.list + (long long)blockIdx.x * (p.most + 1) + 1,
             blockIdx.y >> 1, p.splits);
}

}  // namespace wc
