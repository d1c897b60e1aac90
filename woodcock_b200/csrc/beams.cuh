// Beam search over a paged cache: the best continuations of a request's beams, and the beams' pages in
// their new order.
#pragma once

#include "common.cuh"
#include "paged_walk.cuh"

namespace wc {

// ---------------------------------------------------------------------------- selection
// score(w, v) = s_w + (z_wv - lse_w), lse_w = log sum_v exp z_wv, the n best of a request's W x V, ties to
// the lower beam, then to the lower token.
//
// Every logit is read once. A block takes a piece of one beam's row into registers (32 values a thread),
// leaves the piece's maximum and sum of exponentials, and its n best: n of the threads' maxima are at
// least some T, so at least n values are, and few more; those are collected and ranked among one
// another. The second kernel, one block a request, has each beam's lse and does the same with the
// candidates' scores.
//
// Ranks are decided in 64 bits. Two beams' scores may lie closer than a 32-bit sum resolves: a score near -20
// has steps of 2^-19, and with 64 x 16 neighbours in rank a step apart now and then. The exponentials
// are of 32 bits, but with arguments corrected to 2^-30, and their sum's error averages over the row.
constexpr int BS_THREADS = 256;
constexpr int BS_PER = 32;                       // values a thread
constexpr int BS_PIECE = BS_THREADS * BS_PER;    // values a block
constexpr int BS_LIST = BS_THREADS * 4;          // a piece of fewer values fits whole
constexpr int BS_MAX_N = 64;
constexpr int BS_MAX_W = 64;
constexpr int BJ_THREADS = 512;
constexpr int BJ_LIST = 2048;

struct BeamSelectParams {
  const void* logits;
  long long request, beam;  // strides in elements
  const float* scores;      // [B][W]
  const uint8_t* finished;  // [B][W] or null
  int B, W, V, n, pieces, pad;
  // workspace
  double2* stat;            // [B W][pieces]: maximum, sum of exponentials (NaN: a logit that is not a number or +inf)
  unsigned long long* cand; // [B W][pieces][n]: argmax_key of value and token, best first; 0: none
  float* out_scores;        // [B][n]
  int *out_parents, *out_tokens;
  int* err;
};

// e^(z - m), z <= m: what z - m and log2(e) lose to rounding is added back, so that the exponent is right to
// 2^-30 of its size. Below e^-100 nothing is left beside the maximum's 1.
__device__ __forceinline__ float exp_diff(float z, float m) {
  const float d = z - m, v = d - z;  // d + e = z - m exactly
  const float e = (z - (d - v)) - (m + v);
  constexpr float kHi = 1.44269502162933349609375f, kLo = 1.925963033500966e-08f;  // log2(e), 24 bits and the rest
  const float t = d * kHi;
  const float r = fmaf(d, kHi, -t) + fmaf(d, kLo, e * kHi);
  // 2^(t + r), r below 2^-18: 2^r = 1 + r ln 2
  const float x = ex2_approx(t);
  return d > -100.f ? fmaf(x, r * 0.69314718f, x) : 0.f;
}

// What a beam proposes: 0 nothing (it is dead, or its score is no number), 1 its tokens, 2 itself (it has ended).
__device__ __forceinline__ int beam_kind(const BeamSelectParams& p, long long row) {
  const float score = p.scores[row];
  return !(score > -INFINITY && score < INFINITY) ? 0 : p.finished && p.finished[row] ? 2 : 1;
}

// The j-th largest of a warp's keys (0: there is none).
__device__ __forceinline__ uint32_t warp_jth(uint32_t key, int j, int lane) {
  uint32_t top = 0;
  for (int i = 0; i < j; ++i) {
    top = __reduce_max_sync(0xffffffffu, key);
    const uint32_t who = __ballot_sync(0xffffffffu, key == top);
    if (lane == __ffs(who) - 1) key = 0;
  }
  return top;
}

// N values from i on; -inf behind the row's end. A row that does not begin on a 16-byte boundary is read value by
// value, so that its sum has the order of any other's: beams that are alike stay tied.
template <typename T>
__device__ __forceinline__ void load_logits(const T* row, bool whole, int i, int V, float (&x)[16 / sizeof(T)]) {
  constexpr int N = 16 / sizeof(T);
  if (whole && i + N <= V) {
    if constexpr (N == 4) {
      const float4 a = ldg_stream_f4(reinterpret_cast<const float4*>(row + i));
      x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w;
    } else {
      const uint4 a = ldg_stream(reinterpret_cast<const uint4*>(row + i));
      const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        x[2 * k] = __uint_as_float(w[k] << 16);
        x[2 * k + 1] = __uint_as_float(w[k] & 0xffff0000u);
      }
    }
  } else {
#pragma unroll
    for (int k = 0; k < N; ++k) {
      x[k] = -INFINITY;
      if (i + k < V) {
        if constexpr (N == 4) x[k] = row[i + k];
        else x[k] = bf16_bits_to_f32(row[i + k]);
      }
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(BS_THREADS) beam_pieces_kernel(const __grid_constant__ BeamSelectParams p) {
  constexpr int N = 16 / sizeof(T), NV = BS_PER / N, WARPS = BS_THREADS / 32;
  __shared__ unsigned long long list[BS_LIST];
  __shared__ float s_max[WARPS];
  __shared__ double s_sum[WARPS];
  __shared__ uint32_t s_key[WARPS];
  __shared__ int s_count, s_bad;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int row = blockIdx.x / p.pieces, piece = blockIdx.x - row * p.pieces;
  const int b = row / p.W;
  const T* z = static_cast<const T*>(p.logits) + b * p.request + (row - b * p.W) * p.beam;
  if (tid == 0) s_count = s_bad = 0;
  pdl_wait();
  pdl_launch_dependents();
  if (beam_kind(p, row) != 1) return;  // its logits do not matter
  const bool whole = (reinterpret_cast<unsigned long long>(z) & 15) == 0;
  const int first = piece * BS_PIECE;
  float x[NV][N];
#pragma unroll
  for (int v = 0; v < NV; ++v) load_logits<T>(z, whole, first + (v * BS_THREADS + tid) * N, p.V, x[v]);
  float top = -INFINITY;
  bool bad = false;
#pragma unroll
  for (int v = 0; v < NV; ++v)
#pragma unroll
    for (int k = 0; k < N; ++k) {
      bad |= !(x[v][k] < INFINITY);
      x[v][k] += 0.f;  // -0 ranks with +0
      top = fmaxf(top, x[v][k]);
    }
  const uint32_t mine = uint32_t(argmax_key(top, 0) >> 32);
  const uint32_t jth = warp_jth(mine, (p.n + WARPS - 1) / WARPS, lane);
  const float wtop = warp_max(top);
  if (lane == 0) {
    s_max[warp] = wtop;
    s_key[warp] = jth;
  }
  __syncthreads();
  if (bad) s_bad = 1;
  float m = s_max[0];
  uint32_t least = s_key[0];
#pragma unroll
  for (int i = 1; i < WARPS; ++i) {
    m = fmaxf(m, s_max[i]);
    least = min(least, s_key[i]);
  }
  const float bound = argmax_key_value((unsigned long long)(max(least, 0x00800000u)) << 32);  // above -inf
  float sum = 0.f;
  const float mg = m == -INFINITY ? 0.f : m;
#pragma unroll
  for (int v = 0; v < NV; ++v)
#pragma unroll
    for (int k = 0; k < N; ++k) {
      if (x[v][k] > -INFINITY) sum += exp_diff(x[v][k], mg);
      if (x[v][k] >= bound) {
        const int at = atomicAdd(&s_count, 1);
        if (at < BS_LIST) list[at] = argmax_key(x[v][k], uint32_t(first + (v * BS_THREADS + tid) * N + k));
      }
    }
  const double ws = warp_sum_d(double(sum));
  if (lane == 0) s_sum[warp] = ws;
  __syncthreads();
  unsigned long long* out = p.cand + (long long)blockIdx.x * p.n;
  if (tid == 0) {
    double s = 0;
    for (int i = 0; i < WARPS; ++i) s += s_sum[i];
    if (s_bad) raise_error(p.err, kErrLogits);
    p.stat[blockIdx.x] = make_double2(m, s_bad ? NAN : s);
  }
  int count = s_count;
  if (count > BS_LIST) {
    // Too many values at the bound (equal ones, or values in few threads): the n-th best key, bit by bit.
    unsigned long long nth = 0;
    for (int bit = 63; bit >= 0; --bit) {
      const unsigned long long probe = nth | (1ull << bit);
      int c = 0;
#pragma unroll
      for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int k = 0; k < N; ++k)
          c += x[v][k] >= bound && argmax_key(x[v][k], uint32_t(first + (v * BS_THREADS + tid) * N + k)) >= probe;
      c = __reduce_add_sync(0xffffffffu, c);
      __syncthreads();
      if (lane == 0) s_key[warp] = c;
      __syncthreads();
      c = 0;
      for (int i = 0; i < WARPS; ++i) c += s_key[i];
      if (c >= p.n) nth = probe;
    }
    __syncthreads();
    if (tid == 0) s_count = 0;
    __syncthreads();
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int k = 0; k < N; ++k) {
        const unsigned long long key = argmax_key(x[v][k], uint32_t(first + (v * BS_THREADS + tid) * N + k));
        if (x[v][k] >= bound && key >= nth) list[atomicAdd(&s_count, 1)] = key;  // n of them: keys differ
      }
    __syncthreads();
    count = s_count;
  }
  for (int i = tid; i < count; i += BS_THREADS) {
    const unsigned long long key = list[i];
    int rank = 0;
    for (int k = 0; k < count; ++k) rank += list[k] > key;
    if (rank < p.n) out[rank] = key;
  }
  for (int i = count + tid; i < p.n; i += BS_THREADS) out[i] = 0;
}

// A double's order as an unsigned number.
__device__ __forceinline__ unsigned long long order_of(double x) {
  const unsigned long long u = (unsigned long long)__double_as_longlong(x);
  return (u >> 63) ? ~u : u | (1ull << 63);
}
__device__ __forceinline__ double value_of(unsigned long long k) {
  return __longlong_as_double((long long)((k >> 63) ? k & ~(1ull << 63) : ~k));
}

// One block a request. Bound by latency: statistics, candidates, their ranks.
__global__ void __launch_bounds__(BJ_THREADS) beam_join_kernel(const __grid_constant__ BeamSelectParams p) {
  constexpr int WARPS = BJ_THREADS / 32;
  __shared__ unsigned long long key[BJ_LIST];
  __shared__ uint32_t place[BJ_LIST];       // beam * V + token
  __shared__ double s_score[BS_MAX_W], s_lse[BS_MAX_W];
  __shared__ int s_kind[BS_MAX_W];
  __shared__ uint32_t s_key[WARPS];
  __shared__ int s_count;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, b = blockIdx.x;
  if (tid == 0) s_count = 0;
  pdl_wait();
  for (int w = warp; w < p.W; w += WARPS) {
    const long long row = (long long)b * p.W + w;
    const double2* st = p.stat + row * p.pieces;
    const int kind = beam_kind(p, row);
    double m = -INFINITY, s = 0;
    for (int i = lane; kind == 1 && i < p.pieces; i += 32) {
      const double2 y = st[i];
      const double mn = fmax(m, y.x);
      if (!(y.x == -INFINITY && y.y == 0)) s = s * exp(m - mn) + y.y * exp(y.x - mn);
      m = mn;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const double m2 = __shfl_xor_sync(0xffffffffu, m, o), s2 = __shfl_xor_sync(0xffffffffu, s, o);
      const double mn = fmax(m, m2);
      if (mn > -INFINITY) s = s * exp(m - mn) + s2 * exp(m2 - mn);
      m = mn;
    }
    if (lane == 0) {
      const float score = p.scores[row];
      if (!(score < INFINITY)) raise_error(p.err, kErrLogits);
      s_score[w] = score;
      s_lse[w] = m + log(s);
      s_kind[w] = kind != 1 || (m > -INFINITY && s > 0) ? kind : 0;  // not without a token, nor where s is no number
    }
  }
  __syncthreads();
  const int per = p.pieces * p.n, total = p.W * per;
  const unsigned long long* cand = p.cand + (long long)b * total;
  // candidate i: its score's order (0: none) and its place
  auto look = [&](int i, uint32_t& at) -> unsigned long long {
    const int w = i / per, kind = s_kind[w];
    if (kind == 1) {
      const unsigned long long c = cand[i];
      if (!c) return 0;
      at = uint32_t(w) * uint32_t(p.V) + argmax_key_index(c);
      return order_of(s_score[w] + (double(argmax_key_value(c)) - s_lse[w]));
    }
    if (kind == 2 && i == w * per) {
      at = uint32_t(w) * uint32_t(p.V) + uint32_t(p.pad);
      return order_of(s_score[w]);
    }
    return 0;
  };
  uint32_t top = 0;
  for (int i = tid; i < total; i += BJ_THREADS) {
    uint32_t at;
    top = max(top, uint32_t(look(i, at) >> 32));
  }
  const uint32_t jth = warp_jth(top, (p.n + WARPS - 1) / WARPS, lane);
  if (lane == 0) s_key[warp] = jth;
  __syncthreads();
  uint32_t least = s_key[0];
#pragma unroll
  for (int i = 1; i < WARPS; ++i) least = min(least, s_key[i]);
  least = max(least, 1u);
  for (int i = tid; i < total; i += BJ_THREADS) {
    uint32_t at;
    const unsigned long long k = look(i, at);
    if (uint32_t(k >> 32) >= least) {
      const int to = atomicAdd(&s_count, 1);
      if (to < BJ_LIST) {
        key[to] = k;
        place[to] = at;
      }
    }
  }
  __syncthreads();
  int count = s_count;
  if (count > BJ_LIST) {
    // Scores that are all but equal: the n-th best of (score, place), bit by bit.
    auto counted = [&](auto test) {
      int c = 0;
      for (int i = tid; i < total; i += BJ_THREADS) {
        uint32_t at = 0;
        const unsigned long long k = look(i, at);
        c += k != 0 && test(k, at);
      }
      c = __reduce_add_sync(0xffffffffu, c);
      __syncthreads();
      if (lane == 0) s_key[warp] = c;
      __syncthreads();
      c = 0;
      for (int i = 0; i < WARPS; ++i) c += s_key[i];
      return c;
    };
    unsigned long long nth = 0;
    for (int bit = 63; bit >= 0; --bit) {
      const unsigned long long probe = nth | (1ull << bit);
      if (counted([&](unsigned long long k, uint32_t) { return k >= probe; }) >= p.n) nth = probe;
    }
    const int more = p.n - counted([&](unsigned long long k, uint32_t) { return k > nth; });
    uint32_t last = 0xffffffffu;  // the lowest place up to which `more` of the equal ones lie
    for (int bit = 31; bit >= 0; --bit) {
      const uint32_t probe = last & ~(1u << bit);
      if (counted([&](unsigned long long k, uint32_t at) { return k == nth && at <= probe; }) >= more) last = probe;
    }
    __syncthreads();
    if (tid == 0) s_count = 0;
    __syncthreads();
    for (int i = tid; i < total; i += BJ_THREADS) {
      uint32_t at = 0;
      const unsigned long long k = look(i, at);
      if (k > nth || (k != 0 && k == nth && at <= last)) {
        const int to = atomicAdd(&s_count, 1);
        key[to] = k;
        place[to] = at;
      }
    }
    __syncthreads();
    count = s_count;
  }
  const long long out = (long long)b * p.n;
  for (int i = tid; i < count; i += BJ_THREADS) {
    const unsigned long long k = key[i];
    const uint32_t at = place[i];
    int rank = 0;
    for (int j = 0; j < count; ++j) rank += key[j] > k || (key[j] == k && place[j] < at);
    if (rank < p.n) {
      p.out_scores[out + rank] = float(value_of(k));
      p.out_parents[out + rank] = int(at / uint32_t(p.V));
      p.out_tokens[out + rank] = int(at % uint32_t(p.V));
    }
  }
  for (int i = count + tid; i < p.n; i += BJ_THREADS) {
    p.out_scores[out + i] = -INFINITY;
    p.out_parents[out + i] = 0;
    p.out_tokens[out + i] = 0;
  }
}

// ---------------------------------------------------------------------------- reordering
// Beam w of a request continues beam parents[w]. A page that is full is history: every child refers to
// its parent's. In the column that is being filled all beams' pages differ: a parent's first child keeps
// the page, the i-th further child of the request takes the i-th dead beam's and the filled rows are copied
// there (a beam is dead when it has no child; there are as many of them as further children). Pages
// behind that column stay with their beams. What is read is a living beam's page, what is written a dead
// one's, so nothing has to be ordered.
constexpr int BR_THREADS = 256;

struct BeamReorderParams {
  PagePool K, V;
  long long k_layer, v_layer;
  int pages, page_log2, Hk, row_chunks, esize_log2, layers;
  const int* table;   // [B W][table_ld]
  int table_ld, cols;
  const int* lens;    // [B W]: alike in a request
  const int* parents; // [B][W]
  int* table_out;     // [B W][out_ld]
  int out_ld;
  int W, parts;       // blocks per request and layer
  int* err;
};

__global__ void __launch_bounds__(BR_THREADS) beam_reorder_kernel(const __grid_constant__ BeamReorderParams p) {
  __shared__ int s_parent[BS_MAX_W], s_heir[BS_MAX_W], s_page[BS_MAX_W], s_src[BS_MAX_W], s_dst[BS_MAX_W];
  const int tid = threadIdx.x, b = blockIdx.x, layer = blockIdx.y, part = blockIdx.z;
  pdl_wait();
  pdl_launch_dependents();
  const long long row0 = (long long)b * p.W;
  const int n = p.lens[row0], full = n >> p.page_log2, rest = n & ((1 << p.page_log2) - 1);
  int bad = 0;
  if (n < 0 || full > p.cols || (full == p.cols && rest)) bad |= kErrCapacity;
  if (tid < p.W) {
    const int parent = p.parents[row0 + tid];
    if (parent < 0 || parent >= p.W || p.lens[row0 + tid] != n) bad |= kErrTree;
    s_parent[tid] = parent;
    int page = -1;
    if (!bad && rest) {
      page = p.table[(row0 + tid) * p.table_ld + full];
      if (page < 0 || page >= p.pages) bad |= kErrPage;
    }
    s_page[tid] = page;
  }
  __syncthreads();
  bool further = false, dead = true;
  if (tid < p.W) {
    for (int w = 0; w < p.W; ++w) {
      further |= w < tid && s_parent[w] == s_parent[tid];
      dead &= s_parent[w] != tid;
      if (rest && w < tid && s_page[w] == s_page[tid]) bad |= kErrPage;  // a page that two beams would fill
    }
  }
  // numbers of further children and of dead beams up to each; both are few, in beam order
  __shared__ unsigned long long s_further, s_dead;
  if (tid == 0) s_further = s_dead = 0;
  __syncthreads();
  if (further) atomicOr(&s_further, 1ull << tid);
  if (tid < p.W && dead) atomicOr(&s_dead, 1ull << tid);
  const bool stop = __syncthreads_or(bad);
  if (bad) raise_error(p.err, bad);
  const int extra = __popcll(s_further);
  if (!stop && tid < p.W) {
    int heir = s_parent[tid];
    if (further) {
      const int i = __popcll(s_further & ((1ull << tid) - 1));
      unsigned long long d = s_dead;
      for (int k = 0; k < i; ++k) d &= d - 1;
      heir = __ffsll((long long)d) - 1;
      s_src[i] = s_page[s_parent[tid]];
      s_dst[i] = s_page[heir];
    }
    s_heir[tid] = heir;
  }
  __syncthreads();
  if (layer == 0) {
    for (int i = tid + part * BR_THREADS; i < p.W * p.cols; i += p.parts * BR_THREADS) {
      const int w = i / p.cols, c = i - w * p.cols;
      const int from = stop || c > full || (c == full && !rest) ? w : c < full ? s_parent[w] : s_heir[w];
      p.table_out[(row0 + w) * p.out_ld + c] = p.table[(row0 + from) * p.table_ld + c];
    }
  }
  if (stop || !rest) return;
  // 16-byte pieces: further child, K or V and head, row, piece of the row
  const int span = rest * p.row_chunks;
  const long long units = (long long)extra * 2 * p.Hk * span;
  const long long step = (long long)p.parts * BR_THREADS;
  for (long long u0 = (long long)part * BR_THREADS + tid; u0 < units; u0 += 4 * step) {
    uint4 x[4];
    char* to[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const long long u = u0 + k * step;
      to[k] = nullptr;
      if (u < units) {
        const int g = int(u / span), c = int(u - (long long)g * span);
        const int e = g / (2 * p.Hk), hv = g - e * 2 * p.Hk, head = hv >> 1;
        const PagePool& pool = (hv & 1) ? p.V : p.K;
        const int r = c / p.row_chunks, piece = c - r * p.row_chunks;
        char* base = static_cast<char*>(pool.ptr) +
                     ((((hv & 1) ? p.v_layer : p.k_layer) * layer + head * pool.head + r * pool.row) << p.esize_log2) +
                     piece * 16;
        x[k] = *reinterpret_cast<const uint4*>(base + ((s_src[e] * pool.page) << p.esize_log2));
        to[k] = base + ((s_dst[e] * pool.page) << p.esize_log2);
      }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (to[k]) *reinterpret_cast<uint4*>(to[k]) = x[k];
  }
}

}  // namespace wc
