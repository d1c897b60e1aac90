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
// Every logit is read once. A block has a piece of one beam's row, a few rounds of 32 values a thread; four
// blocks an SM, so that some load while others work. The first round gives a bound: the n-th of the threads'
// maxima, which n values at least reach; what reaches it, then and later, is collected, and the piece leaves
// at least its n best and its sum of exponentials. The second kernel, one block a request, has each beam's lse
// and does the same with the candidates' scores.
//
// Ranks are decided in 64 bits: two beams' scores may lie closer than a 32-bit sum resolves, as a score near -20
// has steps of 2^-19. The exponentials are of 32 bits, 2^(z c - R) with c, log2(e) in 32 bits, and an integer R, so that
// sums with other R are joined without a rounding. c is 1.34e-8 of itself too small, so lse = R / c + log sum, which
// shifts with the row and has that share of z's distance from R alone. With d, the mean distance of a row's terms
// from its maximum (at most log V), lse is off by less than 2^-24 (d + 1) for the exponents' rounding, 2^-26 d for c, 2^-22
// for ex2 and, at worst, 2^-21 a round for the additions: under 2^-18 up to five rounds a piece and V below 2^18.
//
// 64 x 8 beams over 151,936 fp32 logits: 68 us (two rounds a piece 75, five 68, seven 71, ten 74), 4.7 TB/s in the first kernel.
constexpr int BS_THREADS = 256;
constexpr int BS_PER = 32;                       // values a thread and round
constexpr int BS_ROUND = BS_THREADS * BS_PER;
constexpr int BS_LIST = 1024;
constexpr int BS_MAX_N = 64;
constexpr int BS_MAX_W = 64;
constexpr int BJ_THREADS = 512;
constexpr int BJ_LIST = 2048;
// Exponents are taken against integers: a logit times log2(e), rounded to 32 bits, then up. Up to 2^20 that leaves less
// than 1.1 above the exact product; from 2^31 on the rounding alone would make a sum infinite or 0. Logits
// below -2^21 / log2(e) are no maximum of a piece that is summed this way, and add 0 to it.
constexpr double kLog2eUsed = kLog2e;  // as the exponents have it
constexpr float BS_FLOOR = -0x1p21f, BS_FAR = 0x1p20f;

struct BeamSelectParams {
  const void* logits;
  long long request, beam;  // strides in elements
  const float* scores;      // [B][W]
  const uint8_t* finished;  // [B][W] or null
  int B, W, V, n, pieces, rounds, pad;
  // workspace
  double2* stat;            // [B W][pieces]: R and the sum of 2^(z c - R); sum 0: no token, not finite: no numbers
  unsigned long long* cand; // [B W][pieces][2 n]: argmax_key of value and token, in any order
  int* counts;              // [B W][pieces]
  float* out_scores;        // [B][n]
  int *out_parents, *out_tokens;
  int* err;
};

// What a beam proposes: 0 nothing (it is dead, or its score is no number), 1 its tokens, 2 itself (it has ended).
__device__ __forceinline__ int beam_kind(const BeamSelectParams& p, long long row) {
  const float score = p.scores[row];
  return !(score > -INFINITY && score < INFINITY) ? 0 : p.finished && p.finished[row] ? 2 : 1;
}

// A bound that the keys of n threads of a block reach, and of few more; 1 where fewer threads have a key (0: none).
// Halves the span between the lowest key and the highest.
template <int kThreads>
__device__ __forceinline__ uint32_t reached_by(uint32_t key, int n, uint32_t* s_low, uint32_t* s_high) {
  const uint32_t wl = __reduce_min_sync(0xffffffffu, key ? key : 0xffffffffu), wh = __reduce_max_sync(0xffffffffu, key);
  if (threadIdx.x % 32 == 0) {
    s_low[threadIdx.x / 32] = wl;
    s_high[threadIdx.x / 32] = wh;
  }
  if (__syncthreads_count(key != 0) < n) return 1;
  uint32_t low = s_low[0], high = s_high[0];
#pragma unroll
  for (int i = 1; i < kThreads / 32; ++i) {
    low = min(low, s_low[i]);
    high = max(high, s_high[i]);
  }
#pragma unroll 1
  while (high - low > 64) {  // keys 64 apart are as good as one: the bound stays at or below the n-th
    const uint32_t mid = low + (high - low) / 2 + 1;
    const int c = __syncthreads_count(key >= mid);
    if (c >= n) low = mid;
    else high = mid - 1;
    if (c >= n && c <= n + n / 4) break;
  }
  return low;
}

// 16 bytes of a row, four fp32 or eight bf16 values.
template <typename T>
struct Logits {
  static constexpr int N = 16 / sizeof(T);
  uint4 w;
  __device__ __forceinline__ float at(int k) const {
    const uint32_t x[4] = {w.x, w.y, w.z, w.w};
    if constexpr (N == 4) return __uint_as_float(x[k]);
    else return __uint_as_float(k & 1 ? x[k / 2] & 0xffff0000u : x[k / 2] << 16);
  }
  __device__ __forceinline__ void load(const T* row, int i) { w = ldg_stream(reinterpret_cast<const uint4*>(row + i)); }
  // Values from i on; -inf behind the row's end. A row that does not begin on a 16-byte boundary is read value by
  // value, so that its sum has the order of any other's: beams that are alike stay tied.
  __device__ __forceinline__ void load_edge(const T* row, bool whole, int i, int V) {
    if (whole && i + N <= V) {
      load(row, i);
    } else {
      uint32_t x[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if constexpr (N == 4) {
          x[k] = i + k < V ? __float_as_uint(row[i + k]) : 0xff800000u;
        } else {
          const uint32_t lo = i + 2 * k < V ? row[i + 2 * k] : 0xff80u, hi = i + 2 * k + 1 < V ? row[i + 2 * k + 1] : 0xff80u;
          x[k] = lo | (hi << 16);
        }
      }
      w = make_uint4(x[0], x[1], x[2], x[3]);
    }
  }
};

// Too many values at the bound (equal ones, values in few threads, values that rise behind the first round): the n best
// of a row's [first, end), the n-th found bit by bit. Reads the values again, 65 times, so that the way that is always
// taken does not keep them. 64 x 8 beams over 151,936 tokens where every piece comes here (all logits alike or rising; a
// hundred tokens in a run and the rest at a finite mask, while -inf is below every bound: 56 us): 2.7 ms, else 68 us.
template <typename T>
__device__ __noinline__ void beam_pieces_again(const T* z, int first, int end, float bound, int n, unsigned long long* list,
                                               uint32_t* s_sum, int* s_count) {
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  auto key = [&](int i) -> unsigned long long {
    float x;
    if constexpr (sizeof(T) == 4) x = z[i];
    else x = bf16_bits_to_f32(z[i]);
    return x >= bound ? argmax_key(x + 0.f, uint32_t(i)) : 0;
  };
  unsigned long long nth = 0;
#pragma unroll 1
  for (int bit = 63; bit >= 0; --bit) {
    const unsigned long long probe = nth | (1ull << bit);
    int c = 0;
    for (int i = first + tid; i < end; i += BS_THREADS) c += key(i) >= probe;
    c = __reduce_add_sync(0xffffffffu, c);
    __syncthreads();
    if (lane == 0) s_sum[warp] = c;
    __syncthreads();
    c = 0;
    for (int i = 0; i < BS_THREADS / 32; ++i) c += s_sum[i];
    if (c >= n) nth = probe;
  }
  __syncthreads();
  if (tid == 0) *s_count = 0;
  __syncthreads();
  for (int i = first + tid; i < end; i += BS_THREADS) {
    const unsigned long long k = key(i);
    if (k >= nth) list[atomicAdd(s_count, 1)] = k;  // n of them: keys differ
  }
  __syncthreads();
}

// A piece whose maximum lies far from 0 (a mask's value in every place, a type's lowest): its sum relative to the maximum
// itself, for thread 0.
template <typename T>
__device__ __noinline__ double beam_piece_extreme(const T* z, int first, int end, float m, double* s_sum) {
  double sum = 0;
  for (int i = first + int(threadIdx.x); i < end; i += BS_THREADS) {
    float x;
    if constexpr (sizeof(T) == 4) x = z[i];
    else x = bf16_bits_to_f32(z[i]);
    sum += ex2_approx((x - m) * kLog2e);
  }
  sum = warp_sum_d(sum);
  __syncthreads();
  if (threadIdx.x % 32 == 0) s_sum[threadIdx.x / 32] = sum;
  __syncthreads();
  sum = 0;
  for (int i = 0; i < BS_THREADS / 32; ++i) sum += s_sum[i];
  return sum;
}

template <typename T>
__global__ void __launch_bounds__(BS_THREADS, 4) beam_pieces_kernel(const __grid_constant__ BeamSelectParams p) {
  constexpr int N = 16 / sizeof(T), NV = BS_PER / N, WARPS = BS_THREADS / 32;
  __shared__ unsigned long long list[BS_LIST];
  __shared__ float s_max[WARPS], s_ref[WARPS];
  __shared__ double s_sum[WARPS];
  __shared__ uint32_t s_key[2 * WARPS];
  __shared__ int s_count;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int row = blockIdx.x / p.pieces, piece = blockIdx.x - row * p.pieces;
  const int b = row / p.W;
  const T* z = static_cast<const T*>(p.logits) + b * p.request + (row - b * p.W) * p.beam;
  if (tid == 0) s_count = 0;
  pdl_wait();
  pdl_launch_dependents();
  if (beam_kind(p, row) != 1) return;  // its logits do not matter
  const bool whole = (reinterpret_cast<unsigned long long>(z) & 15) == 0;
  const int first = piece * p.rounds * BS_ROUND, end = min(first + p.rounds * BS_ROUND, p.V);
  float best = -INFINITY, ref = BS_FLOOR, sum[4] = {0.f, 0.f, 0.f, 0.f}, bound = 0.f;
#pragma unroll 1
  for (int at = first; at < end; at += BS_ROUND) {
    Logits<T> x[NV];
    if (whole && at + BS_ROUND <= p.V) {
#pragma unroll
      for (int v = 0; v < NV; ++v) x[v].load(z, at + (v * BS_THREADS + tid) * N);
    } else {
#pragma unroll
      for (int v = 0; v < NV; ++v) x[v].load_edge(z, whole, at + (v * BS_THREADS + tid) * N, p.V);
    }
    float vtop[NV], top = -INFINITY;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      vtop[v] = fmaxf(x[v].at(0), x[v].at(1));
#pragma unroll
      for (int k = 2; k < N; ++k) vtop[v] = fmaxf(vtop[v], x[v].at(k));
      top = fmaxf(top, vtop[v]);
    }
    best = fmaxf(best, top);
    const float r = fmaxf(ref, ceilf(top * kLog2e));
    if (r > ref) {
      const float less = ex2_approx(ref - r);  // of integers: exact
#pragma unroll
      for (int k = 0; k < 4; ++k) sum[k] *= less;
      ref = r;
    }
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int k = 0; k < N; ++k) sum[k & 3] += ex2_approx(fmaf(x[v].at(k), kLog2e, -ref));
    if (at == first)  // n threads' maxima are at the bound or above; -inf is not
      bound = argmax_key_value((unsigned long long)(max(reached_by<BS_THREADS>(uint32_t(argmax_key(top + 0.f, 0) >> 32), p.n,
                                                                               s_key, s_key + WARPS), 0x00800000u)) << 32);
    if (top >= bound) {
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        if (vtop[v] >= bound) {
#pragma unroll
          for (int k = 0; k < N; ++k)
            if (x[v].at(k) >= bound) {
              const int to = atomicAdd(&s_count, 1);
              // -0 ranks with +0
              if (to < BS_LIST) list[to] = argmax_key(x[v].at(k) + 0.f, uint32_t(at + (v * BS_THREADS + tid) * N + k));
            }
        }
      }
    }  }
  {
    const float wref = warp_max(ref), wbest = warp_max(best);
    const double s = warp_sum_d(double((sum[0] + sum[1]) + (sum[2] + sum[3])) * double(ex2_approx(ref - wref)));
    if (lane == 0) {
      s_sum[warp] = s;
      s_ref[warp] = wref;
      s_max[warp] = wbest;
    }
  }
  __syncthreads();
  unsigned long long* out = p.cand + (long long)blockIdx.x * 2 * p.n;
  float m = s_max[0], R = s_ref[0];
#pragma unroll
  for (int i = 1; i < WARPS; ++i) {
    m = fmaxf(m, s_max[i]);
    R = fmaxf(R, s_ref[i]);
  }
  double total = 0, reference = R;
  if (fabsf(m) > BS_FAR && fabsf(m) < INFINITY) {
    total = beam_piece_extreme(z, first, end, m, s_sum);
    reference = double(m) * kLog2eUsed;  // exact, and so is the quotient
  } else if (tid == 0) {
    for (int i = 0; i < WARPS; ++i) total += s_sum[i] * double(ex2_approx(s_ref[i] - R));
  }
  if (tid == 0) {
    if (!(total < INFINITY)) raise_error(p.err, kErrLogits);
    p.stat[blockIdx.x] = make_double2(reference, total);
  }
  int count = s_count;
  if (count > BS_LIST) {
    beam_pieces_again(z, first, end, bound, p.n, list, s_key, &s_count);
    count = s_count;
  }
  if (tid == 0) p.counts[blockIdx.x] = count <= 2 * p.n ? count : p.n;
  if (count <= 2 * p.n) {  // as they are
    if (tid < count) out[tid] = list[tid];
    return;
  }
  for (int i0 = 0; i0 < count; i0 += BS_THREADS / 4) {  // the n best, four lanes a candidate
    const int i = i0 + tid / 4;
    const unsigned long long key = i < count ? list[i] : ~0ull;
    int rank = 0;
    for (int k = tid % 4; k < count; k += 4) rank += list[k] > key;
    rank += __shfl_xor_sync(0xffffffffu, rank, 1);
    rank += __shfl_xor_sync(0xffffffffu, rank, 2);
    if (i < count && rank < p.n && tid % 4 == 0) out[rank] = key;
  }
}

// A double's order as an unsigned number.
__device__ __forceinline__ unsigned long long order_of(double x) {
  const unsigned long long u = (unsigned long long)__double_as_longlong(x);
  return (u >> 63) ? ~u : u | (1ull << 63);
}
__device__ __forceinline__ double value_of(unsigned long long k) {
  return __longlong_as_double((long long)((k >> 63) ? k & ~(1ull << 63) : ~k));
}

// One block a request. Bound by latency: statistics, candidates, their ranks (64 requests of 32 lists: 8 us).
__global__ void __launch_bounds__(BJ_THREADS) beam_join_kernel(const __grid_constant__ BeamSelectParams p) {
  constexpr int WARPS = BJ_THREADS / 32;
  __shared__ unsigned long long key[BJ_LIST];
  __shared__ uint32_t place[BJ_LIST];       // beam * V + token
  __shared__ double s_score[BS_MAX_W], s_lse[BS_MAX_W];
  __shared__ int s_kind[BS_MAX_W];
  __shared__ int s_sum[WARPS];
  __shared__ int s_count;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, b = blockIdx.x;
  if (tid == 0) s_count = 0;
  pdl_wait();
  // Each beam's log of the sum of exponentials, 16 lanes a beam.
  for (int w0 = 0; w0 < p.W; w0 += BJ_THREADS / 16) {
    const int w = w0 + tid / 16, part = tid % 16;
    const long long row = (long long)b * p.W + min(w, p.W - 1);
    const double2* st = p.stat + row * p.pieces;
    const float score = p.scores[row];
    const int kind = beam_kind(p, row), n = kind == 1 ? p.pieces : 0;
    double m = -INFINITY, s = 0;
    for (int i = part; i < n; i += 16)
      if (st[i].y != 0) m = fmax(m, st[i].x);
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) m = fmax(m, __shfl_xor_sync(0xffffffffu, m, o));
    for (int i = part; i < n; i += 16) {
      const double2 y = st[i];
      if (y.y != 0) s += y.y * exp2(y.x - m);
    }
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (part == 0 && w < p.W) {
      if (!(score < INFINITY)) raise_error(p.err, kErrLogits);
      s_score[w] = score;
      // far from 0 the quotient has to be exact
      s_lse[w] = (fabs(m) > 2 * BS_FAR ? m / kLog2eUsed : m * (1 / kLog2eUsed)) + log(s);
      s_kind[w] = kind != 1 || (s > 0 && s < INFINITY) ? kind : 0;  // not without a token, nor where s is no number
    }
  }
  __syncthreads();
  // Candidates, eight of a thread at a time: score's order (0: none) and place. A list's places lie over 8, 16 or 32
  // threads, of longer lists 2 or 4 in a thread. A ninth is the beam itself where it has ended.
  constexpr int U = 8;
  const int slots = 2 * p.n, lists = p.W * p.pieces;
  const int wide = slots <= 8 ? 3 : slots <= 16 ? 4 : 5, more = slots <= 32 ? 0 : slots <= 64 ? 1 : 2;  // log2
  const int step = BJ_THREADS >> wide, units = ((lists + step - 1) / step) << more;
  const unsigned long long* cand = p.cand + (long long)b * lists * slots;
  const int* counts = p.counts + (long long)b * lists;
  unsigned long long k[U + 1];
  uint32_t at[U + 1];
  k[U] = at[U] = 0;
  if (tid < p.W && s_kind[tid] == 2) {
    k[U] = order_of(s_score[tid]);
    at[U] = uint32_t(tid) * uint32_t(p.V) + uint32_t(p.pad);
  }
  // list / pieces: the half keeps a quotient's border further away than rounding goes (beams x pieces < 2^18 + 64)
  const float each_piece = 1.f / float(p.pieces);
  auto fill = [&](int u0) {
    int w[U], held[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int list = ((u0 + u) >> more) * step + (tid >> wide);
      w[u] = min(int((float(list) + 0.5f) * each_piece), p.W - 1);
      held[u] = list < lists ? counts[list] : 0;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int list = ((u0 + u) >> more) * step + (tid >> wide);
      const int j = (tid & ((1 << wide) - 1)) + (((u0 + u) & ((1 << more) - 1)) << wide);
      k[u] = s_kind[w[u]] == 1 && j < held[u] ? cand[(long long)list * slots + j] : 0;
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (k[u]) {
        at[u] = uint32_t(w[u]) * uint32_t(p.V) + argmax_key_index(k[u]);
        k[u] = order_of(s_score[w[u]] + (double(argmax_key_value(k[u])) - s_lse[w[u]]));
      }
  };
  // f for every candidate; what fits in one fill is not fetched again
  bool filled = false;
  auto each = [&](auto f) {
    for (int u0 = 0; u0 < units; u0 += U) {
      if (!filled) fill(u0);
      filled = units <= U;
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (k[u]) f(k[u], at[u]);
    }
    if (k[U]) f(k[U], at[U]);
  };
  uint32_t top = 0;
  each([&](unsigned long long x, uint32_t) { top = max(top, uint32_t(x >> 32)); });
  __shared__ uint32_t s_low[WARPS], s_high[WARPS];
  const uint32_t least = reached_by<BJ_THREADS>(top, p.n, s_low, s_high);
  if (__any_sync(0xffffffffu, top >= least))
    each([&](unsigned long long x, uint32_t where) {
      if (uint32_t(x >> 32) >= least) {
        const int to = atomicAdd(&s_count, 1);
        if (to < BJ_LIST) {
          key[to] = x;
          place[to] = where;
        }
      }
    });
  __syncthreads();
  int count = s_count;
  if (count > BJ_LIST) {
    // Scores that are all but equal: the n-th best of (score, place), bit by bit.
    auto counted = [&](auto test) {
      int c = 0;
      each([&](unsigned long long x, uint32_t where) { c += test(x, where); });
      c = __reduce_add_sync(0xffffffffu, c);
      __syncthreads();
      if (lane == 0) s_sum[warp] = c;
      __syncthreads();
      c = 0;
      for (int i = 0; i < WARPS; ++i) c += s_sum[i];
      return c;
    };
    unsigned long long nth = 0;
#pragma unroll 1
    for (int bit = 63; bit >= 0; --bit) {
      const unsigned long long probe = nth | (1ull << bit);
      if (counted([&](unsigned long long x, uint32_t) { return x >= probe; }) >= p.n) nth = probe;
    }
    const int left = p.n - counted([&](unsigned long long x, uint32_t) { return x > nth; });
    uint32_t last = 0xffffffffu;  // the lowest place up to which `left` of the equal ones lie
#pragma unroll 1
    for (int bit = 31; bit >= 0; --bit) {
      const uint32_t probe = last & ~(1u << bit);
      if (counted([&](unsigned long long x, uint32_t where) { return x == nth && where <= probe; }) >= left) last = probe;
    }
    __syncthreads();
    if (tid == 0) s_count = 0;
    __syncthreads();
    each([&](unsigned long long x, uint32_t where) {
      if (x > nth || (x == nth && where <= last)) {
        const int to = atomicAdd(&s_count, 1);
        key[to] = x;
        place[to] = where;
      }
    });
    __syncthreads();
    count = s_count;
  }
  const long long out = (long long)b * p.n;
  // four lanes a candidate
  for (int i0 = 0; i0 < count; i0 += BJ_THREADS / 4) {
    const int i = i0 + tid / 4;
    const unsigned long long mine = i < count ? key[i] : ~0ull;
    const uint32_t where = i < count ? place[i] : 0;
    int rank = 0;
    for (int j = tid % 4; j < count; j += 4) {
      const unsigned long long y = key[j];
      rank += y > mine || (y == mine && place[j] < where);
    }
    rank += __shfl_xor_sync(0xffffffffu, rank, 1);
    rank += __shfl_xor_sync(0xffffffffu, rank, 2);
    if (i < count && rank < p.n && tid % 4 == 0) {
      p.out_scores[out + rank] = float(value_of(mine));
      p.out_parents[out + rank] = int(where / uint32_t(p.V));
      p.out_tokens[out + rank] = int(where % uint32_t(p.V));
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
constexpr int BR_PARTS = 4;  // blocks for a request and layer. 32 x 8 beams: 1 163 us, 2 154, 4 150, 8 150, 16 204; 1 x 4: 5.9, 4.7, 4.1, 4.2, 4.4

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
  // Copies of a page's filled rows of one head: further child, head, K or V. Their addresses are found 64 at a time,
  // so that a thread, whose place in the rows stays, has eight of them on their way for an addition each.
  __shared__ char *s_from[64], *s_to[64];
  const int span = rest * p.row_chunks, groups = extra * 2 * p.Hk;
  for (int g0 = part; g0 < groups; g0 += 64 * p.parts) {
    const int n = min(64, (groups - g0 + p.parts - 1) / p.parts);
    __syncthreads();
    if (tid < n) {
      const int g = g0 + tid * p.parts, e = g / (2 * p.Hk), hv = g - e * 2 * p.Hk, head = hv >> 1;
      const PagePool& pool = (hv & 1) ? p.V : p.K;
      char* base = static_cast<char*>(pool.ptr) + ((((hv & 1) ? p.v_layer : p.k_layer) * layer + head * pool.head) << p.esize_log2);
      s_from[tid] = base + ((s_src[e] * pool.page) << p.esize_log2);
      s_to[tid] = base + ((s_dst[e] * pool.page) << p.esize_log2);
    }
    __syncthreads();
    for (int c = tid; c < span; c += BR_THREADS) {
      const int r = c / p.row_chunks, piece = (c - r * p.row_chunks) * 16;
      const long long at_k = ((r * p.K.row) << p.esize_log2) + piece, at_v = ((r * p.V.row) << p.esize_log2) + piece;
      for (int i0 = 0; i0 < n; i0 += 8) {
        uint4 x[8];
#pragma unroll
        for (int u = 0; u < 8; ++u)
          if (i0 + u < n) x[u] = *reinterpret_cast<const uint4*>(s_from[i0 + u] + ((g0 + (i0 + u) * p.parts) & 1 ? at_v : at_k));
#pragma unroll
        for (int u = 0; u < 8; ++u)
          if (i0 + u < n) *reinterpret_cast<uint4*>(s_to[i0 + u] + ((g0 + (i0 + u) * p.parts) & 1 ? at_v : at_k)) = x[u];
      }
    }
  }
}

}  // namespace wc
