// Beam search: the choice of the next beams and the reordering of their cache.
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>

#include <tuple>

#include "common.cuh"
#include "launch.h"
#include "status.h"

namespace dsv3 {

namespace {

typedef __nv_bfloat16 bf16;

constexpr int kMaxBeams = 32;
constexpr int kPickThreads = 512;
constexpr int kListCap = 512;      // candidates at or above a CTA's threshold that it ranks in shared memory

// Order-preserving map of a float to an unsigned key (larger float, larger
// key); 0 stands for "no candidate" and lies below the key of -inf.
__device__ __forceinline__ uint32_t order_key(float x) {
  const uint32_t u = __float_as_uint(x);
  return u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) {
  return __uint_as_float(k ^ ((k >> 31) ? 0x80000000u : 0xffffffffu));
}
// (key, index) as one number: a larger one is the better candidate, that is the
// larger value, and of equal values the lower index.
__device__ __forceinline__ uint64_t entry_of(uint32_t key, uint32_t index) { return (uint64_t)key << 32 | ~index; }
__device__ __forceinline__ uint32_t entry_index(uint64_t e) { return ~(uint32_t)e; }

// A logit or score as the selection sees it: NaN counts as -inf, +inf (below) as the largest
// finite float, so that the log-sum-exp of a row is always defined; -0 becomes 0,
// whose key differs.
constexpr float kLargest = 3.402823466e38f;
constexpr uint32_t kLowestKey = 0x007fffffu;   // of -inf
__device__ __forceinline__ float number_of(float x) { return fmaxf(x, -INFINITY) + 0.f; }
__device__ __forceinline__ float number_of(bf16 x) { return number_of(__bfloat162float(x)); }

// Logits that differ by more than kTieWindow have different scores where
// 3 (max - logit) + |score| < kTieReach: a score is score + ((x - max) - log sum),
// three roundings of at most 2^-24 of their results, and log sum is at most 22 (V <
// 2^31), so that two scores differ by 2^-23 (3 (max - x) + 44 + |score|) less than
// their logits, at most.  Half of the window is kept for its own rounding.
constexpr float kTieWindow = 1.f / 2048, kTieReach = 2000.f;
__device__ __forceinline__ uint32_t below_window(uint32_t key) {
  return key <= kLowestKey ? key : order_key(key_value(key) - kTieWindow);
}

// e^x for x <= 0, flushed to zero where it would be denormal.
__device__ __forceinline__ float exp_of(float x) { return ex2_approx(x * 1.4426950408889634f); }

// A key that at least k of a CTA's candidates reach and few more do (22 of 8,192
// for k = 8 on random data): the k-th largest of the warps' maxima, or with fewer
// than k warps the smallest over the warps of their r-th largest lane maximum, r =
// ceil(k / warps).  `top` is the lane's largest key, 0 where it has none.  One
// barrier.
template <int THREADS>
__device__ __forceinline__ uint32_t cta_threshold(int k, uint32_t top) {
  constexpr int W = THREADS / 32;
  __shared__ uint32_t s_low[W];
  const int lane = threadIdx.x & 31;
  uint32_t left = top, low = 0;
  for (int i = 0; i < (k + W - 1) / W; ++i) {
    low = __reduce_max_sync(0xffffffffu, left);
    const unsigned who = __ballot_sync(0xffffffffu, left == low);
    if (lane == __ffs(who) - 1) left = 0;
  }
  if (lane == 0) s_low[threadIdx.x >> 5] = low;
  __syncthreads();
  const int me = lane & (W - 1);
  const uint32_t mine = s_low[me];
  if (k > W) return __reduce_min_sync(0xffffffffu, mine);
  int rank = 0;
#pragma unroll
  for (int w = 0; w < W; ++w) {
    const uint32_t other = __shfl_sync(0xffffffffu, mine, w);
    rank += other > mine || (other == mine && w < me);
  }
  return __shfl_sync(0xffffffffu, mine, __ffs(__ballot_sync(0xffffffffu, rank == k - 1)) - 1);
}

// The k best of the candidates whose key reaches `threshold`, ranked by counting
// in shared memory.  `each(least, f)` calls f(entry) for the thread's candidates
// whose key is `least` or more; `any` says whether it may have one.
// Where more reach the threshold than the list holds (many equal values) the best
// are taken one at a time.  put(rank, entry) is called once per rank; a rank
// without a candidate gets 0.  *s_n is 0 on entry, and the caller's barrier comes
// before the next use.
template <int THREADS, typename Each, typename Put>
__device__ __forceinline__ void cta_rank(int k, uint32_t threshold, bool any, int* s_n, Each each, Put put) {
  constexpr int W = THREADS / 32;
  __shared__ uint64_t s_list[kListCap];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (any)
    each(max(threshold, 1u), [&](uint64_t e) {
      const int at = atomicAdd(s_n, 1);
      if (at < kListCap) s_list[at] = e;
    });
  __syncthreads();
  const int n = *s_n;
  if (n <= kListCap) {
    for (int i = tid; i < n; i += THREADS) {
      const uint64_t e = s_list[i];
      int rank = 0;
#pragma unroll 4
      for (int j = 0; j < n; ++j) rank += s_list[j] > e;
      if (rank < k) put(rank, e);
    }
    for (int i = n + tid; i < k; i += THREADS) put(i, (uint64_t)0);
    return;
  }
  uint64_t last = ~(uint64_t)0;
  for (int r = 0; r < k; ++r) {
    uint64_t best = 0;
    each(1u, [&](uint64_t e) {
      if (e < last && e > best) best = e;
    });
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const uint64_t other = __shfl_xor_sync(0xffffffffu, best, o);
      if (other > best) best = other;
    }
    __syncthreads();                     // the last round's entries are read
    if (lane == 0) s_list[warp] = best;
    __syncthreads();
    for (int w = 0; w < W; ++w)
      if (s_list[w] > best) best = s_list[w];
    if (tid == 0) put(r, best);
    last = best;
  }
}

// A CTA walks `chunk` consecutive segments of PER * THREADS logits, rows one after
// another, and leaves one record per row that it touches: maximum, sum of
// exponentials, the K largest of its part and, of the logits left out, the largest
// that lies within kTieWindow of them.  Every thread keeps a running
// maximum and sum, the CTA a list of the K best so far; a segment that holds
// nothing above the last of them costs one barrier.  The logits of the next
// segment are on their way while this one is looked at.  A thread's elements go
// by their index in the row, never by its address, so that sums and scores are
// the same wherever a row lies.  32 x 8 rows of 102,400 fp32 take 34 us (16 at the
// copy rate): the ranking of a part's first segments bounds it, not the reads.
template <typename T, int THREADS, int PER, bool ALIGNED>
__global__ void __launch_bounds__(THREADS, 3) beam_scan_kernel(const T* __restrict__ logits, long ldb, long ldk,
                                                                            int units, int nseg, int chunk, int runs,
                                                                            int K, int V,
                                                                            const bool* __restrict__ finished,
                                                                            float2* __restrict__ stat,
                                                                            uint64_t* __restrict__ cand,
                                                                            uint32_t* __restrict__ left) {
  constexpr int VE = 16 / sizeof(T), NV = PER / VE, W = THREADS / 32;
  __shared__ float2 red[W];
  __shared__ uint64_t best[2][kMaxBeams + 1];
  __shared__ int s_n;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int u0 = blockIdx.x * chunk, u1 = min(u0 + chunk, units);
  uint4 raw[NV];                          // of the next segment, as loaded
  int row = u0 / nseg, seg = u0 % nseg;   // that segment
  const bool even = ldb == ldk * K;       // rows at one stride
  // Loads it: by 16 bytes, by 4 bytes where rows are not all ALIGNED, and what a
  // row does not fill, or a row at an odd address, element by element.  False where
  // the row is finished.
  auto fetch = [&]() {
    if (finished != nullptr && finished[row]) return false;
    const T* x = logits + (even ? row * ldk : (row / K) * ldb + (row % K) * ldk);
    const int first = seg * PER * THREADS + tid * VE;
    if ((seg + 1) * PER * THREADS <= V && (ALIGNED || (reinterpret_cast<uintptr_t>(x) & 3) == 0)) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const T* p = x + first + j * THREADS * VE;
        if constexpr (ALIGNED) {
          raw[j] = __ldg(reinterpret_cast<const uint4*>(p));
        } else {
          const uint32_t* q = reinterpret_cast<const uint32_t*>(p);
          raw[j] = make_uint4(__ldg(q), __ldg(q + 1), __ldg(q + 2), __ldg(q + 3));
        }
      }
    } else {
      const T low = (T)-INFINITY;
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        T* e = reinterpret_cast<T*>(&raw[j]);
#pragma unroll
        for (int i = 0; i < VE; ++i) {
          const int at = first + j * THREADS * VE + i;
          e[i] = at < V ? x[at] : low;
        }
      }
    }
    return true;
  };
  bool next_live = u0 < u1 && fetch();
  float m = -kLargest, s = 0.f;
  uint32_t floor = 1;                     // key that later logits have to reach
  int cur = 0;
  for (int u = u0; u < u1; ++u) {
    const bool live = next_live, begin = u == u0 || seg == 0, end = u + 1 == u1 || seg == nseg - 1;
    const int first = seg * PER * THREADS + tid * VE, this_row = row;
    float v[PER];
    if (live) {
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int i = 0; i < VE; ++i) v[j * VE + i] = number_of(reinterpret_cast<const T*>(&raw[j])[i]);
    }
    if (u + 1 < u1) {
      if (++seg == nseg) {
        seg = 0;
        ++row;
      }
      next_live = fetch();
    }
    if (!live) continue;
    float top = v[0];
#pragma unroll
    for (int i = 1; i < PER; ++i) top = fmaxf(top, v[i]);
    if (top > kLargest) {
#pragma unroll
      for (int i = 0; i < PER; ++i) v[i] = fminf(v[i], kLargest);
      top = kLargest;
    }
    if (begin) {
      m = -kLargest;
      s = 0.f;
    }
    const float now = fmaxf(m, top);
    s *= exp_of(m - now);
#pragma unroll
    for (int i = 0; i < PER; ++i) s += exp_of(v[i] - now);
    m = now;
    const uint32_t key = first < V ? order_key(top) : 0u;
    if (tid == 0) s_n = 0;
    const uint32_t threshold = begin ? below_window(cta_threshold<THREADS>(K, key)) : floor;
    const bool any = key >= threshold && key > 0;
    if (begin || __syncthreads_or(any)) {
      cta_rank<THREADS>(
          K + 1, threshold, any || (!begin && tid <= K), &s_n,
          [&](uint32_t least, auto&& f) {
            const float low = key_value(least);          // (a NaN for keys below that of -inf)
#pragma unroll
            for (int i = 0; i < PER; ++i)
              if (!(v[i] < low)) {
                const int at = first + (i / VE) * THREADS * VE + i % VE;
                const uint32_t k = order_key(v[i]);
                if (at < V && k >= least) f(entry_of(k, (uint32_t)at));
              }
            if (!begin && tid <= K && best[cur][tid] != 0) f(best[cur][tid]);
          },
          [&](int rank, uint64_t e) { best[cur ^ 1][rank] = e; });
      __syncthreads();
      cur ^= 1;
      // Later indices lose ties of equal logits, but logits in the window below the
      // K-th best are ranked too, so that the one after it is known; where that one
      // equals it already (masked rows) nothing is left to know.
      const uint32_t last = (uint32_t)(best[cur][K - 1] >> 32), next = (uint32_t)(best[cur][K] >> 32);
      floor = last == next ? last + 1 : below_window(last);
    }
    if (end) {
      const float wm = warp_max(m);
      const float ws = warp_sum(s * exp_of(m - wm));
      if (lane == 0) red[warp] = make_float2(wm, ws);
      __syncthreads();
      const size_t at = (size_t)this_row * runs + (blockIdx.x - this_row * nseg / chunk);
      if (tid < K) cand[at * K + tid] = best[cur][tid];
      if (tid == K) left[at] = (uint32_t)(best[cur][K] >> 32);
      if (warp == W - 1) {
        const float2 r = lane < W ? red[lane] : make_float2(-kLargest, 0.f);
        const float M = warp_max(r.x);
        const float sum = warp_sum(r.y * exp_of(r.x - M));
        if (lane == 0) stat[at] = make_float2(M, sum);
      }
    }
  }
}

// The logits again, for the rare case below.
struct BeamLogits {
  const void* at;
  long ldb, ldk;
  bool narrow;                // bf16
  __device__ __forceinline__ float operator()(int b, int r, int v) const {
    const long i = b * ldb + r * ldk + v;
    const float x = narrow ? number_of(static_cast<const bf16*>(at)[i]) : number_of(static_cast<const float*>(at)[i]);
    return fminf(x, kLargest);
  }
};

// One CTA per batch entry: log-sum-exp of its beams, then the K best candidates.
//
// A row's part keeps its K largest logits, and a score is a rounded and so not
// strictly growing function of the logit: a candidate that a part left out cannot
// beat the K-th best score, but it can equal it at a lower index.  Where the parts'
// records do not rule that out, and only there, the entry's rows are read again for
// the candidates that score exactly the K-th best.
__global__ void __launch_bounds__(kPickThreads) beam_pick_kernel(BeamLogits logits, const float2* __restrict__ stat,
                                                                 const uint64_t* __restrict__ cand,
                                                                 const uint32_t* __restrict__ left,
                                                                 const float* __restrict__ scores,
                                                                 const bool* __restrict__ finished, int K, int V,
                                                                 int nseg, int chunk, int runs, int eos,
                                                                 float* __restrict__ o_score,
                                                                 int* __restrict__ o_parent, int* __restrict__ o_token,
                                                                 bool* __restrict__ o_done) {
  const int b = blockIdx.x, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  __shared__ float s_max[kMaxBeams], s_log[kMaxBeams], s_score[kMaxBeams];
  __shared__ bool s_done[kMaxBeams];
  __shared__ int s_runs[kMaxBeams], s_n;
  __shared__ float s_val[kMaxBeams];      // the scores chosen
  __shared__ int s_ties[kPickThreads / 32];
  const size_t row0 = (size_t)b * K;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  for (int r = warp; r < K; r += kPickThreads / 32) {
    const bool done = finished != nullptr && finished[row0 + r];
    const float2* st = stat + (row0 + r) * runs;
    const int row = (int)row0 + r, n = ((row + 1) * nseg - 1) / chunk - row * nseg / chunk + 1;   // parts of the row
    float m = -kLargest, s = 0.f;
    if (!done) {
      for (int i = lane; i < n; i += 32) m = fmaxf(m, st[i].x);
      m = warp_max(m);
      for (int i = lane; i < n; i += 32) s += st[i].y * expf(st[i].x - m);
      s = warp_sum(s);
    }
    if (lane == 0) {
      s_max[r] = m;
      s_log[r] = logf(s);
      s_score[r] = fminf(number_of(scores[row0 + r]), kLargest);
      s_done[r] = done;
      s_runs[r] = n;
    }
  }
  if (tid == 0) s_n = 0;
  __syncthreads();
  const int per = runs * K;               // candidates per beam, at most
  // score of a logit, and whether a beam has such candidates (the others: -inf)
  auto score_of = [&](int r, float x) { return s_score[r] + ((x - s_max[r]) - s_log[r]); };
  auto live = [&](int r) { return !s_done[r] && s_score[r] > -INFINITY && s_log[r] > -INFINITY; };
  // smallest logit that part c % runs of beam c / runs kept, 0 if it kept all
  auto least_kept = [&](int c) -> uint32_t {
    const int r = c / runs;
    return c < K * runs && live(r) && c % runs < s_runs[r] ? cand[row0 * per + (size_t)c * K + K - 1] >> 32 : 0;
  };
  const uint32_t least0 = least_kept(tid);       // (on its way while the candidates are ranked)
  auto candidate = [&](int c) -> uint64_t {
    const int r = c / per, i = c % per;
    const float sc = s_score[r];
    uint32_t v;
    float val = -INFINITY;
    if (s_done[r]) {                      // the end token at the unchanged score, others at -inf
      if (i >= K) return 0;
      v = i == 0 ? eos : (i - 1 < eos ? i - 1 : i);
      if (i == 0) val = sc;
    } else if (!live(r)) {
      if (i >= K) return 0;
      v = i;
    } else {
      if (i >= s_runs[r] * K) return 0;
      const uint64_t e = cand[row0 * per + c];
      if (e == 0) return 0;
      v = entry_index(e);
      val = score_of(r, key_value((uint32_t)(e >> 32)));
    }
    return v < (uint32_t)V ? entry_of(order_key(val), r * V + v) : 0;
  };
  auto choose = [&](int rank, float val, int r, int v) {
    o_score[row0 + rank] = val;
    o_parent[row0 + rank] = r;
    o_token[row0 + rank] = v;
    o_done[row0 + rank] = s_done[r] || v == eos;
  };
  uint32_t top = 0;
  for (int c = tid; c < K * per; c += kPickThreads) top = max(top, (uint32_t)(candidate(c) >> 32));
  const uint32_t threshold = cta_threshold<kPickThreads>(K, top);
  cta_rank<kPickThreads>(
      K, threshold, top >= threshold && top > 0, &s_n,
      [&](uint32_t least, auto&& f) {
        for (int c = tid; c < K * per; c += kPickThreads) {
          const uint64_t e = candidate(c);
          if (e >> 32 >= least) f(e);
        }
      },
      [&](int rank, uint64_t e) {
        const uint32_t at = entry_index(e);
        s_val[rank] = key_value((uint32_t)(e >> 32));
        choose(rank, s_val[rank], at / V, at % V);
      });
  __syncthreads();
  const float cut = s_val[K - 1];
  bool tie = false;
  for (int c = tid; c < K * runs; c += kPickThreads) {
    const int r = c / runs;
    const uint32_t least = c == tid ? least0 : least_kept(c);
    const float x = key_value(least);
    if (least == 0 || score_of(r, x) != cut) continue;
    if (x > -INFINITY && !(3.f * (s_max[r] - x) + fabsf(s_score[r]) < kTieReach)) {
      tie = true;
      continue;
    }
    const uint32_t out = left[row0 * runs + c];
    if (out == least) {
      // equal logits at higher indices are left out, which does no harm unless a
      // smaller logit may score the same, or a larger one, perhaps behind them, does
      const uint32_t step = logits.narrow ? 0x10000u : 1u;     // to the next value of the logits' type
      const uint64_t* list = cand + row0 * per + (size_t)c * K;
      int j = K - 2;
      while (j >= 0 && (uint32_t)(list[j] >> 32) == least) --j;
      tie |= (x > -INFINITY && score_of(r, key_value(least - step)) == cut) ||
             (j >= 0 && score_of(r, key_value((uint32_t)(list[j] >> 32))) == cut);
    } else if (out != 0) {
      tie |= score_of(r, key_value(out)) == cut;
    }
  }
  if (!__syncthreads_or(tie)) return;
  // the scores above the cut stand; behind them, the lowest indices that score it
  int n = 0;
  while (s_val[n] > cut) ++n;
  constexpr int PER = 8;                  // consecutive tokens of a thread
  for (int r = 0; r < K && n < K; ++r) {
    const bool alive = live(r);
    if (alive && score_of(r, s_max[r]) < cut) continue;
    if (!alive && cut > -INFINITY) {      // at most the end token of a finished beam
      if (s_done[r] && s_score[r] == cut) {
        if (tid == 0) choose(n, cut, r, eos);
        ++n;
      }
      continue;
    }
    for (int v0 = 0; v0 < V && n < K; v0 += PER * kPickThreads) {
      const int first = v0 + tid * PER;
      unsigned hit = 0;
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const int v = first + i;
        if (v < V) {
          const float val = alive ? score_of(r, logits(b, r, v)) : s_done[r] && v == eos ? s_score[r] : -INFINITY;
          hit |= (unsigned)(val == cut) << i;
        }
      }
      if (!__syncthreads_or(hit)) continue;
      int upto = __popc(hit);
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += x;
      }
      if (lane == 31) s_ties[warp] = upto;
      __syncthreads();
      int rank = n + upto - __popc(hit);
      for (int w = 0; w < kPickThreads / 32; ++w) {
        if (w < warp) rank += s_ties[w];
        n += s_ties[w];
      }
      for (; hit != 0 && rank < K; hit &= hit - 1) choose(rank++, cut, r, first + __ffs(hit) - 1);
      __syncthreads();                    // the counts are read
    }
  }
}

// Grid (x, layer, group).  CTA x < parts * splits copies 16 KB of the page that
// is being filled, for every splits-th copy of its group; the last x (layer 0
// only) writes the group's new table rows.  Bound by the copied bytes.
constexpr int kCopyThreads = 256, kCopyVecs = 4;

__global__ void __launch_bounds__(kCopyThreads) beam_reorder_kernel(uint4* __restrict__ pages, long ld_layer, long ld_page,
                                                                    int row16, int page, int pool,
                                                                    const int* __restrict__ table, long ldt, int cols,
                                                                    const int* __restrict__ parents, int K,
                                                                    const int* __restrict__ lens, int* __restrict__ out,
                                                                    int parts, int splits, unsigned int* status) {
  __shared__ int s_src[kMaxBeams], s_dst[kMaxBeams], s_par[kMaxBeams], s_cur[kMaxBeams], s_spare[kMaxBeams], s_n;
  const int b = blockIdx.z, layer = blockIdx.y;
  const bool writes_table = (int)blockIdx.x == parts * splits;
  if (writes_table && layer > 0) return;
  // a length outside the table is reported; a negative one counts as zero
  const int given = lens[b], len = max(given, 0);
  if (writes_table && threadIdx.x == 0 && (given < 0 || given > (long)cols * page))
    record_error(status, DSV3_ERR_BOUNDS);
  const int col = len / page, rem = len % page;
  const int part = blockIdx.x % parts, split = blockIdx.x / parts;
  const int n16 = rem * row16;
  const int first = part * kCopyThreads * kCopyVecs + threadIdx.x;
  if (!writes_table && part * kCopyThreads * kCopyVecs >= n16) return;
  const int* tb = table + (size_t)b * K * ldt;
  if (threadIdx.x < 32) {
    const int lane = threadIdx.x;
    const bool beam = lane < K;
    int p = beam ? parents[b * K + lane] : -1;
    const int cur = beam && col < cols ? tb[lane * ldt + col] : -1;
    const bool bad_parent = beam && (p < 0 || p >= K);
    const bool bad_page = beam && rem > 0 && (cur < 0 || cur >= pool);
    if (bad_parent) p = lane;
    if (bad_parent || bad_page) record_error(status, DSV3_ERR_BOUNDS);
    // the first child of a parent keeps its page, the j-th of the further
    // children takes that of the j-th beam without a child
    const unsigned below = (1u << lane) - 1;
    const unsigned alike = __match_any_sync(0xffffffffu, p);     // all lanes take part
    const bool again = beam && (alike & below) != 0;
    const unsigned has = __reduce_or_sync(0xffffffffu, beam ? 1u << p : 0u);
    const bool dead = beam && !(has >> lane & 1);
    const unsigned agains = __ballot_sync(0xffffffffu, again), deads = __ballot_sync(0xffffffffu, dead);
    const bool ok = !__any_sync(0xffffffffu, bad_page);
    s_cur[lane] = cur;
    if (dead) s_spare[__popc(deads & below)] = cur;
    __syncwarp();
    const int j = __popc(agains & below);
    if (beam) {
      const int src = s_cur[p], dst = again ? s_spare[j] : src;
      s_par[lane] = p;
      s_dst[lane] = dst;                  // by child, for the table
      if (again) s_src[j] = src;
    }
    __syncwarp();
    if (!writes_table) {
      const int dst = s_dst[lane];
      __syncwarp();
      if (again) s_dst[j] = dst;          // by copy
      if (lane == 0) s_n = ok ? __popc(agains) : 0;
    }
  }
  __syncthreads();
  if (writes_table) {
    int* ob = out + (size_t)b * K * cols;
    for (int i = threadIdx.x; i < K * cols; i += kCopyThreads) {
      const int r = i / cols, c = i % cols;
      ob[i] = c < col ? tb[s_par[r] * ldt + c] : c == col && rem > 0 ? s_dst[r] : tb[r * ldt + c];
    }
    return;
  }
  for (int d = split; d < s_n; d += splits) {
    const uint4* src = pages + layer * ld_layer + s_src[d] * ld_page;
    uint4* dst = pages + layer * ld_layer + s_dst[d] * ld_page;
    uint4 v[kCopyVecs];
#pragma unroll
    for (int u = 0; u < kCopyVecs; ++u)
      if (first + u * kCopyThreads < n16) v[u] = src[first + u * kCopyThreads];
#pragma unroll
    for (int u = 0; u < kCopyVecs; ++u)
      if (first + u * kCopyThreads < n16) dst[first + u * kCopyThreads] = v[u];
  }
}

}  // namespace

std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor> beam_select(const at::Tensor& logits,
                                                                       const at::Tensor& scores,
                                                                       const c10::optional<at::Tensor>& finished,
                                                                       int64_t eos) {
  const char* op = "beam_select";
  TORCH_CHECK(logits.is_cuda() && logits.dim() == 3 && logits.stride(2) == 1 &&
                  (logits.scalar_type() == at::kFloat || logits.scalar_type() == at::kBFloat16),
              op, ": logits must be a CUDA bf16 or fp32 tensor [B, K, V] with unit stride in the last dimension");
  const int64_t B = logits.size(0), K = logits.size(1), V = logits.size(2);
  // (the last segment of a row counts up to 4,095 past V in 32 bits)
  TORCH_CHECK(K >= 1 && K <= kMaxBeams && V >= K && K * V < (1ll << 31) - 4096, op,
              ": 1 to 32 beams, at least as many tokens as beams and K * V below 2^31 - 4096");
  TORCH_CHECK(scores.scalar_type() == at::kFloat && scores.is_contiguous() && scores.dim() == 2 &&
                  scores.size(0) == B && scores.size(1) == K && scores.device() == logits.device(),
              op, ": scores must be a contiguous fp32 tensor [B, K]");
  const bool* done = nullptr;
  if (finished) {
    TORCH_CHECK(finished->scalar_type() == at::kBool && finished->is_contiguous() && finished->dim() == 2 &&
                    finished->size(0) == B && finished->size(1) == K && finished->device() == logits.device(),
                op, ": finished must be a contiguous bool tensor [B, K]");
    TORCH_CHECK(eos >= 0 && eos < V, op, ": finished beams need an end token inside the vocabulary");
    done = finished->data_ptr<bool>();
  }
  TORCH_CHECK(B * K * ((V + 2047) / 2048) < (1ll << 31), op, ": too many rows");
  const at::cuda::CUDAGuard guard(logits.device());
  auto st = at::cuda::getCurrentCUDAStream();
  // (straight to the allocator: five tensors through the dispatcher cost more
  // host time than the two launches)
  auto make = [&](at::IntArrayRef sizes, at::ScalarType t) {
    return at::Tensor(at::detail::empty_cuda(sizes, t, logits.device(), c10::nullopt));
  };
  auto o_score = make({B, K}, at::kFloat), o_parent = make({B, K}, at::kInt), o_token = make({B, K}, at::kInt),
       o_done = make({B, K}, at::kBool);
  if (B == 0) return {o_score, o_parent, o_token, o_done};
  // segments of 4,096 logits where that gives three CTAs per SM, else of 2,048: with
  // few rows the latency of a segment counts, not its overhead
  const int64_t sms = at::cuda::getCurrentDeviceProperties()->multiProcessorCount, es = logits.element_size();
  const int span = B * K * ((V + 4095) / 4096) >= 3 * sms ? 4096 : 2048;
  const int nseg = (int)((V + span - 1) / span);
  const bool aligned = reinterpret_cast<uintptr_t>(logits.data_ptr()) % 16 == 0 && logits.stride(0) * es % 16 == 0 &&
                       logits.stride(1) * es % 16 == 0;
  const int64_t units = B * K * nseg, ctas = sms * 3;
  const int chunk = (int)((units + ctas - 1) / ctas), runs = (nseg - 1) / chunk + 2;   // parts of a row, at most
  auto work = make({B * K * runs * (3 + 2 * K)}, at::kFloat);
  float2* stat = reinterpret_cast<float2*>(work.data_ptr());
  uint64_t* cand = reinterpret_cast<uint64_t*>(stat + B * K * runs);
  uint32_t* left = reinterpret_cast<uint32_t*>(cand + B * K * runs * K);
#define DSV3_SCAN(T_, PER_, ALIGNED_)                                                                          \
  beam_scan_kernel<T_, 256, PER_, ALIGNED_><<<(unsigned)((units + chunk - 1) / chunk), 256, 0, st>>>(          \
      reinterpret_cast<const T_*>(logits.data_ptr()), logits.stride(0), logits.stride(1), (int)units, nseg, chunk, \
      runs, (int)K, (int)V, done, stat, cand, left)
#define DSV3_SCAN_TYPE(T_)                              \
  do {                                                  \
    if (span == 4096 && aligned) DSV3_SCAN(T_, 16, true); \
    else if (span == 4096) DSV3_SCAN(T_, 16, false);    \
    else if (aligned) DSV3_SCAN(T_, 8, true);           \
    else DSV3_SCAN(T_, 8, false);                       \
  } while (0)
  if (logits.scalar_type() == at::kFloat) DSV3_SCAN_TYPE(float);
  else DSV3_SCAN_TYPE(bf16);
#undef DSV3_SCAN_TYPE
#undef DSV3_SCAN
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  const BeamLogits again{logits.data_ptr(), (long)logits.stride(0), (long)logits.stride(1),
                         logits.scalar_type() == at::kBFloat16};
  C10_CUDA_CHECK(launch_dependent(beam_pick_kernel, dim3((unsigned)B), kPickThreads, st, again, (const float2*)stat,
                                  (const uint64_t*)cand, (const uint32_t*)left,
                                  (const float*)scores.data_ptr<float>(), done, (int)K, (int)V, nseg, chunk, runs,
                                  eos >= 0 && eos < V ? (int)eos : -1, o_score.data_ptr<float>(),
                                  o_parent.data_ptr<int>(), o_token.data_ptr<int>(), o_done.data_ptr<bool>()));
  return {o_score, o_parent, o_token, o_done};
}

at::Tensor beam_reorder(at::Tensor& pages, const at::Tensor& table, const at::Tensor& parents,
                        const at::Tensor& lens) {
  const char* op = "beam_reorder";
  TORCH_CHECK(pages.is_cuda() && pages.dim() == 4 &&
                  (pages.numel() == 0 || (pages.stride(3) == 1 && pages.stride(2) == pages.size(3))), op,
              ": pages must be a CUDA tensor [layers, pool, page, width] with contiguous pages");
  const int64_t es = pages.element_size(), width = pages.size(3), page = pages.size(2);
  TORCH_CHECK(pages.numel() == 0 ||
                  (width * es % 16 == 0 && pages.stride(0) * es % 16 == 0 && pages.stride(1) * es % 16 == 0 &&
                   reinterpret_cast<uintptr_t>(pages.data_ptr()) % 16 == 0),
              op, ": page rows must be 16-byte aligned");
  TORCH_CHECK(parents.dim() == 2 && parents.scalar_type() == at::kInt && parents.is_contiguous() &&
                  parents.device() == pages.device(),
              op, ": parents must be a contiguous int32 tensor [B, K]");
  const int64_t B = parents.size(0), K = parents.size(1);
  TORCH_CHECK(K >= 1 && K <= kMaxBeams, op, ": 1 to 32 beams");
  TORCH_CHECK(table.dim() == 2 && table.scalar_type() == at::kInt && table.stride(1) == 1 && table.size(0) == B * K &&
                  table.device() == pages.device(),
              op, ": block_table must be int32 [B * K, columns] with unit stride in the last dimension");
  TORCH_CHECK(lens.dim() == 1 && lens.scalar_type() == at::kInt && lens.is_contiguous() && lens.size(0) == B &&
                  lens.device() == pages.device(),
              op, ": seq_lens must be a contiguous int32 tensor [B]");
  TORCH_CHECK(page >= 1, op, ": an empty page");
  TORCH_CHECK(B <= 65535 && pages.size(0) <= 65535 && pages.size(1) < (1ll << 31), op, ": too many groups or layers");
  const at::cuda::CUDAGuard guard(pages.device());
  auto out = at::Tensor(at::detail::empty_cuda({B * K, table.size(1)}, at::kInt, pages.device(), c10::nullopt));
  if (B == 0 || table.size(1) == 0) return out;
  const int row16 = (int)(width * es / 16);
  const int64_t layers = pages.numel() == 0 ? 0 : pages.size(0);
  const int64_t vecs = page * row16, per = kCopyThreads * kCopyVecs;
  const int parts = (int)std::max<int64_t>(1, (vecs + per - 1) / per);
  // about K / e copies per group when parents are random; none without layers, where
  // the one CTA of a group writes its table
  const int splits = layers == 0 ? 0 : (int)std::max<int64_t>(1, K / 2);
  const dim3 grid(parts * splits + 1, (unsigned)std::max<int64_t>(1, layers), (unsigned)B);
  beam_reorder_kernel<<<grid, kCopyThreads, 0, at::cuda::getCurrentCUDAStream()>>>(
      reinterpret_cast<uint4*>(pages.data_ptr()), pages.stride(0) * es / 16, pages.stride(1) * es / 16, row16,
      (int)page, (int)pages.size(1), table.data_ptr<int>(), table.stride(0), (int)table.size(1),
      parents.data_ptr<int>(), (int)K, lens.data_ptr<int>(), out.data_ptr<int>(), parts, splits, status_ptr());
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  return out;
}

void register_beam(pybind11::module_& m) {
  m.def("beam_select", &beam_select, "next beams over (beam, token) candidates", pybind11::arg("logits"),
        pybind11::arg("scores"), pybind11::arg("finished") = pybind11::none(), pybind11::arg("eos") = -1);
  m.def("beam_reorder", &beam_reorder, "block tables of the chosen beams and the copy of their unfinished page");
}

}  // namespace dsv3
