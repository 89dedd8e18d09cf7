// tcgen05 attention of a ragged batch over a paged latent cache (sm_100a).
// Included by paged.cu inside its anonymous namespace, after Ragged.
//
// The rows of sequence b are its (token, head) pairs, n_b * H of them, cut
// into row tiles of N; a key tile is 128 cached rows.  Both products are
// computed transposed, so that the cached rows are the 128-wide M side of the
// first and the latent columns the M side of the second, and one copy of a key
// tile in shared memory serves both:
//
//   S^T [128 keys x N rows] = K [128 x D] . Q^T                 (K-major A)
//   P^T = 2^(scale log2(e) S^T - m)                             (bf16, [key][row])
//   O^T [R x N rows]       += V^T [R x 128 keys] . P^T          (the same K, read MN-major)
//
// The cache row [latent | rotated key] is read as 64-column chunks [128 x 64]
// with a 128-byte swizzle; chunk pairs 0 .. LP-1 cover the latent (LP =
// ceil(R / 128)), and where D reaches past them one more tail chunk holds the
// rest of the rotated key.  Columns past D are zero-filled by TMA, rows past
// the cached length are masked in S and zeroed in shared memory before the
// second product (pages are never assumed to be initialised past that).
//
// A softmax thread owns one key and N / 2 of the rows: there is no per-row
// maximum over keys at hand, and none is needed.  Each row keeps a reference m
// that any score may exceed by up to 2^8 without harm (sums and O are fp32, P
// has the same relative precision at any scale); the 128 threads of a column
// half vote per tile, and only when one exceeds it are the column maxima
// computed, m moved and O^T rescaled.  Row sums are kept per thread and added
// up once per item, over the bf16-rounded P that the second product uses, so
// that a row's weights sum to one exactly.
//
// Work: all (sequence, row tile, key tile) triples in one order, cut into equal
// shares, one per CTA (one persistent CTA per SM).  Every CTA derives its share
// from the lengths on the device: the number of key tiles of a sequence's
// first n row tiles has a closed form (floor_sum).  A row tile that lies in one
// share is written out at once; one that is cut writes (m, sum, O) partials,
// which a second kernel merges in share order, so results do not depend on
// timing.
//
// Warps: 0 TMA, 1 MMA (and TMEM), 2..9 softmax and epilogue.  Every wait is
// bounded; after one ran out the softmax warps go on without waiting, so that
// they meet at their barriers, and the others stop.

constexpr int kPaThreads = 320;
constexpr int kPaChunk = 128 * 128;          // [128 keys x 64 columns] bf16, bytes
constexpr int kPaPair = 2 * kPaChunk;
constexpr int kPaMaxSlots = 8;
constexpr float kPaUnset = -1e30f;           // reference of a row that has seen no key

struct PagedPlan {
  int N, LP, nch, tail;       // row tile, latent chunk pairs, chunks, 1 if there is a tail chunk
  int slots, tails;           // ring slots (pairs), tail slots
  int alias;                  // P shares the (single) tail slot
  int look;                   // S of the next tile is issued before PV of this one
  int off_q, off_p, off_t, off_misc, smem, tmem_cols;
};

// Shared memory of a plan: ring | tail slots | P | Q | misc, with as many ring
// slots as fit.  P needs its own buffer unless even one whole key tile would
// not fit next to it; then it takes the tail slot, which S has read by the time
// P is written.
inline bool paged_plan(int N, int R, int D, PagedPlan& p) {
  p.N = N;
  p.LP = (R + 127) / 128;
  p.nch = (D + 63) / 64;
  p.tail = D > 128 * p.LP ? 1 : 0;
  const int limit = 232448;
  const int q = p.nch * N * 128, P = (N + 63) / 64 * kPaChunk, misc = 8 * N + 1024 + 512;
  for (int mode = 0; mode < 3; ++mode) {     // two tail slots, one, one shared with P
    p.tails = p.tail ? (mode == 0 ? 2 : 1) : 0;
    p.alias = p.tail && mode == 2;
    if (p.alias && N > 64) continue;
    const int fixed = q + (p.alias ? 0 : P) + p.tails * kPaChunk + misc;
    const int fit = (limit - fixed) / kPaPair;
    if (limit - fixed < 0 || fit < p.LP) continue;
    p.slots = fit < kPaMaxSlots ? fit : kPaMaxSlots;
    p.look = p.slots >= 2 * p.LP && (!p.tail || p.tails == 2);
    if (mode == 0 && p.tail && !p.look) continue;   // the second tail slot only pays with lookahead
    p.off_t = p.slots * kPaPair;
    p.off_p = p.alias ? p.off_t : p.off_t + p.tails * kPaChunk;
    p.off_q = (p.alias ? p.off_t + kPaChunk : p.off_p + P);
    p.off_misc = p.off_q + q;
    p.smem = p.off_misc + misc;
    const int cols = (2 + p.LP) * N;
    p.tmem_cols = 32;
    while (p.tmem_cols < cols) p.tmem_cols *= 2;
    return p.tmem_cols <= 512;
  }
  return false;
}

// sum_{i=0}^{n-1} floor((a i + b) / m) for a, b >= 0 (Euclid-like reduction, a
// few steps).
__device__ __forceinline__ long long floor_sum(long long n, long long m, long long a, long long b) {
  long long ans = 0;
  while (n > 0) {
    if (a >= m) {
      ans += (n - 1) * n / 2 * (a / m);
      a %= m;
    }
    if (b >= m) {
      ans += n * (b / m);
      b %= m;
    }
    const long long y = a * n + b;
    if (y < m) break;
    n = y / m;
    b = y % m;
    const long long t = m;
    m = a;
    a = t;
  }
  return ans;
}

// One sequence as the scheduler sees it.
struct PagedSeq {
  int tok0, n, len;           // first token, new tokens, cached length
  int rows, tiles;            // (token, head) rows, row tiles of N
};

template <int N>
__device__ __forceinline__ PagedSeq paged_seq(const Ragged& r, int b, int H, int total) {
  PagedSeq s;
  const int c0 = __ldg(r.cu + b), c1 = __ldg(r.cu + b + 1);
  s.tok0 = c0;
  s.n = (c0 >= 0 && c1 <= total && c1 > c0) ? c1 - c0 : 0;
  s.len = min(max(__ldg(r.lens + b), 0), r.cols * r.page);
  s.rows = s.n * H;
  s.tiles = (s.rows + N - 1) / N;
  return s;
}

// Key tiles of row tile rt: up to the position of its last row, at least one
// (a row that sees nothing is still written).
template <int N>
__device__ __forceinline__ int paged_key_tiles(const PagedSeq& s, int rt, int H) {
  const int last = min((rt + 1) * N, s.rows) - 1;
  const int keys = s.len - s.n + last / H + 1;
  return max(1, (keys + 127) / 128);
}

// Key tiles of row tiles 0 .. k-1.
template <int N>
__device__ __forceinline__ long long paged_tiles_before(const PagedSeq& s, int k, int H) {
  if (k <= 0) return 0;
  long long ans = 0;
  int full = k;
  if (k == s.tiles) {         // the last row tile may be short
    full = k - 1;
    ans = paged_key_tiles<N>(s, k - 1, H);
  }
  // row tile i ends at row x = (i + 1) N - 1, at position p = len - n + x / H:
  // p / 128 + 1 = ((len - n) H + x) / (128 H) + 1 tiles, one where p < 0
  const long long m = 128ll * H, c = (long long)(s.len - s.n) * H + N - 1;
  int first = 0;
  if (c < 0) first = (int)min((long long)full, (-c + N - 1) / N);
  ans += full + floor_sum(full - first, m, N, c + (long long)first * N);
  return ans;
}

// A CTA's share as a walk over items: (sequence, row tile, key tiles t0 .. t1).
template <int N>
struct PagedWalk {
  const Ragged& r;
  int H, total;
  long long left;
  int b, rt, t0, t1, nt;
  PagedSeq s;
  __device__ __forceinline__ PagedWalk(const Ragged& r_, int H_, int total_, long long count, int b0, int rt0, int tile0)
      : r(r_), H(H_), total(total_), left(count), b(b0), rt(rt0), t0(tile0) {
    if (left > 0) {
      s = paged_seq<N>(r, b, H, total);
      nt = paged_key_tiles<N>(s, rt, H);
      t1 = (int)min((long long)nt, t0 + left);
    }
  }
  __device__ __forceinline__ bool ok() const { return left > 0; }
  __device__ __forceinline__ void next() {
    left -= t1 - t0;
    if (left <= 0) return;
    t0 = 0;
    if (++rt >= s.tiles) {
      rt = 0;
      do {
        if (++b >= r.B) {
          left = 0;
          return;
        }
        s = paged_seq<N>(r, b, H, total);
      } while (s.tiles == 0);
    }
    nt = paged_key_tiles<N>(s, rt, H);
    t1 = (int)min((long long)nt, left);
  }
};

// NC consecutive 32-bit TMEM columns of this thread's lane (no wait).
__device__ __forceinline__ void tmem_ld8(uint32_t taddr, uint32_t* r) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(taddr));
}
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t* r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr), "r"(r[0]),
               "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
template <int NC>
__device__ __forceinline__ void tmem_ld_cols(uint32_t taddr, uint32_t (&r)[NC]) {
  if constexpr (NC == 8) {
    tmem_ld8(taddr, r);
  } else {
#pragma unroll
    for (int i = 0; i < NC; i += 16) tmem_ld16(taddr + i, *reinterpret_cast<uint32_t(*)[16]>(&r[i]));
  }
}

// Barrier of the 128 threads of one column half, with the OR of a predicate.
__device__ __forceinline__ bool half_any(int half, bool v) {
  uint32_t out;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 q, %1, 0;\n\t"
      "barrier.cta.red.or.pred p, %2, 128, q;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(out)
      : "r"((uint32_t)v), "r"(half + 1)
      : "memory");
  return out != 0;
}
__device__ __forceinline__ void half_sync(int half) {
  asm volatile("barrier.cta.sync %0, 128;" ::"r"(half + 1) : "memory");
}

__device__ __forceinline__ uint32_t float_key(float x) {
  const uint32_t u = __float_as_uint(x);
  return u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float float_unkey(uint32_t k) {
  return __uint_as_float(k ^ ((k >> 31) ? 0x80000000u : 0xffffffffu));
}

// Start of this CTA's share, found by the whole CTA.
struct PagedStart {
  long long count;            // key tiles in the share
  long long share;
  long long first;            // flat index of its first key tile
  int b, rt, tile;
};

template <int N>
__device__ __forceinline__ void paged_find(const Ragged& r, int H, int total, int min_share, PagedStart* out,
                                           long long* warp_sum, unsigned int* status) {
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  constexpr int NW = kPaThreads / 32;
  // round 0 adds up all sequences; round 1 finds the one that holds the share's first tile
  long long W = 0, target = 0;
  for (int round = 0; round < 2; ++round) {
    long long base = 0;
    for (int b0 = 0; b0 < r.B; b0 += kPaThreads) {
      const int b = b0 + tid;
      PagedSeq s;
      s.tiles = 0;
      long long t = 0;
      if (b < r.B) {
        s = paged_seq<N>(r, b, H, total);
        t = paged_tiles_before<N>(s, s.tiles, H);
        if (round == 0 && blockIdx.x == 0) {
          const bool bad = __ldg(r.lens + b) > r.cols * r.page || __ldg(r.cu + b + 1) > total ||
                           __ldg(r.cu + b + 1) < __ldg(r.cu + b) || (b == 0 && __ldg(r.cu) != 0) ||
                           (b == r.B - 1 && __ldg(r.cu + b + 1) != total);
          if (bad) record_error(status, DSV3_ERR_BOUNDS);
        }
      }
      long long inc = t;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long v = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += v;
      }
      if (lane == 31) warp_sum[warp] = inc;
      __syncthreads();
      long long before = base, all = base;
      for (int w = 0; w < NW; ++w) {
        if (w < warp) before += warp_sum[w];
        all += warp_sum[w];
      }
      const long long lo = before + inc - t, hi = before + inc;
      if (round == 1 && t > 0 && lo <= target && target < hi) {
        // last row tile that starts at or before the target
        int a = 0, z = s.tiles - 1;
        while (a < z) {
          const int mid = (a + z + 1) >> 1;
          if (lo + paged_tiles_before<N>(s, mid, H) <= target) a = mid;
          else z = mid - 1;
        }
        out->b = b;
        out->rt = a;
        out->tile = (int)(target - lo - paged_tiles_before<N>(s, a, H));
      }
      base = all;
      __syncthreads();
    }
    if (round == 0) {
      W = base;
      long long share = (W + gridDim.x - 1) / gridDim.x;
      if (share < min_share) share = min_share;
      target = share * blockIdx.x;
      if (tid == 0) {
        out->share = share;
        out->first = target;
        out->count = min(share, W - target);
        out->b = out->rt = out->tile = 0;
      }
      if (target >= W) break;
    }
  }
  __syncthreads();
}

template <int N>
__global__ void __launch_bounds__(kPaThreads, 1) paged_attention_tc_kernel(
    const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_kv, PagedPlan pl, Ragged rg,
    int total, int H, int R, int D, float scale_log2, int min_share, bf16* __restrict__ out,
    float* __restrict__ part_o, float2* __restrict__ part_ml, int4* __restrict__ rec, unsigned int* status) {
  constexpr int NC = N / 2;
  extern __shared__ __align__(1024) uint8_t smem[];
  float* mref = reinterpret_cast<float*>(smem + pl.off_misc);            // [N]
  int* lim = reinterpret_cast<int*>(mref + N);                           // [N] keys that a row sees
  float* red = reinterpret_cast<float*>(lim + N);                        // [2][32][4]
  uint64_t* pair_full = reinterpret_cast<uint64_t*>(red + 256);
  uint64_t* pair_empty = pair_full + kPaMaxSlots;
  uint64_t* tail_full = pair_empty + kPaMaxSlots;
  uint64_t* tail_empty = tail_full + 2;
  uint64_t* q_full = tail_empty + 2;
  uint64_t* q_empty = q_full + 1;
  uint64_t* s_full = q_empty + 1;     // [2]
  uint64_t* p_ready = s_full + 2;
  uint64_t* pv_done = p_ready + 1;
  uint64_t* o_free = pv_done + 1;
  uint64_t* drain = o_free + 1;
  PagedStart* start = reinterpret_cast<PagedStart*>(drain + 1);
  long long* scan = reinterpret_cast<long long*>(start + 1);             // [kPaThreads / 32]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(scan + kPaThreads / 32);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < pl.slots; ++i) {
      mbar_init(&pair_full[i], 1);
      mbar_init(&pair_empty[i], 1);
    }
    for (int i = 0; i < pl.tails; ++i) {
      mbar_init(&tail_full[i], 1);
      mbar_init(&tail_empty[i], 1);
    }
    mbar_init(q_full, 1);
    mbar_init(q_empty, 1);
    mbar_init(&s_full[0], 1);
    mbar_init(&s_full[1], 1);
    mbar_init(p_ready, 8);
    mbar_init(pv_done, 1);
    mbar_init(o_free, 8);
    mbar_init(drain, 1);
    *abort_flag = 0;
    fence_barrier_init();
    tma_prefetch_desc(&tm_q);
    tma_prefetch_desc(&tm_kv);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, pl.tmem_cols);
    tmem_relinquish();
  }
  paged_find<N>(rg, H, total, min_share, start, scan, status);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const long long count = start->count;
  const uint32_t smem0 = smem_u32(smem);
  const int boxes = rg.page >= 128 ? 1 : 128 / rg.page;        // TMA boxes per chunk

  if (warp == 0) {
    // ------------------------------------------------------------ producer
    uint32_t pu = 0, tu = 0, items = 0;      // pair uses, tail uses
    bool ok = count > 0;
    for (PagedWalk<N> w(rg, H, total, ok ? count : 0, start->b, start->rt, start->tile); w.ok() && ok; w.next(), ++items) {
      if (lane == 0) {
        ok = mbar_wait_bounded(q_empty, (items & 1u) ^ 1u, abort_flag, status, DSV3_ERR_WAIT_EMPTY);
        if (ok) {
          mbar_arrive_expect_tx(q_full, pl.nch * N * 128);
          const int row = w.s.tok0 * H + w.rt * N;
          for (int c = 0; c < pl.nch; ++c) tma_load_2d(smem + pl.off_q + c * N * 128, &tm_q, q_full, 64 * c, row);
        }
      }
      ok = __shfl_sync(0xffffffffu, ok, 0);
      for (int t = w.t0; t < w.t1 && ok; ++t) {
        // page of this lane's box; one outside the pool reads as zeros
        int pg = rg.pool;
        const int key = t * 128 + lane * (128 / boxes);
        if (lane < boxes && key < w.s.len) {
          pg = rg.table[w.b * rg.ldt + key / rg.page];
          if (pg < 0 || pg >= rg.pool) {
            record_error(status, DSV3_ERR_BOUNDS);
            pg = rg.pool;
          }
        }
        const int row = key & (rg.page - 1);
        const int dst = lane * (128 / boxes) * 128;
        for (int m = 0; m <= pl.LP && ok; ++m) {
          if (m == pl.LP && !pl.tail) break;
          const bool is_tail = m == pl.LP;
          const int c0 = 2 * m, nc = is_tail ? 1 : min(2, pl.nch - c0);
          const int slot = is_tail ? tu % pl.tails : pu % pl.slots;
          const uint32_t ph = (is_tail ? tu / pl.tails : pu / pl.slots) & 1u;
          uint64_t* full = is_tail ? &tail_full[slot] : &pair_full[slot];
          uint64_t* empty = is_tail ? &tail_empty[slot] : &pair_empty[slot];
          uint8_t* at = smem + (is_tail ? pl.off_t + slot * kPaChunk : slot * kPaPair);
          if (lane == 0) {
            ok = mbar_wait_bounded(empty, ph ^ 1u, abort_flag, status, DSV3_ERR_WAIT_EMPTY);
            if (ok) mbar_arrive_expect_tx(full, nc * kPaChunk);
          }
          ok = __shfl_sync(0xffffffffu, ok, 0);
          if (ok && lane < boxes)
            for (int c = 0; c < nc; ++c) tma_load_3d(at + c * kPaChunk + dst, &tm_kv, full, 64 * (c0 + c), row, pg);
          if (ok) {
            if (is_tail) ++tu;
            else ++pu;
          }
        }
      }
      if (!ok) break;
    }
    // every issued copy lands before the CTA may exit
    if (lane == 0) {
      for (uint32_t i = pu > (uint32_t)pl.slots ? pu - pl.slots : 0; i < pu; ++i)
        mbar_wait_bounded(&pair_full[i % pl.slots], (i / pl.slots) & 1u, nullptr, status, DSV3_ERR_WAIT_FULL);
      for (uint32_t i = tu > (uint32_t)pl.tails ? tu - pl.tails : 0; i < tu; ++i)
        mbar_wait_bounded(&tail_full[i % pl.tails], (i / pl.tails) & 1u, nullptr, status, DSV3_ERR_WAIT_FULL);
      if (items > 0) mbar_wait_bounded(q_full, (items - 1) & 1u, nullptr, status, DSV3_ERR_WAIT_FULL);
    }
  } else if (warp == 1) {
    // ---------------------------------------------------------- MMA issuer
    if (lane == 0 && count > 0) {
      constexpr uint32_t I_S = idesc_bf16_f32(128, N, 0, 0);     // S^T = K Q^T
      constexpr uint32_t I_O = idesc_bf16_f32(128, N, 1, 1);     // O^T += V^T P^T, both read MN-major
      PagedWalk<N> ws(rg, H, total, count, start->b, start->rt, start->tile);   // walk of S
      PagedWalk<N> wp(rg, H, total, count, start->b, start->rt, start->tile);   // walk of PV
      int ts = ws.t0, tp = wp.t0;
      uint32_t gs = 0, gp = 0, s_items = 0, p_items = 0, tu = 0;
      bool ok = true, issued = false;
      // S^T of the next tile in order
      auto issue_s = [&]() {
        if (ts == ws.t0) {
          if (!mbar_wait_bounded(q_full, s_items & 1u, abort_flag, status, DSV3_ERR_WAIT_FULL)) return false;
        }
        const uint32_t d = tmem + (gs & 1u) * N;
        uint32_t acc = 0;
        for (int m = 0; m <= pl.LP; ++m) {
          if (m == pl.LP && !pl.tail) break;
          const bool is_tail = m == pl.LP;
          const uint32_t u = is_tail ? tu : gs * pl.LP + m;
          const int ring = is_tail ? pl.tails : pl.slots;
          const int slot = u % ring;
          if (!mbar_wait_bounded(is_tail ? &tail_full[slot] : &pair_full[slot], (u / ring) & 1u, abort_flag, status,
                                 DSV3_ERR_WAIT_FULL))
            return false;
          tc_fence_after();
          const int nc = is_tail ? 1 : min(2, pl.nch - 2 * m);
          const uint32_t at = smem0 + (is_tail ? pl.off_t + slot * kPaChunk : slot * kPaPair);
          for (int c = 0; c < nc; ++c) {
            const int ch = 2 * m + c, ks = min(4, (D - 64 * ch + 15) / 16);
            for (int kk = 0; kk < ks; ++kk) {
              umma_bf16(d, smem_desc_sw128(at + c * kPaChunk + kk * 32, 16, 1024),
                        smem_desc_sw128(smem0 + pl.off_q + ch * N * 128 + kk * 32, 16, 1024), I_S, acc);
              acc = 1;
            }
          }
          issued = true;
          if (is_tail) {
            if (!pl.alias) umma_commit(&tail_empty[slot]);
            ++tu;
          }
        }
        umma_commit(&s_full[gs & 1u]);
        ++gs;
        if (++ts >= ws.t1) {
          umma_commit(q_empty);
          ++s_items;
          ws.next();
          ts = ws.t0;
        }
        return true;
      };
      ok = issue_s();
      while (ok && wp.ok()) {
        if (pl.look && ws.ok()) ok = issue_s();
        if (!ok) break;
        if (!mbar_wait_bounded(p_ready, gp & 1u, abort_flag, status, DSV3_ERR_WAIT_FULL)) break;
        const bool first = tp == wp.t0;
        if (first && p_items > 0 &&
            !mbar_wait_bounded(o_free, (p_items - 1) & 1u, abort_flag, status, DSV3_ERR_WAIT_TMEM))
          break;
        tc_fence_after();
        for (int m = 0; m < pl.LP; ++m) {
          const int slot = (gp * pl.LP + m) % pl.slots;
          for (int kk = 0; kk < 8; ++kk)
            umma_bf16(tmem + (2 + m) * N, smem_desc_sw128(smem0 + slot * kPaPair + kk * 2048, kPaChunk, 1024),
                      smem_desc_sw128(smem0 + pl.off_p + kk * 2048, kPaChunk, 1024), I_O, !first || kk > 0);
          umma_commit(&pair_empty[slot]);
        }
        if (pl.alias) umma_commit(&tail_empty[0]);
        umma_commit(pv_done);
        issued = true;
        ++gp;
        if (++tp >= wp.t1) {
          ++p_items;
          wp.next();
          tp = wp.t0;
        }
        if (!pl.look && ws.ok()) ok = issue_s();
      }
      if (issued) {   // no MMA may still write TMEM when it is freed
        umma_commit(drain);
        mbar_wait_bounded(drain, 0, nullptr, status, DSV3_ERR_WAIT_TMEM);
      }
    }
  } else {
    // ---------------------------------------------------- softmax / epilogue
    const int half = (warp - 2) >> 2;              // columns half * NC ..
    const int quarter = warp & 3;                  // TMEM lanes 32 * quarter ..
    const int key = quarter * 32 + lane;           // key of S^T, latent column of O^T
    const int ht = (warp - 2 - 4 * half) * 32 + lane;
    const uint32_t lane_base = (uint32_t)(quarter * 32) << 16;
    const int col0 = half * NC;
    float* myred = red + half * 128;               // [32][4]
    float4* mref4 = reinterpret_cast<float4*>(mref + col0);
    const int4* lim4 = reinterpret_cast<const int4*>(lim + col0);
    uint32_t g = 0;
    int4 my_rec = make_int4(-1, 0, 0, 0);
    for (PagedWalk<N> w(rg, H, total, count, start->b, start->rt, start->tile); w.ok(); w.next()) {
      const int base = w.s.len - w.s.n;
      const int nr = min(N, w.s.rows - w.rt * N);
      half_sync(half);                             // the last item's references are read
      if (ht < NC) {
        const int n = col0 + ht;
        mref[n] = kPaUnset;
        lim[n] = n < nr ? base + (w.rt * N + n) / H + 1 : 0;
      }
      half_sync(half);
      const int seen_by_all = base + (w.rt * N) / H + 1;      // keys that every row sees
      float l[NC];
#pragma unroll
      for (int c = 0; c < NC; ++c) l[c] = 0.f;
      for (int t = w.t0; t < w.t1; ++t, ++g) {
        mbar_wait_bounded(&s_full[g & 1u], (g >> 1) & 1u, abort_flag, status, DSV3_ERR_WAIT_TMEM);
        tc_fence_after();
        uint32_t sr[NC];
        tmem_ld_cols<NC>(tmem + lane_base + (g & 1u) * N + col0, sr);
        tmem_ld_wait();
        const int pos = t * 128 + key;
        if (t * 128 + 128 > seen_by_all) {
#pragma unroll
          for (int c = 0; c < NC; c += 4) {
            const int4 k4 = lim4[c / 4];
            if (pos >= k4.x) sr[c] = 0xff800000u;
            if (pos >= k4.y) sr[c + 1] = 0xff800000u;
            if (pos >= k4.z) sr[c + 2] = 0xff800000u;
            if (pos >= k4.w) sr[c + 3] = 0xff800000u;
          }
        }
        float over = -INFINITY;
#pragma unroll
        for (int c = 0; c < NC; c += 4) {
          const float4 m4 = mref4[c / 4];
          over = fmaxf(over, fmaf(__uint_as_float(sr[c]), scale_log2, -m4.x));
          over = fmaxf(over, fmaf(__uint_as_float(sr[c + 1]), scale_log2, -m4.y));
          over = fmaxf(over, fmaf(__uint_as_float(sr[c + 2]), scale_log2, -m4.z));
          over = fmaxf(over, fmaf(__uint_as_float(sr[c + 3]), scale_log2, -m4.w));
        }
        const bool move = half_any(half, over > 8.f);
        // P and O^T of the previous tile are no longer in use by the tensor core
        if (g > 0) mbar_wait_bounded(pv_done, (g - 1) & 1u, abort_flag, status, DSV3_ERR_WAIT_TMEM);
        tc_fence_after();
        if (move) {
#pragma unroll
          for (int c0 = 0; c0 < NC; c0 += 32) {
            constexpr int W = NC < 32 ? NC : 32;
            uint32_t mine = 0;
#pragma unroll
            for (int c = 0; c < W; ++c) {
              const uint32_t k = __reduce_max_sync(0xffffffffu, float_key(__uint_as_float(sr[c0 + c]) * scale_log2));
              if (lane == c) mine = k;
            }
            if (lane < W) myred[lane * 4 + (warp - 2 - 4 * half)] = float_unkey(mine);
            half_sync(half);
            float keep = kPaUnset;
#pragma unroll
            for (int c = 0; c < W; c += 8) {
              float corr[8];
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                const float4 r4 = *reinterpret_cast<const float4*>(myred + (c + i) * 4);
                const float old = mref[col0 + c0 + c + i];
                const float top = fmaxf(fmaxf(fmaxf(r4.x, r4.y), fmaxf(r4.z, r4.w)), old);
                corr[i] = ex2_approx(old - top);
                l[c0 + c + i] *= corr[i];
                if (lane == c + i) keep = top;
              }
              if (t > w.t0) {
                for (int m = 0; m < pl.LP; ++m) {
                  uint32_t o[8];
                  const uint32_t at = tmem + lane_base + (2 + m) * N + col0 + c0 + c;
                  tmem_ld8(at, o);
                  tmem_ld_wait();
#pragma unroll
                  for (int i = 0; i < 8; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * corr[i]);
                  tmem_st8(at, o);
                }
              }
            }
            half_sync(half);                       // all threads have read the old references
            if (ht < W) mref[col0 + c0 + lane] = keep;
          }
          tmem_st_wait();
          half_sync(half);
        }
        uint8_t* prow = smem + pl.off_p + key * 128;
#pragma unroll
        for (int c = 0; c < NC; c += 8) {
          uint32_t pk[4];
#pragma unroll
          for (int i = 0; i < 8; i += 4) {
            const float4 m4 = mref4[(c + i) / 4];
            const float p0 = ex2_approx(fmaf(__uint_as_float(sr[c + i]), scale_log2, -m4.x));
            const float p1 = ex2_approx(fmaf(__uint_as_float(sr[c + i + 1]), scale_log2, -m4.y));
            const float p2 = ex2_approx(fmaf(__uint_as_float(sr[c + i + 2]), scale_log2, -m4.z));
            const float p3 = ex2_approx(fmaf(__uint_as_float(sr[c + i + 3]), scale_log2, -m4.w));
            pk[i / 2] = pack_bf16x2(p0, p1);
            pk[i / 2 + 1] = pack_bf16x2(p2, p3);
            l[c + i] += __uint_as_float(pk[i / 2] << 16);
            l[c + i + 1] += __uint_as_float(pk[i / 2] & 0xffff0000u);
            l[c + i + 2] += __uint_as_float(pk[i / 2 + 1] << 16);
            l[c + i + 3] += __uint_as_float(pk[i / 2 + 1] & 0xffff0000u);
          }
          const int n = col0 + c;
          *reinterpret_cast<uint4*>(prow + (n >> 6) * kPaChunk + ((((n & 63) >> 3) ^ (key & 7)) << 4)) =
              make_uint4(pk[0], pk[1], pk[2], pk[3]);
        }
        // rows of the pages past the cached length hold anything: zero them, so
        // that their zero weights do not meet an infinity or NaN
        if (t * 128 + 128 > w.s.len && pos >= w.s.len) {
          for (int c = half; c < 2 * pl.LP; c += 2) {
            const int slot = (g * pl.LP + (c >> 1)) % pl.slots;
            uint4* z = reinterpret_cast<uint4*>(smem + slot * kPaPair + (c & 1) * kPaChunk + key * 128);
#pragma unroll
            for (int i = 0; i < 8; ++i) z[i] = make_uint4(0, 0, 0, 0);
          }
        }
        fence_proxy_async_smem();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(p_ready);
      }
      // ---- item epilogue
      mbar_wait_bounded(pv_done, (g - 1) & 1u, abort_flag, status, DSV3_ERR_WAIT_TMEM);
      tc_fence_after();
      const bool whole = w.t0 == 0 && w.t1 == w.nt;
      const int slot = 2 * blockIdx.x + (w.t0 == 0 ? 1 : 0);
      const long long row0 = (long long)w.s.tok0 * H + (long long)w.rt * N;
      if (!whole && w.t0 == 0) {
        const long long s0 = start->first + (count - w.left);
        my_rec = make_int4((int)row0, nr, (int)((s0 + w.nt - 1) / start->share), 0);
      }
#pragma unroll
      for (int c0 = 0; c0 < NC; c0 += 32) {
        constexpr int W = NC < 32 ? NC : 32;
        half_sync(half);
#pragma unroll
        for (int c = 0; c < W; ++c) {
          const float v = warp_sum(l[c0 + c]);
          if (lane == c) myred[c * 4 + (warp - 2 - 4 * half)] = v;
        }
        half_sync(half);
        if (!whole && ht < W) {
          const float4 r4 = *reinterpret_cast<const float4*>(myred + lane * 4);
          const int n = col0 + c0 + lane;
          part_ml[(size_t)slot * N + n] = make_float2(mref[n], (r4.x + r4.y) + (r4.z + r4.w));
        }
#pragma unroll
        for (int c = 0; c < W; c += 8) {
          float inv[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float4 r4 = *reinterpret_cast<const float4*>(myred + (c + i) * 4);
            const float sum = (r4.x + r4.y) + (r4.z + r4.w);
            inv[i] = sum > 0.f ? 1.f / sum : (sum == sum ? 0.f : sum);
          }
          for (int m = 0; m < pl.LP; ++m) {
            uint32_t o[8];
            tmem_ld8(tmem + lane_base + (2 + m) * N + col0 + c0 + c, o);
            tmem_ld_wait();
            const int r = 128 * m + key;
            if (r < R) {
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                const int n = col0 + c0 + c + i;
                if (n < nr) {
                  if (whole) out[(size_t)(row0 + n) * R + r] = __float2bfloat16(__uint_as_float(o[i]) * inv[i]);
                  else part_o[((size_t)slot * N + n) * R + r] = __uint_as_float(o[i]);
                }
              }
            }
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(o_free);
    }
    if (threadIdx.x == 64) rec[blockIdx.x] = my_rec;
  }
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, pl.tmem_cols);
  }
}

// Joins the partials of row tiles that were cut: CTA (g, y) takes rows of the
// one that begins in share g.  The parts are added in share order.
template <int N>
__global__ void __launch_bounds__(128) paged_merge_kernel(const float* __restrict__ part_o,
                                                          const float2* __restrict__ part_ml,
                                                          const int4* __restrict__ rec, int R,
                                                          bf16* __restrict__ out) {
  const int g = blockIdx.x;
  const int4 rc = rec[g];
  const int n = blockIdx.y;
  if (rc.x < 0 || n >= rc.y) return;
  const int parts = rc.z - g + 1;
  // part 0 is slot 2 g + 1, part i > 0 slot 2 (g + i)
  float M = -INFINITY;
  for (int i = 0; i < parts; ++i) {
    const float2 ml = part_ml[(size_t)(i ? 2 * (g + i) : 2 * g + 1) * N + n];
    if (ml.y > 0.f) M = fmaxf(M, ml.x);
  }
  float sum = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  const int r = threadIdx.x * 4;
  for (int i = 0; i < parts; ++i) {
    const size_t at = (size_t)(i ? 2 * (g + i) : 2 * g + 1) * N + n;
    const float2 ml = part_ml[at];
    if (ml.y == 0.f) continue;
    const float wgt = ex2_approx(ml.x - M);
    sum += ml.y * wgt;
    if (r < R) {
      const float4 o = *reinterpret_cast<const float4*>(part_o + at * R + r);
      acc.x += o.x * wgt;
      acc.y += o.y * wgt;
      acc.z += o.z * wgt;
      acc.w += o.w * wgt;
    }
  }
  if (r < R) {
    const float inv = sum > 0.f ? 1.f / sum : (sum == sum ? 0.f : sum);
    uint2 v;
    v.x = pack_bf16x2(acc.x * inv, acc.y * inv);
    v.y = pack_bf16x2(acc.z * inv, acc.w * inv);
    *reinterpret_cast<uint2*>(out + (size_t)(rc.x + n) * R + r) = v;
  }
}
