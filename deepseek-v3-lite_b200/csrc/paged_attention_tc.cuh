// tcgen05 attention of a ragged batch over a paged latent cache (sm_100a).
// Included by paged.cu inside its anonymous namespace, after Ragged.
//
// The rows of sequence b are its (token, head) pairs, n_b * H of them, cut
// into row tiles of N; a key tile is KT cached rows.  Both products are
// computed transposed, so that the cached rows are the M side of the first and
// the latent columns the M side of the second, and one copy of a key tile in
// shared memory serves both:
//
//   S^T [KT keys x N rows] = K [KT x D] . Q^T                   (K-major A)
//   P^T = 2^(scale log2(e) S^T - m)                             (bf16, [key][row])
//   O^T [R x N rows]      += V^T [R x KT keys] . P^T            (the same K, read MN-major)
//
// KT is 64: with R 512 and N 64 the shared memory then holds two key tiles (128
// rows left no room for a second; 441 us against 361 us for 4 x 512 new tokens when
// it was chosen), and an MMA of 64 keys and 64 rows takes 32 cycles against 48 of
// 128 keys.
//
// P is bf16 because an MMA takes one type for both of its operands and the cache is
// bf16.  Each weight is then off by 2^-9 at most, as the result is by its own
// rounding; all else (scores, references, sums, O, partials) is fp32.
//
// The cache row [latent | rotated key] is read as 64-column chunks [KT x 64]
// with a 128-byte swizzle; chunk pairs 0 .. LP-1 cover the latent (LP =
// ceil(R / 128)), and where D reaches past them one more tail chunk holds the
// rest of the rotated key.  Columns past D are zero-filled by TMA, rows past
// the cached length are masked in S and zeroed in shared memory before the
// second product (pages are never assumed to be initialised past that).
//
// A softmax thread owns one key and a few of the rows: there is no per-row
// maximum over keys at hand, and none is needed.  Each row keeps a reference m
// that any score may exceed by up to 2^8 without harm (sums and O are fp32, P
// has the same relative precision at any scale); the 128 threads of a warpgroup
// vote per tile, and only when one exceeds it are the rows' maxima computed, m
// moved and O^T rescaled.  Row sums are kept per thread and added
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
// Warps: 0 TMA, 1 first product (and TMEM), then two or four warpgroups of softmax
// and epilogue, and one warp for the second product.  Every wait is
// bounded; after one ran out the softmax warps go on without waiting, so that
// they meet at their barriers, and the others stop.
//
// Measured on the device, without the merge (R 512, 16 heads, pages of 64): 64
// requests with 512 to 4,096 rows, one token each, 40 us (169 MB, floor 26 us; 4.1
// TB/s with a cold L2); two of 100,000 rows 60 us (floor 42 us); 4 x 512 new tokens
// on 3,000 to 4,096 rows 365 us with the merge, 630 TFLOP/s: tensor pipe active in
// 44% of the cycles, its operand path in 48%, which is S^T with 64 keys on the M side
// and 64 rows on the N side of both.  R 192, 16 ragged chunks of up to 509 tokens: 79
// us, tensor pipe 28%, bound by the softmax and by the turn from one row tile to the
// next.

// Softmax warpgroups of a row tile, each with its share of the rows: two for few
// rows; four for 64 and 128, where the softmax of a tile takes longer than its MMAs
// (2,200 cycles against 1,400 for 128 rows of R 192, with two).
constexpr int pa_groups(int N) { return N >= 64 ? 4 : 2; }
constexpr int pa_threads(int N) { return 32 * (3 + 4 * pa_groups(N)); }   // TMA, S, softmax, PV
constexpr int KT = 64;                       // key tile
constexpr int kPaMaxSlots = 16;
constexpr int kPaSmem = 232448;              // shared memory of a CTA, at most
constexpr float kPaUnset = -1e30f;           // reference of a row that has seen no key
constexpr float kPaNever = 1e30f;            // of one that sees none, or lies past the sequence's rows: the tile
                                             // holds the next sequence's queries there, whose scores have no vote
constexpr float kPaLead = 12.f;              // first reference above the first key's score (log2)

struct PagedPlan {
  int LP, nch, tail;          // latent chunk pairs, chunks, 1 if there is a tail chunk
  int slots, tails;           // ring slots (pairs), tail slots
  int pbufs;                  // buffers of P
  int off_q, off_p, off_t, off_misc, smem, tmem_cols;
};

// Shared memory of a plan: ring | tail slots | P | Q | misc, with as many ring
// slots as fit; at least two key tiles' worth, so that one loads while the
// other is in use.
inline bool paged_plan(int N, int R, int D, PagedPlan& p) {
  const int chunk = KT * 128;
  p.LP = (R + 127) / 128;
  p.nch = (D + 63) / 64;
  p.tail = D > 128 * p.LP ? 1 : 0;
  p.tails = p.tail ? 2 : 0;
  const int q = p.nch * N * 128, P = (N + 63) / 64 * chunk, misc = 28 * N + 448 + pa_threads(N) / 4;
  // a second P buffer where the ring still holds two key tiles with it
  for (p.pbufs = 2;; --p.pbufs) {
    const int fit = (kPaSmem - q - p.pbufs * P - p.tails * chunk - misc) / (2 * chunk);
    p.slots = fit < kPaMaxSlots ? fit : kPaMaxSlots;
    if (p.slots >= 2 * p.LP || p.pbufs == 1) break;
  }
  p.off_t = p.slots * 2 * chunk;
  p.off_p = p.off_t + p.tails * chunk;
  p.off_q = p.off_p + p.pbufs * P;
  p.off_misc = p.off_q + q;
  p.smem = p.off_misc + misc;
  p.tmem_cols = 32;
  while (p.tmem_cols < (2 + p.LP) * N) p.tmem_cols *= 2;
  return p.slots >= 2 * p.LP && p.tmem_cols <= 512;
}

// sum_{i=0}^{n-1} floor((a i + b) / m) for a, b >= 0 (Euclid-like reduction, a
// few steps).  T is 32 bits wide where a n + b fits: its division is several
// times cheaper.
template <typename T>
__device__ __forceinline__ long long floor_sum(T n, T m, T a, T b) {
  long long ans = 0;
  while (n > 0) {
    if (a >= m) {
      ans += (long long)(n - 1) * n / 2 * (a / m);
      a %= m;
    }
    if (b >= m) {
      ans += (long long)n * (b / m);
      b %= m;
    }
    const T y = a * n + b;
    if (y < m) break;
    n = y / m;
    b = y % m;
    const T t = m;
    m = a;
    a = t;
  }
  return ans;
}

// One sequence as the scheduler sees it.
struct PagedSeq {
  int tok0, end, n, len;      // first token, the one after the last, new tokens, cached length
  int rows, tiles;            // (token, head) rows, row tiles of N
};

template <int N>
__device__ __forceinline__ PagedSeq paged_seq(const Ragged& r, int b, int H, int total) {
  PagedSeq s;
  const int c0 = __ldg(r.cu + b), c1 = __ldg(r.cu + b + 1);
  s.tok0 = c0;
  s.end = c1;
  s.n = (c0 >= 0 && c1 <= total && c1 > c0) ? c1 - c0 : 0;
  s.len = min(max(__ldg(r.lens + b), 0), r.cols * r.page);
  s.rows = s.n * H;
  s.tiles = (s.rows + N - 1) / N;
  return s;
}

// A value that all lanes of the warp hold, marked as such for the compiler: loop
// bounds and descriptors derived from it stay in uniform registers, and MMAs
// under such control flow issue without moves or divergent branches (32 cycles
// apiece against 67 to 200).
__device__ __forceinline__ int warp_uniform(int x) { return __shfl_sync(0xffffffffu, x, 0); }

// Key tiles of row tile rt: up to the position of its last row, at least one
// (a row that sees nothing is still written).
template <int N>
__device__ __forceinline__ int paged_key_tiles(const PagedSeq& s, int rt, int H) {
  const int last = min((rt + 1) * N, s.rows) - 1;
  const int keys = s.len - s.n + last / H + 1;
  return max(1, (keys + KT - 1) / KT);
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
  // p / KT + 1 = ((len - n) H + x) / (KT H) + 1 tiles, one where p < 0
  const long long c = (long long)(s.len - s.n) * H + N - 1;
  int first = 0;
  if (c < 0) first = (int)min((long long)full, (-c + N - 1) / N);
  const long long b = c + (long long)first * N;
  if (b + (long long)full * N < (1ll << 31))
    return ans + full + floor_sum<uint32_t>(full - first, (uint32_t)KT * H, N, (uint32_t)b);
  return ans + full + floor_sum<long long>(full - first, (long long)KT * H, N, b);
}

// A CTA's share as a walk over items: (sequence, row tile, key tiles t0 .. t1).
template <int N>
struct PagedWalk {
  const Ragged& r;
  int H, total;
  int left;
  int b, rt, t0, t1, nt;
  PagedSeq s;
  __device__ __forceinline__ PagedWalk(const Ragged& r_, int H_, int total_, int count, int b0, int rt0, int tile0)
      : r(r_), H(H_), total(total_), left(count), b(b0), rt(rt0), t0(tile0) {
    if (left > 0) {
      load();
      nt = paged_key_tiles<N>(s, rt, H);
      t1 = min(nt, t0 + left);
    }
  }
  __device__ __forceinline__ void load() {
    s = paged_seq<N>(r, b, H, total);
    s.tok0 = warp_uniform(s.tok0);
    s.n = warp_uniform(s.n);
    s.len = warp_uniform(s.len);
    s.rows = s.n * H;
    s.tiles = (s.rows + N - 1) / N;
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
        load();
      } while (s.tiles == 0);
    }
    nt = paged_key_tiles<N>(s, rt, H);
    t1 = min(nt, left);
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
// Lanes 0..15 of the warp's quarter: threads 0..15 get W columns at taddr,
// threads 16..31 those SPLIT columns further of the same lanes.
template <int SPLIT, int W>
__device__ __forceinline__ void tmem_ld_half(uint32_t taddr, uint32_t* r) {
  if constexpr (W == 4) {
    asm volatile("tcgen05.ld.sync.aligned.16x32bx2.x4.b32 {%0, %1, %2, %3}, [%4], %5;"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(taddr), "n"(SPLIT));
  } else if constexpr (W == 8) {
    asm volatile("tcgen05.ld.sync.aligned.16x32bx2.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8], %9;"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "r"(taddr), "n"(SPLIT));
  } else {
#pragma unroll
    for (int i = 0; i < W; i += 16)
      asm volatile(
          "tcgen05.ld.sync.aligned.16x32bx2.x16.b32 "
          "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16], %17;"
          : "=r"(r[i]), "=r"(r[i + 1]), "=r"(r[i + 2]), "=r"(r[i + 3]), "=r"(r[i + 4]), "=r"(r[i + 5]), "=r"(r[i + 6]),
            "=r"(r[i + 7]), "=r"(r[i + 8]), "=r"(r[i + 9]), "=r"(r[i + 10]), "=r"(r[i + 11]), "=r"(r[i + 12]),
            "=r"(r[i + 13]), "=r"(r[i + 14]), "=r"(r[i + 15])
          : "r"(taddr + i), "n"(SPLIT));
  }
}
// Barrier of the 128 threads of a softmax warpgroup, with the OR of a predicate.
__device__ __forceinline__ bool wg_any(int wg, bool v) {
  uint32_t out;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 q, %1, 0;\n\t"
      "barrier.cta.red.or.pred p, %2, 128, q;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(out)
      : "r"((uint32_t)v), "r"(wg + 1)
      : "memory");
  return out != 0;
}
__device__ __forceinline__ void wg_sync(int wg) {
  asm volatile("barrier.cta.sync %0, 128;" ::"r"(wg + 1) : "memory");
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
  int count;                  // key tiles in the share
  int share;
  int first;                  // flat index of its first key tile
  int local;                  // its index within sequence b
  int b, rt, tile, found;
  int gap;                    // the offsets do not cover every token once
  int excess;                 // more key tiles than 32 bits count
};

template <int N>
__device__ __forceinline__ void paged_find(const Ragged& r, int H, int total, PagedStart* out, int2* scan,
                                           unsigned int* status) {
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  constexpr int THREADS = pa_threads(N), NW = THREADS / 32;
  if (tid == 0) out->gap = out->excess = 0;
  // round 0 adds up all sequences; round 1 finds the one that holds the share's
  // first tile (a batch of up to THREADS sequences is still in registers)
  int target = 0, t = 0;
  PagedSeq s;
  s.tiles = 0;
  for (int round = 0; round < 2; ++round) {
    int base = 0, thousands = 0;             // key tiles, and by 1,024 rounded up per sequence
    for (int b0 = 0; b0 < r.B; b0 += THREADS) {
      const int b = b0 + tid;
      bool gap = false;
      int more = 0;
      if (round == 0 || r.B > THREADS) {
        s.tiles = 0;
        t = 0;
        if (b < r.B) {
          s = paged_seq<N>(r, b, H, total);
          const long long tiles = paged_tiles_before<N>(s, s.tiles, H);
          t = (int)tiles;
          if (round == 0) {
            more = (int)min((tiles + 1023) >> 10, 1ll << 21);
            gap = s.end > total || s.end < s.tok0 || (b == 0 && s.tok0 != 0) || (b == r.B - 1 && s.end != total);
            if (blockIdx.x == 0 && (gap || __ldg(r.lens + b) > r.cols * r.page)) record_error(status, DSV3_ERR_BOUNDS);
          }
        }
      }
      int inc = t;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += v;
      }
      more = __reduce_add_sync(0xffffffffu, more);
      if (lane == 31) scan[warp] = make_int2(inc, more);
      __syncthreads();
      if (gap) out->gap = 1;
      int before = base, all = base;
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        const int2 v = scan[w];
        if (w < warp) before += v.x;
        all += v.x;
        thousands += v.y;                      // (at most 19 warps of 32 x 2^21)
      }
      thousands = min(thousands, 1 << 21);
      if (round == 1 && t > 0 && before + inc - t <= target && target < before + inc) {
        out->b = b;
        out->local = target - (before + inc - t);
        if (s.tiles == 1) {
          out->tile = (int)out->local;
          out->found = 1;
        }
      }
      base = all;
      __syncthreads();
    }
    if (round == 0) {
      if (thousands >= (1 << 21) - 1024) {     // reported, and nothing is computed
        if (tid == 0) {
          out->excess = 1;
          if (blockIdx.x == 0) record_error(status, DSV3_ERR_BOUNDS);
        }
        base = 0;
      }
      int share = (base + gridDim.x - 1) / gridDim.x;
      target = share * blockIdx.x;
      if (tid == 0) {
        out->share = share;
        out->first = target;
        out->count = min(share, base - target);
        out->b = out->rt = out->tile = 0;
        out->local = 0;
        out->found = 0;
      }
      if (target >= base) break;
    }
  }
  __syncthreads();
  if (out->count > 0 && !out->found) {   // the row tile of that sequence: every thread tries one candidate
    const int local = out->local;
    s = paged_seq<N>(r, out->b, H, total);
    int lo = 0, hi = s.tiles;                    // the answer lies in [lo, hi)
    while (hi > lo) {
      const int step = (hi - lo + THREADS - 1) / THREADS, k = lo + tid * step;
      const int k1 = min(k + step, hi);
      if (k < hi) {
        const long long at = paged_tiles_before<N>(s, k, H);
        if (at <= local && (k1 == s.tiles || local < paged_tiles_before<N>(s, k1, H))) {
          out->rt = k;
          out->tile = (int)(local - at);
        }
      }
      __syncthreads();
      lo = out->rt;
      hi = step > 1 ? min(lo + step, hi) : lo;
      __syncthreads();
    }
  }
}

// Zeroes the result of the tokens that no sequence holds, or of all; the whole CTA,
// a token per CTA in turn.  Only for metadata that are reported as wrong.
__device__ __forceinline__ void paged_clear(const Ragged& r, bool all, int total, size_t row_bytes, uint8_t* out) {
#pragma unroll 1
  for (int t = blockIdx.x; t < total; t += gridDim.x) {
    bool held = false;
#pragma unroll 1
    for (int b = threadIdx.x; b < r.B; b += blockDim.x) {
      const int c0 = __ldg(r.cu + b), c1 = __ldg(r.cu + b + 1);
      held |= !all && c0 >= 0 && c1 <= total && c0 <= t && t < c1;
    }
    if (__syncthreads_or(held)) continue;
#pragma unroll 1
    for (size_t i = threadIdx.x * 16; i < row_bytes; i += blockDim.x * 16)
      *reinterpret_cast<uint4*>(out + t * row_bytes + i) = make_uint4(0, 0, 0, 0);
  }
}

// Combines W values per lane over groups of L lanes, column by column: W / 2
// exchanges, then W / 4 ..., since a lane keeps only half of its columns at each
// step.  Lane i of a group ends with column i * W / L.
template <int W, int L, typename Op>
__device__ __forceinline__ float fold_columns(float (&v)[W], int lane, Op op) {
  int o = L / 2;
#pragma unroll
  for (int w = W; w > 1; w >>= 1, o >>= 1) {
    const bool up = lane & o;
#pragma unroll
    for (int i = 0; i < w / 2; ++i) {
      const float send = up ? v[i] : v[i + w / 2], keep = up ? v[i + w / 2] : v[i];
      v[i] = op(keep, __shfl_xor_sync(0xffffffffu, send, o));
    }
  }
  for (; o > 0; o >>= 1) v[0] = op(v[0], __shfl_xor_sync(0xffffffffu, v[0], o));
  return v[0];
}

// One MMA by the lane whose `leader` is set.  The whole warp runs the issuing
// code with the same values: descriptors then stay in uniform registers, where
// the instruction wants them (one lane in a divergent branch moved each operand
// there first and issued an MMA in 90 to 190 cycles).
__device__ __forceinline__ void umma_lead(uint32_t leader, uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t hi,
                                          uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t.reg .b64 da, db;\n\t"
      "setp.ne.b32 p, %6, 0;\n\t"
      "setp.ne.b32 q, %0, 0;\n\t"
      "mov.b64 da, {%2, %4};\n\t"
      "mov.b64 db, {%3, %4};\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%1], da, db, %5, p;\n\t}" ::"r"(leader),
      "r"(d), "r"(a_lo), "r"(b_lo), "r"(hi), "r"(idesc), "r"(acc)
      : "memory");
}
__device__ __forceinline__ void commit_lead(uint32_t leader, uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred q;\n\t"
      "setp.ne.b32 q, %0, 0;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%1];\n\t}" ::"r"(leader),
      "r"(smem_u32(bar))
      : "memory");
}
// The TMA loads and barrier arrivals of the producer are issued the same way.
__device__ __forceinline__ void expect_lead(uint32_t leader, uint64_t* bar, uint32_t bytes) {
  asm volatile(
      "{\n\t.reg .pred q;\n\t"
      "setp.ne.b32 q, %0, 0;\n\t"
      "@q mbarrier.arrive.expect_tx.shared::cta.b64 _, [%1], %2;\n\t}" ::"r"(leader),
      "r"(smem_u32(bar)), "r"(bytes)
      : "memory");
}
__device__ __forceinline__ void tma_lead_2d(uint32_t leader, uint32_t dst, const void* desc, uint64_t* bar, int c0,
                                            int c1) {
  asm volatile(
      "{\n\t.reg .pred q;\n\t"
      "setp.ne.b32 q, %0, 0;\n\t"
      "@q cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%1], [%2, {%4, %5}], [%3];\n\t}" ::
          "r"(leader),
      "r"(dst), "l"(desc), "r"(smem_u32(bar)), "r"(c0), "r"(c1)
      : "memory");
}
__device__ __forceinline__ void tma_lead_3d(uint32_t leader, uint32_t dst, const void* desc, uint64_t* bar, int c0,
                                            int c1, int c2) {
  asm volatile(
      "{\n\t.reg .pred q;\n\t"
      "setp.ne.b32 q, %0, 0;\n\t"
      "@q cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%1], [%2, {%4, %5, %6}], "
      "[%3];\n\t}" ::"r"(leader),
      "r"(dst), "l"(desc), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2)
      : "memory");
}
// The issuing lane.  It has to come from elect.sync: under `lane == 0` the
// compiler wraps each MMA in a divergent branch (90 to 200 cycles apiece).
__device__ __forceinline__ uint32_t elect_lead() {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(r));
  return r;
}

// mbar_wait_bounded with a hint to sleep up to 20 us per try: some 300 threads
// wait at any time here, and their polling slowed the issuing warps down.
__device__ __forceinline__ bool pa_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag, unsigned int* status,
                                        unsigned int code) {
  uint64_t t0 = 0;
  while (true) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity), "r"(20000u)
        : "memory");
    if (ok) return true;
    if (*abort_flag) return false;
    const uint64_t now = globaltimer_ns();
    if (t0 == 0) t0 = now;
    if (now - t0 > DSV3_WAIT_BUDGET_NS) {
      record_error(status, code);
      *abort_flag = 1;
      return false;
    }
  }
}

// Low words of the shared-memory descriptors (128-byte swizzle, 1024 bytes
// between groups of eight rows) and the high word that both share.
constexpr uint32_t kPaDescHi = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t desc_k(uint32_t addr) { return (addr >> 4) | (1u << 16); }
template <int CHUNK>
__device__ __forceinline__ uint32_t desc_mn(uint32_t addr) {
  return (addr >> 4) | ((uint32_t)(CHUNK >> 4) << 16);
}

// Position in a ring of slots.
struct Ring {
  int n, slot = 0;
  uint32_t phase = 0;
  __device__ __forceinline__ explicit Ring(int n_) : n(n_) {}
  __device__ __forceinline__ void next() {
    if (++slot >= n) {
      slot = 0;
      phase ^= 1u;
    }
  }
};

template <int N>
__global__ void __launch_bounds__(pa_threads(N), 1) paged_attention_tc_kernel(
    const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_kv, const __grid_constant__ PagedPlan pl,
    const __grid_constant__ Ragged rg,
    int total, int H, int R, int D, float scale_log2, bf16* __restrict__ out,
    float* __restrict__ part_o, float2* __restrict__ part_ml, int4* __restrict__ rec, unsigned int* status) {
  constexpr int G = pa_groups(N), PBUF = (N + 63) / 64 * KT * 128;
  constexpr int CHUNK = KT * 128, PAIR = 2 * CHUNK;  // [KT keys x 64 columns], two of them (bytes)
  extern __shared__ __align__(1024) uint8_t smem[];
  float* mref = reinterpret_cast<float*>(smem + pl.off_misc);            // [N]
  int* lim = reinterpret_cast<int*>(mref + N);                           // [N] keys that a row sees
  float* corr = reinterpret_cast<float*>(lim + N);                       // [N] rescaling, 1 / sum, or maximum keys
  float* red = corr + N;                                                 // [N][4]
  uint64_t* pair_full = reinterpret_cast<uint64_t*>(red + 4 * N);
  uint64_t* pair_empty = pair_full + kPaMaxSlots;
  uint64_t* tail_full = pair_empty + kPaMaxSlots;
  uint64_t* tail_empty = tail_full + 2;
  uint64_t* q_full = tail_empty + 2;
  uint64_t* q_empty = q_full + 1;
  uint64_t* s_full = q_empty + 1;     // [2]
  uint64_t* p_ready = s_full + 2;
  uint64_t* pv_done = p_ready + 2;    // p_ready, pv_done, s_full, s_free: one per parity of the tile
  uint64_t* o_free = pv_done + 2;
  uint64_t* s_free = o_free + 1;      // [2]
  uint64_t* drain = s_free + 2;       // [2]
  PagedStart* start = reinterpret_cast<PagedStart*>(drain + 2);
  int2* scan = reinterpret_cast<int2*>(start + 1);           // [threads / 32]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(scan + pa_threads(N) / 32);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
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
    mbar_init(&p_ready[0], 4 * G);
    mbar_init(&p_ready[1], 4 * G);
    mbar_init(&pv_done[0], 1);
    mbar_init(&pv_done[1], 1);
    mbar_init(o_free, 4 * G);
    mbar_init(&s_free[0], 4 * G);
    mbar_init(&s_free[1], 4 * G);
    mbar_init(&drain[0], 1);
    mbar_init(&drain[1], 1);
    *abort_flag = 0;
    fence_barrier_init();
    tma_prefetch_desc(&tm_q);
    tma_prefetch_desc(&tm_kv);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, pl.tmem_cols);
    tmem_relinquish();
  }
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  paged_find<N>(rg, H, total, start, scan, status);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (start->gap | start->excess)
    paged_clear(rg, start->excess, total, (size_t)H * R * 2, reinterpret_cast<uint8_t*>(out));
  const uint32_t tmem = warp_uniform(*tmem_slot);
  const int count = warp_uniform(start->count), b_0 = warp_uniform(start->b), rt_0 = warp_uniform(start->rt),
            tile_0 = warp_uniform(start->tile);
  const uint32_t smem0 = smem_u32(smem);
  const int boxes = rg.page >= KT ? 1 : KT / rg.page;        // TMA boxes per chunk

  if (warp == 0) {
    // ------------------------------------------------------------ producer
    const uint32_t lead = elect_lead();
    Ring pr(pl.slots), tr(pl.tail ? pl.tails : 1);
    uint32_t pu = 0, tu = 0, items = 0;      // pair uses, tail uses
    bool ok = true;
    for (PagedWalk<N> w(rg, H, total, count, b_0, rt_0, tile_0); w.ok() && ok; w.next()) {
      ok = pa_wait(q_empty, (items & 1u) ^ 1u, abort_flag, status, DSV3_ERR_WAIT_EMPTY);
      if (!ok) break;
      ++items;
      expect_lead(lead, q_full, pl.nch * N * 128);
      const int qrow = w.s.tok0 * H + w.rt * N;
      for (int c = 0; c < pl.nch; ++c) tma_lead_2d(lead, smem0 + pl.off_q + c * N * 128, &tm_q, q_full, 64 * c, qrow);
      for (int t = w.t0; t < w.t1 && ok; ++t) {
        // page of this lane's box; one outside the pool reads as zeros
        int pg = rg.pool;
        const int key = t * KT + lane * (KT / boxes);
        if (lane < boxes && key < w.s.len) {
          pg = rg.table[w.b * rg.ldt + key / rg.page];
          if (pg < 0 || pg >= rg.pool) {
            record_error(status, DSV3_ERR_BOUNDS);
            pg = rg.pool;
          }
        }
        const int row = t * KT & (rg.page - 1);
        for (int m = 0; m < pl.LP + pl.tail; ++m) {
          const bool is_tail = m == pl.LP;
          const int c0 = 2 * m, nc = is_tail ? 1 : min(2, pl.nch - c0);
          const int slot = is_tail ? tr.slot : pr.slot;
          uint64_t* full = is_tail ? &tail_full[slot] : &pair_full[slot];
          const uint32_t at = smem0 + (is_tail ? pl.off_t + slot * CHUNK : slot * PAIR);
          ok = pa_wait(is_tail ? &tail_empty[slot] : &pair_empty[slot], (is_tail ? tr.phase : pr.phase) ^ 1u, abort_flag,
                       status, DSV3_ERR_WAIT_EMPTY);
          if (!ok) break;
          expect_lead(lead, full, nc * CHUNK);
          for (int i = 0; i < boxes; ++i) {
            const int p = __shfl_sync(0xffffffffu, pg, i);
            const uint32_t dst = at + i * (KT / boxes) * 128;
            tma_lead_3d(lead, dst, &tm_kv, full, 64 * c0, row, p);
            if (nc > 1) tma_lead_3d(lead, dst + CHUNK, &tm_kv, full, 64 * c0 + 64, row, p);
          }
          if (is_tail) {
            tr.next();
            ++tu;
          } else {
            pr.next();
            ++pu;
          }
        }
      }
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
    // --------------------------------------------------------- S^T = K Q^T
    if (count > 0) {
      constexpr uint32_t I_S = idesc_bf16_f32(KT, N, 0, 0);
      const uint32_t lead = elect_lead();
      Ring sr(pl.slots), tr(pl.tail ? pl.tails : 1);
      uint32_t g = 0, items = 0;
      bool ok = true, issued = false;
      for (PagedWalk<N> w(rg, H, total, count, b_0, rt_0, tile_0); w.ok() && ok; w.next(), ++items) {
        ok = pa_wait(q_full, items & 1u, abort_flag, status, DSV3_ERR_WAIT_FULL);
        for (int t = w.t0; t < w.t1 && ok; ++t, ++g) {
          // two S^T buffers: this one's last tile has been read
          if (g > 1 && !pa_wait(&s_free[g & 1u], ((g >> 1) & 1u) ^ 1u, abort_flag, status, DSV3_ERR_WAIT_TMEM)) {
            ok = false;
            break;
          }
          const uint32_t d = tmem + (g & 1u) * N;
          uint32_t acc = 0, q_lo = desc_k(smem0 + pl.off_q);
          for (int m = 0; m < pl.LP + pl.tail; ++m) {
            const bool is_tail = m == pl.LP;
            const int slot = is_tail ? tr.slot : sr.slot;
            if (!pa_wait(is_tail ? &tail_full[slot] : &pair_full[slot], is_tail ? tr.phase : sr.phase, abort_flag,
                         status, DSV3_ERR_WAIT_FULL)) {
              ok = false;
              break;
            }
            tc_fence_after();
            uint32_t a_lo = desc_k(smem0 + (is_tail ? pl.off_t + slot * CHUNK : slot * PAIR));
            // 64-column chunks of this pair: whole ones as four MMAs, what is left
            // of the row as its steps of 16
            const int left = min(128, D - 128 * m);
            for (int c = 0; c < left / 64; ++c) {
              umma_lead(lead, d, a_lo, q_lo, kPaDescHi, I_S, acc);
#pragma unroll
              for (int kk = 1; kk < 4; ++kk) umma_lead(lead, d, a_lo + 2 * kk, q_lo + 2 * kk, kPaDescHi, I_S, 1u);
              acc = 1;
              a_lo += CHUNK >> 4;
              q_lo += N * 128 >> 4;
            }
#pragma unroll 1
            for (int k = 0; k < left % 64; k += 16) {
              umma_lead(lead, d, a_lo + k / 8, q_lo + k / 8, kPaDescHi, I_S, acc);
              acc = 1;
            }
            issued = true;
            if (is_tail) {
              commit_lead(lead, &tail_empty[slot]);
              tr.next();
            } else {
              sr.next();
            }
          }
          if (ok) commit_lead(lead, &s_full[g & 1u]);
        }
        if (ok) commit_lead(lead, q_empty);
      }
      if (issued) {   // no MMA may still write TMEM when it is freed
        commit_lead(lead, drain);
        mbar_wait_bounded(drain, 0, nullptr, status, DSV3_ERR_WAIT_TMEM);
      }
      __syncwarp();
    }
  } else if (warp == 2 + 4 * G) {
    // ------------------------------------------------------ O^T += V^T P^T
    // A warp of its own: S^T of a later tile and PV of this one become ready in
    // either order, and neither waits behind the other.
    if (count > 0) {
      constexpr uint32_t I_O = idesc_bf16_f32(128, N, 1, 1);     // both read MN-major
      const uint32_t lead = elect_lead();
      Ring vr(pl.slots);
      uint32_t g = 0, items = 0;
      bool ok = true, issued = false;
      for (PagedWalk<N> w(rg, H, total, count, b_0, rt_0, tile_0); w.ok() && ok; w.next(), ++items) {
        for (int t = w.t0; t < w.t1 && ok; ++t, ++g) {
          ok = pa_wait(&p_ready[g & 1u], (g >> 1) & 1u, abort_flag, status, DSV3_ERR_WAIT_FULL);
          // the last item's O^T has been read out
          if (ok && t == w.t0 && items > 0)
            ok = pa_wait(o_free, (items - 1) & 1u, abort_flag, status, DSV3_ERR_WAIT_TMEM);
          if (!ok) break;
          tc_fence_after();
          const uint32_t acc = t > w.t0;
          const uint32_t p_lo = desc_mn<CHUNK>(smem0 + pl.off_p + (g & 1u) * (pl.pbufs - 1) * PBUF);
          for (int m = 0; m < pl.LP; ++m) {
            const uint32_t v_lo = desc_mn<CHUNK>(smem0 + vr.slot * PAIR), d = tmem + (2 + m) * N;
            umma_lead(lead, d, v_lo, p_lo, kPaDescHi, I_O, acc);
#pragma unroll
            for (int kk = 1; kk < KT / 16; ++kk)
              umma_lead(lead, d, v_lo + 128 * kk, p_lo + 128 * kk, kPaDescHi, I_O, 1u);
            commit_lead(lead, &pair_empty[vr.slot]);
            vr.next();
          }
          commit_lead(lead, &pv_done[g & 1u]);
          issued = true;
        }
      }
      if (issued) {
        commit_lead(lead, drain + 1);
        mbar_wait_bounded(drain + 1, 0, nullptr, status, DSV3_ERR_WAIT_TMEM);
      }
      __syncwarp();
    }
  } else {
    // ---------------------------------------------------- softmax / epilogue
    const int wg = (warp - 2) >> 2;              // its rows are wg * NH ..
    const int quarter = warp & 3;                  // TMEM lanes 32 * quarter ..
    // A key tile of 64 fills 16 TMEM lanes of each quarter; the two half warps
    // then take different columns of the same 16 keys.
    constexpr int NH = N / G;                      // rows of a warpgroup
    constexpr int NC = NH / 2;                     // rows of a thread
    constexpr int L = 16;                          // lanes that hold different keys
    const int side = lane >> 4;
    const int key = quarter * L + (lane & (L - 1));
    const int ht = (warp - 2 - 4 * wg) * 32 + lane;
    const uint32_t lane_base = (uint32_t)(quarter * 32) << 16;
    const int col0 = wg * NH + side * NC;
    float* myred = red + wg * NH * 4;            // [NH][4]
    float4* mref4 = reinterpret_cast<float4*>(mref + col0);
    const int4* lim4 = reinterpret_cast<const int4*>(lim + col0);
    uint32_t g = 0;
    int4 my_rec = make_int4(-1, 0, 0, 0);
    for (PagedWalk<N> w(rg, H, total, count, b_0, rt_0, tile_0); w.ok(); w.next()) {
      const int base = w.s.len - w.s.n;
      const int nr = min(N, w.s.rows - w.rt * N);
      wg_sync(wg);                             // the last item's references are read
      if (ht < NH) {
        const int n = wg * NH + ht;
        reinterpret_cast<uint32_t*>(corr)[n] = 0u;
        lim[n] = n < nr ? base + (w.rt * N + n) / H + 1 : 0;
      }
      wg_sync(wg);
      const int seen_by_all = base + (w.rt * N) / H + 1;      // keys that every row sees
      float l[NC];
#pragma unroll
      for (int c = 0; c < NC; ++c) l[c] = 0.f;
      for (int t = w.t0; t < w.t1; ++t, ++g) {
        pa_wait(&s_full[g & 1u], (g >> 1) & 1u, abort_flag, status, DSV3_ERR_WAIT_TMEM);
        tc_fence_after();
        uint32_t sr[NC];
        tmem_ld_half<NC, NC>(tmem + lane_base + (g & 1u) * N + wg * NH, sr);
        tmem_ld_wait();
        const int pos = t * KT + key;
        if (t * KT + KT > seen_by_all) {
#pragma unroll
          for (int c = 0; c < NC; c += 4) {
            const int4 k4 = lim4[c / 4];
            if (pos >= k4.x) sr[c] = 0xff800000u;
            if (pos >= k4.y) sr[c + 1] = 0xff800000u;
            if (pos >= k4.z) sr[c + 2] = 0xff800000u;
            if (pos >= k4.w) sr[c + 3] = 0xff800000u;
          }
        }
        // The first references are the scores of the tile's first key plus 12:
        // scores up to 2^20 times its weight pass without a move, and weights
        // lose nothing by starting at 2^-12 (a maximum over the tile first cost
        // 1,700 to 8,000 cycles per item).  A row that does not see that key
        // sees none of this tile.
        if (t == w.t0) {
          if (key == 0) {
#pragma unroll
            for (int c = 0; c < NC; c += 4) {
              const int4 k4 = lim4[c / 4];
              float4 m4;
              m4.x = k4.x > 0 ? fmaxf(fmaf(__uint_as_float(sr[c]), scale_log2, kPaLead), kPaUnset) : kPaNever;
              m4.y = k4.y > 0 ? fmaxf(fmaf(__uint_as_float(sr[c + 1]), scale_log2, kPaLead), kPaUnset) : kPaNever;
              m4.z = k4.z > 0 ? fmaxf(fmaf(__uint_as_float(sr[c + 2]), scale_log2, kPaLead), kPaUnset) : kPaNever;
              m4.w = k4.w > 0 ? fmaxf(fmaf(__uint_as_float(sr[c + 3]), scale_log2, kPaLead), kPaUnset) : kPaNever;
              mref4[c / 4] = m4;
            }
          }
          wg_sync(wg);
        }
        // p = 2^(s - m) at the present references; where one is passed by more
        // than 2^8 the warpgroup moves them and computes p again
        uint32_t pk[NC / 2];
        for (int attempt = 0;; ++attempt) {
          float over = -INFINITY;
#pragma unroll
          for (int c = 0; c < NC; c += 4) {
            const float4 m4 = mref4[c / 4];
            const float d0 = fmaf(__uint_as_float(sr[c]), scale_log2, -m4.x);
            const float d1 = fmaf(__uint_as_float(sr[c + 1]), scale_log2, -m4.y);
            const float d2 = fmaf(__uint_as_float(sr[c + 2]), scale_log2, -m4.z);
            const float d3 = fmaf(__uint_as_float(sr[c + 3]), scale_log2, -m4.w);
            over = fmaxf(fmaxf(over, fmaxf(d0, d1)), fmaxf(d2, d3));
            pk[c / 2] = pack_bf16x2(ex2_approx(d0), ex2_approx(d1));
            pk[c / 2 + 1] = pack_bf16x2(ex2_approx(d2), ex2_approx(d3));
          }
          if (!wg_any(wg, over > 8.f) || attempt == 1) break;
          // column maxima of the tile: S^T is read again in slices, so that this
          // rare path is a short loop (unrolled over registers it ran from
          // instruction-cache misses, 14,000 cycles)
          constexpr int W = NC < 16 ? NC : 16;
#pragma unroll 1
          for (int c0 = 0; c0 < NC; c0 += W) {
            uint32_t u[W];
            float v[W];
            tmem_ld_half<NC, W>(tmem + lane_base + (g & 1u) * N + wg * NH + c0, u);
            tmem_ld_wait();
#pragma unroll
            for (int c = 0; c < W; ++c)
              v[c] = pos < lim[col0 + c0 + c] ? __uint_as_float(u[c]) * scale_log2 : -INFINITY;
            const float top = fold_columns<W, L>(v, lane, [](float x, float y) { return fmaxf(x, y); });
            if (lane % (L / W) == 0)
              atomicMax(reinterpret_cast<unsigned int*>(corr) + col0 + c0 + (lane & (L - 1)) * W / L, float_key(top));
          }
          wg_sync(wg);
          if (ht < NH) {
            const int n = wg * NH + ht;
            const float old = mref[n], top = float_unkey(reinterpret_cast<uint32_t*>(corr)[n]);
            const float now = fmaxf(old, top);
            mref[n] = now;
            corr[n] = ex2_approx(old - now);
          }
          wg_sync(wg);
#pragma unroll
          for (int c = 0; c < NC; c += 4) {
            const float4 f = *reinterpret_cast<const float4*>(corr + col0 + c);
            l[c] *= f.x;
            l[c + 1] *= f.y;
            l[c + 2] *= f.z;
            l[c + 3] *= f.w;
          }
          if (t > w.t0) {   // the first tile of an item overwrites O^T
            pa_wait(&pv_done[(g - 1) & 1u], ((g - 1) >> 1) & 1u, abort_flag, status, DSV3_ERR_WAIT_TMEM);
            tc_fence_after();
#pragma unroll 1
            for (int i = 0; i < pl.LP * (NH / 8); ++i) {
              const int m = i / (NH / 8), c = wg * NH + i % (NH / 8) * 8;
              uint32_t o[8];
              tmem_ld8(tmem + lane_base + (2 + m) * N + c, o);
              tmem_ld_wait();
#pragma unroll
              for (int j = 0; j < 8; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * corr[c + j]);
              tmem_st8(tmem + lane_base + (2 + m) * N + c, o);
            }
            tmem_st_wait();
          }
          wg_sync(wg);
          if (ht < NH) reinterpret_cast<uint32_t*>(corr)[wg * NH + ht] = 0u;
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&s_free[g & 1u]);
        // the tile that last used this P buffer is through
        if (g >= (uint32_t)pl.pbufs) {
          const uint32_t u = g - pl.pbufs;
          pa_wait(&pv_done[u & 1u], (u >> 1) & 1u, abort_flag, status, DSV3_ERR_WAIT_TMEM);
        }
        uint8_t* prow = smem + pl.off_p + (g & 1u) * (pl.pbufs - 1) * PBUF + key * 128;
        if constexpr (NC == 4) {
          *reinterpret_cast<uint2*>(prow + (((col0 >> 3) ^ (key & 7)) << 4) + (col0 & 4) * 2) = make_uint2(pk[0], pk[1]);
        } else {
#pragma unroll
          for (int c = 0; c < NC; c += 8) {
            const int n = col0 + c;
            *reinterpret_cast<uint4*>(prow + (n >> 6) * CHUNK + ((((n & 63) >> 3) ^ (key & 7)) << 4)) =
                make_uint4(pk[c / 2], pk[c / 2 + 1], pk[c / 2 + 2], pk[c / 2 + 3]);
          }
        }
        // rows of the pages past the cached length hold anything: zero them, so
        // that their zero weights do not meet an infinity or NaN
        if (t * KT + KT > w.s.len && pos >= w.s.len) {
          for (int c = wg * 2 + side; c < 2 * pl.LP; c += 2 * G) {
            const int slot = (g * pl.LP + (c >> 1)) % pl.slots;
            uint4* z = reinterpret_cast<uint4*>(smem + slot * PAIR + (c & 1) * CHUNK + key * 128);
#pragma unroll
            for (int i = 0; i < 8; ++i) z[(i + lane) & 7] = make_uint4(0, 0, 0, 0);   // spread over the banks
          }
        }
        fence_proxy_async_smem();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_ready[g & 1u]);
        // row sums over the rounded weights, while the tensor core runs
#pragma unroll
        for (int c = 0; c < NC; c += 2) {
          l[c] += __uint_as_float(pk[c / 2] << 16);
          l[c + 1] += __uint_as_float(pk[c / 2] & 0xffff0000u);
        }
      }
      // ---- item epilogue
      pa_wait(&pv_done[(g - 1) & 1u], ((g - 1) >> 1) & 1u, abort_flag, status, DSV3_ERR_WAIT_TMEM);
      tc_fence_after();
      const bool whole = w.t0 == 0 && w.t1 == w.nt;
      const int slot = 2 * blockIdx.x + (w.t0 == 0 ? 1 : 0);
      const long long row0 = (long long)w.s.tok0 * H + (long long)w.rt * N;
      if (!whole && w.t0 == 0) {
        const int s0 = start->first + (count - w.left);
        my_rec = make_int4((int)row0, nr, (s0 + w.nt - 1) / start->share, 0);
      }
      constexpr int WL = NC < L ? NC : L;            // rows of a half warp folded at a time
#pragma unroll
      for (int c0 = 0; c0 < NC; c0 += WL) {
        const float v = fold_columns<WL, L>(*reinterpret_cast<float(*)[WL]>(&l[c0]), lane,
                                            [](float x, float y) { return x + y; });
        if (c0 > 0) wg_sync(wg);               // the last columns are read
        if (lane % (L / WL) == 0) myred[(side * WL + (lane & (L - 1)) * WL / L) * 4 + (warp - 2 - 4 * wg)] = v;
        wg_sync(wg);
        if (ht < 2 * WL) {
          const float4 r4 = *reinterpret_cast<const float4*>(myred + ht * 4);
          const float sum = (r4.x + r4.y) + (r4.z + r4.w);
          const int n = wg * NH + ht / WL * NC + c0 + ht % WL;
          if (!whole) part_ml[(size_t)slot * N + n] = make_float2(mref[n], sum);
          corr[n] = !whole ? 1.f : (sum > 0.f ? 1.f / sum : (sum == sum ? 0.f : sum));
        }
      }
      wg_sync(wg);
      constexpr int W = NH < 32 ? NH : 32;
      // O^T out: a thread holds one latent column of W rows; the warp turns eight
      // rows (four of fp32 partials) at a time into 16-byte stores in 512 bytes of
      // the idle P buffer (4-byte stores from registers took 24 cycles each,
      // 14,000 per item of 128 rows)
      uint8_t* stage = smem + pl.off_p + (warp - 2) * 512;
#pragma unroll 1
      for (int i = 0; i < pl.LP * (NH / W); ++i) {
        const int m = i / (NH / W), n0 = wg * NH + i % (NH / W) * W;
        const int r0 = 128 * m + quarter * 32;
        if (n0 >= nr || r0 >= R) continue;
        uint32_t o[W];
        tmem_ld_cols<W>(tmem + lane_base + (2 + m) * N + n0, o);
        tmem_ld_wait();
        if (whole) {
          const int row = lane >> 2, r = r0 + (lane & 3) * 8;
#pragma unroll
          for (int j = 0; j < W; j += 8) {
#pragma unroll
            for (int k = 0; k < 8; ++k)
              *reinterpret_cast<bf16*>(stage + k * 64 + lane * 2) =
                  __float2bfloat16(__uint_as_float(o[j + k]) * corr[n0 + j + k]);
            __syncwarp();
            const uint4 v = *reinterpret_cast<const uint4*>(stage + lane * 16);
            if (n0 + j + row < nr && r < R)
              *reinterpret_cast<uint4*>(out + (size_t)(row0 + n0 + j + row) * R + r) = v;
            __syncwarp();
          }
        } else {
          const int row = lane >> 3, r = r0 + (lane & 7) * 4;
#pragma unroll
          for (int j = 0; j < W; j += 4) {
#pragma unroll
            for (int k = 0; k < 4; ++k) *reinterpret_cast<uint32_t*>(stage + k * 128 + lane * 4) = o[j + k];
            __syncwarp();
            const uint4 v = *reinterpret_cast<const uint4*>(stage + lane * 16);
            if (n0 + j + row < nr && r < R)
              *reinterpret_cast<uint4*>(part_o + ((size_t)slot * N + n0 + j + row) * R + r) = v;
            __syncwarp();
          }
        }
      }
      // no warpgroup writes the next item's P over another's stage
      asm volatile("barrier.cta.sync 8, %0;" ::"n"(128 * G) : "memory");
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

// Joins the partials of row tiles that were cut.  rec[g] describes the one that
// begins in share g and goes on: part 0 is slot 2 g + 1, part i slot 2 (g + i).
// The parts are added in a fixed order.  Where shares outnumber row tiles (few
// rows over long contexts, FEW) a CTA joins one row, its threads split over the
// parts; else a warp joins one row, of two or three parts as a rule.
template <int N, bool FEW>
__global__ void __launch_bounds__(FEW ? 512 : 256) paged_merge_kernel(const float* __restrict__ part_o,
                                                                    const float2* __restrict__ part_ml,
                                                                    const int4* __restrict__ rec, int shares, int R,
                                                                    bf16* __restrict__ out) {
  __shared__ int s_g;
  __shared__ float s_m[32];
  __shared__ float4 s_acc[FEW ? 512 : 1];
  __shared__ float s_sum[FEW ? 256 : 1];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  int g = blockIdx.x, n;
  if constexpr (FEW) {
    // the blockIdx.x-th row tile that was cut
    if (warp == 0) {
      int skip = blockIdx.x, found = -1;
      for (int i = 0; i < shares && found < 0; i += 32) {
        const unsigned hit = __ballot_sync(0xffffffffu, i + lane < shares && rec[min(i + lane, shares - 1)].x >= 0);
        const int c = __popc(hit);
        if (skip < c) {
          const bool me = (hit >> lane & 1) && __popc(hit & ((1u << lane) - 1)) == skip;
          found = i + __ffs(__ballot_sync(0xffffffffu, me)) - 1;
        }
        skip -= c;
      }
      if (lane == 0) s_g = found;
    }
    __syncthreads();
    g = s_g;
    if (g < 0) return;
    n = blockIdx.y;
  } else {
    n = blockIdx.y * 8 + warp;
  }
  const int4 rc = rec[g];
  if (rc.x < 0 || n >= rc.y) return;
  const int parts = rc.z - g + 1;
  auto at = [&](int i) { return (size_t)(i ? 2 * (g + i) : 2 * g + 1) * N + n; };
  float M = -INFINITY;
  for (int i = FEW ? tid : lane; i < parts; i += FEW ? 512 : 32) {
    const float2 ml = part_ml[at(i)];
    if (ml.y > 0.f) M = fmaxf(M, ml.x);
  }
  M = warp_max(M);
  if constexpr (!FEW) {
    // a lane holds up to 4 x 4 latent columns: one pass over the parts, all loads
    // of a part in flight together
    float sum = 0.f;
    float4 acc[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) acc[c] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 2
    for (int i = 0; i < parts; ++i) {
      const size_t k = at(i);
      const float2 ml = part_ml[k];
      float4 o[4];
#pragma unroll
      for (int c = 0; c < 4; ++c)
        if (lane * 4 + 128 * c < R) o[c] = *reinterpret_cast<const float4*>(part_o + k * R + lane * 4 + 128 * c);
      const float wgt = ml.y == 0.f ? 0.f : ex2_approx(ml.x - M);
      sum += ml.y * wgt;
      if (wgt != 0.f) {
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          acc[c].x += o[c].x * wgt;
          acc[c].y += o[c].y * wgt;
          acc[c].z += o[c].z * wgt;
          acc[c].w += o[c].w * wgt;
        }
      }
    }
    const float inv = sum > 0.f ? 1.f / sum : (sum == sum ? 0.f : sum);
#pragma unroll
    for (int c = 0; c < 4; ++c)
      if (lane * 4 + 128 * c < R)
        *reinterpret_cast<uint2*>(out + (size_t)(rc.x + n) * R + lane * 4 + 128 * c) =
            make_uint2(pack_bf16x2(acc[c].x * inv, acc[c].y * inv), pack_bf16x2(acc[c].z * inv, acc[c].w * inv));
  } else {
    // R / 4 threads of a part hold four latent columns each; the parts of a thread
    // group are added first, then the groups in order
    if (lane == 0) s_m[warp] = M;
    __syncthreads();
    M = warp_max(s_m[lane & 15]);
    const int tpp = R / 4, groups = 512 / tpp, grp = tid / tpp, r = (tid % tpp) * 4;
    float sum = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    if (grp < groups) {
#pragma unroll 4
      for (int i = grp; i < parts; i += groups) {
        const size_t k = at(i);
        const float2 ml = part_ml[k];
        const float4 o = *reinterpret_cast<const float4*>(part_o + k * R + r);
        const float wgt = ml.y == 0.f ? 0.f : ex2_approx(ml.x - M);
        sum += ml.y * wgt;
        if (wgt != 0.f) {
          acc.x += o.x * wgt;
          acc.y += o.y * wgt;
          acc.z += o.z * wgt;
          acc.w += o.w * wgt;
        }
      }
    }
    s_acc[tid] = acc;
    if (tid % tpp == 0 && grp < groups) s_sum[grp] = sum;
    __syncthreads();
    if (grp > 0) return;
    for (int i = 1; i < groups; ++i) {
      const float4 o = s_acc[i * tpp + tid];
      acc.x += o.x;
      acc.y += o.y;
      acc.z += o.z;
      acc.w += o.w;
      sum += s_sum[i];
    }
    const float inv = sum > 0.f ? 1.f / sum : (sum == sum ? 0.f : sum);
    *reinterpret_cast<uint2*>(out + (size_t)(rc.x + n) * R + r) =
        make_uint2(pack_bf16x2(acc.x * inv, acc.y * inv), pack_bf16x2(acc.z * inv, acc.w * inv));
  }
}
