// Beam search: the choice of the next beams and the reordering of their cache.
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include <tuple>

#include "common.cuh"
#include "status.h"

namespace dsv3 {

namespace {

typedef __nv_bfloat16 bf16;

constexpr int kMaxBeams = 32;
constexpr int kSelThreads = 256;
constexpr int kSelPer = 32;                        // logits per thread
constexpr int kSelSeg = kSelThreads * kSelPer;     // logits per CTA

// Order-preserving map of a float to an unsigned key (larger float, larger
// key); 0 stands for "no candidate" and lies below the key of -inf.
__device__ __forceinline__ uint32_t order_key(float x) {
  const uint32_t u = __float_as_uint(x);
  return u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) {
  return __uint_as_float(k ^ ((k >> 31) ? 0x80000000u : 0xffffffffu));
}

// A logit as the selection sees it: NaN counts as -inf, +inf as the largest
// finite float, so that the log-sum-exp of a row is always defined.
__device__ __forceinline__ float clean_logit(float x) { return fminf(fmaxf(x, -INFINITY), 3.402823466e38f); }
__device__ __forceinline__ float load_logit(const float* p) { return clean_logit(*p); }
__device__ __forceinline__ float load_logit(const bf16* p) { return clean_logit(__bfloat162float(*p)); }

// Top `k` of (key, index) pairs held by a warp, `n` per lane: larger key first, ties to the lower index.
// Lane 0 emits through `put(rank, key, index)`.
template <int N, typename Put>
__device__ __forceinline__ void warp_top(uint32_t (&key)[N], const uint32_t (&idx)[N], int k, int lane, Put put) {
  for (int j = 0; j < k; ++j) {
    uint32_t bk = 0, bi = 0xffffffffu;
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (key[i] > bk || (key[i] == bk && idx[i] < bi)) {
        bk = key[i];
        bi = idx[i];
      }
    const uint32_t top = __reduce_max_sync(0xffffffffu, bk);
    const uint32_t at = __reduce_min_sync(0xffffffffu, bk == top ? bi : 0xffffffffu);
    if (lane == 0) put(j, top, at);
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (idx[i] == at) key[i] = 0;
  }
}

// One CTA per (segment of a row): maximum, sum of exponentials and the `k` largest logits.
template <typename T>
__global__ void __launch_bounds__(kSelThreads) beam_scan_kernel(const T* __restrict__ logits, long ldb, long ldk, int K,
                                                                int V, int k, const bool* __restrict__ finished,
                                                                float2* __restrict__ stat,
                                                                uint2* __restrict__ cand) {
  const int row = blockIdx.y, seg = blockIdx.x, nseg = gridDim.x;
  if (finished != nullptr && finished[row]) return;
  const T* x = logits + (row / K) * ldb + (row % K) * ldk;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  __shared__ float red[2][kSelThreads / 32];
  __shared__ uint2 top_s[kSelThreads / 32][kMaxBeams];
  uint32_t key[kSelPer], idx[kSelPer];
  float mx = -3.402823466e38f;
#pragma unroll
  for (int i = 0; i < kSelPer; ++i) {
    const int v = seg * kSelSeg + i * kSelThreads + tid;
    idx[i] = v < V ? v : 0xfffffffeu;
    const float f = v < V ? load_logit(x + v) : -INFINITY;
    key[i] = v < V ? order_key(f) : 0;
    mx = fmaxf(mx, f);
  }
  mx = warp_max(mx);
  if (lane == 0) red[0][warp] = mx;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kSelThreads / 32; ++i) mx = fmaxf(mx, red[0][i]);
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < kSelPer; ++i) s += key[i] ? __expf(key_value(key[i]) - mx) : 0.f;
  s = warp_sum(s);
  if (lane == 0) red[1][warp] = s;
  warp_top(key, idx, k, lane, [&](int j, uint32_t kk, uint32_t ii) { top_s[warp][j] = make_uint2(kk, ii); });
  __syncthreads();
  if (warp == 0) {
    uint32_t k2[kMaxBeams / 4], i2[kMaxBeams / 4];
#pragma unroll
    for (int i = 0; i < kMaxBeams / 4; ++i) {
      const int e = i * 32 + lane, w = e / k;
      k2[i] = w < kSelThreads / 32 ? top_s[w][e % k].x : 0;
      i2[i] = w < kSelThreads / 32 ? top_s[w][e % k].y : 0xfffffffeu;
    }
    uint2* o = cand + ((size_t)row * nseg + seg) * k;
    warp_top(k2, i2, k, lane, [&](int j, uint32_t kk, uint32_t ii) { o[j] = make_uint2(kk, ii); });
    if (lane == 0) {
      float t = 0.f;
      for (int i = 0; i < kSelThreads / 32; ++i) t += red[1][i];
      stat[(size_t)row * nseg + seg] = make_float2(mx, t);
    }
  }
}

// One CTA per batch entry: log-sum-exp of its beams, then the K best candidates.
__global__ void __launch_bounds__(256) beam_pick_kernel(const float2* __restrict__ stat, const uint2* __restrict__ cand,
                                                        const float* __restrict__ scores,
                                                        const bool* __restrict__ finished, int K, int V, int nseg,
                                                        int eos, float* __restrict__ o_score, int* __restrict__ o_parent,
                                                        int* __restrict__ o_token, bool* __restrict__ o_done) {
  const int b = blockIdx.x, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  __shared__ float s_max[kMaxBeams], s_log[kMaxBeams];
  __shared__ uint32_t s_key[8], s_at[8];
  for (int r = warp; r < K; r += 8) {
    const size_t row = (size_t)b * K + r;
    float m = -3.402823466e38f, s = 0.f;
    if (!(finished != nullptr && finished[row])) {
      for (int i = lane; i < nseg; i += 32) m = fmaxf(m, stat[row * nseg + i].x);
      m = warp_max(m);
      for (int i = lane; i < nseg; i += 32) s += stat[row * nseg + i].y * expf(stat[row * nseg + i].x - m);
      s = warp_sum(s);
    }
    if (lane == 0) {
      s_max[r] = m;
      s_log[r] = logf(s);
    }
  }
  __syncthreads();
  const int per = nseg * K;       // candidates per beam
  uint32_t last_key = 0xffffffffu, last_at = 0;
  for (int j = 0; j < K; ++j) {
    // best candidate after (last_key, last_at) in the order (key descending, flat index ascending)
    uint32_t bk = 0, bi = 0xffffffffu;
    for (int c = tid; c < K * per; c += 256) {
      const int r = c / per, i = c % per;
      const size_t row = (size_t)b * K + r;
      const float sc = scores[row];
      uint32_t v;
      float val;
      if (finished != nullptr && finished[row]) {
        if (i >= K) continue;
        v = i == 0 ? eos : (i - 1 < eos ? i - 1 : i);
        val = i == 0 ? sc : -INFINITY;
      } else if (!(sc > -INFINITY) || s_log[r] == -INFINITY) {
        if (i >= K) continue;
        v = i;
        val = -INFINITY;
      } else {
        const uint2 e = cand[row * per + i];
        if (e.x == 0) continue;
        v = e.y;
        val = sc + ((key_value(e.x) - s_max[r]) - s_log[r]);
      }
      if (v >= V) continue;
      const uint32_t k2 = order_key(val), at = r * V + v;
      const bool after = k2 < last_key || (k2 == last_key && at > last_at);
      if (after && (k2 > bk || (k2 == bk && at < bi))) {
        bk = k2;
        bi = at;
      }
    }
    const uint32_t wk = __reduce_max_sync(0xffffffffu, bk);
    const uint32_t wi = __reduce_min_sync(0xffffffffu, bk == wk ? bi : 0xffffffffu);
    if (lane == 0) {
      s_key[warp] = wk;
      s_at[warp] = wi;
    }
    __syncthreads();
    last_key = 0;
    last_at = 0xffffffffu;
    for (int w = 0; w < 8; ++w)
      if (s_key[w] > last_key || (s_key[w] == last_key && s_at[w] < last_at)) {
        last_key = s_key[w];
        last_at = s_at[w];
      }
    __syncthreads();
    if (tid == 0) {
      const int p = last_at / V, v = last_at % V;
      o_score[b * K + j] = key_value(last_key);
      o_parent[b * K + j] = p;
      o_token[b * K + j] = v;
      o_done[b * K + j] = (finished != nullptr && finished[(size_t)b * K + p]) || v == eos;
    }
  }
}

// Grid (part, layer, group): part < parts copies its share of the page that is
// being filled, part == parts (layer 0 only) writes the group's new table rows.
__global__ void __launch_bounds__(256) beam_reorder_kernel(uint4* __restrict__ pages, long ld_layer, long ld_page,
                                                           int row16, int page, int pool, const int* __restrict__ table,
                                                           long ldt, int cols, const int* __restrict__ parents, int K,
                                                           const int* __restrict__ lens, int* __restrict__ out,
                                                           int parts, unsigned int* status) {
  __shared__ int s_src[kMaxBeams], s_dst[kMaxBeams], s_par[kMaxBeams], s_n;
  const int b = blockIdx.z, layer = blockIdx.y, part = blockIdx.x;
  if (part == parts && layer > 0) return;
  const int len = lens[b];
  const int col = len / page, rem = len % page;
  if (part < parts && rem == 0) return;
  const int* tb = table + (size_t)b * K * ldt;
  if (threadIdx.x < 32) {
    const int lane = threadIdx.x;
    int p = lane < K ? parents[b * K + lane] : -1;
    bool bad = lane < K && (p < 0 || p >= K);
    if (bad) p = lane;
    int cur = lane < K && col < cols ? tb[lane * ldt + col] : -1;
    if (lane < K && rem > 0 && (cur < 0 || cur >= pool)) bad = true;
    if (bad) record_error(status, DSV3_ERR_BOUNDS);
    const bool ok = !__any_sync(0xffffffffu, lane < K && rem > 0 && (cur < 0 || cur >= pool));
    // children of the same parent; the first keeps its page, the j-th other takes the j-th childless beam's
    const unsigned mine = __match_any_sync(0xffffffffu, p) & (K == 32 ? 0xffffffffu : (1u << K) - 1);
    const bool again = lane < K && (mine & ((1u << lane) - 1)) != 0;
    unsigned has = __reduce_or_sync(0xffffffffu, lane < K ? 1u << p : 0u);
    const unsigned dead = ~has & (K == 32 ? 0xffffffffu : (1u << K) - 1);
    const unsigned agains = __ballot_sync(0xffffffffu, again);
    const int j = __popc(agains & ((1u << lane) - 1));
    const int from = p < 0 ? 0 : p;
    const int src = __shfl_sync(0xffffffffu, cur, from);
    const int spare = again ? __fns(dead, 0, j + 1) : from;
    const int dst = __shfl_sync(0xffffffffu, cur, spare);
    if (lane < K) {
      s_par[lane] = p;
      s_dst[lane] = dst;
    }
    __syncwarp();
    if (part < parts) {
      if (again) {
        s_src[j] = src;
        s_dst[j] = dst;
      }
      if (lane == 0) s_n = ok ? __popc(agains) : 0;
    }
  }
  __syncthreads();
  if (part == parts) {
    int* ob = out + (size_t)b * K * cols;
    for (int i = threadIdx.x; i < K * cols; i += 256) {
      const int r = i / cols, c = i % cols;
      int v;
      if (c < col) v = tb[s_par[r] * ldt + c];
      else if (c == col && rem > 0) v = s_dst[r];
      else v = tb[r * ldt + c];
      ob[i] = v;
    }
    return;
  }
  const int n16 = rem * row16;
  for (int d = 0; d < s_n; ++d) {
    const uint4* src = pages + layer * ld_layer + s_src[d] * ld_page;
    uint4* dst = pages + layer * ld_layer + s_dst[d] * ld_page;
    for (int i = part * 256 + threadIdx.x; i < n16; i += parts * 256) dst[i] = src[i];
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
  TORCH_CHECK(K >= 1 && K <= kMaxBeams && V >= K && K * V < (1ll << 31), op,
              ": 1 to 32 beams, at least as many tokens as beams and K * V below 2^31");
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
  TORCH_CHECK(B * K <= 65535, op, ": too many rows");
  const at::cuda::CUDAGuard guard(logits.device());
  auto st = at::cuda::getCurrentCUDAStream();
  auto iopt = scores.options().dtype(at::kInt);
  auto o_score = at::empty({B, K}, scores.options()), o_parent = at::empty({B, K}, iopt),
       o_token = at::empty({B, K}, iopt), o_done = at::empty({B, K}, scores.options().dtype(at::kBool));
  if (B == 0) return {o_score, o_parent, o_token, o_done};
  const int nseg = (int)((V + kSelSeg - 1) / kSelSeg);
  auto work = at::empty({B * K * nseg * (1 + K) * 2}, scores.options());
  float2* stat = reinterpret_cast<float2*>(work.data_ptr());
  uint2* cand = reinterpret_cast<uint2*>(stat + B * K * nseg);
  const dim3 grid(nseg, (unsigned)(B * K));
  if (logits.scalar_type() == at::kFloat)
    beam_scan_kernel<float><<<grid, kSelThreads, 0, st>>>(logits.data_ptr<float>(), logits.stride(0),
                                                          logits.stride(1), (int)K, (int)V, (int)K, done, stat, cand);
  else
    beam_scan_kernel<bf16><<<grid, kSelThreads, 0, st>>>(reinterpret_cast<const bf16*>(logits.data_ptr()),
                                                         logits.stride(0), logits.stride(1), (int)K, (int)V, (int)K,
                                                         done, stat, cand);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  beam_pick_kernel<<<(int)B, 256, 0, st>>>(stat, cand, scores.data_ptr<float>(), done, (int)K, (int)V, nseg, (int)eos,
                                           o_score.data_ptr<float>(), o_parent.data_ptr<int>(),
                                           o_token.data_ptr<int>(), o_done.data_ptr<bool>());
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  return {o_score, o_parent, o_token, o_done};
}

at::Tensor beam_reorder(at::Tensor& pages, const at::Tensor& table, const at::Tensor& parents,
                        const at::Tensor& lens) {
  const char* op = "beam_reorder";
  TORCH_CHECK(pages.is_cuda() && pages.dim() == 4 && pages.stride(3) == 1 && pages.stride(2) == pages.size(3), op,
              ": pages must be a CUDA tensor [layers, pool, page, width] with contiguous pages");
  const int64_t es = pages.element_size(), width = pages.size(3), page = pages.size(2);
  TORCH_CHECK(width * es % 16 == 0 && pages.stride(0) * es % 16 == 0 && pages.stride(1) * es % 16 == 0 &&
                  reinterpret_cast<uintptr_t>(pages.data_ptr()) % 16 == 0 && page >= 1,
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
  TORCH_CHECK(B <= 65535 && pages.size(0) <= 65535 && pages.size(1) < (1ll << 31), op, ": too many groups or layers");
  const at::cuda::CUDAGuard guard(pages.device());
  auto out = at::empty({B * K, table.size(1)}, table.options());
  if (B == 0 || table.size(1) == 0) return out;
  const int row16 = (int)(width * es / 16);
  const int parts = (int)((page * row16 + 1023) / 1024);
  const dim3 grid(parts + 1, (unsigned)std::max<int64_t>(1, pages.size(0)), (unsigned)B);
  beam_reorder_kernel<<<grid, 256, 0, at::cuda::getCurrentCUDAStream()>>>(
      reinterpret_cast<uint4*>(pages.data_ptr()), pages.stride(0) * es / 16, pages.stride(1) * es / 16, row16,
      (int)page, (int)pages.size(1), table.data_ptr<int>(), table.stride(0), (int)table.size(1),
      parents.data_ptr<int>(), (int)K, lens.data_ptr<int>(), out.data_ptr<int>(), parts, status_ptr());
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  return out;
}

void register_beam(pybind11::module_& m) {
  m.def("beam_select", &beam_select, "next beams over (beam, token) candidates", pybind11::arg("logits"),
        pybind11::arg("scores"), pybind11::arg("finished") = pybind11::none(), pybind11::arg("eos") = -1);
  m.def("beam_reorder", &beam_reorder, "block tables of the chosen beams and the copy of their unfinished page");
}

}  // namespace dsv3
