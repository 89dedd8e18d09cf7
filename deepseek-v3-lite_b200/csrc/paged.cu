// Paged latent cache: the write of new rows and the absorbed attention that
// reads them.
//
// A cache page holds `page` rows of D = R + dr bf16 values, the RMS-normalised
// latent (R) followed by the rotated shared key (dr); block_table[b, j] is the
// page of positions [j * page, (j + 1) * page) of sequence b.  A call works on
// a ragged batch: the new tokens of sequence b are rows cu[b] .. cu[b + 1) of
// the token-major inputs, and seq_lens[b] is its cached length including them,
// so token i of sequence b sits at position seq_lens[b] - n_b + i.  Lengths,
// offsets and tables are read on the device only: no host synchronisation, and
// a captured graph stays valid while they change.
//
// Error messages carry numbers as strings (std::to_string): formatting an
// integer through a stream crashes where the extension's compiler links its own
// static libstdc++ next to the one that torch loaded.
//
// A position outside the table, a page outside the pool or a token outside the
// batch's offsets is skipped and recorded in the device status word.
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>

#include <atomic>
#include <string>

#include "common.cuh"
#include "launch.h"
#include "status.h"
#include "tma_host.h"

namespace dsv3 {

namespace {

typedef __nv_bfloat16 bf16;

struct Ragged {
  const int* table;  // [B, cols], row stride ldt
  long ldt;
  const int* cu;     // [B + 1]
  const int* lens;   // [B]
  int B, cols, page, pool;
};

// Sequence of token t: the number of sequences that end at or before t.  Every
// lane counts its own share of the offsets, so the loads are independent and a
// warp waits for memory once whatever the batch (a binary search would wait
// log2(B) times).
__device__ __forceinline__ int ragged_seq(const Ragged& r, int t, int lane) {
  int n = 0;
  for (int j = lane; j < r.B; j += 32) n += __ldg(r.cu + j + 1) <= t;
  return __reduce_add_sync(0xffffffffu, n);
}

// ------------------------------------------------------------------- append
// Cache row of token t: *pos its position, null where it has none (reported).
__device__ __forceinline__ bf16* append_row(const Ragged& rg, int t, int lane, int npos, bf16* pages, long ld_page,
                                            long ld_row, int* pos, unsigned int* status) {
  const int b = ragged_seq(rg, t, lane);
  int pg = -1, col = 0;
  if (b < rg.B && t >= rg.cu[b]) {          // (not in front of the first offset)
    *pos = rg.lens[b] - rg.cu[b + 1] + t;
    col = *pos / rg.page;
    if (*pos >= 0 && *pos < npos && col < rg.cols) pg = rg.table[b * rg.ldt + col];
  }
  if (pg < 0 || pg >= rg.pool) {
    if (lane == 0) record_error(status, DSV3_ERR_BOUNDS);
    return nullptr;
  }
  return pages + (size_t)pg * ld_page + (size_t)(*pos - col * rg.page) * ld_row;
}

// row = [ x / sqrt(mean(x^2) + eps) * w | rotated pairs ] per token, one warp
// per token, statistics in fp32, any sizes.
template <typename T>
__global__ void __launch_bounds__(128) latent_append_kernel(const T* __restrict__ x, long ldx, int total, int R,
                                                            int dr, float eps, const float* __restrict__ w,
                                                            const float* __restrict__ cosv,
                                                            const float* __restrict__ sinv, int npos, Ragged rg,
                                                            bf16* __restrict__ pages, long ld_page, long ld_row,
                                                            unsigned int* status) {
  const int t = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (t >= total) return;
  int pos = 0;
  bf16* out = append_row(rg, t, lane, npos, pages, ld_page, ld_row, &pos, status);
  if (out == nullptr) return;
  const T* xr = x + (size_t)t * ldx;
  float ss = 0.f;
  for (int i = lane; i < R; i += 32) {
    const float v = (float)xr[i];
    ss += v * v;
  }
  const float inv = rsqrtf(warp_sum(ss) / R + eps);
  for (int i = lane; i < R; i += 32) out[i] = __float2bfloat16((float)xr[i] * inv * w[i]);
  for (int i = lane; i < dr / 2; i += 32) {
    const float c = cosv[(size_t)pos * (dr / 2) + i], s = sinv[(size_t)pos * (dr / 2) + i];
    const float a = (float)xr[R + 2 * i], d = (float)xr[R + 2 * i + 1];
    out[R + 2 * i] = __float2bfloat16(a * c - d * s);
    out[R + 2 * i + 1] = __float2bfloat16(a * s + d * c);
  }
}

__device__ __forceinline__ void load8(const float* p, float (&v)[8]) {
  const float4 a = __ldg(reinterpret_cast<const float4*>(p)), b = __ldg(reinterpret_cast<const float4*>(p) + 1);
  v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
}
__device__ __forceinline__ void load8(const bf16* p, float (&v)[8]) {
  const uint4 u = __ldg(reinterpret_cast<const uint4*>(p));
  const uint16_t* h = reinterpret_cast<const uint16_t*>(&u);
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = bf16_bits_to_float(h[i]);
}

// The same where rows are 16-byte aligned, R and dr multiples of 8 and R + dr at
// most 768: a lane takes up to three groups of 8 columns, read once, on their way
// while the token's sequence and page are looked up.  Bound by that latency for a
// decode step (64 rows: 3.1 us on the device), by it and the bytes for a prompt
// (8,300 rows of 576: 6.6 us, of which the bytes take 3.0 at the copy rate).
template <typename T>
__global__ void __launch_bounds__(128) latent_append_vec_kernel(const T* __restrict__ x, long ldx, int total, int R,
                                                                int dr, float eps, const float* __restrict__ w,
                                                                const float* __restrict__ cosv,
                                                                const float* __restrict__ sinv, int npos, Ragged rg,
                                                                bf16* __restrict__ pages, long ld_page, long ld_row,
                                                                unsigned int* status) {
  const int t = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (t >= total) return;
  const T* xr = x + (size_t)t * ldx;
  const int groups = (R + dr) / 8, latent = R / 8;
  float v[3][8], f[3][8];
#pragma unroll
  for (int k = 0; k < 3; ++k)
    if (lane + 32 * k < groups) load8(xr + 8 * (lane + 32 * k), v[k]);
  float ss = 0.f;
#pragma unroll
  for (int k = 0; k < 3; ++k)
    if (lane + 32 * k < latent) {
      load8(w + 8 * (lane + 32 * k), f[k]);
#pragma unroll
      for (int i = 0; i < 8; ++i) ss += v[k][i] * v[k][i];
    }
  int pos = 0;
  bf16* out = append_row(rg, t, lane, npos, pages, ld_page, ld_row, &pos, status);
  if (out == nullptr) return;
  const float inv = rsqrtf(warp_sum(ss) / R + eps);
#pragma unroll
  for (int k = 0; k < 3; ++k) {
    const int g = lane + 32 * k;
    if (g >= groups) break;
    if (g < latent) {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[k][i] *= inv * f[k][i];
    } else {
      const size_t at = (size_t)pos * (dr / 2) + (g - latent) * 4;
      const float4 c = __ldg(reinterpret_cast<const float4*>(cosv + at));
      const float4 s = __ldg(reinterpret_cast<const float4*>(sinv + at));
      const float cc[4] = {c.x, c.y, c.z, c.w}, sn[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float a = v[k][2 * i], d = v[k][2 * i + 1];
        v[k][2 * i] = a * cc[i] - d * sn[i];
        v[k][2 * i + 1] = a * sn[i] + d * cc[i];
      }
    }
    *reinterpret_cast<uint4*>(out + 8 * g) = make_uint4(pack_bf16x2(v[k][0], v[k][1]), pack_bf16x2(v[k][2], v[k][3]),
                                                        pack_bf16x2(v[k][4], v[k][5]), pack_bf16x2(v[k][6], v[k][7]));
  }
}

// ---------------------------------------------------------------- attention
#include "paged_attention_tc.cuh"

// --------------------------------------------------------------- host side
// Opt a kernel in to the full shared memory of a CTA, once per device (the call
// costs host time on every launch otherwise).
template <typename Kern>
void allow_shared_memory(Kern kern, std::atomic<uint64_t>& done) {
  int dev = 0;
  C10_CUDA_CHECK(cudaGetDevice(&dev));
  const uint64_t bit = 1ull << (dev & 63);
  if (done.load(std::memory_order_acquire) & bit) return;
  C10_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kPaSmem));
  done.fetch_or(bit, std::memory_order_release);
}

Ragged check_ragged(const char* op, const at::Tensor& ref, const at::Tensor& pages, const at::Tensor& table,
                    const at::Tensor& cu, const at::Tensor& lens) {
  TORCH_CHECK(pages.is_cuda() && pages.dim() == 3 && pages.scalar_type() == at::kBFloat16 && pages.stride(2) == 1,
              op, ": pages must be a CUDA bf16 tensor [pool, page, R + dr] with unit stride in the last dimension");
  TORCH_CHECK(table.dim() == 2 && table.scalar_type() == at::kInt && table.stride(1) == 1,
              op, ": block_table must be int32 [B, columns] with unit stride in the last dimension");
  TORCH_CHECK(lens.dim() == 1 && lens.scalar_type() == at::kInt && lens.is_contiguous() &&
                  lens.size(0) == table.size(0),
              op, ": seq_lens must be a contiguous int32 tensor [B]");
  TORCH_CHECK(cu.dim() == 1 && cu.scalar_type() == at::kInt && cu.is_contiguous() && cu.size(0) == lens.size(0) + 1,
              op, ": cu_seqlens must be a contiguous int32 tensor [B + 1]");
  TORCH_CHECK(ref.device() == pages.device() && table.device() == pages.device() && cu.device() == pages.device() &&
                  lens.device() == pages.device(),
              op, ": all tensors must be on the device of pages");
  const int64_t page = pages.size(1);
  TORCH_CHECK(page >= 8 && page <= 256 && (page & (page - 1)) == 0, op,
              ": the page size must be a power of two from 8 to 256, got ", std::to_string(page));
  TORCH_CHECK(pages.stride(0) % 8 == 0 && pages.stride(1) % 8 == 0 &&
                  reinterpret_cast<uintptr_t>(pages.data_ptr()) % 16 == 0,
              op, ": page rows must be 16-byte aligned");
  TORCH_CHECK(pages.size(0) >= 1 && table.size(1) >= 1, op, ": an empty pool or table");
  TORCH_CHECK(pages.size(0) * page < (1ll << 31) && table.size(1) * page < (1ll << 31), op,
              ": the pool and a sequence hold fewer than 2^31 rows");
  Ragged r;
  r.table = table.data_ptr<int>();
  r.ldt = table.stride(0);
  r.cu = cu.data_ptr<int>();
  r.lens = lens.data_ptr<int>();
  r.B = table.size(0);
  r.cols = table.size(1);
  r.page = page;
  r.pool = pages.size(0);
  return r;
}

}  // namespace

void latent_cache_append(at::Tensor& pages, const at::Tensor& kv_a, const at::Tensor& weight, const at::Tensor& cosv,
                         const at::Tensor& sinv, const at::Tensor& table, const at::Tensor& cu,
                         const at::Tensor& lens, double eps) {
  const char* op = "latent_cache_append";
  TORCH_CHECK(kv_a.dim() == 2 && kv_a.stride(1) == 1 &&
                  (kv_a.scalar_type() == at::kBFloat16 || kv_a.scalar_type() == at::kFloat),
              op, ": kv_a must be bf16 or fp32 [T, R + dr] with unit stride in the last dimension");
  const Ragged rg = check_ragged(op, kv_a, pages, table, cu, lens);
  TORCH_CHECK(weight.dim() == 1 && weight.scalar_type() == at::kFloat && weight.is_contiguous(), op,
              ": weight must be a contiguous fp32 tensor [R]");
  TORCH_CHECK(cosv.dim() == 2 && cosv.scalar_type() == at::kFloat && cosv.is_contiguous() &&
                  sinv.scalar_type() == at::kFloat && sinv.is_contiguous() && sinv.sizes() == cosv.sizes(),
              op, ": cos and sin must be contiguous fp32 tables [positions, dr / 2]");
  const int64_t R = weight.size(0), dr = 2 * cosv.size(1);
  TORCH_CHECK(kv_a.size(1) == R + dr && pages.size(2) == R + dr, op, ": kv_a and pages must be R + dr = ",
              std::to_string(R + dr), " wide");
  TORCH_CHECK(weight.device() == pages.device() && cosv.device() == pages.device() &&
                  sinv.device() == pages.device(),
              op, ": all tensors must be on the device of pages");
  const int64_t T = kv_a.size(0);
  TORCH_CHECK(T < (1ll << 31), op, ": too many tokens");
  if (T == 0) return;
  TORCH_CHECK(rg.B > 0, op, ": tokens without a sequence");
  const at::cuda::CUDAGuard guard(pages.device());
  auto st = at::cuda::getCurrentCUDAStream();
  const int grid = (int)((T + 3) / 4);
  auto aligned = [](const at::Tensor& x) { return reinterpret_cast<uintptr_t>(x.data_ptr()) % 16 == 0; };
  const bool vec = R % 8 == 0 && dr % 8 == 0 && R + dr <= 768 && kv_a.stride(0) * kv_a.element_size() % 16 == 0 &&
                   aligned(kv_a) && aligned(weight) && aligned(cosv) && aligned(sinv);
#define DSV3_APPEND(K_, T_)                                                                                      \
  K_<T_><<<grid, 128, 0, st>>>(reinterpret_cast<const T_*>(kv_a.data_ptr()), kv_a.stride(0), (int)T, (int)R,     \
                               (int)dr, (float)eps, weight.data_ptr<float>(), cosv.data_ptr<float>(),            \
                               sinv.data_ptr<float>(), (int)cosv.size(0), rg,                                    \
                               reinterpret_cast<bf16*>(pages.data_ptr()), pages.stride(0), pages.stride(1),      \
                               status_ptr())
  if (kv_a.scalar_type() == at::kFloat) {
    if (vec) DSV3_APPEND(latent_append_vec_kernel, float);
    else DSV3_APPEND(latent_append_kernel, float);
  } else {
    if (vec) DSV3_APPEND(latent_append_vec_kernel, bf16);
    else DSV3_APPEND(latent_append_kernel, bf16);
  }
#undef DSV3_APPEND
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

at::Tensor paged_latent_attention(const at::Tensor& q, const at::Tensor& pages, const at::Tensor& table,
                                  const at::Tensor& cu, const at::Tensor& lens, int64_t R, double scale) {
  const char* op = "paged_latent_attention";
  TORCH_CHECK(q.dim() == 3 && q.scalar_type() == at::kBFloat16 && q.is_contiguous(), op,
              ": q must be a contiguous bf16 tensor [T, H, R + dr]");
  const Ragged rg = check_ragged(op, q, pages, table, cu, lens);
  const int64_t T = q.size(0), H = q.size(1), D = q.size(2);
  TORCH_CHECK(pages.size(2) == D, op, ": q and pages must have the same width, got ", std::to_string(D),
              " and ", std::to_string(pages.size(2)));
  TORCH_CHECK(R % 8 == 0 && R >= 8 && R <= 512 && D % 8 == 0 && D > R && D - R <= 64, op,
              ": the latent rank must be a multiple of 8 up to 512 and the rotary width one up to 64, got ",
              std::to_string(R), " and ", std::to_string(D - R));
  TORCH_CHECK(H >= 1 && H <= 4096 && T * H < (1ll << 31), op, ": 1 to 4096 heads and T * H below 2^31");
  TORCH_CHECK(scale > 0, op, ": scale must be positive");
  auto out = at::Tensor(at::detail::empty_cuda({T, H, R}, at::kBFloat16, pages.device(), c10::nullopt));
  if (T == 0) return out;
  TORCH_CHECK(rg.B > 0, op, ": tokens without a sequence");
  const at::cuda::CUDAGuard guard(pages.device());
  const int sms = at::cuda::getCurrentDeviceProperties()->multiProcessorCount;
  // Row tile, from the rows per sequence on average: 16 up to 16 (12 heads of R 192
  // over 64 x 2,048 rows 24.6 us against 26.7 with 32); 32 up to 32 where every
  // sequence has one token (24 heads 26.7 against 30.4 with 64; of R 512, 32 heads,
  // 45.4 against 50.6), while a ragged batch of the same average may hold chunks,
  // which want 64; 64 up to 64 (32 x 5 tokens of 12 heads 26.7 against 28.7 with
  // 128); then 128 (8 x 256 tokens 77.5 against 98.4 with 64) where the output
  // columns of 128 rows fit in TMEM.
  const int64_t rows = (T * H + rg.B - 1) / rg.B;
  const int N = rows <= 16 ? 16 : rows <= 32 && T == rg.B ? 32 : rows <= 64 || R > 256 ? 64 : 128;
  PagedPlan pl;
  TORCH_CHECK(paged_plan(N, (int)R, (int)D, pl), op, ": no shared-memory plan");
  auto work = at::Tensor(
      at::detail::empty_cuda({sms * (2 * N * (R + 2) + 4)}, at::kFloat, pages.device(), c10::nullopt));
  int4* rec = reinterpret_cast<int4*>(work.data_ptr<float>());
  float2* ml = reinterpret_cast<float2*>(rec + sms);
  float* part = reinterpret_cast<float*>(ml + 2 * (int64_t)sms * N);
  const uint64_t qd[2] = {(uint64_t)D, (uint64_t)(T * H)}, qs[1] = {(uint64_t)D * 2};
  const uint32_t qb[2] = {64, (uint32_t)N};
  const CUtensorMap tm_q = make_map(q.data_ptr(), 2, qd, qs, qb);
  const uint64_t kd[3] = {(uint64_t)D, (uint64_t)rg.page, (uint64_t)rg.pool};
  const uint64_t ks[2] = {(uint64_t)pages.stride(1) * 2, (uint64_t)pages.stride(0) * 2};
  const uint32_t kb[3] = {64, (uint32_t)std::min(rg.page, KT), 1};
  const CUtensorMap tm_kv = make_map(pages.data_ptr(), 3, kd, ks, kb);
  auto st = at::cuda::getCurrentCUDAStream();
  const int64_t cuts = std::min<int64_t>(sms, T * H / N + rg.B);   // row tiles that can be cut, at most
  const bool few = cuts * 4 <= sms;
  bf16* o = reinterpret_cast<bf16*>(out.data_ptr());
  static std::atomic<uint64_t> opted[4];   // devices on which each variant may take all shared memory
  const int variant = N == 16 ? 0 : N == 32 ? 1 : N == 64 ? 2 : 3;
#define DSV3_PAGED(N_)                                                                                           \
  do {                                                                                                           \
    allow_shared_memory(paged_attention_tc_kernel<N_>, opted[variant]);                                      \
    paged_attention_tc_kernel<N_><<<sms, pa_threads(N_), pl.smem, st>>>(                                             \
        tm_q, tm_kv, pl, rg, (int)T, (int)H, (int)R, (int)D, (float)(scale * 1.4426950408889634), o, part, ml, \
        rec, status_ptr());                                                                                      \
    C10_CUDA_KERNEL_LAUNCH_CHECK();                                                                              \
    C10_CUDA_CHECK(few ? launch_dependent(paged_merge_kernel<N_, true>, dim3((unsigned)cuts, N_), 512, st,       \
                                          (const float*)part, (const float2*)ml, (const int4*)rec, sms, (int)R, o) \
                       : launch_dependent(paged_merge_kernel<N_, false>, dim3(sms, N_ / 8), 256, st,             \
                                          (const float*)part, (const float2*)ml, (const int4*)rec, sms, (int)R, o)); \
  } while (0)
  if (N == 16) DSV3_PAGED(16);
  else if (N == 32) DSV3_PAGED(32);
  else if (N == 64) DSV3_PAGED(64);
  else DSV3_PAGED(128);
#undef DSV3_PAGED
  return out;
}

void register_paged(pybind11::module_& m) {
  m.def("latent_cache_append", &latent_cache_append,
        "normalised latent and rotated key of new tokens into the pages of a latent cache");
  m.def("paged_latent_attention", &paged_latent_attention,
        "absorbed attention of a ragged batch of new tokens over a paged latent cache");
}

}  // namespace dsv3
