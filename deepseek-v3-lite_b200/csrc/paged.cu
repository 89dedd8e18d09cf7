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
#include <c10/cuda/CUDAGuard.h>

#include <string>

#include "common.cuh"
#include "status.h"

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
// row = [ x / sqrt(mean(x^2) + eps) * w | rotated pairs ] per token, one warp
// per token, statistics in fp32.
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
  const int b = ragged_seq(rg, t, lane);
  if (b >= rg.B) {
    if (lane == 0) record_error(status, DSV3_ERR_BOUNDS);
    return;
  }
  const int pos = rg.lens[b] - rg.cu[b + 1] + t;
  const int col = pos / rg.page;
  int pg = -1;
  if (pos >= 0 && pos < npos && col < rg.cols) pg = rg.table[b * rg.ldt + col];
  if (pg < 0 || pg >= rg.pool) {
    if (lane == 0) record_error(status, DSV3_ERR_BOUNDS);
    return;
  }
  const T* xr = x + (size_t)t * ldx;
  bf16* out = pages + (size_t)pg * ld_page + (size_t)(pos - col * rg.page) * ld_row;
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

// ---------------------------------------------------------------- attention
// out[t, h] = sum_j softmax_j(scale * q[t, h] . k_j) k_j[:R] over the cached
// rows j at or before the token's position.  One warp per (token, head) with a
// running maximum and sum.
constexpr int kMaxPerLane = 18;  // D <= 576

__global__ void __launch_bounds__(128) paged_attention_kernel(const bf16* __restrict__ q, int total, int H, int R,
                                                              int D, Ragged rg, const bf16* __restrict__ pages,
                                                              long ld_page, long ld_row, float scale,
                                                              bf16* __restrict__ out, unsigned int* status) {
  const int item = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (item >= total * H) return;
  const int t = item / H;
  const int b = ragged_seq(rg, t, lane);
  int keys = 0;
  if (b < rg.B) {
    const int len = min(rg.lens[b], rg.cols * rg.page);
    keys = min(rg.lens[b] - rg.cu[b + 1] + t + 1, len);
    if (len < rg.lens[b] && lane == 0) record_error(status, DSV3_ERR_BOUNDS);
  } else if (lane == 0) {
    record_error(status, DSV3_ERR_BOUNDS);
  }
  float qv[kMaxPerLane], acc[kMaxPerLane], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int i = 0; i < kMaxPerLane; ++i) {
    acc[i] = 0.f;
    qv[i] = lane + 32 * i < D ? __bfloat162float(q[(size_t)item * D + lane + 32 * i]) : 0.f;
  }
  for (int j = 0; j < keys; ++j) {
    const int pg = rg.table[b * rg.ldt + j / rg.page];
    if (pg < 0 || pg >= rg.pool) {
      if (lane == 0) record_error(status, DSV3_ERR_BOUNDS);
      continue;
    }
    const bf16* kr = pages + (size_t)pg * ld_page + (size_t)(j % rg.page) * ld_row;
    float kv[kMaxPerLane], s = 0.f;
#pragma unroll
    for (int i = 0; i < kMaxPerLane; ++i) {
      kv[i] = lane + 32 * i < D ? __bfloat162float(kr[lane + 32 * i]) : 0.f;
      s += qv[i] * kv[i];
    }
    s = warp_sum(s) * scale;
    const float nm = fmaxf(m, s);
    if (nm == -INFINITY) continue;
    const float c = expf(m - nm), p = expf(s - nm);
    l = l * c + p;
#pragma unroll
    for (int i = 0; i < kMaxPerLane; ++i) acc[i] = acc[i] * c + p * kv[i];
    m = nm;
  }
  const float inv = l > 0.f ? 1.f / l : 0.f;
#pragma unroll
  for (int i = 0; i < kMaxPerLane; ++i)
    if (lane + 32 * i < R) out[(size_t)item * R + lane + 32 * i] = __float2bfloat16(acc[i] * inv);
}

// --------------------------------------------------------------- host side
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
#define DSV3_APPEND(T_, P_)                                                                                        \
  latent_append_kernel<T_><<<grid, 128, 0, st>>>(P_, kv_a.stride(0), (int)T, (int)R, (int)dr, (float)eps,         \
      weight.data_ptr<float>(), cosv.data_ptr<float>(), sinv.data_ptr<float>(), (int)cosv.size(0), rg,             \
      reinterpret_cast<bf16*>(pages.data_ptr()), pages.stride(0), pages.stride(1), status_ptr())
  if (kv_a.scalar_type() == at::kFloat) DSV3_APPEND(float, kv_a.data_ptr<float>());
  else DSV3_APPEND(bf16, reinterpret_cast<const bf16*>(kv_a.data_ptr()));
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
  TORCH_CHECK(H >= 1 && T * H < (1ll << 31), op, ": T * H must be below 2^31");
  auto out = at::empty({T, H, R}, q.options());
  if (T == 0) return out;
  TORCH_CHECK(rg.B > 0, op, ": tokens without a sequence");
  const at::cuda::CUDAGuard guard(pages.device());
  paged_attention_kernel<<<(int)((T * H + 3) / 4), 128, 0, at::cuda::getCurrentCUDAStream()>>>(
      reinterpret_cast<const bf16*>(q.data_ptr()), (int)T, (int)H, (int)R, (int)D, rg,
      reinterpret_cast<const bf16*>(pages.data_ptr()), pages.stride(0), pages.stride(1), (float)scale,
      reinterpret_cast<bf16*>(out.data_ptr()), status_ptr());
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  return out;
}

void register_paged(pybind11::module_& m) {
  m.def("latent_cache_append", &latent_cache_append,
        "normalised latent and rotated key of new tokens into the pages of a latent cache");
  m.def("paged_latent_attention", &paged_latent_attention,
        "absorbed attention of a ragged batch of new tokens over a paged latent cache");
}

}  // namespace dsv3
