// Layer normalisation (sm_100a), forward and backward, with the residual add fused.
//
//   mu = mean(x), r = 1 / sqrt(mean((x - mu)^2) + eps), xh = (x - mu) r, y = xh w + b
//   dx = r (g - mean(g) - xh mean(g xh)) [+ dres],  g = dy w
//   dw = sum over rows of dy xh,  db = sum over rows of dy
//
// The variance is taken around the row's own mean (a second pass over the row), so a row
// with a large common offset loses nothing.  Statistics, sums and gradients are fp32; only
// the stored activations are rounded to the caller's type.  Every sum has a fixed order (no
// atomics), so two runs on the same inputs agree bit for bit.
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include "common.cuh"
#include "host_utils.h"

namespace pb {
namespace {

__device__ __forceinline__ float ldf(const float* p) { return *p; }
__device__ __forceinline__ float ldf(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ void stf(float* p, float v) { *p = v; }
__device__ __forceinline__ void stf(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

// Sum over the block in a fixed order; every thread gets the result.
__device__ __forceinline__ float block_sum(float v, float* red) {
  v = warp_sum(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x / 32] = v;
  __syncthreads();
  float t = 0.f;
  for (int k = 0; k < static_cast<int>(blockDim.x / 32); ++k) t += red[k];
  return t;
}

// One block per row.
template <typename TI, typename TO>
__global__ void ln_fwd_kernel(const TI* __restrict__ xp, const __nv_bfloat16* __restrict__ delta,
                              const float* __restrict__ w, const float* __restrict__ b, float* __restrict__ x_out,
                              TO* __restrict__ y, float* __restrict__ mean, float* __restrict__ rstd, int n,
                              float eps) {
  __shared__ float red[32];
  const long row = blockIdx.x;
  const long off = row * n;
  auto value = [&](int c) {
    const float v = ldf(xp + off + c);
    return delta != nullptr ? v + ldf(delta + off + c) : v;
  };
  float s = 0.f;
  for (int c = threadIdx.x; c < n; c += blockDim.x) {
    const float v = value(c);
    if (x_out != nullptr) x_out[off + c] = v;
    s += v;
  }
  const float mu = block_sum(s, red) / n;
  float ss = 0.f;
  for (int c = threadIdx.x; c < n; c += blockDim.x) {
    const float d = value(c) - mu;
    ss += d * d;
  }
  const float r = rsqrtf(block_sum(ss, red) / n + eps);
  if (threadIdx.x == 0) {
    mean[row] = mu;
    rstd[row] = r;
  }
  for (int c = threadIdx.x; c < n; c += blockDim.x)
    stf(y + off + c, (value(c) - mu) * r * w[c] + (b != nullptr ? b[c] : 0.f));
}

template <typename TI, typename TD>
__global__ void ln_bwd_dx_kernel(const TD* __restrict__ dy, const TI* __restrict__ x, const float* __restrict__ w,
                                 const float* __restrict__ mean, const float* __restrict__ rstd,
                                 const float* __restrict__ dres, TI* __restrict__ dx,
                                 __nv_bfloat16* __restrict__ dx_bf16, int n) {
  __shared__ float red[32];
  const long row = blockIdx.x;
  const long off = row * n;
  const float mu = mean[row], r = rstd[row];
  float s1 = 0.f, s2 = 0.f;
  for (int c = threadIdx.x; c < n; c += blockDim.x) {
    const float g = ldf(dy + off + c) * w[c];
    s1 += g;
    s2 += g * ((ldf(x + off + c) - mu) * r);
  }
  s1 = block_sum(s1, red) / n;
  s2 = block_sum(s2, red) / n;
  for (int c = threadIdx.x; c < n; c += blockDim.x) {
    const float g = ldf(dy + off + c) * w[c];
    const float xh = (ldf(x + off + c) - mu) * r;
    float d = r * (g - s1 - xh * s2);
    if (dres != nullptr) d += dres[off + c];
    stf(dx + off + c, d);
    if (dx_bf16 != nullptr) stf(dx_bf16 + off + c, d);
  }
}

// Column sums: a block owns 32 columns, its 8 warps take every eighth row.
template <typename TI, typename TD>
__global__ void ln_bwd_dw_kernel(const TD* __restrict__ dy, const TI* __restrict__ x, const float* __restrict__ mean,
                                 const float* __restrict__ rstd, float* __restrict__ dw, float* __restrict__ db,
                                 int rows, int n, bool accumulate) {
  __shared__ float red[2][8][32];
  const int lane = threadIdx.x & 31, wid = threadIdx.x / 32;
  const int c = blockIdx.x * 32 + lane;
  float sw = 0.f, sb = 0.f;
  if (c < n) {
    for (int row = wid; row < rows; row += 8) {
      const long at = static_cast<long>(row) * n + c;
      const float d = ldf(dy + at);
      sw += d * ((ldf(x + at) - mean[row]) * rstd[row]);
      sb += d;
    }
  }
  red[0][wid][lane] = sw;
  red[1][wid][lane] = sb;
  __syncthreads();
  if (wid != 0 || c >= n) return;
  for (int k = 1; k < 8; ++k) {
    sw += red[0][k][lane];
    sb += red[1][k][lane];
  }
  dw[c] = accumulate ? dw[c] + sw : sw;
  if (db != nullptr) db[c] = accumulate ? db[c] + sb : sb;
}

void check_vec(const at::Tensor& t, int64_t n, const at::Tensor& like, const char* what) {
  TORCH_CHECK(t.is_cuda() && t.device() == like.device() && t.scalar_type() == at::kFloat && t.is_contiguous() &&
                  t.numel() == n,
              "layernorm: ", what, " must be a contiguous fp32 CUDA tensor of ", n, " elements on the device of x");
}
void check_act(const at::Tensor& t, const at::Tensor& like, const char* what) {
  TORCH_CHECK(t.is_cuda() && t.device() == like.device() && t.is_contiguous() && t.sizes() == like.sizes() &&
                  (t.scalar_type() == at::kFloat || t.scalar_type() == at::kBFloat16),
              "layernorm: ", what, " must be a contiguous fp32 or bf16 CUDA tensor of x's shape and device");
}

template <typename F>
void by_type(const at::Tensor& t, F&& f) {
  if (t.scalar_type() == at::kFloat) f(static_cast<float*>(t.data_ptr()));
  else f(static_cast<__nv_bfloat16*>(t.data_ptr()));
}

}  // namespace

// x [rows, n] fp32 or bf16, ``delta`` (bf16, with an fp32 x): the row is x + delta, returned
// as the first tensor.  -> {x + delta or x, y, mean, rstd}.
std::vector<at::Tensor> add_layernorm_fwd(at::Tensor x, c10::optional<at::Tensor> delta, at::Tensor w,
                                          c10::optional<at::Tensor> b, double eps, bool out_bf16) {
  TORCH_CHECK(x.dim() == 2 && x.size(1) > 0, "layernorm: x must be [rows, n] with n > 0");
  check_act(x, x, "x");
  const int64_t rows = x.size(0), n = x.size(1);
  TORCH_CHECK(rows < (1LL << 31) && n < (1LL << 31), "layernorm: rows and n must fit 32 bits");
  check_vec(w, n, x, "weight");
  if (b.has_value()) check_vec(*b, n, x, "bias");
  const __nv_bfloat16* dp = nullptr;
  at::Tensor xo = x;
  const c10::cuda::CUDAGuard guard(x.device());
  if (delta.has_value()) {
    check_act(*delta, x, "delta");
    TORCH_CHECK(x.scalar_type() == at::kFloat && delta->scalar_type() == at::kBFloat16,
                "add_layernorm: fp32 x and bf16 delta");
    xo = at::empty_like(x);
    dp = static_cast<const __nv_bfloat16*>(delta->data_ptr());
  }
  auto y = at::empty(x.sizes(), x.options().dtype(out_bf16 ? at::kBFloat16 : x.scalar_type()));
  auto mean = at::empty({rows}, x.options().dtype(at::kFloat));
  auto rstd = at::empty({rows}, x.options().dtype(at::kFloat));
  if (rows == 0) return {xo, y, mean, rstd};
  auto s = at::cuda::getCurrentCUDAStream();
  const float* bp = b.has_value() ? b->data_ptr<float>() : nullptr;
  float* xop = delta.has_value() ? xo.data_ptr<float>() : nullptr;
  by_type(x, [&](auto* xp) {
    by_type(y, [&](auto* yp) {
      ln_fwd_kernel<<<rows, 256, 0, s>>>(xp, dp, w.data_ptr<float>(), bp, xop, yp, mean.data_ptr<float>(),
                                         rstd.data_ptr<float>(), (int)n, (float)eps);
    });
  });
  PB_CUDA_CHECK(cudaGetLastError());
  return {xo, y, mean, rstd};
}

// -> dx (x's type).  ``dres`` (fp32) is added to dx, ``dx_bf16`` receives a bf16 copy; dw and
// db are written into ``dw_out`` / ``db_out`` (added to them when ``accumulate``).
at::Tensor layernorm_bwd(at::Tensor dy, at::Tensor x, at::Tensor w, at::Tensor mean, at::Tensor rstd,
                         c10::optional<at::Tensor> dres, c10::optional<at::Tensor> dx_bf16, at::Tensor dw_out,
                         c10::optional<at::Tensor> db_out, bool accumulate) {
  TORCH_CHECK(x.dim() == 2 && x.size(1) > 0, "layernorm: x must be [rows, n] with n > 0");
  check_act(x, x, "x");
  check_act(dy, x, "dy");
  const int64_t rows = x.size(0), n = x.size(1);
  TORCH_CHECK(rows < (1LL << 31) && n < (1LL << 31), "layernorm: rows and n must fit 32 bits");
  check_vec(w, n, x, "weight");
  check_vec(mean, rows, x, "mean");
  check_vec(rstd, rows, x, "rstd");
  check_vec(dw_out, n, x, "dw_out");
  if (db_out.has_value()) check_vec(*db_out, n, x, "db_out");
  if (dres.has_value()) {
    check_act(*dres, x, "dres");
    TORCH_CHECK(dres->scalar_type() == at::kFloat, "layernorm: dres must be fp32");
  }
  if (dx_bf16.has_value()) {
    check_act(*dx_bf16, x, "dx_bf16");
    TORCH_CHECK(dx_bf16->scalar_type() == at::kBFloat16, "layernorm: dx_bf16 must be bf16");
  }
  const c10::cuda::CUDAGuard guard(x.device());
  auto dx = at::empty_like(x);
  auto s = at::cuda::getCurrentCUDAStream();
  const float* dr = dres.has_value() ? dres->data_ptr<float>() : nullptr;
  auto* dxb = dx_bf16.has_value() ? static_cast<__nv_bfloat16*>(dx_bf16->data_ptr()) : nullptr;
  float* dbp = db_out.has_value() ? db_out->data_ptr<float>() : nullptr;
  by_type(x, [&](auto* xp) {
    by_type(dy, [&](auto* dyp) {
      if (rows > 0)
        ln_bwd_dx_kernel<<<rows, 256, 0, s>>>(dyp, xp, w.data_ptr<float>(), mean.data_ptr<float>(),
                                              rstd.data_ptr<float>(), dr, static_cast<decltype(xp)>(dx.data_ptr()),
                                              dxb, (int)n);
      ln_bwd_dw_kernel<<<(n + 31) / 32, 256, 0, s>>>(dyp, xp, mean.data_ptr<float>(), rstd.data_ptr<float>(),
                                                     dw_out.data_ptr<float>(), dbp, (int)rows, (int)n, accumulate);
    });
  });
  PB_CUDA_CHECK(cudaGetLastError());
  return dx;
}

}  // namespace pb
