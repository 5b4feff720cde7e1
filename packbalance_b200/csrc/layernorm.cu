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

#include <type_traits>

#include "common.cuh"
#include "host_utils.h"

namespace pb {
namespace {

__device__ __forceinline__ float ldf(const float* p) { return *p; }
__device__ __forceinline__ float ldf(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ void stf(float* p, float v) { *p = v; }
__device__ __forceinline__ void stf(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

// ---- rows held in registers --------------------------------------------------------
// T threads hold a row, K pieces of V elements each (16 bytes where rows allow it, else single
// elements), so a row is read once; rows are dealt to a persistent grid and the next row's
// loads are issued before the current row is reduced.  Weight, bias and the backward's column
// sums stay in registers over all of a thread's rows.  Both directions wait for HBM only; what
// has to be right for that is bytes in flight: 256 threads x 16 elements x 2 rows per SM and more.
template <typename T_, int V>
struct Piece;  // V consecutive elements as loaded
template <>
struct Piece<float, 4> {
  float4 r;
  __device__ __forceinline__ void load(const float* p) { r = __ldcs(reinterpret_cast<const float4*>(p)); }
  __device__ __forceinline__ void get(float* v) const { v[0] = r.x; v[1] = r.y; v[2] = r.z; v[3] = r.w; }
};
template <>
struct Piece<__nv_bfloat16, 4> {
  uint2 r;
  __device__ __forceinline__ void load(const __nv_bfloat16* p) { r = __ldcs(reinterpret_cast<const uint2*>(p)); }
  __device__ __forceinline__ void get(float* v) const {
    const float2 a = unpack_bf16x2(r.x), b = unpack_bf16x2(r.y);
    v[0] = a.x; v[1] = a.y; v[2] = b.x; v[3] = b.y;
  }
};
template <>
struct Piece<__nv_bfloat16, 8> {
  uint4 r;
  __device__ __forceinline__ void load(const __nv_bfloat16* p) { r = __ldcs(reinterpret_cast<const uint4*>(p)); }
  __device__ __forceinline__ void get(float* v) const {
    const uint32_t* w = &r.x;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float2 a = unpack_bf16x2(w[k]);
      v[2 * k] = a.x;
      v[2 * k + 1] = a.y;
    }
  }
};
template <typename T_>
struct Piece<T_, 1> {
  T_ r;
  __device__ __forceinline__ void load(const T_* p) { r = *p; }
  __device__ __forceinline__ void get(float* v) const { *v = ldf(&r); }
};
template <int V>
__device__ __forceinline__ void put(float* p, const float* v) {
  if constexpr (V == 1) *p = *v;
  else
#pragma unroll
    for (int k = 0; k < V; k += 4)
      *reinterpret_cast<float4*>(p + k) = make_float4(v[k], v[k + 1], v[k + 2], v[k + 3]);
}
template <int V>
__device__ __forceinline__ void put(__nv_bfloat16* p, const float* v) {
  if constexpr (V == 1) *p = __float2bfloat16_rn(*v);
  else if constexpr (V == 4) *reinterpret_cast<uint2*>(p) = make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
  else
    *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]),
                                              pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
}

constexpr int ln_threads(int t) { return t < 256 ? 256 : t; }

// Sum over the T threads of a row, in a fixed order; every one gets it.  ``red``: T / 32 floats
// of this group, used alternately (``flip``) so that one barrier per sum is enough.
template <int T>
__device__ __forceinline__ float row_sum(float v, float* red, int& flip) {
  v = warp_sum(v);
  if constexpr (T == 32) return v;
  constexpr int W = T / 32;
  float* r = red + flip * W;
  flip ^= 1;
  const int t = threadIdx.x % T;
  if ((t & 31) == 0) r[t / 32] = v;
  if constexpr (T >= 256) __syncthreads();
  else asm volatile("bar.sync %0, %1;" ::"r"(1 + static_cast<int>(threadIdx.x) / T), "n"(T) : "memory");
  float s = 0.f;
#pragma unroll
  for (int k = 0; k < W; ++k) s += r[k];
  return s;
}

template <int T, int V, int K, typename TI, typename TO, bool ADD>
__global__ void __launch_bounds__(ln_threads(T))
    ln_fwd_reg_kernel(const TI* __restrict__ xp, const __nv_bfloat16* __restrict__ delta, const float* __restrict__ w,
                      const float* __restrict__ b, float* __restrict__ x_out, TO* __restrict__ y,
                      float* __restrict__ mean, float* __restrict__ rstd, int rows, int n, float eps) {
  constexpr int G = ln_threads(T) / T;
  __shared__ float red[G][2 * (T / 32)];
  const int t = threadIdx.x % T, grp = threadIdx.x / T;
  int flip = 0;
  float wv[K * V], bv[K * V];
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const int c = (k * T + t) * V + e;
      wv[k * V + e] = c < n ? w[c] : 0.f;
      bv[k * V + e] = c < n && b != nullptr ? b[c] : 0.f;
    }
  Piece<TI, V> px[K];
  Piece<__nv_bfloat16, V> pd[ADD ? K : 1];
  auto fetch = [&](long row) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = (k * T + t) * V;
      if (c < n) {
        px[k].load(xp + row * n + c);
        if constexpr (ADD) pd[k].load(delta + row * n + c);
      }
    }
  };
  const long stride = static_cast<long>(gridDim.x) * G;
  long row = static_cast<long>(blockIdx.x) * G + grp;
  if (row < rows) fetch(row);
  for (; row < rows; row += stride) {
    float v[K * V];
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = (k * T + t) * V;
      if (c < n) {
        px[k].get(v + k * V);
        if constexpr (ADD) {
          float d[V];
          pd[k].get(d);
#pragma unroll
          for (int e = 0; e < V; ++e) v[k * V + e] += d[e];
          put<V>(x_out + row * n + c, v + k * V);
        }
      } else {
#pragma unroll
        for (int e = 0; e < V; ++e) v[k * V + e] = 0.f;
      }
#pragma unroll
      for (int e = 0; e < V; ++e) s += v[k * V + e];
    }
    if (row + stride < rows) fetch(row + stride);
    const float mu = row_sum<T>(s, red[grp], flip) / n;
    float ss = 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k)
      if ((k * T + t) * V < n) {
#pragma unroll
        for (int e = 0; e < V; ++e) {
          v[k * V + e] -= mu;
          ss += v[k * V + e] * v[k * V + e];
        }
      }
    const float r = rsqrtf(row_sum<T>(ss, red[grp], flip) / n + eps);
    if (t == 0 && mean != nullptr) {
      mean[row] = mu;
      rstd[row] = r;
    }
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = (k * T + t) * V;
      if (c < n) {
        float o[V];
#pragma unroll
        for (int e = 0; e < V; ++e) o[e] = v[k * V + e] * r * wv[k * V + e] + bv[k * V + e];
        put<V>(y + row * n + c, o);
      }
    }
  }
}

// ``part``: [gridDim.x][2][n], this block's sums for dw and db.
template <int T, int V, int K, typename TI, typename TD, bool RES>
__global__ void __launch_bounds__(ln_threads(T))
    ln_bwd_reg_kernel(const TD* __restrict__ dy, const TI* __restrict__ x, const float* __restrict__ w,
                      const float* __restrict__ mean, const float* __restrict__ rstd, const float* __restrict__ dres,
                      TI* __restrict__ dx, __nv_bfloat16* __restrict__ dx_bf16, float* __restrict__ part, int rows,
                      int n) {
  constexpr int G = ln_threads(T) / T;
  __shared__ float red[G][4 * (T / 32)];
  extern __shared__ float cols[];  // [2][T * K * V] (G > 1)
  const int t = threadIdx.x % T, grp = threadIdx.x / T;
  int flip = 0;
  float wv[K * V], aw[K * V], ab[K * V];
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const int c = (k * T + t) * V + e;
      wv[k * V + e] = c < n ? w[c] : 0.f;
      aw[k * V + e] = ab[k * V + e] = 0.f;
    }
  Piece<TI, V> px[K];
  Piece<TD, V> pg[K];
  Piece<float, V == 8 ? 4 : V> pr[RES ? K : 1];
  float mu_n = 0.f, r_n = 0.f;
  auto fetch = [&](long row) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = (k * T + t) * V;
      if (c < n) {
        px[k].load(x + row * n + c);
        pg[k].load(dy + row * n + c);
        if constexpr (RES) pr[k].load(dres + row * n + c);
      }
    }
    mu_n = mean[row];
    r_n = rstd[row];
  };
  const long stride = static_cast<long>(gridDim.x) * G;
  long row = static_cast<long>(blockIdx.x) * G + grp;
  if (row < rows) fetch(row);
  for (; row < rows; row += stride) {
    const float mu = mu_n, r = r_n;
    float xh[K * V], g[K * V], res[RES ? K * V : 1];
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if ((k * T + t) * V < n) {
        px[k].get(xh + k * V);
        pg[k].get(g + k * V);
        if constexpr (RES) pr[k].get(res + k * V);
      } else {
#pragma unroll
        for (int e = 0; e < V; ++e) {
          xh[k * V + e] = mu;
          g[k * V + e] = 0.f;
        }
      }
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const int i = k * V + e;
        xh[i] = (xh[i] - mu) * r;
        aw[i] += g[i] * xh[i];
        ab[i] += g[i];
        g[i] *= wv[i];
        s1 += g[i];
        s2 += g[i] * xh[i];
      }
    }
    if (row + stride < rows) fetch(row + stride);
    // both sums behind one barrier
    s1 = warp_sum(s1);
    s2 = warp_sum(s2);
    if constexpr (T > 32) {
      constexpr int W = T / 32;
      float* q = red[grp] + flip * 2 * W;
      flip ^= 1;
      if ((t & 31) == 0) {
        q[t / 32] = s1;
        q[W + t / 32] = s2;
      }
      if constexpr (T >= 256) __syncthreads();
      else asm volatile("bar.sync %0, %1;" ::"r"(1 + grp), "n"(T) : "memory");
      s1 = s2 = 0.f;
#pragma unroll
      for (int k = 0; k < W; ++k) {
        s1 += q[k];
        s2 += q[W + k];
      }
    }
    s1 /= n;
    s2 /= n;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = (k * T + t) * V;
      if (c < n) {
        float o[V];
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const int i = k * V + e;
          o[e] = r * (g[i] - s1 - xh[i] * s2);
          if constexpr (RES) o[e] += res[i];
        }
        put<V>(dx + row * n + c, o);
        if constexpr (RES) {
          if (dx_bf16 != nullptr) put<V>(dx_bf16 + row * n + c, o);
        }
      }
    }
  }
  if constexpr (G > 1) {  // the groups' sums, added in group order
    float* cw = cols;
    float* cb = cols + T * K * V;
    for (int q = 0; q < G; ++q) {
      if (grp == q) {
#pragma unroll
        for (int i = 0; i < K * V; ++i) {
          cw[i * T + t] = q == 0 ? aw[i] : cw[i * T + t] + aw[i];
          cb[i * T + t] = q == 0 ? ab[i] : cb[i * T + t] + ab[i];
        }
      }
      __syncthreads();
    }
    if (grp != 0) return;
#pragma unroll
    for (int i = 0; i < K * V; ++i) {
      aw[i] = cw[i * T + t];
      ab[i] = cb[i * T + t];
    }
  }
  float* pw = part + static_cast<long>(blockIdx.x) * 2 * n;
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const int c = (k * T + t) * V + e;
      if (c < n) {
        pw[c] = aw[k * V + e];
        pw[n + c] = ab[k * V + e];
      }
    }
}

// dw, db (+)= the blocks' sums, in block order per warp and then in warp order.  A block takes 32
// of the 2 n columns, its 32 warps every 32nd partial row.
__global__ void __launch_bounds__(1024)
    ln_dw_reduce_kernel(const float* __restrict__ part, int blocks, int n, float* __restrict__ dw,
                        float* __restrict__ db, bool accumulate) {
  __shared__ float red[32][33];
  const int lane = threadIdx.x & 31, wid = threadIdx.x / 32;
  const long c = static_cast<long>(blockIdx.x) * 32 + lane;
  float s = 0.f;
  if (c < 2L * n) {
#pragma unroll 4
    for (int k = wid; k < blocks; k += 32) s += part[static_cast<long>(k) * 2 * n + c];
  }
  red[wid][lane] = s;
  __syncthreads();
  if (wid != 0 || c >= 2L * n) return;
  for (int k = 1; k < 32; ++k) s += red[k][lane];
  float* out = c < n ? dw + c : (db != nullptr ? db + (c - n) : nullptr);
  if (out != nullptr) *out = accumulate ? *out + s : s;
}

// ---- rows of any width -------------------------------------------------------------
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
  if (threadIdx.x == 0 && mean != nullptr) {
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

// Threads per row T and pieces per thread K for n elements in pieces of V.  K as large as the
// registers allow (16 elements; fewer threads per row mean cheaper sums), then T the power of
// two that leaves the fewest lanes idle; 0: the row does not fit.
struct RowPlan {
  int T, K;
};
RowPlan row_plan(int64_t n, int V) {
  const int64_t pieces = (n + V - 1) / V;
  const int most = V == 1 ? 16 : 16 / V;
  RowPlan best{0, 0};
  int64_t best_cost = 0;
  for (int T = 32; T <= 1024; T *= 2) {
    int K = static_cast<int>((pieces + T - 1) / T);
    if (K > most) continue;
    if (V == 1) K = K <= 2 ? 2 : (K <= 4 ? 4 : (K <= 8 ? 8 : (K <= 12 ? 12 : 16)));  // compiled sizes
    const int64_t cost = static_cast<int64_t>(T) * K * 64 + T;  // lanes x pieces, then threads
    if (best.T == 0 || cost < best_cost) {
      best = {T, K};
      best_cost = cost;
    }
  }
  return best;
}

template <int V, typename F>
bool with_plan(const RowPlan& p, F&& f) {
  auto with_k = [&](auto t) {
    constexpr int T = decltype(t)::value;
    auto is = [&](auto k) {
      if (p.K != decltype(k)::value) return false;
      f(t, k);
      return true;
    };
    if constexpr (V == 1)
      return is(std::integral_constant<int, 2>{}) || is(std::integral_constant<int, 4>{}) ||
             is(std::integral_constant<int, 8>{}) || is(std::integral_constant<int, 12>{}) ||
             is(std::integral_constant<int, 16>{});
    else if constexpr (V == 4)
      return is(std::integral_constant<int, 1>{}) || is(std::integral_constant<int, 2>{}) ||
             is(std::integral_constant<int, 3>{}) || is(std::integral_constant<int, 4>{});
    else return is(std::integral_constant<int, 1>{}) || is(std::integral_constant<int, 2>{});
  };
  switch (p.T) {
    case 32: return with_k(std::integral_constant<int, 32>{});
    case 64: return with_k(std::integral_constant<int, 64>{});
    case 128: return with_k(std::integral_constant<int, 128>{});
    case 256: return with_k(std::integral_constant<int, 256>{});
    case 512: return with_k(std::integral_constant<int, 512>{});
    case 1024: return with_k(std::integral_constant<int, 1024>{});
  }
  return false;
}

// Blocks of a persistent launch: what fits on the GPU at once, or fewer for few rows.
template <typename Kern>
int row_blocks(Kern kern, int threads, size_t smem, int64_t rows, int groups, int dev) {
  static int per_sm[64] = {0};  // one instance per kernel
  if (per_sm[dev] == 0) {
    int n = 0;
    PB_CUDA_CHECK(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kern, threads, smem));
    per_sm[dev] = std::max(1, n);
  }
  return static_cast<int>(std::min<int64_t>((rows + groups - 1) / groups, static_cast<int64_t>(per_sm[dev]) * num_sms(dev)));
}

bool aligned(const at::Tensor& t, size_t bytes) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % bytes == 0; }

}  // namespace

// x [rows, n] fp32 or bf16, ``delta`` (bf16, with an fp32 x): the row is x + delta, returned
// as the first tensor.  -> {x + delta or x, y, mean, rstd}; the statistics only if ``stats``.
std::vector<at::Tensor> add_layernorm_fwd(at::Tensor x, c10::optional<at::Tensor> delta, at::Tensor w,
                                          c10::optional<at::Tensor> b, double eps, bool out_bf16, bool stats) {
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
  at::Tensor mean, rstd;
  if (stats) {
    mean = at::empty({rows}, x.options().dtype(at::kFloat));
    rstd = at::empty({rows}, x.options().dtype(at::kFloat));
  }
  if (rows == 0) return {xo, y, mean, rstd};
  auto s = at::cuda::getCurrentCUDAStream();
  const float* bp = b.has_value() ? b->data_ptr<float>() : nullptr;
  float* xop = delta.has_value() ? xo.data_ptr<float>() : nullptr;
  const int dev = x.device().index();
  float* mp = stats ? mean.data_ptr<float>() : nullptr;
  float* rp = stats ? rstd.data_ptr<float>() : nullptr;
  by_type(x, [&](auto* xp) {
    by_type(y, [&](auto* yp) {
      using TI = std::remove_pointer_t<decltype(xp)>;
      using TO = std::remove_pointer_t<decltype(yp)>;
      // 16 bytes of x at a time where every row starts on such a boundary
      constexpr int V = sizeof(TI) == 4 ? 4 : 8;
      auto launch = [&](auto v, auto add) {
        constexpr int VV = decltype(v)::value;
        constexpr bool ADD = decltype(add)::value;
        return with_plan<VV>(row_plan(n, VV), [&](auto t, auto k) {
          constexpr int T = decltype(t)::value;
          auto kern = ln_fwd_reg_kernel<T, VV, decltype(k)::value, TI, TO, ADD>;
          constexpr int threads = ln_threads(T);
          const int grid = row_blocks(kern, threads, 0, rows, threads / T, dev);
          kern<<<grid, threads, 0, s>>>(xp, dp, w.data_ptr<float>(), bp, xop, yp, mp, rp, (int)rows, (int)n, (float)eps);
        });
      };
      if constexpr (std::is_same_v<TI, __nv_bfloat16> && std::is_same_v<TO, float>) {
        return;  // not a combination this function makes
      } else {
        const bool wide = n % V == 0 && aligned(x, 16) && aligned(y, 16) && (dp == nullptr || aligned(*delta, 8));
        bool done;
        if constexpr (std::is_same_v<TI, float> && std::is_same_v<TO, __nv_bfloat16>)
          done = dp != nullptr ? (wide ? launch(std::integral_constant<int, V>{}, std::true_type{})
                                       : launch(std::integral_constant<int, 1>{}, std::true_type{}))
                               : (wide ? launch(std::integral_constant<int, V>{}, std::false_type{})
                                       : launch(std::integral_constant<int, 1>{}, std::false_type{}));
        else
          done = dp == nullptr && (wide ? launch(std::integral_constant<int, V>{}, std::false_type{})
                                        : launch(std::integral_constant<int, 1>{}, std::false_type{}));
        if (!done)
          ln_fwd_kernel<<<rows, 256, 0, s>>>(xp, dp, w.data_ptr<float>(), bp, xop, yp, mp, rp, (int)n, (float)eps);
      }
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
  const int dev = x.device().index();
  by_type(x, [&](auto* xp) {
    by_type(dy, [&](auto* dyp) {
      using TI = std::remove_pointer_t<decltype(xp)>;
      using TD = std::remove_pointer_t<decltype(dyp)>;
      auto* dxp = static_cast<TI*>(dx.data_ptr());
      constexpr int V = sizeof(TI) == 4 ? 4 : 8;
      auto launch = [&](auto v, auto res) {
        constexpr int VV = decltype(v)::value;
        constexpr bool RES = decltype(res)::value;
        return with_plan<VV>(row_plan(n, VV), [&](auto t, auto k) {
          constexpr int T = decltype(t)::value, K = decltype(k)::value;
          auto kern = ln_bwd_reg_kernel<T, VV, K, TI, TD, RES>;
          constexpr int threads = ln_threads(T);
          constexpr size_t smem = threads > T ? 2 * T * K * VV * sizeof(float) : 0;
          const int grid = row_blocks(kern, threads, smem, rows, threads / T, dev);
          auto part = at::empty({grid, 2, n}, x.options().dtype(at::kFloat));
          kern<<<grid, threads, smem, s>>>(dyp, xp, w.data_ptr<float>(), mean.data_ptr<float>(),
                                           rstd.data_ptr<float>(), dr, dxp, dxb, part.template data_ptr<float>(),
                                           (int)rows, (int)n);
          ln_dw_reduce_kernel<<<(2 * n + 31) / 32, 1024, 0, s>>>(part.template data_ptr<float>(), grid, (int)n,
                                                                dw_out.data_ptr<float>(), dbp, accumulate);
        });
      };
      bool done = false;
      if (rows > 0) {
        if constexpr (std::is_same_v<TI, float>) {
          const bool wide = n % V == 0 && aligned(x, 16) && aligned(dy, 16) && aligned(dx, 16) &&
                            (dr == nullptr || aligned(*dres, 16)) && (dxb == nullptr || aligned(*dx_bf16, 8));
          if (dr != nullptr)
            done = wide ? launch(std::integral_constant<int, V>{}, std::true_type{})
                        : launch(std::integral_constant<int, 1>{}, std::true_type{});
          else if (dxb == nullptr)
            done = wide ? launch(std::integral_constant<int, V>{}, std::false_type{})
                        : launch(std::integral_constant<int, 1>{}, std::false_type{});
        } else if constexpr (std::is_same_v<TD, __nv_bfloat16>) {
          if (dr == nullptr && dxb == nullptr)
            done = n % V == 0 && aligned(x, 16) && aligned(dy, 16) && aligned(dx, 16)
                       ? launch(std::integral_constant<int, V>{}, std::false_type{})
                       : launch(std::integral_constant<int, 1>{}, std::false_type{});
        }
      }
      if (done) return;
      if (rows > 0)
        ln_bwd_dx_kernel<<<rows, 256, 0, s>>>(dyp, xp, w.data_ptr<float>(), mean.data_ptr<float>(),
                                              rstd.data_ptr<float>(), dr, dxp, dxb, (int)n);
      ln_bwd_dw_kernel<<<(n + 31) / 32, 256, 0, s>>>(dyp, xp, mean.data_ptr<float>(), rstd.data_ptr<float>(),
                                                     dw_out.data_ptr<float>(), dbp, (int)rows, (int)n, accumulate);
    });
  });
  PB_CUDA_CHECK(cudaGetLastError());
  return dx;
}

}  // namespace pb
