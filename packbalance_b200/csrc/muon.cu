// Newton-Schulz orthogonalisation of batches of matrices and the Muon update (sm_100a).
//
//   orthogonalize   X0 = U / (|U|_F + eps), then ``steps`` times X <- a X + (b A + c A A) X,
//                   A = X X^T; the result in bf16.
//   muon_update     m += (1 - mu)(s g - m); u = s g + mu (m - s g) with Nesterov, else m;
//                   p = p (1 - lr wd) - lr * 0.2 sqrt(max(rows, cols)) * orthogonalised u,
//                   s = min(1, max_norm / (norm + 1e-6)) the clip factor.
//
// Two passes over the inputs come first: the norm has to be known before the first fp16
// rounding, so pass 1 updates the momentum and sums u^2 per 8192-element chunk, and pass 2
// reads momentum and gradient again, adds up its matrix's chunk sums (in chunk order: no
// atomics, the result does not depend on scheduling) and writes X0 as fp16 high and low parts.
// Both are memory-bound (the 100M model's 75.5M elements, 12 bytes each: 138 and 142 us, 6.6 and
// 6.4 TB/s).  The products follow
// as three launches per step (ns_gemm.cuh).
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include <cooperative_groups.h>

#include <algorithm>
#include <array>
#include <cmath>
#include <map>

#include "common.cuh"
#include "host_utils.h"
#include "ns_gemm.cuh"

namespace pb {
namespace {

namespace cg = cooperative_groups;

constexpr float kXScale = 256.f;   // X is held as 256 X
constexpr float kAScale = 1024.f;  // A and P as 1024 A, 1024 P
constexpr int kChunk = 8192;       // elements per block of the two elementwise passes

struct MatTable {
  const void* g[kNsMats];  // gradients (or the matrices to orthogonalise)
  float* m[kNsMats];       // momenta (null: none)
};
// One shape's share of the elementwise passes.
struct PassGroup {
  int mat0, batch;       // matrices [mat0, mat0 + batch) of the table
  int rows, cols, ld;    // ld: padded row length of X
  long numel;            // rows * cols
  int chunks;            // chunks per matrix
  int block_end;         // running total of blocks
  int part0;             // index of the group's first partial sum
  int vec;               // 4-element accesses allowed
  __half* hi;            // X0 [batch][rows][ld] and its low part (null: none)
  __half* low;
};
struct PassArgs {
  PassGroup g[kNsGroups];
  int groups;
  double* part;
  const float* norm;     // gradient norm (null: no clipping, always update)
  float mu, max_norm, eps;
  int nesterov;
};

__device__ __forceinline__ float4 load4(const float* p) { return *reinterpret_cast<const float4*>(p); }
__device__ __forceinline__ float4 load4(const __nv_bfloat16* p) {
  const uint2 u = *reinterpret_cast<const uint2*>(p);
  const float2 a = unpack_bf16x2(u.x), b = unpack_bf16x2(u.y);
  return make_float4(a.x, a.y, b.x, b.y);
}
__device__ __forceinline__ float load1(const float* p) { return *p; }
__device__ __forceinline__ float load1(const __nv_bfloat16* p) { return __bfloat162float(*p); }

__device__ __forceinline__ double square(float v) { return static_cast<double>(v) * v; }

__device__ __forceinline__ int pass_group(const PassArgs& a, int block, int& local) {
  int g = 0, base = 0;
  while (g + 1 < a.groups && block >= a.g[g].block_end) base = a.g[g++].block_end;
  local = block - base;
  return g;
}

// Sums of squares are held in 64 bits: squares of large or tiny entries neither overflow nor
// vanish, and the passes wait for memory anyway.
__device__ __forceinline__ double block_total(double v, double* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffff, v, o);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x / 32] = v;
  __syncthreads();
  double t = 0.0;
  for (int k = 0; k < static_cast<int>(blockDim.x / 32); ++k) t += red[k];
  return t;
}

// Clip factor; false: the norm is not finite and nothing may change.
__device__ __forceinline__ bool clip_factor(const PassArgs& a, float& s) {
  s = 1.f;
  if (a.norm == nullptr) return true;
  const float n = *a.norm;
  if (!isfinite(n)) return false;
  if (a.max_norm > 0.f) s = fminf(1.f, a.max_norm / (n + 1e-6f));
  return true;
}

__device__ __forceinline__ float momentum(float g, float m, float mu) { return m + (1.f - mu) * (g - m); }
__device__ __forceinline__ float direction(float g, float m, const PassArgs& a) {
  return a.nesterov ? g + a.mu * (m - g) : m;
}

// Pass 1: momentum update and the chunk's sum of squares of the update direction.
template <typename TG, bool MOM>
__global__ void __launch_bounds__(256) ns_norm_kernel(const __grid_constant__ PassArgs a,
                                                       const __grid_constant__ MatTable t) {
  __shared__ double red[8];
  int local;
  const PassGroup& g = a.g[pass_group(a, blockIdx.x, local)];
  float s;
  if (!clip_factor(a, s)) return;
  const int mat = local / g.chunks;
  const long lo = static_cast<long>(local % g.chunks) * kChunk;
  const long hi = min(lo + kChunk, g.numel);
  const TG* gp = static_cast<const TG*>(t.g[g.mat0 + mat]);
  float* mp = MOM ? t.m[g.mat0 + mat] : nullptr;
  double ss = 0.0;
  if (g.vec) {
#pragma unroll 4
    for (long i = lo + threadIdx.x * 4; i < hi; i += 1024) {
      float4 gv = load4(gp + i);
      if constexpr (MOM) {
        float4 mv = load4(mp + i);
        gv.x *= s; gv.y *= s; gv.z *= s; gv.w *= s;
        mv.x = momentum(gv.x, mv.x, a.mu);
        mv.y = momentum(gv.y, mv.y, a.mu);
        mv.z = momentum(gv.z, mv.z, a.mu);
        mv.w = momentum(gv.w, mv.w, a.mu);
        *reinterpret_cast<float4*>(mp + i) = mv;
        gv.x = direction(gv.x, mv.x, a);
        gv.y = direction(gv.y, mv.y, a);
        gv.z = direction(gv.z, mv.z, a);
        gv.w = direction(gv.w, mv.w, a);
      }
      ss += square(gv.x) + square(gv.y) + square(gv.z) + square(gv.w);
    }
  } else {
    for (long i = lo + threadIdx.x; i < hi; i += 256) {
      float u = load1(gp + i);
      if constexpr (MOM) {
        u *= s;
        const float m = momentum(u, mp[i], a.mu);
        mp[i] = m;
        u = direction(u, m, a);
      }
      ss += square(u);
    }
  }
  ss = block_total(ss, red);
  if (threadIdx.x == 0) a.part[g.part0 + local] = ss;
}

// Pass 2: X0 = u / (|u| + eps) as fp16 high and low parts.
template <typename TG, bool MOM>
__global__ void __launch_bounds__(256) ns_init_kernel(const __grid_constant__ PassArgs a,
                                                       const __grid_constant__ MatTable t) {
  __shared__ double red[8];
  int local;
  const PassGroup& g = a.g[pass_group(a, blockIdx.x, local)];
  grid_dependency_wait();
  float s;
  if (!clip_factor(a, s)) return;
  const int mat = local / g.chunks;
  double ss = 0.0;
  for (int k = threadIdx.x; k < g.chunks; k += 256) ss += a.part[g.part0 + mat * g.chunks + k];
  const float scale = static_cast<float>(kXScale / (sqrt(block_total(ss, red)) + a.eps));
  const long lo = static_cast<long>(local % g.chunks) * kChunk;
  const long hi = min(lo + kChunk, g.numel);
  const TG* gp = static_cast<const TG*>(t.g[g.mat0 + mat]);
  const float* mp = MOM ? t.m[g.mat0 + mat] : nullptr;
  const long base = static_cast<long>(mat) * g.rows * g.ld;
  if (g.vec) {
#pragma unroll 4
    for (long i = lo + threadIdx.x * 4; i < hi; i += 1024) {
      float4 u = load4(gp + i);
      if constexpr (MOM) {
        const float4 mv = load4(mp + i);
        u.x = direction(u.x * s, mv.x, a);
        u.y = direction(u.y * s, mv.y, a);
        u.z = direction(u.z * s, mv.z, a);
        u.w = direction(u.w * s, mv.w, a);
      }
      u.x *= scale; u.y *= scale; u.z *= scale; u.w *= scale;
      const long at = base + (g.ld == g.cols ? i : i / g.cols * g.ld + i % g.cols);
      const uint2 h = make_uint2(pack_f16x2(u.x, u.y), pack_f16x2(u.z, u.w));
      *reinterpret_cast<uint2*>(g.hi + at) = h;
      if (g.low != nullptr) {
        const float2 h0 = __half22float2(*reinterpret_cast<const __half2*>(&h.x));
        const float2 h1 = __half22float2(*reinterpret_cast<const __half2*>(&h.y));
        *reinterpret_cast<uint2*>(g.low + at) =
            make_uint2(pack_f16x2((u.x - h0.x) * kNsLowScale, (u.y - h0.y) * kNsLowScale),
                       pack_f16x2((u.z - h1.x) * kNsLowScale, (u.w - h1.y) * kNsLowScale));
      }
    }
  } else {
    for (long i = lo + threadIdx.x; i < hi; i += 256) {
      float u = load1(gp + i);
      if constexpr (MOM) u = direction(u * s, mp[i], a);
      u *= scale;
      const long at = base + i / g.cols * g.ld + i % g.cols;
      const __half h = __float2half_rn(u);
      g.hi[at] = h;
      if (g.low != nullptr) g.low[at] = __float2half_rn((u - __half2float(h)) * kNsLowScale);
    }
  }
}

// ---- small matrices: one block or cluster each, fp32 throughout -------------------
// With 32 rows or fewer the products are too small for tensor-core tiles, and rounding to fp16
// no longer averages out (a 2 x 2 matrix can end 1e-2 off, a 64 x 64 one 1.9e-3).  So the
// blocks of one cluster (1 to 8) hold X, each a slice of the long side (fp32; in shared memory,
// or in ``scratch`` when it does not fit), and run the whole update in one launch: momentum,
// norm, every step, and the store.  The blocks' partial Gram matrices are added in block order
// through distributed shared memory; the polynomial is computed by every block for itself.
// Bound by its passes over shared memory: the Gram phase reads 8 values per 16 multiply-adds, and
// its 36 blocks of 32 rows make three uneven rounds of 16 warps; below a few thousand columns by
// the latency of 15 dependent passes.  Measured: 1 x 32 x 768 78 us, 12 x 16 x 768 31 us,
// 23 x 32 x 3232 202 us, 100 x 8 x 4096 89 us.
//   Gram   a warp takes 4 x 4 blocks of row pairs, its lanes run along the long side
//   apply  a thread takes one column: R values in registers, P from shared memory
struct SmallArgs {
  int rows, cols, steps;
  float a, b, c, eps, mu, max_norm;
  int nesterov;
  float step;          // step length per unit of learning rate (STEP)
  __nv_bfloat16* dst;  // result [batch][rows][cols] (null: update the parameters)
  float* scratch;      // [batch][blocks of a cluster][R][ld] (null: shared memory)
  int slice;           // long-side elements per block
};
constexpr int kSmallRows = 32;
constexpr int kSmallThreads = 512;
__host__ __device__ constexpr int small_ld(int long_side) { return long_side | 1; }

template <int R, typename TG, bool MOM>
__global__ void __launch_bounds__(kSmallThreads)
    ns_small_kernel(const __grid_constant__ SmallArgs a, const __grid_constant__ MatTable t,
                    const __grid_constant__ NsStepArgs st) {
  extern __shared__ float small_smem[];
  __shared__ double red[kSmallThreads / 32], norm_part;
  __shared__ float part[R][R + 1], gram[R][R + 1];
  __shared__ __align__(16) float poly[R][R + 4];
  cg::cluster_group cluster = cg::this_cluster();
  const int blocks = cluster.num_blocks(), rank = cluster.block_rank();
  const int mat = blockIdx.x / blocks, tid = threadIdx.x, lane = tid & 31, warp = tid / 32;
  const bool tall = a.rows > a.cols;
  const unsigned r = tall ? a.cols : a.rows;
  const int total = tall ? a.rows : a.cols, ld = small_ld(a.slice);
  const int c0 = min(rank * a.slice, total), c = min(a.slice, total - c0);  // this block's slice
  float* x = a.scratch != nullptr ? a.scratch + static_cast<long>(blockIdx.x) * R * ld : small_smem;
  // Element ``e`` of the slice, in memory order: its row of X, its column, its place in the matrix.
  struct At {
    int i, j;
    long k;
  };
  auto at = [&](unsigned e) {  // 32-bit divisions: the host keeps slices below 2^26 columns
    if (tall) return At{static_cast<int>(e % r), static_cast<int>(e / r), static_cast<long>(c0) * r + e};
    const int i = static_cast<int>(e / static_cast<unsigned>(c)), j = static_cast<int>(e % static_cast<unsigned>(c));
    return At{i, j, static_cast<long>(i) * a.cols + c0 + j};
  };
  const unsigned elems = static_cast<unsigned>(r) * c;
  float s = 1.f;
  if (st.norm != nullptr) {  // the same for every block of the cluster
    const float n = *st.norm;
    if (!isfinite(n)) return;
    if (a.max_norm > 0.f) s = fminf(1.f, a.max_norm / (n + 1e-6f));
  }
  const TG* gp = static_cast<const TG*>(t.g[mat]);
  double ss = 0.0;
  for (unsigned e = tid; e < elems; e += kSmallThreads) {
    const At q = at(e);
    float u = load1(gp + q.k);
    if constexpr (MOM) {
      u *= s;
      const float m = momentum(u, t.m[mat][q.k], a.mu);
      t.m[mat][q.k] = m;
      u = a.nesterov ? u + a.mu * (m - u) : m;
    }
    ss += square(u);
    x[static_cast<long>(q.i) * ld + q.j] = u;
  }
  for (int k = tid; k < c; k += kSmallThreads)
    for (int i = static_cast<int>(r); i < R; ++i) x[static_cast<long>(i) * ld + k] = 0.f;
  ss = block_total(ss, red);
  if (blocks > 1) {
    if (tid == 0) norm_part = ss;
    cluster.sync();
    ss = 0.0;
    for (int b = 0; b < blocks; ++b) ss += *cluster.map_shared_rank(&norm_part, b);
  }
  const double inv = 1.0 / (sqrt(ss) + a.eps);
  __syncthreads();
  for (int k = tid; k < c; k += kSmallThreads)
    for (int i = 0; i < static_cast<int>(r); ++i) x[static_cast<long>(i) * ld + k] = static_cast<float>(x[static_cast<long>(i) * ld + k] * inv);
  __syncthreads();
  constexpr int RB = R / 4;
  for (int step = 0; step < a.steps; ++step) {
    for (int blk = warp; blk < RB * (RB + 1) / 2; blk += kSmallThreads / 32) {
      int bi = 0, k = blk;
      while (k >= RB - bi) k -= RB - bi++;
      const int bj = bi + k;
      float acc[4][4] = {};
      for (int e = lane; e < c; e += 32) {
        float u[4], v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          u[i] = x[static_cast<long>(4 * bi + i) * ld + e];
          v[i] = x[static_cast<long>(4 * bj + i) * ld + e];
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[i][j] += u[i] * v[j];
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float v = warp_sum(acc[i][j]);
          if (lane == 0) {
            part[4 * bi + i][4 * bj + j] = v;
            part[4 * bj + j][4 * bi + i] = v;
          }
        }
    }
    // every block's partial sums are there; and, before any block writes its next ones, read
    if (blocks > 1) cluster.sync();
    else __syncthreads();
    for (int e = tid; e < R * R; e += kSmallThreads) {
      float v = 0.f;
      if (blocks > 1)
        for (int b = 0; b < blocks; ++b) v += *cluster.map_shared_rank(&part[e / R][e % R], b);
      else v = part[e / R][e % R];
      gram[e / R][e % R] = v;
    }
    if (blocks > 1) cluster.sync();
    else __syncthreads();
    for (int e = tid; e < R * R; e += kSmallThreads) {
      const int i = e / R, j = e % R;
      float v = 0.f;
#pragma unroll
      for (int k = 0; k < R; ++k) v += gram[i][k] * gram[k][j];
      poly[i][j] = a.c * v + a.b * gram[i][j] + (i == j ? a.a : 0.f);
    }
    __syncthreads();
    for (int k = tid; k < c; k += kSmallThreads) {
      float v[R];
#pragma unroll
      for (int i = 0; i < R; ++i) v[i] = x[static_cast<long>(i) * ld + k];
#pragma unroll 4
      for (int i = 0; i < R; ++i) {
        float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int j = 0; j < R; j += 4) {
          const float4 w = *reinterpret_cast<const float4*>(&poly[i][j]);
          y.x += w.x * v[j];
          y.y += w.y * v[j + 1];
          y.z += w.z * v[j + 2];
          y.w += w.w * v[j + 3];
        }
        x[static_cast<long>(i) * ld + k] = (y.x + y.y) + (y.z + y.w);
      }
    }
    __syncthreads();
  }
  float lr = 0.f, decay = 1.f;
  if (a.dst == nullptr) {
    lr = st.hp != nullptr ? *st.hp : st.lr;
    decay = 1.f - lr * st.weight_decay;
  }
  const long numel = static_cast<long>(a.rows) * a.cols;
  for (unsigned e = tid; e < elems; e += kSmallThreads) {
    const At q = at(e);
    const float o = x[static_cast<long>(q.i) * ld + q.j];
    if (a.dst != nullptr) {
      a.dst[mat * numel + q.k] = __float2bfloat16_rn(o);
    } else {
      const float w = st.p[mat][q.k] * decay - lr * a.step * o;
      st.p[mat][q.k] = w;
      if (st.shadow[mat] != nullptr) st.shadow[mat][q.k] = __float2bfloat16_rn(w);
    }
  }
}

// AdamW on chosen ranges of flat buffers (the parameters Muon does not take); the second
// moment has its own, compact buffer.
struct AdamRange {
  long at, numel, v_at;
};
constexpr int kAdamRanges = 512;
struct AdamRanges {
  AdamRange r[kAdamRanges];
  int count;
};
constexpr int kAdamChunk = 4096;

__global__ void __launch_bounds__(256) adamw_ranges_kernel(
    const __grid_constant__ AdamRanges rs, float* __restrict__ p, const float* __restrict__ g, float* __restrict__ m,
    float* __restrict__ v, __nv_bfloat16* __restrict__ shadow, const float* __restrict__ norm,
    int* __restrict__ skipped, float lr, float b1, float b2, float eps, float wd, float bc1, float bc2, float max_norm,
    const float* __restrict__ hp) {
  if (hp != nullptr) {
    lr = hp[0];
    bc1 = hp[1];
    bc2 = hp[2];
  }
  const float nv = *norm;
  const bool bad = !isfinite(nv);
  if (blockIdx.x == 0 && threadIdx.x == 0) *skipped = bad ? 1 : 0;
  if (bad) return;
  const float gs = max_norm > 0.f ? fminf(1.f, max_norm / (nv + 1e-6f)) : 1.f;
  const float step = lr / bc1, inv_sqrt_bc2 = rsqrtf(bc2), decay = 1.f - lr * wd;
  long chunk = blockIdx.x;
  for (int k = 0; k < rs.count; ++k) {
    const AdamRange r = rs.r[k];
    const long n = (r.numel + kAdamChunk - 1) / kAdamChunk;
    for (; chunk < n; chunk += gridDim.x) {
      const long hi = min((chunk + 1) * kAdamChunk, r.numel);
      for (long i = chunk * kAdamChunk + threadIdx.x; i < hi; i += 256) {
        const long at = r.at + i;
        const float gk = g[at] * gs;
        const float mk = b1 * m[at] + (1.f - b1) * gk;
        const float vk = b2 * v[r.v_at + i] + (1.f - b2) * gk * gk;
        const float w = p[at] * decay - step * mk / (sqrtf(vk) * inv_sqrt_bc2 + eps);
        m[at] = mk;
        v[r.v_at + i] = vk;
        p[at] = w;
        if (shadow != nullptr) shadow[at] = __float2bfloat16_rn(w);
      }
    }
    chunk -= n;
  }
}

// ------------------------------------ host ----------------------------------------
CUtensorMap map3(const void* ptr, CUtensorMapDataType type, int64_t cols, int64_t rows, int64_t batch, int64_t ld,
                 uint32_t box, CUtensorMapSwizzle swizzle) {
  CUtensorMap m;
  cuuint64_t dims[3] = {(cuuint64_t)cols, (cuuint64_t)rows, (cuuint64_t)batch};
  cuuint64_t strides[2] = {(cuuint64_t)ld * 2, (cuuint64_t)(rows * ld) * 2};
  cuuint32_t boxes[3] = {box, box, 1};
  cuuint32_t estr[3] = {1, 1, 1};
  CUresult r = tmap_encoder()(&m, type, 3, const_cast<void*>(ptr), dims, strides, boxes, estr,
                              CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  TORCH_CHECK(r == CUDA_SUCCESS, "newton-schulz: tensor map of ", batch, " x ", rows, " x ", cols, " failed (",
              static_cast<int>(r), ")");
  return m;
}
CUtensorMap load_map(const __half* p, int64_t cols, int64_t rows, int64_t batch, int64_t ld) {
  return map3(p, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, cols, rows, batch, ld, 64, CU_TENSOR_MAP_SWIZZLE_128B);
}
CUtensorMap store_map(const void* p, int64_t cols, int64_t rows, int64_t batch, int64_t ld, bool bf16) {
  return map3(p, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, cols, rows, batch, ld, 32,
              CU_TENSOR_MAP_SWIZZLE_64B);
}

// Matrices of one shape and where the iteration keeps them.
struct Shape {
  int64_t rows = 0, cols = 0;
  std::vector<int> mats;  // indices into the caller's matrix list
  int64_t batch() const { return static_cast<int64_t>(mats.size()); }
  int64_t r() const { return std::min(rows, cols); }
  int64_t ld() const { return (cols + 7) / 8 * 8; }
  int64_t ldr() const { return (r() + 7) / 8 * 8; }
  bool tall() const { return rows > cols; }
  int64_t bytes() const { return 2 * (3 * rows * ld() + 2 * r() * ldr()); }  // workspace of one matrix
  __half *x[2] = {nullptr, nullptr}, *low = nullptr, *gram = nullptr, *poly = nullptr;
};

template <int CG, int MODE, class Step>
void ns_launch(const NsArgs& args, const Step& step, int dev, cudaStream_t stream) {
  using C = NsCfg<CG>;
  auto kern = ns_gemm_kernel<CG, MODE, Step>;
  static int max_clusters[64] = {0};
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;  // see grid_dependency_wait
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = CG;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg{};
  cfg.blockDim = dim3(C::THREADS, 1, 1);
  cfg.dynamicSmemBytes = C::SMEM_BYTES;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = CG == 2 ? 2 : 1;
  if (max_clusters[dev] == 0) {
    PB_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM_BYTES));
    int n = num_sms(dev) / CG;
    if (CG == 2) {
      cfg.gridDim = dim3(2 * n, 1, 1);
      PB_CUDA_CHECK(cudaOccupancyMaxActiveClusters(&n, kern, &cfg));
    }
    max_clusters[dev] = std::max(1, n);
  }
  cfg.gridDim = pb::smem_max(kern, dim3(CG * std::min(args.tiles, max_clusters[dev]), 1, 1));
  PB_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kern, args, step));
}

// Tile counts of every group; returns the total.
template <int CG, bool SYM>
int64_t count_tiles(NsArgs& a) {
  constexpr int T = NsCfg<CG>::T;
  int64_t total = 0;
  for (int k = 0; k < a.groups; ++k) {
    NsGroup& g = a.g[k];
    const int tm = (g.M + T - 1) / T, tn = (g.N + T - 1) / T;
    int64_t per = static_cast<int64_t>(tm) * tn;
    if (SYM) {
      per = 0;
      for (int i = 0; i < tm; ++i) per += tn - ns_first_col<CG>(i);
    }
    TORCH_CHECK(per < (1LL << 31), "newton-schulz: too many tiles");
    g.tiles_n = tn;
    g.tiles_per_mat = static_cast<int>(per);
    total += per * g.batch;
    TORCH_CHECK(total < (1LL << 31), "newton-schulz: too many tiles");
    g.tile_end = static_cast<int>(total);
  }
  a.tiles = static_cast<int>(total);
  return total;
}

template <int MODE, class Step>
void ns_product(NsArgs& a, const Step& step, int dev, cudaStream_t s) {
  constexpr bool SYM = MODE == NS_GRAM || MODE == NS_POLY;
  // A 256-wide tile on a CTA pair and a 128-wide tile on one CTA take the same time (the pair's
  // tensor cores finish a k-block in the time in which one CTA's 32 KB of operands arrive), so
  // the smaller number of waves wins, and at equal numbers the smaller tiles, whose epilogue is
  // half as long.
  const int64_t sms = num_sms(dev), pairs = sms / 2;
  const int64_t waves2 = (count_tiles<2, SYM>(a) + pairs - 1) / pairs, waves1 = (count_tiles<1, SYM>(a) + sms - 1) / sms;
  if (waves1 <= waves2) {
    ns_launch<1, MODE, Step>(a, step, dev, s);
  } else {
    count_tiles<2, SYM>(a);
    ns_launch<2, MODE, Step>(a, step, dev, s);
  }
}

struct Iteration {
  int steps;
  float a, b, c;
};

// The products on prepared X0; ``last`` fills the last product's groups and launches it.
template <class Last>
void ns_iterate(std::vector<Shape>& shapes, const Iteration& it, int dev, cudaStream_t s, Last&& last) {
  NsArgs gram{}, poly{}, apply{};
  const int n = static_cast<int>(shapes.size());
  gram.groups = poly.groups = apply.groups = n;
  gram.status = poly.status = apply.status = status_ptr(dev);
  gram.alpha = kAScale / (kXScale * kXScale);
  poly.alpha = it.c / kAScale;
  poly.beta = it.b;
  poly.diag = it.a * kAScale;
  apply.alpha = 1.f / kAScale;
  apply.beta = it.a / kNsLowScale;
  for (int k = 0, at = 0; k < n; ++k) {
    gram.g[k].batch = poly.g[k].batch = apply.g[k].batch = (int)shapes[k].batch();
    apply.g[k].mat0 = at;
    at += (int)shapes[k].batch();
  }
  // everything but which of the two X buffers is read is the same in every step
  std::vector<std::array<CUtensorMap, 2>> x_load(n), x_store(n);
  for (int k = 0; k < n; ++k) {
    Shape& sh = shapes[k];
    const int64_t r = sh.r(), B = sh.batch();
    for (int i = 0; i < (it.steps > 1 ? 2 : 1); ++i) {
      x_load[k][i] = load_map(sh.x[i], sh.cols, sh.rows, B, sh.ld());
      x_store[k][i] = store_map(sh.x[i], sh.cols, sh.rows, B, sh.ld(), false);
    }
    NsGroup& g = gram.g[k];
    g.a_mn = g.b_mn = sh.tall();
    g.M = g.N = (int)r;
    g.K = (int)std::max(sh.rows, sh.cols);
    g.out = store_map(sh.gram, r, r, B, sh.ldr(), false);
    NsGroup& q = poly.g[k];
    q.a = q.b = load_map(sh.gram, r, r, B, sh.ldr());
    q.out = store_map(sh.poly, r, r, B, sh.ldr(), false);
    q.add = sh.gram;
    q.add_batch = r * sh.ldr();
    q.add_ld = (int)sh.ldr();
    q.a_sym = q.b_sym = 1;
    q.M = q.N = q.K = (int)r;
    NsGroup& y = apply.g[k];
    (sh.tall() ? y.b : y.a) = load_map(sh.poly, r, r, B, sh.ldr());
    y.a_sym = !sh.tall();
    y.b_sym = sh.tall();
    y.b_mn = !sh.tall();
    y.M = (int)sh.rows;
    y.N = (int)sh.cols;
    y.K = (int)r;
    y.add_batch = sh.rows * sh.ld();
    y.add_ld = (int)sh.ld();
    if (it.steps > 3) y.low = store_map(sh.low, sh.cols, sh.rows, B, sh.ld(), false);
    for (NsGroup* p : {&g, &q, &y}) p->k_blocks = (p->K + 63) / 64;
  }
  for (int step = 0, cur = 0; step < it.steps; ++step, cur ^= 1) {
    const bool final = step + 1 == it.steps;
    for (int k = 0; k < n; ++k) {
      gram.g[k].a = gram.g[k].b = x_load[k][cur];
      NsGroup& y = apply.g[k];
      (shapes[k].tall() ? y.a : y.b) = x_load[k][cur];
      // the input carries a low part while at least two steps follow this one
      y.add = step + 2 < it.steps ? shapes[k].low : nullptr;
      y.store_low = step + 3 < it.steps;
      if (!final) y.out = x_store[k][cur ^ 1];
    }
    ns_product<NS_GRAM>(gram, NsNoStep{}, dev, s);
    ns_product<NS_POLY>(poly, NsNoStep{}, dev, s);
    if (!final) ns_product<NS_APPLY>(apply, NsNoStep{}, dev, s);
    else {
      apply.alpha = 1.f / (kAScale * kXScale);
      last(apply);
    }
  }
}

// Matrices go through the iteration in parts of at most this much workspace (one at least).  Without
// a bound the hidden matrices of an 8B decoder would take 50 GB at once, and a captured step keeps
// what it took.  Measured, four layers of such a decoder: 57.0 ms without a bound, 56.6 with 2 GB,
// 57.3 with 1 GB, 58.2 with 256 MB; eight layers of a 1.1B one: 13.2, 13.4, 13.6 and 14.5 ms.
constexpr int64_t kNsWorkspace = 2LL << 30;
// Workspace of each of the fewest, equally large parts of ``total`` bytes.
int64_t part_bytes(int64_t total) {
  const int64_t parts = std::max<int64_t>(1, (total + kNsWorkspace - 1) / kNsWorkspace);
  return (total + parts - 1) / parts;
}

// Workspace of one run: X twice, its low part, the Gram and polynomial matrices of every
// shape, and the partial sums.  From the caller's stream-ordered allocator.
at::Tensor make_workspace(std::vector<Shape>& shapes, const Iteration& it, int64_t partials, const at::Tensor& like,
                          double*& part) {
  int64_t bytes = 0;
  auto take = [&](int64_t n) {
    const int64_t at = bytes;
    bytes += (n + 255) / 256 * 256;
    return at;
  };
  std::vector<std::array<int64_t, 5>> at(shapes.size());
  for (size_t k = 0; k < shapes.size(); ++k) {
    const Shape& s = shapes[k];
    const int64_t xb = s.batch() * s.rows * s.ld() * 2, ab = s.batch() * s.r() * s.ldr() * 2;
    at[k] = {take(xb), it.steps > 1 ? take(xb) : 0, it.steps > 2 ? take(xb) : -1, take(ab), take(ab)};
  }
  const int64_t pat = take(partials * 8);
  auto ws = at::empty({bytes}, like.options().dtype(at::kByte));
  uint8_t* base = static_cast<uint8_t*>(ws.data_ptr());
  for (size_t k = 0; k < shapes.size(); ++k) {
    Shape& s = shapes[k];
    s.x[0] = reinterpret_cast<__half*>(base + at[k][0]);
    s.x[1] = reinterpret_cast<__half*>(base + at[k][1]);
    s.low = at[k][2] < 0 ? nullptr : reinterpret_cast<__half*>(base + at[k][2]);
    s.gram = reinterpret_cast<__half*>(base + at[k][3]);
    s.poly = reinterpret_cast<__half*>(base + at[k][4]);
  }
  part = reinterpret_cast<double*>(base + pat);
  return ws;
}

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

// Elementwise passes over ``shapes`` (tables in shape order).
template <typename TG, bool MOM>
void ns_passes(PassArgs& a, const MatTable& t, int blocks, cudaStream_t s) {
  ns_norm_kernel<TG, MOM><<<blocks, 256, 0, s>>>(a, t);
  PB_CUDA_CHECK(cudaGetLastError());
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(blocks, 1, 1);
  cfg.blockDim = dim3(256, 1, 1);
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  PB_CUDA_CHECK(cudaLaunchKernelEx(&cfg, ns_init_kernel<TG, MOM>, a, t));
}

int64_t chunks_of(const Shape& s) { return (s.rows * s.cols + kChunk - 1) / kChunk; }

int fill_passes(PassArgs& a, const std::vector<Shape>& shapes, const MatTable& t, bool mom, bool bf16) {
  int64_t blocks = 0;
  int mat0 = 0;
  a.groups = static_cast<int>(shapes.size());
  for (size_t k = 0; k < shapes.size(); ++k) {
    const Shape& s = shapes[k];
    PassGroup& g = a.g[k];
    g.mat0 = mat0;
    g.batch = (int)s.batch();
    g.rows = (int)s.rows;
    g.cols = (int)s.cols;
    g.ld = (int)s.ld();
    g.numel = s.rows * s.cols;
    g.chunks = (int)chunks_of(s);
    g.part0 = (int)blocks;
    blocks += s.batch() * chunks_of(s);
    g.block_end = (int)blocks;
    g.hi = s.x[0];
    g.low = s.low;
    // 4 elements at a time: whole rows of such pieces and aligned tables
    bool vec = s.cols % 4 == 0;
    for (int i = 0; i < g.batch; ++i)
      vec = vec && reinterpret_cast<uintptr_t>(t.g[mat0 + i]) % (bf16 ? 8 : 16) == 0 &&
            (!mom || aligned16(t.m[mat0 + i]));
    g.vec = vec;
    mat0 += g.batch;
  }
  TORCH_CHECK(blocks < (1LL << 31), "newton-schulz: too many elements");
  return static_cast<int>(blocks);
}

// Whether a shape goes to the one-block kernel.
bool is_small(int64_t rows, int64_t cols) { return std::min(rows, cols) <= kSmallRows; }

template <int R, typename TG, bool MOM>
void launch_small(SmallArgs a, const MatTable& t, const NsStepArgs& st, int batch, const at::Tensor& like,
                  cudaStream_t s) {
  const int64_t side = std::max(a.rows, a.cols);
  auto bytes = [&](int blocks) { return R * small_ld((side + blocks - 1) / blocks) * sizeof(float); };
  constexpr size_t kMost = 200 * 1024;
  // more blocks per matrix while each still has 256 columns and the GPU has room for them, or
  // until the slices fit in shared memory
  const int64_t sms = num_sms(like.device().index());
  int blocks = 1;
  while (blocks < 8 && side > 256 * blocks && (2 * blocks * batch <= 2 * sms || bytes(blocks) > kMost)) blocks *= 2;
  TORCH_CHECK((side + blocks - 1) / blocks < (1LL << 26), "newton-schulz: ", side, " is too long for a matrix of ",
              std::min(a.rows, a.cols), " rows");
  a.slice = static_cast<int>((side + blocks - 1) / blocks);
  size_t smem = bytes(blocks);
  at::Tensor scratch;
  if (smem > kMost) {
    scratch = at::empty({batch * blocks * static_cast<int64_t>(smem / sizeof(float))}, like.options().dtype(at::kFloat));
    a.scratch = scratch.data_ptr<float>();
    smem = 0;
  }
  auto kern = ns_small_kernel<R, TG, MOM>;
  if (smem > 32 * 1024)
    PB_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kMost));
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = blocks;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(batch * blocks, 1, 1);
  cfg.blockDim = dim3(kSmallThreads, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  PB_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kern, a, t, st));
}

template <typename TG, bool MOM>
void run_small(const SmallArgs& a, const MatTable& t, const NsStepArgs& st, int batch, const at::Tensor& like,
               cudaStream_t s) {
  const int r = std::min(a.rows, a.cols);
  if (r <= 8) launch_small<8, TG, MOM>(a, t, st, batch, like, s);
  else if (r <= 16) launch_small<16, TG, MOM>(a, t, st, batch, like, s);
  else launch_small<32, TG, MOM>(a, t, st, batch, like, s);
}

Iteration check_iteration(int64_t steps, const std::vector<double>& coef) {
  TORCH_CHECK(steps >= 1 && steps <= 100, "newton-schulz: steps must be 1 to 100, got ", steps);
  TORCH_CHECK(coef.size() == 3, "newton-schulz: three coefficients");
  for (double c : coef) TORCH_CHECK(std::isfinite(c), "newton-schulz: coefficients must be finite");
  return Iteration{(int)steps, (float)coef[0], (float)coef[1], (float)coef[2]};
}

// Memory that one call writes must not be listed twice, nor read as a gradient.
using Ranges = std::vector<std::pair<uintptr_t, uintptr_t>>;
void check_disjoint(Ranges ranges, const Ranges& reads) {
  std::sort(ranges.begin(), ranges.end());
  for (size_t k = 1; k < ranges.size(); ++k)
    TORCH_CHECK(ranges[k - 1].second <= ranges[k].first,
                "muon_update: parameters, momenta and shadows must not overlap or be listed twice");
  for (const auto& r : reads) {
    const auto next = std::upper_bound(ranges.begin(), ranges.end(), r);
    TORCH_CHECK((next == ranges.end() || r.second <= next->first) &&
                    (next == ranges.begin() || std::prev(next)->second <= r.first),
                "muon_update: gradients must not overlap parameters, momenta or shadows");
  }
}

// Cost of one matrix of a shape, to place the longest work first.
double shape_cost(const Shape& s) { return double(s.r()) * s.r() * std::max(s.rows, s.cols); }

}  // namespace

// x [batch, rows, cols] fp32 or bf16, contiguous -> the orthogonalised matrices, bf16.
at::Tensor ns_orthogonalize(at::Tensor x, int64_t steps, std::vector<double> coef, double eps) {
  TORCH_CHECK(x.is_cuda() && x.dim() == 3 && x.is_contiguous(),
              "orthogonalize: x must be a contiguous CUDA tensor [batch, rows, cols]");
  const bool bf16 = x.scalar_type() == at::kBFloat16;
  TORCH_CHECK(bf16 || x.scalar_type() == at::kFloat, "orthogonalize: x must be fp32 or bf16");
  TORCH_CHECK(x.size(1) < (1LL << 30) && x.size(2) < (1LL << 30), "orthogonalize: matrix too large");
  const Iteration it = check_iteration(steps, coef);
  const c10::cuda::CUDAGuard guard(x.device());
  auto out = at::empty(x.sizes(), x.options().dtype(at::kBFloat16));
  if (x.numel() == 0) return out;
  const int dev = x.device().index();
  auto s = at::cuda::getCurrentCUDAStream();
  const int64_t rows = x.size(1), cols = x.size(2), numel = rows * cols;
  Shape shape;
  shape.rows = rows;
  shape.cols = cols;
  const int64_t one = shape.bytes(), fit = (part_bytes(x.size(0) * one) + one - 1) / one;
  const int64_t most = is_small(rows, cols) ? kNsMats : std::min<int64_t>(kNsMats, fit);
  for (int64_t b0 = 0, nb; b0 < x.size(0); b0 += nb) {
    nb = std::min(most, x.size(0) - b0);
    std::vector<Shape> shapes(1, shape);
    MatTable t{};
    for (int64_t i = 0; i < nb; ++i) {
      shapes[0].mats.push_back((int)i);
      t.g[i] = static_cast<const char*>(x.data_ptr()) + (b0 + i) * numel * x.element_size();
    }
    if (is_small(rows, cols)) {
      SmallArgs sa{(int)rows, (int)cols, it.steps, it.a, it.b, it.c, (float)eps, 0.f, 0.f, 0, 0.f,
                   static_cast<__nv_bfloat16*>(out.data_ptr()) + b0 * numel, nullptr};
      if (bf16) run_small<__nv_bfloat16, false>(sa, t, NsStepArgs{}, (int)nb, x, s);
      else run_small<float, false>(sa, t, NsStepArgs{}, (int)nb, x, s);
      continue;
    }
    PassArgs pa{};
    auto ws = make_workspace(shapes, it, nb * chunks_of(shapes[0]), x, pa.part);
    pa.eps = (float)eps;
    const int blocks = fill_passes(pa, shapes, t, false, bf16);
    if (bf16) ns_passes<__nv_bfloat16, false>(pa, t, blocks, s);
    else ns_passes<float, false>(pa, t, blocks, s);
    ns_iterate(shapes, it, dev, s, [&](NsArgs& a) {
      NsGroup& g = a.g[0];
      g.dst = static_cast<__nv_bfloat16*>(out.data_ptr()) + b0 * numel;
      g.dst_tma = cols % 8 == 0 && aligned16(g.dst);
      if (g.dst_tma) g.out = store_map(g.dst, cols, rows, nb, cols, true);
      ns_product<NS_LAST>(a, NsNoStep{}, dev, s);
    });
  }
  return out;
}

// In-place Muon update of matrices given as lists of contiguous fp32 tensors [..., rows, cols]
// (leading dimensions count matrices).  ``shadows``: bf16 copies to refresh, or empty.
// ``norm`` (fp32 device scalar): gradient norm for clipping to ``max_norm`` and the skip when
// it is not finite.  ``hp`` (fp32, device): learning rate read on the device.
void muon_update(std::vector<at::Tensor> params, std::vector<at::Tensor> grads, std::vector<at::Tensor> momenta,
                 std::vector<at::Tensor> shadows, double lr, double mu, bool nesterov, double weight_decay,
                 int64_t steps, std::vector<double> coef, double eps, c10::optional<at::Tensor> norm, double max_norm,
                 c10::optional<at::Tensor> hp) {
  const size_t n = params.size();
  TORCH_CHECK(grads.size() == n && momenta.size() == n && (shadows.empty() || shadows.size() == n),
              "muon_update: ", n, " parameters, ", grads.size(), " gradients, ", momenta.size(), " momenta, ",
              shadows.size(), " shadows");
  const Iteration it = check_iteration(steps, coef);
  if (n == 0) return;
  const auto device = params[0].device();
  auto scalar_ok = [&](const at::Tensor& t) {
    return t.is_cuda() && t.device() == device && t.scalar_type() == at::kFloat && t.numel() >= 1;
  };
  TORCH_CHECK(!norm.has_value() || scalar_ok(*norm), "muon_update: norm must be an fp32 scalar on the parameters' device");
  TORCH_CHECK(!hp.has_value() || scalar_ok(*hp), "muon_update: hp must be fp32 on the parameters' device");
  std::map<std::pair<int64_t, int64_t>, Shape> by_shape;
  struct Mat {
    float* p;
    const float* g;
    float* m;
    __nv_bfloat16* sh;
  };
  std::vector<Mat> mats;
  Ranges written, read;
  auto note = [](Ranges& to, const at::Tensor& t) {
    const auto lo = reinterpret_cast<uintptr_t>(t.data_ptr());
    if (t.numel() > 0) to.emplace_back(lo, lo + t.numel() * t.element_size());
  };
  for (size_t k = 0; k < n; ++k) {
    const at::Tensor &p = params[k], &g = grads[k], &m = momenta[k];
    for (const at::Tensor* t : {&p, &g, &m})
      TORCH_CHECK(t->is_cuda() && t->device() == device && t->scalar_type() == at::kFloat && t->is_contiguous() &&
                      t->dim() >= 2 && t->sizes() == p.sizes(),
                  "muon_update: entry ", k, " must be contiguous fp32 [..., rows, cols] tensors of one shape on one device");
    const int64_t rows = p.size(-2), cols = p.size(-1), numel = rows * cols;
    TORCH_CHECK(rows < (1LL << 30) && cols < (1LL << 30), "muon_update: matrix too large");
    __nv_bfloat16* sh = nullptr;
    if (!shadows.empty()) {
      const at::Tensor& w = shadows[k];
      TORCH_CHECK(w.is_cuda() && w.device() == device && w.scalar_type() == at::kBFloat16 && w.is_contiguous() &&
                      w.numel() == p.numel(),
                  "muon_update: shadow ", k, " must be contiguous bf16 of its parameter's size");
      sh = static_cast<__nv_bfloat16*>(w.data_ptr());
      note(written, w);
    }
    note(written, p);
    note(written, m);
    note(read, g);
    if (p.numel() == 0) continue;
    Shape& s = by_shape[{rows, cols}];
    s.rows = rows;
    s.cols = cols;
    for (int64_t i = 0; i < p.numel() / numel; ++i) {
      s.mats.push_back((int)mats.size());
      mats.push_back({p.data_ptr<float>() + i * numel, g.data_ptr<float>() + i * numel, m.data_ptr<float>() + i * numel,
                      sh == nullptr ? nullptr : sh + i * numel});
    }
  }
  check_disjoint(std::move(written), read);
  const c10::cuda::CUDAGuard guard(device);
  const int dev = device.index();
  auto s = at::cuda::getCurrentCUDAStream();
  auto table = [&](const std::vector<Shape>& shapes, MatTable& t, NsStepArgs& st) {
    int at = 0;
    for (const Shape& sh : shapes)
      for (int i : sh.mats) {
        t.g[at] = mats[i].g;
        t.m[at] = mats[i].m;
        st.p[at] = mats[i].p;
        st.shadow[at] = mats[i].sh;
        ++at;
      }
    st.norm = norm.has_value() ? norm->data_ptr<float>() : nullptr;
    st.hp = hp.has_value() ? hp->data_ptr<float>() : nullptr;
    st.lr = (float)lr;
    st.weight_decay = (float)weight_decay;
  };
  auto step_length = [](const Shape& sh) { return 0.2f * std::sqrt((float)std::max(sh.rows, sh.cols)); };
  std::vector<Shape> all;
  for (auto& [key, shape] : by_shape) {
    if (!is_small(shape.rows, shape.cols)) {
      all.push_back(std::move(shape));
      continue;
    }
    for (size_t i = 0; i < shape.mats.size(); i += kNsMats) {
      std::vector<Shape> one(1);
      one[0].rows = shape.rows;
      one[0].cols = shape.cols;
      one[0].mats.assign(shape.mats.begin() + i, shape.mats.begin() + std::min(i + kNsMats, shape.mats.size()));
      MatTable t{};
      NsStepArgs st{};
      table(one, t, st);
      run_small<float, true>(SmallArgs{(int)shape.rows, (int)shape.cols, it.steps, it.a, it.b, it.c, (float)eps,
                                       (float)mu, (float)max_norm, nesterov, step_length(shape), nullptr, nullptr},
                             t, st, (int)one[0].batch(), params[0], s);
    }
  }
  // longest tiles first, so that the last wave is made of short ones
  std::sort(all.begin(), all.end(), [](const Shape& x, const Shape& y) { return shape_cost(x) > shape_cost(y); });
  // launches take kNsGroups shapes, kNsMats matrices and kNsWorkspace bytes at a time
  int64_t total = 0;
  for (const Shape& sh : all) total += sh.batch() * sh.bytes();
  const int64_t target = part_bytes(total);
  size_t k = 0, used = 0;
  while (k < all.size()) {
    std::vector<Shape> shapes;
    int64_t room = kNsMats, partials = 0, bytes = 0;
    while (k < all.size() && shapes.size() < (size_t)kNsGroups && room > 0 && bytes < target) {
      const int64_t one = all[k].bytes(), left = all[k].batch() - (int64_t)used;
      int64_t take = std::min({room, left, (target - bytes + one - 1) / one});
      if (bytes + take * one > kNsWorkspace) take = (kNsWorkspace - bytes) / one;
      if (take <= 0) {
        if (!shapes.empty()) break;
        take = 1;  // larger than the bound by itself
      }
      bytes += take * one;
      Shape part;
      part.rows = all[k].rows;
      part.cols = all[k].cols;
      part.mats.assign(all[k].mats.begin() + used, all[k].mats.begin() + used + take);
      partials += part.batch() * chunks_of(part);
      shapes.push_back(std::move(part));
      room -= take;
      used += take;
      if (used == all[k].mats.size()) {
        ++k;
        used = 0;
      }
    }
    MatTable t{};
    NsStepArgs st{};
    table(shapes, t, st);
    PassArgs pa{};
    auto ws = make_workspace(shapes, it, partials, params[0], pa.part);
    pa.norm = st.norm;
    pa.mu = (float)mu;
    pa.max_norm = (float)max_norm;
    pa.eps = (float)eps;
    pa.nesterov = nesterov;
    const int blocks = fill_passes(pa, shapes, t, true, false);
    ns_passes<float, true>(pa, t, blocks, s);
    ns_iterate(shapes, it, dev, s, [&](NsArgs& a) {
      for (int j = 0; j < a.groups; ++j)
        {
        NsGroup& g = a.g[j];
        g.step = step_length(shapes[j]);
        g.vec = g.N % 4 == 0;
        for (int i = 0; i < g.batch; ++i)
          g.vec = g.vec && aligned16(st.p[g.mat0 + i]) && reinterpret_cast<uintptr_t>(st.shadow[g.mat0 + i]) % 8 == 0;
      }
      ns_product<NS_STEP>(a, st, dev, s);
    });
  }
}

// AdamW on ranges [at, at + numel) of the flat buffers, second moments at v_at of ``v``:
// ``ranges`` is at, numel, v_at repeated.
void adamw_ranges(at::Tensor p, at::Tensor g, at::Tensor m, at::Tensor v, c10::optional<at::Tensor> shadow,
                  std::vector<int64_t> ranges, at::Tensor norm, at::Tensor skipped, double lr, double b1, double b2,
                  double eps, double wd, double bc1, double bc2, double max_norm, c10::optional<at::Tensor> hp) {
  for (const at::Tensor* t : {&p, &g, &m, &v})
    TORCH_CHECK(t->is_cuda() && t->device() == p.device() && t->scalar_type() == at::kFloat && t->is_contiguous(),
                "adamw_ranges: contiguous fp32 CUDA buffers on one device");
  TORCH_CHECK(g.numel() == p.numel() && m.numel() == p.numel(), "adamw_ranges: buffers of one size");
  TORCH_CHECK(!shadow.has_value() || (shadow->device() == p.device() && shadow->scalar_type() == at::kBFloat16 &&
                                      shadow->is_contiguous() && shadow->numel() == p.numel()),
              "adamw_ranges: bf16 shadow of the same size");
  TORCH_CHECK(norm.device() == p.device() && norm.scalar_type() == at::kFloat && norm.numel() == 1 &&
                  skipped.device() == p.device() && skipped.scalar_type() == at::kInt && skipped.numel() == 1,
              "adamw_ranges: fp32 norm and int32 skipped scalars on the buffers' device");
  TORCH_CHECK(!hp.has_value() || (hp->device() == p.device() && hp->scalar_type() == at::kFloat && hp->numel() >= 3),
              "adamw_ranges: hp holds lr and the two bias corrections");
  TORCH_CHECK(ranges.size() % 3 == 0, "adamw_ranges: ranges are triples");
  for (size_t k = 0; k < ranges.size(); k += 3)
    TORCH_CHECK(ranges[k] >= 0 && ranges[k + 1] >= 0 && ranges[k + 2] >= 0 && ranges[k] + ranges[k + 1] <= p.numel() &&
                    ranges[k + 2] + ranges[k + 1] <= v.numel(),
                "adamw_ranges: range ", k / 3, " is outside its buffers");
  const c10::cuda::CUDAGuard guard(p.device());
  auto s = at::cuda::getCurrentCUDAStream();
  size_t k = 0;
  do {  // at least one launch: it writes ``skipped``
    AdamRanges rs{};
    int64_t chunks = 0;
    for (; k < ranges.size() && rs.count < kAdamRanges; k += 3) {
      rs.r[rs.count++] = {ranges[k], ranges[k + 1], ranges[k + 2]};
      chunks += (ranges[k + 1] + kAdamChunk - 1) / kAdamChunk;
    }
    const int grid = (int)std::max<int64_t>(1, std::min<int64_t>(chunks, 8L * num_sms(p.device().index())));
    adamw_ranges_kernel<<<grid, 256, 0, s>>>(
        rs, p.data_ptr<float>(), g.data_ptr<float>(), m.data_ptr<float>(), v.data_ptr<float>(),
        shadow.has_value() ? static_cast<__nv_bfloat16*>(shadow->data_ptr()) : nullptr, norm.data_ptr<float>(),
        skipped.data_ptr<int>(), (float)lr, (float)b1, (float)b2, (float)eps, (float)wd, (float)bc1, (float)bc2,
        (float)max_norm, hp.has_value() ? hp->data_ptr<float>() : nullptr);
    PB_CUDA_CHECK(cudaGetLastError());
  } while (k < ranges.size());
}

}  // namespace pb
