// Layer normalisation (sm_100a), forward and backward, with the residual add fused.
//
//   mu = mean(x), r = 1 / sqrt(mean((x - mu)^2) + eps), xh = (x - mu) r, y = xh w + b
//   dx = r (g - mean(g) - xh mean(g xh)) [+ dres],  g = dy w
//   dw = sum over rows of dy xh,  db = sum over rows of dy
//
// The variance is taken around the row's own mean (a second pass over the row).  The mean is the
// unevaluated sum of two floats: the sum of the row over n, and the mean of the differences from
// that.  A row whose offset is far larger than its spread has a first part that is off by a few of
// its own last places, and at an offset of 1e4 one of those is 1e-3; the second part takes that out
// again.  Statistics, sums and gradients are fp32; only the stored activations are rounded to the
// caller's type.  Every sum has a fixed order (no
// atomics), so two runs on the same inputs agree bit for bit.
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include <type_traits>
#include <utility>

#include "common.cuh"
#include "host_utils.h"

namespace pb {
namespace {

__device__ __forceinline__ float ldf(const float* p) { return *p; }
__device__ __forceinline__ float ldf(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ void stf(float* p, float v) { *p = v; }
__device__ __forceinline__ void stf(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

// ---- rows held in registers --------------------------------------------------------
// T threads hold a row, K pieces of V elements each, so a row is read once; rows are dealt to a
// persistent grid.  Weight, bias and the backward's column sums stay in registers over all of a
// thread's rows.  What bounds both directions is HBM, and what has to be right for that is bytes
// in flight.  Rows whose every operand starts on a 16-byte boundary arrive by bulk copies in a
// ring of shared-memory slots (RING), several rows ahead; other rows come one element at a time
// through registers (V = 1), one row ahead.
// Measured (B200): 16384 x 4096 bf16 forward 51.5 us (5.2 TB/s, 0.80 of the measured copy), backward
// with the column sums 82 us (4.9 TB/s); 8192 x 768 with the residual add 14.6 us (5.2 TB/s, partly L2),
// its backward from an fp32 dy 24.7 us; 4001 x 1409 fp32 12.5 and 18 us.
// The backward holds weight, column sums, xh and g besides the row: at 512 threads with a residual
// gradient (above 6144 columns) and at 1024 (above 8192) not all of that fits, and it spills:
// 16384 x 8192 fp32 with a residual gradient 507 us (4.2 TB/s; bf16 without one 150 us, 5.4 TB/s),
// 8192 x 12288 fp32 420 us (2.9 TB/s), bf16 1050 us (0.6 TB/s).
//
// Arithmetic is on pairs of fp32 (one instruction each on sm_100a): one element at a time the
// kernels issued 18 and 25 instructions per element and waited for those, not for HBM.
struct f2 {
  unsigned long long v;
};
__device__ __forceinline__ f2 mk2(float a, float b) {
  f2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 un2(f2 p) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(p.v));
  return r;
}
__device__ __forceinline__ f2 add2(f2 a, f2 b) {
  f2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ f2 mul2(f2 a, f2 b) {
  f2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ f2 fma2(f2 a, f2 b, f2 c) {
  f2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
__device__ __forceinline__ float sum2(f2 p) {
  const float2 q = un2(p);
  return q.x + q.y;
}

template <typename T_, int V>
struct Piece;  // V consecutive elements as loaded
template <>
struct Piece<float, 4> {
  float4 r;
  __device__ __forceinline__ void load(const float* p) { r = *reinterpret_cast<const float4*>(p); }
  __device__ __forceinline__ void get(float* v) const { v[0] = r.x; v[1] = r.y; v[2] = r.z; v[3] = r.w; }
};
template <>
struct Piece<__nv_bfloat16, 4> {
  uint2 r;
  __device__ __forceinline__ void load(const __nv_bfloat16* p) { r = *reinterpret_cast<const uint2*>(p); }
  __device__ __forceinline__ void get(float* v) const {
    const float2 a = unpack_bf16x2(r.x), b = unpack_bf16x2(r.y);
    v[0] = a.x; v[1] = a.y; v[2] = b.x; v[3] = b.y;
  }
};
template <>
struct Piece<__nv_bfloat16, 8> {
  uint4 r;
  __device__ __forceinline__ void load(const __nv_bfloat16* p) { r = *reinterpret_cast<const uint4*>(p); }
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

// A mean of this many deviations gets its second part; below, the first part's error is a few
// times 2^-24 of the deviation.  For every row the forward would take 55.9 instead of 51.5 us at
// 16384 x 4096 bf16, where it waits for its instructions.
constexpr float kFarMean = 8.f;

// 1 / sqrt(var + eps) from the mean square of the differences from a mean that is off by ``dmu``.
// (The rounded difference may be below zero; NaN stays.)
__device__ __forceinline__ float rstd_of(float msq, float dmu, float eps) {
  const float var = fmaf(-dmu, dmu, msq);
  return rsqrtf((var < 0.f ? 0.f : var) + eps);
}

constexpr int ln_threads(int t) { return t < 256 ? 256 : t; }

// Sums of N (1 or 2) values over the T threads of a row, in a fixed order; every thread gets them.
// ``red``: 2 N T / 32 floats of this group, its halves used in turn (``flip``), so that one
// barrier per call is enough.
template <int T, int N>
__device__ __forceinline__ void row_sums(float (&v)[N], float* red, int& flip) {
  const int t = threadIdx.x % T, lane = t & 31;
  if constexpr (N == 2) {
    // the lower half of the warp goes on with the first sum, the upper half with the second
    const bool up = lane >= 16;
    float a = (up ? v[1] : v[0]) + __shfl_xor_sync(0xffffffff, up ? v[0] : v[1], 16);
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) a += __shfl_xor_sync(0xffffffff, a, o);
    v[0] = a;  // lanes 0 and 16 hold the sums
    if constexpr (T == 32) {
      v[0] = __shfl_sync(0xffffffff, a, 0);
      v[1] = __shfl_sync(0xffffffff, a, 16);
    }
  } else {
    v[0] = warp_sum(v[0]);
  }
  if constexpr (T > 32) {
    constexpr int W = T / 32;
    float* r = red + flip * N * W;
    flip ^= 1;
    if (lane % (32 / N) == 0) r[lane / (32 / N) * W + t / 32] = v[0];
    if constexpr (T >= 256) __syncthreads();
    else asm volatile("bar.sync %0, %1;" ::"r"(1 + static_cast<int>(threadIdx.x) / T), "n"(T) : "memory");
#pragma unroll
    for (int i = 0; i < N; ++i) {
      v[i] = 0.f;
      if constexpr (W % 4 == 0) {
#pragma unroll
        for (int k = 0; k < W; k += 4) {
          const float4 q = *reinterpret_cast<const float4*>(r + i * W + k);
          v[i] += (q.x + q.y) + (q.z + q.w);
        }
      } else {
#pragma unroll
        for (int k = 0; k < W; ++k) v[i] += r[i * W + k];
      }
    }
  }
}

// One group's ring: ``slots`` slots of one row each (up to three operands back to back), filled
// by the group's first thread.  A slot is refilled after a barrier that every thread reaches with
// the slot's row in registers, so it needs no barrier of its own for that.
struct RowRing {
  uint64_t* full;
  uint8_t* base;
  int slots, slot_bytes, slot;
  uint32_t phase;
  __device__ __forceinline__ void init(uint8_t* smem, int groups, int grp, int n_slots, int bytes) {
    slots = n_slots;
    slot_bytes = bytes;
    slot = 0;
    phase = 0;
    full = reinterpret_cast<uint64_t*>(smem) + grp * n_slots;
    base = smem + ((groups * n_slots * 8 + 15) & ~15) + static_cast<long>(grp) * n_slots * bytes;
  }
  __device__ __forceinline__ uint8_t* row() { return base + slot * slot_bytes; }
  // The slot's row has landed (bounded; a timeout is recorded and the row's values are undefined).
  __device__ __forceinline__ void wait(int* status) { mbar_wait(full + slot, phase, status, 601, nullptr); }
  __device__ __forceinline__ void next() {
    if (++slot == slots) {
      slot = 0;
      phase ^= 1;
    }
  }
};

template <int T, int V, int K, typename TI, typename TO, bool ADD>
__global__ void __launch_bounds__(ln_threads(T))
    ln_fwd_reg_kernel(const TI* __restrict__ xp, const __nv_bfloat16* __restrict__ delta, const float* __restrict__ w,
                      const float* __restrict__ b, float* __restrict__ x_out, TO* __restrict__ y,
                      float* __restrict__ mean, float* __restrict__ rstd, int rows, int n, float eps, int slots,
                      int* status) {
  constexpr int G = ln_threads(T) / T;
  constexpr bool RING = V > 1;
  constexpr int P = K * V / 2;  // pairs
  const float inv_n = 1.f / n;
  __shared__ __align__(16) float red[G][2 * (T / 32)];
  extern __shared__ __align__(16) uint8_t ring_smem[];
  const int t = threadIdx.x % T, grp = threadIdx.x / T;
  int flip = 0;
  const long stride = static_cast<long>(gridDim.x) * G;
  long row = static_cast<long>(blockIdx.x) * G + grp;
  RowRing ring;
  const int xb = n * static_cast<int>(sizeof(TI)), db = ADD ? n * 2 : 0;
  auto refill = [&](int slot, long r) {
    mbar_arrive_expect_tx(ring.full + slot, xb + db);
    uint8_t* d = ring.base + slot * ring.slot_bytes;
    bulk_load(d, xp + r * n, xb, ring.full + slot);
    if constexpr (ADD) bulk_load(d + xb, delta + r * n, db, ring.full + slot);
  };
  if constexpr (RING) {
    ring.init(ring_smem, G, grp, slots, xb + db);
    if (t == 0) {
      for (int k = 0; k < slots; ++k) mbar_init(ring.full + k, 1);
      fence_mbar_init();
      for (int k = 0; k < slots; ++k)
        if (row + k * stride < rows) refill(k, row + k * stride);
    }
    __syncthreads();
  }
  f2 wv[P], bv[P];
#pragma unroll
  for (int i = 0; i < P; ++i) {
    float a[2], c2[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int j = 2 * i + e, c = (j / V * T + t) * V + j % V;
      a[e] = c < n ? w[c] : 0.f;
      c2[e] = c < n && b != nullptr ? b[c] : 0.f;
    }
    wv[i] = mk2(a[0], a[1]);
    bv[i] = mk2(c2[0], c2[1]);
  }
  Piece<TI, V> px[K];
  Piece<__nv_bfloat16, V> pd[ADD ? K : 1];
  auto fetch = [&](const TI* xr, const __nv_bfloat16* dr) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = (k * T + t) * V;
      if (c < n) {
        px[k].load(xr + c);
        if constexpr (ADD) pd[k].load(dr + c);
      }
    }
  };
  if (!RING && row < rows) fetch(xp + row * n, delta + row * n);
  for (; row < rows; row += stride) {
    if constexpr (RING) {
      ring.wait(status);
      fetch(reinterpret_cast<const TI*>(ring.row()), reinterpret_cast<const __nv_bfloat16*>(ring.row() + xb));
    }
    f2 v[P];
    f2 acc = mk2(0.f, 0.f);
    {
      float u[K * V];
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const int c = (k * T + t) * V;
        if (c < n) {
          px[k].get(u + k * V);
          if constexpr (ADD) {
            float d[V];
            pd[k].get(d);
#pragma unroll
            for (int e = 0; e < V; ++e) u[k * V + e] += d[e];
            put<V>(x_out + row * n + c, u + k * V);
          }
        } else {
#pragma unroll
          for (int e = 0; e < V; ++e) u[k * V + e] = 0.f;
        }
      }
#pragma unroll
      for (int i = 0; i < P; ++i) {
        v[i] = mk2(u[2 * i], u[2 * i + 1]);
        acc = add2(acc, v[i]);
      }
    }
    if (!RING && row + stride < rows) fetch(xp + (row + stride) * n, delta + (row + stride) * n);
    float s[1] = {sum2(acc)};
    row_sums<T>(s, red[grp], flip);
    if constexpr (RING) {
      if constexpr (T == 32) __syncwarp();
      if (t == 0 && row + ring.slots * stride < rows) refill(ring.slot, row + ring.slots * stride);
      ring.next();
    }
    const float mu = s[0] * inv_n;
    const f2 minus = mk2(-mu, -mu);
    acc = mk2(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < P; ++i) {
      v[i] = add2(v[i], minus);
      // a pair lies in one piece, or (V = 1) in two, the second of which may be past the row
      constexpr bool split = V == 1;
      if ((2 * i / V * T + t) * V < n) {
        if (split && ((2 * i + 1) * T + t) >= n) {
          const float a = un2(v[i]).x;
          acc = fma2(mk2(a, 0.f), mk2(a, 0.f), acc);
        } else {
          acc = fma2(v[i], v[i], acc);
        }
      }
    }
    s[0] = sum2(acc);
    row_sums<T>(s, red[grp], flip);
    const float msq = s[0] * inv_n;
    float dmu = 0.f, r = rsqrtf(msq + eps);
    if (fabsf(mu) * r > kFarMean) {  // the same for all threads of the row
      acc = mk2(0.f, 0.f);
#pragma unroll
      for (int i = 0; i < P; ++i) {
        if ((2 * i / V * T + t) * V < n) {
          const bool half = V == 1 && (2 * i + 1) * T + t >= n;
          acc = add2(acc, half ? mk2(un2(v[i]).x, 0.f) : v[i]);
        }
      }
      s[0] = sum2(acc);
      row_sums<T>(s, red[grp], flip);
      dmu = s[0] * inv_n;
      r = rstd_of(msq, dmu, eps);
    }
    if (t == 0 && mean != nullptr) {
      mean[2 * row] = mu;
      mean[2 * row + 1] = dmu;
      rstd[row] = r;
    }
    const f2 r2 = mk2(r, r), dr = mk2(-dmu * r, -dmu * r);
    float o[K * V];
#pragma unroll
    for (int i = 0; i < P; ++i) {
      const float2 q = un2(fma2(fma2(v[i], r2, dr), wv[i], bv[i]));
      o[2 * i] = q.x;
      o[2 * i + 1] = q.y;
    }
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = (k * T + t) * V;
      if (c < n) put<V>(y + row * n + c, o + k * V);
    }
  }
}

// ``part``: [gridDim.x][2][n], this block's sums for dw and db.
template <int T, int V, int K, typename TI, typename TD, bool RES>
__global__ void __launch_bounds__(ln_threads(T))
    ln_bwd_reg_kernel(const TD* __restrict__ dy, const TI* __restrict__ x, const float* __restrict__ w,
                      const float* __restrict__ mean, const float* __restrict__ rstd, const float* __restrict__ dres,
                      TI* __restrict__ dx, __nv_bfloat16* __restrict__ dx_bf16, float* __restrict__ part, int rows,
                      int n, int slots, int* status) {
  constexpr int G = ln_threads(T) / T;
  constexpr bool RING = V > 1;
  constexpr int P = K * V / 2;  // pairs
  const float inv_n = 1.f / n;
  __shared__ __align__(16) float red[G][4 * (T / 32)];
  extern __shared__ __align__(16) uint8_t ring_smem[];
  // [2][T * K * V] after the last row (G > 1), in the slots' memory; not over the ring's mbarriers,
  // whose memory may not be used otherwise while they are valid
  float* cols = reinterpret_cast<float*>(ring_smem + (RING ? (G * slots * 8 + 15) & ~15 : 0));
  const int t = threadIdx.x % T, grp = threadIdx.x / T;
  int flip = 0;
  const long stride = static_cast<long>(gridDim.x) * G;
  long row = static_cast<long>(blockIdx.x) * G + grp;
  RowRing ring;
  const int xb = n * static_cast<int>(sizeof(TI)), gb = n * static_cast<int>(sizeof(TD)), rb = RES ? n * 4 : 0;
  auto refill = [&](int slot, long r) {
    mbar_arrive_expect_tx(ring.full + slot, xb + gb + rb);
    uint8_t* d = ring.base + slot * ring.slot_bytes;
    bulk_load(d, x + r * n, xb, ring.full + slot);
    bulk_load(d + xb, dy + r * n, gb, ring.full + slot);
    if constexpr (RES) bulk_load(d + xb + gb, dres + r * n, rb, ring.full + slot);
  };
  if constexpr (RING) {
    ring.init(ring_smem, G, grp, slots, xb + gb + rb);
    if (t == 0) {
      for (int k = 0; k < slots; ++k) mbar_init(ring.full + k, 1);
      fence_mbar_init();
      for (int k = 0; k < slots; ++k)
        if (row + k * stride < rows) refill(k, row + k * stride);
    }
    __syncthreads();
  }
  f2 wv[P], aw[P], ab[P];
#pragma unroll
  for (int i = 0; i < P; ++i) {
    float a[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int j = 2 * i + e, c = (j / V * T + t) * V + j % V;
      a[e] = c < n ? w[c] : 0.f;
    }
    wv[i] = mk2(a[0], a[1]);
    aw[i] = ab[i] = mk2(0.f, 0.f);
  }
  Piece<TI, V> px[K];
  Piece<TD, V> pg[K];
  Piece<float, V == 8 ? 4 : V> pr[RES ? K : 1];
  auto fetch = [&](const TI* xr, const TD* gr, const float* rr) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = (k * T + t) * V;
      if (c < n) {
        px[k].load(xr + c);
        pg[k].load(gr + c);
        if constexpr (RES) pr[k].load(rr + c);
      }
    }
  };
  float mu_n = 0.f, dmu_n = 0.f, r_n = 0.f;
  if (row < rows) {
    mu_n = mean[2 * row];
    dmu_n = mean[2 * row + 1];
    r_n = rstd[row];
    if (!RING) fetch(x + row * n, dy + row * n, dres + row * n);
  }
  for (; row < rows; row += stride) {
    const float mu = mu_n, r = r_n, dmu_r = -dmu_n * r_n;
    if constexpr (RING) {
      ring.wait(status);
      const uint8_t* q = ring.row();
      fetch(reinterpret_cast<const TI*>(q), reinterpret_cast<const TD*>(q + xb),
            reinterpret_cast<const float*>(q + xb + gb));
    }
    const long after = row + stride;
    if (after < rows) {
      mu_n = mean[2 * after];
      dmu_n = mean[2 * after + 1];
      r_n = rstd[after];
    }
    f2 xh[P], g[P];
    float res[RES ? K * V : 1];
    f2 a1 = mk2(0.f, 0.f), a2 = mk2(0.f, 0.f);
    {
      const f2 r2 = mk2(r, r), dr = mk2(dmu_r, dmu_r);
      float u[K * V], q[K * V];
#pragma unroll
      for (int k = 0; k < K; ++k) {
        if ((k * T + t) * V < n) {
          px[k].get(u + k * V);
          pg[k].get(q + k * V);
          if constexpr (RES) pr[k].get(res + k * V);
        } else {
#pragma unroll
          for (int e = 0; e < V; ++e) {
            u[k * V + e] = 0.f;
            q[k * V + e] = 0.f;
          }
        }
      }
      if (!RING && after < rows) fetch(x + after * n, dy + after * n, dres + after * n);
#pragma unroll
      for (int i = 0; i < P; ++i) {
        // (x - mu) r - dmu r, the difference rounded first: x r - mu r would lose a row's common offset
        const f2 d = add2(mk2(u[2 * i], u[2 * i + 1]), mk2(-mu, -mu));
        xh[i] = fma2(d, r2, dr);
        g[i] = mk2(q[2 * i], q[2 * i + 1]);
        const f2 t2 = mul2(g[i], xh[i]);
        aw[i] = add2(aw[i], t2);
        ab[i] = add2(ab[i], g[i]);
        a1 = fma2(g[i], wv[i], a1);
        a2 = fma2(t2, wv[i], a2);
      }
    }
    float s[2] = {sum2(a1), sum2(a2)};
    row_sums<T>(s, red[grp], flip);
    if constexpr (RING) {
      if constexpr (T == 32) __syncwarp();
      if (t == 0 && row + ring.slots * stride < rows) refill(ring.slot, row + ring.slots * stride);
      ring.next();
    }
    // dx = g w r - xh (r s2 / n) - r s1 / n
    const float m1 = -r * (s[0] * inv_n), m2 = -r * (s[1] * inv_n);
    const f2 r2 = mk2(r, r), c1 = mk2(m1, m1), c2 = mk2(m2, m2);
    float o[K * V];
#pragma unroll
    for (int i = 0; i < P; ++i) {
      const float2 q = un2(fma2(mul2(g[i], wv[i]), r2, fma2(xh[i], c2, c1)));
      o[2 * i] = q.x;
      o[2 * i + 1] = q.y;
      if constexpr (RES) {
        o[2 * i] += res[2 * i];
        o[2 * i + 1] += res[2 * i + 1];
      }
    }
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = (k * T + t) * V;
      if (c < n) {
        put<V>(dx + row * n + c, o + k * V);
        if constexpr (sizeof(TI) == 4) {
          if (dx_bf16 != nullptr) put<V>(dx_bf16 + row * n + c, o + k * V);
        }
      }
    }
  }
  float fw[K * V], fb[K * V];
#pragma unroll
  for (int i = 0; i < P; ++i) {
    const float2 p = un2(aw[i]), q = un2(ab[i]);
    fw[2 * i] = p.x;
    fw[2 * i + 1] = p.y;
    fb[2 * i] = q.x;
    fb[2 * i + 1] = q.y;
  }
  if constexpr (G > 1) {  // the groups' sums, added in group order
    __syncthreads();      // the ring's memory is free
    float* cw = cols;
    float* cb = cols + T * K * V;
    for (int q = 0; q < G; ++q) {
      if (grp == q) {
#pragma unroll
        for (int i = 0; i < K * V; ++i) {
          cw[i * T + t] = q == 0 ? fw[i] : cw[i * T + t] + fw[i];
          cb[i * T + t] = q == 0 ? fb[i] : cb[i * T + t] + fb[i];
        }
      }
      __syncthreads();
    }
    if (grp != 0) return;
#pragma unroll
    for (int i = 0; i < K * V; ++i) {
      fw[i] = cw[i * T + t];
      fb[i] = cb[i * T + t];
    }
  }
  float* pw = part + static_cast<long>(blockIdx.x) * 2 * n;
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const int c = (k * T + t) * V + e;
      if (c < n) {
        pw[c] = fw[k * V + e];
        pw[n + c] = fb[k * V + e];
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
  s = 0.f;
  for (int c = threadIdx.x; c < n; c += blockDim.x) {
    const float d = value(c) - mu;
    s += d;
    ss += d * d;
  }
  const float dmu = block_sum(s, red) / n;
  const float r = rstd_of(block_sum(ss, red) / n, dmu, eps);
  if (threadIdx.x == 0 && mean != nullptr) {
    mean[2 * row] = mu;
    mean[2 * row + 1] = dmu;
    rstd[row] = r;
  }
  for (int c = threadIdx.x; c < n; c += blockDim.x)
    stf(y + off + c, ((value(c) - mu) - dmu) * r * w[c] + (b != nullptr ? b[c] : 0.f));
}

template <typename TI, typename TD>
__global__ void ln_bwd_dx_kernel(const TD* __restrict__ dy, const TI* __restrict__ x, const float* __restrict__ w,
                                 const float* __restrict__ mean, const float* __restrict__ rstd,
                                 const float* __restrict__ dres, TI* __restrict__ dx,
                                 __nv_bfloat16* __restrict__ dx_bf16, int n) {
  __shared__ float red[32];
  const long row = blockIdx.x;
  const long off = row * n;
  const float mu = mean[2 * row], dmu = mean[2 * row + 1], r = rstd[row];
  float s1 = 0.f, s2 = 0.f;
  for (int c = threadIdx.x; c < n; c += blockDim.x) {
    const float g = ldf(dy + off + c) * w[c];
    s1 += g;
    s2 += g * (((ldf(x + off + c) - mu) - dmu) * r);
  }
  s1 = block_sum(s1, red) / n;
  s2 = block_sum(s2, red) / n;
  for (int c = threadIdx.x; c < n; c += blockDim.x) {
    const float g = ldf(dy + off + c) * w[c];
    const float xh = ((ldf(x + off + c) - mu) - dmu) * r;
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
      sw += d * (((ldf(x + at) - mean[2L * row]) - mean[2L * row + 1]) * rstd[row]);
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

// Threads per row T and pieces per thread K for n elements in pieces of V, at most E elements
// per thread: the fewest threads that hold the row (a row's sums cost each thread about 30
// instructions however few elements it has), then the smallest compiled K.
template <int V, int E, typename F>
bool with_plan(int64_t n, F&& f) {
  constexpr int most = E / V;
  const int64_t pieces = (n + V - 1) / V;
  int T = 32;
  while (T < 1024 && pieces > static_cast<int64_t>(T) * most) T *= 2;
  const int64_t K = (pieces + T - 1) / T;
  if (K > most) return false;
  auto with_t = [&](auto t) {
    constexpr int TT = decltype(t)::value;
    if (T != TT) return false;
    auto try_k = [&](auto k) {
      constexpr int KK = decltype(k)::value;
      if constexpr (KK < 1 || KK > most || KK * V % 2 != 0) return false;
      else {
        if (K > KK) return false;
        f(t, k);
        return true;
      }
    };
    // a row longer than 32 threads hold fills more than half of the pieces: half as many threads
    // would hold it otherwise
    if constexpr (TT == 32) {
      if (try_k(std::integral_constant<int, most / 8>{}) || try_k(std::integral_constant<int, most / 4>{}) ||
          try_k(std::integral_constant<int, most / 2>{}))
        return true;
    }
    if constexpr (most * 3 / 4 > most / 2) {
      if (try_k(std::integral_constant<int, most * 3 / 4>{})) return true;
    }
    return try_k(std::integral_constant<int, most>{});
  };
  return with_t(std::integral_constant<int, 32>{}) || with_t(std::integral_constant<int, 64>{}) ||
         with_t(std::integral_constant<int, 128>{}) || with_t(std::integral_constant<int, 256>{}) ||
         with_t(std::integral_constant<int, 512>{}) || with_t(std::integral_constant<int, 1024>{});
}
// Elements per thread.  At 16384 x 4096 bf16 16 measured 50 us forward and 86 us backward where 8
// took 74 and 124 (the sums' cost per element) and 32 took 68 and 105 (too few resident rows).
constexpr int kFwdElems = 16, kBwdElems = 16;

// Shape of a persistent launch: ring slots per group, shared memory and blocks.  64 KB of slots
// per block of 256 threads: with 32 KB the backward at 16384 x 4096 took 115 us instead of 87 (one
// row ahead), with 104 KB no less than with 64.
struct RowLaunch {
  int slots, blocks;
  size_t smem;
};
constexpr int kRingBytes = 64 * 1024;
constexpr int kRingMost = 220 * 1024;
template <auto Kern>
RowLaunch row_launch(int threads, int groups, int64_t row_bytes, size_t least, int64_t rows, int dev) {
  RowLaunch l{0, 0, least};
  if (row_bytes > 0) {
    const int64_t one = groups * (row_bytes + 8);
    const int64_t room = std::min(kRingBytes * (threads / 256), kRingMost - 64);
    l.slots = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(8, room / one)));
    TORCH_CHECK(l.slots * one <= kRingMost - 64, "layernorm: row of ", row_bytes, " bytes does not fit");
    l.smem = std::max(least, static_cast<size_t>(groups * l.slots * row_bytes)) + (groups * l.slots * 8 + 15) / 16 * 16;
  }
  static int most[64] = {0};  // of this kernel
  // 48 KB need no opt-in, but they include the kernel's static arrays (at most 512 bytes)
  if (l.smem > 47 * 1024 && most[dev] == 0) {
    PB_CUDA_CHECK(cudaFuncSetAttribute(Kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kRingMost));
    most[dev] = 1;
  }
  // resident blocks at the shared-memory size last asked for (the query costs as much as a launch)
  thread_local std::pair<size_t, int> resident[64] = {};
  int& n = resident[dev].second;
  if (n == 0 || resident[dev].first != l.smem) {
    resident[dev].first = l.smem;
    PB_CUDA_CHECK(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, Kern, threads, l.smem));
  }
  l.blocks = static_cast<int>(std::min<int64_t>((rows + groups - 1) / groups,
                                                static_cast<int64_t>(std::max(1, n)) * num_sms(dev)));
  return l;
}

bool aligned(const at::Tensor& t, size_t bytes) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % bytes == 0; }

}  // namespace

// x [rows, n] fp32 or bf16, ``delta`` (bf16, with an fp32 x): the row is x + delta, returned
// as the first tensor.  -> {x + delta or x, y, mean [rows, 2], rstd [rows]}: the row's mean is the sum
// of its two floats.  The statistics only if ``stats``.
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
    mean = at::empty({rows, 2}, x.options().dtype(at::kFloat));
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
        return with_plan<VV, kFwdElems>(n, [&](auto t, auto k) {
          constexpr int T = decltype(t)::value;
          constexpr auto kern = ln_fwd_reg_kernel<T, VV, decltype(k)::value, TI, TO, ADD>;
          constexpr int threads = ln_threads(T);
          const int64_t row_bytes = VV > 1 ? n * (int64_t)(sizeof(TI) + (ADD ? 2 : 0)) : 0;
          const RowLaunch l = row_launch<kern>(threads, threads / T, row_bytes, 0, rows, dev);
          kern<<<l.blocks, threads, l.smem, s>>>(xp, dp, w.data_ptr<float>(), bp, xop, yp, mp, rp, (int)rows, (int)n,
                                                 (float)eps, l.slots, status_ptr(dev));
        });
      };
      // a bf16 x is normalised into bf16 and has no delta (checked above)
      constexpr bool XF = sizeof(TI) == 4, YF = sizeof(TO) == 4;
      bool done = false;
      if constexpr (XF || !YF) {
        const bool wide = n % (dp == nullptr ? V : 8) == 0 && aligned(x, 16) && aligned(y, 16) &&
                          (dp == nullptr || aligned(*delta, 16));
        if constexpr (XF && !YF) {
          if (dp != nullptr)
            done = wide ? launch(std::integral_constant<int, V>{}, std::true_type{})
                        : launch(std::integral_constant<int, 1>{}, std::true_type{});
        }
        if (dp == nullptr)
          done = wide ? launch(std::integral_constant<int, V>{}, std::false_type{})
                      : launch(std::integral_constant<int, 1>{}, std::false_type{});
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
  check_vec(mean, 2 * rows, x, "mean");
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
  TORCH_CHECK(x.scalar_type() == at::kFloat ||
                  (dy.scalar_type() == at::kBFloat16 && !dres.has_value() && !dx_bf16.has_value()),
              "layernorm: a bf16 x has a bf16 dy, no dres and no dx_bf16");
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
        return with_plan<VV, kBwdElems>(n, [&](auto t, auto k) {
          constexpr int T = decltype(t)::value, K = decltype(k)::value;
          constexpr auto kern = ln_bwd_reg_kernel<T, VV, K, TI, TD, RES>;
          constexpr int threads = ln_threads(T);
          constexpr size_t least = threads > T ? 2 * T * K * VV * sizeof(float) : 0;
          const int64_t row_bytes = VV > 1 ? n * (int64_t)(sizeof(TI) + sizeof(TD) + (RES ? 4 : 0)) : 0;
          const RowLaunch l = row_launch<kern>(threads, threads / T, row_bytes, least, rows, dev);
          auto part = at::empty({l.blocks, 2, n}, x.options().dtype(at::kFloat));
          kern<<<l.blocks, threads, l.smem, s>>>(dyp, xp, w.data_ptr<float>(), mean.data_ptr<float>(),
                                           rstd.data_ptr<float>(), dr, dxp, dxb, part.template data_ptr<float>(),
                                           (int)rows, (int)n, l.slots, status_ptr(dev));
          ln_dw_reduce_kernel<<<(2 * n + 31) / 32, 1024, 0, s>>>(part.template data_ptr<float>(), l.blocks, (int)n,
                                                                dw_out.data_ptr<float>(), dbp, accumulate);
        });
      };
      constexpr bool XF = sizeof(TI) == 4, DF = sizeof(TD) == 4;
      if constexpr (XF || !DF) {  // checked above
        const bool wide = n % (DF ? V : 8) == 0 && aligned(x, 16) && aligned(dy, 16) && aligned(dx, 16) &&
                          (dr == nullptr || aligned(*dres, 16)) && (dxb == nullptr || aligned(*dx_bf16, 8));
        bool done = false;
        if constexpr (XF) {
          if (rows > 0 && dr != nullptr)
            done = wide ? launch(std::integral_constant<int, V>{}, std::true_type{})
                        : launch(std::integral_constant<int, 1>{}, std::true_type{});
        }
        // (the bf16 dy of an fp32 x comes with a residual gradient: the sum's two results)
        if constexpr (XF == DF) {
          if (rows > 0 && dr == nullptr)
            done = wide ? launch(std::integral_constant<int, V>{}, std::false_type{})
                        : launch(std::integral_constant<int, 1>{}, std::false_type{});
        }
        if (done) return;
        if (rows > 0)
          ln_bwd_dx_kernel<<<rows, 256, 0, s>>>(dyp, xp, w.data_ptr<float>(), mean.data_ptr<float>(),
                                                rstd.data_ptr<float>(), dr, dxp, dxb, (int)n);
        ln_bwd_dw_kernel<<<(n + 31) / 32, 256, 0, s>>>(dyp, xp, mean.data_ptr<float>(), rstd.data_ptr<float>(),
                                                       dw_out.data_ptr<float>(), dbp, (int)rows, (int)n, accumulate);
      }
    });
  });
  PB_CUDA_CHECK(cudaGetLastError());
  return dx;
}

}  // namespace pb
