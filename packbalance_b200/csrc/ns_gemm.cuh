// Batched tcgen05 products of the Newton-Schulz iteration (sm_100a).
//
// One step on a matrix X [m, n] is, with r = min(m, n),
//
//   A = X X^T (wide, m <= n) or X^T X (tall)      GRAM    r x r, symmetric
//   P = a I + b A + c A A                         POLY    r x r, symmetric
//   X <- P X (wide) or X P (tall)                 APPLY / LAST / STEP   m x n
//
// A launch does one of these products for every matrix of up to kNsGroups groups; a group is
// a set of matrices of one shape, stored back to back, so one 3-D tensor map addresses all of
// them and its bounds zero-fill ragged edges.  X is never transposed: both operands of a
// tcgen05.mma may be K-major or MN-major, and the group says which.
//
// Numbers.  Operands are fp16 (11 significant bits; bf16 iterates lose an order of magnitude
// against the 64-bit iteration), held at fixed power-of-two scales that keep everything the
// iteration produces (|X| <= ~1.2, |A| <= ~1.5, |P| <= 3.5 in the 2-norm) in fp16's normal
// range.  Accumulation is fp32.  Small singular values grow 3.4-fold per step, and with them
// the rounding of X in the directions X hardly has: so the early iterates carry their
// rounding error as a second fp16 matrix ``low`` (scaled by 2^11, which makes it about as large as
// X's own values), which enters through the linear term, X' = P hi + a low.  Simulated against 64
// bits over Gaussian matrices, power-law spectra and one to sixteen dominant directions plus noise,
// the result is off by at most 3.7e-3 of its norm from 64 rows on (Gaussian 1.9e-3) and 5.2e-3
// for 33 to 63 rows, where fewer roundings average out.  ``low`` in e4m3 takes 2 to 6 % less
// time (the 100M model's update 1.69 instead of 1.77 ms) and is off by up to 5.1e-3 with one
// dominant direction; without it 4e-2.
//
// Kernel structure: that of the CTA-pair GEMM (gemm_pair.cuh), whose barrier and abort
// protocol is kept.  CG = 2: a pair of CTAs computes a 256 x 256 tile with cta_group::2; CG =
// 1: one CTA computes 128 x 128, for launches too small to fill the GPU with pairs.  Either
// way a CTA stages 128 rows of each operand per 64-deep k-block (32 KB), loaded as four
// 64 x 64 boxes.  GRAM and POLY compute and store only the 256 x 256 blocks on and above the
// diagonal.  Whoever reads such a matrix takes a block below the diagonal from its mirror
// image: the same box load with the coordinates swapped, and that k-block's MMAs told that
// the operand is MN-major.  So symmetry halves the stores as well as the products.
//   warp 0 TMA producer, warp 1 TMEM allocation and MMA issue, warps 2-9 epilogue: two per
//   quarter of the TMEM lanes, each finishing half of the tile's columns.
//
// Measured (B200, the 100M model's 84 matrices, device time of a launch within the whole update): the
// first GRAM 58 us (0.95 PFLOP/s of useful work), the later ones, under the power cap, 72 to 84; POLY
// 57 to 64 us (K = 768 or less: epilogue and pipeline start); APPLY 107 us, 170 where it reads and
// writes low parts (604 MB at 3.6 TB/s); STEP 176 us (755 MB at 4.3 TB/s).
#pragma once

#include <cuda_fp16.h>

#include "gemm_pair.cuh"

namespace pb {

enum NsMode : int {
  NS_GRAM = 0,   // out = alpha acc
  NS_POLY = 1,   // out = alpha acc + beta add + diag I
  NS_APPLY = 2,  // out, low = split(alpha acc + beta add)  (``add``: the input's low part, or none)
  NS_LAST = 3,   // bf16 result
  NS_STEP = 4,   // p = decay p - step alpha acc (fp32), and the bf16 copy of p
};

constexpr int kNsGroups = 8;     // shapes per launch
constexpr int kNsMats = 192;     // matrices per launch of the pointer tables
constexpr float kNsLowScale = 2048.f;

struct NsGroup {
  CUtensorMap a, b;      // operands: 64 x 64 boxes of fp16 [batch][rows][cols]
  CUtensorMap out, low;  // 32 x 32 boxes of the results
  const __half* add;     // POLY, APPLY: addend, indexed as the result (APPLY: the low part, or null)
  long add_batch;        // elements between the addend's matrices
  int add_ld;
  int M, N, K;
  int a_mn, b_mn;        // operand is MN-major
  int a_sym, b_sym;      // operand is symmetric, blocks on and above the diagonal stored
  int batch;             // matrices
  int k_blocks;
  int tiles_n;           // tiles per row (symmetric: per side)
  int tiles_per_mat;
  int tile_end;          // running total over the groups
  int store_low;         // APPLY: the result's low part is wanted
  int vec;               // STEP: 16-byte accesses to the parameters
  int mat0;              // STEP: index of the group's first matrix in the pointer table
  __nv_bfloat16* dst;    // LAST: [batch][M][N]
  int dst_tma;           // LAST: ``out`` maps dst (rows are whole 16-byte pieces)
  float step;            // STEP: step length per unit of learning rate
};
struct NsArgs {
  NsGroup g[kNsGroups];
  int groups;
  int tiles;
  float alpha, beta, diag;
  int* status;
};
struct NsStepArgs {
  float* p[kNsMats];
  __nv_bfloat16* shadow[kNsMats];
  const float* norm;  // gradient norm; not finite: nothing is updated (null: always update)
  const float* hp;    // learning rate on the device (null: ``lr``)
  float lr, weight_decay;
};
struct NsNoStep {};

template <int CG_>
struct NsCfg {
  static constexpr int CG = CG_;
  static constexpr int BM = 128;
  static constexpr int T = BM * CG;  // tile rows and columns
  static constexpr int BK = 64;
  static constexpr int OP_BYTES = BM * BK * 2;  // this CTA's share of either operand of a k-block
  static constexpr int STAGE_BYTES = 2 * OP_BYTES;
  static constexpr int STAGES = 6;
  static constexpr int EPI_WARPS = 8;
  static constexpr int THREADS = 64 + 32 * EPI_WARPS;
  using Stg = StagerT<2>;
  static constexpr int EPI_OFF = STAGES * STAGE_BYTES;
  static constexpr uint32_t TMEM_COLS = 2 * T;
  static constexpr int SMEM_BYTES = EPI_OFF + EPI_WARPS * Stg::kBytes + 1024;
  static_assert(SMEM_BYTES <= 232448, "shared memory budget");
};

// kind::f16 instruction descriptor with fp16 operands (formats 0) and fp32 accumulation.
__device__ __forceinline__ uint32_t ns_idesc(int t, int a_mn, int b_mn) {
  return (1u << 4) | (static_cast<uint32_t>(a_mn) << 15) | (static_cast<uint32_t>(b_mn) << 16) |
         (static_cast<uint32_t>(t >> 3) << 17) | (static_cast<uint32_t>(t >> 4) << 24);
}

__device__ __forceinline__ void grid_dependency_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void grid_dependents_go() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

struct NsTile {
  int g, mat, i, j;
};
// First tile column that is computed in tile row ``i`` of a symmetric result: 256 x 256 blocks
// are whole, so with 128-wide tiles the block's first.
template <int CG>
__host__ __device__ __forceinline__ int ns_first_col(int i) {
  return CG == 2 ? i : i & ~1;
}
// Tile index -> group, matrix and tile row / column.
template <int CG, bool SYM>
__device__ __forceinline__ NsTile ns_tile(const NsArgs& a, int tile) {
  int g = 0, base = 0;
  while (g + 1 < a.groups && tile >= a.g[g].tile_end) base = a.g[g++].tile_end;
  const int per = a.g[g].tiles_per_mat, tn = a.g[g].tiles_n;
  const int local = tile - base;
  NsTile t{g, local / per, 0, 0};
  int k = local % per;
  if (SYM) {
    while (k >= tn - ns_first_col<CG>(t.i)) k -= tn - ns_first_col<CG>(t.i++);
    t.j = ns_first_col<CG>(t.i) + k;
  } else {
    t.i = k / tn;
    t.j = k % tn;
  }
  return t;
}
// Is the operand MN-major in k-block ``kb`` of a tile whose rows start at ``row``?
__device__ __forceinline__ int ns_is_mn(int mn, int sym, int row, int kb) {
  return sym ? (kb * 64) / 256 < row / 256 : mn;
}

template <int CG>
__device__ __forceinline__ void ns_load(void* dst, const CUtensorMap* map, uint32_t bar, int c0, int c1, int c2) {
  if constexpr (CG == 2)
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1), "r"(c2)
        : "memory");
  else
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1), "r"(c2)
        : "memory");
}

// 128 rows (K-major) or columns (MN-major) of an operand from ``row``, k-block ``k0``.
template <int CG>
__device__ __forceinline__ void ns_load_operand(uint8_t* dst, const CUtensorMap* map, uint32_t bar, int mn, int row,
                                                int k0, int mat) {
  const int x = mn ? row : k0, y = mn ? k0 : row;
  ns_load<CG>(dst, map, bar, x, y, mat);
  ns_load<CG>(dst + 8192, map, bar, mn ? x + 64 : x, mn ? y : y + 64, mat);
}

// One MMA; the operands' shared-memory descriptors share their high word (stride 1024, version,
// swizzle) and are put together here.
template <int CG>
__device__ __forceinline__ void ns_mma(uint32_t d_tmem, uint32_t a_lo, uint32_t b_lo, uint32_t hi, uint32_t idesc,
                                       uint32_t accumulate) {
  if constexpr (CG == 2)
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\t"
        "mov.b64 a, {%1, %3};\n\tmov.b64 b, {%2, %3};\n\t"
        "setp.ne.b32 p, %5, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], a, b, %4, p;\n\t}" ::"r"(d_tmem),
        "r"(a_lo), "r"(b_lo), "r"(hi), "r"(idesc), "r"(accumulate)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\t"
        "mov.b64 a, {%1, %3};\n\tmov.b64 b, {%2, %3};\n\t"
        "setp.ne.b32 p, %5, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %4, p;\n\t}" ::"r"(d_tmem),
        "r"(a_lo), "r"(b_lo), "r"(hi), "r"(idesc), "r"(accumulate)
        : "memory");
}

// One lane of a converged warp.
__device__ __forceinline__ bool elect_one() {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok));
  return ok != 0;
}
// Bounded wait of a whole, converged warp: all lanes try at once, and only if that fails does
// lane 0 go on polling for the others.
__device__ __forceinline__ bool ns_wait(uint64_t* bar, uint32_t parity, int* status, int code, volatile int* abort) {
  if (__all_sync(0xffffffff, mbar_try_wait(bar, parity))) return true;
  return mbar_wait_warp(bar, parity, status, code, abort);
}

__device__ __forceinline__ void ns_store(const CUtensorMap* map, const uint8_t* s, int col, int row, int mat) {
  fence_async_smem();
  __syncwarp();
  if ((threadIdx.x & 31) == 0) {
    asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%2, %3, %4}], [%1];" ::"l"(
                     reinterpret_cast<uint64_t>(map)),
                 "r"(smem_u32(s)), "r"(col), "r"(row), "r"(mat)
                 : "memory");
    bulk_commit();
  }
}

__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// 32 values of this lane's row -> 64-byte row of a 64B-swizzled [32 x 32] fp16 box.
__device__ __forceinline__ void stage_f16(uint8_t* s, const float (&v)[32]) {
  const int r = threadIdx.x & 31;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    uint4 q = make_uint4(pack_f16x2(v[8 * j], v[8 * j + 1]), pack_f16x2(v[8 * j + 2], v[8 * j + 3]),
                         pack_f16x2(v[8 * j + 4], v[8 * j + 5]), pack_f16x2(v[8 * j + 6], v[8 * j + 7]));
    *reinterpret_cast<uint4*>(s + r * 64 + ((j ^ ((r >> 1) & 3)) << 4)) = q;
  }
}
// 32 fp16 of this lane's row of the addend, columns [col, col + 32); pieces at or beyond ``ld``
// (the padded row length, a multiple of 8) read as zero.  Coherent loads: APPLY stores the new low
// part over the one that it reads here.
__device__ __forceinline__ void ns_load_add(const __half* row, bool ok, int col, int ld, uint4 (&q)[4]) {
#pragma unroll
  for (int j = 0; j < 4; ++j)
    q[j] = ok && col + 8 * j < ld ? *(reinterpret_cast<const uint4*>(row + col) + j) : make_uint4(0, 0, 0, 0);
}
__device__ __forceinline__ void ns_add(float (&v)[32], const uint4 (&q)[4], float alpha, float beta) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t* w = &q[j].x;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(w + k));
      v[8 * j + 2 * k] = alpha * v[8 * j + 2 * k] + beta * f.x;
      v[8 * j + 2 * k + 1] = alpha * v[8 * j + 2 * k + 1] + beta * f.y;
    }
  }
}

// A 32 x 32 fp32 block through shared memory: this lane's row in, any row's 16-byte pieces out
// (piece q of row r at q ^ (r & 7): neither direction has bank conflicts).
__device__ __forceinline__ void ns_block_in(float* s, const float (&v)[32]) {
  const int r = threadIdx.x & 31;
#pragma unroll
  for (int q = 0; q < 8; ++q)
    *reinterpret_cast<float4*>(s + r * 32 + ((q ^ (r & 7)) << 2)) =
        make_float4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
  __syncwarp();
}
__device__ __forceinline__ float4 ns_block_piece(const float* s, int r, int q) {
  return *reinterpret_cast<const float4*>(s + r * 32 + ((q ^ (r & 7)) << 2));
}
__device__ __forceinline__ float ns_block_at(const float* s, int r, int c) {
  return s[r * 32 + ((((c >> 2) ^ (r & 7)) << 2) | (c & 3))];
}

// What the epilogue of ``tile`` will read for this warp's rows (the low part, the parameters)
// starts moving into L2 while the tile before it is finished: the parameters, and the low parts of
// all matrices together, are larger than L2, and the DRAM latency was otherwise paid once per 32
// columns.
template <int CG, int MODE, class Step>
__device__ __forceinline__ void ns_prefetch(const NsArgs& a, const Step& sa, int tile, int row_in_tile, int c0) {
  using C = NsCfg<CG>;
  if constexpr (MODE == NS_APPLY || MODE == NS_STEP) {
    if (tile >= a.tiles) return;
    const NsTile t = ns_tile<CG, false>(a, tile);
    const NsGroup& g = a.g[t.g];
    const int row = t.i * C::T + row_in_tile, col = t.j * C::T + c0;
    if (row >= g.M) return;
    const char* p = nullptr;
    int piece = 0;  // columns per 128-byte line
    if constexpr (MODE == NS_APPLY) {
      if (g.add == nullptr) return;
      p = reinterpret_cast<const char*>(g.add + t.mat * g.add_batch + static_cast<long>(row) * g.add_ld + col);
      piece = 64;
    } else {
      p = reinterpret_cast<const char*>(sa.p[g.mat0 + t.mat] + static_cast<long>(row) * g.N + col);
      piece = 32;
    }
    for (int c = 0; c < C::T / 2 && col + c < g.N; c += piece, p += 128)
      asm volatile("prefetch.global.L2 [%0];" ::"l"(p));
  }
}

// Epilogue of one tile for the 32 rows from ``row0`` and the tile columns [c0, c0 + T / 2);
// ``tacc`` is the accumulator's address at those rows and columns.  Inputs that do not depend on
// the products are requested before ``wait()`` waits for the accumulator (false: give up).
template <int CG, int MODE, class Step, class Wait>
__device__ __forceinline__ bool ns_epilogue(const NsArgs& a, const Step& sa, const NsTile& t, typename NsCfg<CG>::Stg& st,
                                            uint32_t tacc, int row0, int c0, Wait&& wait) {
  using C = NsCfg<CG>;
  constexpr int W = C::T / 2;
  const NsGroup& g = a.g[t.g];
  const int lane = threadIdx.x & 31;
  const int row = row0 + lane;
  const int col0 = t.j * C::T + c0;
  if constexpr (MODE == NS_GRAM || MODE == NS_POLY || MODE == NS_APPLY) {
    const bool ok = row < g.M;
    const bool with_add = MODE == NS_POLY || (MODE == NS_APPLY && g.add != nullptr);
    uint4 q[MODE == NS_GRAM ? 1 : W / 32][4];
    if constexpr (MODE != NS_GRAM) {
      if (with_add) {
        const __half* from = g.add + t.mat * g.add_batch + static_cast<long>(ok ? row : 0) * g.add_ld;
#pragma unroll
        for (int k = 0; k < W / 32; ++k) ns_load_add(from, ok, col0 + 32 * k, g.add_ld, q[k]);
      }
    }
    if (!wait()) return false;
#pragma unroll
    for (int k = 0; k < W / 32; ++k) {
      const int col = col0 + 32 * k;
      if (col >= g.N) break;  // uniform across the warp
      float v[32];
      tmem_load_f32(tacc + 32 * k, v);
      if (with_add) {
        ns_add(v, q[MODE == NS_GRAM ? 0 : k], a.alpha, a.beta);
      } else {
#pragma unroll
        for (int j = 0; j < 32; ++j) v[j] *= a.alpha;
      }
      if constexpr (MODE == NS_POLY) {
        if (col < row0 + 32 && row0 < col + 32) {
#pragma unroll
          for (int j = 0; j < 32; ++j)
            if (col + j == row) v[j] += a.diag;
        }
      }
      uint8_t* s = st.acquire();
      stage_f16(s, v);
      ns_store(&g.out, s, col, row0, t.mat);
      st.release();
      if constexpr (MODE == NS_APPLY) {
        if (g.store_low) {
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] = (v[j] - __half2float(__float2half_rn(v[j]))) * kNsLowScale;
          s = st.acquire();
          stage_f16(s, v);
          ns_store(&g.low, s, col, row0, t.mat);
          st.release();
        }
      }
    }
  } else if constexpr (MODE == NS_LAST) {
    if (!wait()) return false;
    if (g.dst_tma) {
      tmem_walk(tacc, W, [&](int c, float (&v)[32]) {
        const int col = col0 + c;
        if (col >= g.N) return;
        uint8_t* s = st.acquire();
        stage_bf16(s, v, a.alpha);
        ns_store(&g.out, s, col, row0, t.mat);
        st.release();
      });
    } else {
      // rows that do not start on 16-byte boundaries: 64-byte row pieces with plain stores
      float* s = reinterpret_cast<float*>(st.base);
      __nv_bfloat16* d = g.dst + static_cast<long>(t.mat) * g.M * g.N;
      const int rows = min(32, g.M - row0);
      tmem_walk(tacc, W, [&](int c, float (&v)[32]) {
        const int col = col0 + c;
        if (col >= g.N) return;
        ns_block_in(s, v);
        if (col + lane < g.N)
          for (int k = 0; k < rows; ++k)
            d[static_cast<long>(row0 + k) * g.N + col + lane] = __float2bfloat16_rn(ns_block_at(s, k, lane) * a.alpha);
        __syncwarp();
      });
    }
  } else {
    // The parameters of the next 32 columns are on their way while this block is updated: the
    // launch reads and writes 4 bytes per element, more than its products cost.
    if (sa.norm != nullptr && !isfinite(*sa.norm)) return wait();
    const float lr = sa.hp != nullptr ? *sa.hp : sa.lr;
    const float decay = 1.f - lr * sa.weight_decay;
    const float step = lr * g.step * a.alpha;
    float* p = sa.p[g.mat0 + t.mat];
    __nv_bfloat16* sh = sa.shadow[g.mat0 + t.mat];
    float* s = reinterpret_cast<float*>(st.base);
    if (g.vec) {
      // A lane takes the 16-byte piece lane % 8 of rows lane / 8, + 4, + 8, ...; as a piece is
      // used, the one 32 columns on is requested into its registers.  (Holding two blocks ahead
      // spilled, and with 225 KB of shared memory in use a spill's reload comes from L2: 253 us
      // instead of 172 for the 100M model's last product.)
      const int r0 = lane >> 3, q = lane & 7;
      const int rows = (g.M - row0 - r0 + 3) / 4;  // this lane's rows in range
      const long base = static_cast<long>(row0 + r0) * g.N + col0 + 4 * q;
      const int pitch = 4 * g.N, cols = g.N - col0 - 4 * q;
      const float* next = p + base;
      float4 buf[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        buf[k] = k < rows && cols > 0 ? *reinterpret_cast<const float4*>(next) : make_float4(0.f, 0.f, 0.f, 0.f);
        next += pitch;
      }
      if (!wait()) return false;
#pragma unroll 1
      for (int c = 0; c < W; c += 32) {
        if (col0 + c >= g.N) break;  // uniform across the warp
        {
          float v[32];
          tmem_load_f32(tacc + c, v);
          ns_block_in(s, v);
        }
        float* at = p + base + c;
        __nv_bfloat16* to = sh == nullptr ? nullptr : sh + base + c;
        const bool more = c + 32 < W && cols > c + 32;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const float4 o = ns_block_piece(s, r0 + 4 * k, q);
          float4 w = buf[k];
          if (more && k < rows) buf[k] = *reinterpret_cast<const float4*>(at + 32);
          w.x = w.x * decay - step * o.x;
          w.y = w.y * decay - step * o.y;
          w.z = w.z * decay - step * o.z;
          w.w = w.w * decay - step * o.w;
          if (k < rows && cols > c) {
            *reinterpret_cast<float4*>(at) = w;
            if (sh != nullptr) *reinterpret_cast<uint2*>(to) = make_uint2(pack_bf16x2(w.x, w.y), pack_bf16x2(w.z, w.w));
          }
          at += pitch;
          if (sh != nullptr) to += pitch;
        }
        __syncwarp();
      }
    } else {
      if (!wait()) return false;
      const int rows = min(32, g.M - row0);
      tmem_walk(tacc, W, [&](int c, float (&v)[32]) {
        const int col = col0 + c;
        if (col >= g.N) return;
        ns_block_in(s, v);
        if (col + lane < g.N) {
#pragma unroll 1
          for (int k0 = 0; k0 < rows; k0 += 8) {
            float w[8];
#pragma unroll
            for (int k = 0; k < 8; ++k)
              w[k] = k0 + k < rows ? p[static_cast<long>(row0 + k0 + k) * g.N + col + lane] : 0.f;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              if (k0 + k >= rows) break;
              const float u = w[k] * decay - step * ns_block_at(s, k0 + k, lane);
              const long at = static_cast<long>(row0 + k0 + k) * g.N + col + lane;
              p[at] = u;
              if (sh != nullptr) sh[at] = __float2bfloat16_rn(u);
            }
          }
        }
        __syncwarp();
      });
    }
  }
  return true;
}

// NsCfg::THREADS threads; CG == 2 with cluster dimension (2, 1, 1).
template <int CG, int MODE, class Step>
__global__ void __launch_bounds__(NsCfg<CG>::THREADS, 1)
    ns_gemm_kernel(const __grid_constant__ NsArgs args, const __grid_constant__ Step step) {
  using C = NsCfg<CG>;
  constexpr bool SYM = MODE == NS_GRAM || MODE == NS_POLY;
  __shared__ __align__(8) uint64_t full_bar[C::STAGES];
  __shared__ __align__(8) uint64_t empty_bar[C::STAGES];
  __shared__ __align__(8) uint64_t accf_bar[2];
  __shared__ __align__(8) uint64_t acce_bar[2];
  __shared__ __align__(8) uint64_t drain_bar;
  __shared__ uint32_t tmem_base_sh;
  __shared__ volatile int abort_sh;
  __shared__ volatile uint32_t odd_done_sh;  // even CTA: the odd producer's issued k-blocks | kOddDone
  __shared__ volatile uint32_t odd_one_sh;   // and its one_mask
  extern __shared__ uint8_t dyn_smem[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(dyn_smem) + 1023) & ~uintptr_t(1023));

  const int warp = threadIdx.x / 32;
  const int lane = threadIdx.x % 32;
  const uint32_t cta = CG == 2 ? cluster_ctarank() : 0;  // CTA 0 issues the MMAs
  const int first = blockIdx.x / CG, stride = gridDim.x / CG;
  if (threadIdx.x == 0) {
    odd_done_sh = odd_one_sh = 0;
    for (int s = 0; s < C::STAGES; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(&accf_bar[s], 1);
      mbar_init(&acce_bar[s], C::EPI_WARPS * CG);
    }
    mbar_init(&drain_bar, 1);
    abort_sh = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    if constexpr (CG == 2) {
      tmem_alloc_pair(&tmem_base_sh, C::TMEM_COLS);
      tmem_relinquish_pair();
    } else {
      tmem_alloc(&tmem_base_sh, C::TMEM_COLS);
      tmem_relinquish();
    }
  }
  tc_fence_before();
  if constexpr (CG == 2) cluster_sync();
  else __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = tmem_base_sh;
  // The launch before this one may still be finishing on other SMs: everything above overlaps its
  // tail, everything below reads what it wrote.
  grid_dependency_wait();
  grid_dependents_go();

  // Warps 0 and 1 run their loops with all lanes converged and elect one to issue.  A k-block's
  // MMAs take 512 cycles; measured per k-block the issuing warp spends about 190 on its barrier,
  // 290 on the four MMAs and 90 on the commit, the producer 360 on four box loads.  A tile on
  // the diagonal of a symmetric product has twice the same operand and loads it once.
  if (warp == 0) {
    const uint32_t full0 = CG == 2 ? cluster_addr(smem_u32(&full_bar[0]), 0) : smem_u32(&full_bar[0]);
    const bool leader = elect_one();
    int stage = 0;
    uint32_t phase = 0;
    uint32_t armed_mask = 0, armed_phase = 0;  // CTA 0: per stage, armed and its phase
    uint32_t n_kb = 0;                         // k-blocks armed (CTA 0) / issued (CTA 1)
    uint32_t one_mask = 0;                     // per stage: its last k-block has one operand
    bool ok = true;
    for (int tile = first; tile < args.tiles && ok; tile += stride) {
      const NsTile t = ns_tile<CG, SYM>(args, tile);
      const NsGroup& g = args.g[t.g];
      const int row_a = t.i * C::T + static_cast<int>(cta) * C::BM;
      const int row_b = t.j * C::T + static_cast<int>(cta) * C::BM;
      const int a_mn = g.a_mn, b_mn = g.b_mn, a_sym = g.a_sym, b_sym = g.b_sym, kbs = g.k_blocks;
      const bool one = SYM && t.i == t.j;  // both operands are the same rows of the same matrix
      for (int kb = 0; kb < kbs; ++kb) {
        if (!ns_wait(&empty_bar[stage], phase ^ 1, args.status, 141, &abort_sh)) {
          ok = false;
          break;
        }
        if (cta == 0) {
          if (leader) mbar_arrive_expect_tx(&full_bar[stage], CG * (one ? C::OP_BYTES : C::STAGE_BYTES));
          armed_mask |= 1u << stage;
          armed_phase = (armed_phase & ~(1u << stage)) | (phase << stage);
        }
        one_mask = (one_mask & ~(1u << stage)) | (static_cast<uint32_t>(one) << stage);
        ++n_kb;
        uint8_t* sa = smem + stage * C::STAGE_BYTES;
        if (leader) {
          ns_load_operand<CG>(sa, &g.a, full0 + stage * 8, ns_is_mn(a_mn, a_sym, row_a, kb), row_a, kb * C::BK, t.mat);
          if (!one)
            ns_load_operand<CG>(sa + C::OP_BYTES, &g.b, full0 + stage * 8, ns_is_mn(b_mn, b_sym, row_b, kb), row_b,
                                kb * C::BK, t.mat);
        }
        __syncwarp();
        if (++stage == C::STAGES) {
          stage = 0;
          phase ^= 1;
        }
      }
    }
    if (leader) {
      // Abort protocol of gemm_pair.cuh: no load of either CTA is in flight at the exit.
      if (CG == 2 && cta == 1) {
        st_release_cluster(cluster_addr(smem_u32((const void*)&odd_one_sh), 0), one_mask);
        st_release_cluster(cluster_addr(smem_u32((const void*)&odd_done_sh), 0), n_kb | kOddDone);
      } else if (!ok) {
        if constexpr (CG == 2) {
          st_release_cluster(cluster_addr(smem_u32((const void*)&abort_sh), 1), 1u);
          uint32_t done = 0;
          const uint64_t t0 = globaltimer();
          while (!((done = ld_acquire_cluster(&odd_done_sh)) & kOddDone)) {
            if (globaltimer() - t0 > 2 * PB_WAIT_TIMEOUT_NS) {
              report_error(args.status, 147);
              break;
            }
          }
          if (done & kOddDone) {
            const uint32_t n_odd = done & ~kOddDone;
            for (uint32_t kb = n_kb; kb < n_odd && kb < n_kb + C::STAGES; ++kb) {
              mbar_arrive_expect_tx(&full_bar[stage], (odd_one_sh >> stage) & 1u ? C::OP_BYTES : C::STAGE_BYTES);
              armed_mask |= 1u << stage;
              armed_phase = (armed_phase & ~(1u << stage)) | (phase << stage);
              if (++stage == C::STAGES) {
                stage = 0;
                phase ^= 1;
              }
            }
          }
        }
        for (int s = 0; s < C::STAGES; ++s)
          if (armed_mask & (1u << s)) mbar_wait(&full_bar[s], (armed_phase >> s) & 1u, args.status, 142, nullptr);
      }
    }
  } else if (warp == 1) {
    if (cta == 0) {
      const bool leader = elect_one();
      int stage = 0;
      uint32_t phase = 0;
      int acc = 0;
      uint32_t acc_phase = 0;
      bool ok = true;
      const uint32_t smem_base = smem_u32(smem);
      const uint32_t desc_hi = static_cast<uint32_t>(sdesc_sw128(0, 0, 1024) >> 32);
      for (int tile = first; tile < args.tiles && ok; tile += stride) {
        const NsTile t = ns_tile<CG, SYM>(args, tile);
        const NsGroup& g = args.g[t.g];
        const int kbs = g.k_blocks, g_amn = g.a_mn, g_asym = g.a_sym, g_bmn = g.b_mn, g_bsym = g.b_sym;
        const int row_a = t.i * C::T, row_b = t.j * C::T;
        const bool one = SYM && t.i == t.j;
        if (!mbar_wait_warp(&acce_bar[acc], acc_phase ^ 1, args.status, 143, &abort_sh)) break;
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + acc * C::T;
        // A symmetric operand is MN-major below its diagonal block and K-major from there on, so
        // the k-blocks fall into at most three runs of one kind each; within a run only the stage
        // address changes.
        const int cut_a = g_asym ? min(kbs, row_a / 256 * 4) : (g_amn ? kbs : 0);
        const int cut_b = g_bsym ? min(kbs, row_b / 256 * 4) : (g_bmn ? kbs : 0);
        for (int kb = 0; kb < kbs && ok;) {
          const bool a_mn = kb < cut_a, b_mn = kb < cut_b;
          const int end = min(a_mn ? cut_a : kbs, b_mn ? cut_b : kbs);
          const uint32_t idesc = ns_idesc(C::T, a_mn, b_mn);
          // 32 bytes per 16-deep step of a K-major operand, 16 rows of 128 bytes of an MN-major one
          const uint32_t step_a = a_mn ? 2048 >> 4 : 32 >> 4, step_b = b_mn ? 2048 >> 4 : 32 >> 4;
          const uint32_t a_lbo = (a_mn ? 8192u : 16u) >> 4 << 16, b_lbo = (b_mn ? 8192u : 16u) >> 4 << 16;
          for (; kb < end; ++kb) {
            if (!ns_wait(&full_bar[stage], phase, args.status, 144, &abort_sh)) {
              ok = false;
              break;
            }
            tc_fence_after();
            const int cur = stage;
            if (++stage == C::STAGES) {
              stage = 0;
              phase ^= 1;
            }
            const uint32_t s0 = (smem_base + cur * C::STAGE_BYTES) >> 4;
            const uint32_t ad = s0 | a_lbo, bd = (s0 + (one ? 0 : C::OP_BYTES >> 4)) | b_lbo;
            if (leader) {
#pragma unroll
              for (int kk = 0; kk < C::BK / 16; ++kk)
                ns_mma<CG>(d_tmem, ad + kk * step_a, bd + kk * step_b, desc_hi, idesc, (kb > 0 || kk > 0) ? 1u : 0u);
              if constexpr (CG == 2) umma_commit_both(&empty_bar[cur]);
              else umma_commit(&empty_bar[cur]);
            }
            __syncwarp();
          }
        }
        if (!ok) break;
        if (leader) {
          if constexpr (CG == 2) umma_commit_both(&accf_bar[acc]);
          else umma_commit(&accf_bar[acc]);
        }
        __syncwarp();
        acc ^= 1;
        if (acc == 0) acc_phase ^= 1;
      }
      // All MMAs issued by this warp must finish before TMEM is released.
      if (leader) {
        if constexpr (CG == 2) umma_commit_pair_local(&drain_bar);
        else umma_commit(&drain_bar);
        mbar_wait(&drain_bar, 0, args.status, 145, nullptr);
      }
      __syncwarp();
    }
  } else {
    const int q = warp & 3, half = (warp - 2) / 4;  // TMEM lanes 32 q.., columns T / 2 half..
    const uint32_t acce0 = CG == 2 ? cluster_addr(smem_u32(&acce_bar[0]), 0) : 0;
    typename C::Stg st{smem + C::EPI_OFF + (warp - 2) * C::Stg::kBytes, 0, false};
    const int row_in_tile = static_cast<int>(cta) * C::BM + q * 32;
    int acc = 0;
    uint32_t acc_phase = 0;
    ns_prefetch<CG, MODE>(args, step, first, row_in_tile + lane, half * (C::T / 2));
    for (int tile = first; tile < args.tiles; tile += stride) {
      const NsTile t = ns_tile<CG, SYM>(args, tile);
      const uint32_t tacc = tmem_base + (static_cast<uint32_t>(q * 32) << 16) + acc * C::T + half * (C::T / 2);
      const int row0 = t.i * C::T + row_in_tile;
      auto wait = [&] {
        const bool ok = mbar_wait_warp(&accf_bar[acc], acc_phase, args.status, 146, &abort_sh);
        tc_fence_after();
        return ok;
      };
      ns_prefetch<CG, MODE>(args, step, tile + stride, row_in_tile + lane, half * (C::T / 2));
      bool ok;
      if (row0 < args.g[t.g].M && t.j * C::T + half * (C::T / 2) < args.g[t.g].N)
        ok = ns_epilogue<CG, MODE>(args, step, t, st, tacc, row0, half * (C::T / 2), wait);
      else ok = wait();
      if (!ok) break;
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if constexpr (CG == 2) mbar_arrive_cluster(acce0 + acc * 8);
        else mbar_arrive(&acce_bar[acc]);
      }
      acc ^= 1;
      if (acc == 0) acc_phase ^= 1;
    }
    if (lane == 0) bulk_wait_all<0>();
    __syncwarp();
  }
  tc_fence_before();
  if constexpr (CG == 2) cluster_sync();
  else __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    if constexpr (CG == 2) tmem_dealloc_pair(tmem_base, C::TMEM_COLS);
    else tmem_dealloc(tmem_base, C::TMEM_COLS);
  }
}

}  // namespace pb
