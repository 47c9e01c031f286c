// The tiled matrix product behind dense.hip: D[m][n] = sum_k A[m][k] B[n][k] on the bf16 matrix cores,
// with the epilogues of the dense and gated operators.
//
// Operands are bf16 "planes": a bf16 matrix is one plane, an fp32 matrix three whose sum is the matrix,
// x = x1 + x2 + x3 exactly (8 + 8 + 8 mantissa bits). The product of two three-plane
// operands takes the six plane products x_i w_j with i + j <= 4 (Henry, Tang, Heinecke, "Leveraging the
// bfloat16 Artificial Intelligence Datatype For Higher-Precision Computations", 2019): what is left out
// is at most 2^-23 |x||w|, the products of planes are exact (8 x 8 bits) and their sums are
// fp32. Six bf16 instructions replace sixteen times slower fp32 ones. Against a one-plane operand three
// plane products are the whole product.
//
// Layout rules (the host stages operands that break them): rows 16-byte aligned, k contiguous, ld and the
// k extent multiples of 64 elements with zeros behind the matrix's own columns. Rows are guarded by the
// buffer descriptors: a row past the end reads zeros.
#pragma once

#include <algorithm>

#include "aimx_common.h"

namespace aimx {
namespace dense {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef uint16_t u16x4 __attribute__((ext_vector_type(4)));

// fp32 -> bf16 bits, round to nearest even; NaN stays NaN
__device__ __forceinline__ uint16_t to_bf16(float v) {
  union { __bf16 b; uint16_t u; } c;
  c.b = (__bf16)v;
  return c.u;
}
__device__ __forceinline__ float from_bf16(uint16_t u) { return __uint_as_float((uint32_t)u << 16); }

// The three planes of v, each the nearest bf16 of what is left: |x2| <= 2^-8 |x|, |x3| <= 2^-16 |x|, and the
// third is exact (24 = 8 + 8 + 8 bits). A NaN or infinity goes whole into the first plane; what it then
// multiplies in the other operand's lower planes may be zero, so an infinite operand can make a NaN
// where the one-plane product has an infinity.
__device__ __forceinline__ void split3(float v, uint16_t (&p)[3]) {
  p[0] = to_bf16(v);
  p[1] = p[2] = 0;
  if ((p[0] & 0x7f80u) == 0x7f80u) {  // not finite, or within half a step of the largest value: cut off instead
    if ((__float_as_uint(v) & 0x7f800000u) == 0x7f800000u) return;
    p[0] = (uint16_t)(__float_as_uint(v) >> 16);
  }
  const float r1 = v - from_bf16(p[0]);
  p[1] = to_bf16(r1);
  p[2] = to_bf16(r1 - from_bf16(p[1]));
}

// One operand of a product. `half` rows come from p, the rows behind them from p2 (the gated forward's two
// weights); plane q is at + q * plane elements.
struct Operand {
  const uint16_t* p;
  const uint16_t* p2;
  int64_t ld, plane, rows;
};

struct Problem {
  Operand a, b;
  int64_t M, N, K;       // N: columns of the result (of one half where the epilogue is gated); K % 64 == 0
  void* y;               // [M][N], ld ldy (nullptr: only pre)
  void* y2;              // rows >= y_rows of the result go to y2 (weight gradients of two weights)
  int64_t ldy, y_rows;
  const void* bias;      // [N], of the output's type; bias2: of the second half
  const void* bias2;
  const void* res;       // [M][N], ld ldr
  int64_t ldr;
  float* pre;            // [M][halves * N] fp32, before the activation
  float* slab;           // split-k partial sums [splits][M][N]
  int32_t act, splits, vec;
};

enum Epi : int { kPlain = 0, kGated = 1, kSlab = 2 };

template <int PA_, int PB_, int TM_, int TN_, int WGM_, int WGN_, int BK_>
struct Config {
  static constexpr int PA = PA_, PB = PB_, TM = TM_, TN = TN_, WGM = WGM_, WGN = WGN_, BK = BK_;
  static constexpr int kThreads = WGM * WGN * kWave;
  static constexpr int WTM = TM / WGM, WTN = TN / WGN, FM = WTM / 16, FN = WTN / 16;
  static constexpr int U = BK / 8;                   // 16-byte units of a row
  static constexpr int kRowsPerLoad = kWave / U;     // rows that one wave's load covers
  static constexpr int kStage = (PA * TM + PB * TN) * BK * 2;  // bytes
};

// Position of k unit c of row r: the units of neighbouring rows are spread over the banks, so that the 16
// rows a fragment read takes at one k unit fall into different ones (the loads write LDS linearly: the
// permutation is in the global addresses).
template <int U>
__device__ __forceinline__ int swz(int r, int c) {
  return U == 8 ? (c ^ (r & 7)) : (c ^ ((r >> 1) & 3));
}

__device__ __forceinline__ float act_fast(int kind, float v) {
  // hardware exp2 and reciprocal (about 2^-21): for results that are rounded to 8 bits
  if (kind == ACT_SILU) return v * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-1.44269504f * v));
  return act_fwd(kind, v);
}

template <typename T>
__device__ __forceinline__ float load1(const T* p);
template <>
__device__ __forceinline__ float load1<float>(const float* p) { return *p; }
template <>
__device__ __forceinline__ float load1<uint16_t>(const uint16_t* p) { return from_bf16(*p); }

// four consecutive values; vec: the address is a multiple of 4 elements and all four exist
template <typename T>
__device__ __forceinline__ floatx4 load4(const T* p, bool vec, int64_t left) {
  floatx4 v;
  if (vec) {
    if constexpr (sizeof(T) == 4) {
      v = *reinterpret_cast<const floatx4*>(p);
    } else {
      const u16x4 h = *reinterpret_cast<const u16x4*>(p);
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = from_bf16(h[i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = i < left ? load1(p + i) : 0.f;
  }
  return v;
}
template <typename T>
__device__ __forceinline__ void store4(T* p, floatx4 v, bool vec, int64_t left) {
  if (vec) {
    if constexpr (sizeof(T) == 4) {
      *reinterpret_cast<floatx4*>(p) = v;
    } else {
      u16x4 h;
#pragma unroll
      for (int i = 0; i < 4; ++i) h[i] = to_bf16(v[i]);
      *reinterpret_cast<u16x4*>(p) = h;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < left) {
        if constexpr (sizeof(T) == 4) p[i] = v[i];
        else p[i] = to_bf16(v[i]);
      }
  }
}

// One workgroup: one TM x TN tile (kGated: TN / 2 columns of each half) over one k range. Operands go
// straight from global memory into LDS (16 bytes a lane, no registers), two stages: stage t + 1 is in flight
// through the matrix work of stage t. The weight is the instruction's first operand, so that a lane holds
// four consecutive columns of one row: 8- and 16-byte stores.
template <typename C, int EPI, typename T>
__global__ __launch_bounds__(C::kThreads) void k_dense(const Problem p, const int tiles_m, const int tiles_n) {
#ifdef __HIP_DEVICE_COMPILE__  // the host pass drops the stub of a body with the LDS load builtin
  constexpr int PA = C::PA, PB = C::PB, TM = C::TM, TN = C::TN, BK = C::BK, U = C::U;
  constexpr int kHalves = EPI == kGated ? 2 : 1, TC = TN / kHalves;  // columns of a half in a tile
  constexpr int kALoads = TM / C::kRowsPerLoad, kBLoads = TN / C::kRowsPerLoad;
  constexpr int kWaves = C::kThreads / kWave;
  static_assert(kALoads % kWaves == 0 && kBLoads % kWaves == 0, "every wave issues whole loads");
  static_assert(C::WTN / kHalves >= C::kRowsPerLoad, "a load lies inside one half");
  __shared__ __attribute__((aligned(1024))) char lds[2 * C::kStage];

  // Workgroups go to the 8 XCDs in turn: give each XCD a contiguous run of tiles, so that neighbours share
  // operand rows in one L2; within it, 8 tile rows at a time.
  const int nblk = tiles_m * tiles_n;
  int pid = blockIdx.x;
  {
    const int q = nblk >> 3, r = nblk & 7, x = pid & 7;
    pid = (x < r ? x * (q + 1) : r * (q + 1) + (x - r) * q) + (pid >> 3);
  }
  constexpr int kGroup = 8;
  const int group = pid / (kGroup * tiles_n), first = group * kGroup;
  const int gsz = min(tiles_m - first, kGroup), in = pid - group * kGroup * tiles_n;
  const int64_t m0 = (int64_t)(first + in % gsz) * TM, n0 = (int64_t)(in / gsz) * TC;

  const int split = blockIdx.y;
  const int64_t steps = p.K / BK;
  const int64_t s0 = steps * split / p.splits, s1 = steps * (split + 1) / p.splits;

  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int wm = wave / C::WGN, wn = wave % C::WGN;

  // Descriptors: one per plane, over the tile's rows from its first k
  __amdgpu_buffer_rsrc_t ra[PA], rb[PB][kHalves];
  {
    const int64_t left = p.a.rows - m0;
    const uint32_t bytes = (uint32_t)(min((int64_t)TM, max(left, (int64_t)0)) * p.a.ld * 2);
#pragma unroll
    for (int q = 0; q < PA; ++q) ra[q] = buffer_rsrc(p.a.p + q * p.a.plane + m0 * p.a.ld, bytes);
  }
  {
    const int64_t left = p.b.rows - n0;
    const uint32_t bytes = (uint32_t)(min((int64_t)TC, max(left, (int64_t)0)) * p.b.ld * 2);
#pragma unroll
    for (int q = 0; q < PB; ++q) {
      rb[q][0] = buffer_rsrc(p.b.p + q * p.b.plane + n0 * p.b.ld, bytes);
      if (kHalves == 2) rb[q][kHalves - 1] = buffer_rsrc(p.b.p2 + q * p.b.plane + n0 * p.b.ld, bytes);
    }
  }
  const int lr = lane / U, lu = lane % U;  // the row and unit of this lane in a load
  const uint32_t lda2 = (uint32_t)p.a.ld * 2, ldb2 = (uint32_t)p.b.ld * 2;

  auto load_stage = [&](int64_t step, int buf) {
    const uint32_t kb = (uint32_t)(step * BK * 2);
    char* base = lds + buf * C::kStage;
#pragma unroll
    for (int j = 0; j < kALoads / kWaves; ++j) {
      const int row = (j * kWaves + wave) * C::kRowsPerLoad + lr;
      const uint32_t off = (uint32_t)row * lda2 + swz<U>(row, lu) * 16;
#pragma unroll
      for (int q = 0; q < PA; ++q)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(
            ra[q], (__attribute__((address_space(3))) void*)(base + (q * TM * U + (j * kWaves + wave) * kWave) * 16), 16,
            off, kb, 0, 0);
    }
    base += PA * TM * BK * 2;
#pragma unroll
    for (int j = 0; j < kBLoads / kWaves; ++j) {
      const int r0 = (j * kWaves + wave) * C::kRowsPerLoad, row = r0 + lr;
      // LDS row -> row of a half: a wave's WTN columns are WTN / 2 of the first half, then of the second
      int src = row, half = 0;
      if (kHalves == 2) {
        constexpr int WH = C::WTN / 2;
        half = (r0 / WH) & 1;
        src = row / C::WTN * WH + row % WH;
      }
      const uint32_t off = (uint32_t)src * ldb2 + swz<U>(row, lu) * 16;
#pragma unroll
      for (int q = 0; q < PB; ++q) {
        auto dst = (__attribute__((address_space(3))) void*)(base + (q * TN * U + (j * kWaves + wave) * kWave) * 16);
        if (kHalves == 1 || half == 0)
          __builtin_amdgcn_raw_ptr_buffer_load_lds(rb[q][0], dst, 16, off, kb, 0, 0);
        else
          __builtin_amdgcn_raw_ptr_buffer_load_lds(rb[q][kHalves - 1], dst, 16, off, kb, 0, 0);
      }
    }
  };

  floatx4 acc[C::FN][C::FM];
#pragma unroll
  for (int i = 0; i < C::FN; ++i)
#pragma unroll
    for (int j = 0; j < C::FM; ++j) acc[i][j] = floatx4{0.f, 0.f, 0.f, 0.f};

  const int fr = lane & 15, fc = lane >> 4;  // fragment row, k unit
  if (s0 < s1) load_stage(s0, 0);
  for (int64_t s = s0; s < s1; ++s) {
    const int buf = (int)(s - s0) & 1;
    // this wave's loads of stage s are in LDS; after the barrier everyone's are, and nobody reads the
    // other buffer any more
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (s + 1 < s1) load_stage(s + 1, buf ^ 1);
    const char* sa = lds + buf * C::kStage;
    const char* sb = sa + PA * TM * BK * 2;
#pragma unroll
    for (int kk = 0; kk < BK / 32; ++kk) {
      bf16x8 fa[PA][C::FM], fb[PB][C::FN];
#pragma unroll
      for (int q = 0; q < PB; ++q)
#pragma unroll
        for (int i = 0; i < C::FN; ++i) {
          const int r = wn * C::WTN + i * 16 + fr;
          fb[q][i] = *reinterpret_cast<const bf16x8*>(sb + ((q * TN + r) * U + swz<U>(r, kk * 4 + fc)) * 16);
        }
#pragma unroll
      for (int q = 0; q < PA; ++q)
#pragma unroll
        for (int j = 0; j < C::FM; ++j) {
          const int r = wm * C::WTM + j * 16 + fr;
          fa[q][j] = *reinterpret_cast<const bf16x8*>(sa + ((q * TM + r) * U + swz<U>(r, kk * 4 + fc)) * 16);
        }
      // small plane products first
#pragma unroll
      for (int sum = (PA == 3 || PB == 3) ? 2 : 0; sum >= 0; --sum)
#pragma unroll
        for (int qa = 0; qa < PA; ++qa) {
          const int qb = sum - qa;
          if (qb < 0 || qb >= PB) continue;
#pragma unroll
          for (int i = 0; i < C::FN; ++i)
#pragma unroll
            for (int j = 0; j < C::FM; ++j)
              acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fb[qb][i], fa[qa][j], acc[i][j], 0, 0, 0);
        }
    }
  }

  // ------------------------------------------------------------------------------------------
  constexpr int FH = C::FN / kHalves;
  const bool vec = p.vec;
#pragma unroll
  for (int j = 0; j < C::FM; ++j) {
    const int64_t m = m0 + wm * C::WTM + j * 16 + fr;
    if (m >= p.M) continue;
#pragma unroll
    for (int i = 0; i < FH; ++i) {
      const int64_t n = n0 + wn * (C::WTN / kHalves) + i * 16 + fc * 4;
      if (n >= p.N) continue;
      const int64_t left = p.N - n;
      const bool v4 = vec && left >= 4;
      floatx4 v = acc[i][j];
      if constexpr (EPI == kSlab) {
        store4(p.slab + ((int64_t)split * p.M + m) * p.N + n, v, v4, left);
      } else if constexpr (EPI == kGated) {
        floatx4 u = acc[i + FH][j];
        if (p.bias) v += load4((const T*)p.bias + n, v4, left);
        if (p.bias2) u += load4((const T*)p.bias2 + n, v4, left);
        if (p.pre) {
          store4(p.pre + m * 2 * p.N + n, v, v4, left);
          store4(p.pre + m * 2 * p.N + p.N + n, u, v4, left);
        }
        if (p.y) {
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] = (sizeof(T) == 2 ? act_fast(p.act, v[e]) : act_fwd(p.act, v[e])) * u[e];
          store4((T*)p.y + m * p.ldy + n, v, v4, left);
        }
      } else {
        if (p.bias) v += load4((const T*)p.bias + n, v4, left);
        if (p.pre) store4(p.pre + m * p.N + n, v, v4, left);
        if (p.y) {
          if (p.act >= 0) {
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = sizeof(T) == 2 ? act_fast(p.act, v[e]) : act_fwd(p.act, v[e]);
          }
          if (p.res) v += load4((const T*)p.res + m * p.ldr + n, v4, left);
          T* y = m < p.y_rows ? (T*)p.y + m * p.ldy : (T*)p.y2 + (m - p.y_rows) * p.ldy;
          store4(y + n, v, v4, left);
        }
      }
    }
  }
#endif
}

// A tile shape (0: the largest) and the number of k ranges of one launch.
struct Plan {
  int tile, splits;
};
// `columns`: of both halves together. may_split: a plain product whose partial sums may go to slabs.
Plan plan_one(int64_t M, int64_t columns, int64_t K, bool may_split);
Plan plan_split(int64_t M, int64_t columns, int64_t K, bool may_split);
// Launchers (dense_bf16.hip: one plane a side; dense_split.hip: three planes on one side or both, fp32 out).
// p.splits > 1: the partial sums go to p.slab and reduce_slabs (dense.hip) applies the epilogue.
int launch_one(const Problem& p, int tile, int halves, bool fp32_out, hipStream_t st);
int launch_split(const Problem& p, int tile, int pa, int pb, int halves, hipStream_t st);

template <typename C, int EPI, typename T>
int launch_config(const Problem& p, hipStream_t st) {
  constexpr int TC = C::TN / (EPI == kGated ? 2 : 1);
  const int64_t tm = cdiv(p.M, C::TM), tn = cdiv(p.N, TC);
  if (tm * tn > (int64_t)INT32_MAX) return AIMX_EARG;
  hipLaunchKernelGGL((k_dense<C, EPI, T>), dim3((unsigned)(tm * tn), (unsigned)p.splits), dim3(C::kThreads), 0, st, p,
                     (int)tm, (int)tn);
  AIMX_CHECK_LAUNCH();
  return AIMX_OK;
}

}  // namespace dense
}  // namespace aimx
