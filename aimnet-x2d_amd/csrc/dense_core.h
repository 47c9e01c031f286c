// The tiled matrix product behind dense.hip: D[m][n] = sum_k A[m][k] B[n][k] on the bf16 matrix cores,
// with the epilogues of the dense and gated operators.
//
// Operands are bf16 "planes": a bf16 matrix is one plane, an fp32 matrix three whose sum is the matrix,
// x = x1 + x2 + x3 exactly (8 + 8 + 8 mantissa bits) from 2^-110 on; below, where the third plane's last bit would
// be less than bf16's least subnormal 2^-133, within 2^-134. The product of two three-plane
// operands takes the six plane products x_i w_j with i + j <= 4 (Henry, Tang, Heinecke, "Leveraging the
// bfloat16 Artificial Intelligence Datatype For Higher-Precision Computations", 2019): what is left out
// is at most 2^-23 |x||w|, the products of planes are exact (8 x 8 bits) and their sums are
// fp32. Six bf16 instructions replace sixteen times slower fp32 ones. Against a one-plane operand three
// plane products are the whole product.
//
// An operand is read along its rows (k contiguous) or across them: a matrix whose rows run along k (the
// weight in dx, both operands in dW) goes into LDS as it is and is transposed by the fragment reads
// (ds_read_b64_tr_b16), so no product needs a transposed copy.
//
// Layout rules (the host stages operands that break them): rows 16-byte aligned. Along the rows: the k extent a
// multiple of 64 elements, zeros behind the matrix's own columns. Across: columns a multiple of 8. Rows and k
// past the end read zeros through the buffer descriptors, which end with the matrix.
// Bound: the matrix cores, then LDS reads (a 128 x 64 wave tile reads 12 KB per 32 matrix instructions, three
// quarters of LDS's rate; a 64 x 64 one all of it), then the epilogue where k is short. Measured, us and TFLOP/s of a
// launch: 32768 x 1024 over k = 8192 (dx) 450, 1220; 8192 x 1024 over k = 32768 (dW) 452, 1215; the gated forward
// 32768 x 1024 -> 2 x 4096 538, 1022, its gradient epilogue 695; 20480 x 512 -> 2 x 2048 113, 760. Three planes
// a side, as fp32: 32768 x 2048 over k = 1024 639 to 656, 209 to 215.
#pragma once

#include <algorithm>

#include "aimx_common.h"

namespace aimx {
namespace dense {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef uint16_t u16x4 __attribute__((ext_vector_type(4)));
typedef uint16_t u16x8 __attribute__((ext_vector_type(8)));
// the same in memory at any element: gfx950 takes 8- and 16-byte accesses at such addresses (within 8 % of the aligned
// rate), so no row needs an alignment
typedef float floatx4e __attribute__((ext_vector_type(4), aligned(4)));
typedef uint16_t u16x4e __attribute__((ext_vector_type(4), aligned(2)));
typedef uint16_t u16x8e __attribute__((ext_vector_type(8), aligned(2)));

// fp32 -> bf16 bits, round to nearest even; NaN stays NaN
__device__ __forceinline__ uint16_t to_bf16(float v) {
  union { __bf16 b; uint16_t u; } c;
  c.b = (__bf16)v;
  return c.u;
}
__device__ __forceinline__ float from_bf16(uint16_t u) { return __uint_as_float((uint32_t)u << 16); }

// The three planes of v, each the nearest bf16 of what is left: |x2| <= 2^-8 |x|, |x3| <= 2^-16 |x|, and the
// third is exact (24 = 8 + 8 + 8 bits; |x| >= 2^-110). A NaN or infinity goes whole into the first plane; what it then
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

// One operand of a product: `rows` rows of `cols` elements, planes `plane` elements apart. p2: the second weight (the
// gated forward's second half of columns; across the rows, the second half of k).
struct Operand {
  const uint16_t* p;
  const uint16_t* p2;
  int64_t ld, plane, rows, cols;
};

struct Problem {
  Operand a, b;
  int64_t M, N, K;       // N: columns of the result (of one half where the epilogue is gated); K % 64 == 0
  int64_t k_half;        // k of one half of an operand read across its rows (K where there is one)
  void* y;               // [M][N], ld ldy (nullptr: only pre)
  void* y2;              // rows >= y_rows of the result go to y2 (weight gradients of two weights)
  int64_t ldy, y_rows, y_valid;  // of each half's rows, y_valid are written
  const void* bias;      // [N], of the output's type; bias2: of the second half
  const void* bias2;
  const void* res;       // [M][N], ld ldr; the backward epilogues: dy
  int64_t ldr;
  float* pre;            // [M][halves][n8] fp32, before the activation
  float* slab;           // split-k partial sums [splits][M][N]
  uint16_t* rows;        // backward epilogues: the gradient before the activation, planes of [M][halves * np]
  int64_t rows_plane;
  float* sums;           // backward epilogues, nullable: column sums [tiles of rows * WGM][halves * N]
  int64_t n8, np;        // N rounded up to 8, to 64
  int32_t act, splits;
};

// kDenseGrad / kGatedGrad: the product is the forward's, computed again; what leaves the kernel is the gradient
// before the activation, dP = dy act'(p) or [dG | dU]
enum Epi : int { kPlain = 0, kGated = 1, kSlab = 2, kDenseGrad = 3, kGatedGrad = 4 };
// the operands read across their rows: none (forward), b (dx), both (dW)
enum Across : int { kNone = 0, kB = 1, kBoth = 2 };

template <int PA_, int PB_, int TM_, int TN_, int WGM_, int WGN_, int BK_>
struct Config {
  static constexpr int PA = PA_, PB = PB_, TM = TM_, TN = TN_, WGM = WGM_, WGN = WGN_, BK = BK_;
  static_assert(WGM == 2, "kWavesM");
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

// Across the rows, LDS holds [k][rows]: 32-byte blocks of 16 rows, permuted by k so that the values of k that half a
// wave's transposing read touches (2 groups of 8, 4 of each) lie in different banks.
template <int ROWS>
__device__ __forceinline__ int swz_t(int k, int block) {
  return block ^ (((k & 3) | ((k >> 1) & 4)) & (ROWS / 16 - 1));
}

// Activations of several values with one branch on the kind: a branch per value costs more than the value's
// arithmetic. FAST: hardware exp2 and reciprocal (about 2^-21 each) in silu, for results rounded to 8 bits.
template <bool FAST, int KIND>
__device__ __forceinline__ void act_one(float v, float& a, float& da) {
  if constexpr (FAST && KIND == ACT_SILU) {
    const float s = __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-1.44269504f * v));
    a = v * s;
    da = s * (1.f + v * (1.f - s));
  } else if constexpr (KIND == ACT_SILU) {
    const float s = 1.f / (1.f + expf(-v));
    a = v / (1.f + expf(-v));
    da = s * (1.f + v * (1.f - s));
  } else {
    a = act_fwd(KIND, v);
    da = act_grad(KIND, v);
  }
}
template <bool FAST, int KIND, int N>
__device__ __forceinline__ void act_each(const float (&v)[N], float (&a)[N], float (&da)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) act_one<FAST, KIND>(v[i], a[i], da[i]);
}
// a(v) and a'(v); what the caller does not use is not computed
template <bool FAST, int N>
__device__ __forceinline__ void act_all(int kind, const float (&v)[N], float (&a)[N], float (&da)[N]) {
  switch (kind) {
    case ACT_RELU: return act_each<FAST, ACT_RELU>(v, a, da);
    case ACT_LEAKYRELU: return act_each<FAST, ACT_LEAKYRELU>(v, a, da);
    case ACT_ELU: return act_each<FAST, ACT_ELU>(v, a, da);
    case ACT_GELU: return act_each<FAST, ACT_GELU>(v, a, da);
    case ACT_SILU: return act_each<FAST, ACT_SILU>(v, a, da);
    default: return act_each<FAST, ACT_NONE>(v, a, da);
  }
}

template <typename T>
__device__ __forceinline__ float load1(const T* p);
template <>
__device__ __forceinline__ float load1<float>(const float* p) { return *p; }
template <>
__device__ __forceinline__ float load1<uint16_t>(const uint16_t* p) { return from_bf16(*p); }

// four consecutive values, `left` of which exist (the others: zero)
template <typename T>
__device__ __forceinline__ floatx4 load4(const T* p, int64_t left) {
  floatx4 v;
  if (left >= 4) {
    if constexpr (sizeof(T) == 4) {
      v = *reinterpret_cast<const floatx4e*>(p);
    } else {
      const u16x4 h = *reinterpret_cast<const u16x4e*>(p);
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
__device__ __forceinline__ void store4(T* p, floatx4 v, int64_t left) {
  if (left >= 4) {
    if constexpr (sizeof(T) == 4) {
      *reinterpret_cast<floatx4e*>(p) = v;
    } else {
      u16x4 h;
#pragma unroll
      for (int i = 0; i < 4; ++i) h[i] = to_bf16(v[i]);
      *reinterpret_cast<u16x4e*>(p) = h;
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
// 8 values from p, `left` of which exist (the others: zero)
template <typename T>
__device__ __forceinline__ void load8(const T* p, int64_t left, float (&v)[8]) {
  if (left >= 8) {
    if constexpr (sizeof(T) == 4) {
      const floatx4 a = *reinterpret_cast<const floatx4e*>(p), b = *reinterpret_cast<const floatx4e*>(p + 4);
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = a[i], v[4 + i] = b[i];
    } else {
      const u16x8 a = *reinterpret_cast<const u16x8e*>(p);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = from_bf16(a[i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < left ? load1(p + i) : 0.f;
  }
}
template <typename T>
__device__ __forceinline__ void store8(T* p, int64_t left, const float (&v)[8]) {
  if (left >= 8) {
    if constexpr (sizeof(T) == 4) {
      *reinterpret_cast<floatx4e*>(p) = floatx4{v[0], v[1], v[2], v[3]};
      *reinterpret_cast<floatx4e*>(p + 4) = floatx4{v[4], v[5], v[6], v[7]};
    } else {
      u16x8 o;
#pragma unroll
      for (int i = 0; i < 8; ++i) o[i] = to_bf16(v[i]);
      *reinterpret_cast<u16x8e*>(p) = o;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < left) {
        if constexpr (sizeof(T) == 4) p[i] = v[i];
        else p[i] = to_bf16(v[i]);
      }
  }
}

// Four values loaded from up to 3 columns in front of where they belong (the last ones of a row whose length is no
// multiple of 4), converted and shifted into place where they are used.
template <typename T>
struct Raw4 {
  typedef T t4 __attribute__((ext_vector_type(4)));
  typedef T t4e __attribute__((ext_vector_type(4), aligned(sizeof(T))));
  t4 h;
  __device__ __forceinline__ void load(const T* p) { h = *reinterpret_cast<const t4e*>(p); }
  __device__ __forceinline__ floatx4 get() const {
    if constexpr (sizeof(T) == 4) return h;
    else return floatx4{from_bf16(h[0]), from_bf16(h[1]), from_bf16(h[2]), from_bf16(h[3])};
  }
  __device__ __forceinline__ floatx4 get(int shift) const {
    const floatx4 v = get();
    floatx4 o;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      o[e] = 0.f;
#pragma unroll
      for (int k = 0; e + k < 4; ++k) o[e] = shift == k ? v[e + k] : o[e];
    }
    return o;
  }
};

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));

// Loads of one operand's stage into LDS, straight from global memory (16 bytes a lane, no registers).
template <typename C, bool T, int P, int ROWS, int HALVES, int WT>
struct Loader {
  static constexpr int kWaves = C::kThreads / kWave;
  static constexpr int kLoads = ROWS * C::U / kWave / kWaves;  // of a wave, per plane
  static constexpr int UR = ROWS / 8;                          // units of a k row, across
  // rows (across: of k) that all waves' j-th loads cover: the permutations repeat after as many, so a lane keeps one
  // offset and load j adds to it
  static constexpr int kStep = kWaves * (T ? kWave / UR : C::kRowsPerLoad);
  static_assert(ROWS * C::U % (kWave * kWaves) == 0, "every wave issues whole loads");
  static_assert(kStep % (T ? 16 : 8) == 0, "the permutations repeat");
  static_assert(T || HALVES == 1 || ((kStep % WT == 0 || WT / 2 % kStep == 0) && WT / 2 >= C::kRowsPerLoad),
                "a load lies inside one half");
  const Operand& o;
  int64_t row0;
  int wave;
  uint32_t off;  // of this lane in load 0
  __amdgpu_buffer_rsrc_t r[T ? 1 : P][HALVES];

  // the row of a half (gated: a wave's WT columns are WT / 2 of the first half, then of the second) that LDS row
  // `row` holds
  static __device__ __forceinline__ constexpr int source_row(int row) {
    return HALVES == 1 ? row : row / WT * (WT / 2) + row % (WT / 2);
  }

  __device__ __forceinline__ Loader(const Operand& o_, int64_t row0_, int wave_, int lane) : o(o_), row0(row0_), wave(wave_) {
    const int u = wave * kWave + lane;
    if constexpr (T) {
      const int k = u / UR, c = u % UR;
      off = (uint32_t)k * (uint32_t)o.ld * 2 + swz_t<ROWS>(k, c >> 1) * 32 + (c & 1) * 16;
    } else {
      const int row = u / C::U;
      off = (uint32_t)source_row(row) * (uint32_t)o.ld * 2 + swz<C::U>(row, u % C::U) * 16;
      // one descriptor per plane and half, over the tile's rows
      const int64_t left = o.rows - row0;
      const uint32_t bytes = (uint32_t)(min((int64_t)(ROWS / HALVES), max(left, (int64_t)0)) * o.ld * 2);
#pragma unroll
      for (int q = 0; q < P; ++q) {
        r[q][0] = buffer_rsrc(o.p + q * o.plane + row0 * o.ld, bytes);
        if (HALVES == 2) r[q][HALVES - 1] = buffer_rsrc(o.p2 + q * o.plane + row0 * o.ld, bytes);
      }
    }
  }

  // Rows are skipped by the offset that the descriptor's range is checked against: a scalar offset is subtracted from the
  // range first, which would wrap where fewer bytes are left than it skips. Along the rows the scalar is k, which
  // stays inside the first row (0 where the tile has no row).
  __device__ __forceinline__ void load(char* base, int64_t step, int64_t k_half) const {
    typedef __attribute__((address_space(3))) void lds_void;
    const uint32_t ld2 = (uint32_t)o.ld * 2;
    if constexpr (T) {
      int64_t k0 = step * C::BK;
      const uint16_t* p = o.p;
      if (k0 >= k_half) p = o.p2, k0 -= k_half;
      // the descriptor of these k rows ends with the matrix
      const int64_t kr = min((int64_t)C::BK, o.rows - k0);
      const uint32_t bytes = kr > 0 && row0 < o.cols ? (uint32_t)(((kr - 1) * o.ld + o.cols - row0) * 2) : 0;
#pragma unroll
      for (int q = 0; q < P; ++q) {
        const __amdgpu_buffer_rsrc_t d = buffer_rsrc(p + q * o.plane + k0 * o.ld + row0, bytes);
#pragma unroll
        for (int j = 0; j < kLoads; ++j)
          __builtin_amdgcn_raw_ptr_buffer_load_lds(
              d, (lds_void*)(base + (q * ROWS * C::U + (j * kWaves + wave) * kWave) * 16), 16, off + j * kStep * ld2, 0, 0,
              0);
      }
    } else {
      const uint32_t kb = row0 < o.rows ? (uint32_t)(step * C::BK * 2) : 0u;
#pragma unroll
      for (int j = 0; j < kLoads; ++j) {
        const int half = HALVES == 1 ? 0 : ((j * kStep + wave * C::kRowsPerLoad) / (WT / 2)) & 1;
        const uint32_t at = off + source_row(j * kStep) * ld2;
#pragma unroll
        for (int q = 0; q < P; ++q) {
          lds_void* dst = (lds_void*)(base + (q * ROWS * C::U + (j * kWaves + wave) * kWave) * 16);
          if (half == 0) __builtin_amdgcn_raw_ptr_buffer_load_lds(r[q][0], dst, 16, at, kb, 0, 0);
          else __builtin_amdgcn_raw_ptr_buffer_load_lds(r[q][HALVES - 1], dst, 16, at, kb, 0, 0);
        }
      }
    }
  }

  // Fragments of 16 rows, F of them from row `row`, at k = kk * 32 .. + 31: lane = row % 16, 8 values of k from
  // 8 (lane / 16) on.
  template <int F>
  static __device__ __forceinline__ void fragments(const char* base, int q, int row, int kk, int lane, bf16x8 (&f)[F]) {
    if constexpr (T) {
      // k = kk * 32 + 8 (lane / 16) + 4 i + (lane % 16) / 4 for the halves i of the 8 values: the blocks'
      // permutation depends on the lane alone
      const int kl = (lane >> 4) * 8 + ((lane & 15) >> 2);
      const char* at0 = base + ((q * C::BK + kk * 32 + kl) * (ROWS / 8)) * 16 + (lane & 3) * 8;
#pragma unroll
      for (int j = 0; j < F; ++j) {
        auto at = (__attribute__((address_space(3))) s16x4*)(at0 + swz_t<ROWS>(kl, (row >> 4) + j) * 32);
        const s16x4 l = __builtin_amdgcn_ds_read_tr16_b64_v4i16(at), h = __builtin_amdgcn_ds_read_tr16_b64_v4i16(at + ROWS);
        f[j] = __builtin_bit_cast(bf16x8, __builtin_shufflevector(l, h, 0, 1, 2, 3, 4, 5, 6, 7));
      }
    } else {
#pragma unroll
      for (int j = 0; j < F; ++j) {
        const int r = row + j * 16 + (lane & 15);
        f[j] = *reinterpret_cast<const bf16x8*>(base + ((q * ROWS + r) * C::U + swz<C::U>(r, kk * 4 + (lane >> 4))) * 16);
      }
    }
  }
};

template <typename C, int EPI, typename T, bool WIDE>
__device__ __forceinline__ void epilogue(const Problem& p, floatx4 (&acc)[C::FN][C::FM], int tm, int64_t m0, int64_t n0,
                                         int wm, int wn, int lane, int split) {
  constexpr int kHalves = EPI == kGated || EPI == kGatedGrad ? 2 : 1, FH = C::FN / kHalves;
  constexpr bool kFast = sizeof(T) == 2, kGrad = EPI == kDenseGrad || EPI == kGatedGrad;
  constexpr int PL = kGrad && sizeof(T) == 4 && C::PB == 3 ? 3 : 1;
  const int fr = lane & 15, fc = lane >> 4;
  int64_t nn[FH], nl[FH];  // a lane's first columns, where they are loaded from
  floatx4 b0[FH], b1[FH], total[kHalves][FH];
#pragma unroll
  for (int i = 0; i < FH; ++i) {
    nn[i] = n0 + wn * (C::WTN / kHalves) + i * 16 + fc * 4;
    nl[i] = min(nn[i], p.N - 4);
    b0[i] = b1[i] = floatx4{0.f, 0.f, 0.f, 0.f};
    if constexpr (EPI != kSlab) {
      if (p.bias) b0[i] = load4((const T*)p.bias + nn[i], p.N - nn[i]);
      if (kHalves == 2 && p.bias2) b1[i] = load4((const T*)p.bias2 + nn[i], p.N - nn[i]);
    }
#pragma unroll
    for (int h = 0; h < kHalves; ++h) total[h][i] = floatx4{0.f, 0.f, 0.f, 0.f};
  }
  constexpr bool kRes = EPI == kPlain || kGrad;
  const bool whole = p.N % 4 == 0;
  // a row's operand: in flight where rows hold at least 4 columns, else read where it is used
  auto operand = [&](const Raw4<T>& d, int64_t m, int i) __attribute__((always_inline)) -> floatx4 {
    if constexpr (!WIDE) return load4((const T*)p.res + m * p.ldr + nn[i], p.N - nn[i]);
    const int64_t shift = nn[i] - nl[i];
    if (whole) return shift > 0 ? floatx4{0.f, 0.f, 0.f, 0.f} : d.get();
    return d.get((int)min(shift, (int64_t)4));
  };
  // rows whose operands are in flight together, 32 registers of them
  constexpr int kMost = 32 / sizeof(T) / FH, kAhead = kMost < 1 ? 1 : kMost < C::FM ? kMost : C::FM;
#pragma unroll
  for (int j0 = 0; j0 < C::FM; j0 += kAhead) {
    Raw4<T> d[kAhead][FH];
    if constexpr (kRes && WIDE) {
      if (p.res) {
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
          const int64_t m = min(m0 + wm * C::WTM + (j0 + j) * 16 + fr, p.M - 1);
#pragma unroll
          for (int i = 0; i < FH; ++i) d[j][i].load((const T*)p.res + m * p.ldr + nl[i]);
        }
      }
    }
#pragma unroll
    for (int jj = 0; jj < kAhead; ++jj) {
      const int j = j0 + jj;
      const int64_t m = m0 + wm * C::WTM + j * 16 + fr;
      if (m >= p.M) continue;
      float v[FH * 4], a[FH * 4], da[FH * 4];
#pragma unroll
      for (int i = 0; i < FH; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) a[4 * i + e] = v[4 * i + e] = acc[i][j][e] + b0[i][e];
      if constexpr (EPI == kGated || EPI == kPlain) {
        if (p.pre) {
#pragma unroll
          for (int i = 0; i < FH; ++i) {
            if (nn[i] >= p.N) continue;
            float* at = p.pre + m * kHalves * p.n8 + nn[i];
            *reinterpret_cast<floatx4*>(at) = floatx4{v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]};
            if constexpr (kHalves == 2) *reinterpret_cast<floatx4*>(at + p.n8) = acc[i + FH][j] + b1[i];
          }
        }
      }
      if constexpr (kGrad || EPI == kGated) {
        act_all<kFast>(p.act, v, a, da);
      } else if constexpr (EPI == kPlain) {
        if (p.act >= 0) act_all<kFast>(p.act, v, a, da);
      }
#pragma unroll
      for (int i = 0; i < FH; ++i) {
        const int64_t n = nn[i], left = p.N - n;
        if (n >= (kGrad ? p.np : p.N)) continue;
        floatx4 o = {a[4 * i], a[4 * i + 1], a[4 * i + 2], a[4 * i + 3]};
        if constexpr (kGrad) {
          floatx4 out[kHalves];
          const floatx4 dd = operand(d[jj][i], m, i);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            if constexpr (kHalves == 2) {
              out[0][e] = dd[e] * (acc[i + FH][j][e] + b1[i][e]) * da[4 * i + e];
              out[kHalves - 1][e] = dd[e] * o[e];
            } else {
              out[0][e] = dd[e] * da[4 * i + e];
            }
          }
          // Columns behind N only pad the rows. Their sums are x times zero, NaN where x is infinite, and 0 * NaN would
          // reach dx, which reads them.
          if (left < 4) {
#pragma unroll
            for (int h = 0; h < kHalves; ++h)
#pragma unroll
              for (int e = 0; e < 4; ++e) out[h][e] = e < left ? out[h][e] : 0.f;
          }
#pragma unroll
          for (int h = 0; h < kHalves; ++h) {
            total[h][i] += out[h];
            u16x4 w[PL];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              if constexpr (PL == 1) {
                w[0][e] = to_bf16(out[h][e]);
              } else {
                uint16_t q3[3];
                split3(out[h][e], q3);
#pragma unroll
                for (int q = 0; q < PL; ++q) w[q][e] = q3[q];
              }
            }
            uint16_t* at = p.rows + (m * kHalves + h) * p.np + n;
#pragma unroll
            for (int q = 0; q < PL; ++q) *reinterpret_cast<u16x4*>(at + q * p.rows_plane) = w[q];
          }
        } else if constexpr (EPI == kSlab) {
          store4(p.slab + ((int64_t)split * p.M + m) * p.N + n, o, left);
        } else if constexpr (EPI == kGated) {
          store4((T*)p.y + m * p.ldy + n, o * (acc[i + FH][j] + b1[i]), left);
        } else {
          if (p.res) o += operand(d[jj][i], m, i);
          const int64_t r = m < p.y_rows ? m : m - p.y_rows;
          if (r < p.y_valid) store4((T*)(m < p.y_rows ? p.y : p.y2) + r * p.ldy + n, o, left);
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    __builtin_amdgcn_sched_barrier(0);  // or the addresses of every row are live at once
  }
  if constexpr (kGrad) {
    if (p.sums) {  // the 16 rows of a fragment in a fixed tree
#pragma unroll
      for (int i = 0; i < FH; ++i)
#pragma unroll
        for (int h = 0; h < kHalves; ++h)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float t = total[h][i][e];
#pragma unroll
            for (int o = 1; o < 16; o <<= 1) t += __shfl_xor(t, o);
            if (fr == 0 && nn[i] + e < p.N)
              p.sums[((int64_t)tm * C::WGM + wm) * kHalves * p.N + h * p.N + nn[i] + e] = t;
          }
    }
  }
}

// One workgroup: one TM x TN tile (gated: TN / 2 columns of each half) over one k range. Two LDS stages: stage t + 1 is
// in flight through the matrix work of stage t. The weight is the instruction's first operand, so that a lane
// holds four consecutive columns of one row: 8- and 16-byte stores.
template <typename C, int EPI, int ACROSS, typename T>
__global__ __launch_bounds__(C::kThreads) void k_dense(const Problem p, const int tiles_m, const int tiles_n) {
#ifdef __HIP_DEVICE_COMPILE__  // the host pass drops the stub of a body with the LDS load builtin
  constexpr int PA = C::PA, PB = C::PB, TM = C::TM, TN = C::TN, BK = C::BK;
  constexpr int kHalves = EPI == kGated || EPI == kGatedGrad ? 2 : 1, TC = TN / kHalves;  // columns of a half in a tile
  static_assert(kHalves == 1 || ACROSS == kNone, "the gated epilogues belong to the forward product");
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
  const int tm = first + in % gsz;
  const int64_t m0 = (int64_t)tm * TM, n0 = (int64_t)(in / gsz) * TC;

  const int split = blockIdx.y;
  const int64_t steps = p.K / BK;
  const int64_t s0 = steps * split / p.splits, s1 = steps * (split + 1) / p.splits;

  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int wm = wave / C::WGN, wn = wave % C::WGN;
  using LA = Loader<C, ACROSS == kBoth, PA, TM, 1, C::WTM>;
  using LB = Loader<C, ACROSS != kNone, PB, TN, kHalves, C::WTN>;
  const LA la(p.a, m0, wave, lane);
  const LB lb(p.b, n0, wave, lane);

  floatx4 acc[C::FN][C::FM];
#pragma unroll
  for (int i = 0; i < C::FN; ++i)
#pragma unroll
    for (int j = 0; j < C::FM; ++j) acc[i][j] = floatx4{0.f, 0.f, 0.f, 0.f};

  auto load = [&](char* at, int64_t step) __attribute__((always_inline)) {
    la.load(at, step, p.k_half);
    lb.load(at + PA * TM * BK * 2, step, p.k_half);
  };
  struct Set {
    bf16x8 a[PA][C::FM], b[PB][C::FN];
  };
  auto read = [&](const char* at, int kk, Set& t) __attribute__((always_inline)) {
#pragma unroll
    for (int q = 0; q < PB; ++q) LB::template fragments<C::FN>(at + PA * TM * BK * 2, q, wn * C::WTN, kk, lane, t.b[q]);
#pragma unroll
    for (int q = 0; q < PA; ++q) LA::template fragments<C::FM>(at, q, wm * C::WTM, kk, lane, t.a[q]);
  };
  auto multiply = [&](const Set& t) __attribute__((always_inline)) {
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
            acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(t.b[qb][i], t.a[qa][j], acc[i][j], 0, 0, 0);
      }
  };
  constexpr int kVmcnt0 = 0x0f70;  // s_waitcnt vmcnt(0), the other counters as they are
  // The stages' addresses are __restrict: without it the compiler takes every transposing read to depend on the
  // loads into LDS in flight and waits for them first.
  if constexpr (C::kThreads == 512) {
    // Two groups of four waves, one of each on a SIMD, half a step apart: while one reads its fragments the other
    // has the matrix cores. Every phase ends at a barrier; the second group starts one barrier late and the first
    // ends with one more.
    //   phase 2 i:      first reads set i          second multiplies set i - 1
    //   phase 2 i + 1:  first multiplies set i     second reads set i
    // A group loads its share of stage s + 1 as it begins to read stage s: by then both groups' reads of stage s - 1,
    // whose place it takes, have ended (the other's last one a barrier ago). Both wait for their shares before
    // the barrier in front of the first group's first read of stage s + 1.
    // The barrier alone: __syncthreads would wait for the loads into LDS at every one.
    constexpr int kLgkmcnt0 = 0xc07f;
    auto phase = [&]() __attribute__((always_inline)) {
      asm volatile("" ::: "memory");
      __builtin_amdgcn_sched_barrier(0);
      __builtin_amdgcn_s_barrier();
      __builtin_amdgcn_sched_barrier(0);
      asm volatile("" ::: "memory");
    };
    const bool second = wave >= 4;
    auto stage = [&](char* __restrict next, const char* __restrict now, int64_t s) __attribute__((always_inline)) {
#pragma unroll
      for (int kk = 0; kk < BK / 32; ++kk) {
        Set f;
        if (kk == 0 && s + 1 < s1) load(next, s + 1);
        read(now, kk, f);
        if (kk == BK / 32 - 1 && second) __builtin_amdgcn_s_waitcnt(kVmcnt0);
        __builtin_amdgcn_s_waitcnt(kLgkmcnt0);
        phase();
        __builtin_amdgcn_s_setprio(1);
        multiply(f);
        __builtin_amdgcn_s_setprio(0);
        if (kk == BK / 32 - 1 && !second) __builtin_amdgcn_s_waitcnt(kVmcnt0);
        phase();
      }
    };
    if (s0 < s1) load(lds, s0);
    __builtin_amdgcn_s_waitcnt(kVmcnt0);
    __syncthreads();
    if (second) phase();
    for (int64_t s = s0; s < s1; ++s) {
      const int buf = (int)(s - s0) & 1;
      stage(lds + (buf ^ 1) * C::kStage, lds + buf * C::kStage, s);
    }
    if (!second) phase();
  } else {
    // one stage: its fragments and their products, while the next stage comes in
    auto stage = [&](char* __restrict next, const char* __restrict now, int64_t s) __attribute__((always_inline)) {
      if (s + 1 < s1) load(next, s + 1);
#pragma unroll
      for (int kk = 0; kk < BK / 32; ++kk) {
        Set f;
        read(now, kk, f);
        multiply(f);
      }
    };
    if (s0 < s1) load(lds, s0);
    for (int64_t s = s0; s < s1; ++s) {
      const int buf = (int)(s - s0) & 1;
      // this wave's loads of stage s are in LDS; after the barrier everyone's are, and nobody reads the
      // other buffer any more
      __builtin_amdgcn_s_waitcnt(kVmcnt0);
      __syncthreads();
      stage(lds + (buf ^ 1) * C::kStage, lds + buf * C::kStage, s);
    }
  }

  // ------------------------------------------------------------------------------------------
  // The epilogue's operands come by unconditional loads (of the last row and the last four columns in place of those
  // past the end), several rows' in flight together; rows of fewer than four columns have a form of their own.
  if (p.N >= 4) epilogue<C, EPI, T, true>(p, acc, tm, m0, n0, wm, wn, lane, split);
  else epilogue<C, EPI, T, false>(p, acc, tm, m0, n0, wm, wn, lane, split);
#endif
}

// A tile shape and the number of k ranges of one launch, picked by an estimate of its time.
struct Shape {
  int tile;        // index of the launchers
  int64_t rows, cols, bk;
  int per_cu;      // workgroups that fit a CU
  double step, end;  // us: one k step of a workgroup with its CU full, its prologue and epilogue (measured)
};
struct Plan {
  int tile, splits;
  int64_t rows;
};
constexpr int kWavesM = 2;  // rows of waves of every tile: a tile leaves that many parts of column sums
constexpr int kCus = 256;
// `columns`: of both halves together. may_split: a plain product whose partial sums may go to slabs.
inline Plan pick(const Shape* shapes, int n, int64_t M, int64_t columns, int64_t K, bool may_split) {
  Plan best{shapes[0].tile, 1, shapes[0].rows};
  double least = 1e30;
  for (int i = 0; i < n; ++i) {
    const Shape& s = shapes[i];
    const int64_t tiles = std::max<int64_t>(1, cdiv(M, s.rows) * cdiv(columns, s.cols)), steps = K / s.bk;
    const int64_t most = may_split ? std::max<int64_t>(1, std::min<int64_t>(steps * s.bk / 256, 64)) : 1;
    for (int64_t k = 1; k <= most; ++k) {
      const int64_t all = tiles * k, slots = (int64_t)kCus * s.per_cu, rest = all % slots;
      // workgroups that share a CU with fewer are faster, alone about twice as fast as among three
      const double part = rest == 0 ? 0. : s.per_cu == 1 ? 1. : std::max(0.47, 0.2 + 0.8 * (double)rest / (double)slots);
      const double rounds = (double)(all / slots) + part;
      double t = rounds * ((double)cdiv(steps, k) * s.step + s.end);
      // one more launch reads the slabs, which the caches hold in part: 8 of 4 MB in 6.8 us
      if (k > 1) t += 4. + (double)(3 * k + 2) * (double)M * (double)columns / 4.5e6;
      if (t < least) least = t, best = Plan{s.tile, (int)k, s.rows};
      if (all > 16 * slots) break;
    }
  }
  return best;
}
Plan plan_one(int64_t M, int64_t columns, int64_t K, bool may_split);
Plan plan_split(int64_t M, int64_t columns, int64_t K, bool may_split, bool fp32);
// Launchers (dense_bf16.hip: one plane a side; dense_split.hip: three planes on one side or both).
// epi: kPlain, kGated, kDenseGrad or kGatedGrad. p.splits > 1 (kPlain): the partial sums go to p.slab, and the
// caller's reduction applies the epilogue.
int launch_one(const Problem& p, int tile, int epi, int across, bool fp32, hipStream_t st);
int launch_split(const Problem& p, int tile, int pa, int pb, int epi, int across, bool fp32, hipStream_t st);

// a dispatch counts its work items of a dimension in 32 bits
inline bool grid_ok(int64_t blocks, int64_t threads) { return blocks <= (int64_t)UINT32_MAX / threads; }

template <typename C, int EPI, int ACROSS, typename T>
int launch_config(const Problem& p, hipStream_t st) {
  constexpr int TC = C::TN / (EPI == kGated || EPI == kGatedGrad ? 2 : 1);
  // the backward epilogues write the padding behind column N too
  const int64_t tm = cdiv(p.M, C::TM), tn = cdiv(EPI == kDenseGrad || EPI == kGatedGrad ? p.np : p.N, TC);
  if (!grid_ok(tm * tn, C::kThreads)) return AIMX_EARG;
  hipLaunchKernelGGL((k_dense<C, EPI, ACROSS, T>), dim3((unsigned)(tm * tn), (unsigned)p.splits), dim3(C::kThreads), 0,
                     st, p, (int)tm, (int)tn);
  AIMX_CHECK_LAUNCH();
  return AIMX_OK;
}

// the operand orders that occur with each epilogue
template <typename C, typename T>
int launch_epi(const Problem& p, int epi, int across, hipStream_t st) {
  if (p.splits > 1) {
    if (across == kNone) return launch_config<C, kSlab, kNone, float>(p, st);
    return across == kB ? launch_config<C, kSlab, kB, float>(p, st) : launch_config<C, kSlab, kBoth, float>(p, st);
  }
  switch (epi) {
    case kGated: return launch_config<C, kGated, kNone, T>(p, st);
    case kDenseGrad: return launch_config<C, kDenseGrad, kNone, T>(p, st);
    case kGatedGrad: return launch_config<C, kGatedGrad, kNone, T>(p, st);
    default: break;
  }
  if (across == kNone) return launch_config<C, kPlain, kNone, T>(p, st);
  return across == kB ? launch_config<C, kPlain, kB, T>(p, st) : launch_config<C, kPlain, kBoth, T>(p, st);
}

}  // namespace dense
}  // namespace aimx
