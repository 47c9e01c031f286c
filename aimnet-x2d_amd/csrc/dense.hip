// Dense and gated products with their gradients (aimx_dense_*, include/aimx.h).
//
//   halves 1:  p = x W^T + b            y = act(p) + res
//   halves 2:  g = x Wg^T + bg, u = x Wu^T + bu    y = act(g) * u
// Backward, from dy and the fp32 pre-activations (kept by the forward, or computed again from x or from the
// 8-bit form of x):
//   dP = dy act'(p)    |    dG = dy u act'(g), dU = dy act(g)
//   dx = dP W          |    dx = dG Wg + dU Wu, one product over both halves' columns
//   dW = dP^T x, db = column sums of dP (fp32, before dP is rounded)
// Every product is D[m][n] = sum_k A[m][k] B[n][k] (dense_core.h); the operands whose rows run along the
// wrong axis are transposed while they are staged: the kernels below also pad, split fp32 into planes and
// unpack 8-bit values, in the one pass over them that this needs.
//
// Roundings to fewer bits: y, dx, dW and db once, to the tensors' type. bf16 tensors: dP / dG / dU are
// rounded to bf16 for the matrix instructions (their sums for db are not); with the result's own rounding
// that makes sqrt(2) of the error of rounding the result alone. fp32 tensors: none.
#include "dense_core.h"

namespace aimx {
namespace dense {
namespace {

inline int64_t up64(int64_t v) { return (v + 63) / 64 * 64; }

// --------------------------------------------------------------------------------------------
// Staging
// --------------------------------------------------------------------------------------------
enum Src : int { kF32 = 0, kBf16 = 1, kQ8 = 2 };

struct Segment {
  const void* src;    // [R][C], ld
  const int8_t* exp;  // kQ8: [R][cdiv(C, 32)]
  int64_t ld, R, C;
  uint16_t* dst;
  int64_t ldd, plane;
  int64_t first;  // first work item of this segment
};
struct Segments {
  Segment s[3];
  int32_t n;
  int64_t items;
};

template <int SRC>
__device__ __forceinline__ float source(const Segment& s, int64_t r, int64_t c) {
  if constexpr (SRC == kF32) return ((const float*)s.src)[r * s.ld + c];
  if constexpr (SRC == kBf16) return from_bf16(((const uint16_t*)s.src)[r * s.ld + c]);
  const int e = s.exp[r * ((s.C + 31) / 32) + c / 32];
  return e == 127 ? __uint_as_float(0x7fc00000u) : ldexpf((float)((const int8_t*)s.src)[r * s.ld + c], e);
}

template <int PL>
__device__ __forceinline__ void store_planes8(uint16_t* dst, int64_t plane, const float (&v)[8]) {
  typedef uint16_t u16x8 __attribute__((ext_vector_type(8)));
  u16x8 o[PL];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if constexpr (PL == 1) {
      o[0][i] = to_bf16(v[i]);
    } else {
      uint16_t p[3];
      split3(v[i], p);
#pragma unroll
      for (int q = 0; q < 3; ++q) o[q][i] = p[q];
    }
  }
#pragma unroll
  for (int q = 0; q < PL; ++q) *reinterpret_cast<u16x8*>(dst + q * plane) = o[q];
}

__device__ __forceinline__ const Segment& segment_of(const Segments& a, int64_t item) {
  int k = 0;
  while (k + 1 < a.n && a.s[k + 1].first <= item) ++k;
  return a.s[k];
}

// Rows as they are: planes [PL][R][ldd], zeros behind column C. An item is 8 columns of a row.
template <int SRC, int PL>
__global__ __launch_bounds__(256) void k_stage(const Segments a) {
  for (int64_t item = blockIdx.x * (int64_t)256 + threadIdx.x; item < a.items; item += (int64_t)gridDim.x * 256) {
    const Segment& s = segment_of(a, item);
    const int64_t w = s.ldd / 8, i = item - s.first, r = i / w, c = (i - r * w) * 8;
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = c + e < s.C ? source<SRC>(s, r, c + e) : 0.f;
    store_planes8<PL>(s.dst + r * s.ldd + c, s.plane, v);
  }
}

// Transposed: dst[c][r], planes of [C][ldd], zeros for R <= r < up64(R). An item is a 64 x 64 tile.
template <int SRC, int PL>
__global__ __launch_bounds__(256) void k_stage_t(const Segments a) {
  __shared__ float tile[64][65];
  const Segment& s = segment_of(a, blockIdx.x);
  const int64_t tc = (s.C + 63) / 64, i = blockIdx.x - s.first, r0 = i / tc * 64, c0 = (i - i / tc * tc) * 64;
  {
    const int c = threadIdx.x & 63, r = threadIdx.x >> 6;
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const int64_t rr = r0 + r + 4 * j, cc = c0 + c;
      tile[r + 4 * j][c] = rr < s.R && cc < s.C ? source<SRC>(s, rr, cc) : 0.f;
    }
  }
  __syncthreads();
  const int r8 = (threadIdx.x & 7) * 8;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int c = (threadIdx.x >> 3) + 32 * j;
    if (c0 + c >= s.C) continue;
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = tile[r8 + e][c];
    store_planes8<PL>(s.dst + (c0 + c) * s.ldd + r0 + r8, s.plane, v);
  }
}

// The gradient before the activation: rows [PL][M][halves * Np] (the first operand of dx), transposed
// [PL][halves * N][Mp] (the first operand of dW) and each 64-row tile's column sums, whichever is asked for.
struct Dpre {
  const void* dy;
  int64_t ldd, M, N, Np, Mp;
  const float* pre;  // [M][halves * N]; nullptr: no activation
  uint16_t* rows;
  uint16_t* cols;
  int64_t rows_plane, cols_plane;
  float* sums;  // [cdiv(M, 64)][halves * N]
  int32_t act;
};
template <typename T, int PL, int HALVES>
__global__ __launch_bounds__(256) void k_dpre(const Dpre a) {
  __shared__ float tile[HALVES][64][65];
  __shared__ float part[HALVES][4][64];
  const int64_t tn = a.Np / 64, tm = blockIdx.x / tn, m0 = tm * 64, n0 = (blockIdx.x - tm * tn) * 64;
  {
    const int c = threadIdx.x & 63, r = threadIdx.x >> 6;
    const int64_t n = n0 + c;
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const int64_t m = m0 + r + 4 * j;
      const bool ok = m < a.M && n < a.N;
      float d = ok ? load1((const T*)a.dy + m * a.ldd + n) : 0.f;
      if constexpr (HALVES == 2) {
        float dg = 0.f, du = 0.f;
        if (ok) {
          const float g = a.pre[m * 2 * a.N + n], u = a.pre[m * 2 * a.N + a.N + n];
          dg = d * u * act_grad(a.act, g);
          du = d * act_fwd(a.act, g);
        }
        tile[0][r + 4 * j][c] = dg;
        tile[1][r + 4 * j][c] = du;
      } else {
        if (ok && a.pre) d *= act_grad(a.act, a.pre[m * a.N + n]);
        tile[0][r + 4 * j][c] = d;
      }
    }
  }
  __syncthreads();
  const int e8 = (threadIdx.x & 7) * 8;
#pragma unroll
  for (int h = 0; h < HALVES; ++h) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int t = (threadIdx.x >> 3) + 32 * j;
      float v[8];
      if (a.rows && m0 + t < a.M) {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = tile[h][t][e8 + e];
        store_planes8<PL>(a.rows + (m0 + t) * HALVES * a.Np + h * a.Np + n0 + e8, a.rows_plane, v);
      }
      if (a.cols && n0 + t < a.N) {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = tile[h][e8 + e][t];
        store_planes8<PL>(a.cols + (h * a.N + n0 + t) * a.Mp + m0 + e8, a.cols_plane, v);
      }
    }
    if (a.sums) {
      const int c = threadIdx.x & 63, w = threadIdx.x >> 6;
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < 16; ++i) s += tile[h][w * 16 + i][c];
      part[h][w][c] = s;
    }
  }
  if (!a.sums) return;
  __syncthreads();
  if (threadIdx.x < 64 * HALVES) {
    const int h = threadIdx.x >> 6, c = threadIdx.x & 63;
    if (n0 + c < a.N)
      a.sums[tm * HALVES * a.N + h * a.N + n0 + c] = (part[h][0][c] + part[h][1][c]) + (part[h][2][c] + part[h][3][c]);
  }
}

// db: the tiles' column sums, 16 interleaved runs per column added in a fixed order
template <typename T>
__global__ __launch_bounds__(1024) void k_column_sums(const float* __restrict__ sums, int64_t tiles, int64_t N,
                                                      int32_t halves, T* __restrict__ d0, T* __restrict__ d1) {
  __shared__ float part[16][64];
  const int c = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int64_t total = N * halves, n = blockIdx.x * (int64_t)64 + c;
  float s = 0.f;
  if (n < total)
    for (int64_t t = w; t < tiles; t += 16) s += sums[t * total + n];
  part[w][c] = s;
  __syncthreads();
  if (w == 0 && n < total) {
    float v = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) v += part[i][c];
    T* d = n < N ? d0 + n : d1 + (n - N);
    if constexpr (sizeof(T) == 4) *d = v;
    else *d = to_bf16(v);
  }
}

// The partial sums of a split product in slab order, then the plain epilogue. 4 columns an item.
template <typename T>
__global__ __launch_bounds__(256) void k_reduce_slabs(const Problem p) {
  const int64_t w = (p.N + 3) / 4, items = p.M * w;
  for (int64_t it = blockIdx.x * (int64_t)256 + threadIdx.x; it < items; it += (int64_t)gridDim.x * 256) {
    const int64_t m = it / w, n = (it - m * w) * 4, left = p.N - n;
    const bool v4 = p.vec && left >= 4;
    floatx4 v = {0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < p.splits; ++s) v += load4(p.slab + ((int64_t)s * p.M + m) * p.N + n, v4, left);
    if (p.bias) v += load4((const T*)p.bias + n, v4, left);
    if (p.pre) store4(p.pre + m * p.N + n, v, v4, left);
    if (!p.y) continue;
    if (p.act >= 0) {
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = act_fwd(p.act, v[e]);
    }
    if (p.res) v += load4((const T*)p.res + m * p.ldr + n, v4, left);
    T* y = m < p.y_rows ? (T*)p.y + m * p.ldy : (T*)p.y2 + (m - p.y_rows) * p.ldy;
    store4(y + n, v, v4, left);
  }
}

// --------------------------------------------------------------------------------------------
// Host
// --------------------------------------------------------------------------------------------
// A workspace handed out in 256-byte steps; with no base it only counts.
struct Carve {
  char* base;
  size_t used = 0;
  template <typename P>
  P* take(int64_t n) {
    P* p = base ? (P*)(base + used) : nullptr;
    used += ((size_t)n * sizeof(P) + 255) & ~(size_t)255;
    return p;
  }
};

inline bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

struct Ctx {
  hipStream_t st;
  bool dry;  // count the workspace, launch nothing
  int rc = AIMX_OK;
};

template <int SRC, int PL>
void stage_go(Ctx& c, Segments& a, bool transpose) {
  if (a.items == 0) return;
  if (transpose)
    hipLaunchKernelGGL((k_stage_t<SRC, PL>), dim3((unsigned)a.items), dim3(256), 0, c.st, a);
  else
    hipLaunchKernelGGL((k_stage<SRC, PL>), dim3((unsigned)std::min<int64_t>(cdiv(a.items, 256), 16384)), dim3(256), 0,
                       c.st, a);
  c.rc = (int)hipGetLastError();
}

// Launches a list of segments of one kind of source.
void stage(Ctx& c, Segments& a, int src, int planes, bool transpose) {
  if (c.dry || c.rc || a.n == 0) return;
  a.items = 0;
  for (int i = 0; i < a.n; ++i) {
    a.s[i].first = a.items;
    a.items += transpose ? cdiv(a.s[i].R, 64) * cdiv(a.s[i].C, 64) : a.s[i].R * (a.s[i].ldd / 8);
  }
  if (transpose && a.items > INT32_MAX) {
    c.rc = AIMX_EARG;
    return;
  }
  if (src == kF32) return planes == 3 ? stage_go<kF32, 3>(c, a, transpose) : stage_go<kF32, 1>(c, a, transpose);
  if (src == kBf16) return stage_go<kBf16, 1>(c, a, transpose);
  return stage_go<kQ8, 1>(c, a, transpose);
}

void product(Ctx& c, Carve& ws, Problem p, int pa, int pb, int halves, bool fp32, bool may_split) {
  if (p.M == 0) return;
  const bool one = pa == 1 && pb == 1;
  const Plan t = one ? plan_one(p.M, p.N * halves, p.K, may_split) : plan_split(p.M, p.N * halves, p.K, may_split);
  p.splits = t.splits;
  if (t.splits > 1) p.slab = ws.take<float>((int64_t)t.splits * p.M * p.N);
  if (c.dry || c.rc) return;
  // 8- and 16-byte accesses of 4 columns: every row of every tensor starts at a multiple of 4 elements
  const size_t b = fp32 ? 4 : 2;
  auto four = [&](const void* q, int64_t ld) { return !q || (((uintptr_t)q % (4 * b)) == 0 && ld % 4 == 0); };
  p.vec = p.N % 4 == 0 && four(p.y, p.ldy) && four(p.y2, p.ldy) && four(p.res, p.ldr) && four(p.bias, 0) &&
          four(p.bias2, 0) && aligned16(p.pre);
  if (p.y_rows == 0) p.y_rows = p.M;
  c.rc = one ? launch_one(p, t.tile, halves, fp32, c.st) : launch_split(p, t.tile, pa, pb, halves, c.st);
  if (c.rc || t.splits == 1) return;
  const dim3 grid((unsigned)std::min<int64_t>(cdiv(p.M * cdiv(p.N, 4), 256), 16384));
  if (fp32) hipLaunchKernelGGL(k_reduce_slabs<float>, grid, dim3(256), 0, c.st, p);
  else hipLaunchKernelGGL(k_reduce_slabs<uint16_t>, grid, dim3(256), 0, c.st, p);
  c.rc = (int)hipGetLastError();
}

bool valid(const AimxDense* d) {
  if (!d || d->M < 0 || d->N < 1 || d->K < 1 || (d->halves != 1 && d->halves != 2)) return false;
  if (d->dtype != AIMX_DTYPE_F32 && d->dtype != AIMX_DTYPE_BF16) return false;
  if (d->act < AIMX_ACT_NONE || d->act > AIMX_ACT_SILU) return false;
  if (d->precision != AIMX_PREC_FP32 && d->precision != AIMX_PREC_BF16) return false;
  if (!d->w[0] || (d->halves == 2 && (!d->w[1] || d->act < 0)) || d->ldw < d->K) return false;
  if (d->x && d->ldx < d->K) return false;
  if (d->res && (d->halves == 2 || d->ldr < d->N)) return false;
  // offsets inside a tile's rows are 32 bits wide
  const int64_t most = (int64_t)1 << 21;
  return d->M <= (int64_t)1 << 40 && d->N <= most && d->K <= most && d->ldx <= most && d->ldw <= most;
}

struct Kind {
  bool fp32;
  int planes, src;
  size_t bytes;
};
Kind kind_of(const AimxDense* d) {
  const bool f = d->dtype == AIMX_DTYPE_F32;
  return {f, f && d->precision == AIMX_PREC_FP32 ? 3 : 1, f ? kF32 : kBf16, f ? (size_t)4 : (size_t)2};
}

// a bf16 matrix the products can read where it is
bool in_place(const Kind& k, const void* p, int64_t ld, int64_t cols) {
  return !k.fp32 && aligned16(p) && ld % 8 == 0 && cols % 64 == 0;
}

Segment& add(Segments& a, const void* src, int64_t ld, int64_t R, int64_t C, uint16_t* dst, int64_t ldd, int64_t plane) {
  Segment& s = a.s[a.n++];
  s = Segment{src, nullptr, ld, R, C, dst, ldd, plane, 0};
  return s;
}

// x W^T with the forward's epilogue. From the 8-bit form of x where d->x is null. w_only: y is not
// written, only pre.
void forward(Ctx& c, Carve& ws, const AimxDense* d, float* pre, bool pre_only) {
  const Kind k = kind_of(d);
  const int64_t Kp = up64(d->K);
  Problem p{};
  p.M = d->M;
  p.N = d->N;
  p.K = Kp;
  p.act = d->act;
  p.pre = pre;
  if (!pre_only) {
    p.y = d->y;
    p.ldy = d->ldy;
    p.res = d->res;
    p.ldr = d->ldr;
  }
  p.bias = d->b[0];
  p.bias2 = d->b[1];
  Segments same{}, eight{};
  int pa = k.planes;
  p.a = Operand{(const uint16_t*)d->x, nullptr, d->ldx, 0, d->M};
  if (!d->x) {
    pa = 1;
    uint16_t* t = ws.take<uint16_t>(d->M * Kp);
    p.a = Operand{t, nullptr, Kp, 0, d->M};
    add(eight, d->q, (d->K + 31) / 32 * 32, d->M, d->K, t, Kp, 0).exp = d->qexp;
  } else if (!in_place(k, d->x, d->ldx, d->K)) {
    const int64_t plane = d->M * Kp;
    uint16_t* t = ws.take<uint16_t>(plane * k.planes);
    p.a = Operand{t, nullptr, Kp, plane, d->M};
    add(same, d->x, d->ldx, d->M, d->K, t, Kp, plane);
  }
  p.b = Operand{(const uint16_t*)d->w[0], (const uint16_t*)d->w[1], d->ldw, 0, d->N};
  if (!in_place(k, d->w[0], d->ldw, d->K) || (d->halves == 2 && !aligned16(d->w[1]))) {
    const int64_t plane = d->N * Kp;
    uint16_t* t[2] = {nullptr, nullptr};
    for (int h = 0; h < d->halves; ++h) {
      t[h] = ws.take<uint16_t>(plane * k.planes);
      add(same, d->w[h], d->ldw, d->N, d->K, t[h], Kp, plane);
    }
    p.b = Operand{t[0], t[1], Kp, plane, d->N};
  }
  stage(c, same, k.src, k.planes, false);
  stage(c, eight, kQ8, 1, false);
  product(c, ws, p, pa, k.planes, d->halves, k.fp32, d->halves == 1);
}

template <typename T, int PL>
void dpre_go(Ctx& c, const Dpre& a, int halves) {
  const dim3 grid((unsigned)(a.Np / 64 * cdiv(a.M, 64)));
  if (halves == 2) hipLaunchKernelGGL((k_dpre<T, PL, 2>), grid, dim3(256), 0, c.st, a);
  else hipLaunchKernelGGL((k_dpre<T, PL, 1>), grid, dim3(256), 0, c.st, a);
  c.rc = (int)hipGetLastError();
}

void backward(Ctx& c, Carve& ws, const AimxDense* d, const AimxDenseGrad* g) {
  const Kind k = kind_of(d);
  const int64_t M = d->M, N = d->N, K = d->K, H = d->halves, Np = up64(N), Mp = up64(M);
  const bool has_dw = g->dw[0] != nullptr, has_db = g->db[0] != nullptr, has_dx = g->dx != nullptr;
  const float* pre = d->pre;
  if (d->act >= 0 && !pre) {
    float* t = ws.take<float>(M * H * N);
    forward(c, ws, d, t, true);
    pre = t;
  }
  Dpre a{};
  a.dy = g->dy;
  a.ldd = g->ldd;
  a.M = M;
  a.N = N;
  a.Np = Np;
  a.Mp = Mp;
  a.act = d->act;
  a.pre = d->act >= 0 ? pre : nullptr;
  Operand rows{};
  if (has_dx) {
    if (d->act < 0 && in_place(k, g->dy, g->ldd, N)) {
      rows = Operand{(const uint16_t*)g->dy, nullptr, g->ldd, 0, M};
    } else {
      a.rows_plane = M * H * Np;
      a.rows = ws.take<uint16_t>(a.rows_plane * k.planes);
      rows = Operand{a.rows, nullptr, H * Np, a.rows_plane, M};
    }
  }
  if (has_dw) {
    a.cols_plane = H * N * Mp;
    a.cols = ws.take<uint16_t>(a.cols_plane * k.planes);
  }
  if (has_db) a.sums = ws.take<float>(cdiv(M, 64) * H * N);
  if (!c.dry && !c.rc && M > 0 && (a.rows || a.cols || a.sums)) {
    if (Np / 64 * cdiv(M, 64) > INT32_MAX) c.rc = AIMX_EARG;
    else if (!k.fp32) dpre_go<uint16_t, 1>(c, a, (int)H);
    else if (k.planes == 3) dpre_go<float, 3>(c, a, (int)H);
    else dpre_go<float, 1>(c, a, (int)H);
  }
  if (has_db && !c.dry && !c.rc) {
    const dim3 grid((unsigned)cdiv(H * N, 64));
    if (k.fp32)
      hipLaunchKernelGGL(k_column_sums<float>, grid, dim3(1024), 0, c.st, a.sums, cdiv(M, 64), N, (int)H,
                         (float*)g->db[0], (float*)g->db[1]);
    else
      hipLaunchKernelGGL(k_column_sums<uint16_t>, grid, dim3(1024), 0, c.st, a.sums, cdiv(M, 64), N, (int)H,
                         (uint16_t*)g->db[0], (uint16_t*)g->db[1]);
    c.rc = (int)hipGetLastError();
  }
  // the transposed x (or its 8-bit form) and weights
  Segments same{}, eight{};
  uint16_t *xt = nullptr, *wt = nullptr;
  const int64_t xplane = K * Mp, wplane = K * H * Np;
  const int px = d->x ? k.planes : 1;
  if (has_dw) {
    xt = ws.take<uint16_t>(xplane * px);
    if (d->x) add(same, d->x, d->ldx, M, K, xt, Mp, xplane);
    else add(eight, d->q, (K + 31) / 32 * 32, M, K, xt, Mp, 0).exp = d->qexp;
  }
  if (has_dx) {
    wt = ws.take<uint16_t>(wplane * k.planes);
    for (int h = 0; h < H; ++h) add(same, d->w[h], d->ldw, N, K, wt ? wt + h * Np : nullptr, H * Np, wplane);
  }
  stage(c, same, k.src, k.planes, true);
  stage(c, eight, kQ8, 1, true);
  if (has_dx) {
    Problem p{};
    p.a = rows;
    p.b = Operand{wt, nullptr, H * Np, wplane, K};
    p.M = M;
    p.N = K;
    p.K = H * Np;
    p.y = g->dx;
    p.ldy = g->lddx;
    p.act = AIMX_ACT_NONE;
    product(c, ws, p, k.planes, k.planes, 1, k.fp32, true);
  }
  if (has_dw) {
    Problem p{};
    p.a = Operand{a.cols, nullptr, Mp, a.cols_plane, H * N};
    p.b = Operand{xt, nullptr, Mp, xplane, K};
    p.M = H * N;
    p.N = K;
    p.K = Mp;
    p.y = g->dw[0];
    p.y2 = g->dw[1];
    p.ldy = K;
    p.y_rows = N;
    p.act = AIMX_ACT_NONE;
    product(c, ws, p, k.planes, px, 1, k.fp32, true);
  }
}

bool valid_grad(const AimxDense* d, const AimxDenseGrad* g) {
  if (!valid(d) || !g) return false;
  const bool second = d->halves == 2;
  if (second && ((g->dw[0] != nullptr) != (g->dw[1] != nullptr) || (g->db[0] != nullptr) != (g->db[1] != nullptr)))
    return false;
  if ((d->M > 0 && !g->dy) || g->ldd < d->N || (g->dx && g->lddx < d->K) || g->ldd > (int64_t)1 << 21) return false;
  if (d->M > (int64_t)1 << 22) return false;  // the transposed operands' rows run along M
  return d->M == 0 || d->x || (d->q && d->qexp);
}

}  // namespace
}  // namespace dense
}  // namespace aimx

using namespace aimx;

extern "C" size_t aimx_dense_workspace_bytes(const AimxDense* d) {
  if (!dense::valid(d)) return 0;
  dense::Ctx c{nullptr, true};
  dense::Carve ws{nullptr};
  dense::forward(c, ws, d, d->pre, false);
  return ws.used;
}

extern "C" int aimx_dense_forward(const AimxDense* d, aimx_stream_t stream) {
  if (!dense::valid(d) || (d->M > 0 && (!d->x || !d->y)) || d->ldy < d->N) return AIMX_EARG;
  if (d->M == 0) return AIMX_OK;
  if (d->workspace_bytes < aimx_dense_workspace_bytes(d) || (d->workspace_bytes && !d->workspace)) return AIMX_EARG;
  if (!dense::aligned16(d->workspace)) return AIMX_EARG;
  dense::Ctx c{(hipStream_t)stream, false};
  dense::Carve ws{(char*)d->workspace};
  dense::forward(c, ws, d, d->pre, false);
  return c.rc;
}

extern "C" size_t aimx_dense_backward_workspace_bytes(const AimxDense* d, const AimxDenseGrad* g) {
  if (!dense::valid_grad(d, g)) return 0;
  dense::Ctx c{nullptr, true};
  dense::Carve ws{nullptr};
  dense::backward(c, ws, d, g);
  return ws.used;
}

extern "C" int aimx_dense_backward(const AimxDense* d, const AimxDenseGrad* g, aimx_stream_t stream) {
  if (!dense::valid_grad(d, g)) return AIMX_EARG;
  const size_t need = aimx_dense_backward_workspace_bytes(d, g);
  if (g->workspace_bytes < need || (need && !g->workspace) || !dense::aligned16(g->workspace)) return AIMX_EARG;
  dense::Ctx c{(hipStream_t)stream, false};
  dense::Carve ws{(char*)g->workspace};
  dense::backward(c, ws, d, g);
  return c.rc;
}
