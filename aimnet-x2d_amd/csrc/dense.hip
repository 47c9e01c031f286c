// Dense and gated products with their gradients (aimx_dense_*, include/aimx.h).
//
//   halves 1:  p = x W^T + b            y = act(p) + res
//   halves 2:  g = x Wg^T + bg, u = x Wu^T + bu    y = act(g) * u
// Backward, from dy and the fp32 pre-activations (kept by the forward, or computed again from x or from the
// 8-bit form of x):
//   dP = dy act'(p)    |    dG = dy u act'(g), dU = dy act(g)
//   dx = dP W          |    dx = dG Wg + dU Wu, one product over both halves' columns
//   dW = dP^T x, db = column sums of dP (fp32, before dP is rounded)
// Every product is D[m][n] = sum_k A[m][k] B[n][k] (dense_core.h), dx and dW with operands read across their rows.
// bf16 tensors: the backward does not read kept pre-activations, it runs the forward product again with an epilogue
// that leaves dP / [dG | dU]: at 20480 x 512 -> 2 x 2048 that is 86 GF, where fp32 values before the activation
// would be 335 MB written and read again. fp32 tensors keep them: their product costs six times as much.
//
// Roundings to fewer bits: y, dx, dW and db once, to the tensors' type. bf16 tensors: dP / dG / dU are
// rounded to bf16 for the matrix instructions (their sums for db are not), unless they are few; with the result's
// own rounding that makes sqrt(2) of the error of rounding the result alone. fp32 tensors: none.
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

typedef int8_t i8x8 __attribute__((ext_vector_type(8)));

template <int PL>
__device__ __forceinline__ void store_planes8(uint16_t* dst, int64_t plane, const float (&v)[8]) {
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

// Planes [PL][R][ldd], zeros behind column C. An item is 8 columns of a row.
template <int SRC, int PL>
__global__ __launch_bounds__(256) void k_stage(const Segments a) {
  for (int64_t item = blockIdx.x * (int64_t)256 + threadIdx.x; item < a.items; item += (int64_t)gridDim.x * 256) {
    int k = 0;
    while (k + 1 < a.n && a.s[k + 1].first <= item) ++k;
    const Segment& s = a.s[k];
    const int64_t w = s.ldd / 8, i = item - s.first, r = i / w, c = (i - r * w) * 8;
    float v[8];
    if constexpr (SRC == kQ8) {
      const int e = c < s.C ? s.exp[r * ((s.C + 31) / 32) + c / 32] : 0;
      i8x8 q = {};
      if (c < s.C) q = *reinterpret_cast<const i8x8*>((const int8_t*)s.src + r * s.ld + c);
#pragma unroll
      for (int j = 0; j < 8; ++j)
        v[j] = c + j < s.C ? (e == 127 ? __uint_as_float(0x7fc00000u) : ldexpf((float)q[j], e)) : 0.f;
    } else if constexpr (SRC == kF32) {
      load8((const float*)s.src + r * s.ld + c, s.C - c, v);
    } else {
      load8((const uint16_t*)s.src + r * s.ld + c, s.C - c, v);
    }
    store_planes8<PL>(s.dst + r * s.ldd + c, s.plane, v);
  }
}

// The gradient before the activation from kept values, or dy itself: planes [PL][M][halves * Np] with zeros behind
// column N (nullptr: not wanted), and the column sums of each 128 rows (nullable).
struct Dpre {
  const void* dy;
  int64_t ldd, M, N, Np, N8;
  const float* pre;  // [M][halves][N8]; nullptr: no activation
  uint16_t* rows;
  int64_t plane;
  float* sums;  // [cdiv(M, 128)][halves * N]
  int32_t act;
};
constexpr int kDpreRows = 128;
template <typename T, int PL, int HALVES>
__global__ __launch_bounds__(256) void k_dpre(const Dpre a) {
  __shared__ float part[HALVES][32][65];
  const int64_t tn = a.Np / 64, tm = blockIdx.x / tn;
  const int c8 = (threadIdx.x & 7) * 8, r = threadIdx.x >> 3;
  const int64_t n = (blockIdx.x - tm * tn) * 64 + c8;
  float total[HALVES][8] = {};
#pragma unroll
  for (int j = 0; j < kDpreRows / 32; ++j) {
    const int64_t m = tm * kDpreRows + j * 32 + r;
    if (m >= a.M) continue;
    float d[8], g[8], u[8], o[8];
    load8((const T*)a.dy + m * a.ldd + n, a.N - n, d);
    if (a.pre && n < a.N8) {
      load8(a.pre + m * HALVES * a.N8 + n, 8, g);
      if constexpr (HALVES == 2) load8(a.pre + m * HALVES * a.N8 + a.N8 + n, 8, u);
    }
#pragma unroll
    for (int h = 0; h < HALVES; ++h) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        o[e] = d[e];
        if (n + e >= a.N) continue;  // behind N: d is zero, pre undefined
        if constexpr (HALVES == 2) o[e] = h == 0 ? d[e] * u[e] * act_grad(a.act, g[e]) : d[e] * act_fwd(a.act, g[e]);
        else if (a.pre) o[e] = d[e] * act_grad(a.act, g[e]);
        total[h][e] += o[e];
      }
      if (a.rows) store_planes8<PL>(a.rows + m * HALVES * a.Np + h * a.Np + n, a.plane, o);
    }
  }
  if (!a.sums) return;
#pragma unroll
  for (int h = 0; h < HALVES; ++h)
#pragma unroll
    for (int e = 0; e < 8; ++e) part[h][r][c8 + e] = total[h][e];
  __syncthreads();
  if (threadIdx.x < 64 * HALVES) {
    const int h = threadIdx.x >> 6, c = threadIdx.x & 63;
    const int64_t col = (blockIdx.x - tm * tn) * 64 + c;
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < 32; ++i) s += part[h][i][c];
    if (col < a.N) a.sums[tm * HALVES * a.N + h * a.N + col] = s;
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
    floatx4 v = {0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < p.splits; ++s) v += load4(p.slab + ((int64_t)s * p.M + m) * p.N + n, left);
    if (p.bias) v += load4((const T*)p.bias + n, left);
    if (p.pre) *reinterpret_cast<floatx4*>(p.pre + m * p.n8 + n) = v;
    if (p.act >= 0) {
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = act_fwd(p.act, v[e]);
    }
    if (p.res) v += load4((const T*)p.res + m * p.ldr + n, left);
    const int64_t r = m < p.y_rows ? m : m - p.y_rows;
    if (r < p.y_valid) store4((T*)(m < p.y_rows ? p.y : p.y2) + r * p.ldy + n, v, left);
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
void stage_go(Ctx& c, const Segments& a) {
  hipLaunchKernelGGL((k_stage<SRC, PL>), dim3((unsigned)std::min<int64_t>(cdiv(a.items, 256), 16384)), dim3(256), 0,
                     c.st, a);
  c.rc = (int)hipGetLastError();
}

// Launches a list of segments of one kind of source.
void stage(Ctx& c, Segments& a, int src, int planes) {
  if (c.dry || c.rc || a.n == 0) return;
  a.items = 0;
  for (int i = 0; i < a.n; ++i) {
    a.s[i].first = a.items;
    a.items += a.s[i].R * (a.s[i].ldd / 8);
  }
  if (a.items == 0) return;
  if (src == kF32) return planes == 3 ? stage_go<kF32, 3>(c, a) : stage_go<kF32, 1>(c, a);
  if (src == kBf16) return stage_go<kBf16, 1>(c, a);
  return stage_go<kQ8, 1>(c, a);
}

// One product and, where its k is split, the sum of its parts.
void product(Ctx& c, Carve& ws, Problem p, int pa, int pb, int epi, int across, bool fp32) {
  if (p.M == 0) return;
  const bool one = pa == 1 && pb == 1;
  const int halves = epi == kGated || epi == kGatedGrad ? 2 : 1;
  const Plan t = one ? plan_one(p.M, p.N * halves, p.K, epi == kPlain) : plan_split(p.M, p.N * halves, p.K, epi == kPlain, fp32);
  p.splits = t.splits;
  if (t.splits > 1) p.slab = ws.take<float>((int64_t)t.splits * p.M * p.N);
  if (c.dry || c.rc) return;
  p.n8 = (p.N + 7) / 8 * 8;
  p.np = up64(p.N);
  if (p.k_half == 0) p.k_half = p.K;
  if (p.y_rows == 0) p.y_rows = p.y_valid = p.M;
  c.rc = one ? launch_one(p, t.tile, epi, across, fp32, c.st) : launch_split(p, t.tile, pa, pb, epi, across, fp32, c.st);
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

// a bf16 matrix the products can read where it is, along its rows (k contiguous) or across them
bool in_place(const Kind& k, const void* p, int64_t ld, int64_t cols, bool along) {
  return !k.fp32 && aligned16(p) && ld % 8 == 0 && cols % (along ? 64 : 8) == 0;
}

void add(Segments& a, const void* src, const int8_t* exp, int64_t ld, int64_t R, int64_t C, uint16_t* dst, int64_t ldd) {
  a.s[a.n++] = Segment{src, exp, ld, R, C, dst, ldd, R * ldd, 0};
}

// x (or its 8-bit form) as an operand; `along` if some product reads it along its rows
Operand operand_x(const AimxDense* d, const Kind& k, Carve& ws, bool along, Segments& same, Segments& eight) {
  if (d->x && in_place(k, d->x, d->ldx, d->K, along)) return {(const uint16_t*)d->x, nullptr, d->ldx, 0, d->M, d->K};
  const int64_t Kp = up64(d->K);
  uint16_t* t = ws.take<uint16_t>(d->M * Kp * (d->x ? k.planes : 1));
  if (d->x) add(same, d->x, nullptr, d->ldx, d->M, d->K, t, Kp);
  else add(eight, d->q, d->qexp, (d->K + 31) / 32 * 32, d->M, d->K, t, Kp);
  return {t, nullptr, Kp, d->M * Kp, d->M, Kp};
}

Operand operand_w(const AimxDense* d, const Kind& k, Carve& ws, bool along, Segments& same) {
  if (in_place(k, d->w[0], d->ldw, d->K, along) && (d->halves == 1 || aligned16(d->w[1])))
    return {(const uint16_t*)d->w[0], (const uint16_t*)d->w[1], d->ldw, 0, d->N, d->K};
  const int64_t Kp = up64(d->K);
  uint16_t* t[2] = {nullptr, nullptr};
  for (int h = 0; h < d->halves; ++h) {
    t[h] = ws.take<uint16_t>(d->N * Kp * k.planes);
    add(same, d->w[h], nullptr, d->ldw, d->N, d->K, t[h], Kp);
  }
  return {t[0], t[1], Kp, d->N * Kp, d->N, Kp};
}

// the forward product's problem
Problem forward_problem(const AimxDense* d, const Operand& x, const Operand& w) {
  Problem p{};
  p.a = x;
  p.b = w;
  p.M = d->M;
  p.N = d->N;
  p.K = up64(d->K);
  p.act = d->act;
  p.bias = d->b[0];
  p.bias2 = d->b[1];
  return p;
}

void forward(Ctx& c, Carve& ws, const AimxDense* d) {
  const Kind k = kind_of(d);
  Segments same{}, none{};
  const Operand x = operand_x(d, k, ws, true, same, none), w = operand_w(d, k, ws, true, same);
  stage(c, same, k.src, k.planes);
  Problem p = forward_problem(d, x, w);
  p.y = d->y;
  p.ldy = d->ldy;
  p.res = d->res;
  p.ldr = d->ldr;
  p.pre = d->pre;
  product(c, ws, p, k.planes, k.planes, d->halves == 2 ? kGated : kPlain, kNone, k.fp32);
}

template <typename T, int PL>
void dpre_go(Ctx& c, const Dpre& a, int halves) {
  const dim3 grid((unsigned)(a.Np / 64 * cdiv(a.M, kDpreRows)));
  if (halves == 2) hipLaunchKernelGGL((k_dpre<T, PL, 2>), grid, dim3(256), 0, c.st, a);
  else hipLaunchKernelGGL((k_dpre<T, PL, 1>), grid, dim3(256), 0, c.st, a);
  c.rc = (int)hipGetLastError();
}

void backward(Ctx& c, Carve& ws, const AimxDense* d, const AimxDenseGrad* g) {
  const Kind k = kind_of(d);
  const int64_t M = d->M, N = d->N, K = d->K, H = d->halves, Np = up64(N);
  const bool has_dw = g->dw[0] != nullptr, has_db = g->db[0] != nullptr, has_dx = g->dx != nullptr;
  const bool again = d->act >= 0 && !d->pre;  // the values before the activation are computed again
  // Rounded to bf16, the gradient before the activation leaves dx and dW at 0.00235 of their norm where rounding the
  // results alone leaves 0.00166, at every size; where it holds few values the error does not average out either (1.5
  // times that of rounding the results at one row of 32). Three planes of it leave 0.00166 and cost 8 to 23 us of a
  // pass up to 65536 values (1 row, 256 -> 2 x 1024: 27 us against 19; 8, 1024 -> 2 x 4096: 56, 46; 500, 256 -> 2 x 64:
  // 42, 19), less than the host takes to enqueue one. At 262144 the kernels are what counts (128, 1024 -> 2 x 1024: 58,
  // 31; 512, 512 -> 512: 44, 25). The forward's values then come as fp32 first.
  const bool fine = !k.fp32 && d->act >= 0 && M * H * N <= 65536;
  const int px = d->x ? k.planes : 1, pd = fine ? 3 : k.planes;
  Segments same{}, eight{};
  Operand x{}, w{}, rows{};
  if (has_dw || again) x = operand_x(d, k, ws, again, same, eight);
  if (has_dx || again) w = operand_w(d, k, ws, again, same);
  stage(c, same, k.src, k.planes);
  stage(c, eight, kQ8, 1);

  // dP / [dG | dU] as an operand and the parts of its column sums
  const int64_t plane = M * H * Np;
  const float* sums = nullptr;
  int64_t parts = 0;
  const float* pre = d->pre;
  if (fine && again) {
    Problem p = forward_problem(d, x, w);
    p.y = ws.take<uint16_t>(M * N);
    p.ldy = N;
    pre = p.pre = ws.take<float>(M * H * ((N + 7) / 8 * 8));
    product(c, ws, p, 1, 1, H == 2 ? kGated : kPlain, kNone, false);
  }
  if (again && !fine) {
    uint16_t* t = ws.take<uint16_t>(plane * k.planes);
    rows = {t, nullptr, H * Np, plane, M, H * Np};
    Problem p = forward_problem(d, x, w);
    p.res = g->dy;
    p.ldr = g->ldd;
    p.rows = t;
    p.rows_plane = plane;
    const Plan at = (px == 1 && k.planes == 1) ? plan_one(M, N * H, p.K, false) : plan_split(M, N * H, p.K, false, k.fp32);
    parts = cdiv(M, at.rows) * kWavesM;
    if (has_db) sums = p.sums = ws.take<float>(parts * H * N);
    product(c, ws, p, px, k.planes, H == 2 ? kGatedGrad : kDenseGrad, kNone, k.fp32);
  } else {
    Dpre a{};
    a.dy = g->dy;
    a.ldd = g->ldd;
    a.M = M;
    a.N = N;
    a.Np = Np;
    a.N8 = (N + 7) / 8 * 8;
    a.pre = d->act >= 0 ? pre : nullptr;
    a.act = d->act;
    if (d->act < 0 && in_place(k, g->dy, g->ldd, N, has_dx)) {
      rows = {(const uint16_t*)g->dy, nullptr, g->ldd, 0, M, N};
    } else if (has_dx || has_dw) {
      a.rows = ws.take<uint16_t>(plane * pd);
      a.plane = plane;
      rows = {a.rows, nullptr, H * Np, plane, M, H * Np};
    }
    parts = cdiv(M, kDpreRows);
    if (has_db) sums = a.sums = ws.take<float>(parts * H * N);
    if (!c.dry && !c.rc && M > 0 && (a.rows || a.sums)) {
      if (!grid_ok(Np / 64 * parts, 256)) c.rc = AIMX_EARG;
      else if (!k.fp32 && fine) dpre_go<uint16_t, 3>(c, a, (int)H);
      else if (!k.fp32) dpre_go<uint16_t, 1>(c, a, (int)H);
      else if (k.planes == 3) dpre_go<float, 3>(c, a, (int)H);
      else dpre_go<float, 1>(c, a, (int)H);
    }
  }
  if (has_db && !c.dry && !c.rc) {
    const dim3 grid((unsigned)cdiv(H * N, 64));
    if (k.fp32)
      hipLaunchKernelGGL(k_column_sums<float>, grid, dim3(1024), 0, c.st, sums, parts, N, (int)H, (float*)g->db[0],
                         (float*)g->db[1]);
    else
      hipLaunchKernelGGL(k_column_sums<uint16_t>, grid, dim3(1024), 0, c.st, sums, parts, N, (int)H,
                         (uint16_t*)g->db[0], (uint16_t*)g->db[1]);
    c.rc = (int)hipGetLastError();
  }
  if (has_dx) {
    Problem p{};
    p.a = rows;
    p.b = w;
    p.M = M;
    p.N = K;
    p.K = H * Np;
    p.k_half = Np;
    p.y = g->dx;
    p.ldy = g->lddx;
    p.act = AIMX_ACT_NONE;
    product(c, ws, p, pd, k.planes, kPlain, kB, k.fp32);
  }
  if (has_dw) {
    Problem p{};
    p.a = rows;
    p.b = x;
    p.M = H == 2 ? H * Np : N;
    p.N = K;
    p.K = up64(M);
    p.y = g->dw[0];
    p.y2 = g->dw[1];
    p.ldy = K;
    p.y_rows = H == 2 ? Np : N;
    p.y_valid = N;
    p.act = AIMX_ACT_NONE;
    product(c, ws, p, pd, px, kPlain, kBoth, k.fp32);
  }
}

bool valid_grad(const AimxDense* d, const AimxDenseGrad* g) {
  if (!valid(d) || !g) return false;
  const bool second = d->halves == 2;
  if (second && ((g->dw[0] != nullptr) != (g->dw[1] != nullptr) || (g->db[0] != nullptr) != (g->db[1] != nullptr)))
    return false;
  if ((d->M > 0 && !g->dy) || g->ldd < d->N || (g->dx && g->lddx < d->K) || g->ldd > (int64_t)1 << 21) return false;
  // The interface's limit, no offset's: dw and db are fp32 sums over the rows, whose error is bounded by M 2^-24 of the
  // magnitudes, a quarter of them here.
  if (d->M > (int64_t)1 << 22) return false;
  if (d->pre && ((uintptr_t)d->pre & 15)) return false;
  if (!d->x) return d->M == 0 || (d->q && d->qexp && ((uintptr_t)d->q & 7) == 0);
  // fp32 products keep the values before the activation where they keep x
  return d->act < 0 || d->pre || kind_of(d).planes == 1;
}

}  // namespace
}  // namespace dense
}  // namespace aimx

using namespace aimx;

extern "C" size_t aimx_dense_workspace_bytes(const AimxDense* d) {
  if (!dense::valid(d)) return 0;
  dense::Ctx c{nullptr, true};
  dense::Carve ws{nullptr};
  dense::forward(c, ws, d);
  return ws.used;
}

extern "C" int aimx_dense_forward(const AimxDense* d, aimx_stream_t stream) {
  if (!dense::valid(d) || (d->M > 0 && (!d->x || !d->y)) || d->ldy < d->N || !dense::aligned16(d->pre)) return AIMX_EARG;
  if (d->M == 0) return AIMX_OK;
  if (d->workspace_bytes < aimx_dense_workspace_bytes(d) || (d->workspace_bytes && !d->workspace)) return AIMX_EARG;
  if (!dense::aligned16(d->workspace)) return AIMX_EARG;
  dense::Ctx c{(hipStream_t)stream, false};
  dense::Carve ws{(char*)d->workspace};
  dense::forward(c, ws, d);
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
