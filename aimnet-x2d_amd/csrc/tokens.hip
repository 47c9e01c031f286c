// Scaled embedding of any table and its gradient by sorted tokens (aimx_token_embedding_*, include/aimx.h).
//
//   forward   out_i = scale * table[index_i]
//   gradient  dtable_v = scale * sum over i with index_i = v of dout_i, in ascending i
//
// The small-table kernels of embed.hip keep every table in LDS; here the table has any size, so the gradient
// sorts the tokens and sums runs of equal ones: a stable radix sort, 8 bits a pass, each wave ranking its own
// consecutive chunk of items (no order between waves is needed, the scanned histogram holds it), then
// segments of the sorted items, one group of lanes each. A run inside a segment is written at once; one that
// crosses segments leaves a partial row per segment, and the segment it begins in adds them in order. So no
// atomics touch a float, the sums are fp32 and the same in every run, and a token with half of all items costs
// no more than its share of segments.
//
// 65536 tokens in a 32000 x 512 bf16 table: the lookup 18 us (67 MB written, 4.4 TB/s with the rows read), the zero fill
// 7.5, the sort's two passes of three launches 31 (latency: 64 workgroups), the runs 18 to 24 (90 MB), their join 10.
// A group of 32 rows a segment: fewer leave more runs to join, more leave too few groups to hide the scattered
// rows' latency (kAhead rows are in flight in each).
#include <algorithm>

#include "dense_core.h"

namespace aimx {
namespace {

using dense::floatx4;

// 16 bytes of a row from p, `left` elements of which exist
template <typename T>
struct Cols {
  static constexpr int kVec = 16 / sizeof(T);
  typedef T vec __attribute__((ext_vector_type(kVec)));
  typedef T vece __attribute__((ext_vector_type(kVec), aligned(sizeof(T))));
  vec v;
  __device__ __forceinline__ void load(const T* p, int64_t left) {
    if (left >= kVec) {
      v = *reinterpret_cast<const vece*>(p);
    } else {
#pragma unroll
      for (int e = 0; e < kVec; ++e) v[e] = e < left ? p[e] : (T)0;
    }
  }
  __device__ __forceinline__ float get(int e) const {
    if constexpr (sizeof(T) == 4) return v[e];
    else return dense::from_bf16(v[e]);
  }
  __device__ __forceinline__ void set(int e, float f) {
    if constexpr (sizeof(T) == 4) v[e] = f;
    else v[e] = dense::to_bf16(f);
  }
  __device__ __forceinline__ void store(T* p, int64_t left) const {
    if (left >= kVec) {
      *reinterpret_cast<vece*>(p) = v;
    } else {
#pragma unroll
      for (int e = 0; e < kVec; ++e)
        if (e < left) p[e] = v[e];
    }
  }
};
template <typename T>
__device__ __forceinline__ void store1(T* p, float f) {
  if constexpr (sizeof(T) == 4) *p = f;
  else *p = dense::to_bf16(f);
}

template <typename T>
__global__ __launch_bounds__(256) void k_token_gather(const int64_t* __restrict__ index, int64_t n,
                                                      const T* __restrict__ table, int64_t V, int64_t D, float scale,
                                                      T* __restrict__ out) {
  constexpr int kVec = Cols<T>::kVec;
  const int64_t w = (D + kVec - 1) / kVec, items = n * w;
  for (int64_t it = blockIdx.x * (int64_t)256 + threadIdx.x; it < items; it += (int64_t)gridDim.x * 256) {
    const int64_t i = it / w, c = (it - i * w) * kVec, v = index[i];
    const bool ok = v >= 0 && v < V;
    Cols<T> a;
    a.load(table + (ok ? v : 0) * D + c, ok ? D - c : 0);
#pragma unroll
    for (int e = 0; e < kVec; ++e) a.set(e, ok ? a.get(e) * scale : 0.f);  // 0 * scale is NaN for an infinite scale
    a.store(out + i * D + c, D - c);
  }
}

// --------------------------------------------------------------------------------------------
// Stable sort of the tokens
// --------------------------------------------------------------------------------------------
constexpr int kSortWaves = 4;
constexpr int kMaxChunks = 1024;

struct Sort {
  const int64_t* index;
  int64_t n, V, pad;
  int64_t chunk, chunks;    // items of a wave, waves
  uint32_t *key[2], *id[2];  // sorted tokens (V: out of range or padding) and their items
  int32_t* hist;            // [256][chunks]
  int32_t* totals;          // [4][256]
};

__device__ __forceinline__ void sort_item(const Sort& s, int pass, int64_t i, uint32_t& key, uint32_t& id) {
  if (pass == 0) {
    const int64_t v = s.index[i];
    key = v >= 0 && v < s.V && v != s.pad ? (uint32_t)v : (uint32_t)s.V;
    id = (uint32_t)i;
  } else {
    key = s.key[(pass - 1) & 1][i];
    id = s.id[(pass - 1) & 1][i];
  }
}

// the gradient's n 16-bit words (a table whose every row may stay unseen) and the sort's totals
__global__ __launch_bounds__(256) void k_token_zero(uint16_t* __restrict__ p, int64_t n, int32_t* __restrict__ totals) {
  if (blockIdx.x == 0)
    for (int i = threadIdx.x; i < 4 * 256; i += 256) totals[i] = 0;
  for (int64_t i = (blockIdx.x * (int64_t)256 + threadIdx.x) * 8; i < n; i += (int64_t)gridDim.x * 256 * 8) {
    if (i + 8 <= n) {
      *reinterpret_cast<floatx4*>(p + i) = floatx4{0.f, 0.f, 0.f, 0.f};
    } else {
      for (int64_t j = i; j < n; ++j) p[j] = 0;
    }
  }
}

__global__ __launch_bounds__(256) void k_token_hist(const Sort s, int pass) {
  __shared__ int32_t cnt[kSortWaves][256];
  const int w = threadIdx.x >> 6, lane = threadIdx.x & 63;
  for (int i = threadIdx.x; i < kSortWaves * 256; i += 256) cnt[i >> 8][i & 255] = 0;
  __syncthreads();
  const int64_t chunk = blockIdx.x * (int64_t)kSortWaves + w;
  if (chunk < s.chunks) {
    const int64_t i0 = chunk * s.chunk, i1 = min(s.n, i0 + s.chunk);
    for (int64_t i = i0 + lane; i < i1; i += 64) {
      uint32_t key, id;
      sort_item(s, pass, i, key, id);
      atomicAdd(&cnt[w][(key >> (8 * pass)) & 255], 1);
    }
  }
  __syncthreads();
  int32_t sum = 0;
#pragma unroll
  for (int j = 0; j < kSortWaves; ++j) {
    const int64_t c = blockIdx.x * (int64_t)kSortWaves + j;
    if (c < s.chunks) s.hist[(int64_t)threadIdx.x * s.chunks + c] = cnt[j][threadIdx.x];
    sum += cnt[j][threadIdx.x];
  }
  if (sum) atomicAdd(&s.totals[pass * 256 + threadIdx.x], sum);
}

// hist[d][c] -> first position of chunk c's items of digit d: a workgroup per digit scans its chunks
__global__ __launch_bounds__(256) void k_token_scan(const Sort s, int pass) {
  __shared__ int32_t red[4], wsum[4];
  const int d = blockIdx.x, t = threadIdx.x, lane = t & 63, w = t >> 6;
  int32_t before = t < d ? s.totals[pass * 256 + t] : 0;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) before += __shfl_xor(before, o);
  if (lane == 0) red[w] = before;
  constexpr int kPer = kMaxChunks / 256;
  int32_t* row = s.hist + (int64_t)d * s.chunks;
  int32_t v[kPer], sum = 0;
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    const int c = t * kPer + j;
    v[j] = c < s.chunks ? row[c] : 0;
    sum += v[j];
  }
  int32_t incl = sum;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int32_t up = __shfl_up(incl, o);
    if (lane >= o) incl += up;
  }
  if (lane == 63) wsum[w] = incl;
  __syncthreads();
  int32_t run = red[0] + red[1] + red[2] + red[3] + incl - sum;
  for (int j = 0; j < w; ++j) run += wsum[j];
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    const int c = t * kPer + j;
    if (c < s.chunks) row[c] = run;
    run += v[j];
  }
}

// A wave places its chunk 64 items at a time: an item's place is the digit's next position plus the number of
// lower lanes with the same digit.
__global__ __launch_bounds__(256) void k_token_scatter(const Sort s, int pass) {
  __shared__ int32_t next_[kSortWaves][256];
  const int w = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int64_t chunk = blockIdx.x * (int64_t)kSortWaves + w;
  if (chunk < s.chunks)
    for (int d = lane; d < 256; d += 64) next_[w][d] = s.hist[(int64_t)d * s.chunks + chunk];
  __syncthreads();
  if (chunk >= s.chunks) return;
  volatile int32_t* next = next_[w];  // other lanes' updates of the last round are read back
  const int64_t i0 = chunk * s.chunk, i1 = min(s.n, i0 + s.chunk);
  for (int64_t i = i0 + lane; i - lane < i1; i += 64) {
    const bool on = i < i1;
    uint32_t key = 0, id = 0;
    if (on) sort_item(s, pass, i, key, id);
    const int digit = (key >> (8 * pass)) & 255;
    uint64_t same = __ballot(on);
#pragma unroll
    for (int b = 0; b < 8; ++b) {
      const bool bit = (digit >> b) & 1;
      const uint64_t m = __ballot(bit);
      same &= bit ? m : ~m;
    }
    const int rank = __popcll(same & (((uint64_t)1 << lane) - 1));
    int32_t pos = 0;
    if (on) {
      pos = next[digit] + rank;
      s.key[pass & 1][pos] = key;
      s.id[pass & 1][pos] = id;
    }
    __builtin_amdgcn_wave_barrier();
    if (on && rank == 0) next[digit] = pos + __popcll(same);
    __builtin_amdgcn_wave_barrier();
  }
}

// --------------------------------------------------------------------------------------------
// Sums of runs
// --------------------------------------------------------------------------------------------
struct Runs {
  const uint32_t *key, *id;
  int64_t n, V, D, ldd, seg, segs;
  int64_t slices;  // column slices of a row
  int32_t group;   // lanes of a slice
  int64_t ldp;     // D rounded up to 8
  float* head;     // [segs][ldp]: the part of a run that began before the segment
  float* tail;     // [segs][ldp]: the part of a run that goes on behind it and began inside
  float scale;
};

constexpr int kAhead = 8;  // rows in flight

template <typename T>
__global__ __launch_bounds__(256) void k_token_runs(const Runs a, const T* __restrict__ dy, T* __restrict__ dtable) {
  constexpr int VEC = Cols<T>::kVec;
  const int64_t worker = (blockIdx.x * (int64_t)256 + threadIdx.x) / a.group;
  const int64_t seg = worker / a.slices;
  const int64_t c = ((worker - seg * a.slices) * a.group + threadIdx.x % a.group) * VEC;
  if (seg >= a.segs || c >= a.D) return;
  const int64_t p0 = seg * a.seg, p1 = min(a.n, p0 + a.seg);
  const uint32_t none = (uint32_t)a.V;
  bool from_before = p0 > 0 && a.key[p0 - 1] == a.key[p0];
  float acc[VEC];
#pragma unroll
  for (int e = 0; e < VEC; ++e) acc[e] = 0.f;
  for (int64_t p = p0; p < p1; p += kAhead) {
    Cols<T> row[kAhead];
    uint32_t key[kAhead + 1];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const int64_t q = min(p + j, p1 - 1);
      key[j] = a.key[q];
      row[j].load(dy + (int64_t)a.id[q] * a.ldd + c, a.D - c);
    }
    key[kAhead] = p + kAhead < a.n ? a.key[p + kAhead] : none + 1;
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const int64_t q = p + j;
      if (q < p1) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) acc[e] += row[j].get(e);
        // the key behind q: of the next row here, or across the segment's end
        uint32_t next = key[j + 1];
        if (q + 1 == p1) next = p1 < a.n ? a.key[p1] : none + 1;
        const bool ends = next != key[j], last = q + 1 == p1;
        if (ends || last) {
          if (key[j] != none) {
            if (from_before || !ends) {
              float* part = (from_before ? a.head : a.tail) + seg * a.ldp + c;
#pragma unroll
              for (int e = 0; e < VEC; ++e) part[e] = acc[e];  // ldp is a multiple of 8
            } else {
              Cols<T> o;
#pragma unroll
              for (int e = 0; e < VEC; ++e) o.set(e, acc[e] * a.scale);
              o.store(dtable + (int64_t)key[j] * a.D + c, a.D - c);
            }
          }
          from_before = false;
#pragma unroll
          for (int e = 0; e < VEC; ++e) acc[e] = 0.f;
        }
      }
    }
  }
}

// The runs that cross segments, 64 columns a workgroup: each of its 16 groups of 16 lanes takes a segment whose last run
// goes on and began in it, and adds the partial rows in order; runs over 16 segments and more are left for the
// whole workgroup, a contiguous part for each group and the groups' sums in order. (A workgroup per segment spent
// 25 us at 65536 tokens finding that most have nothing to do.)
template <typename T>
__global__ __launch_bounds__(256) void k_token_join(const Runs a, T* __restrict__ dtable) {
  __shared__ float part[16][64];
  __shared__ int32_t behind, longs[16];
  const int lane = threadIdx.x & 15, g = threadIdx.x >> 4;
  const int64_t c = blockIdx.y * (int64_t)64 + lane * 4;
  auto at = [&](const float* p, int64_t seg) { return *reinterpret_cast<const floatx4*>(p + seg * a.ldp + c); };
  {
    const int64_t seg = blockIdx.x * (int64_t)16 + g, p1 = (seg + 1) * a.seg;
    bool owner = p1 < a.n;
    uint32_t key = 0;
    if (owner) {
      key = a.key[p1];
      owner = key != (uint32_t)a.V && a.key[p1 - 1] == key && (seg == 0 || a.key[seg * a.seg - 1] != key);
    }
    // the segments behind that begin with the run, 16 looked at
    const int64_t t = seg + 1 + lane;
    const bool same = owner && t < a.segs && a.key[t * a.seg] == key;
    const uint32_t mask = (uint32_t)(__ballot(same) >> (threadIdx.x & 48)) & 0xffffu;
    const int parts = __ffs((int)(~mask)) - 1;  // bit 16 of ~mask is set: at most 16
    if (lane == 0) longs[g] = owner && parts == 16;
    if (owner && parts < 16 && c < a.ldp) {
      floatx4 s = at(a.tail, seg);
      for (int j = 0; j < parts; ++j) s += at(a.head, seg + 1 + j);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (c + e < a.D) store1(dtable + (int64_t)key * a.D + c + e, s[e] * a.scale);
    }
  }
  __syncthreads();
  for (int k = 0; k < 16; ++k) {
    if (!longs[k]) continue;
    const int64_t seg = blockIdx.x * (int64_t)16 + k;
    const uint32_t key = a.key[(seg + 1) * a.seg];
    int64_t parts = 0;
    for (int64_t t0 = seg + 1;; t0 += 256) {
      if (threadIdx.x == 0) behind = 256;
      __syncthreads();
      const int64_t t = t0 + threadIdx.x;
      if (t >= a.segs || a.key[t * a.seg] != key) atomicMin(&behind, (int32_t)threadIdx.x);
      __syncthreads();
      const int32_t got = behind;
      parts += got;
      __syncthreads();
      if (got < 256) break;
    }
    const int64_t t0 = seg + 1 + parts * g / 16, t1 = seg + 1 + parts * (g + 1) / 16;
    floatx4 s = {0.f, 0.f, 0.f, 0.f};
    if (c < a.ldp) {
      if (g == 0) s = at(a.tail, seg);
      int64_t t = t0;
      for (; t + 8 <= t1; t += 8) {
        floatx4 v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = at(a.head, t + j);
#pragma unroll
        for (int j = 0; j < 8; ++j) s += v[j];
      }
      for (; t < t1; ++t) s += at(a.head, t);
    }
    *reinterpret_cast<floatx4*>(&part[g][lane * 4]) = s;
    __syncthreads();
    const int64_t col = blockIdx.y * (int64_t)64 + threadIdx.x;
    if (threadIdx.x < 64 && col < a.D) {
      float f = 0.f;
#pragma unroll
      for (int i = 0; i < 16; ++i) f += part[i][threadIdx.x];
      store1(dtable + (int64_t)key * a.D + col, f * a.scale);
    }
    __syncthreads();
  }
}

// --------------------------------------------------------------------------------------------
inline bool args_ok(int32_t dtype, int64_t n, int64_t V, int64_t D) {
  return (dtype == AIMX_DTYPE_F32 || dtype == AIMX_DTYPE_BF16) && n >= 0 && n < INT32_MAX && V >= 1 && V < INT32_MAX &&
         D >= 1 && D <= (int64_t)1 << 21;  // 64 columns a workgroup in the grid's y
}

struct Layout {
  Sort s;
  Runs r;
  size_t bytes;
};
// the workspace of a gradient; base may be null to count it
Layout layout(char* base, int64_t n, int64_t V, int64_t D) {
  Layout l{};
  size_t used = 0;
  auto take = [&](size_t b) {
    char* p = base ? base + used : nullptr;
    used += (b + 255) & ~(size_t)255;
    return p;
  };
  // 4 rounds of 64 items for a wave at least (65536 tokens, a pass: 14.6 us; 1 round: 16.4), at most kMaxChunks waves
  l.s.chunk = std::max<int64_t>(256, cdiv(cdiv(n, kMaxChunks), 64) * 64);
  l.s.chunks = cdiv(n, l.s.chunk);
  // rows of a segment: enough segments to fill the card, few enough that joining a frequent token's is short
  l.r.seg = std::max<int64_t>(32, cdiv(cdiv(n, 4096), kAhead) * kAhead);
  l.r.segs = cdiv(n, l.r.seg);
  l.s.totals = (int32_t*)take(4 * 256 * 4);
  for (int i = 0; i < 2; ++i) {
    l.s.key[i] = (uint32_t*)take((size_t)n * 4);
    l.s.id[i] = (uint32_t*)take((size_t)n * 4);
  }
  l.s.hist = (int32_t*)take((size_t)l.s.chunks * 256 * 4);
  l.r.ldp = (D + 7) / 8 * 8;
  l.r.head = (float*)take((size_t)l.r.segs * l.r.ldp * 4);
  l.r.tail = (float*)take((size_t)l.r.segs * l.r.ldp * 4);
  l.bytes = used;
  return l;
}

inline bool al16(const void* p) { return ((uintptr_t)p & 15) == 0; }

template <typename T>
int gather(const int64_t* index, int64_t n, const T* table, int64_t V, int64_t D, float scale, T* out, hipStream_t st) {
  const dim3 grid((unsigned)std::min<int64_t>(cdiv(n * cdiv(D, Cols<T>::kVec), 256), 32768));
  hipLaunchKernelGGL((k_token_gather<T>), grid, dim3(256), 0, st, index, n, table, V, D, scale, out);
  AIMX_CHECK_LAUNCH();
  return AIMX_OK;
}

template <typename T>
int grad(const int64_t* index, int64_t n, const T* dy, int64_t ldd, int64_t V, int64_t D, float scale, int64_t pad,
         T* dtable, void* ws, hipStream_t st) {
  Layout l = layout((char*)ws, n, V, D);
  const int64_t words = V * D * (int64_t)sizeof(T) / 2;
  hipLaunchKernelGGL(k_token_zero, dim3((unsigned)std::min<int64_t>(cdiv(words, 2048), 8192)), dim3(256), 0, st,
                     (uint16_t*)dtable, words, l.s.totals);
  AIMX_CHECK_LAUNCH();
  if (n == 0) return AIMX_OK;
  Sort& s = l.s;
  s.index = index;
  s.n = n;
  s.V = V;
  s.pad = pad;
  int passes = 1;
  while (passes < 4 && (V >> (8 * passes)) > 0) ++passes;  // keys up to V
  const dim3 grid((unsigned)cdiv(s.chunks, kSortWaves));
  for (int p = 0; p < passes; ++p) {
    hipLaunchKernelGGL(k_token_hist, grid, dim3(256), 0, st, s, p);
    AIMX_CHECK_LAUNCH();
    hipLaunchKernelGGL(k_token_scan, dim3(256), dim3(256), 0, st, s, p);
    AIMX_CHECK_LAUNCH();
    hipLaunchKernelGGL(k_token_scatter, grid, dim3(256), 0, st, s, p);
    AIMX_CHECK_LAUNCH();
  }
  Runs& r = l.r;
  r.key = s.key[(passes - 1) & 1];
  r.id = s.id[(passes - 1) & 1];
  r.n = n;
  r.V = V;
  r.D = D;
  r.ldd = ldd;
  r.scale = scale;
  const int64_t cols = cdiv(D, Cols<T>::kVec);
  r.group = 1;
  while (r.group < 64 && r.group < cols) r.group *= 2;
  r.slices = cdiv(cols, r.group);
  const int64_t blocks = cdiv(r.segs * r.slices * r.group, 256);
  if (blocks > INT32_MAX) return AIMX_EARG;
  hipLaunchKernelGGL((k_token_runs<T>), dim3((unsigned)blocks), dim3(256), 0, st, r, dy, dtable);
  AIMX_CHECK_LAUNCH();
  if (r.segs > 1) {
    hipLaunchKernelGGL((k_token_join<T>), dim3((unsigned)cdiv(r.segs - 1, 16), (unsigned)cdiv(D, 64)), dim3(256), 0, st, r,
                       dtable);
    AIMX_CHECK_LAUNCH();
  }
  return AIMX_OK;
}

}  // namespace
}  // namespace aimx

using namespace aimx;

extern "C" int aimx_token_embedding_forward(int32_t dtype, const int64_t* index, int64_t n, const void* table, int64_t V,
                                            int64_t D, float scale, void* out, aimx_stream_t stream) {
  if (!args_ok(dtype, n, V, D)) return AIMX_EARG;
  if (n == 0) return AIMX_OK;
  if (!index || !table || !out) return AIMX_EARG;
  if (dtype == AIMX_DTYPE_F32)
    return gather(index, n, (const float*)table, V, D, scale, (float*)out, (hipStream_t)stream);
  return gather(index, n, (const uint16_t*)table, V, D, scale, (uint16_t*)out, (hipStream_t)stream);
}

extern "C" size_t aimx_token_embedding_backward_workspace_bytes(int32_t dtype, int64_t n, int64_t V, int64_t D) {
  return args_ok(dtype, n, V, D) ? layout(nullptr, n, V, D).bytes : 0;
}

extern "C" int aimx_token_embedding_backward(int32_t dtype, const int64_t* index, int64_t n, const void* dy, int64_t ldd,
                                             int64_t V, int64_t D, float scale, int64_t padding_idx, void* dtable,
                                             void* workspace, size_t workspace_bytes, aimx_stream_t stream) {
  if (!args_ok(dtype, n, V, D) || !dtable || !al16(dtable) || (n > 0 && (!index || !dy || ldd < D))) return AIMX_EARG;
  if (!workspace || !al16(workspace) || workspace_bytes < aimx_token_embedding_backward_workspace_bytes(dtype, n, V, D))
    return AIMX_EARG;
  if (dtype == AIMX_DTYPE_F32)
    return grad(index, n, (const float*)dy, ldd, V, D, scale, padding_idx, (float*)dtable, workspace, (hipStream_t)stream);
  return grad(index, n, (const uint16_t*)dy, ldd, V, D, scale, padding_idx, (uint16_t*)dtable, workspace,
              (hipStream_t)stream);
}
