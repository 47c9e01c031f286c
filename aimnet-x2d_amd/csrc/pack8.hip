// Activations in 8 bits (aimx_pack8 / aimx_unpack8, include/aimx.h).
//
// Groups of 32 values along a row share a power-of-two scale: e is the least integer from -126 with
// 127 * 2^e >= max|x|, and q = round(x / 2^e), to nearest even, |q| <= 127. A power of two because q * 2^e is
// then exactly a bf16 (7 bits and an exponent): the matrix instructions of the backward products read the
// checkpoint with no second rounding, as one plane also beside fp32 weights. It costs half a bit on average
// against the scale max / 127. A group that holds a NaN or an infinity keeps the exponent 127 and reads back as
// NaN: a checkpoint never turns a diverged activation into a finite one.
//
// Both directions are bound by memory and move their bytes once: a thread takes 8 values (16 or 32 bytes), the 4
// threads of a group find its largest with two lane exchanges. 32768 x 4096 bf16: packed in 87 us (4.7 TB/s; a copy
// reaches 5.06), unpacked in 64 (6.4, the packed values partly from the cache).
#include <algorithm>

#include "dense_core.h"

namespace aimx {
namespace {

typedef int8_t i8x8 __attribute__((ext_vector_type(8)));

constexpr int kNotFinite = 127;

// e of a group whose largest magnitude is the finite float with these bits: from the exponent field and
// whether the significand passes 127/128 of the next power of two
__device__ __forceinline__ int group_exp(uint32_t top) {
  const int field = (int)(top >> 23);
  if (field == 0) return -126;  // zero and subnormals: 127 * 2^-126 is far above
  // max = m 2^ex, m in [1/2, 1): ex = field - 126; 127 2^(ex-7) >= max iff m <= 127/128
  const bool over = (top & 0x7fffffu) > 0x7e0000u;
  return max(field - 126 - (over ? 6 : 7), -126);
}

template <typename T>
__global__ __launch_bounds__(256) void k_pack8(const T* __restrict__ x, int64_t ld, int64_t M, int64_t K, int64_t Kq,
                                               int8_t* __restrict__ q, int8_t* __restrict__ exps) {
  const int64_t w = Kq / 8, items = M * w;
  // every thread of a group of 4 stays in the loop as long as the group does (w and the block are
  // multiples of 4)
  for (int64_t it = blockIdx.x * (int64_t)256 + threadIdx.x; it < items; it += (int64_t)gridDim.x * 256) {
    const int64_t r = it / w, c = (it - r * w) * 8;
    float v[8];
    dense::load8(x + r * ld + c, K - c, v);
    uint32_t top = 0;  // magnitudes order as their bits, NaN above infinity
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(v[i]) & 0x7fffffffu);
    top = max(top, (uint32_t)__shfl_xor((int)top, 1));
    top = max(top, (uint32_t)__shfl_xor((int)top, 2));
    i8x8 o;
    int e = kNotFinite;
    if (top >= 0x7f800000u) {
#pragma unroll
      for (int i = 0; i < 8; ++i) o[i] = 0;
    } else {
      e = group_exp(top);
      // the largest floats round to 64 * 2^122 = 2^128: one step less keeps them finite
      const float lim = e == 122 ? 63.f : 127.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) o[i] = (int8_t)fminf(fmaxf(rintf(ldexpf(v[i], -e)), -lim), lim);
    }
    *reinterpret_cast<i8x8*>(q + r * Kq + c) = o;
    if ((c & 31) == 0) exps[r * (Kq / 32) + c / 32] = (int8_t)e;
  }
}

template <typename T>
__global__ __launch_bounds__(256) void k_unpack8(const int8_t* __restrict__ q, const int8_t* __restrict__ exps, int64_t M,
                                                 int64_t K, int64_t Kq, T* __restrict__ y, int64_t ld) {
  const int64_t w = (K + 7) / 8, items = M * w;
  for (int64_t it = blockIdx.x * (int64_t)256 + threadIdx.x; it < items; it += (int64_t)gridDim.x * 256) {
    const int64_t r = it / w, c = (it - r * w) * 8;
    const i8x8 a = *reinterpret_cast<const i8x8*>(q + r * Kq + c);
    const int e = exps[r * (Kq / 32) + c / 32];
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = e == kNotFinite ? __uint_as_float(0x7fc00000u) : ldexpf((float)a[i], e);
    dense::store8(y + r * ld + c, K - c, v);
  }
}

inline bool args_ok(int32_t dtype, int64_t M, int64_t K, int64_t ld) {
  return (dtype == AIMX_DTYPE_F32 || dtype == AIMX_DTYPE_BF16) && M >= 0 && K >= 1 && ld >= K &&
         M <= ((int64_t)1 << 56) / K;
}
inline unsigned grid_of(int64_t items) { return (unsigned)std::min<int64_t>(cdiv(items, 256), 32768); }

}  // namespace
}  // namespace aimx

using namespace aimx;

extern "C" int aimx_pack8(int32_t dtype, const void* x, int64_t ldx, int64_t M, int64_t K, int8_t* q, int8_t* exps,
                          aimx_stream_t stream) {
  if (!args_ok(dtype, M, K, ldx)) return AIMX_EARG;
  if (M == 0) return AIMX_OK;
  if (!x || !q || !exps || ((uintptr_t)q & 7)) return AIMX_EARG;
  const int64_t Kq = cdiv(K, 32) * 32;
  const dim3 grid(grid_of(M * (Kq / 8)));
  if (dtype == AIMX_DTYPE_F32)
    hipLaunchKernelGGL(k_pack8<float>, grid, dim3(256), 0, (hipStream_t)stream, (const float*)x, ldx, M, K, Kq, q, exps);
  else
    hipLaunchKernelGGL(k_pack8<uint16_t>, grid, dim3(256), 0, (hipStream_t)stream, (const uint16_t*)x, ldx, M, K, Kq, q,
                       exps);
  AIMX_CHECK_LAUNCH();
  return AIMX_OK;
}

extern "C" int aimx_unpack8(int32_t dtype, const int8_t* q, const int8_t* exps, int64_t M, int64_t K, void* y,
                            int64_t ldy, aimx_stream_t stream) {
  if (!args_ok(dtype, M, K, ldy)) return AIMX_EARG;
  if (M == 0) return AIMX_OK;
  if (!y || !q || !exps || ((uintptr_t)q & 7)) return AIMX_EARG;
  const int64_t Kq = cdiv(K, 32) * 32;
  const dim3 grid(grid_of(M * cdiv(K, 8)));
  if (dtype == AIMX_DTYPE_F32)
    hipLaunchKernelGGL(k_unpack8<float>, grid, dim3(256), 0, (hipStream_t)stream, q, exps, M, K, Kq, (float*)y, ldy);
  else
    hipLaunchKernelGGL(k_unpack8<uint16_t>, grid, dim3(256), 0, (hipStream_t)stream, q, exps, M, K, Kq, (uint16_t*)y,
                       ldy);
  AIMX_CHECK_LAUNCH();
  return AIMX_OK;
}
