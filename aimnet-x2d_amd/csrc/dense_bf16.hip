// One-plane products: bf16 tensors, or fp32 tensors whose operands are rounded to bf16 (autocast).
#include "dense_core.h"

namespace aimx {
namespace dense {
namespace {

using Large = Config<1, 1, 256, 256, 2, 4, 64>;   // 8 waves of 128 x 64, 128 KB of LDS: one workgroup a CU
using Medium = Config<1, 1, 128, 128, 2, 2, 64>;  // 4 waves of 64 x 64, 64 KB: two
using Small = Config<1, 1, 64, 64, 2, 2, 64>;     // 4 waves of 32 x 32, 32 KB: five

template <typename C>
int go(const Problem& p, int halves, bool fp32_out, hipStream_t st) {
  if (p.splits > 1) return launch_config<C, kSlab, float>(p, st);
  if (halves == 2)
    return fp32_out ? launch_config<C, kGated, float>(p, st) : launch_config<C, kGated, uint16_t>(p, st);
  return fp32_out ? launch_config<C, kPlain, float>(p, st) : launch_config<C, kPlain, uint16_t>(p, st);
}

}  // namespace

Plan plan_one(int64_t M, int64_t columns, int64_t K, bool may_split) {
  auto tiles = [&](int64_t t) { return cdiv(M, t) * cdiv(columns, t); };
  const int64_t steps = K / 64;
  const int64_t most = may_split ? std::max<int64_t>(1, steps / 8) : 1;  // a k range has 8 steps at least
  if (tiles(256) * most >= 192) return {0, (int)std::min(most, cdiv(192, tiles(256)))};
  if (tiles(128) * most >= 192) return {1, (int)std::min(most, cdiv(384, tiles(128)))};
  return {2, (int)std::min(most, cdiv(512, tiles(64)))};
}

int launch_one(const Problem& p, int tile, int halves, bool fp32_out, hipStream_t st) {
  if (tile == 0) return go<Large>(p, halves, fp32_out, st);
  if (tile == 1) return go<Medium>(p, halves, fp32_out, st);
  return go<Small>(p, halves, fp32_out, st);
}

}  // namespace dense
}  // namespace aimx
