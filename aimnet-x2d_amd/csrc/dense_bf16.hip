// One-plane products: bf16 tensors, or fp32 tensors whose operands are rounded to bf16 (autocast).
#include "dense_core.h"

namespace aimx {
namespace dense {
namespace {

using Large = Config<1, 1, 256, 256, 2, 4, 64>;   // 8 waves of 128 x 64, 128 KB of LDS: one workgroup a CU
using Medium = Config<1, 1, 128, 128, 2, 2, 64>;  // 4 waves of 64 x 64, 64 KB: two
using Small = Config<1, 1, 64, 64, 2, 2, 64>;     // 4 waves of 32 x 32, 32 KB: five

}  // namespace

// At 20480 x 512 (K = 4096) 160 large tiles take 119 us, in two k ranges 131 and 19 for their sum; at
// 20480 x 2048 (K = 512) three rounds of large tiles take 80 us and five of middle ones 68.
Plan plan_one(int64_t M, int64_t columns, int64_t K, bool may_split) {
  static const Shape shapes[] = {{0, 256, 256, 64, 1, 1.74, 9.}, {1, 128, 128, 64, 2, 1.08, 4.5}, {2, 64, 64, 64, 5, 0.85, 3.}};
  const int64_t force = opt_i64("AIMX_DENSE_TILE", -1);  // test hook (aimx_set_option)
  if (force >= 0 && force < 3) return pick(shapes + force, 1, M, columns, K, may_split);
  return pick(shapes, 3, M, columns, K, may_split);
}

int launch_one(const Problem& p, int tile, int epi, int across, bool fp32, hipStream_t st) {
  if (tile == 0) return fp32 ? launch_epi<Large, float>(p, epi, across, st) : launch_epi<Large, uint16_t>(p, epi, across, st);
  if (tile == 1)
    return fp32 ? launch_epi<Medium, float>(p, epi, across, st) : launch_epi<Medium, uint16_t>(p, epi, across, st);
  return fp32 ? launch_epi<Small, float>(p, epi, across, st) : launch_epi<Small, uint16_t>(p, epi, across, st);
}

}  // namespace dense
}  // namespace aimx
