// One-plane products: bf16 tensors, or fp32 tensors whose operands are rounded to bf16 (autocast).
#include "dense_core.h"

namespace aimx {
namespace dense {
namespace {

using Large = Config<1, 1, 256, 256, 2, 4, 64>;   // 8 waves of 128 x 64, 128 KB of LDS: one workgroup a CU
using Medium = Config<1, 1, 128, 128, 2, 2, 64>;  // 4 waves of 64 x 64, 64 KB: two
using Small = Config<1, 1, 64, 64, 2, 2, 64>;     // 4 waves of 32 x 32, 32 KB: five

}  // namespace

Plan plan_one(int64_t M, int64_t columns, int64_t K, bool may_split) {
  auto tiles = [&](int64_t t, int64_t u) { return std::max<int64_t>(1, cdiv(M, t) * cdiv(columns, u)); };
  const int64_t steps = K / 64;
  const int64_t most = may_split ? std::max<int64_t>(1, steps / 8) : 1;  // a k range has 8 steps at least
  const int64_t force = tune_i64("AIMX_DENSE_TILE", -1), fs = tune_i64("AIMX_DENSE_SPLITS", 0);
  Plan r{2, 1, 2, 64};
  if (tiles(256, 256) * most >= 192) r = {0, (int)std::min(most, cdiv(192, tiles(256, 256))), 2, 256};
  else if (tiles(128, 128) * most >= 192) r = {1, (int)std::min(most, cdiv(384, tiles(128, 128))), 2, 128};
  else r.splits = (int)std::min(most, cdiv(512, tiles(64, 64)));
  if (force >= 0) r.tile = (int)force, r.tile_m = force == 0 ? 256 : force == 1 ? 128 : 64;
  if (fs > 0) r.splits = (int)std::min(may_split ? fs : 1, steps);
  return r;
}

int launch_one(const Problem& p, int tile, int epi, int across, bool fp32, hipStream_t st) {
  if (tile == 0) return fp32 ? launch_epi<Large, float>(p, epi, across, st) : launch_epi<Large, uint16_t>(p, epi, across, st);
  if (tile == 1)
    return fp32 ? launch_epi<Medium, float>(p, epi, across, st) : launch_epi<Medium, uint16_t>(p, epi, across, st);
  return fp32 ? launch_epi<Small, float>(p, epi, across, st) : launch_epi<Small, uint16_t>(p, epi, across, st);
}

}  // namespace dense
}  // namespace aimx
