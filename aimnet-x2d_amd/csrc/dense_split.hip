// Three-plane products: fp32 tensors at fp32 accuracy.
#include "dense_core.h"

namespace aimx {
namespace dense {
namespace {

template <int PA, int PB>
using Medium = Config<PA, PB, 128, 128, 2, 2, 32>;  // 4 waves of 64 x 64; 96 KB of LDS at 3 x 3 planes
template <int PA, int PB>
using Small = Config<PA, PB, 64, 64, 2, 2, 32>;  // 4 waves of 32 x 32; 48 KB

template <typename C>
int go(const Problem& p, int halves, hipStream_t st) {
  if (p.splits > 1) return launch_config<C, kSlab, float>(p, st);
  return halves == 2 ? launch_config<C, kGated, float>(p, st) : launch_config<C, kPlain, float>(p, st);
}

template <int PA, int PB>
int go_planes(const Problem& p, int tile, int halves, hipStream_t st) {
  return tile == 0 ? go<Medium<PA, PB>>(p, halves, st) : go<Small<PA, PB>>(p, halves, st);
}

}  // namespace

Plan plan_split(int64_t M, int64_t columns, int64_t K, bool may_split) {
  auto tiles = [&](int64_t t) { return cdiv(M, t) * cdiv(columns, t); };
  const int64_t most = may_split ? std::max<int64_t>(1, K / 256) : 1;  // a k range has 8 steps at least
  if (tiles(128) * most >= 192) return {0, (int)std::min(most, cdiv(256, tiles(128)))};
  return {1, (int)std::min(most, cdiv(512, tiles(64)))};
}

int launch_split(const Problem& p, int tile, int pa, int pb, int halves, hipStream_t st) {
  if (pa == 3 && pb == 3) return go_planes<3, 3>(p, tile, halves, st);
  if (pa == 1 && pb == 3) return go_planes<1, 3>(p, tile, halves, st);
  if (pa == 3 && pb == 1) return go_planes<3, 1>(p, tile, halves, st);
  return AIMX_EARG;
}

}  // namespace dense
}  // namespace aimx
