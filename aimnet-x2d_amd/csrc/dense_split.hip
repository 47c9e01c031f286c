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
int plain(const Problem& p, int across, hipStream_t st) {
  if (p.splits > 1) {
    if (across == kNone) return launch_config<C, kSlab, kNone, float>(p, st);
    return across == kB ? launch_config<C, kSlab, kB, float>(p, st) : launch_config<C, kSlab, kBoth, float>(p, st);
  }
  if (across == kNone) return launch_config<C, kPlain, kNone, float>(p, st);
  return across == kB ? launch_config<C, kPlain, kB, float>(p, st) : launch_config<C, kPlain, kBoth, float>(p, st);
}

// Only what occurs: the forward and dx are 3 x 3 planes, dW 3 x 3 or, from a checkpoint, 3 x 1; the
// pre-activation values computed again stand on a checkpoint, 1 x 3.
template <template <int, int> class Tile>
int go(const Problem& p, int pa, int pb, int epi, int across, hipStream_t st) {
  if (pa == 3 && pb == 3)
    return epi == kGated ? launch_config<Tile<3, 3>, kGated, kNone, float>(p, st) : plain<Tile<3, 3>>(p, across, st);
  if (pa == 1 && pb == 3) {
    if (epi == kDenseGrad) return launch_config<Tile<1, 3>, kDenseGrad, kNone, float>(p, st);
    if (epi == kGatedGrad) return launch_config<Tile<1, 3>, kGatedGrad, kNone, float>(p, st);
  }
  if (pa == 3 && pb == 1 && across == kBoth)
    return p.splits > 1 ? launch_config<Tile<3, 1>, kSlab, kBoth, float>(p, st)
                        : launch_config<Tile<3, 1>, kPlain, kBoth, float>(p, st);
  return AIMX_EARG;
}

}  // namespace

Plan plan_split(int64_t M, int64_t columns, int64_t K, bool may_split) {
  auto tiles = [&](int64_t t) { return std::max<int64_t>(1, cdiv(M, t) * cdiv(columns, t)); };
  const int64_t most = may_split ? std::max<int64_t>(1, K / 256) : 1;  // a k range has 8 steps at least
  if (tiles(128) * most >= 192) return {0, (int)std::min(most, cdiv(256, tiles(128))), 2, 128};
  return {1, (int)std::min(most, cdiv(512, tiles(64))), 2, 64};
}

int launch_split(const Problem& p, int tile, int pa, int pb, int epi, int across, hipStream_t st) {
  return tile == 0 ? go<Medium>(p, pa, pb, epi, across, st) : go<Small>(p, pa, pb, epi, across, st);
}

}  // namespace dense
}  // namespace aimx
