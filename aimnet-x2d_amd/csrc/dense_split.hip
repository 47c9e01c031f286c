// Three-plane products: fp32 tensors at fp32 accuracy, and the small bf16 backward products whose first operand, the
// gradient before the activation, keeps fp32's accuracy.
#include "dense_core.h"

namespace aimx {
namespace dense {
namespace {

template <int PA, int PB>
using Large = Config<PA, PB, 256, 128, 2, 4, 32>;  // 8 waves of 128 x 32; 144 KB of LDS at 3 x 3 planes
template <int PA, int PB>
using Medium = Config<PA, PB, 128, 128, 2, 4, 32>;  // 8 waves of 64 x 32; 96 KB of LDS at 3 x 3 planes
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

// At 9186 rows, 256 -> 2 x 683: 3168 small tiles 67 us, 792 middle ones 72; at 20480 rows, 512 -> 2 x 2048: 745 and 595.
Plan plan_split(int64_t M, int64_t columns, int64_t K, bool may_split, bool fp32) {
  static const Shape shapes[] = {{0, 128, 128, 32, 1, 1.1, 9.}, {1, 64, 64, 32, 3, 1.5, 4.}, {2, 256, 128, 32, 1, 1.95, 12.}};
  if (!fp32) return pick(shapes + 1, 1, M, columns, K, may_split);
  const int64_t force = opt_i64("AIMX_DENSE_SPLIT_TILE", -1);  // test hook (aimx_set_option)
  if (force >= 0 && force < 3) return pick(shapes + force, 1, M, columns, K, may_split);
  return pick(shapes, 3, M, columns, K, may_split);
}

int launch_split(const Problem& p, int tile, int pa, int pb, int epi, int across, bool fp32, hipStream_t st) {
  if (!fp32) {
    if (pa != 3 || pb != 1 || epi != kPlain || across == kNone) return AIMX_EARG;
    using C = Small<3, 1>;
    if (p.splits > 1) return across == kB ? launch_config<C, kSlab, kB, float>(p, st) : launch_config<C, kSlab, kBoth, float>(p, st);
    return across == kB ? launch_config<C, kPlain, kB, uint16_t>(p, st) : launch_config<C, kPlain, kBoth, uint16_t>(p, st);
  }
  if (tile == 2) return go<Large>(p, pa, pb, epi, across, st);
  return tile == 0 ? go<Medium>(p, pa, pb, epi, across, st) : go<Small>(p, pa, pb, epi, across, st);
}

}  // namespace dense
}  // namespace aimx
