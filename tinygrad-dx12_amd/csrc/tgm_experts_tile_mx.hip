// The grouped products of tgm_experts_apply (tgm_experts_tile.h) for FP4 and FP6 weights.
#include "tgm_experts_tile.h"

namespace tgm {

// Stages in LDS: as many as leave room for two workgroups a compute unit, or fill it.
template <int F>
static int launch_kind(const WGroupArgs& p, int shape, bool wide, int64_t most, hipStream_t st) {
  constexpr bool FP4 = F == TGM_FMT_FP4_E2M1;
  if (shape == 0)
    return wide ? launch_experts_tile<F, 1, 8, FP4 ? 3 : 2>(p, most, st) : launch_experts_tile<F, 1, 4, FP4 ? 4 : 3>(p, most, st);
  if (shape == 1) return wide ? launch_experts_tile<F, 2, 8, 3>(p, most, st) : launch_experts_tile<F, 2, 4, 3>(p, most, st);
  return wide ? launch_experts_tile<F, FP4 ? 4 : 3, 8, 3>(p, most, st) : launch_experts_tile<F, FP4 ? 4 : 3, 4, 3>(p, most, st);
}

int launch_experts_tile_mx(const WGroupArgs& p, int fmt, int shape, bool wide, int64_t most, hipStream_t st) {
  if (fmt == TGM_FMT_FP4_E2M1) return launch_kind<TGM_FMT_FP4_E2M1>(p, shape, wide, most, st);
  if (fmt == TGM_FMT_FP6_E2M3) return launch_kind<TGM_FMT_FP6_E2M3>(p, shape, wide, most, st);
  return launch_kind<TGM_FMT_FP6_E3M2>(p, shape, wide, most, st);
}

}  // namespace tgm
