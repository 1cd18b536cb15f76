// The grouped products of tgm_experts_apply (tgm_gemm_w_tile.h) for FP4 and FP6 weights.
#include "tgm_experts.h"

namespace tgm {

// The 32 x 64 shape holds two stages for FP6, whose third would not fit the LDS.
template <int F>
static int launch_kind(const WGroupArgs& p, int shape, int64_t most, hipStream_t st) {
  constexpr bool FP4 = F == TGM_FMT_FP4_E2M1;
  switch (shape) {
    case 0: return launch_experts_tile<F, 1, 2, 4, FP4 ? 3 : 2>(p, most, st);
    case 1: return launch_experts_tile<F, 2, 2, 2, 3>(p, most, st);
    case 2: return launch_experts_tile<F, 2, 4, 1, 3>(p, most, st);
    default: return launch_experts_tile<F, 4, 8, 1, FP4 ? 3 : 2>(p, most, st);
  }
}

int launch_experts_tile_mx(const WGroupArgs& p, int fmt, int shape, int64_t most, hipStream_t st) {
  if (fmt == TGM_FMT_FP4_E2M1) return launch_kind<TGM_FMT_FP4_E2M1>(p, shape, most, st);
  if (fmt == TGM_FMT_FP6_E2M3) return launch_kind<TGM_FMT_FP6_E2M3>(p, shape, most, st);
  return launch_kind<TGM_FMT_FP6_E3M2>(p, shape, most, st);
}

}  // namespace tgm
