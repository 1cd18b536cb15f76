// The grouped products of tgm_experts_apply (tgm_gemm_w_tile.h) for INT4 and UINT4 weights with f16, bf16 or fp32 scales.
#include "tgm_experts.h"

namespace tgm {

// The 32 x 64 shape holds two stages with scales per 32, whose third would not fit the LDS.
template <int KIND>
static int launch_kind(const WGroupArgs& p, int shape, int64_t most, hipStream_t st) {
  switch (shape) {
    case 0: return launch_experts_tile<KIND, 1, 2, 4, kind_group(KIND) == 32 ? 2 : 3>(p, most, st);
    case 1: return launch_experts_tile<KIND, 2, 2, 2, 3>(p, most, st);
    case 2: return launch_experts_tile<KIND, 2, 4, 1, 3>(p, most, st);
    default: return launch_experts_tile<KIND, 4, 8, 1, 2>(p, most, st);
  }
}

int launch_experts_tile_i4(const WGroupArgs& p, int64_t group, int shape, int64_t most, hipStream_t st) {
  if (!p.scales) return launch_kind<kKindI4>(p, shape, most, st);
  const bool wide = p.sdt == TGM_F32;
  switch (group) {
    case 32: return wide ? launch_kind<kKindI4 + 33>(p, shape, most, st) : launch_kind<kKindI4 + 32>(p, shape, most, st);
    case 64: return wide ? launch_kind<kKindI4 + 65>(p, shape, most, st) : launch_kind<kKindI4 + 64>(p, shape, most, st);
    default: return wide ? launch_kind<kKindI4 + 129>(p, shape, most, st) : launch_kind<kKindI4 + 128>(p, shape, most, st);
  }
}

}  // namespace tgm
