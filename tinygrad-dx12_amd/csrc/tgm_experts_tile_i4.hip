// The grouped products of tgm_experts_apply (tgm_experts_tile.h) for INT4 and UINT4 weights with f16, bf16 or fp32 scales.
#include "tgm_experts_tile.h"

namespace tgm {

template <int KIND>
static int launch_kind(const WGroupArgs& p, int shape, bool wide, int64_t most, hipStream_t st) {
  constexpr bool FINE = kind_group(KIND) == 32;
  if (shape == 0)
    return wide ? launch_experts_tile<KIND, 1, 8, FINE ? 2 : 3>(p, most, st) : launch_experts_tile<KIND, 1, 4, FINE ? 3 : 4>(p, most, st);
  if (shape == 1) return wide ? launch_experts_tile<KIND, 2, 8, 3>(p, most, st) : launch_experts_tile<KIND, 2, 4, 3>(p, most, st);
  return wide ? launch_experts_tile<KIND, 4, 8, FINE ? 2 : 3>(p, most, st) : launch_experts_tile<KIND, 4, 4, 2>(p, most, st);
}

int launch_experts_tile_i4(const WGroupArgs& p, int64_t group, int shape, bool wide, int64_t most, hipStream_t st) {
  if (!p.scales) return launch_kind<kKindI4>(p, shape, wide, most, st);
  const bool f32 = p.sdt == TGM_F32;
  switch (group) {
    case 32: return f32 ? launch_kind<kKindI4 + 33>(p, shape, wide, most, st) : launch_kind<kKindI4 + 32>(p, shape, wide, most, st);
    case 64: return f32 ? launch_kind<kKindI4 + 65>(p, shape, wide, most, st) : launch_kind<kKindI4 + 64>(p, shape, wide, most, st);
    default: return f32 ? launch_kind<kKindI4 + 129>(p, shape, wide, most, st) : launch_kind<kKindI4 + 128>(p, shape, wide, most, st);
  }
}

}  // namespace tgm
