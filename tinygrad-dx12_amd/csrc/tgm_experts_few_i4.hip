// The products of few tokens (tgm_experts_few.h) for INT4 and UINT4 weights with f16, bf16 or fp32 scales.
#include "tgm_experts_few.h"

namespace tgm {

int launch_experts_few_i4(const FewArgs& p, int64_t group, bool up, int groups, hipStream_t st) {
  if (!p.scales) return launch_experts_few<kKindI4>(p, up, groups, st);
  const bool wide = p.sdt == TGM_F32;
  switch (group) {
    case 32: return wide ? launch_experts_few<kKindI4 + 33>(p, up, groups, st) : launch_experts_few<kKindI4 + 32>(p, up, groups, st);
    case 64: return wide ? launch_experts_few<kKindI4 + 65>(p, up, groups, st) : launch_experts_few<kKindI4 + 64>(p, up, groups, st);
    default: return wide ? launch_experts_few<kKindI4 + 129>(p, up, groups, st) : launch_experts_few<kKindI4 + 128>(p, up, groups, st);
  }
}

}  // namespace tgm
