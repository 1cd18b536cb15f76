// The products of few tokens (tgm_experts_few.h) for FP4 and FP6 weights.
#include "tgm_experts_few.h"

namespace tgm {

int launch_experts_few_mx(const FewArgs& p, int fmt, bool up, int groups, hipStream_t st) {
  if (fmt == TGM_FMT_FP4_E2M1) return launch_experts_few<TGM_FMT_FP4_E2M1>(p, up, groups, st);
  if (fmt == TGM_FMT_FP6_E2M3) return launch_experts_few<TGM_FMT_FP6_E2M3>(p, up, groups, st);
  return launch_experts_few<TGM_FMT_FP6_E3M2>(p, up, groups, st);
}

}  // namespace tgm
