// Shared by the kernels of tgm_experts_apply: the products of many experts' rows with their own weights.
#pragma once

#include "../../include/tgm_experts.h"
#include "tgm_gemm_w_tile.h"

namespace tgm {

// Tiles of the grouped products, rows by the rows that experts have on average: of 32, 64 or 128, each 128 or 256 wide.
constexpr int kExpertRows[] = {32, 64, 128};
constexpr int kExpertTileKinds = 3;
constexpr int kMaxExperts = 1024;

// A grouped product on tiles of kExpertRows[shape] rows and 128 or (wide) 256 columns, `most` tile rows at most;
// tgm_experts_tile_{mx,i4}.hip.
int launch_experts_tile_mx(const WGroupArgs& p, int fmt, int shape, bool wide, int64_t most, hipStream_t stream);
int launch_experts_tile_i4(const WGroupArgs& p, int64_t group, int shape, bool wide, int64_t most, hipStream_t stream);

template <int KIND, int FA, int WN, int WK, int NBUF>
int launch_experts_tile(const WGroupArgs& p, int64_t most, hipStream_t stream) {
  using T = WTile<KIND, FA, WN, WK, NBUF>;
  static_assert(T::kFits, "tile shape");
  const int64_t tiles = most * ((p.N + T::kBN - 1) / T::kBN);
  hipLaunchKernelGGL((gemm_w_tile<KIND, FA, WN, WK, NBUF, WGroupArgs>), dim3((unsigned)tiles), dim3(T::kThreads), 0, stream, p);
  return launch_status("tgm_experts_apply");
}

}  // namespace tgm
