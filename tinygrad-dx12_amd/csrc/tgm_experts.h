// Shared by the kernels of tgm_experts_apply: the products of many experts' rows with their own weights.
#pragma once

#include "../../include/tgm_experts.h"
#include "tgm_gemm_w_tile.h"

namespace tgm {

// Tiles of the grouped products, each 128 or 256 wide: of 32 rows, 64, or 128 (FP6: 96, which leave LDS for a third stage).
constexpr int kExpertTileKinds = 3;
constexpr int expert_rows(int64_t format, int shape) {
  return shape < 2 ? 32 << shape : format == TGM_FMT_FP6_E2M3 || format == TGM_FMT_FP6_E3M2 ? 96 : 128;
}
constexpr int kMaxExperts = 1024;

// The product of many experts' rows with their own weights: tile row tm is entry tm of a list that lies on the device, the count
// of them before it.
struct WGroupArgs {
  const uint8_t* a;
  const uint8_t* w;
  const uint8_t* scales;      // E8M0 bytes [N, K / 32] or INT4 group scales [N, K / G] of dtype sdt, of each expert; null: unscaled
  void* c;
  int64_t ldc;
  unsigned lda_bytes;
  int N, K, sdt, is_signed;
  int swiglu;                 // rows of W interleave gate and up: C has N / 2 columns of cdt, silu(gate) * up; otherwise fp32
  int cdt;
  const int* tiles;           // [0] count; from [4] on, per tile {expert, first position, positions, 0}
  // row of A at each position; null: the position itself.  A tile reads whole groups of 4 up to its height, past the last
  // position too
  const int* rows;
  unsigned a_bytes;           // of all rows of A, where rows name them
  int64_t w_bytes, s_bytes;   // of an expert's codes and scales
};

// A grouped product on tiles of expert_rows rows and 128 or (wide) 256 columns, `most` tile rows at most;
// tgm_experts_tile_{mx,i4}.hip.
int launch_experts_tile_mx(const WGroupArgs& p, int fmt, int shape, bool wide, int64_t most, hipStream_t stream);
int launch_experts_tile_i4(const WGroupArgs& p, int64_t group, int shape, bool wide, int64_t most, hipStream_t stream);

}  // namespace tgm
