// The feed-forward block of each token's experts (tgm_experts_apply).
//
//   y[t] = sum_j weights[t, j] down_e . (silu(gate_e . x[t]) * (up_e . x[t])),  e = ids[t, j]
//
// A token and one of its experts is a pair.  Up to 16 tokens and 128 pairs take the two launches of tgm_experts_few.h, more of
// them four:
//
//   experts_plan  puts the pairs in the order of their experts (a position each), and cuts each expert's positions into
//                 tiles of rows;
//   gemm_w_group  gate|up over those tiles, the rows of x gathered as they are loaded, silu(gate) * up in the epilogue:
//                 the hidden activations [position, ffn] in x's type;
//   gemm_w_group  down over the same tiles: a row of fp32 per position;
//   experts_sum   each token's rows, weighted and summed in the order of its choices.
//
// The count of tiles is known on the device alone: a launch covers the most that the pairs can make, and workgroups past
// the count end at once.
#include <math.h>

#include "tgm_experts_few.h"

namespace tgm {

constexpr int kPlanThreads = 1024;

struct PlanArgs {
  const int32_t* ids;
  int pairs, top_k, experts, rows;  // rows of a tile
  int* tiles;                       // [0] count; from [4] on {expert, first position, positions, 0}
  int* source;                      // token of each position
  int* place;                       // position of each pair; -1: no expert
};

// Sum of v over the threads before this one (and all of them in total); buf: one word per wave.
__device__ __forceinline__ int block_before(int v, int* buf, int& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int sum = v;
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) {
    const int o = __shfl_up(sum, m);
    sum += lane >= m ? o : 0;
  }
  __syncthreads();
  if (lane == 63) buf[wave] = sum;
  __syncthreads();
  int before = sum - v;
  total = 0;
#pragma unroll
  for (int w = 0; w < kPlanThreads / 64; ++w) {
    before += w < wave ? buf[w] : 0;
    total += buf[w];
  }
  return before;
}

// One workgroup; a thread's first kPlanEach ids stay in registers, so that all of them are loaded at once and once.  A pair's
// position among those of its expert goes by an atomic's order, which changes nothing else: every row is computed alike
// wherever it stands.
constexpr int kPlanEach = 16;
__global__ void __launch_bounds__(kPlanThreads) experts_plan(PlanArgs a) {
  __shared__ int count[kMaxExperts];
  __shared__ int buf[kPlanThreads / 64];
  const int e = threadIdx.x;
  unsigned ids[kPlanEach];
#pragma unroll
  for (int i = 0; i < kPlanEach; ++i) {
    const int pair = i * kPlanThreads + threadIdx.x;
    ids[i] = pair < a.pairs ? (unsigned)a.ids[pair] : ~0u;
  }
  count[e] = 0;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kPlanEach; ++i)
    if (ids[i] < (unsigned)a.experts) atomicAdd(&count[ids[i]], 1);
  for (int i = kPlanEach * kPlanThreads + threadIdx.x; i < a.pairs; i += kPlanThreads) {
    const unsigned id = (unsigned)a.ids[i];
    if (id < (unsigned)a.experts) atomicAdd(&count[id], 1);
  }
  __syncthreads();
  const int n = count[e];
  int total;
  const int first = block_before(n, buf, total);
  const int tiles = (n + a.rows - 1) / a.rows;
  const int at = block_before(tiles, buf, total);
  if (e == 0) a.tiles[0] = total;
  for (int i = 0; i < tiles; ++i) {
    int* entry = a.tiles + 4 + 4 * (at + i);
    entry[0] = e;
    entry[1] = first + i * a.rows;
    entry[2] = n - i * a.rows < a.rows ? n - i * a.rows : a.rows;
  }
  count[e] = first;
  __syncthreads();
  auto put = [&](int pair, unsigned id) __attribute__((always_inline)) {
    int p = -1;
    if (id < (unsigned)a.experts) {
      p = atomicAdd(&count[id], 1);
      a.source[p] = pair / a.top_k;
    }
    a.place[pair] = p;
  };
#pragma unroll
  for (int i = 0; i < kPlanEach; ++i)
    if (i * kPlanThreads + (int)threadIdx.x < a.pairs) put(i * kPlanThreads + threadIdx.x, ids[i]);
  for (int i = kPlanEach * kPlanThreads + threadIdx.x; i < a.pairs; i += kPlanThreads) put(i, (unsigned)a.ids[i]);
}

// A token's rows, four columns a thread.
__global__ void __launch_bounds__(256) experts_sum(const float* rows, const int* place, const float* weights, int top_k,
                                                   int hidden, void* y, int ydt, int64_t ldy) {
  const int64_t token = blockIdx.x;
  const int col = (blockIdx.y * 256 + threadIdx.x) * 4;
  if (col >= hidden) return;
  f32x4 sum = {0.f, 0.f, 0.f, 0.f};
  for (int j = 0; j < top_k; ++j) {
    const int p = place[token * top_k + j];
    if (p < 0) continue;
    const float w = weights[token * top_k + j];
    const f32x4 v = *(const f32x4*)(rows + (int64_t)p * hidden + col);
#pragma unroll
    for (int i = 0; i < 4; ++i) sum[i] = __builtin_fmaf(w, v[i], sum[i]);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) store_c(y, ydt, token * ldy + col + i, sum[i]);
}

struct ExpertSizes {
  int64_t pairs, most[kExpertTileKinds], tiles, source, place, hidden, rows, bytes;
};
static ExpertSizes expert_sizes(const tgm_experts& e, int64_t tokens, int64_t top_k) {
  ExpertSizes z;
  z.pairs = tokens * top_k;
  int64_t at = 0, most = 0;
  auto take = [&](int64_t bytes) {
    const int64_t here = at;
    at += (bytes + 255) / 256 * 256;
    return here;
  };
  for (int i = 0; i < kExpertTileKinds; ++i) {
    // every expert that a pair names may end in a tile that is not full
    z.most[i] = z.pairs / expert_rows(e.format, i) + (z.pairs < e.experts ? z.pairs : e.experts);
    most = z.most[i] > most ? z.most[i] : most;
  }
  z.tiles = take(16 * (1 + most) > (int64_t)sizeof(FewList) ? 16 * (1 + most) : (int64_t)sizeof(FewList));
  z.source = take(4 * z.pairs);  // read in whole groups of 4 up to a tile's height: at most 512 bytes on, of what follows
  z.place = take(4 * z.pairs);
  z.hidden = take(2 * z.pairs * e.ffn);
  z.rows = take(4 * z.pairs * e.hidden);
  z.bytes = at;
  return z;
}

// Experts that pairs name, taken as chosen at random.
static double experts_named(const tgm_experts& e, int64_t pairs) {
  return (double)e.experts * (1.0 - pow(1.0 - 1.0 / (double)e.experts, (double)pairs));
}
// Rows of the tiles by the rows of x that an expert has on average: the kind of tile.  us of the two products of 64 (FP6: 32)
// experts of 2048 x 1408 on tiles of 32, 64 and 128 (96) rows.  FP4: 24 rows an expert 100, 101, 103; 48 rows 132, 123, 132;
// 72 rows 169, 150, 163; 96 rows 195, 170, 170; 192 rows -, -, 257.  FP6: 32 rows -, 90, 94; 48 rows -, 91, 100; 64 rows 130,
// 110, 99; 96 rows -, 124, 126; 192 rows -, 328, 293.
static int expert_tile(const tgm_experts& e, int64_t pairs) {
  const double mean = (double)pairs / experts_named(e, pairs);
  return mean <= 32.0 ? 0 : mean <= (expert_rows(e.format, 2) == 96 ? 56.0 : 96.0) ? 1 : 2;
}
// Whether tiles of 256 columns are enough to give every compute unit one.  INT4, 17 tile rows x 4096: 38 us, and 41 on 128 columns;
// FP4, 8 tile rows x 4096: 103 and 68.
static bool expert_wide(const tgm_experts& e, int64_t pairs, int64_t columns, int shape, int cus) {
  const double named = experts_named(e, pairs), rows = named + (double)(pairs / expert_rows(e.format, shape)) / 2;
  return rows * (double)((columns + 255) / 256) >= cus;
}

static bool expert_ints(int64_t format) { return format == TGM_FMT_INT4 || format == TGM_FMT_UINT4; }

static int check_experts(const tgm_experts* e, int64_t tokens, int64_t top_k) {
  TGM_CHECK_ARG(e, "null experts");
  TGM_CHECK_ARG(e->format >= TGM_FMT_INT4 && e->format <= TGM_FMT_FP6_E3M2, "unknown format");
  TGM_CHECK_ARG(e->experts >= 1 && e->experts <= kMaxExperts, "a layer holds 1 to %d experts", kMaxExperts);
  TGM_CHECK_ARG(e->hidden >= 128 && e->ffn >= 128 && e->hidden % 128 == 0 && e->ffn % 128 == 0 && e->hidden <= (1 << 17) &&
                    e->ffn <= (1 << 17),
                "hidden and ffn must be multiples of 128 up to 2^17");
  const bool scaled = e->scale_dtype != TGM_NONE;
  if (expert_ints(e->format)) {
    TGM_CHECK_ARG(!scaled || ((e->scale_dtype == TGM_F16 || e->scale_dtype == TGM_BF16 || e->scale_dtype == TGM_F32) &&
                              (e->block_size == 32 || e->block_size == 64 || e->block_size == 128)),
                  "integer weights take f16, bf16 or f32 scales per 32, 64 or 128 values");
  } else {
    TGM_CHECK_ARG(!scaled || (e->scale_dtype == TGM_E8M0 && e->block_size == 32), "float weights take E8M0 scales per 32 values");
  }
  // an expert's codes are one buffer of 32-bit offsets, the last tile's rows past its end included
  const int64_t bits = format_info((int)e->format).bits;
  TGM_CHECK_ARG((2 * e->ffn + 256) * (e->hidden * bits / 8) < (1ll << 32) && (e->hidden + 256) * (e->ffn * bits / 8) < (1ll << 32),
                "the weight of an expert must be less than 4 GiB");
  TGM_CHECK_ARG(tokens >= 0 && tokens < (1 << 24) && top_k >= 1 && top_k <= kMaxExperts && tokens * top_k < (1 << 24),
                "tokens times top_k must be less than 2^24");
  return TGM_OK;
}

}  // namespace tgm

using namespace tgm;

extern "C" int64_t tgm_experts_workspace(const tgm_experts* experts, int64_t tokens, int64_t top_k) {
  clear_error();
  if (check_experts(experts, tokens, top_k) != TGM_OK || tokens == 0) return 0;
  return expert_sizes(*experts, tokens, top_k).bytes;
}

extern "C" int tgm_experts_apply(const tgm_experts* experts, const void* x, int64_t x_dtype, int64_t tokens, int64_t ldx,
                                 const int32_t* ids, const float* weights, int64_t top_k, void* y, int64_t y_dtype,
                                 int64_t ldy, void* workspace, int64_t workspace_bytes, void* stream) {
  clear_error();
  if (const int status = check_experts(experts, tokens, top_k); status != TGM_OK) return status;
  const tgm_experts& e = *experts;
  const bool ints = expert_ints(e.format), scaled = e.scale_dtype != TGM_NONE;
  TGM_CHECK_ARG(x_dtype == (ints ? TGM_F16 : TGM_BF16), "x must be %s beside these weights", ints ? "f16" : "bf16");
  TGM_CHECK_ARG(y_dtype == x_dtype || y_dtype == TGM_F32, "y must be of x's type or f32");
  TGM_CHECK_ARG((ldx >= e.hidden && ldx % 8 == 0 && ldx < (1ll << 31) && ldy >= e.hidden && ldy < (1ll << 36)) || tokens <= 1,
                "rows must be apart, those of x by a multiple of 8");
  if (tokens == 0) return TGM_OK;
  if (tokens == 1) ldx = ldy = e.hidden;
  TGM_CHECK_ARG(((tokens - 1) * ldx + e.hidden) * 2 < (1ll << 31), "x must be less than 2 GiB");
  TGM_CHECK_ARG(x && ids && weights && y && e.gate_up && e.down, "null operand");
  TGM_CHECK_ARG(!scaled || (e.gate_up_scales && e.down_scales), "null scales");
  TGM_CHECK_ARG(((uintptr_t)x & 15) == 0 && ((uintptr_t)e.gate_up & 15) == 0 && ((uintptr_t)e.down & 15) == 0 &&
                    (!scaled || (((uintptr_t)e.gate_up_scales & 3) == 0 && ((uintptr_t)e.down_scales & 3) == 0)),
                "x and the weights must be 16-byte and scales 4-byte aligned");
  const ExpertSizes z = expert_sizes(e, tokens, top_k);
  TGM_CHECK_ARG(workspace && workspace_bytes >= z.bytes && ((uintptr_t)workspace & 15) == 0, "workspace too small or misaligned");
  const int64_t bits = format_info((int)e.format).bits;
  const int64_t per = scaled ? (e.scale_dtype == TGM_E8M0 ? 1 : dtype_size((int)e.scale_dtype)) : 0;
  const int64_t block = scaled ? e.block_size : 128;
  const hipStream_t st = (hipStream_t)stream;
  char* ws = (char*)workspace;
  const int known = stream_cu_count(st), cus = known > 0 ? known : 256;
  if (tokens <= kFewTokens && z.pairs <= kFewPairs) {
    auto product = [&](bool up) {
      FewArgs p{};
      p.w = (const uint8_t*)(up ? e.gate_up : e.down);
      p.scales = scaled ? (const uint8_t*)(up ? e.gate_up_scales : e.down_scales) : nullptr;
      p.N = (int)(up ? 2 * e.ffn : e.hidden), p.K = (int)(up ? e.hidden : e.ffn);
      p.w_bytes = (int64_t)p.N * p.K * bits / 8, p.s_bytes = (int64_t)p.N * (p.K / block) * per;
      p.a = (const uint8_t*)(up ? x : ws + z.hidden), p.lda = 2 * (up ? ldx : e.ffn);
      p.a_bytes = (unsigned)(up ? ((tokens - 1) * ldx + e.hidden) * 2 : z.pairs * e.ffn * 2);
      p.list = ws + z.tiles;
      p.ids = ids, p.weights = weights, p.tokens = (int)tokens, p.top_k = (int)top_k, p.experts = (int)e.experts;
      p.sdt = (int)e.scale_dtype, p.is_signed = e.format == TGM_FMT_INT4;
      p.y = up ? ws + z.hidden : y, p.ldy = up ? e.ffn : ldy, p.ydt = up ? (int)x_dtype : (int)y_dtype;
      int groups;
      if (up) {
        // One workgroup a compute unit.  As many of the rows' slices as waves end together best, where a unit's own work counts
        // as half a group.
        const int waves = ints ? experts_few_waves_i4(scaled ? (int)e.scale_dtype : TGM_NONE, e.block_size) : experts_few_waves_mx((int)e.format);
        const int64_t units = (int64_t)(experts_named(e, z.pairs) + 0.5) * (p.N / 16), all = (int64_t)cus * waves, parts = (p.K + 511) / 512;
        double least = 0.0;
        for (int s = 1; s <= 4 && s <= parts; s *= 2) {
          const double cost = (double)((units * s + all - 1) / all) * ((double)((parts + s - 1) / s) + 0.5);
          if (s == 1 || cost < least) least = cost, p.slices = s;
        }
        const int64_t most = (units * p.slices + waves - 1) / waves;
        groups = (int)(most < cus ? most : cus);
      } else {
        // rounds of one workgroup a compute unit, their rows even
        const int64_t rounds = (p.N + 16 * cus - 1) / (16 * cus);
        p.rows = (int)((p.N + cus * rounds - 1) / (cus * rounds));
        groups = (p.N + p.rows - 1) / p.rows;
      }
      return ints ? launch_experts_few_i4(p, e.block_size, up, groups, st) : launch_experts_few_mx(p, (int)e.format, up, groups, st);
    };
    if (const int status = product(true); status != TGM_OK) return status;
    return product(false);
  }
  const int shape = expert_tile(e, z.pairs);
  const int64_t most_columns = 2 * e.ffn > e.hidden ? 2 * e.ffn : e.hidden;
  TGM_CHECK_ARG(z.most[shape] * ((most_columns + 127) / 128) < (1ll << 31), "too many tiles");
  PlanArgs plan;
  plan.ids = ids, plan.pairs = (int)z.pairs, plan.top_k = (int)top_k, plan.experts = (int)e.experts;
  plan.rows = expert_rows(e.format, shape);
  plan.tiles = (int*)(ws + z.tiles), plan.source = (int*)(ws + z.source), plan.place = (int*)(ws + z.place);
  hipLaunchKernelGGL(experts_plan, dim3(1), dim3(kPlanThreads), 0, st, plan);
  if (const int status = launch_status("tgm_experts_apply"); status != TGM_OK) return status;

  auto product = [&](bool up) {
    WGroupArgs p{};
    p.a = (const uint8_t*)(up ? x : ws + z.hidden);
    p.w = (const uint8_t*)(up ? e.gate_up : e.down);
    p.scales = scaled ? (const uint8_t*)(up ? e.gate_up_scales : e.down_scales) : nullptr;
    p.c = ws + (up ? z.hidden : z.rows);
    p.ldc = up ? e.ffn : e.hidden;
    p.lda_bytes = (unsigned)(2 * (up ? ldx : e.ffn));
    p.N = (int)(up ? 2 * e.ffn : e.hidden), p.K = (int)(up ? e.hidden : e.ffn);
    p.cdt = up ? (int)x_dtype : TGM_F32, p.sdt = (int)e.scale_dtype, p.is_signed = e.format == TGM_FMT_INT4;
    p.swiglu = up;
    p.tiles = plan.tiles, p.rows = up ? plan.source : nullptr;
    p.a_bytes = (unsigned)(((tokens - 1) * ldx + e.hidden) * 2);
    p.w_bytes = (int64_t)p.N * p.K * bits / 8, p.s_bytes = (int64_t)p.N * (p.K / block) * per;
    const bool wide = expert_wide(e, z.pairs, p.N, shape, cus);
    return ints ? launch_experts_tile_i4(p, e.block_size, shape, wide, z.most[shape], st)
                : launch_experts_tile_mx(p, (int)e.format, shape, wide, z.most[shape], st);
  };
  if (const int status = product(true); status != TGM_OK) return status;
  if (const int status = product(false); status != TGM_OK) return status;
  hipLaunchKernelGGL(experts_sum, dim3((unsigned)tokens, (unsigned)((e.hidden + 1023) / 1024)), dim3(256), 0, st,
                     (const float*)(ws + z.rows), plan.place, weights, (int)top_k, (int)e.hidden, y, (int)y_dtype, ldy);
  return launch_status("tgm_experts_apply");
}
