// The experts' products of few tokens (tgm_experts_apply): two launches that stream the weights of the experts which the
// tokens name.
//
// What bounds it: the weights' bytes, each read once, and on the way there the L1, which takes one access for four
// neighbouring lanes of one 64-byte line and four where their lines differ.  The B operand of a 16 x 16 x 32 product wants 16
// weight rows in neighbouring lanes; loaded so, straight into it, codes and scales of 2 experts of 4096 x 14336 took 132
// accesses a KB, and the gate|up product of one token 43 us.  So a wave loads 16 rows x 512 columns in whole lines, and the
// activations of the tokens beside them, two such groups ahead, and turns them in a block of LDS of its own, 12 waves a
// compute unit: 28 us, and 15 for the down product; a bare read in this order takes 21 us for the 117 MB of codes, in 64-byte
// pieces 26.
//
// No sorting of tokens comes first: every workgroup makes the list from the ids by itself (pairs of a token and an expert:
// 128 at most).  An entry of it is an expert and up to four of the tokens that name it; more make a second entry, and the
// weights pass again.
//
//   experts_up_few    a wave takes 16 rows (8 gate and up pairs) of an entry, all of K or a slice of it, and stores
//                     silu(gate) * up, a row per pair;
//   experts_down_few  a workgroup takes `rows` rows of the output and every entry; its waves share the groups of all
//                     entries evenly, weigh each entry's sums per token, and meet in LDS in the waves' order.
//
// D of a product: lane l holds weight row l % 16 of tokens 4 (l / 16) .. + 3.
#pragma once

#include "tgm_experts.h"
#include "tgm_lanes.h"

namespace tgm {

constexpr int kFewTokens = 16, kFewPairs = 128;
constexpr int kFewRows = 4;  // tokens of an entry
struct FewArgs {
  const uint8_t* w;
  const uint8_t* scales;
  int64_t w_bytes, s_bytes;  // of an expert
  const uint8_t* a;          // x, or the hidden activations
  int64_t lda;               // bytes
  unsigned a_bytes;          // of all of it
  const int32_t* ids;
  const float* weights;
  void* list;  // FewList, written by the first launch
  int tokens, top_k, experts;
  int N, K, sdt, is_signed;
  int slices;  // up: waves that share a row's K
  int rows;    // down: output rows of a workgroup
  void* y;     // hidden activations [pair][N / 2], or the output
  int64_t ldy;
  int ydt;
};

// Experts that some token names, each with up to four of the tokens, in the order of the first pair of each entry.  Of pairs of
// one token and one expert the first stands for all of them, with the sum of their weights.
struct __attribute__((aligned(16))) FewList {
  int8_t first[kFewPairs][kFewTokens];  // the pair of this entry and token; -1: the token is not of the entry
  int8_t place[kFewPairs][kFewTokens];  // of each token in the entry; 0 where it is not of it
  int8_t pair[kFewPairs][kFewRows];     // the pairs by place, -1 behind them
  int8_t token[kFewPairs][kFewRows];
  int16_t expert[kFewPairs];
  float weight[kFewPairs];  // of each pair
  int count, unused[3];
};
static_assert(sizeof(FewList) % 16 == 0 && kMaxExperts <= 32767 && kFewPairs <= 128, "a list is copied by 16 bytes");

struct FewScratch {
  int mark[kMaxExperts];
  int ids[kFewPairs];
  float weights[kFewPairs];
  int8_t of[kFewPairs][kFewTokens];     // the pair of an expert, by its first pair's rank, and a token
  int8_t among[kFewPairs][kFewTokens];  // the token's place among the expert's
  int8_t entry[kFewPairs][kFewTokens / kFewRows];
  int waves[4];
};

// Every workgroup makes the list for itself.
__device__ __forceinline__ void few_list(const FewArgs& p, FewList& list, FewScratch& x) {
  const int pairs = p.tokens * p.top_k, tid = threadIdx.x, lane = tid & 63;
  int id = -1;
  float weight = 0.0f;
  if (tid < pairs) id = p.ids[tid], weight = p.weights[tid];
  if (tid < kFewPairs) {
    const u32x4 none = {~0u, ~0u, ~0u, ~0u};
    *(u32x4*)list.first[tid] = none, *(u32x4*)x.of[tid] = none;
    *(u32x4*)list.place[tid] = u32x4{0, 0, 0, 0};
    *(unsigned*)list.pair[tid] = *(unsigned*)list.token[tid] = ~0u;
    x.ids[tid] = id, x.weights[tid] = weight;
  }
  for (int i = tid; i < p.experts; i += blockDim.x) x.mark[i] = kFewPairs;
  __syncthreads();
  const bool named = tid < pairs && (unsigned)id < (unsigned)p.experts;
  if (named) atomicMin(&x.mark[id], tid);
  __syncthreads();
  const bool heads = named && x.mark[id] == tid;  // the first pair of its expert
  unsigned long long set = __ballot(heads);
  if (tid < 128 && lane == 0) x.waves[tid >> 6] = __builtin_popcountll(set);
  __syncthreads();
  if (heads) x.mark[id] = (tid >= 64 ? x.waves[0] : 0) + __builtin_popcountll(set & ((1ull << lane) - 1));
  __syncthreads();
  const int experts = x.waves[0] + x.waves[1];
  const int token = tid / p.top_k, rank = named ? x.mark[id] : 0;
  bool stands = named;  // for all pairs of its token and expert
  if (named) {
    float sum = 0.0f;
    for (int o = 0; o < p.top_k; ++o) {
      const int other = token * p.top_k + o;
      const bool same = x.ids[other] == id;
      stands = stands && !(same && other < tid);
      sum += same ? x.weights[other] : 0.0f;
    }
    list.weight[tid] = sum;
    if (stands) x.of[rank][token] = (int8_t)tid;
  }
  __syncthreads();
  for (int i = tid; i < experts * kFewTokens; i += blockDim.x) {  // 16 lanes an expert
    const int e = i / kFewTokens, t = i % kFewTokens;
    const unsigned tokens = (unsigned)(__ballot(x.of[e][t] >= 0) >> (lane & 48)) & 0xFFFFu;
    x.among[e][t] = (int8_t)__builtin_popcount(tokens & ((1u << t) - 1));
  }
  __syncthreads();
  const int among = stands ? x.among[rank][token] : 0;
  const bool leads = stands && among % kFewRows == 0;  // an entry
  set = __ballot(leads);
  if (tid < 128 && lane == 0) x.waves[2 + (tid >> 6)] = __builtin_popcountll(set);
  __syncthreads();
  if (leads) {
    const int entry = (tid >= 64 ? x.waves[2] : 0) + __builtin_popcountll(set & ((1ull << lane) - 1));
    x.entry[rank][among / kFewRows] = (int8_t)entry;
    list.expert[entry] = (int16_t)id;
  }
  if (tid == 0) list.count = x.waves[2] + x.waves[3];
  __syncthreads();
  if (stands) {
    const int entry = x.entry[rank][among / kFewRows], place = among % kFewRows;
    list.first[entry][token] = list.pair[entry][place] = (int8_t)tid;
    list.place[entry][token] = (int8_t)place;
    list.token[entry][place] = (int8_t)token;
  }
  __syncthreads();
}

// Four steps of 128 columns of 16 weight rows, and of the activations.
template <int KIND>
struct FewGroup {
  static constexpr bool I4 = kind_is_i4(KIND);
  static constexpr int kStep = KIND == TGM_FMT_FP6_E2M3 || KIND == TGM_FMT_FP6_E3M2 ? 96 : 64;  // bytes of a row and step
  static constexpr int kLoads = kStep / 16;                                                     // 16 bytes a lane each
  static constexpr int G = I4 ? kind_group(KIND) : 32;
  static constexpr int kScale = I4 ? (G ? 128 / (G ? G : 1) * kind_scale_bytes(KIND) : 0) : 4;  // bytes of a row and step
  static constexpr int kWords = kScale < 4 ? 1 : kScale / 4;
  // K of product j, for lane group q: 32 q + 8 j, a lane's codes as they lie, or 32 j + 8 q where scales change within a
  // step and no product may span two of them: dword q of each 16 bytes.
  static constexpr bool TURN = I4 && (G == 32 || G == 64);
  // the wave's block of LDS: rows apart by 16 bytes more, so that reads of a column spread over the banks
  static constexpr int kCodes = 4 * kStep + 16, kScales = 16 * kWords + 4, kAct = 1024 + 16;
  static constexpr int kScalesAt = 16 * kCodes, kActAt = kScalesAt + 16 * kScales, kBlock = kActAt + kFewRows * kAct;

  u32x4 codes[kLoads];
  unsigned scale[kWords];
  u32x4 act[kFewRows];
};

// Waves of a workgroup, one workgroup a compute unit, and groups in flight: 6-bit codes and scales that change within a step
// take more registers than 12 waves have.
template <int KIND>
constexpr bool kFewWide = FewGroup<KIND>::kStep == 96 || FewGroup<KIND>::TURN;
template <int KIND>
constexpr int kFewWaves = kFewWide<KIND> ? 8 : 12;
template <int KIND>
constexpr int kFewDepth = kFewWide<KIND> ? 3 : 2;

// Where a wave's loads come from.  Buffer loads: a lane whose offset lies past the end gets zeros and reads nothing, and
// every load is issued, so that the wait for a group counts the same loads of the later ones whatever lanes skip.
constexpr unsigned kFewNone = 0xFFFFFF00u;
template <int KIND>
struct FewSource {
  using G = FewGroup<KIND>;
  __amdgpu_buffer_rsrc_t w, scales, act;
  unsigned w_off[G::kLoads], s_off, a_off[kFewRows];  // of the lane in group 0
  // Bytes from a group's scales to the next, as the loads' scalar offset; 0 without scales, whose buffer is empty: a bounds check
  // against the size less a scalar offset above it would wrap.  Codes' and activations' stays below their buffers' sizes, or
  // passes them by 256 bytes and more, where the wrapped limit is still kFewNone or less.
  int s_group;
};
__device__ __forceinline__ __amdgpu_buffer_rsrc_t few_buffer(const uint8_t* base, unsigned bytes) {
  return __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, (int)bytes, 0x00020000);
}

// The lane's offsets for 16 rows from `row` on, `rows` of them, of an expert's weight.
template <int KIND>
__device__ __forceinline__ void few_rows(FewSource<KIND>& from, const FewArgs& p, int expert, int row, int rows, int steps) {
  using G = FewGroup<KIND>;
  const int lane = threadIdx.x & 63;
  const bool scaled = p.scales != nullptr;
  from.w = few_buffer(p.w + expert * p.w_bytes, (unsigned)p.w_bytes);
  from.scales = few_buffer(p.scales + (scaled ? expert * p.s_bytes : 0), scaled ? (unsigned)p.s_bytes : 0u);
#pragma unroll
  for (int i = 0; i < G::kLoads; ++i) {  // 16 bytes i * 64 + lane of 16 rows of 4 steps
    const int at = 64 * i + lane, r = at / (G::kStep / 4), c = at % (G::kStep / 4);
    from.w_off[i] = r < rows ? (unsigned)(row + r) * (unsigned)(steps * G::kStep) + (unsigned)(16 * c) : kFewNone;
  }
  const int r = lane >> 2;  // step lane % 4 of row lane / 4
  from.s_off = r < rows ? (unsigned)(row + r) * (unsigned)(steps * G::kScale) + (unsigned)((lane & 3) * G::kScale) : kFewNone;
  from.s_group = scaled ? 4 * G::kScale : 0;
}

// Group `group` of a weight's rows, which have `steps` steps, and of the tokens'; what lies past a row's end is zero.
template <int KIND>
__device__ __forceinline__ void few_load(FewGroup<KIND>& g, const FewSource<KIND>& from, int group, int steps) {
  using G = FewGroup<KIND>;
  constexpr int NT = 2;  // codes are read once: they need not stay in the caches
  const int lane = threadIdx.x & 63, left = steps - 4 * group;
#pragma unroll
  for (int i = 0; i < G::kLoads; ++i) {
    const unsigned off = (64 * i + lane) % (G::kStep / 4) * 16 < left * G::kStep ? from.w_off[i] : kFewNone;
    g.codes[i] = __builtin_amdgcn_raw_buffer_load_b128(from.w, off, group * 4 * G::kStep, NT);
  }
  const unsigned s_off = (lane & 3) < left ? from.s_off : kFewNone;
  const int s_at = group * from.s_group;
  if constexpr (G::kScale == 2) {
    g.scale[0] = __builtin_amdgcn_raw_buffer_load_b16(from.scales, s_off, s_at, 0);
  } else if constexpr (G::kScale == 4) {
    g.scale[0] = __builtin_amdgcn_raw_buffer_load_b32(from.scales, s_off, s_at, 0);
  } else if constexpr (G::kScale == 8) {
    const u32x2 v = __builtin_amdgcn_raw_buffer_load_b64(from.scales, s_off, s_at, 0);
    g.scale[0] = v[0], g.scale[1] = v[1];
  } else if constexpr (G::kScale == 16) {
    const u32x4 v = __builtin_amdgcn_raw_buffer_load_b128(from.scales, s_off, s_at, 0);
    g.scale[0] = v[0], g.scale[1] = v[1], g.scale[2] = v[2], g.scale[3] = v[3];
  }
#pragma unroll
  for (int i = 0; i < kFewRows; ++i)
    g.act[i] = __builtin_amdgcn_raw_buffer_load_b128(from.act, lane / 16 < left ? from.a_off[i] : kFewNone, group * 1024, 0);
}

__device__ __forceinline__ void few_fence() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

template <int KIND>
__device__ __forceinline__ void few_write(const FewGroup<KIND>& g, unsigned char* block) {
  using G = FewGroup<KIND>;
  const int lane = threadIdx.x & 63;
  few_fence();  // the products before have read the block
#pragma unroll
  for (int i = 0; i < G::kLoads; ++i) {
    const int at = 64 * i + lane;
    *(u32x4*)(block + at / (G::kStep / 4) * G::kCodes + at % (G::kStep / 4) * 16) = g.codes[i];
  }
  if constexpr (G::kScale > 0) {
#pragma unroll
    for (int i = 0; i < G::kWords; ++i)
      *(unsigned*)(block + G::kScalesAt + (lane >> 2) * G::kScales + ((lane & 3) * G::kWords + i) * 4) = g.scale[i];
  }
#pragma unroll
  for (int i = 0; i < kFewRows; ++i) *(u32x4*)(block + G::kActAt + i * G::kAct + lane * 16) = g.act[i];
  few_fence();
}

// acc += the products of step j of the block; A's row of this lane is row `place` of the activations.  Four sums, so that no
// product waits for the last.
template <int KIND>
__device__ __forceinline__ void few_product(const unsigned char* block, int j, int place, bool scaled, const NibbleConsts& nib,
                                            unsigned sdt, f32x4 (&acc)[4]) {
  using G = FewGroup<KIND>;
  const int lane = threadIdx.x & 63, r = lane & 15, q = lane >> 4;
  u32x4 act[4];
#pragma unroll
  for (int u = 0; u < 4; ++u)
    act[u] = *(const u32x4*)(block + G::kActAt + place * G::kAct + 256 * j + (G::TURN ? 64 * u + 16 * q : 64 * q + 16 * u));
  unsigned scale[G::kWords];
#pragma unroll
  for (int i = 0; i < G::kWords; ++i)
    scale[i] = G::kScale ? *(const unsigned*)(block + G::kScalesAt + r * G::kScales + (j * G::kWords + i) * 4) : 0u;
  const unsigned char* row = block + r * G::kCodes + j * G::kStep;
  if constexpr (G::I4) {
    unsigned d[4];
    if constexpr (G::TURN) {
#pragma unroll
      for (int u = 0; u < 4; ++u) d[u] = *(const unsigned*)(row + 16 * u + 4 * q);
    } else {
      const u32x4 v = *(const u32x4*)(row + 16 * q);
      d[0] = v[0], d[1] = v[1], d[2] = v[2], d[3] = v[3];
    }
    constexpr int PER = G::G ? G::G / 32 : 4;  // products per scale
    f32x4 part = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      part = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(wt_f16x8, act[u]), decode_nibbles(d[u], nib), part, 0, 0, 0);
      if (u % PER == PER - 1) {
        float by = 1.0f;
        if constexpr (G::G != 0) {
          if constexpr (kind_scale_bytes(KIND) == 4) {
            by = bits_f32(scale[u / PER]);
          } else {
            const unsigned h = scale[u / PER / 2] >> (16 * (u / PER % 2)) & 0xFFFFu;
            by = sdt == TGM_F16 ? (float)__builtin_bit_cast(_Float16, (unsigned short)h) : bits_f32(h << 16);
          }
        }
#pragma unroll
        for (int v = 0; v < 4; ++v) acc[j][v] = __builtin_fmaf(by, part[v], acc[j][v]);
        part = f32x4{0.f, 0.f, 0.f, 0.f};
      }
    }
  } else {
    unsigned codes[6];
    if constexpr (G::kStep == 64) {
      const u32x4 v = *(const u32x4*)(row + 16 * q);
      codes[0] = v[0], codes[1] = v[1], codes[2] = v[2], codes[3] = v[3];
    } else {
#pragma unroll
      for (int i = 0; i < 3; ++i) {
        const u32x2 v = *(const u32x2*)(row + 24 * q + 8 * i);
        codes[2 * i] = v[0], codes[2 * i + 1] = v[1];
      }
    }
    wt_bf16x8 b[4];
    decode_mx_block<KIND>(codes, 0, scaled ? scale[0] >> (8 * q) & 0xFFu : 127u, b);
#pragma unroll
    for (int u = 0; u < 4; ++u)
      acc[u] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(wt_bf16x8, act[u]), b[u], acc[u], 0, 0, 0);
  }
}

__device__ __forceinline__ f32x4 few_sum(f32x4 (&acc)[4]) {
  f32x4 sum;
#pragma unroll
  for (int v = 0; v < 4; ++v) sum[v] = (acc[0][v] + acc[1][v]) + (acc[2][v] + acc[3][v]);
#pragma unroll
  for (int i = 0; i < 4; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  return sum;
}

__device__ __forceinline__ NibbleConsts few_nibbles(bool is_signed) {
  NibbleConsts n;
  n.pattern = is_signed ? 0x64006400u ^ 0x00800008u : 0x64006400u;
  n.offset = is_signed ? wt_half2{(_Float16)-1032.0f, (_Float16)-72.0f} : wt_half2{(_Float16)-1024.0f, (_Float16)-64.0f};
  return n;
}

// Workgroup b of `slices` waves a unit takes units b U + (wave / slices), + gridDim.x U, ..., U = waves / slices; a unit is
// 16 rows for one entry.  Past the last unit, waves repeat it and store nothing.
template <int KIND>
__global__ void __launch_bounds__(64 * kFewWaves<KIND>) experts_up_few(FewArgs p) {
  using G = FewGroup<KIND>;
  constexpr int D = kFewDepth<KIND>, WAVES = kFewWaves<KIND>;
  __shared__ FewList list;
  __shared__ __attribute__((aligned(16))) float parts[2][WAVES][16][4];
  __shared__ __attribute__((aligned(16))) unsigned char blocks[WAVES][G::kBlock];
  static_assert(sizeof(blocks) >= sizeof(FewScratch), "the list is made in the blocks' place");
  few_list(p, list, *(FewScratch*)&blocks[0][0]);
  if (blockIdx.x == 0)  // for the second launch
    for (int i = threadIdx.x; i < (int)(sizeof(FewList) / 16); i += 64 * WAVES) ((u32x4*)p.list)[i] = ((const u32x4*)&list)[i];
  const int count = list.count;
  if (count == 0) return;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 15, q = lane >> 4;
  const int slice = wave % p.slices, per_wg = WAVES / p.slices;
  const int tiles = p.N / 16, units = count * tiles;
  const int steps = p.K / 128, groups = (steps + 3) / 4, per = (groups + p.slices - 1) / p.slices;
  const int rounds = (units + (int)gridDim.x * per_wg - 1) / ((int)gridDim.x * per_wg);
  const int u0 = (int)blockIdx.x * per_wg + wave / p.slices;
  const NibbleConsts nib = few_nibbles(p.is_signed);
  const bool scaled = p.scales != nullptr;

  // the loads' cursor, D groups ahead of the products'
  int lr = 0, lg = 0;
  FewSource<KIND> from;
  from.act = few_buffer(p.a, p.a_bytes);
  auto seek = [&]() __attribute__((always_inline)) {
    int u = u0 + lr * (int)gridDim.x * per_wg;
    u = u < units ? u : units - 1;
    const int entry = u / tiles;
    few_rows<KIND>(from, p, __builtin_amdgcn_readfirstlane(list.expert[entry]), (u - entry * tiles) * 16, 16, steps);
    const int tokens = __builtin_amdgcn_readfirstlane(*(const int*)list.token[entry]);
#pragma unroll
    for (int i = 0; i < kFewRows; ++i) {
      const int token = (int8_t)(tokens >> (8 * i));
      from.a_off[i] = token >= 0 ? (unsigned)token * (unsigned)p.lda + (unsigned)(16 * lane) : kFewNone;
    }
  };
  auto load = [&](FewGroup<KIND>& g) __attribute__((always_inline)) {
    few_load<KIND>(g, from, slice * per + lg, steps);
    if (++lg == per) {
      lg = 0;
      if (lr + 1 < rounds) {
        ++lr;
        seek();
      }
    }
  };
  seek();
  FewGroup<KIND> ring[D];
#pragma unroll
  for (int d = 0; d < D; ++d) load(ring[d]);

  f32x4 sums[4] = {};
  int round = 0, group = 0;
  auto finish = [&]() __attribute__((always_inline)) {  // of a unit; lanes 0 .. 15 hold the entry's tokens
    f32x4 acc = few_sum(sums);
    if (p.slices > 1) {
      float(*buf)[16][4] = parts[round & 1];
      if (q == 0) *(f32x4*)buf[wave][r] = acc;
      lds_barrier();
      acc = f32x4{0.f, 0.f, 0.f, 0.f};
      if (slice == 0)
        for (int k = 0; k < p.slices; ++k) {
          const f32x4 part = *(const f32x4*)buf[wave + k][r];
#pragma unroll
          for (int v = 0; v < 4; ++v) acc[v] += part[v];
        }
    }
    const int u = u0 + round * (int)gridDim.x * per_wg, entry = u < units ? u / tiles : 0;
    const int col = (u - entry * tiles) * 8 + r / 2;
    const int pairs = *(const int*)list.pair[entry];
#pragma unroll
    for (int v = 0; v < kFewRows; ++v) {
      const float up = xor1(acc[v]);  // rows 2 i (gate) and 2 i + 1 (up) are neighbours
      const int pair = (int8_t)(pairs >> (8 * v));
      if (u < units && slice == 0 && q == 0 && r % 2 == 0 && pair >= 0)
        store_c(p.y, p.ydt, (int64_t)pair * p.ldy + col, acc[v] / (1.0f + expf(-acc[v])) * up);
    }
  };
  auto product = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      few_product<KIND>(blocks[wave], j, r < kFewRows ? r : 0, scaled, nib, (unsigned)p.sdt, sums);
      if (!kFewWide<KIND>) __builtin_amdgcn_sched_barrier(0);  // a step's operands at a time, for the registers
    }
    if (++group == per) {
      finish();
      group = 0;
      ++round;
    }
  };
  const int total = rounds * per;
  int i = 0;
  for (; i + 2 * D <= total; i += D) {
#pragma unroll
    for (int d = 0; d < D; ++d) {
      few_write<KIND>(ring[d], blocks[wave]);
      load(ring[d]);
      __builtin_amdgcn_sched_barrier(0);
      product();
      __builtin_amdgcn_sched_barrier(0);
    }
  }
  for (; i < total; i += D) {  // no loads past the last group
#pragma unroll
    for (int d = 0; d < D; ++d) {
      if (i + d < total) few_write<KIND>(ring[d], blocks[wave]);
      if (i + d + D < total) load(ring[d]);
      if (i + d < total) product();
    }
  }
}

template <int KIND>
__global__ void __launch_bounds__(64 * kFewWaves<KIND>) experts_down_few(FewArgs p) {
  using G = FewGroup<KIND>;
  constexpr int D = kFewDepth<KIND>, WAVES = kFewWaves<KIND>;
  __shared__ FewList list;
  __shared__ __attribute__((aligned(16))) unsigned char blocks[WAVES][G::kBlock];
  static_assert(sizeof(blocks) >= WAVES * 64 * 4 * sizeof(float), "the waves' sums meet in the blocks' place");
  float(*parts)[64][4] = (float(*)[64][4])&blocks[0][0];
  for (int i = threadIdx.x; i < (int)(sizeof(FewList) / 16); i += 64 * WAVES) ((u32x4*)&list)[i] = ((const u32x4*)p.list)[i];
  __syncthreads();
  const int count = list.count;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 15, q = lane >> 4;
  const int row = (int)blockIdx.x * p.rows, rows = p.N - row < p.rows ? p.N - row : p.rows;
  const int steps = p.K / 128, groups = (steps + 3) / 4;
  const int all = count * groups, per = (all + WAVES - 1) / WAVES;
  const int begin = wave * per < all ? wave * per : all, end = begin + per < all ? begin + per : all;
  const NibbleConsts nib = few_nibbles(p.is_signed);
  const bool scaled = p.scales != nullptr;

  f32x4 sum = {0.f, 0.f, 0.f, 0.f};
  if (begin < end) {
    int lslot = begin / groups, lg = begin - lslot * groups, left = end - begin;
    FewSource<KIND> from;
    from.act = few_buffer(p.a, p.a_bytes);
    auto seek = [&]() __attribute__((always_inline)) {
      few_rows<KIND>(from, p, __builtin_amdgcn_readfirstlane(list.expert[lslot]), row, rows, steps);
      const int pairs = __builtin_amdgcn_readfirstlane(*(const int*)list.pair[lslot]);
#pragma unroll
      for (int i = 0; i < kFewRows; ++i) {
        const int pair = (int8_t)(pairs >> (8 * i));
        from.a_off[i] = pair >= 0 ? (unsigned)pair * (unsigned)p.lda + (unsigned)(16 * lane) : kFewNone;
      }
    };
    auto load = [&](FewGroup<KIND>& g) __attribute__((always_inline)) {
      few_load<KIND>(g, from, lg, steps);
      if (left > 1) {
        --left;
        if (++lg == groups) {
          lg = 0;
          ++lslot;
          seek();
        }
      }
    };
    seek();
    FewGroup<KIND> ring[D];
#pragma unroll
    for (int d = 0; d < D; ++d) load(ring[d]);
    int slot = begin / groups, group = begin - slot * groups, place = list.place[slot][r];
    f32x4 sums[4] = {};
    auto weigh = [&]() __attribute__((always_inline)) {
      const f32x4 acc = few_sum(sums);
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        // tokens that are not of the entry: nothing, also where the weights are not finite
        const int pair = list.first[slot][4 * q + v];
        sum[v] = pair >= 0 ? __builtin_fmaf(list.weight[pair < 0 ? 0 : pair], acc[v], sum[v]) : sum[v];
      }
    };
    auto product = [&]() __attribute__((always_inline)) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        few_product<KIND>(blocks[wave], j, place, scaled, nib, (unsigned)p.sdt, sums);
        if (!kFewWide<KIND>) __builtin_amdgcn_sched_barrier(0);
      }
      if (++group == groups) {
        weigh();
        group = 0;
        if (++slot < count) place = list.place[slot][r];
      }
    };
    int i = begin;
    for (; i + 2 * D <= end; i += D) {
#pragma unroll
      for (int d = 0; d < D; ++d) {
        few_write<KIND>(ring[d], blocks[wave]);
        load(ring[d]);
        __builtin_amdgcn_sched_barrier(0);
        product();
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    for (; i < end; i += D) {  // no loads past the last group
#pragma unroll
      for (int d = 0; d < D; ++d) {
        if (i + d < end) few_write<KIND>(ring[d], blocks[wave]);
        if (i + d + D < end) load(ring[d]);
        if (i + d < end) product();
      }
    }
    if (group > 0) weigh();
  }
  __syncthreads();
  *(f32x4*)parts[wave][lane] = sum;
  __syncthreads();
  // neighbours in a row of the output
  for (int o = threadIdx.x; o < 256; o += 64 * WAVES) {
    const int orow = o & 15, token = o >> 4;
    if (token >= p.tokens || orow >= rows) continue;
    float y = 0.0f;
#pragma unroll
    for (int k = 0; k < WAVES; ++k) y += parts[k][(token >> 2) * 16 + orow][token & 3];
    store_c(p.y, p.ydt, (int64_t)token * p.ldy + row + orow, y);
  }
}

template <int KIND>
int launch_experts_few(const FewArgs& p, bool up, int groups, hipStream_t stream) {
  if (up) hipLaunchKernelGGL((experts_up_few<KIND>), dim3((unsigned)groups), dim3(64 * kFewWaves<KIND>), 0, stream, p);
  else hipLaunchKernelGGL((experts_down_few<KIND>), dim3((unsigned)groups), dim3(64 * kFewWaves<KIND>), 0, stream, p);
  return launch_status("tgm_experts_apply");
}

// One of the two launches, on `groups` workgroups; tgm_experts_few_{mx,i4}.hip.
int launch_experts_few_mx(const FewArgs& p, int fmt, bool up, int groups, hipStream_t stream);
int launch_experts_few_i4(const FewArgs& p, int64_t group, bool up, int groups, hipStream_t stream);
inline int experts_few_waves_mx(int fmt) {
  return fmt == TGM_FMT_FP4_E2M1 ? kFewWaves<TGM_FMT_FP4_E2M1> : kFewWaves<TGM_FMT_FP6_E2M3>;
}
inline int experts_few_waves_i4(int sdt, int64_t group) {
  if (sdt == TGM_NONE) return kFewWaves<kKindI4>;
  const bool wide = sdt == TGM_F32;
  return group == 32 ? (wide ? kFewWaves<kKindI4 + 33> : kFewWaves<kKindI4 + 32>)
                     : group == 64 ? (wide ? kFewWaves<kKindI4 + 65> : kFewWaves<kKindI4 + 64>)
                                   : (wide ? kFewWaves<kKindI4 + 129> : kFewWaves<kKindI4 + 128>);
}

}  // namespace tgm
