// Log probabilities of given tokens, their ranks, the entropy, and the likeliest tokens (tgm_log_probs).
//
// With m the largest logit, d_i = x_i - m, S = sum exp(d_i) and T = sum exp(d_i) d_i:
//
//   log p_i = d_i - log S        entropy = -sum p_i log p_i = log S - T / S
//
// A workgroup reads a stretch of a row into registers, 32 logits a thread (64 of 16 bits where there are many rows), and
// everything else comes from there: the largest, then S, T and the token's rank, then the likeliest tokens.  Those are looked for among the logits that reach a
// bound which enough of them are sure to reach: the n-th largest of the waves' largest logits, or, with more tokens than
// waves, the least over the waves of their q-th largest thread's.  Of independent logits a few dozen reach it; they are
// listed in LDS and each counts those before it.  Where more than the list holds do (many equal ones), the tokens are taken
// one after another instead.
//
// A row that is longer than a stretch, or that would leave compute units idle, takes several, and a second launch joins
// them: S and T scale by exp(m_stretch - m), and the lists' entries that reach a bound count those before them.
//
// What bounds it: HBM with many rows (4000 x 32000 bf16, top 5: 56 us, 4.6 TB/s, where 32 logits a thread take 72), the chain
// of reductions and barriers with few (8 x 32000, top 20: 10.2 us; 131072, top 5: 6.4 in nine stretches, and the join 3; in
// four of 1024 threads 7, in 17 of 256 7.8 and 3.9).
#include <math.h>

#include "../../include/tgm_serving.h"
#include "tgm_common.h"
#include "tgm_lanes.h"

namespace tgm {

constexpr int kLpMost = 1024, kLpTop = 64, kLpList = 512, kLpJoin = 256, kLpStretches = 64;
typedef unsigned long long lp_u64;
typedef unsigned lp_u32x4 __attribute__((ext_vector_type(4)));

struct LpPart {  // of a stretch
  float max, sum, dot;
  int rank;
};

struct LpArgs {
  const void* logits;
  int64_t ld;
  int n, top, stretches;
  const int32_t* tokens;
  float* logprobs;
  int32_t* ranks;
  float* entropy;
  int32_t* top_ids;
  float* top_logprobs;
  LpPart* parts;  // [row][stretch], with several stretches
  lp_u64* lists;  // [row][stretch][top]
};

// Ascending with the value, -0 as +0; 1 a NaN, behind -infinity; 0 no element.
__device__ __forceinline__ unsigned lp_key(float x) {
  if (x != x) return 1u;
  const unsigned b = f32_bits(x + 0.0f);
  return b ^ ((b >> 31) ? 0xFFFFFFFFu : 0x80000000u);
}
__device__ __forceinline__ float lp_unkey(unsigned k) {
  return k == 1u ? NAN : bits_f32(k ^ ((k >> 31) ? 0x80000000u : 0xFFFFFFFFu));
}
// A key and its token as one number: equal keys rank by index.
__device__ __forceinline__ lp_u64 lp_entry(unsigned key, int i) { return (lp_u64)key << 32 | (unsigned)~i; }

__device__ __forceinline__ float lp_wave_max(float v) {
  v = fmaxf(v, xor1(v));
  v = fmaxf(v, xor2(v));
  v = fmaxf(v, xor4(v));
  v = fmaxf(v, xor8(v));
  v = fmaxf(v, __shfl_xor(v, 16));
  return fmaxf(v, __shfl_xor(v, 32));
}
__device__ __forceinline__ float lp_wave_sum(float v) {
  v += xor1(v);
  v += xor2(v);
  v += xor4(v);
  v += xor8(v);
  v += __shfl_xor(v, 16);
  return v + __shfl_xor(v, 32);
}

__device__ __forceinline__ void lp_write(const LpArgs& a, int64_t row, float max, float sum, float dot, int rank, float at,
                                         bool named) {
  const float log_sum = logf(sum);
  a.logprobs[row] = named ? (at - max) - log_sum : 0.0f;
  a.ranks[row] = named ? rank : -1;
  a.entropy[row] = log_sum - dot / sum;
}

template <int DT>
__device__ __forceinline__ float lp_load(const void* p, int64_t i) {
  if constexpr (DT == TGM_F32) return ((const float*)p)[i];
  else if constexpr (DT == TGM_BF16) return bf16_to_f32(((const uint16_t*)p)[i]);
  else return (float)((const _Float16*)p)[i];
}

// Reductions over the 16 lanes of a row, in every lane.
__device__ __forceinline__ float lp_row_max(float v) {
  v = fmaxf(v, xor1(v));
  v = fmaxf(v, xor2(v));
  v = fmaxf(v, xor4(v));
  return fmaxf(v, xor8(v));
}
__device__ __forceinline__ float lp_row_sum(float v) {
  v += xor1(v);
  v += xor2(v);
  v += xor4(v);
  return v + xor8(v);
}
// How many of the 16 lanes of a row hold more than v.
template <int K = 1>
__device__ __forceinline__ int lp_row_above(float v) {
  if constexpr (K < 16) return (dpp<0x120 + K>(v) > v) + lp_row_above<K + 1>(v);  // rotated by K lanes
  else return 0;
}

// Waves of 64 registers, eight on a SIMD: a row's loads go under others' arithmetic.
template <int DT, int EACH>
__global__ void __launch_bounds__(32 * kLpMost / EACH) __attribute__((amdgpu_waves_per_eu(8, 8))) logprob_rows(LpArgs a) {
  constexpr int SIZE = DT == TGM_F32 ? 4 : 2, VEC = 16 / SIZE, NV = EACH / VEC;
  __shared__ float wave_max[16], wave_reach[16], wave_sum[16], wave_dot[16], wave_rank[16];
  __shared__ lp_u64 list[kLpList];
  __shared__ lp_u64 best[16];
  __shared__ int listed;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
  const int64_t row = blockIdx.x / a.stretches;
  const int stretch = blockIdx.x % a.stretches;
  const char* base = (const char*)a.logits + row * a.ld * SIZE;
  // whole aligned vectors: the first may begin before the row and the last end behind it, in its 16 bytes
  const int shift = (int)((uintptr_t)base % 16) / SIZE;
  const lp_u32x4* vectors = (const lp_u32x4*)(base - shift * SIZE);
  const int count = (a.n + shift + VEC - 1) / VEC;
  const int v0 = stretch * (int)blockDim.x * NV + (int)threadIdx.x;
  constexpr unsigned NONE = DT == TGM_F32 ? 0xFF800000u : DT == TGM_BF16 ? 0xFF80FF80u : 0xFC00FC00u;  // -infinity
  lp_u32x4 raw[NV];
#pragma unroll
  for (int q = 0; q < NV; ++q) {
    const int v = v0 + q * (int)blockDim.x;
    raw[q] = v < count ? __builtin_nontemporal_load(vectors + v) : lp_u32x4{NONE, NONE, NONE, NONE};
  }
  const int tok = a.tokens[row];
  const bool named = (unsigned)tok < (unsigned)a.n;
  const float at = named ? lp_load<DT>(base, tok) : 0.0f;
  auto value = [&](int r) __attribute__((always_inline)) {
    const lp_u32x4 v = raw[r / VEC];
    if constexpr (DT == TGM_F32) return bits_f32(v[r % VEC]);
    const unsigned pair = v[r % VEC / 2];
    if constexpr (DT == TGM_BF16) return bits_f32(r % 2 ? pair & 0xFFFF0000u : pair << 16);
    return (float)__builtin_bit_cast(_Float16, (unsigned short)(r % 2 ? pair >> 16 : pair));
  };
  // the first and the last vector: -infinity where there is no element
#pragma unroll
  for (int q = 0; q < NV; ++q) {
    const int v = v0 + q * (int)blockDim.x;
    if (v == 0 || v == count - 1) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        constexpr int PER = 4 / SIZE;
        const unsigned mask = DT == TGM_F32 ? ~0u : i % 2 ? 0xFFFF0000u : 0xFFFFu;
        if ((unsigned)(v * VEC - shift + i) >= (unsigned)a.n) raw[q][i / PER] = (raw[q][i / PER] & ~mask) | (NONE & mask);
      }
    }
  }
  float top = -INFINITY;
#pragma unroll
  for (int r = 0; r < EACH; ++r) {
    top = fmaxf(top, value(r));
    if (r % 8 == 7) __builtin_amdgcn_sched_barrier(0);
  }
  // the stretch's largest, and a bound that `top` logits reach
  if (threadIdx.x == 0) listed = 0;
  const float wave_top = lp_wave_max(top);
  float reach = wave_top;
  if (a.top > waves) {
    float left = top;
    for (int q = (a.top + waves - 1) / waves;;) {
      reach = lp_wave_max(left);
      if (--q == 0) break;
      // one lane that holds it leaves
      const lp_u64 holds = __ballot(left == reach);
      left = holds && lane == __builtin_ctzll(holds) ? -INFINITY : left;
    }
  }
  if (lane == 0) wave_max[wave] = wave_top, wave_reach[wave] = reach;
  __syncthreads();
  const int w16 = lane & 15;
  const float each_max = w16 < waves ? wave_max[w16] : -INFINITY;
  const float max = lp_row_max(each_max);
  float bound;
  if (a.top > waves) bound = -lp_row_max(w16 < waves ? -wave_reach[w16] : -INFINITY);
  else bound = -lp_row_max(lp_row_above(each_max) < a.top ? -each_max : -INFINITY);
  const float zero = max == -INFINITY ? 0.0f : max;
  // unpacked anew: kept from one pass to the next, the values would not fit the registers
#pragma unroll
  for (int q = 0; q < NV; ++q) asm volatile("" : "+v"(raw[q]));
  // The rank counts what is larger, and equal logits before the token: vectors before its own compare with it, later ones with the
  // next number above it, and its own vector's equal ones are counted at the end.  A comparison with a NaN does not hold, so
  // that NaN logits count for no number; a token that is NaN itself is counted apart.
  int rank = 0;
  const float above = at == 0.0f ? bits_f32(1u) : bits_f32(f32_bits(at) + (at > 0.0f ? 1 : -1));  // of +infinity a NaN: none is above
  // exp(x - m) = 2^(x L - m L), L = log2 e.  With m L in two parts, of which the second is left out of every term, one
  // fused step gives an exponent that is off by its own rounding alone; from 2^20 on the second part is not small, and the
  // difference comes first.
  constexpr float L = 1.44269504088896340736f;
  const float zero_l = zero * L, low = fabsf(zero) < 0x1p20f ? __builtin_fmaf(zero, L, -zero_l) : 0.0f;
  float sum = 0.0f, dot = 0.0f;
  auto pass = [&](auto exponent) __attribute__((always_inline)) {
#pragma unroll
    for (int q = 0; q < NV; ++q) {
      const float least = (v0 + q * (int)blockDim.x + 1) * VEC - shift <= tok ? at : above;
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const float x = value(q * VEC + i);
        const float d = exponent(x);
        const float e = __builtin_amdgcn_exp2f(d);
        sum += e;
        dot = __builtin_fmaf(e, fmaxf(d, -1000.0f), dot);  // nothing times infinity adds nothing
        rank += __builtin_popcountll(__ballot(x >= least));
      }
      __builtin_amdgcn_sched_barrier(0);  // ahead of its vector's turn, an unpacked value takes a register
    }
  };
  if (fabsf(zero) < 0x1p20f) pass([&](float x) __attribute__((always_inline)) { return __builtin_fmaf(x, L, -zero_l); });
  else pass([&](float x) __attribute__((always_inline)) { return (x - zero) * L; });
  const int begin = stretch * (int)blockDim.x * EACH - shift, end = begin + (int)blockDim.x * EACH;
  if (named && at != at) {  // behind every number and the NaNs before it
    rank = 0;
    for (int i = begin + (int)threadIdx.x; i < end; i += blockDim.x) {
      const bool in = (unsigned)i < (unsigned)a.n;
      const float x = in ? lp_load<DT>(base, i) : NAN;
      rank += __builtin_popcountll(__ballot(in && (x == x || i < tok)));
    }
  }
  sum = lp_wave_sum(sum), dot = lp_wave_sum(dot);
  // back to sums of exp(d) and exp(d) d: max is finite, or they are 0 or NaN
  dot = (dot - low * sum) * 0.69314718055994530942f;
  const float by = __builtin_amdgcn_exp2f(-low);
  if (lane == 0) wave_sum[wave] = sum * by, wave_dot[wave] = dot * by, wave_rank[wave] = (float)rank;  // at most 2^20
  // list what reaches the bound; of -infinities alone, which all do, nothing
  if (a.top && max > -INFINITY && __any(top >= bound)) {
#pragma unroll
    for (int r = 0; r < EACH; ++r) {
      const float x = value(r);
      if (x >= bound) {
        const int i = (v0 + r / VEC * (int)blockDim.x) * VEC - shift + r % VEC;
        const int o = (unsigned)i < (unsigned)a.n ? atomicAdd(&listed, 1) : kLpList;
        if (o < kLpList) list[o] = lp_entry(lp_key(x), i);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  }
  __syncthreads();
  const int c = listed;
  const int held = (end < a.n ? end : a.n) - (begin > 0 ? begin : 0);  // elements of the stretch; fewer than top end its list
  const bool in_turn = c > kLpList || c < (held < a.top ? held : a.top);
  sum = lp_row_sum(w16 < waves ? wave_sum[w16] : 0.0f);
  dot = lp_row_sum(w16 < waves ? wave_dot[w16] : 0.0f);
  rank = (int)lp_row_sum(w16 < waves ? wave_rank[w16] : 0.0f);
  if (stretch == 0 && named && wave == 0) {
    const int before = (tok + shift) % VEC, i = tok - before + lane;  // in the token's vector
    rank += __builtin_popcountll(__ballot(lane < before && i >= 0 && lp_load<DT>(base, i < 0 ? 0 : i) == at));
    if (at == -INFINITY && VEC - shift <= tok) rank -= shift;  // what the first vector holds before the row
  }
  const bool whole = a.stretches == 1;
  if (threadIdx.x == 0) {
    if (whole) lp_write(a, row, max, sum, dot, rank, at, named);
    else a.parts[blockIdx.x] = LpPart{max, sum, dot, rank};
  }
  if (!a.top) return;
  const float log_sum = logf(sum);
  auto place = [&](int at_place, lp_u64 entry) __attribute__((always_inline)) {
    if (whole) {
      a.top_ids[row * a.top + at_place] = (int)~(unsigned)entry;
      a.top_logprobs[row * a.top + at_place] = (lp_unkey((unsigned)(entry >> 32)) - max) - log_sum;
    } else {
      a.lists[(int64_t)blockIdx.x * a.top + at_place] = entry;
    }
  };
  if (!in_turn) {  // eight lanes an entry
    for (int i = threadIdx.x >> 3; i < c; i += blockDim.x >> 3) {
      const lp_u64 mine = list[i];
      int before = 0;
#pragma unroll 8
      for (int o = lane & 7; o < c; o += 8) before += list[o] > mine;
      float all = (float)before;
      all += xor1(all);
      all += xor2(all);
      all += xor4(all);
      if ((lane & 7) == 0 && (int)all < a.top) place((int)all, mine);
    }
    for (int i = c + (int)threadIdx.x; i < a.top; i += blockDim.x) place(i, 0);
    return;
  }
  // one after another, read again: the largest entry below the last one; 0 where the stretch has no more elements
  lp_u64 last = ~0ull;
  for (int j = 0; j < a.top; ++j) {
    lp_u64 mine = 0;
#pragma unroll 8
    for (int i = begin + (int)threadIdx.x; i < end; i += blockDim.x) {
      const lp_u64 entry = (unsigned)i < (unsigned)a.n ? lp_entry(lp_key(lp_load<DT>(base, i)), i) : 0;
      mine = entry < last && entry > mine ? entry : mine;
    }
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) {
      const lp_u64 o = __shfl_xor(mine, m);
      mine = o > mine ? o : mine;
    }
    __syncthreads();
    if (lane == 0) best[wave] = mine;
    __syncthreads();
    for (int w = 0; w < waves; ++w) mine = best[w] > mine ? best[w] : mine;
    last = mine;
    if (threadIdx.x == 0) place(j, last);
  }
}

// The stretches of a row, a workgroup each.
template <int DT>
__global__ void __launch_bounds__(kLpJoin) logprob_join(LpArgs a) {
  const int64_t row = blockIdx.x;
  const LpPart* parts = a.parts + row * a.stretches;
  const lp_u64* from = a.lists + row * a.stretches * a.top;
  __shared__ lp_u64 lists[kLpStretches * kLpTop], near[kLpList], bound;
  __shared__ int nears, full;
  const int listed = a.stretches * a.top;
  for (int i = threadIdx.x; i < listed; i += kLpJoin) lists[i] = from[i];
  const bool deep = a.top >= a.stretches;
  if (threadIdx.x == 0) nears = full = 0, bound = deep ? ~0ull : 1;
  const int lane = threadIdx.x & 63;  // a stretch each
  LpPart p{-INFINITY, 0.0f, 0.0f, 0};
  if (lane < a.stretches) p = parts[lane];
  const float max = lp_wave_max(p.max);
  const float d = p.max - max, by = p.max == -INFINITY ? 1.0f : expf(d);  // of -infinities alone the sums are 0, or NaN
  const float sum = lp_wave_sum(p.sum * by);
  const float dot = lp_wave_sum(p.max == -INFINITY ? 0.0f : (p.dot + p.sum * fmaxf(d, -1000.0f)) * by);
  const int rank = (int)lp_wave_sum((float)p.rank);  // whole numbers of at most 2^20
  if (threadIdx.x == 0) {
    const int tok = a.tokens[row];
    const bool named = (unsigned)tok < (unsigned)a.n;
    const float at = named ? lp_load<DT>((const char*)a.logits + row * a.ld * (DT == TGM_F32 ? 4 : 2), tok) : 0.0f;
    lp_write(a, row, max, sum, dot, rank, at, named);
  }
  const float log_sum = logf(sum);
  auto place = [&](int before, lp_u64 mine) __attribute__((always_inline)) {
    a.top_ids[row * a.top + before] = (int)~(unsigned)mine;
    a.top_logprobs[row * a.top + before] = (lp_unkey((unsigned)(mine >> 32)) - max) - log_sum;
  };
  // A bound that `top` entries reach, or 1 (0 is no entry): the top-th largest of the lists' first entries, or the least of
  // the q-th entries of those that have so many, as all but the last list do where nothing is masked.
  __syncthreads();
  const int q = deep ? (a.top + a.stretches - 2) / (a.stretches - 1) : 1;
  if ((int)threadIdx.x < a.stretches && a.top) {
    const lp_u64 mine = lists[threadIdx.x * a.top + q - 1];
    if (deep) {
      if (mine) atomicMin(&bound, mine), atomicAdd(&full, 1);
    } else {
      int before = 0;
#pragma unroll 4
      for (int s = 0; s < a.stretches; ++s) before += lists[s * a.top] > mine;
      if (mine && before == a.top - 1) bound = mine;
    }
  }
  __syncthreads();
  const lp_u64 least = deep && full * q < a.top ? 1 : bound;
  for (int i = threadIdx.x; i < listed; i += kLpJoin)
    if (lists[i] >= least) {
      const int o = atomicAdd(&nears, 1);
      if (o < kLpList) near[o] = lists[i];
    }
  __syncthreads();
  const int c = nears;
  if (c <= kLpList) {  // eight lanes an entry, as above
    for (int i = threadIdx.x >> 3; i < c; i += kLpJoin >> 3) {
      const lp_u64 mine = near[i];
      int before = 0;
#pragma unroll 8
      for (int o = lane & 7; o < c; o += 8) before += near[o] > mine;
      float all = (float)before;
      all += xor1(all);
      all += xor2(all);
      all += xor4(all);
      if ((lane & 7) == 0 && (int)all < a.top) place((int)all, mine);
    }
    return;
  }
  for (int i = threadIdx.x; i < listed; i += kLpJoin) {
    const lp_u64 mine = lists[i];
    if (mine < least) continue;
    const int own = i / a.top;
    int before = i - own * a.top;
    for (int s = 0; s < a.stretches && before < a.top; ++s) {
      if (s == own) continue;
      int low = 0, high = a.top;  // entries of list s before mine
      while (low < high) {
        const int mid = (low + high) / 2;
        if (lists[s * a.top + mid] > mine) low = mid + 1;
        else high = mid;
      }
      before += low;
    }
    if (before < a.top) place(before, mine);
  }
}

struct LpSizes {
  int each, threads, stretches;
  int64_t lists, bytes;
};
// Threads of a workgroup and stretches of a row: one where a row fits it, short ones where few rows do not.
static LpSizes lp_sizes(int64_t rows, int64_t vocab, int64_t dtype, int64_t top) {
  const int vec = dtype == TGM_F32 ? 4 : 8;
  const int64_t vectors = (vocab + 2 * vec - 2) / vec;  // at most, by the alignment of the row
  LpSizes z;
  z.each = dtype != TGM_F32 && rows >= 512 ? 64 : 32;
  const int64_t need = (vectors + z.each / vec - 1) / (z.each / vec);  // threads for one stretch
  const int most = 32 * kLpMost / z.each;
  z.threads = need >= most ? most : (int)((need + 63) / 64 * 64);
  if (need > most) {
    for (z.threads = 512; z.threads < most; z.threads *= 2) {
      const int64_t stretches = (need + z.threads - 1) / z.threads;
      if (stretches <= kLpStretches && rows * stretches * z.threads <= 256 * 1024) break;
    }
  }
  z.stretches = (int)((need + z.threads - 1) / z.threads);
  z.lists = (rows * z.stretches * (int64_t)sizeof(LpPart) + 255) / 256 * 256;
  z.bytes = z.stretches == 1 ? 0 : z.lists + rows * z.stretches * top * 8;
  return z;
}

template <int DT>
static void lp_launch(const LpArgs& a, int64_t rows, const LpSizes& z, hipStream_t st) {
  const dim3 grid((unsigned)(rows * z.stretches)), block(z.threads);
  if constexpr (DT != TGM_F32) {
    if (z.each == 64) hipLaunchKernelGGL((logprob_rows<DT, 64>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((logprob_rows<DT, 32>), grid, block, 0, st, a);
  } else {
    hipLaunchKernelGGL((logprob_rows<DT, 32>), grid, block, 0, st, a);
  }
  if (z.stretches > 1) hipLaunchKernelGGL((logprob_join<DT>), dim3((unsigned)rows), dim3(kLpJoin), 0, st, a);
}

static int lp_check(int64_t dtype, int64_t rows, int64_t vocab, int64_t top) {
  TGM_CHECK_ARG(dtype == TGM_F32 || dtype == TGM_F16 || dtype == TGM_BF16, "logits must be f32, f16 or bf16");
  TGM_CHECK_ARG(rows >= 0 && rows < (1ll << 24), "invalid row count");
  TGM_CHECK_ARG(vocab > 0 && vocab <= (1 << 20), "the vocabulary must hold 1 to 2^20 tokens");
  TGM_CHECK_ARG(top >= 0 && top <= kLpTop && top <= vocab, "top must be 0 to %d tokens of the vocabulary", kLpTop);
  return TGM_OK;
}

}  // namespace tgm

using namespace tgm;

extern "C" int64_t tgm_log_probs_workspace(int64_t rows, int64_t vocab, int64_t dtype, int64_t top) {
  clear_error();
  return lp_check(dtype, rows, vocab, top) == TGM_OK ? lp_sizes(rows, vocab, dtype, top).bytes : 0;
}

extern "C" int tgm_log_probs(const void* logits, int64_t dtype, int64_t rows, int64_t vocab, int64_t ld, const int32_t* tokens,
                             int64_t top, float* logprobs, int32_t* ranks, float* entropy, int32_t* top_ids,
                             float* top_logprobs, void* workspace, int64_t workspace_bytes, void* stream) {
  clear_error();
  if (const int status = lp_check(dtype, rows, vocab, top); status != TGM_OK) return status;
  TGM_CHECK_ARG((ld >= vocab && ld < (1ll << 36)) || rows <= 1, "the row stride is less than a row, or too large");
  if (rows == 0) return TGM_OK;
  TGM_CHECK_ARG(logits && tokens && logprobs && ranks && entropy && (!top || (top_ids && top_logprobs)), "null operand");
  TGM_CHECK_ARG((uintptr_t)logits % dtype_size((int)dtype) == 0, "misaligned logits");
  const LpSizes z = lp_sizes(rows, vocab, dtype, top);
  TGM_CHECK_ARG(rows * z.stretches < (1ll << 31), "too many rows");
  TGM_CHECK_ARG(!z.bytes || (workspace && workspace_bytes >= z.bytes && ((uintptr_t)workspace & 15) == 0),
                "workspace too small or misaligned");
  LpArgs a;
  a.logits = logits, a.ld = ld, a.n = (int)vocab, a.top = (int)top, a.stretches = z.stretches, a.tokens = tokens;
  a.logprobs = logprobs, a.ranks = ranks, a.entropy = entropy, a.top_ids = top_ids, a.top_logprobs = top_logprobs;
  a.parts = (LpPart*)workspace, a.lists = (lp_u64*)((char*)workspace + (z.bytes ? z.lists : 0));
  const hipStream_t st = (hipStream_t)stream;
  if (dtype == TGM_F32) lp_launch<TGM_F32>(a, rows, z, st);
  else if (dtype == TGM_F16) lp_launch<TGM_F16>(a, rows, z, st);
  else lp_launch<TGM_BF16>(a, rows, z, st);
  return launch_status("tgm_log_probs");
}
