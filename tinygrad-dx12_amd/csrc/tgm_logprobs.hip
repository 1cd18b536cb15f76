// Log probabilities of given tokens, their ranks, the entropy, and the likeliest tokens (tgm_log_probs).
//
// With m the largest logit, d_i = x_i - m, S = sum exp(d_i) and T = sum exp(d_i) d_i:
//
//   log p_i = d_i - log S        entropy = -sum p_i log p_i = log S - T / S
//
// A workgroup reads a stretch of a row into registers, 32 logits a thread, and everything else comes from there: the
// largest, then S, T and the token's rank, then the likeliest tokens.  Those are looked for among the logits that reach a
// bound which enough of them are sure to reach: the n-th largest of the waves' largest logits, or, with more tokens than
// waves, the least over the waves of their q-th largest thread's.  Of independent logits a few dozen reach it; they are
// listed in LDS and each counts those before it.  Where more than the list holds do (many equal ones), the tokens are taken
// one after another instead.
//
// A row that is longer than a stretch, or that would leave compute units idle, takes several, and a second launch joins
// them: S and T scale by exp(m_stretch - m), and each listed token counts those of the other lists before it.
#include <math.h>

#include "../../include/tgm_serving.h"
#include "tgm_common.h"
#include "tgm_lanes.h"

namespace tgm {

constexpr int kLpMost = 1024, kLpEach = 32, kLpTop = 64, kLpList = 512, kLpJoin = 256;
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

template <int DT>
__global__ void __launch_bounds__(kLpMost) logprob_rows(LpArgs a) {
  constexpr int SIZE = DT == TGM_F32 ? 4 : 2, VEC = 16 / SIZE, NV = kLpEach / VEC;
  __shared__ float wave_a[16], wave_b[16], wave_c[16];
  __shared__ int wave_i[16];
  __shared__ lp_u64 list[kLpList];
  __shared__ lp_u64 best[16];
  __shared__ int listed;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
  const int64_t row = blockIdx.x / a.stretches;
  const int stretch = blockIdx.x % a.stretches;
  const char* base = (const char*)a.logits + row * a.ld * SIZE;
  const int tok = a.tokens[row];
  const bool named = (unsigned)tok < (unsigned)a.n;
  const float at = named ? lp_load<DT>(base, tok) : 0.0f;
  // whole aligned vectors: the first may begin before the row and the last end behind it, in its 16 bytes
  const int shift = (int)((uintptr_t)base % 16) / SIZE;
  const lp_u32x4* vectors = (const lp_u32x4*)(base - shift * SIZE);
  const int count = (a.n + shift + VEC - 1) / VEC;
  const int v0 = stretch * (int)blockDim.x * NV + (int)threadIdx.x;
  lp_u32x4 raw[NV];
#pragma unroll
  for (int q = 0; q < NV; ++q) {
    const int v = v0 + q * (int)blockDim.x;
    raw[q] = v < count ? __builtin_nontemporal_load(vectors + v) : lp_u32x4{};
  }
  auto index = [&](int r) __attribute__((always_inline)) { return (v0 + r / VEC * (int)blockDim.x) * VEC - shift + r % VEC; };
  auto raw_value = [&](int r) __attribute__((always_inline)) {
    const lp_u32x4 v = raw[r / VEC];
    if constexpr (DT == TGM_F32) return bits_f32(v[r % VEC]);
    const unsigned pair = v[r % VEC / 2];
    if constexpr (DT == TGM_BF16) return bits_f32(r % 2 ? pair & 0xFFFF0000u : pair << 16);
    return (float)__builtin_bit_cast(_Float16, (unsigned short)(r % 2 ? pair >> 16 : pair));
  };
  // -infinity where there is no element
  float x[kLpEach];
  float top = -INFINITY;
#pragma unroll
  for (int r = 0; r < kLpEach; ++r) {
    x[r] = (unsigned)index(r) < (unsigned)a.n ? raw_value(r) : -INFINITY;
    top = fmaxf(top, x[r]);
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
  if (lane == 0) wave_a[wave] = wave_top, wave_b[wave] = reach;
  __syncthreads();
  float max = -INFINITY, bound = INFINITY;
  for (int w = 0; w < waves; ++w) {
    const float t = wave_a[w];
    max = fmaxf(max, t);
    if (a.top > waves) {
      bound = fminf(bound, wave_b[w]);
    } else {  // the top-th largest
      int before = 0;
      for (int o = 0; o < waves; ++o) before += wave_a[o] > t || (wave_a[o] == t && o < w);
      bound = before == a.top - 1 ? t : bound;
    }
  }
  const float zero = max == -INFINITY ? 0.0f : max;
  float sum = 0.0f, dot = 0.0f;
  int rank = 0;
#pragma unroll
  for (int r = 0; r < kLpEach; ++r) {
    const float d = x[r] - zero;
    const float e = __builtin_amdgcn_exp2f(d * 1.44269504088896340736f);
    sum += e;
    dot = __builtin_fmaf(e, fmaxf(d, -1000.0f), dot);  // nothing times infinity adds nothing
    rank += x[r] > at || (x[r] == at && (unsigned)index(r) < (unsigned)tok);
  }
  sum = lp_wave_sum(sum), dot = lp_wave_sum(dot);
  const int ranked = (int)lp_wave_sum((float)rank);  // at most 2048
  if (lane == 0) wave_c[wave] = sum, wave_i[wave] = ranked;
  __syncthreads();
  if (lane == 0) wave_b[wave] = dot;
  // list what reaches the bound
  if (a.top && __any(top >= bound)) {
#pragma unroll
    for (int r = 0; r < kLpEach; ++r)
      if (x[r] >= bound && (unsigned)index(r) < (unsigned)a.n) {
        const int o = atomicAdd(&listed, 1);
        if (o < kLpList) list[o] = lp_entry(lp_key(x[r]), index(r));
      }
  }
  __syncthreads();
  sum = 0.0f, dot = 0.0f, rank = 0;
  for (int w = 0; w < waves; ++w) sum += wave_c[w], dot += wave_b[w], rank += wave_i[w];
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
  const int c = listed;
  if (c >= a.top && c <= kLpList) {
    for (int i = threadIdx.x; i < c; i += blockDim.x) {
      const lp_u64 mine = list[i];
      int before = 0;
      for (int o = 0; o < c; ++o) before += list[o] > mine;
      if (before < a.top) place(before, mine);
    }
    return;
  }
  // one after another: the largest entry below the last one; 0 where the stretch has no more elements
  lp_u64 last = ~0ull;
  for (int j = 0; j < a.top; ++j) {
    lp_u64 mine = 0;
#pragma unroll
    for (int r = 0; r < kLpEach; ++r) {
      const int i = index(r);
      const lp_u64 entry = (unsigned)i < (unsigned)a.n ? lp_entry(lp_key(x[r]), i) : 0;
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
  const lp_u64* lists = a.lists + row * a.stretches * a.top;
  float max = -INFINITY;
  for (int s = 0; s < a.stretches; ++s) max = fmaxf(max, parts[s].max);
  float sum = 0.0f, dot = 0.0f;
  int rank = 0;
  for (int s = 0; s < a.stretches; ++s) {
    const LpPart p = parts[s];
    rank += p.rank;
    if (p.max == -INFINITY) {  // a sum of 0, or NaN
      sum += p.sum;
    } else {
      const float d = p.max - max, by = expf(d);
      sum += p.sum * by;
      dot += (p.dot + p.sum * fmaxf(d, -1000.0f)) * by;
    }
  }
  if (threadIdx.x == 0) {
    const int tok = a.tokens[row];
    const bool named = (unsigned)tok < (unsigned)a.n;
    const float at = named ? lp_load<DT>((const char*)a.logits + row * a.ld * (DT == TGM_F32 ? 4 : 2), tok) : 0.0f;
    lp_write(a, row, max, sum, dot, rank, at, named);
  }
  const float log_sum = logf(sum);
  for (int i = threadIdx.x; i < a.stretches * a.top; i += kLpJoin) {
    const lp_u64 mine = lists[i];
    if (mine == 0) continue;  // its stretch had fewer
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
    if (before >= a.top) continue;
    a.top_ids[row * a.top + before] = (int)~(unsigned)mine;
    a.top_logprobs[row * a.top + before] = (lp_unkey((unsigned)(mine >> 32)) - max) - log_sum;
  }
}

struct LpSizes {
  int threads, stretches;
  int64_t lists, bytes;
};
// Threads of a workgroup and stretches of a row.
static LpSizes lp_sizes(int64_t rows, int64_t vocab, int64_t dtype, int64_t top) {
  const int vec = dtype == TGM_F32 ? 4 : 8, each = kLpEach / vec;
  const int64_t vectors = (vocab + 2 * vec - 2) / vec;  // at most, by the alignment of the row
  LpSizes z;
  const int64_t need = (vectors + each - 1) / each;  // threads for one stretch
  z.threads = need >= kLpMost ? kLpMost : (int)((need + 63) / 64 * 64);
  z.stretches = (int)((need + z.threads - 1) / z.threads);
  z.lists = (rows * z.stretches * (int64_t)sizeof(LpPart) + 255) / 256 * 256;
  z.bytes = z.stretches == 1 ? 0 : z.lists + rows * z.stretches * top * 8;
  return z;
}

template <int DT>
static void lp_launch(const LpArgs& a, int64_t rows, const LpSizes& z, hipStream_t st) {
  hipLaunchKernelGGL((logprob_rows<DT>), dim3((unsigned)(rows * z.stretches)), dim3(z.threads), 0, st, a);
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
  TGM_CHECK_ARG(ld >= vocab || rows <= 1, "the row stride is less than a row");
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
