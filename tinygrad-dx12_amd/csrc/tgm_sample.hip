// Token sampling (tgm_sample): temperature, top-k, top-p and min-p, and a draw by inversion.
//
// Weights.  w = exp((x - max) / temperature) is computed in 64 bits (a table of 2^(j / 64) and five terms of the
// exponential series) and held as a whole number of 2^-F, F = 62 - ceil(log2 n) and at most 50: sums of whole numbers do
// not depend on their order, so histograms may be built with atomics and every pass agrees with every other to the last
// unit, and n weights of at most 2^F fit 63 bits.
//
// The kept set.  Sorted by value and, within a value, by index, what top-k and top-p keep is a prefix: all keys above a
// cut, and the first `ties` indices at the cut.  Both cuts are found by descending a radix tree over order-preserving
// keys of the logits (counts for top-k, masses for top-p), without a sort.
#include <math.h>

#include "../../include/tgm_serving.h"
#include "tgm_common.h"

namespace tgm {

constexpr int kSampThreads = 1024, kSampWaves = 16, kSampBins = 2048;
typedef unsigned long long samp_u64;
typedef unsigned samp_u32x4 __attribute__((ext_vector_type(4)));

struct SampleArgs {
  const void* logits;
  int64_t ld;
  int n, fbits, vec;
  const float* u;
  const float* temperature;
  const int32_t* top_k;
  const float* top_p;
  const float* min_p;
  int32_t* tokens;
};

template <int DT>
struct SampKey {
  static constexpr int BITS = DT == TGM_F32 ? 32 : 16;
  static constexpr int LEVELS = DT == TGM_F32 ? 3 : 2;
  // first bit and width of each level's digit, from the top
  __device__ static constexpr int shift(int level) { return DT == TGM_F32 ? (level == 0 ? 21 : (level == 1 ? 10 : 0)) : (level == 0 ? 8 : 0); }
  __device__ static constexpr int width(int level) { return DT == TGM_F32 ? (level == 2 ? 10 : 11) : 8; }
};

// A logit and its key: ascending with the value, equal for equal values (-0 is +0).
template <int DT>
__device__ __forceinline__ float samp_value(const void* row, int64_t i) {
  return load_f32(row, DT, i) + 0.0f;
}
template <int DT>
__device__ __forceinline__ unsigned samp_key(float x) {
  if constexpr (DT == TGM_F32) {
    const unsigned b = f32_bits(x);
    return b ^ ((b >> 31) ? 0xFFFFFFFFu : 0x80000000u);
  } else {
    const unsigned b = DT == TGM_BF16 ? f32_bits(x) >> 16 : (unsigned)__builtin_bit_cast(unsigned short, (_Float16)x);
    return b ^ ((b >> 15) ? 0xFFFFu : 0x8000u);
  }
}
template <int DT>
__device__ __forceinline__ float samp_unkey(unsigned k) {
  if constexpr (DT == TGM_F32) return bits_f32(k ^ ((k >> 31) ? 0x80000000u : 0xFFFFFFFFu));
  const unsigned b = (k ^ ((k >> 15) ? 0x8000u : 0xFFFFu)) & 0xFFFFu;
  if constexpr (DT == TGM_BF16) return bits_f32(b << 16);
  else return (float)__builtin_bit_cast(_Float16, (unsigned short)b);
}

// 2^y for y <= 0 as a whole number of 2^-F (and in 64 bits): 2^y = 2^e T[j] exp(r), 64 y = 64 e + j + 64 r / ln 2.
struct SampExp {
  const double* table;
  double max, rate;  // rate = log2(e) / temperature
  int fbits;
  __device__ __forceinline__ double log2w(float x) const { return x == max ? 0.0 : ((double)x - max) * rate; }
  __device__ __forceinline__ double weight(float x) const {
    const double y = fmax(log2w(x), -1100.0) * 64.0;
    const double k = __builtin_rint(y);
    const int ki = (int)k;
    const double r = (y - k) * (0.69314718055994530942 / 64.0);
    double p = 1.0 / 120.0;
    p = __builtin_fma(p, r, 1.0 / 24.0);
    p = __builtin_fma(p, r, 1.0 / 6.0);
    p = __builtin_fma(p, r, 0.5);
    p = __builtin_fma(p, r, 1.0);
    p = __builtin_fma(p, r, 1.0);
    return __builtin_ldexp(p * table[ki & 63], ki >> 6);
  }
  // w 2^F is at most 2^50: adding 2^52 rounds it to a whole number, which the sum's low 52 bits hold
  __device__ __forceinline__ samp_u64 fix(double w) const {
    const double s = __builtin_ldexp(w, fbits) + 0x1p52;
    return __builtin_bit_cast(samp_u64, s) & 0xFFFFFFFFFFFFFull;
  }
};

template <int DT, typename F>
__device__ __forceinline__ void samp_each(const void* row, int n, int vec, F f) {
  constexpr int V = DT == TGM_F32 ? 4 : 8;
  int done = 0;
  if (vec) {
    const int nv = n / V;
    for (int i = threadIdx.x; i < nv; i += kSampThreads) {
      const samp_u32x4 w = ((const samp_u32x4*)row)[i];
#pragma unroll
      for (int e = 0; e < V; ++e) f(samp_value<DT>(&w, e), i * V + e);
    }
    done = nv * V;
  }
  for (int i = done + threadIdx.x; i < n; i += kSampThreads) f(samp_value<DT>(row, i), i);
}

__device__ __forceinline__ samp_u64 samp_shfl_up(samp_u64 v, int d) {
  const unsigned lo = __shfl_up((unsigned)v, d, 64), hi = __shfl_up((unsigned)(v >> 32), d, 64);
  return ((samp_u64)hi << 32) | lo;
}
__device__ __forceinline__ samp_u64 samp_wave_sum(samp_u64 v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const unsigned lo = __shfl_xor((unsigned)v, o, 64), hi = __shfl_xor((unsigned)(v >> 32), o, 64);
    v += ((samp_u64)hi << 32) | lo;
  }
  return v;
}

struct SampShared {
  samp_u64 mass[kSampBins];
  unsigned count[kSampBins];
  double table[64];
  samp_u64 wave_mass[kSampWaves];
  unsigned wave_count[kSampWaves];
  float fmax_[kSampWaves];
  int idx[kSampWaves];
  // results of a step
  unsigned bin, before_count;
  samp_u64 before_mass;
  int found;
  int64_t at;
};

// Bins from the top: the first non-empty one with which the running count reaches `count` (by_mass 0) or the running
// mass reaches `goal` (by_mass 1); what lies above it goes to before_*.
__device__ __forceinline__ void samp_find(SampShared& sh, int bins, bool by_mass, unsigned goal_count, double goal) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  unsigned c[2] = {0, 0};
  samp_u64 m[2] = {0, 0};
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int b = bins - 1 - (2 * tid + e);
    if (b >= 0) {
      c[e] = sh.count[b];
      m[e] = sh.mass[b];
    }
  }
  unsigned pc = c[0] + c[1];
  samp_u64 pm = m[0] + m[1];
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const unsigned uc = __shfl_up(pc, o, 64);
    const samp_u64 um = samp_shfl_up(pm, o);
    if (lane >= o) {
      pc += uc;
      pm += um;
    }
  }
  if (lane == 63) {
    sh.wave_count[wave] = pc;
    sh.wave_mass[wave] = pm;
  }
  if (tid == 0) sh.found = 0;
  __syncthreads();
  pc -= c[0] + c[1];
  pm -= m[0] + m[1];
  for (int w = 0; w < wave; ++w) {
    pc += sh.wave_count[w];
    pm += sh.wave_mass[w];
  }
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int b = bins - 1 - (2 * tid + e);
    const bool reached = by_mass ? (double)pm >= goal : pc >= goal_count;
    const bool reaches = by_mass ? (double)(pm + m[e]) >= goal : pc + c[e] >= goal_count;
    // the first one of a descent by mass is taken even when the goal is 0
    if (b >= 0 && c[e] > 0 && reaches && (!reached || (by_mass && pc == 0))) {
      sh.bin = (unsigned)b;
      sh.before_count = pc;
      sh.before_mass = pm;
      sh.found = 1;
    }
    pc += c[e];
    pm += m[e];
  }
  __syncthreads();
}

// One workgroup a row: every pass reads the row again (from the caches, as a rule).
template <int DT>
__global__ void __launch_bounds__(kSampThreads) sample_row(const SampleArgs A) {
  __shared__ SampShared sh;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n = A.n;
  const int64_t r = blockIdx.x;
  const char* row = (const char*)A.logits + r * A.ld * (DT == TGM_F32 ? 4 : 2);
  if (tid < 64) {  // 2^(j / 64) by the series of exp(j ln 2 / 64)
    const double x = tid * (0.69314718055994530942 / 64.0);
    double t = 1.0, s = 1.0;
    for (int i = 1; i < 20; ++i) {
      t *= x / i;
      s += t;
    }
    sh.table[tid] = s;
  }
  // the first maximum
  float best = -INFINITY;
  int bi = n;
  samp_each<DT>(row, n, A.vec, [&](float x, int i) {
    if (x > best || (x == best && x > -INFINITY && i < bi)) {
      best = x;
      bi = i;
    }
  });
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const float ob = __shfl_xor(best, o, 64);
    const int oi = __shfl_xor(bi, o, 64);
    if (ob > best || (ob == best && oi < bi)) {
      best = ob;
      bi = oi;
    }
  }
  if (lane == 0) {
    sh.fmax_[wave] = best;
    sh.idx[wave] = bi;
  }
  __syncthreads();
  for (int w = 0; w < kSampWaves; ++w)
    if (sh.fmax_[w] > best || (sh.fmax_[w] == best && sh.idx[w] < bi)) {
      best = sh.fmax_[w];
      bi = sh.idx[w];
    }
  const float temp = A.temperature[r];
  if (!(temp > 0.f) || bi >= n) {  // greedy, or nothing to take
    if (tid == 0) A.tokens[r] = bi < n ? bi : 0;
    return;
  }
  const SampExp ex{sh.table, (double)best, 1.4426950408889634074 / (double)temp, A.fbits};

  unsigned cut = 0, ties = 0xFFFFFFFFu;  // kept: keys above cut, and the first `ties` indices at it
  // A descent: by count over everything, by mass over what the count kept.
  auto descend = [&](bool by_mass, unsigned goal_count, double share) __attribute__((always_inline)) {
    unsigned prefix = 0;
    unsigned above_count = 0;
    samp_u64 above = 0;
    double goal = 0;
    for (int level = 0; level < SampKey<DT>::LEVELS; ++level) {
      const int sft = SampKey<DT>::shift(level), width = SampKey<DT>::width(level), bins = 1 << width;
      for (int i = tid; i < bins; i += kSampThreads) {
        sh.mass[i] = 0;
        sh.count[i] = 0;
      }
      __syncthreads();
      samp_each<DT>(row, n, A.vec, [&](float x, int) {
        if (!(x > -INFINITY)) return;
        const unsigned k = samp_key<DT>(x);
        if (level > 0 && (k >> (sft + width)) != prefix) return;
        if (by_mass && (k < cut || (k == cut && ties != 0xFFFFFFFFu))) return;
        const unsigned d = (k >> sft) & (bins - 1);
        atomicAdd(&sh.count[d], 1u);
        if (by_mass) atomicAdd(&sh.mass[d], ex.fix(ex.weight(x)));
      });
      __syncthreads();
      if (by_mass && ties != 0xFFFFFFFFu && tid == 0 && (level == 0 || (cut >> (sft + width)) == prefix)) {
        const unsigned d = (cut >> sft) & (bins - 1);  // the kept ones of those at the cut
        sh.count[d] += ties;
        sh.mass[d] += (samp_u64)ties * ex.fix(ex.weight(samp_unkey<DT>(cut)));
      }
      __syncthreads();
      if (by_mass && level == 0) {  // the mass of all that is left
        samp_u64 s = 0;
        for (int i = tid; i < bins; i += kSampThreads) s += sh.mass[i];
        s = samp_wave_sum(s);
        if (lane == 0) sh.wave_mass[wave] = s;
        __syncthreads();
        s = 0;
        for (int w = 0; w < kSampWaves; ++w) s += sh.wave_mass[w];
        goal = share * (double)s;
        __syncthreads();
      }
      samp_find(sh, bins, by_mass, goal_count - above_count, goal - (double)above);
      if (!sh.found) return;  // fewer than asked for: all stay
      prefix = (prefix << width) | sh.bin;
      above_count += sh.before_count;
      above += sh.before_mass;
      __syncthreads();
    }
    unsigned keep;
    if (by_mass) {
      const double w = (double)ex.fix(ex.weight(samp_unkey<DT>(prefix)));
      const double need = goal - (double)above;
      const double q = w > 0 ? ceil(need / w) : 0.0;
      keep = q < 1.0 ? 1u : (q > 2147483647.0 ? 0x7FFFFFFFu : (unsigned)q);
      if (prefix == cut && keep > ties) keep = ties;
    } else {
      keep = goal_count - above_count;
    }
    cut = prefix;
    ties = keep;
  };
  const int top_k = A.top_k ? A.top_k[r] : 0;
  if (top_k > 0 && top_k < n) descend(false, (unsigned)top_k, 0.0);
  const float top_p = A.top_p ? A.top_p[r] : 1.f;
  if (top_p < 1.f) descend(true, 0u, (double)top_p);
  const double min_p = A.min_p ? (double)A.min_p[r] : 0.0;

  // the index at which the ties at the cut end: segments of whole waves' steps, a wave each
  const int seg = ((n + kSampWaves - 1) / kSampWaves + 1023) / 1024 * 1024;
  int tie_end = n;
  if (ties != 0xFFFFFFFFu) {
    unsigned cnt = 0;
    for (int64_t i = (int64_t)wave * seg + lane; i < min((int64_t)n, (int64_t)(wave + 1) * seg); i += 64)
      cnt += samp_key<DT>(samp_value<DT>(row, i)) == cut;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) cnt += __shfl_xor(cnt, o, 64);
    if (lane == 0) sh.wave_count[wave] = cnt;
    if (tid == 0) sh.at = n;
    __syncthreads();
    unsigned before = 0;
    for (int w = 0; w < wave; ++w) before += sh.wave_count[w];
    if (before < ties && before + cnt >= ties) {  // one wave at most: it walks its segment
      unsigned left = ties - before;
      for (int64_t i0 = (int64_t)wave * seg; i0 < min((int64_t)n, (int64_t)(wave + 1) * seg); i0 += 64) {
        const int64_t i = i0 + lane;
        const samp_u64 hit = __ballot(i < n && samp_key<DT>(samp_value<DT>(row, i)) == cut);
        const unsigned c = __popcll(hit);
        if (c >= left) {
          const unsigned rank = __popcll(hit & ((2ull << lane) - 1ull));
          if (((hit >> lane) & 1) && rank == left) sh.at = i + 1;
          break;
        }
        left -= c;
      }
    }
    __syncthreads();
    tie_end = (int)sh.at;
  }

  // the draw: weights of the kept in the vocabulary's order; u = 0 takes the first of any weight
  const double u = A.u[r] > 0.f ? (double)A.u[r] : 0.0;
  auto kept = [&](float x, int64_t i) __attribute__((always_inline)) -> samp_u64 {
    if (!(x > -INFINITY)) return 0;
    const unsigned k = samp_key<DT>(x);
    if (k < cut || (k == cut && i >= tie_end)) return 0;
    const double w = ex.weight(x);
    if (!(w >= min_p)) return 0;
    return u > 0 ? ex.fix(w) : (samp_u64)(w > 0);
  };
  int64_t lo = 0, len = seg;  // the waves' segments of a range: first of 1 / 16 of the row, then of the chosen one
  samp_u64 target = 0;
  for (int pass = 0; pass < 2; ++pass) {
    samp_u64 s = 0;
    const int64_t i0 = lo + wave * len, i1 = min((int64_t)n, i0 + len);
    for (int64_t i = i0 + lane; i < i1; i += 64) s += kept(samp_value<DT>(row, i), i);
    s = samp_wave_sum(s);
    __syncthreads();
    if (lane == 0) sh.wave_mass[wave] = s;
    __syncthreads();
    if (pass == 0) {
      samp_u64 total = 0;
      for (int w = 0; w < kSampWaves; ++w) total += sh.wave_mass[w];
      const double t = u * (double)total;
      target = t < (double)total ? (samp_u64)t : total;
      if (target >= total) target = total - 1;  // u of 1 and more: the last
    }
    int w = 0;
    while (w < kSampWaves - 1 && target >= sh.wave_mass[w]) target -= sh.wave_mass[w++];
    lo += w * len;
    len /= kSampWaves;
  }
  if (wave == 0) {  // one wave scans the chosen 1 / 256 of the row
    samp_u64 base = 0;
    const int64_t end = min((int64_t)n, lo + seg / kSampWaves);
    for (int64_t i0 = lo; i0 < end; i0 += 64) {
      const int64_t i = i0 + lane;
      samp_u64 s = i < end ? kept(samp_value<DT>(row, i), i) : 0;
      const samp_u64 own = s;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const samp_u64 up = samp_shfl_up(s, o);
        if (lane >= o) s += up;
      }
      const samp_u64 hit = __ballot(base + s > target && own > 0);
      if (hit) {
        if (lane == __ffsll((unsigned long long)hit) - 1) A.tokens[r] = (int32_t)i;
        break;
      }
      const unsigned lo32 = __shfl((unsigned)s, 63, 64), hi32 = __shfl((unsigned)(s >> 32), 63, 64);
      base += ((samp_u64)hi32 << 32) | lo32;
    }
  }
}

}  // namespace tgm

using namespace tgm;

extern "C" int64_t tgm_sample_workspace(int64_t rows, int64_t vocab, int64_t dtype) { return 0; }

extern "C" int tgm_sample(const void* logits, int64_t dtype, int64_t rows, int64_t vocab, int64_t ld, const float* u,
                          const float* temperature, const int32_t* top_k, const float* top_p, const float* min_p,
                          int32_t* tokens, void* workspace, int64_t workspace_bytes, void* stream) {
  clear_error();
  TGM_CHECK_ARG(dtype == TGM_F32 || dtype == TGM_F16 || dtype == TGM_BF16, "logits must be f32, f16 or bf16");
  TGM_CHECK_ARG(rows >= 0 && rows < (1ll << 24), "invalid row count");
  TGM_CHECK_ARG(vocab > 0 && vocab <= (1 << 20), "the vocabulary must hold 1 to 2^20 tokens");
  TGM_CHECK_ARG(ld >= vocab || rows <= 1, "the row stride is less than a row");
  if (rows == 0) return TGM_OK;
  TGM_CHECK_ARG(logits && u && temperature && tokens, "null operand");
  SampleArgs a;
  a.logits = logits, a.ld = ld, a.n = (int)vocab;
  int lg = 0;
  while ((1ll << lg) < vocab) ++lg;
  a.fbits = 62 - lg > 50 ? 50 : 62 - lg;
  a.vec = ((uintptr_t)logits & 15) == 0 && (ld * dtype_size((int)dtype)) % 16 == 0;
  a.u = u, a.temperature = temperature, a.top_k = top_k, a.top_p = top_p, a.min_p = min_p, a.tokens = tokens;
  const hipStream_t st = (hipStream_t)stream;
  const dim3 grid((unsigned)rows);
  if (dtype == TGM_F32) hipLaunchKernelGGL(sample_row<TGM_F32>, grid, dim3(kSampThreads), 0, st, a);
  else if (dtype == TGM_F16) hipLaunchKernelGGL(sample_row<TGM_F16>, grid, dim3(kSampThreads), 0, st, a);
  else hipLaunchKernelGGL(sample_row<TGM_BF16>, grid, dim3(kSampThreads), 0, st, a);
  return launch_status("tgm_sample");
}
