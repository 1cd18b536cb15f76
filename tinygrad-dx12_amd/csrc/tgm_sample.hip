// Token sampling (tgm_sample): temperature, top-k, top-p and min-p, and a draw by inversion.
//
// Weights.  w = exp((x - max) / temperature) is computed in 64 bits (a table of 2^(j / 64) and five terms of the
// exponential series) and held as a whole number of 2^-F, F = 62 - ceil(log2 n) and at most 50: sums of whole numbers do
// not depend on their order, so histograms may be built with atomics and every pass agrees with every other to the last
// unit, and n weights of at most 2^F fit 63 bits.
//
// The kept set.  Sorted by value and, within a value, by index, what top-k, top-p and min-p keep is a prefix, so one cut
// has to be found, and no row is sorted.  Three launches, a row in several workgroups for the first two:
//
//   sample_bins    counts and masses in bins of 1/40 of a power of two of the weight, from the largest down; weights
//                  that round to 0 are left out (they are never drawn but for u = 0)
//   sample_sift    finds the bin that the cut falls into.  Few tokens down to it (the rule with top-k): they are
//                  listed.  Many: those of the cut's bin alone are listed, and the masses above it summed over segments
//                  of the vocabulary.
//   sample_draw    a workgroup a row: sorts the list in LDS, settles the cut exactly, and draws: over the sorted list,
//                  or over the segments and then inside one of them.
//
// A list holds 2048 tokens.  A row that needs a longer one (thousands of equal logits at the cut, a top_k of thousands),
// and one with u = 0, is settled inside sample_draw by descending a radix tree over order-preserving keys of the logits
// (sample_descend), which needs no list.
#include <math.h>

#include "../../include/tgm_serving.h"
#include "tgm_common.h"

namespace tgm {

constexpr int kSampThreads = 1024, kSampWaves = 16, kSampBins = 2048;
typedef unsigned long long samp_u64;
typedef unsigned samp_u32x4 __attribute__((ext_vector_type(4)));

constexpr int kSampList = 2048, kSampSegs = 1024, kSampMostChunks = 16;
constexpr double kSampPerBin = 40.0;  // bins per power of two of a weight: 2047 of them reach 2^-51

struct SampPlan {  // of a row, from sample_sift
  samp_u64 total, above;  // mass of all, and above the listed tokens
  unsigned mode, bin;
  int top_k, pad;  // 0: no cut
};
enum SampMode { kSampListAll = 0, kSampListBin = 1, kSampDescend = 2 };

struct SampleArgs {
  const void* logits;
  int64_t ld;
  int n, fbits, vec;
  int chunks, chunk, seg, segs;  // workgroups of a row, tokens of each (a multiple of seg), tokens and count of segments
  const float* u;
  const float* temperature;
  const int32_t* top_k;
  const float* top_p;
  const float* min_p;
  int32_t* tokens;
  // workspace, per row
  samp_u64* mass;   // [chunks][bins]
  samp_u64* list;   // [kSampList], unordered
  samp_u64* segsum; // [segs]
  SampPlan* plan;
  unsigned* count;  // [chunks][bins]
  unsigned* listed;
  float* max;
};

// 2^(j / 64)
struct SampTable {
  double v[64];
  constexpr SampTable() : v() {
    for (int j = 0; j < 64; ++j) {  // the series of exp(j ln 2 / 64)
      const double x = j * (0.69314718055994530942 / 64.0);
      double t = 1.0, s = 0.0;
      double term[24] = {};
      for (int i = 0; i < 24; ++i) {
        term[i] = t;
        t = t * x / (i + 1);
      }
      for (int i = 23; i >= 0; --i) s += term[i];  // the small ones first
      v[j] = s;
    }
  }
};
__device__ const SampTable samp_table{};

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
  // bins of 1 / 40 of a power of two, descending with x; kSampBins - 1 for weights that round to 0
  __device__ __forceinline__ int bin(double y) const {
    const double b = y * -kSampPerBin;
    return b < (double)(kSampBins - 1) ? (int)b : kSampBins - 1;
  }
  __device__ __forceinline__ double weight(float x) const { return weight_of(log2w(x)); }
  __device__ __forceinline__ double weight_of(double lw) const {
    const double y = fmax(lw, -1100.0) * 64.0;
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

// f(value, index) over tokens first .. last - 1 of a row, in no order (first a multiple of 8).
template <int DT, int THREADS, typename F>
__device__ __forceinline__ void samp_each(const void* row, int first, int last, int vec, F f) {
  constexpr int V = DT == TGM_F32 ? 4 : 8;
  int done = first;
  if (vec) {
    const int v1 = last / V;
    for (int i = first / V + threadIdx.x; i < v1; i += THREADS) {
      const samp_u32x4 w = ((const samp_u32x4*)row)[i];
#pragma unroll
      for (int e = 0; e < V; ++e) f(samp_value<DT>(&w, e), i * V + e);
    }
    if (v1 * V > done) done = v1 * V;
  }
  for (int i = done + threadIdx.x; i < last; i += THREADS) f(samp_value<DT>(row, i), i);
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
  samp_u64 wave_mass[kSampWaves];
  unsigned wave_count[kSampWaves];
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

// A whole row by one workgroup of 1024 threads without a list: the cuts by descent, then the draw.  Every pass reads the
// row again.
template <int DT>
__device__ void sample_descend(const SampleArgs& A, SampShared& sh, const void* row, int64_t r, const SampExp& ex) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n = A.n;
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
      samp_each<DT, kSampThreads>(row, 0, n, A.vec, [&](float x, int) {
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
      if (total == 0) {  // min_p above 1
        if (tid == 0) A.tokens[r] = 0;
        return;
      }
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

// The row's largest logit (-inf: none), in every thread.
template <int DT, int THREADS>
__device__ __forceinline__ float samp_max(const void* row, int n, int vec, float* part) {
  float best = -INFINITY;
  samp_each<DT, THREADS>(row, 0, n, vec, [&](float x, int) { best = fmaxf(best, x); });  // NaN: the other operand
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) best = fmaxf(best, __shfl_xor(best, o, 64));
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = best;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < THREADS / 64; ++w) best = fmaxf(best, part[w]);
  return best;
}

__device__ __forceinline__ void samp_load_table(double* table) {
  if (threadIdx.x < 64) table[threadIdx.x] = samp_table.v[threadIdx.x];
}

// Grid (chunks, rows).  Every workgroup of a row finds the row's maximum for itself: reading a row from the L2 is
// cheaper than a launch.
constexpr int kBinThreads = 512;
template <int DT>
__global__ void __launch_bounds__(kBinThreads) sample_bins(const SampleArgs A) {
  __shared__ samp_u64 mass[kSampBins];
  __shared__ unsigned count[kSampBins];
  __shared__ double table[64];
  __shared__ float part[kBinThreads / 64];
  const int64_t r = blockIdx.y;
  const int c = blockIdx.x, tid = threadIdx.x;
  const char* row = (const char*)A.logits + r * A.ld * (DT == TGM_F32 ? 4 : 2);
  samp_load_table(table);
  for (int i = tid; i < kSampBins; i += kBinThreads) {
    mass[i] = 0;
    count[i] = 0;
  }
  const float best = samp_max<DT, kBinThreads>(row, A.n, A.vec, part);
  if (c == 0 && tid == 0) {
    A.max[r] = best;
    A.listed[r] = 0;
  }
  const float temp = A.temperature[r];
  if (!(temp > 0.f) || !(best > -INFINITY)) return;
  const SampExp ex{table, (double)best, 1.4426950408889634074 / (double)temp, A.fbits};
  samp_each<DT, kBinThreads>(row, min(c * A.chunk, A.n), min((c + 1) * A.chunk, A.n), A.vec, [&](float x, int) {
    if (!(x > -INFINITY)) return;
    const double y = ex.log2w(x);
    const int b = ex.bin(y);
    if (b == kSampBins - 1) return;
    atomicAdd(&count[b], 1u);
    atomicAdd(&mass[b], ex.fix(ex.weight_of(y)));
  });
  __syncthreads();
  const int64_t o = (r * A.chunks + c) * kSampBins;
  for (int i = tid; i < kSampBins; i += kBinThreads) {
    A.mass[o + i] = mass[i];
    A.count[o + i] = count[i];
  }
}

// Exclusive prefix of v over the workgroup, and its total.
template <int THREADS, typename T>
__device__ __forceinline__ T samp_scan(T v, T* part, T& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  T s = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    T up;
    if constexpr (sizeof(T) == 8) up = samp_shfl_up(s, o);
    else up = __shfl_up(s, o, 64);
    if (lane >= o) s += up;
  }
  __syncthreads();  // the last scan's partials have been read
  if (lane == 63) part[wave] = s;
  __syncthreads();
  T before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 64; ++w) {
    before += w < wave ? part[w] : 0;
    total += part[w];
  }
  return before + s - v;
}

// A listed token: descending order of these is descending by value, ascending by index.
__device__ __forceinline__ samp_u64 samp_entry(unsigned key, int i) { return ((samp_u64)key << 32) | (unsigned)~i; }

// Grid (chunks, rows).
template <int DT>
__global__ void __launch_bounds__(kBinThreads) sample_sift(const SampleArgs A) {
  constexpr int BPT = kSampBins / kBinThreads;
  __shared__ double table[64];
  __shared__ samp_u64 mpart[kBinThreads / 64];
  __shared__ unsigned cpart[kBinThreads / 64];
  __shared__ unsigned kbin, pbin, ksize, psize, pcount;
  __shared__ samp_u64 pabove;
  const int64_t r = blockIdx.y;
  const int c = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const char* row = (const char*)A.logits + r * A.ld * (DT == TGM_F32 ? 4 : 2);
  const float temp = A.temperature[r], best = A.max[r];
  if (!(temp > 0.f) || !(best > -INFINITY)) return;
  samp_load_table(table);
  if (tid == 0) kbin = pbin = kSampBins;
  samp_u64 m[BPT], msum = 0;
  unsigned n[BPT], nsum = 0;
  const int64_t o = r * A.chunks * kSampBins + BPT * tid;
#pragma unroll
  for (int e = 0; e < BPT; ++e) m[e] = n[e] = 0;
  for (int i = 0; i < A.chunks; ++i)
#pragma unroll
    for (int e = 0; e < BPT; ++e) {
      m[e] += A.mass[o + (int64_t)i * kSampBins + e];
      n[e] += A.count[o + (int64_t)i * kSampBins + e];
    }
#pragma unroll
  for (int e = 0; e < BPT; ++e) {
    msum += m[e];
    nsum += n[e];
  }
  samp_u64 total;
  unsigned all;
  samp_u64 mb = samp_scan<kBinThreads>(msum, mpart, total);
  unsigned nb = samp_scan<kBinThreads>(nsum, cpart, all);
  int k = A.top_k ? A.top_k[r] : 0;
  if (k < 0 || k >= A.n || (unsigned)k >= all) k = 0;  // whatever is not counted weighs nothing
  const double p = A.top_p ? (double)A.top_p[r] : 1.0;
  const double goal = p * (double)total;
#pragma unroll
  for (int e = 0; e < BPT; ++e) {
    if (k > 0 && nb < (unsigned)k && nb + n[e] >= (unsigned)k) {
      kbin = BPT * tid + e;
      ksize = nb + n[e];
    }
    if (p < 1.0 && n[e] > 0 && (nb == 0 || (double)mb < goal) && ((double)(mb + m[e]) >= goal)) {
      // the first such bin: with a goal of 0 and less the first one of all
      pbin = BPT * tid + e;
      psize = nb + n[e];
      pcount = n[e];
      pabove = mb;
    }
    mb += m[e];
    nb += n[e];
  }
  __syncthreads();
  SampPlan plan{total, 0, kSampListAll, kSampBins - 2, k, 0};
  if (!(A.u[r] > 0.f)) {
    plan.mode = kSampDescend;
  } else if (k > 0) {
    plan.bin = kbin;
    if (ksize > kSampList) plan.mode = kSampDescend;
  } else if (p < 1.0 && pbin < kSampBins) {
    plan.bin = pbin;
    if (psize > kSampList) {
      plan.mode = pcount > kSampList ? kSampDescend : kSampListBin;
      plan.above = pabove;
    }
  } else if (all > kSampList) {  // everything is kept
    plan.mode = kSampListBin;
    plan.bin = kSampBins - 1;
    plan.above = total;
  }
  if (c == 0 && tid == 0) A.plan[r] = plan;
  if (plan.mode == kSampDescend) return;
  const SampExp ex{table, (double)best, 1.4426950408889634074 / (double)temp, A.fbits};
  auto list = [&](bool hit, float x, int i) __attribute__((always_inline)) {
    const samp_u64 hits = __ballot(hit);
    if (hits == 0) return;
    unsigned at = 0;
    const int first = __ffsll((unsigned long long)hits) - 1;
    if (lane == first) at = atomicAdd(&A.listed[r], (unsigned)__popcll(hits));
    at = __shfl(at, first, 64) + (unsigned)__popcll(hits & ((1ull << lane) - 1ull));
    if (hit && at < kSampList) A.list[r * kSampList + at] = samp_entry(samp_key<DT>(x), i);
  };
  const int begin = min(c * A.chunk, A.n), end = min((c + 1) * A.chunk, A.n);
  if (plan.mode == kSampListAll) {
    samp_each<DT, kBinThreads>(row, begin, end, A.vec,
                               [&](float x, int i) { list(x > -INFINITY && ex.bin(ex.log2w(x)) <= (int)plan.bin, x, i); });
    return;
  }
  const double min_p = A.min_p ? (double)A.min_p[r] : 0.0;
  for (int s = begin / A.seg + wave; s * A.seg < end; s += kBinThreads / 64) {
    samp_u64 sum = 0;
    for (int i0 = s * A.seg; i0 < min((s + 1) * A.seg, end); i0 += 64) {
      const int i = i0 + lane;
      const float x = i < end ? samp_value<DT>(row, i) : -INFINITY;
      bool in_bin = false;
      if (x > -INFINITY) {
        const double y = ex.log2w(x);
        const int b = ex.bin(y);
        in_bin = b == (int)plan.bin && b < kSampBins - 1;
        if (b < (int)plan.bin) {
          const double w = ex.weight_of(y);
          sum += w >= min_p ? ex.fix(w) : 0;
        }
      }
      list(in_bin, x, i);
    }
    sum = samp_wave_sum(sum);
    if (lane == 0) A.segsum[r * A.segs + s] = sum;
  }
}

// Bitonic sort of size (a power of two, at most 2048) entries in LDS by 1024 threads, descending.
__device__ __forceinline__ void samp_sort(samp_u64* v, int size) {
  for (int k = 2; k <= size; k <<= 1)
    for (int j = k >> 1; j > 0; j >>= 1) {
      __syncthreads();
      const int t = threadIdx.x;
      if (t < size / 2) {
        const int a = 2 * t - (t & (j - 1)), b = a + j;
        const samp_u64 x = v[a], y = v[b];
        if ((x < y) == ((a & k) == 0)) {
          v[a] = y;
          v[b] = x;
        }
      }
    }
  __syncthreads();
}

struct SampList {
  samp_u64 entry[kSampList], weight[kSampList], seg[kSampSegs];
};

template <int DT>
__global__ void __launch_bounds__(kSampThreads) sample_draw(const SampleArgs A) {
  __shared__ union {
    SampShared sh;
    SampList li;
  } u_;
  __shared__ double table[64];
  __shared__ samp_u64 part[kSampWaves];
  __shared__ unsigned kept_count;
  __shared__ int seg_at;
  __shared__ samp_u64 seg_left;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n = A.n;
  const int64_t r = blockIdx.x;
  const char* row = (const char*)A.logits + r * A.ld * (DT == TGM_F32 ? 4 : 2);
  const float temp = A.temperature[r], best = A.max[r];
  if (!(best > -INFINITY)) {  // nothing to take
    if (tid == 0) A.tokens[r] = 0;
    return;
  }
  if (!(temp > 0.f)) {  // the first maximum
    int at = n;
    samp_each<DT, kSampThreads>(row, 0, n, A.vec, [&](float x, int i) {
      if (x == best && i < at) at = i;
    });
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) at = min(at, __shfl_xor(at, o, 64));
    if (tid == 0) seg_at = n;
    __syncthreads();
    if (lane == 0) atomicMin(&seg_at, at);
    __syncthreads();
    if (tid == 0) A.tokens[r] = seg_at;
    return;
  }
  samp_load_table(table);
  if (tid == 0) kept_count = 0;
  const SampExp ex{table, (double)best, 1.4426950408889634074 / (double)temp, A.fbits};
  const SampPlan plan = A.plan[r];
  __syncthreads();
  if (plan.mode == kSampDescend) {
    sample_descend<DT>(A, u_.sh, row, r, ex);
    return;
  }
  SampList& li = u_.li;
  const int listed = min((int)A.listed[r], kSampList);
  int size = 64;
  while (size < listed) size <<= 1;
  for (int i = tid; i < size; i += kSampThreads) li.entry[i] = i < listed ? A.list[r * kSampList + i] : 0;
  samp_sort(li.entry, size);
  // weights in rank order (two ranks a thread), and what the cuts keep of them
  const double p = A.top_p ? (double)A.top_p[r] : 1.0, min_p = A.min_p ? (double)A.min_p[r] : 0.0;
  samp_u64 e[2], w[2];
  double wd[2];
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    const int i = 2 * tid + q;
    e[q] = i < size ? li.entry[i] : 0;
    const bool in = i < listed && (plan.top_k == 0 || i < plan.top_k);
    wd[q] = in ? ex.weight(samp_unkey<DT>((unsigned)(e[q] >> 32))) : -1.0;
    w[q] = in ? ex.fix(wd[q]) : 0;
  }
  samp_u64 sum;
  samp_u64 before = plan.above + samp_scan<kSampThreads>(w[0] + w[1], part, sum);
  const double goal = p * (double)(plan.top_k > 0 ? sum : plan.total);
  unsigned mine = 0;
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    const int i = 2 * tid + q;
    // in the mode of a listed bin at least one token lies above it
    const bool keep = wd[q] >= 0.0 && wd[q] >= min_p &&
                      (!(p < 1.0) || (double)before < goal || (i == 0 && plan.mode == kSampListAll));
    before += w[q];
    if (!keep) w[q] = 0;
    mine += keep;
    if (i < size) li.weight[i] = w[q];
    // next: the kept ones by index, so that the draw runs in the vocabulary's order
    if (i < size && plan.mode == kSampListAll) li.entry[i] = keep ? (((e[q] & 0xFFFFFFFFull) << 32) | (unsigned)(i + 1)) : 0;
  }
  const double u = (double)A.u[r];
  auto target_of = [&](samp_u64 total) __attribute__((always_inline)) -> samp_u64 {
    const double t = u * (double)total;
    const samp_u64 target = t < (double)total ? (samp_u64)t : total;
    return target >= total ? total - 1 : target;  // u of 1 and more: the last
  };
  if (plan.mode == kSampListAll) {
    samp_sort(li.entry, size);  // by ~index, descending: ascending indices first, dropped ones last
    samp_u64 x[2];
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const int i = 2 * tid + q;
      e[q] = i < size ? li.entry[i] : 0;
      x[q] = e[q] ? li.weight[(unsigned)e[q] - 1] : 0;
    }
    samp_u64 total;
    samp_u64 at = samp_scan<kSampThreads>(x[0] + x[1], part, total);
    if (total == 0) {  // min_p above 1
      if (tid == 0) A.tokens[r] = 0;
      return;
    }
    const samp_u64 target = target_of(total);
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      if (x[q] > 0 && at <= target && at + x[q] > target) A.tokens[r] = (int32_t)~(unsigned)(e[q] >> 32);
      at += x[q];
    }
    return;
  }
  // the segments' masses with the kept ones of the cut's bin
  if (mine) atomicAdd(&kept_count, mine);
  li.seg[tid] = tid < A.segs ? A.segsum[r * A.segs + tid] : 0;
  __syncthreads();
#pragma unroll
  for (int q = 0; q < 2; ++q)
    if (w[q]) atomicAdd(&li.seg[~(unsigned)e[q] / (unsigned)A.seg], w[q]);
  __syncthreads();
  const samp_u64 cut = kept_count ? li.entry[kept_count - 1] : ~0ull;  // the last one kept of the bin
  const samp_u64 own = li.seg[tid];
  samp_u64 total;
  const samp_u64 at = samp_scan<kSampThreads>(own, part, total);
  if (total == 0) {
    if (tid == 0) A.tokens[r] = 0;
    return;
  }
  const samp_u64 target = target_of(total);
  if (at <= target && at + own > target) {
    seg_at = tid;
    seg_left = target - at;
  }
  __syncthreads();
  if (wave > 0) return;
  samp_u64 base = 0;
  const int first = seg_at * A.seg, end = min(first + A.seg, n);
  for (int i0 = first; i0 < end; i0 += 64) {
    const int i = i0 + lane;
    const float x = i < end ? samp_value<DT>(row, i) : -INFINITY;
    samp_u64 s = 0;
    if (x > -INFINITY) {
      const double y = ex.log2w(x);
      const int b = ex.bin(y);
      const double wx = ex.weight_of(y);
      if (wx >= min_p && (b < (int)plan.bin || (b == (int)plan.bin && samp_entry(samp_key<DT>(x), i) >= cut))) s = ex.fix(wx);
    }
    const samp_u64 one = s;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const samp_u64 up = samp_shfl_up(s, o);
      if (lane >= o) s += up;
    }
    const samp_u64 hit = __ballot(one > 0 && base + s > seg_left);
    if (hit) {
      if (lane == __ffsll((unsigned long long)hit) - 1) A.tokens[r] = (int32_t)i;
      return;
    }
    const unsigned lo32 = __shfl((unsigned)s, 63, 64), hi32 = __shfl((unsigned)(s >> 32), 63, 64);
    base += ((samp_u64)hi32 << 32) | lo32;
  }
}

struct SampSizes {
  int chunks, chunk, seg, segs;
  int64_t mass, list, segsum, plan, count, listed, max, bytes;
};

static SampSizes samp_sizes(int64_t rows, int64_t vocab) {
  SampSizes z;
  z.seg = vocab <= 256 * kSampSegs ? 256 : 1024;
  z.segs = (int)((vocab + z.seg - 1) / z.seg);
  // two workgroups a CU, 2048 tokens each at least
  int64_t c = (512 + rows - 1) / rows;
  const int64_t most = (vocab + 2047) / 2048;
  c = c > most ? most : c;
  c = c > kSampMostChunks ? kSampMostChunks : c;
  z.chunk = (int)((vocab + c * z.seg - 1) / (c * z.seg)) * z.seg;
  z.chunks = (int)((vocab + z.chunk - 1) / z.chunk);
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t o = at;
    at += (bytes + 15) / 16 * 16;
    return o;
  };
  z.mass = take(rows * z.chunks * kSampBins * 8);
  z.list = take(rows * kSampList * 8);
  z.segsum = take(rows * z.segs * 8);
  z.plan = take(rows * (int64_t)sizeof(SampPlan));
  z.count = take(rows * z.chunks * kSampBins * 4);
  z.listed = take(rows * 4);
  z.max = take(rows * 4);
  z.bytes = at;
  return z;
}

template <int DT>
static void sample_launch(const SampleArgs& a, int64_t rows, hipStream_t st) {
  for (int64_t r0 = 0; r0 < rows; r0 += 65535) {  // a grid's second dimension
    SampleArgs b = a;
    const int64_t n = rows - r0 < 65535 ? rows - r0 : 65535;
    b.logits = (const char*)a.logits + r0 * a.ld * (DT == TGM_F32 ? 4 : 2);
    b.u += r0, b.temperature += r0, b.tokens += r0;
    if (b.top_k) b.top_k += r0;
    if (b.top_p) b.top_p += r0;
    if (b.min_p) b.min_p += r0;
    b.mass += r0 * a.chunks * kSampBins, b.count += r0 * a.chunks * kSampBins, b.list += r0 * kSampList;
    b.segsum += r0 * a.segs, b.plan += r0, b.listed += r0, b.max += r0;
    const dim3 grid((unsigned)a.chunks, (unsigned)n);
    hipLaunchKernelGGL(sample_bins<DT>, grid, dim3(kBinThreads), 0, st, b);
    hipLaunchKernelGGL(sample_sift<DT>, grid, dim3(kBinThreads), 0, st, b);
    hipLaunchKernelGGL(sample_draw<DT>, dim3((unsigned)n), dim3(kSampThreads), 0, st, b);
  }
}

}  // namespace tgm

using namespace tgm;

extern "C" int64_t tgm_sample_workspace(int64_t rows, int64_t vocab, int64_t dtype) {
  if (rows <= 0 || rows >= (1ll << 24) || vocab <= 0 || vocab > (1 << 20)) return 0;
  return samp_sizes(rows, vocab).bytes;
}

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
  const SampSizes z = samp_sizes(rows, vocab);
  TGM_CHECK_ARG(workspace && workspace_bytes >= z.bytes && ((uintptr_t)workspace & 15) == 0, "workspace too small or misaligned");
  SampleArgs a;
  a.logits = logits, a.ld = ld, a.n = (int)vocab;
  a.chunks = z.chunks, a.chunk = z.chunk, a.seg = z.seg, a.segs = z.segs;
  int lg = 0;
  while ((1ll << lg) < vocab) ++lg;
  a.fbits = 62 - lg > 50 ? 50 : 62 - lg;
  a.vec = ((uintptr_t)logits & 15) == 0 && (rows == 1 || (ld * dtype_size((int)dtype)) % 16 == 0);
  a.u = u, a.temperature = temperature, a.top_k = top_k, a.top_p = top_p, a.min_p = min_p, a.tokens = tokens;
  char* ws = (char*)workspace;
  a.mass = (samp_u64*)(ws + z.mass), a.list = (samp_u64*)(ws + z.list), a.segsum = (samp_u64*)(ws + z.segsum);
  a.plan = (SampPlan*)(ws + z.plan), a.count = (unsigned*)(ws + z.count), a.listed = (unsigned*)(ws + z.listed);
  a.max = (float*)(ws + z.max);
  const hipStream_t st = (hipStream_t)stream;
  if (dtype == TGM_F32) sample_launch<TGM_F32>(a, rows, st);
  else if (dtype == TGM_F16) sample_launch<TGM_F16>(a, rows, st);
  else sample_launch<TGM_BF16>(a, rows, st);
  return launch_status("tgm_sample");
}
