// Token sampling (tgm_sample): temperature, top-k, top-p and min-p, and a draw by inversion.
//
// Weights.  w = exp((x - max) / temperature) is computed in 64 bits (a table of 2^(j / 64) and five terms of the
// exponential series) and held as a whole number of 2^-F, F = 62 - ceil(log2 n) and at most 50: sums of whole numbers do
// not depend on their order, so histograms may be built with atomics and every pass agrees with every other to the last
// unit, and n weights of at most 2^F fit 63 bits.
//
// The kept set.  Sorted by value and, within a value, by index, what top-k, top-p and min-p keep is a prefix, so one cut
// has to be found, and no row is sorted.  Two launches:
//
//   sample_bins   (a row in several workgroups) counts and masses in bins of 1/40 of a power of two of the weight, from
//                 the largest down; weights that round to 0 are left out (they are never drawn but for u = 0)
//   sample_draw   (a workgroup a row) finds the bin that the cut falls into.  Few tokens down to it (the rule with
//                 top-k): it lists them in LDS, sorts them, settles the cut and draws among them.  Many: it lists those of
//                 the cut's bin alone; the bins above it give the kept mass of each workgroup's part of the vocabulary,
//                 which picks the part that the draw falls into, and only that part is weighed again.
//
// A list holds 2048 tokens.  A row that needs a longer one (thousands of equal logits at the cut, a top_k of thousands),
// and one with u = 0, is settled by descending a radix tree over order-preserving keys of the logits (sample_descend),
// which needs no list.
//
// What bounds it: one row of 32000 fp32 logits, every filter on, takes 18.7 us (6 + 13 in the two kernels), a chain of
// barriers and latencies in one workgroup; 64 rows of 131072 bf16 logits, top-p alone, take 50 (20 + 30): in sample_bins
// about 35 vector instructions a token, most of them in 64 bits, and two LDS atomics, in sample_draw a row's 256 KB through
// one CU.  The descent alone, one workgroup a row, took 63 and 270 us.
#include <math.h>

#include "../../include/tgm_serving.h"
#include "tgm_common.h"

namespace tgm {

constexpr int kCutThreads = 256;  // of sample_draw, 8 bins each
constexpr int kSampThreads = 1024, kSampWaves = 16, kSampBins = 2048;
typedef unsigned long long samp_u64;
typedef unsigned samp_u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned samp_u32x4 __attribute__((ext_vector_type(4)));
typedef samp_u64 samp_u64x2 __attribute__((ext_vector_type(2)));

constexpr int kSampList = 2048, kSampQueue = 2 * kSampList, kSampMostChunks = 16;
constexpr double kSampPerBin = 40.0;  // bins per power of two of a weight: 2047 of them reach 2^-51

struct SampleArgs {
  const void* logits;
  int64_t ld;
  int n, fbits;
  int chunks, chunk;  // workgroups of a row in sample_bins, tokens of each
  int rows;
  const float* u;
  const float* temperature;
  const int32_t* top_k;
  const float* top_p;
  const float* min_p;
  int32_t* tokens;
  // workspace, per row
  samp_u64* mass;   // [chunks][bins]
  unsigned* count;  // [chunks][bins]
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

template <int DT>
__device__ __forceinline__ float samp_load(const void* row, int64_t i) {
  if constexpr (DT == TGM_F16) return (float)((const _Float16*)row)[i];
  else return load_f32(row, DT, i);
}
// A logit and its key: ascending with the value, equal for equal values (-0 is +0).
template <int DT>
__device__ __forceinline__ float samp_value(const void* row, int64_t i) {
  return samp_load<DT>(row, i) + 0.0f;
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
  __device__ __forceinline__ SampExp(const double* t, float best, float temperature, int f)
      : table(t), max(best), rate(1.4426950408889634074 / (double)temperature), fbits(f) {}
  // the minimum turns inf - inf, a maximum of +inf itself, into 0
  __device__ __forceinline__ double log2w(float x) const { return fmin(((double)x - max) * rate, 0.0); }
  // bins of 1 / 40 of a power of two, descending with x; kSampBins - 1 for weights that round to 0
  __device__ __forceinline__ int bin(double y) const {
    const double b = y * -kSampPerBin;
    return b < (double)(kSampBins - 1) ? (int)b : kSampBins - 1;
  }
  // 2^(lw + more), lw above -1100
  __device__ __forceinline__ double power(double lw, int more) const {
    const double y = lw * 64.0;
    const double k = __builtin_rint(y);
    const int ki = (int)k;
    const double r = (y - k) * (0.69314718055994530942 / 64.0);
    double p = 1.0 / 120.0;
    p = __builtin_fma(p, r, 1.0 / 24.0);
    p = __builtin_fma(p, r, 1.0 / 6.0);
    p = __builtin_fma(p, r, 0.5);
    p = __builtin_fma(p, r, 1.0);
    p = __builtin_fma(p, r, 1.0);
    return __builtin_ldexp(p * table[ki & 63], (ki >> 6) + more);
  }
  __device__ __forceinline__ double weight(float x) const { return power(fmax(log2w(x), -1100.0), 0); }
  // w 2^F is at most 2^50: adding 2^52 rounds it to a whole number, which the sum's low 52 bits hold
  __device__ __forceinline__ samp_u64 fix(double w) const { return whole(__builtin_ldexp(w, fbits)); }
  __device__ __forceinline__ samp_u64 fix_of(double lw) const { return whole(power(lw, fbits)); }  // the same
  __device__ __forceinline__ samp_u64 whole(double w) const {
    return __builtin_bit_cast(samp_u64, w + 0x1p52) & 0xFFFFFFFFFFFFFull;
  }
};

// The first token of a row whose address is a multiple of 16.
template <int DT>
__device__ __forceinline__ int samp_aligned(const void* row) {
  return (int)((16u - ((unsigned)(uintptr_t)row & 15u)) & 15u) / (DT == TGM_F32 ? 4 : 2);
}

// f(value, index) over tokens first .. last - 1 of a row, in no order: whole 16-byte vectors where they are aligned, the
// few tokens before and behind one by one.
template <int DT, int THREADS, typename F>
__device__ __forceinline__ void samp_each(const void* row, int first, int last, F f) {
  constexpr int V = DT == TGM_F32 ? 4 : 8;
  const int al = samp_aligned<DT>(row);
  const int begin = first <= al ? al : first + (V - 1) - (first - al + V - 1) % V;  // first + 0 .. V - 1
  const int vectors = last > begin ? (last - begin) / V : 0;
  const samp_u32x4* v = (const samp_u32x4*)((const char*)row + (int64_t)begin * (16 / V));
#pragma unroll 8
  for (int i = threadIdx.x; i < vectors; i += THREADS) {
    const samp_u32x4 w = v[i];
#pragma unroll
    for (int e = 0; e < V; ++e) f(samp_value<DT>(&w, e), begin + i * V + e);
  }
  const int head = min(begin, last) - first;  // under V
  if ((int)threadIdx.x < head) f(samp_value<DT>(row, first + threadIdx.x), first + (int)threadIdx.x);
  const int tail = begin + vectors * V + (int)threadIdx.x;
  if (tail < last && begin < last) f(samp_value<DT>(row, tail), tail);
}

// Inclusive prefix sum over the wave by DPP moves alone: shifts within rows of 16, then the rows' totals.
template <int CTRL, int ROWS>
__device__ __forceinline__ samp_u64 samp_dpp(samp_u64 v) {
  const unsigned lo = __builtin_amdgcn_update_dpp(0, (int)(unsigned)v, CTRL, ROWS, 0xF, false);
  const unsigned hi = __builtin_amdgcn_update_dpp(0, (int)(unsigned)(v >> 32), CTRL, ROWS, 0xF, false);
  return ((samp_u64)hi << 32) | lo;
}
__device__ __forceinline__ samp_u64 samp_wave_scan(samp_u64 v) {
  v += samp_dpp<0x111, 0xF>(v);  // row_shr:1
  v += samp_dpp<0x112, 0xF>(v);
  v += samp_dpp<0x114, 0xF>(v);
  v += samp_dpp<0x118, 0xF>(v);
  v += samp_dpp<0x142, 0xA>(v);  // row_bcast:15 into rows 1 and 3
  v += samp_dpp<0x143, 0xC>(v);  // row_bcast:31 into rows 2 and 3
  return v;
}
__device__ __forceinline__ samp_u64 samp_lane(samp_u64 v, int lane) {
  const unsigned lo = __builtin_amdgcn_readlane((int)(unsigned)v, lane);
  const unsigned hi = __builtin_amdgcn_readlane((int)(unsigned)(v >> 32), lane);
  return ((samp_u64)hi << 32) | lo;
}
__device__ __forceinline__ samp_u64 samp_wave_sum(samp_u64 v) { return samp_lane(samp_wave_scan(v), 63); }

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
  unsigned pc = (unsigned)samp_wave_scan(c[0] + c[1]);
  samp_u64 pm = samp_wave_scan(m[0] + m[1]);
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
      samp_each<DT, kSampThreads>(row, 0, n, [&](float x, int) {
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
      const samp_u64 own = i < end ? kept(samp_value<DT>(row, i), i) : 0;
      const samp_u64 s = samp_wave_scan(own);
      const samp_u64 hit = __ballot(base + s > target && own > 0);
      if (hit) {
        if (lane == __ffsll((unsigned long long)hit) - 1) A.tokens[r] = (int32_t)i;
        break;
      }
      base += samp_lane(s, 63);
    }
  }
}

// The row's largest logit (-inf: none), in every thread.
template <int DT, int THREADS>
__device__ __forceinline__ float samp_max(const void* row, int n, float* part) {
  float best = -INFINITY;
  samp_each<DT, THREADS>(row, 0, n, [&](float x, int) { best = fmaxf(best, x); });  // NaN: the other operand
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

// Workgroups go to the 8 XCDs in turn: every workgroup of row r is number r mod 8 of its eight, so that a row stays in one
// XCD's L2.  Each finds the row's maximum for itself, which costs less than a launch.
constexpr int kBinThreads = 512;
template <int DT>
__global__ void __launch_bounds__(kBinThreads) sample_bins(const SampleArgs A) {
  __shared__ samp_u64 mass[kSampBins];
  __shared__ unsigned count[kSampBins];
  __shared__ double table[64];
  __shared__ float part[kBinThreads / 64];
  const int local = blockIdx.x / 8, c = local % A.chunks, tid = threadIdx.x;
  const int64_t r = (int64_t)(local / A.chunks) * 8 + blockIdx.x % 8;
  if (r >= A.rows) return;
  const char* row = (const char*)A.logits + r * A.ld * (DT == TGM_F32 ? 4 : 2);
  samp_load_table(table);
  for (int i = tid; i < kSampBins; i += kBinThreads) {
    mass[i] = 0;
    count[i] = 0;
  }
  const float best = samp_max<DT, kBinThreads>(row, A.n, part);
  if (c == 0 && tid == 0) A.max[r] = best;
  const float temp = A.temperature[r];
  if (!(temp > 0.f) || !(best > -INFINITY)) return;
  const SampExp ex(table, best, temp, A.fbits);
  samp_each<DT, kBinThreads>(row, min(c * A.chunk, A.n), min((c + 1) * A.chunk, A.n), [&](float x, int) {
    if (!(x > -INFINITY)) return;
    const double y = ex.log2w(x);
    const int b = ex.bin(y);
    if (b == kSampBins - 1) return;
    atomicAdd(&count[b], 1u);
    atomicAdd(&mass[b], ex.fix_of(y));
  });
  __syncthreads();
  const int64_t o = (r * A.chunks + c) * kSampBins;
  for (int i = tid; i < kSampBins; i += kBinThreads) {
    A.mass[o + i] = mass[i];
    A.count[o + i] = count[i];
  }
}

// Exclusive prefix of v over the workgroup's first WAVES waves (the others pass 0), and its total.
template <int WAVES>
__device__ __forceinline__ samp_u64 samp_scan(samp_u64 v, samp_u64* part, samp_u64& total) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const samp_u64 s = samp_wave_scan(v);
  __syncthreads();  // the last scan's partials have been read
  if (lane == 63 && wave < WAVES) part[wave] = s;
  __syncthreads();
  const samp_u64 p = samp_wave_scan(lane < WAVES ? part[lane] : 0);
  total = samp_lane(p, 63);
  const samp_u64 before = wave > 0 ? samp_lane(p, wave - 1) : 0;  // wave is uniform
  return before + s - v;
}

// A listed token: descending order of these is descending by value, ascending by index.
__device__ __forceinline__ samp_u64 samp_entry(unsigned key, int i) { return ((samp_u64)key << 32) | (unsigned)~i; }

// Sorts size (a power of two from 64 to 2048) entries in LDS by 1024 threads, descending; no two entries are alike.
// Up to 256 by counting the larger ones, several threads an entry, three barriers in all (64 entries take about 0.3 us
// where a network of 21 steps takes 2; 512 take 8, and by the network 4), beyond by a bitonic network whose steps within
// 128 entries need no barrier.  `rank` holds 256 counters.
__device__ __forceinline__ void samp_sort(samp_u64* v, unsigned* rank, int size) {
  const int t = threadIdx.x;
  if (size <= 256) {
    const int i = t & (size - 1), share = size * size / kSampThreads, j0 = (t / size) * share;
    if (t < size) rank[t] = 0;
    __syncthreads();
    const samp_u64 mine = v[i];
    unsigned n = 0;
#pragma unroll 4
    for (int j = j0; j < j0 + share; ++j) n += v[j] > mine;
    if (n) atomicAdd(&rank[i], n);
    __syncthreads();
    if (t < size) v[rank[t]] = mine;
    __syncthreads();
    return;
  }
  bool across = true;  // whether the last step, or what came before, went across waves
  for (int k = 2; k <= size; k <<= 1)
    for (int j = k >> 1; j > 0; j >>= 1) {
      // with j below 128 a wave's 64 pairs stay within 128 entries of its own
      if (across || j >= 128) __syncthreads();
      else {
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
      }
      across = j >= 128;
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
  samp_u64 entry[kSampList], weight[kSampList];
  unsigned rank[256];
};
// What sample_draw goes by: the cut's bin, and whether everything down to it is listed or that bin alone.
enum SampMode { kSampListAll = 0, kSampListBin = 1, kSampDescend = 2 };
struct SampCut {
  unsigned bin, size, count;  // tokens down to the bin, and in it
  samp_u64 above;             // mass above it
};

template <int DT>
__global__ void __launch_bounds__(kSampThreads) sample_draw(const SampleArgs A) {
  __shared__ union {
    SampShared sh;
    SampList li;
    struct {
      samp_u64 mass[kSampBins];
      unsigned count[kSampBins];
    } bins;
  } u_;
  __shared__ double table[64];
  __shared__ samp_u64 part[kSampWaves], chunk_mass[kSampMostChunks];
  __shared__ unsigned listed_, queued_, kept_count;
  __shared__ SampCut kcut, pcut, mcut, last;
  __shared__ int first_at;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), n = A.n;
  const int64_t r = blockIdx.x;
  const char* row = (const char*)A.logits + r * A.ld * (DT == TGM_F32 ? 4 : 2);
  const float temp = A.temperature[r], best = A.max[r];
  if (!(best > -INFINITY)) {  // nothing to take
    if (tid == 0) A.tokens[r] = 0;
    return;
  }
  if (!(temp > 0.f)) {  // the first maximum
    int at = n;
    samp_each<DT, kSampThreads>(row, 0, n, [&](float x, int i) {
      if (x == best && i < at) at = i;
    });
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) at = min(at, __shfl_xor(at, o, 64));
    if (tid == 0) first_at = n;
    __syncthreads();
    if (lane == 0) atomicMin(&first_at, at);
    __syncthreads();
    if (tid == 0) A.tokens[r] = first_at;
    return;
  }
  samp_load_table(table);
  if (tid == 0) {
    listed_ = queued_ = kept_count = 0;
    kcut.bin = pcut.bin = mcut.bin = last.bin = kSampBins;
  }
  if (tid < kSampMostChunks) chunk_mass[tid] = 0;
  const SampExp ex(table, best, temp, A.fbits);
  const double p = A.top_p ? (double)A.top_p[r] : 1.0, min_p = A.min_p ? (double)A.min_p[r] : 0.0;

  // all parts of the row, two bins a thread
  {
    samp_u64 m[2] = {0, 0};
    unsigned c[2] = {0, 0};
    const int64_t o = r * A.chunks * kSampBins + 2 * tid;
#pragma unroll
    for (int i0 = 0; i0 < kSampMostChunks; i0 += 8) {  // eight parts' loads in flight
      samp_u64x2 mi[8];
      samp_u32x2 ci[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        mi[i] = samp_u64x2{0, 0};
        ci[i] = samp_u32x2{0, 0};
        if (i0 + i < A.chunks) {
          mi[i] = *(const samp_u64x2*)(A.mass + o + (int64_t)(i0 + i) * kSampBins);
          ci[i] = *(const samp_u32x2*)(A.count + o + (int64_t)(i0 + i) * kSampBins);
        }
      }
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          m[q] += mi[i][q];
          c[q] += ci[i][q];
        }
    }
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      u_.bins.mass[2 * tid + q] = m[q];
      u_.bins.count[2 * tid + q] = c[q];
    }
  }
  __syncthreads();
  // prefixes and cuts: four waves with eight bins a thread (sixteen waves spend more on the scan than on its terms)
  samp_u64 m[8] = {}, msum = 0;
  unsigned c[8] = {}, csum = 0;
  if (tid < kCutThreads)
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      m[q] = u_.bins.mass[8 * tid + q];
      c[q] = u_.bins.count[8 * tid + q];
      msum += m[q];
      csum += c[q];
    }
  samp_u64 total, all;
  samp_u64 mb = samp_scan<kCutThreads / 64>(msum, part, total);
  unsigned nb = (unsigned)samp_scan<kCutThreads / 64>(csum, part, all);
  int k = A.top_k ? A.top_k[r] : 0;
  if (k < 0 || k >= n || (unsigned)k >= (unsigned)all) k = 0;  // what is not counted weighs nothing
  const double goal_p = p * (double)total;
  if (tid < kCutThreads) {
    // the bin of min_p: tokens above it weigh more, tokens below it less
    const int mbin = min_p > 0.0 ? (min_p >= 1.0 ? 0 : ex.bin(log2(min_p))) : kSampBins - 2;
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      const int b = 8 * tid + q;
      const SampCut here{(unsigned)b, nb + c[q], c[q], mb};
      if (k > 0 && nb < (unsigned)k && nb + c[q] >= (unsigned)k) kcut = here;
      // the first bin with which the mass reaches the goal, with a goal of 0 and less the first one of all
      if (p < 1.0 && c[q] > 0 && (nb == 0 || (double)mb < goal_p) && (double)(mb + m[q]) >= goal_p) pcut = here;
      if (b == mbin) mcut = here;
      mb += m[q];
      nb += c[q];
    }
  }
  __syncthreads();
  SampCut cut = mcut;  // everything that min_p leaves
  if (k > 0) {
    if (p < 1.0 || kcut.bin < cut.bin) cut = kcut;  // top-p goes by the mass that top-k left
  } else if (p < 1.0 && pcut.bin < cut.bin) {
    cut = pcut;
  }
  // up to 512 tokens are sorted faster than a part of the vocabulary is weighed, more of them slower
  int mode = kSampDescend;
  if (A.u[r] > 0.f) {
    if (cut.size <= (k > 0 ? kSampList : 512)) mode = kSampListAll;
    else if (k == 0 && cut.count <= kSampList) mode = kSampListBin;
  }
  if (mode == kSampDescend) {
    sample_descend<DT>(A, u_.sh, row, r, ex);
    return;
  }

  // The list.  Which tokens may belong to it is asked in 32 bits, with bounds half a bin too wide.
  SampList& li = u_.li;
  const double step = 1.0 / (kSampPerBin * ex.rate);
  const double low = (double)best - ((double)cut.bin + 1.5) * step;
  const double high = mode == kSampListAll ? (double)best : (double)best - ((double)cut.bin - 0.5) * step;
  // else bins near 32 bits' resolution, or bounds beyond their range (an infinite temperature: an infinite step)
  const bool narrow = step > (double)fabsf(best) * 0x1p-20 && fabs((double)best) < 0x1p120 && fabs(low) < 0x1p120 && fabs(high) < 0x1p120;
  const float middle = narrow ? (float)(0.5 * (low + high)) : 0.f, reach = narrow ? (float)(0.5 * (high - low) + step) : INFINITY;
  __syncthreads();  // the bins have been read
  auto consider = [&](float x, int i) __attribute__((always_inline)) {
    if (!(fabsf(x - middle) <= reach)) return;  // NaN too
    const int b = ex.bin(ex.log2w(x));
    if (b > (int)cut.bin || b >= kSampBins - 1 || (mode == kSampListBin && b != (int)cut.bin)) return;
    const unsigned at = atomicAdd(&listed_, 1u);
    if (at < kSampList) li.entry[at] = samp_entry(samp_key<DT>(x), i);
  };
  // Whole 16-byte vectors first: the few that may hold such a token are queued, and looked into by as many threads
  // afterwards (a test and a branch for each token of the row cost three times as much).
  constexpr int V = DT == TGM_F32 ? 4 : 8;
  const int al = min(samp_aligned<DT>(row), n), nv = (n - al) / V;
  const samp_u32x4* vectors = (const samp_u32x4*)(row + (int64_t)al * (16 / V));
  unsigned* queue = (unsigned*)li.weight;
#pragma unroll 8
  for (int i = tid; i < nv; i += kSampThreads) {
    const samp_u32x4 word = vectors[i];
    float d = INFINITY;  // the smallest distance; NaN does not count
#pragma unroll
    for (int q = 0; q < V; ++q) d = fminf(d, fabsf(samp_load<DT>(&word, q) - middle));
    if (d <= reach) {
      const unsigned at = atomicAdd(&queued_, 1u);
      if (at < kSampQueue) queue[at] = (unsigned)i;
    }
  }
  __syncthreads();
  const int queued = (int)queued_;
  if (queued <= kSampQueue) {
    for (int j = tid; j < queued * V; j += kSampThreads) {
      const int i = al + (int)queue[j / V] * V + j % V;
      consider(samp_value<DT>(row, i), i);
    }
  } else {
    for (int i = tid; i < nv * V; i += kSampThreads) consider(samp_value<DT>(row, al + i), al + i);
  }
  if (tid < al) consider(samp_value<DT>(row, tid), tid);
  if (al + nv * V + tid < n) consider(samp_value<DT>(row, al + nv * V + tid), al + nv * V + tid);
  if (mode == kSampListBin && wave < A.chunks) {  // kept mass of each part of the vocabulary, but for the cut's bin
    const samp_u64* part_mass = A.mass + (r * A.chunks + wave) * kSampBins;
    samp_u64 s = 0;
    for (int b = lane; b < (int)cut.bin; b += 64) s += part_mass[b];
    s = samp_wave_sum(s);
    if (lane == 0) chunk_mass[wave] = s;
  }
  __syncthreads();
  const int listed = min((int)listed_, kSampList);
  int size = 64;
  while (size < listed) size <<= 1;
  for (int i = listed + tid; i < size; i += kSampThreads) li.entry[i] = (samp_u64)(i + 1);  // below every token's
  samp_sort(li.entry, li.rank, size);
  // weights in rank order (two ranks a thread), and what the cuts keep of them
  samp_u64 e[2], w[2];
  double wd[2];
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    const int i = 2 * tid + q;
    e[q] = i < size ? li.entry[i] : 0;
    const bool in = i < listed && (k == 0 || i < k);
    wd[q] = in ? ex.weight(samp_unkey<DT>((unsigned)(e[q] >> 32))) : -1.0;
    w[q] = in ? ex.fix(wd[q]) : 0;
  }
  samp_u64 sum;
  samp_u64 before = samp_scan<kSampWaves>(w[0] + w[1], part, sum) + (mode == kSampListBin ? cut.above : 0);
  const double goal = p * (double)(k > 0 ? sum : total);
  unsigned mine = 0;
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    const int i = 2 * tid + q;
    // the first token of all stays whatever top-p asks for; a bin that is listed alone may be the first one
    const bool keep = wd[q] >= 0.0 && wd[q] >= min_p &&
                      (!(p < 1.0) || (double)before < goal || (i == 0 && (mode == kSampListAll || cut.size == cut.count)));
    before += w[q];
    if (!keep) w[q] = 0;
    mine += keep;
    if (i < size) li.weight[i] = w[q];
    // next: the kept ones by index, so that the draw runs in the vocabulary's order
    if (i < size && mode == kSampListAll) li.entry[i] = keep ? (((e[q] & 0xFFFFFFFFull) << 32) | (unsigned)(i + 1)) : (samp_u64)(i + 1);
  }
  const double u = (double)A.u[r];
  auto target_of = [&](samp_u64 sum_) __attribute__((always_inline)) -> samp_u64 {
    const double t = u * (double)sum_;
    const samp_u64 target = t < (double)sum_ ? (samp_u64)t : sum_;
    return target >= sum_ ? sum_ - 1 : target;  // u of 1 and more: the last
  };
  if (mode == kSampListAll) {
    samp_sort(li.entry, li.rank, size);  // by ~index, descending: ascending indices first, dropped ones last
    samp_u64 x[2];
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const int i = 2 * tid + q;
      e[q] = i < size ? li.entry[i] : 0;
      x[q] = e[q] >> 32 ? li.weight[(unsigned)e[q] - 1] : 0;
    }
    samp_u64 kept;
    samp_u64 at = samp_scan<kSampWaves>(x[0] + x[1], part, kept);
    if (kept == 0) {  // min_p above 1
      if (tid == 0) A.tokens[r] = 0;
      return;
    }
    const samp_u64 target = target_of(kept);
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      if (x[q] > 0 && at <= target && at + x[q] > target) A.tokens[r] = (int32_t)~(unsigned)(e[q] >> 32);
      at += x[q];
    }
    return;
  }
  // the part of the vocabulary that the draw falls into
  if (mine) atomicAdd(&kept_count, mine);
#pragma unroll
  for (int q = 0; q < 2; ++q)
    if (w[q]) atomicAdd(&chunk_mass[~(unsigned)e[q] / (unsigned)A.chunk], w[q]);
  __syncthreads();
  const samp_u64 lowest_kept = kept_count ? li.entry[kept_count - 1] : ~0ull;  // of the cut's bin
  samp_u64 kept = 0;
  for (int i = 0; i < A.chunks; ++i) kept += chunk_mass[i];
  if (kept == 0) {
    if (tid == 0) A.tokens[r] = 0;
    return;
  }
  samp_u64 left = target_of(kept);
  int ch = 0;
  while (ch < A.chunks - 1 && left >= chunk_mass[ch]) left -= chunk_mass[ch++];
  const int end = min((ch + 1) * A.chunk, n);
  const int begin = ch * A.chunk;
  // 8 neighbours a thread, from an aligned token at or before the part's first
  for (int first = begin - ((begin - al) & 7); first < end; first += 8 * kSampThreads) {
    samp_u64 x[8], s = 0;
    float v[8];
    const int i0 = first + 8 * tid;
    if (i0 >= begin && i0 + 8 <= end) {
      constexpr int W = 8 / V;
#pragma unroll
      for (int h = 0; h < W; ++h) {
        const samp_u32x4 word = *(const samp_u32x4*)(row + (int64_t)(i0 + h * V) * (16 / V));
#pragma unroll
        for (int q = 0; q < V; ++q) v[h * V + q] = samp_value<DT>(&word, q);
      }
    } else {
#pragma unroll
      for (int q = 0; q < 8; ++q) v[q] = i0 + q >= begin && i0 + q < end ? samp_value<DT>(row, i0 + q) : -INFINITY;
    }
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      x[q] = 0;
      if (v[q] > -INFINITY) {
        const double y = ex.log2w(v[q]);
        const int b = ex.bin(y);
        if (b < (int)cut.bin || (b == (int)cut.bin && samp_entry(samp_key<DT>(v[q]), i0 + q) >= lowest_kept)) x[q] = ex.fix_of(y);
      }
      s += x[q];
    }
    samp_u64 tile;
    samp_u64 at = samp_scan<kSampWaves>(s, part, tile);
    if (left < tile) {
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        if (x[q] > 0 && at <= left && at + x[q] > left) A.tokens[r] = i0 + q;
        at += x[q];
      }
      return;
    }
    left -= tile;
  }
}

struct SampSizes {
  int chunks, chunk;
  int64_t mass, count, max, bytes;
};

// Rows go in slabs, one after the other over one workspace (24 KB a part of a row).
constexpr int64_t kSampSlab = 2048;

static SampSizes samp_sizes(int64_t rows, int64_t vocab) {
  SampSizes z;
  if (rows > kSampSlab) rows = kSampSlab;
  // two workgroups a CU, 4096 tokens each at least: every part adds 24 KB to what sample_draw reads
  int64_t c = (512 + rows - 1) / rows;
  const int64_t most = (vocab + 4095) / 4096;
  c = c > most ? most : c;
  c = c > kSampMostChunks ? kSampMostChunks : c;
  z.chunk = (int)((vocab + c * 1024 - 1) / (c * 1024)) * 1024;
  z.chunks = (int)((vocab + z.chunk - 1) / z.chunk);
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t o = at;
    at += (bytes + 15) / 16 * 16;
    return o;
  };
  z.mass = take(rows * z.chunks * kSampBins * 8);
  z.count = take(rows * z.chunks * kSampBins * 4);
  z.max = take(rows * 4);
  z.bytes = at;
  return z;
}

template <int DT>
static void sample_launch(const SampleArgs& a, int64_t rows, hipStream_t st) {
  for (int64_t r0 = 0; r0 < rows; r0 += kSampSlab) {
    SampleArgs b = a;
    b.rows = (int)(rows - r0 < kSampSlab ? rows - r0 : kSampSlab);
    b.logits = (const char*)a.logits + r0 * a.ld * (DT == TGM_F32 ? 4 : 2);
    b.u += r0, b.temperature += r0, b.tokens += r0;
    if (b.top_k) b.top_k += r0;
    if (b.top_p) b.top_p += r0;
    if (b.min_p) b.min_p += r0;
    const unsigned eights = (unsigned)((b.rows + 7) / 8);
    hipLaunchKernelGGL(sample_bins<DT>, dim3(8 * eights * (unsigned)b.chunks), dim3(kBinThreads), 0, st, b);
    hipLaunchKernelGGL(sample_draw<DT>, dim3((unsigned)b.rows), dim3(kSampThreads), 0, st, b);
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
  a.chunks = z.chunks, a.chunk = z.chunk, a.rows = 0;
  int lg = 0;
  while ((1ll << lg) < vocab) ++lg;
  a.fbits = 62 - lg > 50 ? 50 : 62 - lg;
  a.u = u, a.temperature = temperature, a.top_k = top_k, a.top_p = top_p, a.min_p = min_p, a.tokens = tokens;
  char* ws = (char*)workspace;
  a.mass = (samp_u64*)(ws + z.mass), a.count = (unsigned*)(ws + z.count), a.max = (float*)(ws + z.max);
  const hipStream_t st = (hipStream_t)stream;
  if (dtype == TGM_F32) sample_launch<TGM_F32>(a, rows, st);
  else if (dtype == TGM_F16) sample_launch<TGM_F16>(a, rows, st);
  else sample_launch<TGM_BF16>(a, rows, st);
  return launch_status("tgm_sample");
}
