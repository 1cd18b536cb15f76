// The choice of experts (tgm_route): scores, keys, groups, the top k and their weights, in one launch.
//
// A token's logits lie in W lanes, R consecutive ones a lane, so that a wave holds 64 / W tokens and the steps of a
// reduction over one token are a reduction over all of them.  The k largest keys come one after another: the largest of a
// lane's R and of the W lanes, then the lowest expert that has it, whose number goes to a list in LDS.  At the end a lane
// takes an entry of the list and computes its weight from the logit.
//
// The keys' order is that of 64 bits, which are needed next to a border only.  Without a bias the logits' own order is the
// keys' and 32 bits hold it exactly.  With one, keys are computed in 32 bits first, and the list goes on to the first
// distance that is larger than their errors allow.  Where neighbours in it are nearer, its entries' keys are computed in 64
// bits, one a lane, and put in order; where it does not end in time, where groups on either side of their border are that
// near, or where a row has a NaN, the wave does the choice again in 64 bits.
//
// What bounds it: instructions.  8192 tokens of 256 experts in 8 groups read 8.4 MB, 2 us of memory time, and take 11 to 12 (some
// 3 more with expf and a division in the keys, whose errors the list allows for): a sigmoid an expert, the two largest of each
// group, eight rounds of a maximum over 16 lanes.  With 32 or 64 lanes a token the rounds are longer and the time the same.  A
// wave that does the choice again takes 9 more, which the launch waits for: one set of such inputs in eight has one.
#include <float.h>
#include <math.h>

#include "../../include/tgm_experts.h"
#include "tgm_common.h"
#include "tgm_lanes.h"

namespace tgm {

constexpr int kRouteThreads = 256, kRouteMaxGroups = 64;

struct RouteArgs {
  const void* logits;
  int64_t ld;
  const float* bias;
  int32_t* ids;
  float* weights;
  int64_t tokens;
  int experts, groups, top_groups, top_k;
  int sigmoid, renormalize, vectors;
  float scale;
};

// Keys that order as their values do; 0 is left out, 1 a NaN's place behind -infinity, -0 is +0.
__device__ __forceinline__ unsigned route_key(float x) {
  if (x != x) return 1u;
  const unsigned b = f32_bits(x + 0.0f);
  return b ^ ((b >> 31) ? 0xFFFFFFFFu : 0x80000000u);
}
__device__ __forceinline__ unsigned long long route_key(double x) {
  if (x != x) return 1ull;
  const unsigned long long b = __builtin_bit_cast(unsigned long long, x + 0.0);
  return b ^ ((b >> 63) ? ~0ull : 0x8000000000000000ull);
}
__device__ __forceinline__ float route_value(unsigned k) {
  return bits_f32(k ^ ((k >> 31) ? 0x80000000u : 0xFFFFFFFFu));
}

// The value of lane l ^ M.
template <int M>
__device__ __forceinline__ unsigned lane_xor(unsigned v) {
  const float f = __builtin_bit_cast(float, v);
  if constexpr (M == 1) return f32_bits(xor1(f));
  else if constexpr (M == 2) return f32_bits(xor2(f));
  else if constexpr (M == 4) return f32_bits(xor4(f));
  else if constexpr (M == 8) return f32_bits(xor8(f));
  else return (unsigned)__shfl_xor((int)v, M);
}
template <int M>
__device__ __forceinline__ unsigned long long lane_xor(unsigned long long v) {
  return (unsigned long long)lane_xor<M>((unsigned)v) | (unsigned long long)lane_xor<M>((unsigned)(v >> 32)) << 32;
}
template <int M>
__device__ __forceinline__ float lane_xor(float v) { return bits_f32(lane_xor<M>(f32_bits(v))); }
template <int M>
__device__ __forceinline__ double lane_xor(double v) {
  return __builtin_bit_cast(double, lane_xor<M>(__builtin_bit_cast(unsigned long long, v)));
}

template <int W, int M = 1, class T>
__device__ __forceinline__ T lanes_sum(T v) {
  if constexpr (M < W) return lanes_sum<W, M * 2>(v + lane_xor<M>(v));
  else return v;
}
template <int W, int M = 1, class T>
__device__ __forceinline__ T lanes_max(T v) {
  if constexpr (M < W) {
    const T o = lane_xor<M>(v);
    return lanes_max<W, M * 2>(o > v ? o : v);
  } else {
    return v;
  }
}
template <int W, int M = 1>
__device__ __forceinline__ int lanes_min(int v) {
  if constexpr (M < W) {
    const int o = (int)lane_xor<M>((unsigned)v);
    return lanes_min<W, M * 2>(o < v ? o : v);
  } else {
    return v;
  }
}
// The two largest of v1 >= v2 over the lanes.
template <int W, int M = 1, class T>
__device__ __forceinline__ void lanes_two(T& v1, T& v2) {
  if constexpr (M < W) {
    const T o1 = lane_xor<M>(v1), o2 = lane_xor<M>(v2);
    const T low = v1 < o1 ? v1 : o1;
    v1 = v1 < o1 ? o1 : v1;
    const T two = v2 < o2 ? o2 : v2;
    v2 = low < two ? two : low;
    lanes_two<W, M * 2>(v1, v2);
  }
}

__device__ __forceinline__ void wave_lds_fence() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// Leaves out the keys of all but the best groups.  V: the type that groups' sums are held in; in 32 bits they may be off by
// tol and by two roundings of the keys and one of their sum each.  Returns whether a group that stays and one that goes are nearer than that.
template <int W, int R, class V, class Key>
__device__ __forceinline__ bool route_groups(const RouteArgs& a, int l, const V (&c)[R], Key (&key)[R], V* sums, V tol) {
  const int per = a.experts / a.groups, lanes = per / R;
  // groups of whole lanes, 2^i of them: each lane looks through its own
  const bool whole = per % R == 0 && (lanes & (lanes - 1)) == 0;
  auto two = [&](int first, int end, V& v1, V& v2) __attribute__((always_inline)) {
    v1 = v2 = -INFINITY;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int e = l * R + r;
      const V v = e >= first && e < end && key[r] > 1 ? c[r] : (V)-INFINITY;
      v2 = v > v1 ? v1 : (v > v2 ? v : v2);
      v1 = v > v1 ? v : v1;
    }
  };
  V v1, v2;
  float size = 0.0f;  // the largest terms of a sum, if they are finite
  if (whole) {
    two(0, a.experts, v1, v2);
    if (lanes > 1) lanes_two<2, 1>(v1, v2);
    if (lanes > 2) lanes_two<4, 2>(v1, v2);
    if (W > 8 && lanes > 4) lanes_two<8, 4>(v1, v2);
    if (W > 8 && lanes > 8) lanes_two<16, 8>(v1, v2);
    if constexpr (W > 32) {
      if (lanes > 16) lanes_two<32, 16>(v1, v2);
    }
    size = fabsf((float)v1) + fabsf((float)v2);
    if (l % lanes == 0 && l / lanes < a.groups) sums[l / lanes] = per > 1 ? v1 + v2 : v1;
  } else {
    for (int g = 0; g < a.groups; ++g) {
      two(g * per, (g + 1) * per, v1, v2);
      lanes_two<W>(v1, v2);
      const float s = fabsf((float)v1) + fabsf((float)v2);
      size = s < INFINITY ? fmaxf(size, s) : size;
      if (l == 0) sums[g] = per > 1 ? v1 + v2 : v1;
    }
  }
  wave_lds_fence();
  // the least that stays and the largest that goes
  unsigned long long kept = 0;
  V least = INFINITY, most = -INFINITY;
  for (int g0 = 0; g0 < a.groups; g0 += W) {
    const int g = g0 + l;
    int rank = 0;
    const V v = g < a.groups ? sums[g] : (V)0;
    const Key kv = route_key(v);
#pragma unroll 8
    for (int o = 0; o < a.groups; ++o) {
      const Key ku = route_key(sums[o]);
      rank += ku > kv || (ku == kv && o < g);
    }
    const bool stays = g < a.groups && rank < a.top_groups;
    if (stays) least = v < least ? v : least;
    else if (g < a.groups) most = v > most ? v : most;
    const unsigned long long in = __ballot(stays);
    const unsigned long long mine = W == 64 ? in : (in >> ((threadIdx.x & 63) / W * W)) & ((1ull << (W & 63)) - 1);
    kept |= mine << g0;
  }
  wave_lds_fence();
  if (whole) {
    const bool stays = kept >> (l / lanes < 63 ? l / lanes : 63) & 1;
#pragma unroll
    for (int r = 0; r < R; ++r) key[r] = stays || l * R + r >= a.experts ? key[r] : 0;
  } else {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int e = l * R + r;
      if (e < a.experts && !(kept >> (e / per) & 1)) key[r] = 0;
    }
  }
  if constexpr (sizeof(V) == 8) return false;
  least = -lanes_max<W>(-least), most = lanes_max<W>(most);
  size = lanes_max<W>(size < INFINITY ? size : 0.0f);
  return !(least - most > tol + 2.4e-7f * size);
}

// The keys of a list go on to kRouteMore entries past the top k.
constexpr int kRouteMore = 4;

// Lists the experts of the largest keys, the top k of them and, with `check`, on to the first that is clearly less than its
// neighbour; key 0 is none.  Returns the entries, and whether two neighbours are nearer than the errors of 32-bit keys
// allow; -1 where the list does not end in time.
template <int W, int R, class Key>
__device__ __forceinline__ int route_choose(const RouteArgs& a, int l, Key (&key)[R], int* list, bool check, float tol, bool& near) {
  float last = 0.0f;
  bool open = true;
  int entries = 0;
  near = false;
  const int rounds = a.top_k + (check ? kRouteMore : 0);
  for (int j = 0; j < rounds; ++j) {
    Key best = key[0];
#pragma unroll
    for (int r = 1; r < R; ++r) best = key[r] > best ? key[r] : best;
    best = lanes_max<W>(best);
    if (check) {
      const float v = route_value((unsigned)best);
      // no key is left, or this one is clearly less; a NaN or equal infinities are near
      const bool clear = best == 0 || last - v > tol + 1.2e-7f * (fabsf(last) + fabsf(v));
      if (j > 0 && open) near |= !clear;
      open = open && !(j >= a.top_k && clear);
      last = v;
      if (j >= a.top_k && !__any(open)) break;
    }
    int e = 1 << 20;
#pragma unroll
    for (int r = R - 1; r >= 0; --r) e = key[r] == best ? l * R + r : e;
    e = lanes_min<W>(e);
#pragma unroll
    for (int r = 0; r < R; ++r) key[r] = l * R + r == e ? 0 : key[r];
    if (open && l == 0) list[j] = e;
    entries += open;
  }
  return check && open ? -1 : entries;
}

template <int DT, int W, int R>
__global__ void __launch_bounds__(kRouteThreads) route_rows(RouteArgs a) {
  constexpr int SLOTS = kRouteThreads / W;
  __shared__ double sums[SLOTS][kRouteMaxGroups];  // of groups, then the listed experts' keys
  extern __shared__ int lists[];                   // [slot][top_k + kRouteMore]
  const int l = threadIdx.x % W, slot = threadIdx.x / W;
  int* list = lists + slot * (a.top_k + kRouteMore);
  const int64_t token = (int64_t)blockIdx.x * SLOTS + slot;
  const bool live = token < a.tokens;
  const int64_t base = (live ? token : a.tokens - 1) * a.ld;  // waves stay whole: exchanges run in every lane
  float x[R];
  if constexpr (R >= 4) {
    if (a.vectors) {  // rows of whole, aligned vectors of four
#pragma unroll
      for (int q = 0; q < R / 4; ++q) {
        const int e = l * R + 4 * q;
        if constexpr (DT == TGM_F32) {
          typedef float f4 __attribute__((ext_vector_type(4)));
          const f4 v = e < a.experts ? *(const f4*)((const float*)a.logits + base + e) : f4{};
          x[4 * q] = v[0], x[4 * q + 1] = v[1], x[4 * q + 2] = v[2], x[4 * q + 3] = v[3];
        } else {
          typedef unsigned short u4 __attribute__((ext_vector_type(4)));
          const u4 v = e < a.experts ? *(const u4*)((const unsigned short*)a.logits + base + e) : u4{};
#pragma unroll
          for (int i = 0; i < 4; ++i)
            x[4 * q + i] = DT == TGM_BF16 ? bf16_to_f32(v[i]) : (float)__builtin_bit_cast(_Float16, (unsigned short)v[i]);
        }
      }
    }
  }
  if (R < 4 || !a.vectors) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int e = l * R + r;
      x[r] = e < a.experts ? load_f32(a.logits, DT, base + e) : 0.0f;
    }
  }
  bool bad = false;
  float top = -INFINITY;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    x[r] = l * R + r < a.experts ? x[r] : -INFINITY;
    bad |= x[r] != x[r];
    top = fmaxf(top, x[r]);
  }
  const bool soft = !a.sigmoid, limited = a.top_groups < a.groups, biased = a.bias != nullptr;
  if (soft) top = lanes_max<W>(top);
  bad |= soft && top == INFINITY;
  const unsigned long long seen = __ballot(bad);
  bad = ((W == 64 ? seen : seen >> ((threadIdx.x & 63) / W * W) & ((1ull << (W & 63)) - 1))) != 0;
  const float zero = top == -INFINITY ? 0.0f : top;
  unsigned key[R];
  float sum = 1.0f;
  bool near = false, again = false;
  int entries;
  if (biased || limited) {
    float c[R];
    sum = 0.0f;
    if (soft) {
#pragma unroll
      for (int r = 0; r < R; ++r) {
        c[r] = expf(x[r] - zero);
        sum += c[r];
      }
    } else {
#pragma unroll
      for (int r = 0; r < R; ++r) c[r] = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(x[r] * -1.44269504f));
    }
    sum = soft ? lanes_sum<W>(sum) : 1.0f;
    const float inv = sum > 0.0f ? 1.0f / sum : 0.0f;
    // Errors of two scores.  Sigmoid, 1 / (1 + 2^t): t is off by 1.5 half steps, which changes p by p (1 - p) |x| 1.5 2^-24, at
    // most 0.34 2^-24; the power, the sum and the quotient by 2^-25, 2^-24 and 2^-23: together less than 2.4e-7.  Softmax: of the
    // largest, inv, a difference of logits up to 104 (below, the score is 0), exp, R + 6 sums and two products, 2^-16.
    const float tol = soft ? 3.1e-5f * inv + 1e-37f : 5e-7f;
    float b[R];
#pragma unroll
    for (int r = 0; r < R; ++r) b[r] = 0.0f;
    if (biased) {
      if (R >= 4 && a.vectors && (uintptr_t)a.bias % 16 == 0) {
#pragma unroll
        for (int q = 0; q < R / 4; ++q) {
          typedef float f4 __attribute__((ext_vector_type(4)));
          const int e = l * R + 4 * q;
          const f4 v = e < a.experts ? *(const f4*)(a.bias + e) : f4{};
          b[4 * q] = v[0], b[4 * q + 1] = v[1], b[4 * q + 2] = v[2], b[4 * q + 3] = v[3];
        }
      } else {
#pragma unroll
        for (int r = 0; r < R; ++r) b[r] = l * R + r < a.experts ? a.bias[l * R + r] : 0.0f;
      }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int e = l * R + r;
      c[r] = c[r] * inv + b[r];
      key[r] = e < a.experts ? route_key(biased ? c[r] : x[r]) : 0u;
    }
    // rows that are not finite have neither errors as above nor, under a softmax, keys that are numbers
    again = bad;
    if (limited) again |= route_groups<W, R>(a, l, c, key, (float*)sums[slot], 2 * tol);
    entries = route_choose<W, R>(a, l, key, list, biased, tol, near);
    again |= entries < 0 || (near && entries > W);
  } else {
    if (soft && !a.renormalize) {
      sum = 0.0f;
#pragma unroll
      for (int r = 0; r < R; ++r) sum += expf(x[r] - zero);
      sum = lanes_sum<W>(sum);
    }
#pragma unroll
    for (int r = 0; r < R; ++r) key[r] = l * R + r < a.experts ? route_key(x[r]) : 0u;
    entries = route_choose<W, R>(a, l, key, list, false, 0.0f, near);
  }
  if (__any(near || again)) {
    double total = 1.0;
    if (soft) {
      total = 0.0;
#pragma unroll
      for (int r = 0; r < R; ++r) total += exp((double)x[r] - (double)zero);
      total = lanes_sum<W>(total);
    }
    auto wide_key = [&](float v, int e) __attribute__((always_inline)) {
      const double p = soft ? exp((double)v - (double)zero) : 1.0 / (1.0 + exp(-(double)v));
      return (total == 0.0 ? 0.0 : p / total) + (biased ? (double)a.bias[e] : 0.0);
    };
    if (__any(again)) {  // the whole wave
      unsigned long long wide[R];
      double c[R];
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const int e = l * R + r;
        c[r] = e < a.experts ? wide_key(x[r], e) : 0.0;
        wide[r] = e < a.experts ? route_key(biased ? c[r] : (double)x[r]) : 0ull;
      }
      if (limited) route_groups<W, R>(a, l, c, wide, sums[slot], 0.0);
      bool unused;
      route_choose<W, R>(a, l, wide, list, false, 0.0f, unused);
    } else {
      wave_lds_fence();
      const bool holds = near && l < entries;
      const int e = holds ? list[l] : 0;
      const unsigned long long mine = holds ? route_key(wide_key(load_f32(a.logits, DT, base + e), e)) : 0ull;
      if (holds) sums[slot][l] = __builtin_bit_cast(double, mine);
      wave_lds_fence();
      int rank = 0;
      for (int o = 0; o < (near ? entries : 0); ++o) {
        const unsigned long long k = __builtin_bit_cast(unsigned long long, sums[slot][o]);
        rank += k > mine || (k == mine && list[o] < e);
      }
      wave_lds_fence();
      if (holds && rank < a.top_k) list[rank] = e;
    }
  }
  wave_lds_fence();

  // The weights, an entry a lane.  Their scores are e^x of a softmax, over its sum, or e^min(x, 0) / (1 + e^-|x|), all of them times
  // e^-from: from the row's largest logit, and in renormalised ones from the largest chosen, which a bias may have picked far
  // below it and which may be low itself, so that the chosen ones' sum is at least a half.
  const int own = l < a.top_k ? list[l] : 0;
  const float mine = load_f32(a.logits, DT, base + own);
  auto logit = [&](int j) __attribute__((always_inline)) { return j < W ? mine : load_f32(a.logits, DT, base + list[j]); };
  float from = soft ? zero : 0.0f;
  if (a.renormalize) {
    float most = -INFINITY;
    for (int j = l; j < a.top_k; j += W) most = fmaxf(most, logit(j));
    most = lanes_max<W>(most);
    from = most == -INFINITY ? 0.0f : soft ? most : fminf(most, 0.0f);
  }
  auto score = [&](float v) __attribute__((always_inline)) {
    return soft ? expf(v - from) : expf(fminf(v, 0.0f) - from) / (1.0f + expf(-fabsf(v)));
  };
  const float first = score(mine);
  float chosen = l < a.top_k ? first : 0.0f;
  for (int j = l + W; j < a.top_k; j += W) chosen += score(logit(j));
  chosen = a.renormalize ? lanes_sum<W>(chosen) : sum;
  if (!live) return;
  for (int j = l; j < a.top_k; j += W) {
    const float part = (j < W ? first : score(logit(j))) / chosen;
    a.ids[token * a.top_k + j] = j < W ? own : list[j];
    a.weights[token * a.top_k + j] = bad ? NAN : chosen > 0.0f ? part * a.scale : 0.0f;
  }
}

template <int DT>
static void route_launch(const RouteArgs& a, hipStream_t st) {
  // few lanes a token make few exchanges; up to 16 of its logits a lane stay in registers
#define TGM_ROUTE(W, R)                                                                                             \
  hipLaunchKernelGGL((route_rows<DT, W, R>), dim3((unsigned)((a.tokens + kRouteThreads / W - 1) / (kRouteThreads / W))), \
                     dim3(kRouteThreads), kRouteThreads / W * (a.top_k + kRouteMore) * sizeof(int), st, a)
  if (a.experts <= 8) TGM_ROUTE(8, 1);
  else if (a.experts <= 16) TGM_ROUTE(16, 1);
  else if (a.experts <= 32) TGM_ROUTE(16, 2);
  else if (a.experts <= 64) TGM_ROUTE(16, 4);
  else if (a.experts <= 128) TGM_ROUTE(16, 8);
  else if (a.experts <= 256) TGM_ROUTE(16, 16);
  else if (a.experts <= 512) TGM_ROUTE(32, 16);
  else TGM_ROUTE(64, 16);
#undef TGM_ROUTE
}

}  // namespace tgm

using namespace tgm;

extern "C" int tgm_route(const void* logits, int64_t dtype, int64_t tokens, int64_t experts, int64_t ld, const float* bias,
                         int64_t score, int64_t groups, int64_t top_groups, int64_t top_k, int64_t renormalize, double scale,
                         int32_t* ids, float* weights, void* stream) {
  clear_error();
  TGM_CHECK_ARG(dtype == TGM_F32 || dtype == TGM_F16 || dtype == TGM_BF16, "logits must be f32, f16 or bf16");
  TGM_CHECK_ARG(tokens >= 0 && tokens < (1ll << 24), "invalid token count");
  TGM_CHECK_ARG(experts >= 1 && experts <= 1024, "a router chooses among 1 to 1024 experts");
  TGM_CHECK_ARG((ld >= experts && ld < (1ll << 36)) || tokens <= 1, "the row stride is less than a row, or too large");
  TGM_CHECK_ARG(score == TGM_ROUTE_SOFTMAX || score == TGM_ROUTE_SIGMOID, "unknown score");
  TGM_CHECK_ARG(groups >= 1 && groups <= kRouteMaxGroups && experts % groups == 0,
                "groups must be 1 to %d and divide the experts", kRouteMaxGroups);
  TGM_CHECK_ARG(top_groups >= 1 && top_groups <= groups, "top_groups must be 1 to groups");
  TGM_CHECK_ARG(top_k >= 1 && top_k <= experts / groups * top_groups, "top_k must be 1 to the experts of top_groups groups");
  TGM_CHECK_ARG(fabs(scale) <= FLT_MAX, "scale must be a finite number of 32 bits");
  if (tokens == 0) return TGM_OK;
  TGM_CHECK_ARG(logits && ids && weights, "null operand");
  RouteArgs a;
  a.logits = logits, a.ld = tokens > 1 ? ld : experts, a.bias = bias, a.ids = ids, a.weights = weights, a.tokens = tokens;
  a.experts = (int)experts, a.groups = (int)groups, a.top_groups = (int)top_groups, a.top_k = (int)top_k;
  a.sigmoid = score == TGM_ROUTE_SIGMOID, a.renormalize = renormalize != 0, a.scale = (float)scale;
  const int size = dtype_size((int)dtype);
  a.vectors = experts % 4 == 0 && a.ld % 4 == 0 && (uintptr_t)logits % (4 * size) == 0;
  const hipStream_t st = (hipStream_t)stream;
  if (dtype == TGM_F32) route_launch<TGM_F32>(a, st);
  else if (dtype == TGM_F16) route_launch<TGM_F16>(a, st);
  else route_launch<TGM_BF16>(a, st);
  return launch_status("tgm_route");
}
