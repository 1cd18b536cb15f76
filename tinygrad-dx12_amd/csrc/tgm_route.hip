// The choice of experts (tgm_route): scores, keys, groups, the top k and their weights, in one launch.
//
// A token's logits lie in W lanes, R consecutive ones a lane, so that a wave holds 64 / W tokens and the steps of a
// reduction over one token are a reduction over all of them.  The k largest keys come one after another: a lane looks
// through its R keys, log2(W) exchanges settle the token's best, and its lane marks it with its rank.
//
// The keys' order is that of 64 bits, which are needed next to a border only.  Without a bias the logits' own order is the
// keys' and 32 bits hold it exactly.  With one, keys are computed in 32 bits first; where two that the choice compares, or
// two groups, are nearer than their errors allow, the wave does the choice again in 64 bits.
//
// What bounds it: instructions.  8192 tokens of 256 experts read 8.4 MB, 2 us of memory time.
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
template <int W, int M = 1>
__device__ __forceinline__ float lanes_max(float v) {
  if constexpr (M < W) return lanes_max<W, M * 2>(fmaxf(v, lane_xor<M>(v)));
  else return v;
}
// The largest key and, of equal ones, the lowest expert.
template <int W, int M = 1, class Key>
__device__ __forceinline__ void lanes_best(Key& key, int& e) {
  if constexpr (M < W) {
    const Key k = lane_xor<M>(key);
    const int o = (int)lane_xor<M>((unsigned)e);
    const bool take = k > key || (k == key && o < e);
    key = take ? k : key;
    e = take ? o : e;
    lanes_best<W, M * 2>(key, e);
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

// Leaves out the keys of all but the best groups.  V: the type that groups' sums are held in; tol: their values may be off
// by tol + 2.4e-7 of them each.  Returns whether two groups are nearer than that.
template <int W, int R, class V, class Key>
__device__ __forceinline__ bool route_groups(const RouteArgs& a, int l, const V (&c)[R], Key (&key)[R], V* sums, V tol) {
  const int per = a.experts / a.groups;
  for (int g = 0; g < a.groups; ++g) {
    V v1 = -INFINITY, v2 = -INFINITY;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int e = l * R + r;
      const V v = e >= g * per && e < (g + 1) * per && key[r] > 1 ? c[r] : (V)-INFINITY;
      v2 = v > v1 ? v1 : (v > v2 ? v : v2);
      v1 = v > v1 ? v : v1;
    }
    lanes_two<W>(v1, v2);
    if (l == 0) sums[g] = per > 1 ? v1 + v2 : v1;
  }
  wave_lds_fence();
  bool near = false;
  unsigned long long kept = 0;
  for (int g0 = 0; g0 < a.groups; g0 += W) {
    const int g = g0 + l;
    int rank = 0;
    const V v = g < a.groups ? sums[g] : (V)0;
    if (g < a.groups)
      for (int o = 0; o < a.groups; ++o) {
        const V u = sums[o];
        const Key ku = route_key(u), kv = route_key(v);
        rank += ku > kv || (ku == kv && o < g);
        if constexpr (sizeof(V) == 4) near |= o != g && !(fabsf(u - v) > tol + 2.4e-7f * (fabsf(u) + fabsf(v)));
      }
    const unsigned long long in = __ballot(g < a.groups && rank < a.top_groups);
    const unsigned long long mine = W == 64 ? in : (in >> ((threadIdx.x & 63) / W * W)) & ((1ull << (W & 63)) - 1);
    kept |= mine << g0;
  }
  wave_lds_fence();
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int e = l * R + r;
    if (e < a.experts && !(kept >> (e / per) & 1)) key[r] = 0;
  }
  return near;
}

// Marks the top k of the keys with their ranks (from 1).  Returns whether two neighbours of the order, the first that is
// left out among them, are nearer than their errors (32-bit keys of sums with a bias).
template <int W, int R, class Key>
__device__ __forceinline__ bool route_choose(const RouteArgs& a, int l, Key (&key)[R], int (&rank)[R], bool check, float tol) {
  bool near = false;
  float last = 0.0f;
  const int rounds = a.top_k + (check && a.top_k < a.experts ? 1 : 0);
  for (int j = 0; j < rounds; ++j) {
    Key best = key[0];
    int at = 0;
#pragma unroll
    for (int r = 1; r < R; ++r) {
      at = key[r] > best ? r : at;
      best = key[r] > best ? key[r] : best;
    }
    int e = l * R + at;
    lanes_best<W>(best, e);
    if constexpr (sizeof(Key) == 4) {
      if (check) {
        const float v = route_value(best);
        // a key that is left out is no rival; a NaN or equal infinities are near, and the 64 bits decide
        if (j > 0 && best != 0) near |= !(last - v > tol + 2.4e-7f * (fabsf(last) + fabsf(v)));
        last = v;
      }
    }
    if (j < a.top_k && e / R == l) {
#pragma unroll
      for (int r = 0; r < R; ++r) {
        rank[r] = e % R == r ? j + 1 : rank[r];
        key[r] = e % R == r ? 0 : key[r];
      }
    }
  }
  return near;
}

template <int DT, int W, int R>
__global__ void __launch_bounds__(kRouteThreads) route_rows(RouteArgs a) {
  __shared__ double sums[kRouteThreads / W][kRouteMaxGroups];
  const int l = threadIdx.x % W, slot = threadIdx.x / W;
  const int64_t token = (int64_t)blockIdx.x * (kRouteThreads / W) + slot;
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
    const bool in = l * R + r < a.experts;
    x[r] = in ? x[r] : -INFINITY;
    bad |= x[r] != x[r];
    top = fmaxf(top, x[r]);
  }
  top = lanes_max<W>(top);
  bad |= !a.sigmoid && top == INFINITY;
  const unsigned long long seen = __ballot(bad);
  bad = ((W == 64 ? seen : seen >> ((threadIdx.x & 63) / W * W) & ((1ull << (W & 63)) - 1))) != 0;

  // scores, under a softmax still to be divided by their sum
  float p[R], sum = 0.0f;
  const float zero = top == -INFINITY ? 0.0f : top;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    p[r] = a.sigmoid ? 1.0f / (1.0f + expf(-x[r])) : expf(x[r] - zero);
    sum += p[r];
  }
  sum = a.sigmoid ? 1.0f : lanes_sum<W>(sum);
  const float inv = sum > 0.0f ? 1.0f / sum : 0.0f;

  unsigned key[R];
  int rank[R];
  const bool limited = a.top_groups < a.groups, biased = a.bias != nullptr;
  bool near = false;
  {
    // errors of a score: 20 roundings and a difference of logits under a softmax, whose largest is inv; 4 of a sigmoid
    const float tol = a.sigmoid ? 1e-6f : 4e-5f * inv + 1e-37f;
    float c[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int e = l * R + r;
      rank[r] = 0;
      c[r] = p[r] * inv + (biased && e < a.experts ? a.bias[e] : 0.0f);
      c[r] = x[r] != x[r] ? x[r] : c[r];
      key[r] = e < a.experts ? route_key(biased ? c[r] : x[r]) : 0u;
    }
    if (limited) near = route_groups<W, R>(a, l, c, key, (float*)sums[slot], tol);
    near |= route_choose<W, R>(a, l, key, rank, biased, tol);
  }
  if (__any(near && !bad)) {  // the whole wave again, in 64 bits
    unsigned long long key64[R];
    double c[R], total = 0.0;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      c[r] = a.sigmoid ? 1.0 / (1.0 + exp(-(double)x[r])) : exp((double)x[r] - (double)zero);
      total += c[r];
    }
    total = a.sigmoid ? 1.0 : lanes_sum<W>(total);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int e = l * R + r;
      rank[r] = 0;
      c[r] = (total > 0.0 ? c[r] / total : 0.0) + (biased && e < a.experts ? (double)a.bias[e] : 0.0);
      c[r] = x[r] != x[r] ? (double)x[r] : c[r];
      key64[r] = e < a.experts ? route_key(biased ? c[r] : (double)x[r]) : 0ull;
    }
    if (limited) route_groups<W, R>(a, l, c, key64, sums[slot], 0.0);
    route_choose<W, R>(a, l, key64, rank, false, 0.0f);
  }

  float chosen = 0.0f;
#pragma unroll
  for (int r = 0; r < R; ++r) chosen += rank[r] ? p[r] : 0.0f;
  chosen = a.renormalize ? lanes_sum<W>(chosen) : sum;
  const float by = chosen > 0.0f ? a.scale / chosen : 0.0f;
  if (!live) return;
#pragma unroll
  for (int r = 0; r < R; ++r)
    if (rank[r]) {
      const int64_t o = token * a.top_k + rank[r] - 1;
      a.ids[o] = l * R + r;
      a.weights[o] = bad ? NAN : p[r] * by;
    }
}

template <int DT>
static void route_launch(const RouteArgs& a, hipStream_t st) {
  // few lanes a token make few exchanges; up to 16 of its logits a lane stay in registers
#define TGM_ROUTE(W, R)                                                                                             \
  hipLaunchKernelGGL((route_rows<DT, W, R>), dim3((unsigned)((a.tokens + kRouteThreads / W - 1) / (kRouteThreads / W))), \
                     dim3(kRouteThreads), 0, st, a)
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
  TGM_CHECK_ARG(ld >= experts || tokens <= 1, "the row stride is less than a row");
  TGM_CHECK_ARG(score == TGM_ROUTE_SOFTMAX || score == TGM_ROUTE_SIGMOID, "unknown score");
  TGM_CHECK_ARG(groups >= 1 && groups <= kRouteMaxGroups && experts % groups == 0,
                "groups must be 1 to %d and divide the experts", kRouteMaxGroups);
  TGM_CHECK_ARG(top_groups >= 1 && top_groups <= groups, "top_groups must be 1 to groups");
  TGM_CHECK_ARG(top_k >= 1 && top_k <= experts / groups * top_groups, "top_k must be 1 to the experts of top_groups groups");
  TGM_CHECK_ARG(scale == scale && scale - scale == 0.0, "scale must be finite");
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
