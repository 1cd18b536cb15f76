// Rotary positions on a wave: the angles of one token, and the rotation of 16 values of a head a lane.
#pragma once

#include "tgm_kv.h"

namespace tgm {

// Modes of a rotation.  Half layout over the whole head: a lane's two chunks of 8 values are partners.
// Interleaved: partners are neighbours.  Half layout over a part of the head: partners lie elsewhere and are
// read one by one.
enum RotMode { kRotNone = 0, kRotHalf = 1, kRotInterleaved = 2, kRotPart = 3 };

struct RotArgs {
  const double* freq;
  double gain;
  int pairs;  // rotary_dim / 2
};

// sin and cos in 64 bits: x is brought to |r| <= pi / 4 by n = rint(x 2 / pi) multiples of pi / 2 held in two
// doubles (fused products, so r is within 2^-53 for |x| < 2^31), and both Taylor series are summed to the
// term whose successor is below 2^-58.
__device__ __forceinline__ void rot_sincos(double x, double& s, double& c) {
  const double n = __builtin_rint(x * 0x1.45f306dc9c883p-1);
  double r = __builtin_fma(-n, 0x1.921fb54442d18p+0, x);
  r = __builtin_fma(-n, 0x1.1a62633145c07p-54, r);
  const double z = r * r;
  double a = 1.0 / 355687428096000.0;  // 17!
  a = __builtin_fma(a, z, -1.0 / 1307674368000.0);
  a = __builtin_fma(a, z, 1.0 / 6227020800.0);
  a = __builtin_fma(a, z, -1.0 / 39916800.0);
  a = __builtin_fma(a, z, 1.0 / 362880.0);
  a = __builtin_fma(a, z, -1.0 / 5040.0);
  a = __builtin_fma(a, z, 1.0 / 120.0);
  a = __builtin_fma(a, z, -1.0 / 6.0);
  const double sr = __builtin_fma(a * z, r, r);
  double b = 1.0 / 20922789888000.0;  // 16!
  b = __builtin_fma(b, z, -1.0 / 87178291200.0);
  b = __builtin_fma(b, z, 1.0 / 479001600.0);
  b = __builtin_fma(b, z, -1.0 / 3628800.0);
  b = __builtin_fma(b, z, 1.0 / 40320.0);
  b = __builtin_fma(b, z, -1.0 / 720.0);
  b = __builtin_fma(b, z, 1.0 / 24.0);
  b = __builtin_fma(b, z, -0.5);
  const double cr = __builtin_fma(b, z, 1.0);
  const int q = (int)(long long)n & 3;  // a long long first: |n| reaches 2^31
  s = q & 1 ? cr : sr;
  c = q & 1 ? sr : cr;
  if (q & 2) s = -s;
  if ((q + 1) & 2) c = -c;
}

__device__ __forceinline__ void rot_wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// One wave's angles of the token at position `pos`, cosine and sine of each pair times the gain, into its own
// LDS block.
__device__ __forceinline__ void rot_angles(const RotArgs& rot, int pos, int lane, double2* cs) {
  for (int i = lane; i < rot.pairs; i += 64) {
    double s, c;
    rot_sincos((double)pos * rot.freq[i], s, c);
    cs[i] = double2{c * rot.gain, s * rot.gain};
  }
  rot_wave_sync();
}

// A lane's cosines and sines: 8 pairs, in registers over the heads of a token.
template <int HD, int MODE>
struct RotLane {
  double c[8], s[8];
  __device__ __forceinline__ void load(const RotArgs& rot, const double2* cs, int chunk) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int i = MODE == kRotHalf ? 8 * chunk + e : (e < 4 ? 4 * chunk + e : HD / 4 + 4 * chunk + e - 4);
      const double2 v = i < rot.pairs ? cs[i] : double2{1.0, 0.0};
      c[e] = v.x;
      s[e] = v.y;
    }
  }
};

// The chunks a (values 8 chunk ..) and b (HD / 2 + 8 chunk ..) of a head, rotated.  `x` and `at` find the head in
// memory for partners that lie elsewhere.
template <int DT, int HD, int MODE>
__device__ __forceinline__ void rot_apply(const RotArgs& rot, const RotLane<HD, MODE>& t, const double2* cs, int chunk,
                                          const void* x, int64_t at, float (&a)[8], float (&b)[8]) {
#pragma clang fp contract(off)  // else the rounding to 32 bits may be merged with the caller's to 16
  if constexpr (MODE == kRotHalf) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const double u = a[e], v = b[e];
      a[e] = (float)__builtin_fma(u, t.c[e], -(v * t.s[e]));
      b[e] = (float)__builtin_fma(v, t.c[e], u * t.s[e]);
    }
  } else if constexpr (MODE == kRotInterleaved) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const double u = a[2 * e], v = a[2 * e + 1], y = b[2 * e], z = b[2 * e + 1];
      if (4 * chunk + e < rot.pairs) {
        a[2 * e] = (float)__builtin_fma(u, t.c[e], -(v * t.s[e]));
        a[2 * e + 1] = (float)__builtin_fma(v, t.c[e], u * t.s[e]);
      }
      if (HD / 4 + 4 * chunk + e < rot.pairs) {
        b[2 * e] = (float)__builtin_fma(y, t.c[4 + e], -(z * t.s[4 + e]));
        b[2 * e + 1] = (float)__builtin_fma(z, t.c[4 + e], y * t.s[4 + e]);
      }
    }
  } else if constexpr (MODE == kRotPart) {
    auto turn = [&](int d, float own) {
      if (d >= 2 * rot.pairs) return own;
      const bool lower = d < rot.pairs;
      const double2 v = cs[lower ? d : d - rot.pairs];
      const double other = load_f32(x, DT, at + (lower ? d + rot.pairs : d - rot.pairs));
      return (float)__builtin_fma((double)own, v.x, lower ? -(other * v.y) : other * v.y);
    };
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      a[e] = turn(8 * chunk + e, a[e]);
      b[e] = turn(HD / 2 + 8 * chunk + e, b[e]);
    }
  }
}

inline int rot_mode(const tgm_rotary* r, int64_t head_dim) {
  if (!r || r->rotary_dim == 0) return kRotNone;
  if (r->layout == TGM_ROTARY_INTERLEAVED) return kRotInterleaved;
  return r->rotary_dim == head_dim ? kRotHalf : kRotPart;
}

inline int rot_check(const tgm_rotary* r, int64_t head_dim) {
  TGM_CHECK_ARG(r->rotary_dim >= 0 && r->rotary_dim % 2 == 0 && r->rotary_dim <= head_dim,
                "rotary_dim must be even and at most head_dim");
  TGM_CHECK_ARG(r->layout == TGM_ROTARY_HALF || r->layout == TGM_ROTARY_INTERLEAVED, "unknown rotary layout");
  TGM_CHECK_ARG(r->freq || r->rotary_dim == 0, "null frequencies");
  return TGM_OK;
}

inline bool heads_dtype_ok(int64_t dt) { return dt == TGM_F32 || dt == TGM_F16 || dt == TGM_BF16; }
// 16-byte loads of 8 values (4 at a time in 32 bits) start at every head of every token.
inline bool heads_vec(const tgm_heads* t, const void* data) {
  const int64_t step = 16 / dtype_size((int)t->dtype);
  return ((uintptr_t)data & 15) == 0 && t->stride_b % step == 0 && t->stride_t % step == 0 && t->stride_h % step == 0;
}

}  // namespace tgm
