// Attention over the quantised paged cache: what its kernels share (tgm_kv_attend).
//
// For token t of sequence b (its last visible position p = lengths[b] - T + t) and query head h of kv head
// j = h / G:   out = sum_{k <= p} softmax_k(scale q . K_k) V_k,   K and V decoded from their codes and scales.
//
// Numbers.  Codes times their power-of-two scales are exact in bf16 (at most four significant bits), so K and V enter
// the matrix instructions as they are.  q is split into bf16 terms that together hold all its bits (bf16 1, f16 2,
// f32 3), each probability into 2 terms (16 bits; the output keeps 8 or 11) or, for f32 output, 3 (24 bits).  Products
// of bf16 values are exact in fp32, sums, maxima and the softmax's sum are fp32; the output is rounded once.
//
// What is not finite shows: a row with a NaN among its scores, or with one of +infinity, is NaN (its sum of weights is, in
// every split that holds such a score).  Zeros are for rows whose weights are all zero: no position is seen, or every
// score is -infinity.
//
// A masked position's value codes are replaced by zeros before they meet a probability of zero, so that whatever lies
// in memory that was never written (NaN codes among it) does not reach the sums.
#pragma once

#include "tgm_kv.h"

namespace tgm {

typedef __attribute__((__vector_size__(8 * sizeof(__bf16)))) __bf16 at_bf16x8;
typedef short at_s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) at_s16x4 at_lds_s16x4;

struct AttendArgs {
  const void* q;
  int64_t qb, qt, qh;
  int qvec;
  KvStore ks, vs;
  KvPages pg;
  const int32_t* lengths;
  int B, T, H, HK, G;
  int k0, kcap;        // positions k0 .. kcap - 1 are this launch's
  int chunk;           // positions per split
  int slot0, slots;    // this launch's first partial of a row, and partials per row (1: the output itself)
  int common;          // attend_many: every sequence's rows against row 0's pages
  int prefix;          // attend_few: positions below it lie in row 0's pages
  float sl;            // scale * log2(e)
  float* part;         // [row][slot][HD] sums, then [row][slot][2] maximum (log2 units) and sum of weights
  void* out;
};

template <int DT>
struct AttendTerms {
  static constexpr int Q = DT == TGM_BF16 ? 1 : (DT == TGM_F16 ? 2 : 3);
  static constexpr int P = DT == TGM_F32 ? 3 : 2;
};

// The bf16 terms of 8 fp32 values: t[0] = bf16(x), each next one the bf16 of what is left.
// Two values a conversion: the compiler does not pair them by itself.
template <int N>
__device__ __forceinline__ void at_split(float (&r)[8], at_bf16x8 (&t)[N]) {
#pragma unroll
  for (int s = 0; s < N; ++s) {
    u32x4 w;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      unsigned pair = bf16x2_bits(r[2 * i], r[2 * i + 1]);
      asm("" : "+v"(pair));  // else the low half is converted a second time for the difference
      w[i] = pair;
      if (s + 1 < N) {
        r[2 * i] -= bits_f32(w[i] << 16);
        r[2 * i + 1] -= bits_f32(w[i] & 0xFFFF0000u);
      }
    }
    t[s] = __builtin_bit_cast(at_bf16x8, w);
  }
}

__device__ __forceinline__ at_bf16x8 at_tr_pair(const unsigned char* lo, const unsigned char* hi) {
  const at_s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((at_lds_s16x4*)lo);
  const at_s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((at_lds_s16x4*)hi);
  return __builtin_bit_cast(at_bf16x8, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
}

// N bytes (a multiple of 4) of global memory into words, in the widest loads that their alignment (N) allows.
template <int N>
__device__ __forceinline__ void at_load(const uint8_t* p, unsigned (&w)[N / 4]) {
  if constexpr (N >= 16) {
#pragma unroll
    for (int i = 0; i < N / 16; ++i) {
      const u32x4 x = *(const u32x4*)(p + 16 * i);
#pragma unroll
      for (int e = 0; e < 4; ++e) w[4 * i + e] = x[e];
    }
  } else {
    static_assert(N == 8, "8, 16 or 32 bytes");
    const u32x2 x = *(const u32x2*)p;
    w[0] = x[0];
    w[1] = x[1];
  }
}

// 8 codes from word index i of a lane's words (fp8: words 2 i, 2 i + 1; fp4: word i) as bf16.
template <int BITS, int N>
__device__ __forceinline__ u32x4 at_codes8(const unsigned (&w)[N], int i, float s) {
  u32x2 a, b;
  if constexpr (BITS == 8) {
    a = kv_bf16x4<8>(w[2 * i], 0, s);
    b = kv_bf16x4<8>(w[2 * i + 1], 0, s);
  } else {
    a = kv_bf16x4<4>(w[i], 0, s);
    b = kv_bf16x4<4>(w[i], 1, s);
  }
  return u32x4{a[0], a[1], b[0], b[1]};
}

template <int DT>
__device__ __forceinline__ void at_store(void* out, int64_t i, float v) {
  if constexpr (DT == TGM_F32) ((float*)out)[i] = v;
  else if constexpr (DT == TGM_BF16) ((uint16_t*)out)[i] = f32_to_bf16(v);
  else ((_Float16*)out)[i] = (_Float16)v;
}

// Cached positions of a sequence, within what 32-bit position arithmetic takes.
__device__ __forceinline__ int at_length(const AttendArgs& A, int b) { return min(max(A.lengths[b], 0), 1 << 30); }
__device__ __forceinline__ int64_t at_rows(const AttendArgs& A) { return (int64_t)A.B * A.T * A.H; }
__device__ __forceinline__ float* at_ml(const AttendArgs& A, int hd, int64_t row, int slot) {
  return A.part + at_rows(A) * A.slots * hd + (row * A.slots + slot) * 2;
}

// Launchers, one translation unit per query type.
struct AttendLaunch {
  AttendArgs a;
  int kb, vb, hd;  // bits of a key's and a value's code, head_dim
  int splits;
};
template <int DT>
void attend_few(const AttendLaunch& l, hipStream_t st);
template <int DT>
void attend_many(const AttendLaunch& l, hipStream_t st);
template <int DT>
void attend_both(const AttendLaunch& prefix, const AttendLaunch& own, hipStream_t st);  // rows of one tile of attend_few

// Rows (tokens x heads of a group) that attend_few takes.
constexpr int attend_few_tile(int dt) { return dt == TGM_F32 ? 5 : 8; }  // rows of one column tile
constexpr int attend_few_rows(int dt) { return 2 * attend_few_tile(dt); }
constexpr int kFewBlock = 64, kFewWaves = 4;
constexpr int kManyKeys = 64, kManyRows = 128;
constexpr float kLazyLog2 = 8.f;
}  // namespace tgm
