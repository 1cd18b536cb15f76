// Attention of many rows per kv head: chunks of a prompt, and the common prefix of a batch.
//
// Grid (row tiles x splits, kv_heads, batch or 1), 256 threads.  A row is a (token, head of the group) pair of one
// sequence, or of any sequence when the positions are common to all.  A workgroup takes 128 rows, 32 per wave, and walks
// the positions of its split in blocks of 64.  The products are computed transposed, so that a lane pair owns a row
// (32x32 MFMA D layout: lane l holds column l % 32):
//
//   S^T[key, row] = K . Q^T      A = keys (LDS),    B = q (registers)
//   O^T[dim, row] += V^T . P^T   A = V^T (LDS),     B = p (registers)
//
// The codes of a block are loaded to registers while the block before is computed, decoded once by the whole workgroup
// (four threads a position) and stored to LDS as bf16 rows, double buffered, one barrier a block.  16-byte chunks of a
// row are XOR-swizzled so that 16-byte reads of 32 key rows and transposing reads of 4 value rows do not conflict.
//
// What bounds it: per wave and block 48 products (bf16 queries), 1536 cycles at the matrix peak, and about 330 vector
// instructions, 1700 cycles; two waves per SIMD overlap them only in part.  512 tokens over 8500 positions, 32 query and 8
// kv heads of 128, fp4 (69 GFLOP, 104 with the second term of the probabilities) take 107 us, the matrix pipe busy for
// 38 % of it, and 117 with the join.  The reference of the softmax moves only when outgrown (125 us before), and the
// terms are converted in pairs.  One term instead of two would take 96, at 1.4 to 2 times a bf16 output's error; two row
// tiles a wave at one wave per SIMD, or the scores of the next 32 keys beside the softmax of these, took 148 and 135.
#pragma once

#include "tgm_kv_attend.h"

namespace tgm {

// LDS: two stages of keys and values, and whether the pages of a stage's four groups of 16 positions exist.
template <int HD>
struct ManyLds {
  static constexpr int STAGES = 4 * kManyKeys * HD * 2, BYTES = STAGES + 2 * 4 * 4;
};

// Workgroup `at` of the row tiles and splits of kv head j; sequence b where the positions are not common.
template <int DT, int KB, int VB, int HD>
__device__ __forceinline__ void many_body(const AttendArgs& A, unsigned char* lds, int tiles, int at, int j, int seq) {
  constexpr int NQ = AttendTerms<DT>::Q, NP = AttendTerms<DT>::P;
  constexpr int NJ = HD / 16, ND = HD / 32;
  constexpr int ROW = HD * 2, CH = ROW / 16;
  constexpr int BLOCK = kManyKeys * ROW, STAGE = 2 * BLOCK;
  constexpr int KROW = HD * KB / 8, VROW = HD * VB / 8, KL = KROW / 4, VL = VROW / 4;
  int(*okgroup)[4] = (int(*)[4])(lds + ManyLds<HD>::STAGES);
  const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5, l32 = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int z = at / tiles, tile = tiles - 1 - at % tiles;  // the longest rows first
  const int TG = A.T * A.G;
  const int nrows = A.common ? A.B * TG : TG;
  const int r0 = tile * kManyRows + wave * 32;
  const int r = min(r0 + l32, nrows - 1);
  const bool rvalid = r0 + l32 < nrows;
  const int b = A.common ? r / TG : seq;
  const int rt = r - (A.common ? b * TG : 0), t = rt / A.G, h = j * A.G + rt % A.G;
  const int last = min(at_length(A, b), A.kcap + A.T) - A.T + t;  // the last position this row sees
  // positions any row of the workgroup sees: of a prefix those of its longest sequence (behind it nothing may be written)
  int kend = A.kcap;
  if (A.common) {
    int most = 0;
    for (int s = tile * kManyRows / TG + lane; s <= (min(tile * kManyRows + kManyRows, nrows) - 1) / TG; s += 64)
      most = max(most, at_length(A, s));
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) most = max(most, __shfl_xor(most, o, 64));
    kend = min(kend, __builtin_amdgcn_readfirstlane(most));
  } else kend = min(kend, at_length(A, b) - A.T + (min(tile * kManyRows + kManyRows, nrows) - 1) / A.G + 1);
  const int k_lo = A.k0 + z * A.chunk, k_hi = min(k_lo + A.chunk, kend);
  const int nblocks = k_hi > k_lo ? (k_hi - k_lo + kManyKeys - 1) / kManyKeys : 0;
  int wave_min = last;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) wave_min = min(wave_min, __shfl_xor(wave_min, o, 64));

  auto swz_k = [](int key) { return CH == 16 ? key & 15 : (key >> 1) & 7; };
  auto swz_v = [](int key) { return CH == 16 ? (key & 3) * 5 : (((key >> 1) & 1) << 2) | (key & 3); };
  const int32_t* trow = A.pg.table + (A.common ? 0 : b * A.pg.ld);
  const int key = tid >> 2, qd = tid & 3;
  struct Raw {
    unsigned k[KL / 4], v[VL / 4];
    float ks, vs;
    int ok;
  };
  auto load = [&](int kb, Raw& w) __attribute__((always_inline)) {
    const int p = k_lo + kb * kManyKeys + key, page = kv_page(A.pg, trow, p);
    const int64_t ph = (int64_t)(page < 0 ? 0 : page) * A.HK + j;
    const int slot = p & A.pg.mask;
    const int64_t row = (ph << A.pg.shift) + slot, sc = ((ph * (HD / kKvBlock) + qd * (HD / 4) / kKvBlock) << A.pg.shift) + slot;
    at_load<KL>(A.ks.data + row * KROW + qd * KL, w.k);
    at_load<VL>(A.vs.data + row * VROW + qd * VL, w.v);
    w.ks = kv_scale(A.ks.scales[sc]);
    w.vs = kv_scale(A.vs.scales[sc]);
    w.ok = page >= 0;
    if (!w.ok || p >= k_hi) {
      w.vs = 1.f;
#pragma unroll
      for (int e = 0; e < VL / 4; ++e) w.v[e] = 0;
    }
  };
  auto stage = [&](int kb, const Raw& w) __attribute__((always_inline)) {
    unsigned char* st = lds + (kb & 1) * STAGE;
#pragma unroll
    for (int i = 0; i < HD / 32; ++i) {
      const int ch = qd * (HD / 32) + i;
      *(u32x4*)(st + key * ROW + ((ch ^ swz_k(key)) * 16)) = at_codes8<KB>(w.k, i, w.ks);
      *(u32x4*)(st + BLOCK + key * ROW + ((ch ^ swz_v(key)) * 16)) = at_codes8<VB>(w.v, i, w.vs);
    }
    if (lane == 0) okgroup[kb & 1][wave] = w.ok;
  };
  Raw raw;
  if (nblocks > 0) {
    load(0, raw);
    stage(0, raw);
  }

  // q's terms as the B operand of S^T: lane (row, half) holds q[16 s + 8 half + i]
  at_bf16x8 qt[NJ][NQ];
  {
    const int64_t qi = b * A.qb + t * A.qt + h * A.qh;
#pragma unroll
    for (int s = 0; s < NJ; ++s) {
      float x[8];
      kv_load8<DT>(A.q, qi + 16 * s + 8 * half, A.qvec, x);
      at_split<NQ>(x, qt[s]);
    }
  }
  const int vi = lane & 15, vg = lane >> 4;
  const int vkey = 4 * half + (vi >> 2);
  unsigned voff[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d)
    voff[d] = (unsigned)(BLOCK + vkey * ROW + ((4 * d + 2 * (vg & 1) + ((vi & 3) >> 1)) ^ swz_v(vkey)) * 16 + (vi & 1) * 8);

  f32x16 O[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d) O[d] = f32x16{};
  float m = -INFINITY, l = 0.f;
#pragma unroll 1
  for (int kb = 0; kb < nblocks; ++kb) {
    __syncthreads();  // block kb is staged; everybody is done with block kb - 1
    const int first = k_lo + kb * kManyKeys;
    load(kb + 1, raw);  // past the last block: positions that are not seen, staged and not used
    const unsigned char* st = lds + (kb & 1) * STAGE;
    f32x16 S[2] = {f32x16{}, f32x16{}};
#pragma unroll
    for (int s = 0; s < NJ; ++s)
#pragma unroll
      for (int kt = 0; kt < 2; ++kt) {
        const at_bf16x8 a = *(const at_bf16x8*)(st + (kt * 32 + l32) * ROW + (((2 * s + half) ^ swz_k(l32)) * 16));
#pragma unroll
        for (int q = 0; q < NQ; ++q) S[kt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, qt[s][q], S[kt], 0, 0, 0);
      }
    const int* okg = okgroup[kb & 1];
    const int ok0 = okg[0], ok1 = okg[1], ok2 = okg[2], ok3 = okg[3];
    if (first + kManyKeys - 1 > wave_min || first + kManyKeys > k_hi || !(ok0 & ok1 & ok2 & ok3)) {  // uniform
#pragma unroll
      for (int kt = 0; kt < 2; ++kt)
#pragma unroll
        for (int v = 0; v < 16; ++v) {
          const int p = first + kt * 32 + 8 * (v >> 2) + 4 * half + (v & 3);
          const int ok = kt == 0 ? (v < 8 ? ok0 : ok1) : (v < 8 ? ok2 : ok3);
          const bool gone = (p > last) | (p >= k_hi) | !ok;
          S[kt][v] = gone ? -INFINITY : S[kt][v];
        }
    }
    float b4[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      b4[i] = S[i >> 1][8 * (i & 1)];
#pragma unroll
      for (int v = 1; v < 8; ++v) b4[i] = fmaxf(b4[i], S[i >> 1][8 * (i & 1) + v]);
    }
    float bm = fmaxf(fmaxf(b4[0], b4[1]), fmaxf(b4[2], b4[3]));
    float other = bm;
    swap32(bm, other);  // bm: the lower half's in both halves, other: the upper half's
    bm = fmaxf(bm, other);
    bm *= A.sl;
    // The reference of the exponentials moves only when a maximum has outgrown it by 2^8: weights of up to 2^8 lose
    // nothing in fp32 and bf16, and the output is rarely rescaled.
    if (__any(bm > m + kLazyLog2)) {
      const float mn = fmaxf(m, bm);
      const float alpha = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - mn);
      l *= alpha;
#pragma unroll
      for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int v = 0; v < 16; ++v) O[d][v] *= alpha;
      m = mn;
    }
    const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        float x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          x[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(S[kt][8 * u + i], A.sl, -ref));
        }
        l += ((x[0] + x[1]) + (x[2] + x[3])) + ((x[4] + x[5]) + (x[6] + x[7]));
        at_bf16x8 pb[NP];
        at_split<NP>(x, pb);
#pragma unroll
        for (int d = 0; d < ND; ++d) {  // keys 16 u + 4 h .. + 4 of tile kt, then the ones 8 on
          const unsigned char* row = st + voff[d] + (kt * 32 + u * 16) * ROW;
          const at_bf16x8 a = at_tr_pair(row, row + 8 * ROW);
#pragma unroll
          for (int q = 0; q < NP; ++q) O[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, pb[q], O[d], 0, 0, 0);
        }
      }
    stage(kb + 1, raw);
  }
  l += __shfl_xor(l, 32, 64);
  if (!rvalid) return;
  const int64_t row = ((int64_t)b * A.T + t) * A.H + h;
  if (A.slots == 1) {
    const float inv = 1.0f / l;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int g = 0; g < 4; ++g)
#pragma unroll
        for (int i = 0; i < 4; ++i) at_store<DT>(A.out, row * HD + d * 32 + 8 * g + 4 * half + i, l == 0.f ? 0.f : O[d][4 * g + i] * inv);
  } else {
    const int slot = A.slot0 + z;
    float* o = A.part + (row * A.slots + slot) * HD;
    if (l != 0.f) {
#pragma unroll
      for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int g = 0; g < 4; ++g)
          *(f32x4*)(o + d * 32 + 8 * g + 4 * half) = f32x4{O[d][4 * g], O[d][4 * g + 1], O[d][4 * g + 2], O[d][4 * g + 3]};
    }
    if (half == 0) {
      float* ml = at_ml(A, HD, row, slot);
      ml[0] = m;
      ml[1] = l;
    }
  }
}

template <int DT, int KB, int VB, int HD>
__global__ void __launch_bounds__(256, 2) kv_attend_many(const AttendArgs A, int tiles) {
  __shared__ __attribute__((aligned(16))) unsigned char lds[ManyLds<HD>::BYTES];
  many_body<DT, KB, VB, HD>(A, lds, tiles, blockIdx.x, blockIdx.y, blockIdx.z);
}

template <int DT, int KB, int VB, int HD>
static void many_go(const AttendLaunch& l, hipStream_t st) {
  const int64_t rows = (int64_t)l.a.T * l.a.G * (l.a.common ? l.a.B : 1);
  const int tiles = (int)((rows + kManyRows - 1) / kManyRows);
  const dim3 grid((unsigned)(tiles * l.splits), (unsigned)l.a.HK, l.a.common ? 1u : (unsigned)l.a.B);
  hipLaunchKernelGGL((kv_attend_many<DT, KB, VB, HD>), grid, dim3(256), 0, st, l.a, tiles);
}
template <int DT, int HD>
static void many_formats(const AttendLaunch& l, hipStream_t st) {
  if (l.kb == 8 && l.vb == 8) many_go<DT, 8, 8, HD>(l, st);
  else if (l.kb == 8) many_go<DT, 8, 4, HD>(l, st);
  else if (l.vb == 8) many_go<DT, 4, 8, HD>(l, st);
  else many_go<DT, 4, 4, HD>(l, st);
}
template <int DT>
void attend_many(const AttendLaunch& l, hipStream_t st) {
  if (l.hd == 64) many_formats<DT, 64>(l, st);
  else many_formats<DT, 128>(l, st);
}

}  // namespace tgm
