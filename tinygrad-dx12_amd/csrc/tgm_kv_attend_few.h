// Attention of a few rows per kv head (decode): split over positions, joined by attend_merge.
//
// Grid (splits, kv_heads, batch), 256 threads.  A workgroup takes `chunk` positions of one kv head; its four waves take
// blocks of 64 of them in turn, each with its own running maximum, sum and output, and meet once at the end.
//
//   S^T[key, column] = K . Q^T      16x16x32 MFMA, A = keys: straight from global memory to registers
//   O^T[dim, column] += V^T . P^T   A = V^T: decoded to bf16 into the wave's own LDS, read transposed
//
// A column is a (row, term) pair: the terms of a probability stand beside each other, so that a tile of 16 columns
// carries 8 rows of 2 terms or 5 of 3 and the extra terms cost nothing while there are few rows.  The q operand repeats
// a row in its term columns, so every lane of them computes the same softmax and keeps its own term.
//
// A lane's key operand covers a quarter of head_dim of key 4 c + i (c = lane % 16, tile i): its scales of the four tiles
// are four consecutive bytes, the contraction order being free as long as q's operand follows it.  The scores of
// column c in lane group g are then keys 16 g + 4 v + i, and the products with V take the keys with i = 0, 1 and then
// those with i = 2, 3: V goes through LDS in these two halves.
//
// Bound by memory: 16 sequences of up to 32700 positions, 32 query and 8 kv heads of 128, fp8 (640 MB) take 132 us with
// the join, 4.85 TB/s (a copy reaches 5.1), the vector instructions busy for a quarter of it and the matrix pipe for 6 %.
// What keeps the memory busy is waves: three per SIMD that load a block of 64 positions (16 KB) and compute it beat two
// that hold the next block in registers (140), and four, which spill (220).  f32 queries stay at two (16 x 16000 positions:
// 121 us, at three, spilling, 123; 16 x 8000 61 and 58).  Short ones are a chain of latencies: 1000 positions of one sequence take 8 us, and
// the join 3.
#pragma once

#include "tgm_kv_attend.h"

namespace tgm {

// Sizes of the workgroup's LDS: q's operands, each wave's staged values (or its part of the output), each wave's maxima
// and sums.
template <int DT, int HD, int CT>
struct FewLds {
  static constexpr int VALUES = 32 * HD * 2, PART = 16 * (HD + 4) * 4;
  static constexpr int WAVE = VALUES > PART ? VALUES : PART;
  static constexpr int Q = CT * (HD / 32) * AttendTerms<DT>::Q * 1024;
  static constexpr int BYTES = Q + kFewWaves * WAVE + 2 * kFewWaves * 16 * CT * 4;
};

// Split z of kv head j of sequence b.
template <int DT, int KB, int VB, int HD, int CT>
__device__ __forceinline__ void few_body(const AttendArgs& A, unsigned char* lds, int z, int j, int b) {
  constexpr int NQ = AttendTerms<DT>::Q, NP = AttendTerms<DT>::P, RP = 16 / NP;
  constexpr int STEPS = HD / 32, ND = HD / 16;
  constexpr int KROW = HD * KB / 8, VROW = HD * VB / 8;
  constexpr int KL = KROW / 4, VL = VROW * 16 / HD;  // bytes a lane loads of a key and of a value row
  constexpr int LPR = HD / 16, KPL = 64 * LPR / 64;  // lanes per value row; value rows per lane and block
  constexpr int WLDS = FewLds<DT, HD, CT>::WAVE;
  unsigned char* qlds = lds;
  unsigned char* wlds = lds + FewLds<DT, HD, CT>::Q;
  float(*sm)[16 * CT] = (float(*)[16 * CT])(wlds + kFewWaves * WLDS);
  float(*ss)[16 * CT] = sm + kFewWaves;
  const int tid = threadIdx.x, lane = tid & 63, c = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int rows = A.T * A.G;
  const int len = at_length(A, b);
  const int kend = min(len, A.kcap);
  const int k_lo = A.k0 + z * A.chunk, k_hi = min(k_lo + A.chunk, kend);
  if (k_lo >= kend && A.slots > 1) return;  // attend_merge knows

  const int32_t* trow = A.pg.table + b * A.pg.ld;
  // positions below A.prefix lie in row 0's pages
  auto page_of = [&](int pos) __attribute__((always_inline)) { return kv_page(A.pg, pos < A.prefix ? A.pg.table : trow, pos); };
  struct Raw {
    unsigned k[4][KL / 4], v[KPL][VL / 4], ksc, vsc[KPL / 4];
    bool kok, vok;
  };
  auto load = [&](int base, Raw& r) __attribute__((always_inline)) {
    const int kp = base + 4 * c, kpage = page_of(kp);
    r.kok = kpage >= 0;
    const int64_t kph = (int64_t)(kpage < 0 ? 0 : kpage) * A.HK + j;
    const int kslot = kp & A.pg.mask;
    const uint8_t* kd = A.ks.data + ((kph << A.pg.shift) + kslot) * KROW + g * KL;
#pragma unroll
    for (int i = 0; i < 4; ++i) at_load<KL>(kd + i * KROW, r.k[i]);
    r.ksc = *(const unsigned*)(A.ks.scales + ((kph * (HD / kKvBlock) + g * (HD / 4) / kKvBlock) << A.pg.shift) + kslot);
    const int vp = base + KPL * (lane / LPR), vpage = page_of(vp), ch = lane % LPR;
    r.vok = vpage >= 0;
    const int64_t vph = (int64_t)(vpage < 0 ? 0 : vpage) * A.HK + j;
    const int vslot = vp & A.pg.mask;
    const uint8_t* vd = A.vs.data + ((vph << A.pg.shift) + vslot) * VROW + ch * VL;
#pragma unroll
    for (int i = 0; i < KPL; ++i) at_load<VL>(vd + i * VROW, r.v[i]);
    const uint8_t* vs = A.vs.scales + ((vph * (HD / kKvBlock) + ch / 2) << A.pg.shift) + vslot;
#pragma unroll
    for (int i = 0; i < KPL / 4; ++i) r.vsc[i] = *(const unsigned*)(vs + 4 * i);
  };

  // q's operands, in lane order
  for (int f = wave; f < CT * STEPS; f += kFewWaves) {
    const int ct = f / STEPS, i = f % STEPS;
    const int r = ct * RP + c / NP;
    float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (c < RP * NP && r < rows)
      kv_load8<DT>(A.q, b * A.qb + (r / A.G) * A.qt + (j * A.G + r % A.G) * A.qh + g * (HD / 4) + 8 * i, A.qvec, x);
    at_bf16x8 t[NQ];
    at_split<NQ>(x, t);
#pragma unroll
    for (int s = 0; s < NQ; ++s) *(at_bf16x8*)(qlds + (f * NQ + s) * 1024 + lane * 16) = t[s];
  }
  // the last position each of this lane's columns sees, and the first of them
  int last[CT], least = 0x7fffffff;
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    const int r = ct * RP + c / NP;
    last[ct] = c < RP * NP && r < rows ? len - A.T + r / A.G : kend - 1;
  }
  least = len - A.T;  // row 0's
  __syncthreads();

  f32x4 O[CT][ND];
  float m[CT], l[CT];
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    m[ct] = -INFINITY;
    l[ct] = 0.f;
#pragma unroll
    for (int d = 0; d < ND; ++d) O[ct][d] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  unsigned char* vlds = wlds + wave * WLDS;
  // chunk of 16 bytes of a staged row, swizzled so that neither the stores nor the transposing reads conflict
  auto swz = [](int row) {
    return HD == 128 ? (((row >> 1) & 3) << 1) | (((row >> 3) & 1) << 3) | ((row >> 2) & 1) : (((row >> 1) & 3) << 1);
  };
  const int i16 = lane & 15;
  unsigned vread[2][ND];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int row = 8 * g + 2 * (i16 >> 2) + e;
#pragma unroll
    for (int d = 0; d < ND; ++d)
      vread[e][d] = (unsigned)(row * HD * 2 + (((2 * d + ((i16 & 3) >> 1)) ^ swz(row)) * 16) + (i16 & 1) * 8);
  }
#pragma unroll 1
  for (int base = k_lo + wave * kFewBlock; base < k_hi; base += kFewWaves * kFewBlock) {
    Raw cur;
    load(base, cur);
    const unsigned long long kok = __ballot(cur.kok);
    const bool whole = base + kFewBlock <= k_hi && __all(cur.kok);  // every position exists (uniform)
    if (!whole) {
      const int vp = base + KPL * (lane / LPR);
#pragma unroll
      for (int i = 0; i < KPL; ++i)
        if (!cur.vok || vp + i >= k_hi) {
#pragma unroll
          for (int e = 0; e < VL / 4; ++e) cur.v[i][e] = 0;
          cur.vsc[i / 4] &= ~(0xFFu << (8 * (i & 3)));
        }
    }
    // scores
    f32x4 S[CT][4];
#pragma unroll
    for (int ct = 0; ct < CT; ++ct)
#pragma unroll
      for (int i = 0; i < 4; ++i) S[ct][i] = f32x4{0.f, 0.f, 0.f, 0.f};
    float ksc[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) ksc[i] = kv_scale((cur.ksc >> (8 * i)) & 0xFFu);
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
      at_bf16x8 q[CT][NQ];
#pragma unroll
      for (int ct = 0; ct < CT; ++ct)
#pragma unroll
        for (int t = 0; t < NQ; ++t) q[ct][t] = *(const at_bf16x8*)(qlds + ((ct * STEPS + s) * NQ + t) * 1024 + lane * 16);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const at_bf16x8 a = __builtin_bit_cast(at_bf16x8, at_codes8<KB>(cur.k[i], s, ksc[i]));
#pragma unroll
        for (int ct = 0; ct < CT; ++ct)
#pragma unroll
          for (int t = 0; t < NQ; ++t) S[ct][i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, q[ct][t], S[ct][i], 0, 0, 0);
      }
    }
    // softmax: positions 16 g + 4 v + i of the block
    const bool mask = !whole || base + kFewBlock - 1 > least;
    const bool gok = (kok >> (4 * g)) & 1;
    const int term = c % NP;
    at_bf16x8 pb[CT][2];
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
      if (mask) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int v = 0; v < 4; ++v) {
            const int p = base + 16 * g + 4 * v + i;
            const bool gone = (p > last[ct]) | (p >= k_hi) | !gok;
            S[ct][i][v] = gone ? -INFINITY : S[ct][i][v];
          }
      }
      float bm = -INFINITY;
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int v = 0; v < 4; ++v) bm = fmaxf(bm, S[ct][i][v]);
      bm = fmaxf(bm, __shfl_xor(bm, 16, 64));
      bm = fmaxf(bm, __shfl_xor(bm, 32, 64));
      bm *= A.sl;
      // the reference of the exponentials moves only when a maximum has outgrown it by 2^8: weights of up to 2^8 lose
      // nothing in fp32 and bf16, and the output is rarely rescaled
      if (__any(bm > m[ct] + kLazyLog2)) {
        const float mn = fmaxf(m[ct], bm);
        const float alpha = m[ct] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m[ct] - mn);
        l[ct] *= alpha;
#pragma unroll
        for (int d = 0; d < ND; ++d) O[ct][d] *= alpha;
        m[ct] = mn;
      }
      const float ref = m[ct] == -INFINITY ? 0.f : m[ct];
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
        u32x4 words;
#pragma unroll
        for (int e = 0; e < 4; ++e) {  // two values: tile i = 2 hf + e / 2, v = 2 (e % 2) and the next
          const f32x4& s4 = S[ct][2 * hf + (e >> 1)];
          // v_exp_f32: within one unit in the last place; 0 for masked positions
          float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s4[2 * (e & 1)], A.sl, -ref));
          float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s4[2 * (e & 1) + 1], A.sl, -ref));
          l[ct] += p0 + p1;
#pragma unroll
          for (int t = 0; t + 1 < NP; ++t) {
            const unsigned w = bf16x2_bits(p0, p1);
            const float r0 = p0 - bits_f32(w << 16), r1 = p1 - bits_f32(w & 0xFFFF0000u);
            p0 = term > t ? r0 : p0;
            p1 = term > t ? r1 : p1;
          }
          words[e] = bf16x2_bits(p0, p1);
        }
        pb[ct][hf] = __builtin_bit_cast(at_bf16x8, words);
      }
    }
    // values: rows with key % 4 in {2 hf, 2 hf + 1}, staged as row 2 (key / 4) + key % 2
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
#pragma unroll
      for (int i = 0; i < KPL; ++i) {
        if (((i >> 1) & 1) != hf) continue;
        const int key = KPL * (lane / LPR) + i, row = 2 * (key >> 2) + (key & 1);
        const float s = kv_scale((cur.vsc[i / 4] >> (8 * (i & 3))) & 0xFFu);
        const int ch = 2 * (lane % LPR);
        *(u32x4*)(vlds + row * HD * 2 + ((ch ^ swz(row)) * 16)) = at_codes8<VB>(cur.v[i], 0, s);
        *(u32x4*)(vlds + row * HD * 2 + (((ch + 1) ^ swz(row)) * 16)) = at_codes8<VB>(cur.v[i], 1, s);
      }
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_wave_barrier();
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
      for (int d = 0; d < ND; ++d) {
        const at_bf16x8 a = at_tr_pair(vlds + vread[0][d], vlds + vread[1][d]);
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) O[ct][d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, pb[ct][hf], O[ct][d], 0, 0, 0);
      }
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_wave_barrier();
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    }
  }

  // the four waves' parts of each row, summed in their order
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    l[ct] += __shfl_xor(l[ct], 16, 64);
    l[ct] += __shfl_xor(l[ct], 32, 64);
    if (g == 0) {
      sm[wave][ct * 16 + c] = m[ct];
      ss[wave][ct * 16 + c] = l[ct];
    }
  }
  __syncthreads();
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    float M = -INFINITY;
#pragma unroll
    for (int w = 0; w < kFewWaves; ++w) M = fmaxf(M, sm[w][ct * 16 + c]);
    const float ref = M == -INFINITY ? 0.f : M;
    const float f = __builtin_amdgcn_exp2f(m[ct] - ref);
    float* red = (float*)(wlds + wave * WLDS);
#pragma unroll
    for (int d = 0; d < ND; ++d) *(f32x4*)(red + c * (HD + 4) + 16 * d + 4 * g) = O[ct][d] * f;
    __syncthreads();
    for (int idx = tid; idx < RP * HD; idx += 256) {
      const int rr = idx / HD, d = idx % HD, r = ct * RP + rr;
      if (r < rows) {
        const int col = rr * NP;
        float M2 = -INFINITY, L = 0.f, o = 0.f;
#pragma unroll
        for (int w = 0; w < kFewWaves; ++w) M2 = fmaxf(M2, sm[w][ct * 16 + col]);
        const float ref2 = M2 == -INFINITY ? 0.f : M2;
#pragma unroll
        for (int w = 0; w < kFewWaves; ++w) {
          L += ss[w][ct * 16 + col] * __builtin_amdgcn_exp2f(sm[w][ct * 16 + col] - ref2);
          const float* rw = (const float*)(wlds + w * WLDS) + col * (HD + 4) + d;
#pragma unroll
          for (int t = 0; t < NP; ++t) o += rw[t * (HD + 4)];
        }
        const int64_t row = ((int64_t)b * A.T + r / A.G) * A.H + j * A.G + r % A.G;
        if (A.slots == 1) {
          at_store<DT>(A.out, row * HD + d, L == 0.f ? 0.f : o / L);
        } else {
          A.part[(row * A.slots + A.slot0 + z) * HD + d] = o;
          if (d == 0) {
            float* ml = at_ml(A, HD, row, A.slot0 + z);
            ml[0] = M2;
            ml[1] = L;
          }
        }
      }
    }
    __syncthreads();
  }
}

template <int DT, int KB, int VB, int HD, int CT>
__global__ void __launch_bounds__(256, CT == 1 && DT != TGM_F32 ? 3 : 2) kv_attend_few(const AttendArgs A) {
  __shared__ __attribute__((aligned(16))) unsigned char lds[FewLds<DT, HD, CT>::BYTES];
  few_body<DT, KB, VB, HD, CT>(A, lds, blockIdx.x, blockIdx.y, blockIdx.z);
}

template <int DT, int KB, int VB, int HD>
static void few_ct(const AttendLaunch& l, hipStream_t st) {
  const dim3 grid((unsigned)l.splits, (unsigned)l.a.HK, (unsigned)l.a.B);
  constexpr int RP = 16 / AttendTerms<DT>::P;
  if (l.a.T * l.a.G <= RP) hipLaunchKernelGGL((kv_attend_few<DT, KB, VB, HD, 1>), grid, dim3(256), 0, st, l.a);
  else hipLaunchKernelGGL((kv_attend_few<DT, KB, VB, HD, 2>), grid, dim3(256), 0, st, l.a);
}
template <int DT, int HD>
static void few_formats(const AttendLaunch& l, hipStream_t st) {
  if (l.kb == 8 && l.vb == 8) few_ct<DT, 8, 8, HD>(l, st);
  else if (l.kb == 8) few_ct<DT, 8, 4, HD>(l, st);
  else if (l.vb == 8) few_ct<DT, 4, 8, HD>(l, st);
  else few_ct<DT, 4, 4, HD>(l, st);
}
template <int DT>
void attend_few(const AttendLaunch& l, hipStream_t st) {
  if (l.hd == 64) few_formats<DT, 64>(l, st);
  else few_formats<DT, 128>(l, st);
}

}  // namespace tgm
