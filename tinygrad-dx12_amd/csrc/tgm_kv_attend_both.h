// A batch on a common prefix in one launch: the workgroups of attend_few for each sequence's own positions, then those of
// attend_many for the prefix, which start as the first ones end: 64 sequences on 16384 common positions take 59.2 us so,
// 59.8 with the prefix first, 63.2 in two launches.  (The two kinds in turn, one of each on a CU, take 80: a workgroup of
// attend_many gets no more of a CU beside one that waits for memory than beside its like, and there are half as many.)
#pragma once

#include "tgm_kv_attend_few.h"
#include "tgm_kv_attend_many.h"

namespace tgm {

template <int DT, int KB, int VB, int HD>
__global__ void __launch_bounds__(256, 2) kv_attend_both(const AttendArgs P, int tiles, int psplits, const AttendArgs A,
                                                         int splits) {
  constexpr int FEW = FewLds<DT, HD, 1>::BYTES, MANY = ManyLds<HD>::BYTES;
  __shared__ __attribute__((aligned(16))) unsigned char lds[FEW > MANY ? FEW : MANY];
  const int nm = tiles * psplits * P.HK, nf = splits * A.HK * A.B;
  const int rf = (nf + 7) / 8, round = blockIdx.x / 8;  // rounds of eight: one an XCD
  const bool many = round >= rf;
  const int at = (many ? round - rf : round) * 8 + (int)(blockIdx.x % 8);
  if (many) {
    if (at < nm) many_body<DT, KB, VB, HD>(P, lds, tiles, at % (tiles * psplits), at / (tiles * psplits), 0);
  } else {
    if (at < nf) few_body<DT, KB, VB, HD, 1>(A, lds, at % splits, at / splits % A.HK, at / (splits * A.HK));
  }
}

template <int DT, int KB, int VB, int HD>
static void both_go(const AttendLaunch& p, const AttendLaunch& l, hipStream_t st) {
  const int tiles = (int)(((int64_t)p.a.B * p.a.T * p.a.G + kManyRows - 1) / kManyRows);
  const int64_t rounds = ((int64_t)tiles * p.splits * p.a.HK + 7) / 8 + ((int64_t)l.splits * l.a.HK * l.a.B + 7) / 8;
  hipLaunchKernelGGL((kv_attend_both<DT, KB, VB, HD>), dim3((unsigned)(8 * rounds)), dim3(256), 0, st, p.a, tiles, p.splits,
                     l.a, l.splits);
}
template <int DT, int HD>
static void both_formats(const AttendLaunch& p, const AttendLaunch& l, hipStream_t st) {
  if (l.kb == 8 && l.vb == 8) both_go<DT, 8, 8, HD>(p, l, st);
  else if (l.kb == 8) both_go<DT, 8, 4, HD>(p, l, st);
  else if (l.vb == 8) both_go<DT, 4, 8, HD>(p, l, st);
  else both_go<DT, 4, 4, HD>(p, l, st);
}
template <int DT>
void attend_both(const AttendLaunch& prefix, const AttendLaunch& own, hipStream_t st) {
  if (own.hd == 64) both_formats<DT, 64>(prefix, own, st);
  else both_formats<DT, 128>(prefix, own, st);
}

}  // namespace tgm
