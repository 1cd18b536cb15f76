// Attention over the quantised paged cache: how a call is split, and the join of the splits (tgm_kv_attend).
#include "tgm_kv_attend.h"

namespace tgm {

// Bound by the partial sums' bytes: 8.8 us for 16384 rows of four splits (34 MB, out of the caches).
//
// One wave per row: weights of its splits (lane s: slot s), then their weighted sum, four dims a lane and the wave's
// halves (quarters for 64 dims) on slots of their own, several loads in flight.  Slots of the common prefix (below
// `pslots`) are always written, those of a sequence's own positions as far as it reaches.
template <int DT, int HD>
__global__ void __launch_bounds__(256) attend_merge(const AttendArgs A, int pslots) {
  constexpr int L = HD / 4, N = 64 / L, U = 4;  // lanes a slot, slots at a time, loads a lane in flight
  const int lane = threadIdx.x & 63, sub = lane / L, d = 4 * (lane % L);
  const int64_t row = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (row >= at_rows(A)) return;
  const int b = (int)(row / ((int64_t)A.T * A.H));
  const int own = min(at_length(A, b), A.kcap) - A.k0;
  const int n = pslots + (own > 0 ? (own + A.chunk - 1) / A.chunk : 0);
  float m = -INFINITY, l = 0.f;
  if (lane < n) {
    const kv_f32x2 ml = *(const kv_f32x2*)at_ml(A, HD, row, lane);
    m = ml[0];
    l = ml[1];
  }
  float M = m;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor(M, o, 64));
  const float w = l == 0.f ? 0.f : __builtin_amdgcn_exp2f(m - M);
  float sum = l * w;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
  f32x4 acc = f32x4{0.f, 0.f, 0.f, 0.f};
  const float* p = A.part + row * A.slots * HD + d;
  for (int s0 = 0; s0 < n; s0 += N * U) {
    f32x4 x[U];
    float ws[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int s = s0 + u * N + sub;  // 63 at most where s0 < n <= 64
      ws[u] = __shfl(w, s, 64);        // 0 past the last one, and where a slot's sums were not written
      x[u] = f32x4{0.f, 0.f, 0.f, 0.f};
      if (ws[u] != 0.f) x[u] = *(const f32x4*)(p + s * HD);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) acc += x[u] * ws[u];
  }
#pragma unroll
  for (int o = L; o < 64; o <<= 1)
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[e] += __shfl_xor(acc[e], o, 64);
  if (sub == 0) {
    const float inv = sum == 0.f ? 0.f : 1.0f / sum;  // NaN in any split: NaN
#pragma unroll
    for (int e = 0; e < 4; ++e) at_store<DT>(A.out, row * HD + d + e, acc[e] * inv);
  }
}

constexpr int64_t kAlonePairs = 196608;  // (sequence, shared position, kv head) triples that are read without sharing
constexpr int kMaxSlots = 64;  // splits of a row: a lane each in attend_merge

struct AttendPlan {
  bool many;           // a sequence's own positions by attend_many
  int chunk, splits;   // of a sequence's own positions
  int prefix;          // positions that the batch shares, read once for all; below it but for these: own
  int pchunk, psplits; // of the common prefix
  int64_t bytes;
};

static int64_t round_up(int64_t x, int64_t m) { return (x + m - 1) / m * m; }

// Splits of `span` positions over about `want` workgroups per row tile, in chunks that are a multiple of `unit`.  The span
// is the table's, since the lengths are on the device: in a table that is wider than its sequences fewer splits hold work
// (512 tokens over 8500 positions take 123 us in a table of 8512, 348 in one of 32768; one token over 2000 of one
// sequence 11 in a table of up to 8192, 15 of 32768, 36 of 131072).
static void split_span(int64_t span, int64_t want, int64_t unit, int64_t most, int& chunk, int& splits) {
  int64_t n = want < 1 ? 1 : (want > most ? most : want);
  const int64_t c = round_up((span + n - 1) / n, unit);
  chunk = (int)(c < unit ? unit : c);
  splits = (int)(span > 0 ? (span + chunk - 1) / chunk : 1);
}

static AttendPlan attend_plan(const tgm_kv_cache* c, int64_t dt, int64_t heads, int64_t batch, int64_t tokens, int64_t cols,
                              int64_t shared) {
  AttendPlan p{};
  const int64_t G = heads / c->kv_heads, rows = tokens * G, cap = cols * c->page_size;
  // attend_few as far as its columns reach: 16 rows of 16 sequences of 8000 positions take 73 us there and 109 in
  // attend_many (one sequence 15 and 20), f32 with 10 rows 77 and 215 (16 and 32); from there on attend_many takes what its
  // 128 rows take, 110 us for 24 rows (f32 217)
  p.many = rows > attend_few_rows((int)dt);
  // A prefix that a few rows read goes with each sequence, through row 0's pages and out of the caches: the products over
  // 128 rows at a time, most of them empty, take longer.  In common and so, us, fp8, 8 kv heads of 4: 8 sequences on 2048
  // positions 16.2 and 14.1 (bf16), 12 of them 17.5 and 16.9, 16 of them 19.6 and 19.6, 24 of them 20.7 and 24.0; 8 on 4096
  // positions 18.2 and 19.9; f32, whose rows split into three terms, 16 on 2048 26.5 and 24.0, 24 of them 28.2 and 30.7, 12
  // on 4096 32.2 and 30.5.  (One kv head on 16384 positions crosses later: 16 sequences 23.7 and 20.9, 32 of them 25.2 and
  // 29.6.)
  const int64_t alone = dt == TGM_F32 ? 2 * kAlonePairs : kAlonePairs;
  p.prefix = shared > 0 && (p.many || batch * shared * c->kv_heads > alone) ? (int)shared : 0;
  const int64_t own = cap > p.prefix ? cap - p.prefix : 0;
  // attend_many: as many workgroups as run at once, two a CU
  if (p.prefix > 0) {
    const int64_t tiles = (batch * rows + kManyRows - 1) / kManyRows * c->kv_heads;
    split_span(shared, (512 + tiles - 1) / tiles, kManyKeys, kMaxSlots - 16, p.pchunk, p.psplits);
  }
  const int64_t most = kMaxSlots - p.psplits, heads_of_all = c->kv_heads * batch;
  if (p.many) {
    const int64_t tiles = (rows + kManyRows - 1) / kManyRows * heads_of_all;
    split_span(own, 512 / tiles, kManyKeys, most, p.chunk, p.splits);
  } else {
    // six rounds of two workgroups a CU, a split at least one block a wave: fewer leave CUs idle at the end of long ragged
    // batches (16 sequences of up to 32700 positions: 150 us with half as many, 132 so, 133 with twice as many; short ones
    // would take fewer: 32 of up to 4000 37, 45 and 46)
    split_span(own, (6 * 512 + heads_of_all - 1) / heads_of_all, kFewWaves * kFewBlock, most, p.chunk, p.splits);
  }
  const int slots = p.splits + p.psplits;
  p.bytes = slots == 1 ? 0 : batch * tokens * heads * slots * (c->head_dim + 2) * 4;
  return p;
}

template <int DT>
static void attend_go(const AttendPlan& p, AttendLaunch l, int shared, int cap, hipStream_t st) {
  AttendArgs& a = l.a;
  a.slots = p.splits + p.psplits;
  AttendLaunch c = l;
  c.a.k0 = 0, c.a.kcap = p.prefix, c.a.chunk = p.pchunk, c.a.slot0 = 0, c.a.common = 1;
  c.splits = p.psplits;
  a.k0 = p.prefix, a.kcap = cap, a.chunk = p.chunk, a.slot0 = p.psplits, a.common = 0, a.prefix = shared;
  l.splits = p.splits;
  if (p.psplits && a.T * a.G <= attend_few_tile(DT)) {
    attend_both<DT>(c, l, st);
  } else {
    if (p.psplits) attend_many<DT>(c, st);
    if (p.many) attend_many<DT>(l, st);
    else attend_few<DT>(l, st);
  }
  if (a.slots > 1) {
    const dim3 grid((unsigned)(((int64_t)a.B * a.T * a.H + 3) / 4));
    if (l.hd == 64) hipLaunchKernelGGL((attend_merge<DT, 64>), grid, dim3(256), 0, st, a, p.psplits);
    else hipLaunchKernelGGL((attend_merge<DT, 128>), grid, dim3(256), 0, st, a, p.psplits);
  }
}

static bool attend_sizes_ok(const tgm_kv_cache* c, int64_t heads, int64_t batch, int64_t tokens, int64_t cols, int64_t shared) {
  return c && c->kv_heads > 0 && c->page_size > 0 && c->page_size <= 1024 && (c->head_dim == 64 || c->head_dim == 128) &&
         heads > 0 && heads % c->kv_heads == 0 && heads <= 65535 && batch >= 0 && batch <= 65535 && tokens >= 0 &&
         tokens < (1ll << 24) && batch * tokens < (1ll << 24) && batch * tokens * heads < (1ll << 30) && cols >= 0 &&
         cols < (1ll << 30) && cols * c->page_size < (1ll << 30) && shared >= 0 && shared <= cols * c->page_size && shared % c->page_size == 0;
}

}  // namespace tgm

using namespace tgm;

extern "C" int64_t tgm_kv_attend_workspace(const tgm_kv_cache* cache, int64_t q_dtype, int64_t heads, int64_t batch,
                                           int64_t tokens, int64_t table_cols, int64_t shared) {
  if (!attend_sizes_ok(cache, heads, batch, tokens, table_cols, shared) || batch == 0 || tokens == 0) return 0;
  return attend_plan(cache, q_dtype, heads, batch, tokens, table_cols, shared).bytes;
}

extern "C" int tgm_kv_attend(const tgm_kv_cache* cache, const tgm_heads* q, const void* q_data, const int32_t* table,
                             int64_t ld_table, int64_t table_cols, const int32_t* lengths, int64_t batch, int64_t tokens,
                             int64_t shared, double scale, void* workspace, int64_t workspace_bytes, void* out,
                             void* stream) {
  clear_error();
  AttendLaunch l{};
  AttendArgs& a = l.a;
  if (const int e = kv_check(cache, table, ld_table, table_cols, a.ks, a.vs, a.pg)) return e;
  TGM_CHECK_ARG(q, "null argument");
  TGM_CHECK_ARG(q->dtype == TGM_F32 || q->dtype == TGM_F16 || q->dtype == TGM_BF16, "q must be f32, f16 or bf16");
  TGM_CHECK_ARG(q->heads > 0 && q->heads % cache->kv_heads == 0, "heads must be a multiple of kv_heads");
  TGM_CHECK_ARG(shared >= 0 && shared % cache->page_size == 0 && shared <= table_cols * cache->page_size,
                "shared must be a multiple of page_size within the table");
  TGM_CHECK_ARG(attend_sizes_ok(cache, q->heads, batch, tokens, table_cols, shared), "sizes out of range");
  TGM_CHECK_ARG(scale > 0 && scale < 1e30, "scale must be positive");
  if (batch == 0 || tokens == 0) return TGM_OK;
  TGM_CHECK_ARG(q_data && lengths && out && ((uintptr_t)out & 15) == 0, "null or misaligned operand");
  const AttendPlan p = attend_plan(cache, q->dtype, q->heads, batch, tokens, table_cols, shared);
  TGM_CHECK_ARG(p.bytes == 0 || (workspace && workspace_bytes >= p.bytes && ((uintptr_t)workspace & 15) == 0),
                "workspace too small or misaligned");
  a.q = q_data, a.qb = q->stride_b, a.qt = q->stride_t, a.qh = q->stride_h;
  const int64_t step = 16 / dtype_size((int)q->dtype);
  a.qvec = ((uintptr_t)q_data & 15) == 0 && a.qb % step == 0 && a.qt % step == 0 && a.qh % step == 0;
  a.lengths = lengths;
  a.B = (int)batch, a.T = (int)tokens, a.H = (int)q->heads, a.HK = (int)cache->kv_heads, a.G = a.H / a.HK;
  a.sl = (float)(scale * 1.4426950408889634);
  a.part = (float*)workspace;
  a.out = out;
  l.kb = cache->k_format == TGM_KV_FP8_E4M3 ? 8 : 4;
  l.vb = cache->v_format == TGM_KV_FP8_E4M3 ? 8 : 4;
  l.hd = (int)cache->head_dim;
  const int cap = (int)(table_cols * cache->page_size);
  const hipStream_t st = (hipStream_t)stream;
  if (q->dtype == TGM_F32) attend_go<TGM_F32>(p, l, (int)shared, cap, st);
  else if (q->dtype == TGM_F16) attend_go<TGM_F16>(p, l, (int)shared, cap, st);
  else attend_go<TGM_BF16>(p, l, (int)shared, cap, st);
  return launch_status("tgm_kv_attend");
}
