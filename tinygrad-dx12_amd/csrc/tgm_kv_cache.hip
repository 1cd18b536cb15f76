// Writing new keys and values into the quantised paged cache, and reading it back
// (tgm_kv_append, tgm_kv_read).
#include "tgm_rotary.h"

namespace tgm {

struct AppendView {
  void* p;
  int64_t sb, st, sh;
  int vec;
};
struct AppendArgs {
  AppendView q, qo, k, v, ko, vo;
  int vec;  // all of q, k and v take 16-byte loads
  int H, HK, seen;  // seen: dtype of ko and vo, or -1
  KvStore ks, vs;
  int kf, vf;
  KvPages pg;
  RotArgs rot;
  const int32_t* start;
  int64_t waves;
  int T, parts;
};

// A lane's 8 values of a block of 32 (four neighbouring lanes hold it): codes in `lo`, `hi` (fp4: lo alone); returns
// the scale byte.  A block whose largest magnitude is below 2^-60 is multiplied by 2^64 first, so that the scale of the
// conversion is a normal number whatever the block holds; the codes are the same.
__device__ __forceinline__ unsigned kv_quantise8(int fmt, const float (&x)[8], unsigned& lo, unsigned& hi) {
  constexpr float kMost = 3.4028234663852886e38f;
  float v[8], am = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    v[e] = x[e] == x[e] ? __builtin_amdgcn_fmed3f(x[e], -kMost, kMost) : 0.f;
    am = fmaxf(am, fabsf(v[e]));
  }
  am = fmaxf(am, xor1(am));
  am = fmaxf(am, xor2(am));
  const int emax = fmt == TGM_KV_FP8_E4M3 ? 8 : 2;
  const float most = fmt == TGM_KV_FP8_E4M3 ? 448.f : 6.f;
  const int adj = am < 0x1p-60f ? 64 : 0;
  if (adj) {
    am *= 0x1p64f;
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] *= 0x1p64f;
  }
  int shared = am > 0.f ? (int)(f32_bits(am) >> 23) - 127 - emax - adj : 0;
  shared = shared < -127 ? -127 : shared;
  const float s = bits_f32((unsigned)(shared + adj + 127) << 23), lim = most * s;
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = __builtin_amdgcn_fmed3f(v[e], -lim, lim);
  if (fmt == TGM_KV_FP8_E4M3) {
    kv_s16x2 a{}, b{};
    a = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(a, v[0], v[1], s, false);
    a = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(a, v[2], v[3], s, true);
    b = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(b, v[4], v[5], s, false);
    b = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(b, v[6], v[7], s, true);
    lo = __builtin_bit_cast(unsigned, a);
    hi = __builtin_bit_cast(unsigned, b);
  } else {
    lo = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, v[0], v[1], s, 0);
    lo = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(lo, v[2], v[3], s, 1);
    lo = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(lo, v[4], v[5], s, 2);
    lo = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(lo, v[6], v[7], s, 3);
    hi = 0;
  }
  return (unsigned)(shared + 127);
}

// Eight values of a head (dims d0 ..) into the cache and, as the cache holds them, into `out`.
__device__ __forceinline__ void kv_put8(int fmt, const KvStore& st, const KvPages& pg, int HD, int HK, int page, int slot,
                                        int h, int d0, const float (&x)[8], const AppendView& out, int64_t to, int seen) {
  unsigned lo, hi;
  const unsigned e = kv_quantise8(fmt, x, lo, hi);
  if (page >= 0) {
    const int64_t ph = (int64_t)page * HK + h;
    const int64_t row = (ph << pg.shift) + slot;
    if (fmt == TGM_KV_FP8_E4M3) *(u32x2*)(st.data + row * HD + d0) = u32x2{lo, hi};
    else *(unsigned*)(st.data + row * (HD / 2) + d0 / 2) = lo;
    if ((d0 & 31) == 0) st.scales[((ph * (HD / kKvBlock) + d0 / kKvBlock) << pg.shift) + slot] = (uint8_t)e;
  }
  if (seen >= 0) {
    float y[8];
    kv_values8(fmt, lo, hi, y);
    const float s = kv_scale(e);
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] *= s;
    if (seen == TGM_F32) kv_store8<TGM_F32>(out.p, to + d0, out.vec, y);
    else if (seen == TGM_BF16) kv_store8<TGM_BF16>(out.p, to + d0, out.vec, y);
    else kv_store8<TGM_F16>(out.p, to + d0, out.vec, y);
  }
}

// A wave takes one token (and every `parts`-th group of its heads): its angles once, then query, key and value heads
// pass by, HD / 16 lanes a head, 16 values a lane.  Query heads are rotated and written out; key heads are rotated and
// quantised, value heads quantised, four lanes a block of 32, whose maximum crosses them by two DPP moves; the codes are
// gfx950's scaled conversions.  Bound by HBM and by a wave's chain from load to store: two prompts of 4001 tokens, 32
// query and 8 key heads of 128 in bf16 (210 MB) take 49.3 us, 4.25 TB/s; 57.8 without the next head's loads under way.
template <int DT, int HD, int MODE>
__global__ void __launch_bounds__(256) kv_append(const AppendArgs A) {
  constexpr int LPH = HD / 16, HPI = 64 / LPH;
  __shared__ double2 angles[4][HD / 2];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t w = (int64_t)blockIdx.x * 4 + wave;
  if (w >= A.waves) return;
  const int64_t token = w / A.parts;
  const int part = (int)(w - token * A.parts);
  const int b = (int)(token / A.T), t = (int)(token - (int64_t)b * A.T);
  const int chunk = lane % LPH, sub = lane / LPH;
  const int heads = A.H + 2 * A.HK;
  // heads of this lane: the next one's values are under way while one is rotated and stored
  const int64_t qi = b * A.q.sb + t * A.q.st, ki = b * A.k.sb + t * A.k.st, vi = b * A.v.sb + t * A.v.st;
  auto fetch = [&](int h, const void*& x, int64_t& at, float (&u)[8], float (&v)[8]) __attribute__((always_inline)) {
    const bool is_q = h < A.H, is_k = h < A.H + A.HK;
    x = is_q ? A.q.p : (is_k ? A.k.p : A.v.p);
    at = is_q ? qi + h * A.q.sh : (is_k ? ki + (h - A.H) * A.k.sh : vi + (h - A.H - A.HK) * A.v.sh);
    const bool vec = A.vec;  // of all three: uniform
    kv_load8<DT>(x, at + 8 * chunk, vec, u);
    kv_load8<DT>(x, at + HD / 2 + 8 * chunk, vec, v);
  };
  const void *x, *x2;
  int64_t at, at2;
  float u[8], v[8], u2[8], v2[8];
  int h = part * HPI + sub;
  if (h < heads) fetch(h, x, at, u, v);
  const int pos = A.start[b] + t;
  const int page = kv_page(A.pg, A.pg.table + b * A.pg.ld, pos), slot = pos & A.pg.mask;
  RotLane<HD, MODE> turn;
  if constexpr (MODE != kRotNone) rot_angles(A.rot, pos, lane, angles[wave]);
  if constexpr (MODE == kRotHalf || MODE == kRotInterleaved) turn.load(A.rot, angles[wave], chunk);
  for (; h < heads; h += A.parts * HPI) {
    const int next = h + A.parts * HPI;
    if (next < heads) fetch(next, x2, at2, u2, v2);
    const int which = h < A.H ? 0 : (h < A.H + A.HK ? 1 : 2);
    const int hh = which == 0 ? h : (which == 1 ? h - A.H : h - A.H - A.HK);
    if (which < 2) rot_apply<DT, HD, MODE>(A.rot, turn, angles[wave], chunk, x, at, u, v);
    if (which == 0) {
      const int64_t to = b * A.qo.sb + t * A.qo.st + hh * A.qo.sh;
      kv_store8<DT>(A.qo.p, to + 8 * chunk, A.qo.vec, u);
      kv_store8<DT>(A.qo.p, to + HD / 2 + 8 * chunk, A.qo.vec, v);
    } else {
      const AppendView& o = which == 1 ? A.ko : A.vo;
      const KvStore& st = which == 1 ? A.ks : A.vs;
      const int fmt = which == 1 ? A.kf : A.vf;
      const int64_t to = b * o.sb + t * o.st + hh * o.sh;
      kv_put8(fmt, st, A.pg, HD, A.HK, page, slot, hh, 8 * chunk, u, o, to, A.seen);
      kv_put8(fmt, st, A.pg, HD, A.HK, page, slot, hh, HD / 2 + 8 * chunk, v, o, to, A.seen);
    }
    x = x2, at = at2;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      u[e] = u2[e];
      v[e] = v2[e];
    }
  }
}

// Positions back in a floating type: HD / 8 lanes a position, 8 values a lane, all heads of keys and of values in turn,
// so that a position's output is written as one contiguous run.  Bound by HBM: 2 x 16001 positions of 8 heads of 128, fp8
// keys and fp4 values to bf16 (182 MB), 40.7 us, 4.5 TB/s.
template <int DT, int HD>
__global__ void __launch_bounds__(256) kv_read(KvStore ks, KvStore vs, int kf, int vf, KvPages pg, int HK,
                                               const int32_t* __restrict__ first, int64_t count,
                                               void* __restrict__ ko, void* __restrict__ vo) {
  constexpr int LPP = HD / 8, PPW = 256 / LPP;
  const int b = blockIdx.y, c = threadIdx.x % LPP;
  const int64_t i = (int64_t)blockIdx.x * PPW + threadIdx.x / LPP;
  if (i >= count) return;
  const int64_t p64 = first[b] + i;
  const int pos = p64 < 0 || p64 >= (1ll << 30) ? -1 : (int)p64;
  const int page = kv_page(pg, pg.table + b * pg.ld, pos), slot = pos & pg.mask;
  const int64_t out = (b * count + i) * HK * HD + 8 * c;
  auto one = [&](const KvStore& st, int fmt, int h, void* o) __attribute__((always_inline)) {
    float y[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (page >= 0) {
      const int64_t ph = (int64_t)page * HK + h, row = (ph << pg.shift) + slot;
      unsigned lo, hi = 0;
      if (fmt == TGM_KV_FP8_E4M3) {
        const u32x2 w = *(const u32x2*)(st.data + row * HD + 8 * c);
        lo = w[0];
        hi = w[1];
      } else {
        lo = *(const unsigned*)(st.data + row * (HD / 2) + 4 * c);
      }
      const float s = kv_scale(st.scales[((ph * (HD / kKvBlock) + c / 4) << pg.shift) + slot]);
      kv_values8(fmt, lo, hi, y);
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] *= s;
    }
    kv_store8<DT>(o, out + (int64_t)h * HD, true, y);
  };
#pragma unroll 4
  for (int h = 0; h < HK; ++h) one(ks, kf, h, ko);
#pragma unroll 4
  for (int h = 0; h < HK; ++h) one(vs, vf, h, vo);
}

template <int DT, int HD>
static void launch_append(int mode, dim3 grid, hipStream_t st, const AppendArgs& a) {
  if (mode == kRotNone) hipLaunchKernelGGL((kv_append<DT, HD, kRotNone>), grid, dim3(256), 0, st, a);
  else if (mode == kRotHalf) hipLaunchKernelGGL((kv_append<DT, HD, kRotHalf>), grid, dim3(256), 0, st, a);
  else if (mode == kRotInterleaved) hipLaunchKernelGGL((kv_append<DT, HD, kRotInterleaved>), grid, dim3(256), 0, st, a);
  else hipLaunchKernelGGL((kv_append<DT, HD, kRotPart>), grid, dim3(256), 0, st, a);
}

static AppendView append_view(const tgm_heads* t, const void* data) {
  if (!t) return AppendView{nullptr, 0, 0, 0, 0};
  return AppendView{(void*)data, t->stride_b, t->stride_t, t->stride_h, heads_vec(t, data)};
}

}  // namespace tgm

using namespace tgm;

extern "C" int tgm_kv_append(const tgm_kv_cache* cache, const tgm_rotary* rotary, const tgm_heads* q, const void* q_data,
                             const tgm_heads* q_out, void* q_out_data, const tgm_heads* k, const void* k_data,
                             const tgm_heads* v, const void* v_data, const tgm_heads* seen, void* k_seen, void* v_seen,
                             const int32_t* table, int64_t ld_table, int64_t table_cols, const int32_t* start,
                             int64_t batch, int64_t tokens, void* stream) {
  clear_error();
  AppendArgs a;
  if (const int e = kv_check(cache, table, ld_table, table_cols, a.ks, a.vs, a.pg)) return e;
  TGM_CHECK_ARG(k && v && (q != nullptr) == (q_out != nullptr), "null argument");
  if (rotary)
    if (const int e = rot_check(rotary, cache->head_dim)) return e;
  TGM_CHECK_ARG(batch >= 0 && tokens >= 0 && batch < (1ll << 30) && tokens < (1ll << 30) && batch * tokens < (1ll << 30),
                "sizes out of range");
  TGM_CHECK_ARG(heads_dtype_ok(k->dtype) && v->dtype == k->dtype && (!q || (q->dtype == k->dtype && q_out->dtype == k->dtype)),
                "q, k and v must be f32, f16 or bf16 and alike");
  TGM_CHECK_ARG(k->heads == cache->kv_heads && v->heads == cache->kv_heads, "k and v must have the cache's heads");
  TGM_CHECK_ARG(!q || (q->heads > 0 && q->heads <= 65535 && q_out->heads == q->heads), "invalid query heads");
  TGM_CHECK_ARG(!seen || (heads_dtype_ok(seen->dtype) && seen->heads == cache->kv_heads),
                "k_seen and v_seen must be f32, f16 or bf16 and have the cache's heads");
  if (batch == 0 || tokens == 0) return TGM_OK;
  TGM_CHECK_ARG(k_data && v_data && start && (!q || (q_data && q_out_data)) && (!seen || (k_seen && v_seen)), "null operand");
  a.q = append_view(q, q_data), a.qo = append_view(q_out, q_out_data);
  a.k = append_view(k, k_data), a.v = append_view(v, v_data);
  a.ko = append_view(seen, k_seen), a.vo = append_view(seen, v_seen);
  a.H = q ? (int)q->heads : 0, a.HK = (int)cache->kv_heads, a.seen = seen ? (int)seen->dtype : -1;
  a.kf = (int)cache->k_format, a.vf = (int)cache->v_format;
  a.rot = rotary ? RotArgs{rotary->freq, rotary->gain, (int)(rotary->rotary_dim / 2)} : RotArgs{nullptr, 1.0, 0};
  a.vec = (!q || a.q.vec) && a.k.vec && a.v.vec;
  a.start = start, a.T = (int)tokens;
  const int64_t ntok = batch * tokens;
  const int groups = ((a.H + 2 * a.HK) * (int)(cache->head_dim / 16) + 63) / 64;
  const int64_t fill = 2048 / ntok;  // as in tgm_rotate
  a.parts = (int)(fill < 1 ? 1 : (fill < groups ? fill : groups));
  a.waves = ntok * a.parts;
  const dim3 grid((unsigned)((a.waves + 3) / 4));
  const int mode = rot_mode(rotary, cache->head_dim);
  const hipStream_t st = (hipStream_t)stream;
#define TGM_GO(DT) (cache->head_dim == 64 ? launch_append<DT, 64>(mode, grid, st, a) : launch_append<DT, 128>(mode, grid, st, a))
  if (k->dtype == TGM_F32) TGM_GO(TGM_F32);
  else if (k->dtype == TGM_F16) TGM_GO(TGM_F16);
  else TGM_GO(TGM_BF16);
#undef TGM_GO
  return launch_status("tgm_kv_append");
}

extern "C" int tgm_kv_read(const tgm_kv_cache* cache, const int32_t* table, int64_t ld_table, int64_t table_cols,
                           const int32_t* first, int64_t batch, int64_t count, void* k_out, void* v_out, int dtype,
                           void* stream) {
  clear_error();
  KvStore ks, vs;
  KvPages pg;
  if (const int e = kv_check(cache, table, ld_table, table_cols, ks, vs, pg)) return e;
  TGM_CHECK_ARG(heads_dtype_ok(dtype), "outputs must be f32, f16 or bf16");
  TGM_CHECK_ARG(batch >= 0 && batch <= 65535 && count >= 0 && count < (1ll << 30), "sizes out of range");
  if (batch == 0 || count == 0) return TGM_OK;
  TGM_CHECK_ARG(first && k_out && v_out && (((uintptr_t)k_out | (uintptr_t)v_out) & 15) == 0, "outputs must be 16-byte aligned");
  const int ppw = cache->head_dim == 64 ? 32 : 16;
  const dim3 grid((unsigned)((count + ppw - 1) / ppw), (unsigned)batch);
  const hipStream_t st = (hipStream_t)stream;
#define TGM_ONE(DT, HD)                                                                                             \
  hipLaunchKernelGGL((kv_read<DT, HD>), grid, dim3(256), 0, st, ks, vs, (int)cache->k_format, (int)cache->v_format, \
                     pg, (int)cache->kv_heads, first, count, k_out, v_out)
#define TGM_GO(DT)                                  \
  do {                                              \
    if (cache->head_dim == 64) TGM_ONE(DT, 64);     \
    else TGM_ONE(DT, 128);                          \
  } while (0)
  if (dtype == TGM_F32) TGM_GO(TGM_F32);
  else if (dtype == TGM_F16) TGM_GO(TGM_F16);
  else TGM_GO(TGM_BF16);
#undef TGM_GO
#undef TGM_ONE
  return launch_status("tgm_kv_read");
}
