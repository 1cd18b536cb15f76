// Rotary positions of heads [batch, tokens, heads, head_dim] (tgm_rotate).
#include "tgm_rotary.h"

namespace tgm {

struct RotView {
  void* p;
  int64_t sb, st, sh;
  int vec;
};

// Heads of 64 or 128 values.  A wave takes one token (and every `parts`-th group of its heads): its lanes compute
// the token's sines and cosines once, a lane keeps those of its 8 pairs in registers, and the heads pass by, HD / 16
// lanes a head, 16 values a lane in two 16-byte loads.  Bound by HBM: 2 x 4096 tokens of 40 heads of 128 in bf16 (168 MB)
// take 35.3 us, 4.75 TB/s where a copy reaches 5.1.  The 64-bit products cost nothing there; they make the result the
// exact one rounded, so that a rotated key that is quantised afterwards falls on the side of a border that it should.
// Loading the next head beside the rotation of this one is slower here (36.1 us, more registers), unlike in kv_append.
template <int DT, int HD, int MODE>
__global__ void __launch_bounds__(256) rotate_heads(RotArgs rot, RotView x, RotView y, int H, const int32_t* start,
                                                    int64_t waves, int T, int parts) {
  constexpr int LPH = HD / 16, HPI = 64 / LPH;
  __shared__ double2 angles[4][HD / 2];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t w = (int64_t)blockIdx.x * 4 + wave;
  if (w >= waves) return;
  const int64_t token = w / parts;
  const int part = (int)(w - token * parts);
  const int b = (int)(token / T), t = (int)(token - (int64_t)b * T);
  const int chunk = lane % LPH, sub = lane / LPH;
  rot_angles(rot, start[b] + t, lane, angles[wave]);
  RotLane<HD, MODE> turn;
  if constexpr (MODE == kRotHalf || MODE == kRotInterleaved) turn.load(rot, angles[wave], chunk);
  const int64_t xi = b * x.sb + t * x.st, yi = b * y.sb + t * y.st;
  for (int h = part * HPI + sub; h < H; h += parts * HPI) {
    const int64_t at = xi + h * x.sh, to = yi + h * y.sh;
    float u[8], v[8];
    kv_load8<DT>(x.p, at + 8 * chunk, x.vec, u);
    kv_load8<DT>(x.p, at + HD / 2 + 8 * chunk, x.vec, v);
    rot_apply<DT, HD, MODE>(rot, turn, angles[wave], chunk, x.p, at, u, v);
    kv_store8<DT>(y.p, to + 8 * chunk, y.vec, u);
    kv_store8<DT>(y.p, to + HD / 2 + 8 * chunk, y.vec, v);
  }
}

// Any other head_dim: a workgroup takes a token, its angles in LDS (as many pairs at a time as fit), a thread a pair.
constexpr int kRotAnyPairs = 512;
template <int DT>
__global__ void __launch_bounds__(256) rotate_any(RotArgs rot, RotView x, RotView y, int H, int D, int interleaved,
                                                  const int32_t* start, int T) {
#pragma clang fp contract(off)  // else the rounding to 32 bits may be merged with the one to 16
  __shared__ double2 angles[kRotAnyPairs];
  const int64_t token = blockIdx.x;
  const int b = (int)(token / T), t = (int)(token - (int64_t)b * T);
  const int pos = start[b] + t;
  const int64_t xi = b * x.sb + t * x.st, yi = b * y.sb + t * y.st;
  for (int p0 = 0; p0 < rot.pairs; p0 += kRotAnyPairs) {
    const int np = min(kRotAnyPairs, rot.pairs - p0);
    __syncthreads();
    for (int i = threadIdx.x; i < np; i += 256) {
      double s, c;
      rot_sincos((double)pos * rot.freq[p0 + i], s, c);
      angles[i] = double2{c * rot.gain, s * rot.gain};
    }
    __syncthreads();
    for (int64_t k = threadIdx.x; k < (int64_t)H * np; k += 256) {
      const int h = (int)(k / np), i = (int)(k - (int64_t)h * np), j = p0 + i;
      const int d0 = interleaved ? 2 * j : j, d1 = interleaved ? 2 * j + 1 : j + rot.pairs;
      const double u = load_f32(x.p, DT, xi + h * x.sh + d0), v = load_f32(x.p, DT, xi + h * x.sh + d1);
      const double2 a = angles[i];
      store_from_f32(y.p, DT, yi + h * y.sh + d0, (float)__builtin_fma(u, a.x, -(v * a.y)));
      store_from_f32(y.p, DT, yi + h * y.sh + d1, (float)__builtin_fma(v, a.x, u * a.y));
    }
  }
  const int rest = D - 2 * rot.pairs;
  for (int64_t k = threadIdx.x; k < (int64_t)H * rest; k += 256) {
    const int h = (int)(k / rest), d = 2 * rot.pairs + (int)(k - (int64_t)h * rest);
    store_from_f32(y.p, DT, yi + h * y.sh + d, load_f32(x.p, DT, xi + h * x.sh + d));
  }
}

template <int DT, int HD>
static void launch_rotate(int mode, dim3 grid, hipStream_t st, const RotArgs& rot, const RotView& x, const RotView& y,
                          int H, const int32_t* start, int64_t waves, int T, int parts) {
  if (mode == kRotHalf)
    hipLaunchKernelGGL((rotate_heads<DT, HD, kRotHalf>), grid, dim3(256), 0, st, rot, x, y, H, start, waves, T, parts);
  else if (mode == kRotInterleaved)
    hipLaunchKernelGGL((rotate_heads<DT, HD, kRotInterleaved>), grid, dim3(256), 0, st, rot, x, y, H, start, waves, T, parts);
  else
    hipLaunchKernelGGL((rotate_heads<DT, HD, kRotPart>), grid, dim3(256), 0, st, rot, x, y, H, start, waves, T, parts);
}

}  // namespace tgm

using namespace tgm;

extern "C" int tgm_rotate(const tgm_rotary* rotary, const tgm_heads* x, const void* x_data, const tgm_heads* out,
                          void* out_data, const int32_t* start, int64_t batch, int64_t tokens, int64_t head_dim,
                          void* stream) {
  clear_error();
  TGM_CHECK_ARG(rotary && x && out, "null argument");
  TGM_CHECK_ARG(batch >= 0 && tokens >= 0 && x->heads >= 0 && head_dim > 0, "negative size");
  if (const int e = rot_check(rotary, head_dim)) return e;
  TGM_CHECK_ARG(heads_dtype_ok(x->dtype) && out->dtype == x->dtype && out->heads == x->heads,
                "x and out must be f32, f16 or bf16 and alike");
  if (batch == 0 || tokens == 0 || x->heads == 0) return TGM_OK;
  TGM_CHECK_ARG(x_data && out_data && start, "null operand");
  TGM_CHECK_ARG(batch < (1 << 30) && tokens < (1 << 30) && x->heads < (1 << 24) && head_dim < (1 << 20) &&
                    batch * tokens < (1ll << 30), "sizes out of range");
  const RotArgs rot{rotary->freq, rotary->gain, (int)(rotary->rotary_dim / 2)};
  const RotView vx{(void*)x_data, x->stride_b, x->stride_t, x->stride_h, heads_vec(x, x_data)};
  const RotView vy{out_data, out->stride_b, out->stride_t, out->stride_h, heads_vec(out, out_data)};
  const hipStream_t st = (hipStream_t)stream;
  const int64_t ntok = batch * tokens;
  const int H = (int)x->heads, T = (int)tokens;
  if (head_dim == 64 || head_dim == 128) {
    const int groups = (H * (int)(head_dim / 16) + 63) / 64;
    // a wave per token walks all its heads; with few tokens the heads spread over waves, 8 a CU
    const int64_t fill = 2048 / ntok;
    const int parts = (int)(fill < 1 ? 1 : (fill < groups ? fill : groups));
    const int64_t waves = ntok * parts;
    const dim3 grid((unsigned)((waves + 3) / 4));
    int mode = rot_mode(rotary, head_dim);
    if (mode == kRotNone) mode = kRotPart;
#define TGM_GO(DT)                                                                                              \
  (head_dim == 64 ? launch_rotate<DT, 64>(mode, grid, st, rot, vx, vy, H, start, waves, T, parts)               \
                  : launch_rotate<DT, 128>(mode, grid, st, rot, vx, vy, H, start, waves, T, parts))
    if (x->dtype == TGM_F32) TGM_GO(TGM_F32);
    else if (x->dtype == TGM_F16) TGM_GO(TGM_F16);
    else TGM_GO(TGM_BF16);
#undef TGM_GO
  } else {
    const dim3 grid((unsigned)ntok);
    const int il = rotary->layout == TGM_ROTARY_INTERLEAVED, D = (int)head_dim;
    if (x->dtype == TGM_F32) hipLaunchKernelGGL(rotate_any<TGM_F32>, grid, dim3(256), 0, st, rot, vx, vy, H, D, il, start, T);
    else if (x->dtype == TGM_F16) hipLaunchKernelGGL(rotate_any<TGM_F16>, grid, dim3(256), 0, st, rot, vx, vy, H, D, il, start, T);
    else hipLaunchKernelGGL(rotate_any<TGM_BF16>, grid, dim3(256), 0, st, rot, vx, vy, H, D, il, start, T);
  }
  return launch_status("tgm_rotate");
}
