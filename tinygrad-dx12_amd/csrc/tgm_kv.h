// Device-side view of the paged key/value cache and its codes (include/tgm_serving.h).
#pragma once

#include <math.h>

#include "../../include/tgm_serving.h"
#include "tgm_mfma_common.h"
#include "tgm_lanes.h"

namespace tgm {

typedef __bf16 kv_bf16x2 __attribute__((ext_vector_type(2)));
typedef float kv_f32x2 __attribute__((ext_vector_type(2)));
typedef short kv_s16x2 __attribute__((ext_vector_type(2)));

constexpr int kKvBlock = 32;  // values that share a scale

// A key or value store: pages of [heads][slots][row bytes], scales [heads][blocks][slots].
struct KvStore {
  uint8_t* data;
  uint8_t* scales;
};

// How positions map to pages; sizes are checked on the host (page_size a power of two).
struct KvPages {
  const int32_t* table;
  int64_t ld;
  int cols, pages, shift, mask;
};

// Page of a position of the sequence whose table row is given, or -1.
__device__ __forceinline__ int kv_page(const KvPages& pg, const int32_t* row, int pos) {
  const int i = pos >> pg.shift;
  if (pos < 0 || i >= pg.cols) return -1;
  const int p = row[i];
  return (unsigned)p < (unsigned)pg.pages ? p : -1;
}

__device__ __forceinline__ float kv_scale(unsigned e) { return bits_f32(e == 0 ? 0x00400000u : e << 23); }

// 8 codes as exact fp32 values without their scale: fp8 from two words, fp4 from one.
__device__ __forceinline__ void kv_values8(int fmt, unsigned lo, unsigned hi, float (&v)[8]) {
  kv_f32x2 p[4];
  if (fmt == TGM_KV_FP8_E4M3) {
    p[0] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(lo, 1.0f, false);
    p[1] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(lo, 1.0f, true);
    p[2] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(hi, 1.0f, false);
    p[3] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(hi, 1.0f, true);
  } else {
    p[0] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(lo, 1.0f, 0);
    p[1] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(lo, 1.0f, 1);
    p[2] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(lo, 1.0f, 2);
    p[3] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(lo, 1.0f, 3);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = p[i][0];
    v[2 * i + 1] = p[i][1];
  }
}

// 4 codes of the fp8 word w, or the 4 of half `h` of the fp4 word, times a power of two, as bf16 (exact:
// at most four significant bits): the scaled conversion does the product.
template <int BITS>
__device__ __forceinline__ u32x2 kv_bf16x4(unsigned w, int h, float s) {
  if constexpr (BITS == 8)
    return u32x2{__builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, s, false)),
                 __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, s, true))};
  else if (h == 0)
    return u32x2{__builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 0)),
                 __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 1))};
  else
    return u32x2{__builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 2)),
                 __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 3))};
}

// 8 values of a tensor at p as fp32 / stored from fp32; `vec`: p is 16-byte aligned.
template <int DT>
__device__ __forceinline__ void kv_load8(const void* base, int64_t i, bool vec, float (&v)[8]) {
  if constexpr (DT == TGM_F32) {
    const float* p = (const float*)base + i;
    if (vec) {
      const f32x4 a = *(const f32x4*)p, b = *(const f32x4*)(p + 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        v[e] = a[e];
        v[4 + e] = b[e];
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = p[e];
    }
  } else {
    const uint16_t* p = (const uint16_t*)base + i;
    uint16_t h[8];
    if (vec) {
      const u32x4 a = *(const u32x4*)p;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        h[2 * e] = (uint16_t)(a[e] & 0xFFFFu);
        h[2 * e + 1] = (uint16_t)(a[e] >> 16);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) h[e] = p[e];
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = DT == TGM_BF16 ? bf16_to_f32(h[e]) : (float)__builtin_bit_cast(_Float16, h[e]);
  }
}

template <int DT>
__device__ __forceinline__ unsigned kv_pack2(float lo, float hi) {
  if constexpr (DT == TGM_BF16) return bf16x2_bits(lo, hi);
  else return __builtin_bit_cast(unsigned short, (_Float16)lo) | ((unsigned)__builtin_bit_cast(unsigned short, (_Float16)hi) << 16);
}

template <int DT>
__device__ __forceinline__ void kv_store8(void* base, int64_t i, bool vec, const float (&v)[8]) {
  if constexpr (DT == TGM_F32) {
    float* p = (float*)base + i;
    if (vec) {
      *(f32x4*)p = f32x4{v[0], v[1], v[2], v[3]};
      *(f32x4*)(p + 4) = f32x4{v[4], v[5], v[6], v[7]};
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) p[e] = v[e];
    }
  } else {
    const u32x4 w{kv_pack2<DT>(v[0], v[1]), kv_pack2<DT>(v[2], v[3]), kv_pack2<DT>(v[4], v[5]), kv_pack2<DT>(v[6], v[7])};
    uint16_t* p = (uint16_t*)base + i;
    if (vec) {
      *(u32x4*)p = w;
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) p[e] = (uint16_t)(w[e / 2] >> (16 * (e & 1)));
    }
  }
}

// Host-side check of a cache description; fills the device views.
inline int kv_check(const tgm_kv_cache* c, const int32_t* table, int64_t ld_table, int64_t table_cols, KvStore& k,
                    KvStore& v, KvPages& pg) {
  TGM_CHECK_ARG(c && c->k_data && c->k_scales && c->v_data && c->v_scales && table, "null cache or table");
  TGM_CHECK_ARG(c->pages > 0 && c->pages < (1ll << 31) && c->kv_heads > 0 && c->kv_heads <= 65535, "invalid page or head count");
  TGM_CHECK_ARG(c->head_dim == 64 || c->head_dim == 128, "head_dim must be 64 or 128");
  TGM_CHECK_ARG(c->page_size >= 16 && c->page_size <= 1024 && (c->page_size & (c->page_size - 1)) == 0,
                "page_size must be a power of two from 16 to 1024");
  TGM_CHECK_ARG((c->k_format == TGM_KV_FP8_E4M3 || c->k_format == TGM_KV_FP4_E2M1) &&
                    (c->v_format == TGM_KV_FP8_E4M3 || c->v_format == TGM_KV_FP4_E2M1),
                "cache formats are fp8_e4m3 and fp4_e2m1");
  TGM_CHECK_ARG((((uintptr_t)c->k_data | (uintptr_t)c->k_scales | (uintptr_t)c->v_data | (uintptr_t)c->v_scales) & 15) == 0,
                "the stores must be 16-byte aligned");
  TGM_CHECK_ARG(table_cols >= 0 && ld_table >= table_cols && table_cols < (1ll << 30) && table_cols * c->page_size < (1ll << 30),
                "invalid page table");
  int shift = 0;
  while ((1ll << shift) < c->page_size) ++shift;
  k = {(uint8_t*)c->k_data, (uint8_t*)c->k_scales};
  v = {(uint8_t*)c->v_data, (uint8_t*)c->v_scales};
  pg = {table, ld_table, (int)table_cols, (int)c->pages, shift, (int)c->page_size - 1};
  return TGM_OK;
}

}  // namespace tgm
