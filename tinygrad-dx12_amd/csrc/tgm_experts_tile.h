// The grouped products of tgm_experts_apply: the rows of many experts, each with a packed weight of its own.
//
// The tile is that of tgm_gemm_w_tile.h: 32 FA rows of A x 32 WN weight rows, a wave to 32 weight rows, K in steps of 128, NBUF
// stages in LDS or on their way there, one barrier a stage, a stage's loads one after each MFMA; its operand layouts, K order
// and decoders.  Of its own here:
//
//  * The tiles come from a list on the device, and the rows of A may be gathered.
//  * A workgroup goes through tiles, as many workgroups as the chip holds at once.  A tile of a few hundred columns takes 11 to
//    32 stages of 1.5 to 1.9 us, and its start (the list, the row indexes, the first loads' latency) and its stores some 8 us
//    more.  The last stages of a tile load the first of the next, and the sums are stored from the registers, beside them
//    (64 experts of 2048 x 1408, 192 rows each: down 122 -> 90 us).
//  * Of a tile's blocks of 32 rows those without rows are not multiplied.
//  * silu's exponent and quotient are the hardware's, which expf and a division took 3 us of a tile's time for.
#pragma once

#include "tgm_experts.h"

namespace tgm {

// Four neighbouring words that the whole wave reads.
typedef int wg_words4 __attribute__((ext_vector_type(4), aligned(4)));
__device__ __forceinline__ wg_words4 scalar_words4(const int* from) {
  return *(const wg_words4 __attribute__((address_space(4)))*)(uintptr_t)from;
}

struct WGroupAt {  // a tile: an entry's positions m0 .. m_end - 1, weight rows from n0 on
  int m0, m_end, n0, expert;
};

// g / (1 + exp(-g)) to 2^-22 of it: exp(-g) = 2^t (1 + r ln 2), where t + r is -g log2(e) beyond fp32.  Past +-126, where the
// quotient is g or 0, t stays within what r can correct.
__device__ __forceinline__ float group_silu(float g) {
  const float x = -__builtin_amdgcn_fmed3f(g, -126.0f, 126.0f);
  const float log2e = 1.44269504f, rest = 1.92596303e-8f, ln2 = 0.693147182f;
  const float t = x * log2e;
  const float r = __builtin_fmaf(x, rest, __builtin_fmaf(x, log2e, -t));
  return g * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(t) * __builtin_fmaf(r, ln2, 1.0f));
}

// A wave's sums, 32 weight rows from n0 on: fp32, or silu(gate) * up in 16 bits.  Rows past the entry's are past the buffer,
// which drops them.
template <int FA>
__device__ __forceinline__ void store_group(const f32x16 (&acc)[FA], int used, int lane, const WGroupAt& at, int n0,
                                            const WGroupArgs& p) {
  if (n0 >= p.N) return;
  const unsigned ld = (unsigned)p.ldc * (p.swiglu ? 2u : 4u);
  const auto c = __builtin_amdgcn_make_buffer_rsrc((uint8_t*)p.c + (int64_t)at.m0 * ld, 0, (int)((unsigned)(at.m_end - at.m0) * ld),
                                                   0x00020000);
  const unsigned first = 4u * (unsigned)(lane >> 5) * ld;  // the lane's rows: 8 (v / 4) + 4 (lane / 32) + v % 4
  const int l32 = lane & 31;
#pragma unroll
  for (int t = 0; t < FA; ++t) {
    if (t >= used) break;
    if (p.swiglu) {  // an even lane holds a gate column and the next one its up column: each takes one of two rows
      const bool odd = lane & 1;
      const unsigned col = first + (odd ? ld : 0u) + (unsigned)(n0 + l32 - (int)odd);
#pragma unroll
      for (int v = 0; v < 16; v += 2) {
        const float send = odd ? acc[t][v] : acc[t][v + 1];
        const float got = __builtin_bit_cast(
            float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, send), 0xB1, 0xF, 0xF, true));  // quad_perm [1, 0, 3, 2]
        const float y = group_silu(odd ? got : acc[t][v]) * (odd ? acc[t][v + 1] : got);
        const uint16_t bits = p.cdt == TGM_BF16 ? f32_to_bf16(y) : __builtin_bit_cast(uint16_t, (_Float16)y);
        __builtin_amdgcn_raw_buffer_store_b16(bits, c, (int)(col + (unsigned)(32 * t + 8 * (v / 4) + v % 4) * ld), 0, 0);
      }
    } else {
      const unsigned col = first + (unsigned)(n0 + l32) * 4u;
#pragma unroll
      for (int v = 0; v < 16; ++v) {
        const float sum = acc[t][v];  // a bit cast of the vector's element itself takes the first
        __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(unsigned, sum), c,
                                              (int)(col + (unsigned)(32 * t + 8 * (v / 4) + v % 4) * ld), 0, 0);
      }
    }
  }
}

template <int KIND, int FA, int WN, int NBUF>
__global__ void __launch_bounds__(64 * WN)
__attribute__((amdgpu_waves_per_eu(WTile<KIND, FA, WN, 1, NBUF>::kOccupancy, WTile<KIND, FA, WN, 1, NBUF>::kOccupancy)))
gemm_w_group(WGroupArgs p) {
  using T = WTile<KIND, FA, WN, 1, NBUF>;
  constexpr bool I4 = T::kI4;
  constexpr int G = T::kG, NS = T::kNS ? T::kNS : 1;
  __shared__ __attribute__((aligned(16))) unsigned char lds[NBUF * T::kStage];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wn = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int tiles_m = p.tiles[0], tiles_n = (p.N + T::kBN - 1) / T::kBN;
  const int total = tiles_m * tiles_n;
  if ((int)blockIdx.x >= total) return;
  const int nstages = p.K / kWtK;
  const unsigned kbw = (unsigned)p.K / 8u * (T::kRow == 64 ? 4u : 6u);  // packed bytes per W row
  constexpr unsigned ssize = (unsigned)kind_scale_bytes(KIND);           // INT4 scale bytes
  const unsigned srow = I4 ? (G ? (unsigned)(p.K / (G ? G : 1)) * ssize : 0u) : (unsigned)p.K / 32u;  // scale bytes per W row
  const unsigned lds_base = (unsigned)(uintptr_t)(__attribute__((address_space(3))) unsigned char*)lds;

  auto find = [&](int tile) __attribute__((always_inline)) {
    int tm, tn;
    tile_of_ranges((unsigned)tile, p.K, tiles_m, tiles_n, 8, tm, tn);
    const wg_words4 entry = scalar_words4(p.tiles + 4 + 4 * tm);
    return WGroupAt{entry[1], entry[1] + entry[2], tn * T::kBN, entry[0]};
  };
  // Offsets of A: load instruction i = wn + WN q covers rows 4 i .. 4 i + 3 (lane l: row 4 i + l / 16, logical 16-byte column
  // (l % 16) ^ (row % 16)).  Rows past the entry's: past A, which the host keeps below 2 GiB.
  auto rows_of = [&](const WGroupAt& to, unsigned (&off)[T::kLoadsA]) __attribute__((always_inline)) {
#pragma unroll
    for (int q = 0; q < T::kLoadsA; ++q) {
      const int row = 4 * (wn + WN * q) + (lane >> 4);
      int r = row;
      if (p.rows) {  // by scalar loads: waiting for a vector load would wait for every load in flight
        const wg_words4 four = scalar_words4(p.rows + to.m0 + 4 * (wn + WN * q));
        const int lo = lane & 16 ? four[1] : four[0], hi = lane & 16 ? four[3] : four[2];
        r = lane & 32 ? hi : lo;
      }
      off[q] = (row < to.m_end - to.m0 ? (unsigned)r * p.lda_bytes : 0xC0000000u) + (unsigned)(((lane & 15) ^ (row & 15)) * 16);
    }
  };
  // The tile that loads are for: in the last stages of a tile already the next.  W instruction i = wn + WN q fills bytes
  // [1024 i, + 1024) of the W panel.
  WGroupAt at;
  i32x4v ra, rw, rs;
  unsigned voa[T::kLoadsA], vow[T::kLoadsW], vos;
  auto aim = [&](const WGroupAt& to, const unsigned (&off)[T::kLoadsA]) __attribute__((always_inline)) {
    at = to;
    ra = p.rows ? buffer_rsrc(p.a, p.a_bytes)
                : buffer_rsrc(p.a + (int64_t)to.m0 * p.lda_bytes, (unsigned)(to.m_end - to.m0 - 1) * p.lda_bytes + (unsigned)p.K * 2u);
    rw = buffer_rsrc(p.w + to.expert * p.w_bytes, (unsigned)p.N * kbw);
    rs = buffer_rsrc(p.scales + (p.scales ? to.expert * p.s_bytes : 0), p.scales ? (unsigned)p.N * srow : 0u);
#pragma unroll
    for (int q = 0; q < T::kLoadsA; ++q) voa[q] = off[q];
#pragma unroll
    for (int q = 0; q < T::kLoadsW; ++q) {
      const int i = wn + WN * q;
      if constexpr (T::kRow == 64) {
        const int row = 16 * i + (lane >> 2);
        vow[q] = (unsigned)(to.n0 + row) * kbw + (unsigned)(((lane & 3) ^ ((row >> 2) & 3)) * 16);
      } else {
        const int f = 1024 * i + 16 * lane;
        vow[q] = (unsigned)(to.n0 + f / 96) * kbw + (unsigned)(f % 96);
      }
    }
    vos = (unsigned)(to.n0 + 32 * wn + (lane & 31)) * srow;
  };
  // Load piece q (< kLoads) of stage st into buffer buf: the A instructions, then W's, then the scales.  Past the tile's end: the
  // next tile's stages, or the last stage again, so that every wave's count stays.
  int turn = -1, turned = 0;
  auto load_piece = [&](int st, int buf, int q) __attribute__((always_inline)) {
    st -= turned;
    const unsigned s0 = (unsigned)(st < nstages ? st : nstages - 1);
    const unsigned base = lds_base + (unsigned)(buf * T::kStage);
    if (q < T::kLoadsA) {
      lds_dma16(ra, base + (unsigned)(wn + WN * q) * 1024u, voa[q < T::kLoadsA ? q : 0] + s0 * (kWtK * 2));
    } else if (q < T::kLoadsA + T::kLoadsW) {
      const int i = q - T::kLoadsA;
      lds_dma16(rw, base + (unsigned)T::kA + (unsigned)(wn + WN * i) * 1024u,
                vow[i >= 0 && i < T::kLoadsW ? i : 0] + s0 * (unsigned)T::kRow);
    } else {
      const unsigned g = (unsigned)(q - T::kLoadsA - T::kLoadsW);
      const unsigned dst = base + (unsigned)(T::kA + T::kW + wn * T::kS) + g * 256u;
      const unsigned off = vos + (I4 ? (s0 * T::kNS + g) * ssize : s0 * 4u);
      if constexpr (!I4 || ssize == 4) lds_dma4(rs, dst, off);
      else lds_dma2(rs, dst, off);
    }
  };

  const int half = lane >> 5, l32 = lane & 31, w_row = 32 * wn + l32;
  NibbleConsts nib;
  nib.pattern = p.is_signed ? 0x64006400u ^ 0x00800008u : 0x64006400u;
  nib.offset = p.is_signed ? wt_half2{(_Float16)-1032.0f, (_Float16)-72.0f} : wt_half2{(_Float16)-1024.0f, (_Float16)-64.0f};
  const unsigned sshift = p.sdt == TGM_BF16 ? 16u : 0u;
  constexpr int JPG = I4 && G ? G / 16 : 8;  // MFMAs per scale group
  constexpr int RAW = T::kRow / 8;           // dwords of a lane's 64 codes
  constexpr int PD = T::kPD, SL = 2 * PD;    // A is read PD substeps ahead
  f32x16 acc[FA];
  u32x4 fa[SL][FA];                  // A fragments of substeps j (slot j % SL)
  unsigned raw[RAW], rawn[RAW];      // packed codes of this step and the next
  unsigned sbits[NS], sbitsn[NS];    // scale words of this step and the next
  wt_bf16x8 wd[I4 ? 1 : 8];          // decoded MX weights
  wt_f16x8 wi[2];                    // decoded nibbles of substeps j (slot j % 2)
  auto read_a = [&](auto blocks, int buf, int j, u32x4 (&dst)[FA]) __attribute__((always_inline)) {
    const int col = (I4 ? 2 * j + half : 8 * half + j) ^ (l32 & 15);
#pragma unroll
    for (int t = 0; t < decltype(blocks)::value; ++t)
      dst[t] = *(const u32x4*)(lds + buf * T::kStage + (32 * t + l32) * 256 + col * 16);
  };
  auto read_w = [&](int buf, unsigned (&r)[RAW], unsigned (&sb)[NS]) __attribute__((always_inline)) {
    const unsigned char* pw = lds + buf * T::kStage + T::kA;
    if constexpr (I4) {  // dword 2 j + h of the row
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const unsigned* c = (const unsigned*)(pw + w_row * 64 + ((q ^ ((w_row >> 2) & 3)) * 16) + 4 * half);
        r[2 * q] = c[0];
        r[2 * q + 1] = c[2];
      }
    } else {
#pragma unroll
      for (int q = 0; q < RAW / 4; ++q) {
        const u32x4 v = T::kRow == 96 ? *(const u32x4*)(pw + w_row * 96 + 48 * half + 16 * q)
                                      : *(const u32x4*)(pw + w_row * 64 + (((2 * half + q) ^ ((w_row >> 2) & 3)) * 16));
#pragma unroll
        for (int e = 0; e < 4; ++e) r[4 * q + e] = v[e];
      }
    }
    const unsigned* ps = (const unsigned*)(pw + T::kW + wn * T::kS) + l32;
#pragma unroll
    for (int g = 0; g < T::kNS; ++g) sb[g] = ps[64 * g];
  };
  auto mx_block = [&](const unsigned (&r)[RAW], unsigned sb, int blk) __attribute__((always_inline)) {
    if constexpr (!I4) decode_mx_block<KIND>(r, blk, p.scales ? (sb >> (16 * half + 8 * blk)) & 0xFFu : 127u, wd + 4 * blk);
  };

  WGroupAt next;
  unsigned voan[T::kLoadsA];
  // One stage from buffer cur.  On entry fa holds A of its first PD substeps, raw and sbits its weights, and substep 0's weights
  // are decoded.  Before substep 8 - PD, when every LDS read of the stage is done, the wave waits for its share of the next
  // stage, the barrier publishes it and frees this buffer; what is left covers the refill's issue, the next stage's first reads
  // and its first decode.
  auto stage = [&](auto blocks, int st, int prv, int cur, int nxt) __attribute__((always_inline)) {
    constexpr int NF = decltype(blocks)::value;
    f32x16 part[FA];  // the sums of the current scale group
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      __builtin_amdgcn_sched_barrier(0);
      if (j == 8 - PD) {
        wait_loads<(NBUF - 2) * T::kLoads>();  // the stores of the tile before count too: then it waits for them as well
        lds_barrier();
        read_w(nxt, rawn, sbitsn);
        read_a(blocks, nxt, 0, fa[0]);
        if (st + NBUF == turn) {
          aim(next, voan);
          turned = nstages;
        }
      } else if (j > 8 - PD) {
        read_a(blocks, nxt, j + PD - 8, fa[j + PD - 8]);
      } else {
        read_a(blocks, cur, j + PD, fa[(j + PD) % SL]);
      }
      // this substep's share of the loads, one after each MFMA: stage st + NBUF into this buffer from substep
      // 8 - PD on, the rest of stage st + NBUF - 1 into the previous stage's buffer before
      auto pieces = [&](int t) __attribute__((always_inline)) {
#pragma unroll
        for (int q = 0; q < T::kLoads; ++q)
          if (q >= T::first_piece(j) && q < T::end_piece(j) && (q - T::first_piece(j)) % FA == t) {
            __builtin_amdgcn_sched_barrier(0);
            if (j >= 8 - PD) load_piece(st + NBUF, cur, q);
            else load_piece(st + NBUF - 1, prv, q);
            __builtin_amdgcn_sched_barrier(0);
          }
      };
      if constexpr (I4) {
        if (j < 7) wi[(j + 1) & 1] = decode_nibbles(raw[j + 1], nib);
#pragma unroll
        for (int t = 0; t < FA; ++t) {
          if (t < NF) {
            const wt_f16x8 a = __builtin_bit_cast(wt_f16x8, fa[j % SL][t]);
            if constexpr (G == 0) acc[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, wi[j & 1], acc[t], 0, 0, 0);
            else part[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, wi[j & 1], j % JPG ? part[t] : f32x16{}, 0, 0, 0);
          }
          pieces(t);
        }
        if (j == 7) wi[0] = decode_nibbles(rawn[0], nib);
        if (G != 0 && j % JPG == JPG - 1) {
          const unsigned bits = sbits[j / JPG];
          const float sv = ssize == 2 && p.sdt == TGM_F16 ? (float)__builtin_bit_cast(_Float16, (unsigned short)bits)
                                                          : __builtin_bit_cast(float, bits << sshift);
#pragma unroll
          for (int t = 0; t < NF; ++t)
#pragma unroll
            for (int v = 0; v < 16; ++v) acc[t][v] += part[t][v] * sv;
          // pins these sums here, as in tgm_gemm_w_tile.h
#pragma unroll
          for (int t = 0; t < NF; ++t) asm volatile("" : "+v"(acc[t]));
        }
      } else {
        if (j == 2) mx_block(raw, sbits[0], 1);
#pragma unroll
        for (int t = 0; t < FA; ++t) {
          if (t < NF)
            acc[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(wt_bf16x8, fa[j % SL][t]), wd[j], acc[t], 0, 0, 0);
          pieces(t);
        }
        if (j == 7) mx_block(rawn, sbitsn[0], 0);
      }
    }
#pragma unroll
    for (int i = 0; i < RAW; ++i) raw[i] = rawn[i];
#pragma unroll
    for (int g = 0; g < T::kNS; ++g) sbits[g] = sbitsn[g];
  };
  auto first_loads = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int s = 0; s < NBUF; ++s)
#pragma unroll
      for (int q = 0; q < T::kLoads; ++q)
        if (s < NBUF - 1 || q < T::first_piece(0)) load_piece(s, s, q);
    wait_loads<(NBUF - 2) * T::kLoads + T::first_piece(0)>();
    lds_barrier();
  };

  next = find(blockIdx.x);
  rows_of(next, voan);
  aim(next, voan);
  first_loads();
  int prv = NBUF - 1, cur = 0;
  for (int tile = blockIdx.x + gridDim.x;; tile += gridDim.x) {
    const WGroupAt own = at;
    const bool more = tile < total, ahead = more && nstages >= NBUF;
    if (more) {
      next = find(tile);
      rows_of(next, voan);
    }
    turn = ahead ? nstages : -1;
#pragma unroll
    for (int t = 0; t < FA; ++t) acc[t] = f32x16{};
    auto stages = [&](auto blocks) __attribute__((always_inline)) {
      read_w(cur, raw, sbits);
#pragma unroll
      for (int j = 0; j < PD; ++j) read_a(blocks, cur, j, fa[j]);
      if constexpr (I4) wi[0] = decode_nibbles(raw[0], nib);
      else mx_block(raw, sbits[0], 0);
#pragma unroll 1
      for (int st = 0; st < nstages; ++st) {
        const int nxt = cur + 1 < NBUF ? cur + 1 : 0;
        stage(blocks, st, prv, cur, nxt);
        prv = cur;
        cur = nxt;
      }
    };
    const int used = (own.m_end - own.m0 + 31) / 32;
    if (FA > 1 && used == 1) stages(std::integral_constant<int, 1>{});
    else if (FA > 2 && used == 2) stages(std::integral_constant<int, FA < 2 ? FA : 2>{});
    else stages(std::integral_constant<int, FA>{});
    turned = 0;
    store_group<FA>(acc, used, lane, own, own.n0 + 32 * wn, p);
    if (!more) break;
    if (!ahead) {  // too few stages to load ahead in
      wait_loads<0>();
      __syncthreads();  // every wave is done with the buffers
      aim(next, voan);
      prv = NBUF - 1, cur = 0;
      first_loads();
    }
  }
  wait_loads<0>();  // of the last stage's repeats, before another workgroup has this LDS
}

template <int KIND, int FA, int WN, int NBUF>
int launch_experts_tile(const WGroupArgs& p, int64_t most, hipStream_t stream) {
  using T = WTile<KIND, FA, WN, 1, NBUF>;
  static_assert(T::kFits && T::kLds == NBUF * T::kStage, "tile shape");
  const int64_t tiles = most * ((p.N + T::kBN - 1) / T::kBN);
  const int cus = stream_cu_count(stream);
  const int64_t held = (int64_t)(cus > 0 ? cus : 256) * (T::kOccupancy * 4 / WN);
  hipLaunchKernelGGL((gemm_w_group<KIND, FA, WN, NBUF>), dim3((unsigned)(tiles < held ? tiles : held)), dim3(64 * WN), 0, stream, p);
  return launch_status("tgm_experts_apply");
}

}  // namespace tgm
