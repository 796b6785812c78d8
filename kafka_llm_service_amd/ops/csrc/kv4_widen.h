// The 4-bit cache's keys and values widened to bf16, in the order in which the matrix cores take them (pages: kv4.h; kv4_tile.hip).
#pragma once
#include "kv4.h"

namespace kafka {
namespace kv4 {

constexpr int TK = 64;                    // keys of a tile
template <int D>
struct Image {                            // of 64 keys and one head
  static constexpr int PAGE_BYTES = PAGE * D * 2, KBYTES = TK * D * 2, BYTES = 2 * KBYTES;
};

// ---- widening -----------------------------------------------------------------------------------------------------------
// A workgroup per tile and head, a wave per page: 16048 keys of 8 heads of 128, 83 MB, 15.5 us (5.4 TB/s, most of it into the last-level
// cache). K: [page][d / 8][key][8], V: [page][d][16 keys: 0-3, 8-11, 4-7, 12-15], the two halves of
// rows with d & 8 exchanged (attn_tile.h: reads of both without bank conflicts). Keys behind ``last`` become zeros, and whole pages of which
// no row from ``pmin`` on sees a key (the table may name anything there); those of a page that is none no numbers. Tiles: table row,
// block, last key, pmin.
template <int D>
__device__ __forceinline__ void widen_tile(int wg, const uint8_t* __restrict__ kc, const uint8_t* __restrict__ vc, int64_t n_pages,
                                           const int* __restrict__ tables, int64_t ts, const int* __restrict__ tiles, int Hkv, int window,
                                           int first, char* __restrict__ ws) {
  constexpr int KW = D / 32;               // words of K a lane: its quarter of a key
  const int t = wg / Hkv, h = wg % Hkv;
  const int* tl = tiles + 4 * (int64_t)t;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, last = tl[2];
  const int key0 = tl[1] * TK + w * PAGE;
  char* kd = ws + ((int64_t)t * Hkv + h) * Image<D>::BYTES + w * Image<D>::PAGE_BYTES;
  char* vd = kd + Image<D>::KBYTES;
  const int o = lane & 15, c = lane >> 4;
  const bool some = key0 <= last && (key0 + PAGE - 1 > tl[3] - window || key0 < first);
  const int pid = some ? tables[tl[0] * ts + (key0 >> 4)] : 0;
  const bool bad = pid < 0 || pid >= n_pages;
  const int64_t at = ((int64_t)(bad ? 0 : pid) * Hkv + h) * Page<D>::BYTES;
  {  // K: lane = (key, quarter of its elements)
    uint32_t x[KW];
    uint32_t e = kc[at + Page<D>::DATA + o * (D / 32) + c * (D / 32) / 4];
#pragma unroll
    for (int i = 0; i < KW; ++i) x[i] = *reinterpret_cast<const uint32_t*>(kc + at + o * (D / 2) + c * (D / 8) + 4 * i);
    if (!some || key0 + o > last) {
      e = 0;
#pragma unroll
      for (int i = 0; i < KW; ++i) x[i] = 0;
    }
    const float sc = bad ? __builtin_nanf("") : scale_of(e);
#pragma unroll
    for (int i = 0; i < KW; ++i) {
      bf16x8 y = widen8(x[i], sc);
      if (bad) {
#pragma unroll
        for (int j = 0; j < 8; ++j) y[j] = (bf16)__builtin_nanf("");
      }
      *reinterpret_cast<bf16x8*>(kd + ((c * KW + i) * 16 + o) * 16) = y;
    }
  }
  {  // V: lane = (four keys, D / 16 elements)
    constexpr int W = D / 32;
    const u32x4 d = *reinterpret_cast<const u32x4*>(vc + at + (c * (D / 8) + o * (D / 8) / 16) * 16);
    const uint32_t s = *reinterpret_cast<const uint32_t*>(vc + at + Page<D>::DATA + (o * (D / 16) / 32) * 16 + c * 4);
    uint32_t x[W][4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t v = d[i], e = (s >> (8 * i)) & 255u;
      if (D == 64) v >>= 16 * (o & 1);
      if (!some || bad || key0 + 4 * c + i > last) v = 0, e = 0;
      const float sc = scale_of(e);
      x[0][i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(v, sc, 0));
      x[1][i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(v, sc, 1));
      if constexpr (D == 128) {
        x[2][i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(v, sc, 2));
        x[3][i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(v, sc, 3));
      }
    }
#pragma unroll
    for (int m = 0; m < W; ++m)
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        const uint32_t sel = b ? 0x07060302u : 0x05040100u;
        const int row = (D / 16) * o + 2 * m + b;
        u32x2 y = {__builtin_amdgcn_perm(x[m][1], x[m][0], sel), __builtin_amdgcn_perm(x[m][3], x[m][2], sel)};
        *reinterpret_cast<u32x2*>(vd + row * 32 + (((c & 1) ^ ((row >> 3) & 1)) << 4) + (c >> 1) * 8) = y;
      }
  }
}

}  // namespace kv4
}  // namespace kafka
