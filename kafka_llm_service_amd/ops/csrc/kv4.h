// Pages of the 4-bit cache (kv_dtype "mx4"), gfx950.
//
// A page holds 16 keys of one key/value head, D = 64 or 128: elements e2m1 (0, 1/2, 1, 3/2, 2, 3, 4, 6 and their negatives) and one
// power of two for every 32 elements of a key, as a byte of its exponent + 127; K and V pages are as large, 16 (D/2 + D/32) bytes.
//   K data   key o at byte o D/2, element d in byte d/2 (even d: the low half). A lane (key l & 15, quarter c = l >> 4) of
//            v_mfma_f32_16x16x32_bf16 takes the D/4 elements from c D/4 on, one 16-byte piece at D = 128 (all its k-steps, since the
//            order of the sum over d is free as long as Q's fragments follow it) and one scale; a wave's load is the whole page.
//   V data   byte ((o / 4) (D/8) + d / 8) 16 + (o % 4) 4 + (d % 8) / 2: a lane (c = l >> 4, d / 8 = l & 15) gets its eight d's of the
//            keys 4c .. 4c + 3, which are those that the lane's scores of a 16 x 16 tile belong to, in one 16-byte piece.
//   scales   behind the data: K of key o, group g at o D/32 + g (a key's are one word), V at 16 g + o (four keys' are one word).
#pragma once
#include "common.h"

namespace kafka {
namespace kv4 {

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int PAGE = 16;
constexpr int EXP_MIN = -124, EXP_MAX = 125;  // 1/2 * 2^-124 is a normal number, 6 * 2^125 a finite one, in fp32 and bf16

template <int D>
struct Page {
  static constexpr int DATA = PAGE * D / 2, BYTES = DATA + PAGE * D / 32;
};

__device__ __forceinline__ float scale_of(uint32_t byte) { return __uint_as_float(byte << 23); }

// eight elements (a word) times a power of two
__device__ __forceinline__ bf16x8 widen8(uint32_t w, float sc) {
  const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, sc, 0), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, sc, 1);
  const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, sc, 2), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, sc, 3);
  return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// eight numbers as a word of e2m1, divided by the power of two sc: nearest, ties to the even code, the largest beyond 6
__device__ __forceinline__ uint32_t narrow8(bf16x8 x, float sc) {
  uint32_t w = 0;
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, bf16x2{x[0], x[1]}, sc, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, bf16x2{x[2], x[3]}, sc, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, bf16x2{x[4], x[5]}, sc, 2);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, bf16x2{x[6], x[7]}, sc, 3);
  return w;
}

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x6 __attribute__((ext_vector_type(6)));

// a [16 rows][128] in e2m1, a lane's 32 elements of k = 32 (l >> 4) on in its first four words, times 2^(sa - 127); b [128][16 columns] in e2m3, a
// lane's 32 of the same k in six words, times 2^(e - 127), e the byte BYTE of sb (255: no number).
// The instruction adds the products of eight neighbouring k, each cut (towards zero) to multiples of 2^-13 of the largest one's power of two, and
// such sums in fp32 (measured: beside 256 a product of 2^-5 is whole, one of 2^-6 gone, in another eight of k it is whole down to 2^-16). Whole numbers
// of up to 16 steps of 1/8, which e2m3 holds all, times a key's of up to 12 halves lose nothing of that: products are multiples of 1/16 up to 12.
// (The compiler does not know that the product needs every lane of its operands: results are pinned where control flow is uniform.)
template <int BYTE>
__device__ __forceinline__ f32x4 mfma4x6(const uint32_t* a, uint32_t sa, const u32x6& b, uint32_t sb, f32x4 c) {
  const i32x8 x = {(int)a[0], (int)a[1], (int)a[2], (int)a[3], 0, 0, 0, 0};
  const i32x8 y = {(int)b[0], (int)b[1], (int)b[2], (int)b[3], (int)b[4], (int)b[5], 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(x, y, c, 4, 2, 0, (int)sa, BYTE, (int)sb);
}

// The same with the operands in each other's place: a [16 rows][128] in e2m3, b [128][16 columns] in e2m1
template <int BYTE>
__device__ __forceinline__ f32x4 mfma6x4(const u32x6& a, uint32_t sa, const uint32_t* b, uint32_t sb, f32x4 c) {
  const i32x8 x = {(int)a[0], (int)a[1], (int)a[2], (int)a[3], (int)a[4], (int)a[5], 0, 0};
  const i32x8 y = {(int)b[0], (int)b[1], (int)b[2], (int)b[3], 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(x, y, c, 2, 4, BYTE, (int)sa, 0, (int)sb);
}

__device__ __forceinline__ f32x4 mfma16(bf16x8 a, bf16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

}  // namespace kv4
}  // namespace kafka
