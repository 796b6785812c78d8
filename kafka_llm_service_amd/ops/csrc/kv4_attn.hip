// Attention over the 4-bit cache, and the weight that its keys receive (pages: kv4.h; gfx950).
//
// A call's rows are segments of consecutive tokens of one sequence each; the row at position p sees the keys j <= p, with a window only
// those with j > p - window or j < first. A work item is a tile of a segment's tokens and a range of the blocks of 64 keys that
// any of them sees (the first ones, then those from the window's start on: a block in the range is a place in this list).
//
//   S^T[key][row] = K . Q^T    A: K in four bits as it lies, B: Q in four parts of e2m3, 20 bits of fixed point
//   O^T[d][row]  += V^T . P    A: a lane's values of four keys, two neighbouring d's a register as they are widened (exactly), B: P as S^T's
//                              registers hold it, beside zeros for the other d: twice the products, but no register is turned
// The softmax runs in one pass with a running maximum per row; its sums and maxima are fp32, P is rounded to bf16 for the product.
//
// Single tokens are bound by the pages' bytes where the work on them fits beside: the matrix cores take K as it lies, so that what is left is mostly
// the widening of V. 64 threads of 4100 tokens, 32/8 heads of 128: 56 us, 5.1 TB/s (a large copy's rate); one thread of 1511 7.6 us: launch,
// four reads that wait for each other (item, page ids, pages, parts) and the join. Long portions go through kv4_tile.hip.
#include "attn_tile.h"
#include "kv4_widen.h"

#include <type_traits>

namespace kafka {
namespace kv4 {

constexpr int KB = 64;   // keys of a block

struct Item {
  int row, tokens;       // first row, rows
  int pos;               // position of the first
  int table;             // row of the block table
  int lo, hi;            // blocks of its list
  int slot;              // < 0: the rows are written here, else the first of the tile's partial results,
  int part;              // of which this is number part & 0xffff of part >> 16
};

struct Args {
  const bf16* q;
  int64_t qs;
  const uint8_t *kc, *vc;
  int64_t n_pages;
  const int* tables;
  int64_t ts;
  const Item* items;
  int T, Hkv, G;
  int window, first;     // (no window: 2^30)
  float scale2;          // scale * log2(e)
  bf16* out;
  int64_t os;
  float* lse;            // [T][Hq], may be null
  float *part, *plse;    // partial results: from slot Hkv + head * parts on of every split tile [parts][rows of a tile][D], [..][rows of a tile]
  int* counters;         // [slots][Hkv] zeros, and zeros again when the launch has ended
};

__device__ __forceinline__ float vmax(float a, float b) { return __builtin_elementwise_maximum(a, b); }
__device__ __forceinline__ float over_quarters_max(float x) {   // of the lanes with the same l & 15
  x = vmax(x, __shfl_xor(x, 16, 64));
  return vmax(x, __shfl_xor(x, 32, 64));
}
__device__ __forceinline__ float over_quarters_sum(float x) {
  x += __shfl_xor(x, 16, 64);
  return x + __shfl_xor(x, 32, 64);
}

// Of four numbers a lane the sums over the quarters, the c-th one in quarter c: halves, then rows of 16, of two registers change places
__device__ __forceinline__ float quarters_sums(const float (&x)[4]) {
  auto half = [](float a, float b) {
    const auto y = __builtin_amdgcn_permlane32_swap(__float_as_uint(a), __float_as_uint(b), false, false);
    return __uint_as_float(y[0]) + __uint_as_float(y[1]);
  };
  const auto y = __builtin_amdgcn_permlane16_swap(__float_as_uint(half(x[0], x[2])), __float_as_uint(half(x[1], x[3])), false, false);
  return __uint_as_float(y[0]) + __uint_as_float(y[1]);
}

// The list of blocks that a tile of rows at positions [p0, p1] sees
struct Blocks {
  int head, tail, count;   // blocks below ``head``, then from ``tail`` on
  __device__ __forceinline__ Blocks(int p0, int p1, int window, int first) {
    tail = max(0, p0 - window + 1) / KB;
    head = min((first + KB - 1) / KB, tail);
    count = p1 < 0 ? 0 : head + p1 / KB + 1 - tail;
  }
  __device__ __forceinline__ int operator[](int v) const { return v < head ? v : v - head + tail; }
};

struct Widen {
  const int* tiles;
  char* ws;
  uint32_t from;           // first workgroup
};

template <int NP>          // of NP pages
struct KFrag {
  uint32_t d[NP][4];       // a lane's 32 elements of a key
  uint32_t s[NP];
};
template <int NP>
struct VFrag {
  u32x4 d[NP];             // a word for each of four keys
  uint32_t s[NP];
};

// Page ids of 16 blocks of 4 pages, a lane each; of pages that no row at pmin .. pmax sees a key of, page 0 (the table may name anything
// there: pages that a window has left behind are their owner's again). One load for them all, ahead of their use: an id that is fetched in
// front of its page's loads adds a round trip to every block.
struct PageIds {
  int v = 0;
  __device__ __forceinline__ PageIds() {}
  template <class Of>
  __device__ __forceinline__ PageIds(const int* bt, int pmin, int pmax, int window, int first, int lane, Of block) {
    const int i = block(lane >> 2) * 4 + (lane & 3), key = 16 * i;
    v = bt[min(i, pmax >> 4)];
    if (key > pmax || (key + 15 <= pmin - window && key >= first)) v = 0;
  }
  // NP of them from lane ``at`` on. An id that is not of the cache counts as page 0 and sets ``bad``: such rows come out as no numbers.
  template <int NP>
  __device__ __forceinline__ void get(int at, uint32_t n_pages, uint32_t (&pg)[NP], bool& bad) const {
#pragma unroll
    for (int t = 0; t < NP; ++t) {
      const uint32_t p = __builtin_amdgcn_readlane(v, at + t);
      bad |= p >= n_pages;
      pg[t] = p < n_pages ? p : 0;
    }
  }
};

// (heads of 64: both halves of the lanes hold the key, for two parts of Q)
template <int D, int NP>
__device__ __forceinline__ void load_k(KFrag<NP>& f, const uint8_t* kh, uint32_t stride, const uint32_t (&pg)[NP], int lane) {
  const uint32_t key = lane & 15, g = (lane >> 4) & (D / 32 - 1), at = key * (D / 2) + g * 16, sc = Page<D>::DATA + key * (D / 32) + g;
#pragma unroll
  for (int t = 0; t < NP; ++t) {
    const uint8_t* p = kh + (uint64_t)pg[t] * stride;
    const u32x4 x = *reinterpret_cast<const u32x4*>(p + at);
#pragma unroll
    for (int i = 0; i < 4; ++i) f.d[t][i] = x[i];
    f.s[t] = p[sc];
  }
}

template <int D, int NP>
__device__ __forceinline__ void load_v(VFrag<NP>& f, const uint8_t* vh, uint32_t stride, const uint32_t (&pg)[NP], int lane) {
  const uint32_t dl = lane & 15, c = lane >> 4, at = (c * (D / 8) + dl * (D / 8) / 16) * 16, sc = Page<D>::DATA + (dl * (D / 16) / 32) * 16 + c * 4;
#pragma unroll
  for (int t = 0; t < NP; ++t) {
    const uint8_t* p = vh + (uint64_t)pg[t] * stride;
    f.d[t] = *reinterpret_cast<const u32x4*>(p + at);
    f.s[t] = *reinterpret_cast<const uint32_t*>(p + sc);
  }
}

// Q in fixed point, so that the matrix cores take the keys in four bits as they lie: of 32 elements the largest comes to 8 .. 16 steps, and four
// parts hold whole numbers of up to 16 in e2m3, each counting a 32nd of the one before: 20 bits, in which an element is whole down to 2^-11 of
// the largest (bf16 has eight bits) and off by at most 2^-19 of it below. Nothing of the products is cut (kv4.h), so scores are as
// exact as 32 bits make them. In two parts of e4m3, in which the instruction takes twice the cycles, the cut of their products was
// 2^-16 of sum |q_d k_d|, one-sided, and came out in lse and the masses.
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x32 __attribute__((ext_vector_type(32)));
typedef uint32_t u32x16 __attribute__((ext_vector_type(16)));
template <int D>
struct QFrag {
  u32x6 x[D / 32];          // heads of 128: the parts; of 64: parts 0 and 2 in the lower half of the lanes (of k), 1 and 3 in the upper
  uint32_t s;               // their scales, a byte each
};

template <int D, int NQ>
struct Rows {
  QFrag<D> q[NQ];
  int lim[NQ];              // a column's position; -1: no row
  f32x4 o[NQ][D / 16];      // register i of tile n: d = (D / 16) (4 c + i) + n
  float m[NQ], l[NQ];       // maximum so far (times scale, log2), this lane's part of the sum
};

// 16 columns from column R0 of the tile on; a lane takes 32 elements of its column
template <int D>
__device__ __forceinline__ int load_q(QFrag<D>& f, const Args& a, int row, int tokens, int pos, int h, int R0, int lane) {
  const int R = R0 + (lane & 15), tok = R / a.G, g = R - tok * a.G, c = lane >> 4;
  const bool there = tok < tokens;
  const bf16* p = a.q + (int64_t)(row + (there ? tok : 0)) * a.qs + (int64_t)(h * a.G + g) * D + 32 * (c & (D / 32 - 1));
  bf16x8 q[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) q[i] = load_bf16x8(p + 8 * i);
  uint32_t m = 0;                                            // the largest element's bits
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const u32x4 b = __builtin_bit_cast(u32x4, q[i]);
#pragma unroll
    for (int j = 0; j < 4; ++j) m = max(m, max(b[j] & 0x7fffu, (b[j] >> 16) & 0x7fffu));
  }
  if (!there) m = 0;
  const uint32_t e = max(m >> 7, 16u);                       // its exponent
  const float s = there ? __uint_as_float((257u - e) << 23) : 0.f;
  u32x16 x;                                                  // (eight bits from below 2^4 on: f16 holds them and what is left of them exactly)
#pragma unroll
  for (int i = 0; i < 16; ++i)
    x[i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz((float)q[i >> 2][2 * (i & 3)] * s, (float)q[i >> 2][2 * (i & 3) + 1] * s));
  // beyond the nearest whole number (of the sum with 1536, whose last bit is one; the packing rounds alike), 32 times
  auto rest = [&]() {
    const f16x2 big = {(_Float16)1536.f, (_Float16)1536.f};
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const f16x2 y = __builtin_bit_cast(f16x2, (uint32_t)x[i]);
      f16x2 t = y + big;
      asm volatile("" : "+v"(t));
      x[i] = __builtin_bit_cast(uint32_t, (y - (t - big)) * (_Float16)32.f);
    }
  };
  // (packed here: or the compiler packs all parts where they are used, and has what is left of each in registers until then)
  auto pack = [&](u32x6& part) {
    part = __builtin_amdgcn_cvt_scalef32_pk32_fp6_f16(__builtin_bit_cast(f16x32, x), 8.f);
    asm volatile("" : "+v"(part));
  };
  if constexpr (D == 128) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (i) rest();
      pack(f.x[i]);
    }
    f.s = e * 0x01010101u - 0x0f0a0500u;
  } else {
    if (c >= 2) rest();
    pack(f.x[0]);
    rest();
    rest();
    pack(f.x[1]);
    f.s = e * 0x0101u - (c < 2 ? 0x0a00u : 0x0f05u);
  }
  if (m >= 0x7f80u) f.s = ~0u;                               // (a row with an infinity or no number in it is no numbers)
  return there ? pos + tok : -1;
}

// the smallest part first
template <int D, class Product>
__device__ __forceinline__ f32x4 parts_sum(const QFrag<D>& q, Product product) {
  f32x4 s = {0.f, 0.f, 0.f, 0.f};
  if constexpr (D == 128) {
    s = product(q.x[3], std::integral_constant<int, 3>{}, s);
    s = product(q.x[2], std::integral_constant<int, 2>{}, s);
  }
  s = product(q.x[1], std::integral_constant<int, 1>{}, s);
  return product(q.x[0], std::integral_constant<int, 0>{}, s);
}

// Scores of 16 NP keys
template <int D, int NQ, int NP>
__device__ __forceinline__ void scores(const KFrag<NP>& f, const QFrag<D> (&q)[NQ], f32x4 (&s)[NP][NQ]) {
#pragma unroll
  for (int t = 0; t < NP; ++t)
#pragma unroll
    for (int n = 0; n < NQ; ++n)
      s[t][n] = parts_sum<D>(q[n], [&](const u32x6& x, auto i, f32x4 c) { return mfma4x6<decltype(i)::value>(f.d[t], f.s[t], x, q[n].s, c); });
#pragma unroll
  for (int t = 0; t < NP; ++t)
#pragma unroll
    for (int n = 0; n < NQ; ++n) asm volatile("" : "+v"(s[t][n]));
}

__device__ __forceinline__ bool sees(int key, int lim, int window, int first) { return key <= lim && (key > lim - window || key < first); }

// 16 NP keys from key0 on: scores, softmax, values
template <int D, int NQ, int NP>
__device__ __forceinline__ void keys_step(const KFrag<NP>& kf, VFrag<NP>& vf, Rows<D, NQ>& r, int key0, int pmin, int pmax, int window, int first,
                                          float scale2, int lane) {
  const int c = lane >> 4;
  f32x4 s[NP][NQ];
  scores<D, NQ, NP>(kf, r.q, s);
  if (key0 + 16 * NP - 1 > pmin || (key0 <= pmax - window && key0 + 16 * NP > first)) {
#pragma unroll
    for (int n = 0; n < NQ; ++n)
#pragma unroll
      for (int t = 0; t < NP; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (!sees(key0 + 16 * t + 4 * c + i, r.lim[n], window, first)) s[t][n][i] = -INFINITY;
    // where no row sees a key the page may hold anything, also scales that are no numbers: their weight is zero, so must they be
    if (key0 + 16 * NP - 1 > pmax || (key0 <= pmin - window && key0 + 16 * NP > first)) {
#pragma unroll
      for (int t = 0; t < NP; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int key = key0 + 16 * t + 4 * c + i;
          if (key > pmax || (key <= pmin - window && key >= first)) {
            vf.d[t][i] = 0u;
            vf.s[t] &= ~(255u << (8 * i));
          }
        }
    }
  }
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    float mx = vmax(vmax(s[0][n][0], s[0][n][1]), vmax(s[0][n][2], s[0][n][3]));
#pragma unroll
    for (int t = 1; t < NP; ++t) mx = vmax(vmax(vmax(mx, s[t][n][0]), s[t][n][1]), vmax(s[t][n][2], s[t][n][3]));
    // (the maximum is raised only where it has grown by 2^24, which sums of fp32 hold: most steps have nothing to exchange or scale)
    if (__any(!(mx * scale2 <= r.m[n] + 24.f))) {
      mx = vmax(r.m[n], over_quarters_max(mx) * scale2);
      const float f = mx == -INFINITY ? 1.f : fast_exp2(r.m[n] - mx);
      r.l[n] *= f;
#pragma unroll
      for (int d = 0; d < D / 16; ++d) r.o[n][d] *= f;
      r.m[n] = mx;
    }
  }
#pragma unroll
  for (int t = 0; t < NP; ++t) {
    bf16x8 p[NQ][2];                                            // weights of four keys, each beside a zero: for even d's, for odd ones
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      const float use = r.m[n] == -INFINITY ? 0.f : r.m[n];
      u32x4 x, y;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float e = fast_exp2(fmaf(s[t][n][i], scale2, -use));
        r.l[n] += e;
        x[i] = __builtin_bit_cast(uint32_t, bf16x2{(bf16)e, (bf16)0.f});
        y[i] = x[i] << 16;
      }
      p[n][0] = __builtin_bit_cast(bf16x8, x);
      p[n][1] = __builtin_bit_cast(bf16x8, y);
    }
    constexpr int W = D / 32;                                   // pairs of d a lane
    u32x4 x[W];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t w = vf.d[t][i];
      if (D == 64) w >>= 16 * (lane & 1);
      const float sc = __uint_as_float(i < 3 ? vf.s[t] << (23 - 8 * i) : vf.s[t] >> 1);   // (only its exponent counts)
      x[0][i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, sc, 0));
      x[1][i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, sc, 1));
      if constexpr (D == 128) {
        x[2][i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, sc, 2));
        x[3][i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, sc, 3));
      }
    }
#pragma unroll
    for (int m = 0; m < W; ++m)
#pragma unroll
      for (int n = 0; n < NQ; ++n)
#pragma unroll
        for (int b = 0; b < 2; ++b) r.o[n][2 * m + b] = mfma16(__builtin_bit_cast(bf16x8, x[m]), p[n][b], r.o[n][2 * m + b]);
  }
}

// Partial results (normalised, with their sums' logarithms) joined to what (M, L, o) holds: the first n of B
template <int B>
__device__ __forceinline__ void join(float& M, float& L, f32x4& o, const float (&l)[B], const f32x4 (&p)[B], int n) {
  float mx = M;
#pragma unroll
  for (int s = 0; s < B; ++s) mx = vmax(mx, l[s]);              // (those behind the last are the last once more)
  const float use = mx == -INFINITY ? 0.f : mx, f0 = fast_exp2(M - use);
  M = mx;
  L *= f0;
  o *= f0;
#pragma unroll
  for (int s = 0; s < B; ++s) {
    const float f = s < n ? fast_exp2(l[s] - use) : 0.f;
    L += f;
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] = fmaf(p[s][j], f, o[j]);
  }
}

// NW waves take a tile of 16 NQ rows, every NW-th block each; their results meet in LDS. A wave has NB half blocks in registers: one that it
// works on, the others on their way. (The loop's first form fetches without a condition, so that the waits count what is on its way.)
// Three waves a SIMD with two half blocks each: 64 threads of 4100 tokens and 29 of 7900 56.7 and 56.7 us, three halves 57.2 and 57.6, two waves with
// four 58.0 and 57.1, four with one 57.6 and 61.3 (with Q in two parts of e4m3; in four of e2m3 57.4 and 57.2). NQ 2, short portions: values are widened once for 32 rows; 4 portions of 100 rows behind
// 1000 keys, 32/8 heads of 128, 23 us (26 with other inputs each time), as tiles of 256 rows whose keys are widened first 31. That is five times its operations' time: about a
// hundred scalar registers of this form do not fit and go through lanes in the loop, each product with values is done twice, and values are widened for every 32 rows anew.
// WIDEN: the workgroups behind the items' widen the step's long portions' keys on the way (kv4_tile.hip), which as a launch of its own would
// wait for this one, 6 us of mostly waiting (5 tokens and 3 portions of 1100, heads of 64, window 512: 43 us apart, 39.6 together).
template <int D, int NQ, int NW, int NB, bool WIDEN>
__global__ __launch_bounds__(64 * NW, NQ == 1 ? 3 : 2) void attn_kernel(Args a, Widen wd) {
  if constexpr (WIDEN) {
    static_assert(NW == 4, "a wave a page");
    if (blockIdx.x >= wd.from) {
      widen_tile<D>(blockIdx.x - wd.from, a.kc, a.vc, a.n_pages, a.tables, a.ts, wd.tiles, a.Hkv, a.window, a.first, wd.ws);
      return;
    }
  }
  constexpr int LD = D + 4;                                     // (16 lanes a quarter write 16 rows: other banks each)
  __shared__ float sO[NW][16][LD];
  __shared__ float sM[NW][16], sL[NW][16];
  __shared__ bool s_last;
  const Item it = a.items[blockIdx.x / a.Hkv];
  const int h = blockIdx.x % a.Hkv, lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int q = lane & 15, c = lane >> 4;
  // (an item outside of the rows is dropped)
  if (it.row < 0 || it.tokens <= 0 || it.row + it.tokens > a.T || it.tokens * a.G > 16 * NQ) return;
  const int pmin = it.pos, pmax = it.pos + it.tokens - 1;
  const Blocks list(pmin, pmax, a.window, a.first);
  const int* bt = a.tables + it.table * a.ts;
  const int hi = min(it.hi, list.count);
  Rows<D, NQ> r;
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    r.lim[n] = -1;
    r.m[n] = -INFINITY;
    r.l[n] = 0.f;
#pragma unroll
    for (int d = 0; d < D / 16; ++d) r.o[n][d] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  bool bad = false;
  const int v0 = it.lo + w, n = (hi - v0 + NW - 1) / NW * 2;    // halves of this wave's blocks: v0, v0 + NW, ..
  if (hi > v0) {
    auto ids = [&](int k) { return PageIds(bt, pmin, pmax, a.window, a.first, lane, [&](int i) { return list[min(v0 + NW * (k / 2 + i), hi - 1)]; }); };
    PageIds id = ids(0), idn = ids(32);
    const uint32_t stride = a.Hkv * Page<D>::BYTES;             // of a page of all heads
    KFrag<2> kf[NB];
    VFrag<2> vf[NB];
    auto fetch = [&](int x, int k) {
      if (k && k % 32 == 0) {
        id = idn;
        idn = ids(k + 32);
      }
      uint32_t pg[2];
      id.get<2>(k % 32 * 2, (uint32_t)a.n_pages, pg, bad);
      load_k<D, 2>(kf[x], a.kc + h * Page<D>::BYTES, stride, pg, lane);
      load_v<D, 2>(vf[x], a.vc + h * Page<D>::BYTES, stride, pg, lane);
    };
    auto step = [&](int x, int k) {
      keys_step<D, NQ, 2>(kf[x], vf[x], r, list[v0 + NW * (k >> 1)] * KB + 32 * (k & 1), pmin, pmax, a.window, a.first, a.scale2, lane);
    };
#pragma unroll
    for (int x = 0; x < NB; ++x)
      if (x < n) fetch(x, x);
#pragma unroll
    for (int m = 0; m < NQ; ++m) r.lim[m] = load_q<D>(r.q[m], a, it.row, it.tokens, it.pos, h, 16 * m, lane);
    int k = 0;
    for (; k + 2 * NB <= n; k += NB)
#pragma unroll
      for (int x = 0; x < NB; ++x) {
        step(x, k + x);
        fetch(x, k + x + NB);
      }
    for (; k < n; k += NB)
#pragma unroll
      for (int x = 0; x < NB; ++x)
        if (k + x < n) {
          step(x, k + x);
          if (k + x + NB < n) fetch(x, k + x + NB);
        }
  }
  const int Hq = a.Hkv * a.G, parts = it.part >> 16;
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    const int live = min(16, it.tokens * a.G - 16 * n);         // columns of the tile that are rows
    if (live <= 0) break;
    const float l = over_quarters_sum(r.l[n]);
    if (n) __syncthreads();
    if (q < live) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int d = 0; d < D / 16; d += 4)
          *reinterpret_cast<f32x4*>(&sO[w][q][(D / 16) * (4 * c + i) + d]) =
              f32x4{r.o[n][d][i], r.o[n][d + 1][i], r.o[n][d + 2][i], r.o[n][d + 3][i]};
      if (c == 0) {
        sM[w][q] = r.m[n];
        sL[w][q] = bad ? __builtin_nanf("") : l;
      }
    }
    __syncthreads();
    for (int x = threadIdx.x; x < live * (D / 4); x += 64 * NW) {
      const int row = x / (D / 4), d0 = (x % (D / 4)) * 4, R = 16 * n + row, tok = R / a.G, g = R - tok * a.G;
      float M = sM[0][row];
#pragma unroll
      for (int i = 1; i < NW; ++i) M = vmax(M, sM[i][row]);
      float L = 0.f;
      f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < NW; ++i) {
        const float f = M == -INFINITY ? 1.f : fast_exp2(sM[i][row] - M);
        const f32x4 y = *reinterpret_cast<const f32x4*>(&sO[i][row][d0]);
        L = fmaf(f, sL[i][row], L);
#pragma unroll
        for (int j = 0; j < 4; ++j) o[j] = fmaf(f, y[j], o[j]);
      }
      const float inv = L == 0.f ? 0.f : 1.f / L, lse = L == 0.f ? -INFINITY : M + log2f(L);
#pragma unroll
      for (int j = 0; j < 4; ++j) o[j] *= inv;
      if (it.slot < 0) {
        *reinterpret_cast<bf16x4*>(a.out + (int64_t)(it.row + tok) * a.os + (int64_t)(h * a.G + g) * D + d0) =
            bf16x4{(bf16)o[0], (bf16)o[1], (bf16)o[2], (bf16)o[3]};
        if (a.lse && d0 == 0) a.lse[(int64_t)(it.row + tok) * Hq + h * a.G + g] = lse;
      } else {                                                  // (through to where the other XCDs see it)
        const int64_t at = ((int64_t)it.slot * a.Hkv + h * parts + (it.part & 0xffff)) * (16 * NQ) + R;
        store16_slab(a.part + at * D + d0, o);
        if (d0 == 0) __hip_atomic_store(a.plse + at, lse, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      }
    }
  }
  if (it.slot < 0) return;
  // ---- the last workgroup of a split tile joins its parts: each has waited for its stores before it counts itself, and the last one's loads go
  // past this XCD's cache; it leaves the counter zero
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (threadIdx.x == 0) {
    int* n = a.counters + (int64_t)it.slot * a.Hkv + h;
    const bool last = __hip_atomic_fetch_add(n, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == parts - 1;
    if (last) __hip_atomic_store(n, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    s_last = last;
  }
  __syncthreads();
  if (!s_last) return;
  constexpr int B = 8;                                          // parts on their way at a time
  const int64_t at = ((int64_t)it.slot * a.Hkv + h * parts) * (16 * NQ);
  const auto rp = buf_rsrc(a.part + at * D);                    // (at most 2^16 parts of 16 KiB)
  for (int x = threadIdx.x; x < it.tokens * a.G * (D / 4); x += 64 * NW) {
    const int R = x / (D / 4), d0 = (x % (D / 4)) * 4, tok = R / a.G, g = R - tok * a.G;
    float M = -INFINITY, L = 0.f;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    for (int s0 = 0; s0 < parts; s0 += B) {
      float l[B];
      f32x4 p[B];
#pragma unroll
      for (int s = 0; s < B; ++s) {
        const int i = min(s0 + s, parts - 1) * (16 * NQ) + R;
        l[s] = __hip_atomic_load(a.plse + at + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        p[s] = load16_sc1(rp, (i * D + d0) * 4);
      }
      join<B>(M, L, o, l, p, parts - s0);
    }
    const float inv = L == 0.f ? 0.f : 1.f / L;
    *reinterpret_cast<bf16x4*>(a.out + (int64_t)(it.row + tok) * a.os + (int64_t)(h * a.G + g) * D + d0) =
        bf16x4{(bf16)(o[0] * inv), (bf16)(o[1] * inv), (bf16)(o[2] * inv), (bf16)(o[3] * inv)};
    if (a.lse && d0 == 0) a.lse[(int64_t)(it.row + tok) * Hq + h * a.G + g] = L == 0.f ? -INFINITY : M + log2f(L);
  }
}

// Partial results of wide tiles (kv4_tile.hip), a thread for four elements of a row, eight parts on their way: 5 us, a launch and two
// reads that wait for each other. Merge items: first row, rows, first slot, slots.
template <int D>
__global__ __launch_bounds__(256) void merge_kernel(Args a, const int* __restrict__ merges, int tile_rows) {
  constexpr int B = 8;
  const int* it = merges + 4 * (blockIdx.x / a.Hkv);
  const int row0 = it[0], tokens = it[1], slot0 = it[2], n = it[3];
  const int h = blockIdx.x % a.Hkv, R = blockIdx.y * (256 / (D / 4)) + threadIdx.x / (D / 4), d0 = (threadIdx.x % (D / 4)) * 4;
  const int tok = R / a.G, g = R - tok * a.G;
  if (tok >= tokens || row0 + tokens > a.T || R >= tile_rows) return;
  const int64_t at = ((int64_t)slot0 * a.Hkv + h) * tile_rows + R, step = (int64_t)a.Hkv * tile_rows;
  float M = -INFINITY, L = 0.f;
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
  for (int s0 = 0; s0 < n; s0 += B) {
    float l[B];
    f32x4 p[B];
#pragma unroll
    for (int s = 0; s < B; ++s) {
      const int64_t i = at + min(s0 + s, n - 1) * step;
      l[s] = a.plse[i];
      p[s] = *reinterpret_cast<const f32x4*>(a.part + i * D + d0);
    }
    join<B>(M, L, o, l, p, n - s0);
  }
  const float inv = L == 0.f ? 0.f : 1.f / L;
  bf16x4 y;
#pragma unroll
  for (int j = 0; j < 4; ++j) y[j] = (bf16)(o[j] * inv);
  *reinterpret_cast<bf16x4*>(a.out + (int64_t)(row0 + tok) * a.os + (int64_t)(h * a.G + g) * D + d0) = y;
  if (a.lse && d0 == 0) a.lse[(int64_t)(row0 + tok) * (a.Hkv * a.G) + h * a.G + g] = L == 0.f ? -INFINITY : M + log2f(L);
}

// ---- weights of the keys ------------------------------------------------------------------------------------------------
// out[segment][head][key] = base + sum over the segment's rows and the head's queries of 2^(s - lse). Sums meet in a fixed order, so that a
// call's result does not depend on who ends first. Items of few rows: first row, rows, position, table row, segment, first block, behind the last, 0.
struct MassArgs {
  Args a;
  const float* base;      // may be null, or out
  float* out;
  int N;
};

// Here Q is the first operand: a lane has one key and the rows 4 c + i, so its weights add up in registers, and only the four quarters' sums
// meet at the end.

// acc[t] += weights of the block's key 16 t + (l & 15) in 16 rows, of which the lane has those whose lse and positions are ls and lim
__device__ __forceinline__ void add_weights(float (&acc)[4], f32x4 (&s)[4], const f32x4& ls, bool masked, int key0, const int (&lim)[4],
                                            const Args& a, int lane) {
#pragma unroll
  for (int t = 0; t < 4; ++t) asm volatile("" : "+v"(s[t]));
  if (masked) {
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (!sees(key0 + 16 * t + (lane & 15), lim[i], a.window, a.first)) s[t][i] = -INFINITY;
  }
#pragma unroll
  for (int t = 0; t < 4; ++t)
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[t] += fast_exp2(fmaf(s[t][i], a.scale2, -ls[i]));
}

// lse of 16 rows from R0 on
__device__ __forceinline__ float load_lse(const Args& a, int row, int tokens, int h, int R0, int lane) {
  const int R = R0 + (lane & 15), tok = R / a.G, g = R - tok * a.G;
  const float x = a.lse[(int64_t)(row + min(tok, tokens - 1)) * (a.Hkv * a.G) + h * a.G + g];
  return tok >= tokens || x == -INFINITY ? INFINITY : x;
}

// what the lanes l & 15 have of the rows 4 c + i
template <class T>
__device__ __forceinline__ void of_rows(T x, T (&y)[4], int lane) {
#pragma unroll
  for (int i = 0; i < 4; ++i) y[i] = __shfl(x, 4 * (lane >> 4) + i, 64);
}

// Segments of at most 16 rows: four waves take every fourth block of an item's (at most 32), NB of them in registers. What a key had before
// comes with it: a load that is asked for when its sum is there holds up those of the next keys. Bytes bound it, and the start and
// end of workgroups of 28 blocks: 29 threads of 7900 tokens, 8 heads of 128, 140 MB, 31 us, 4.5 TB/s, behind the
// attention over the same pages, 36 by itself over others each time. Heads of 128 take four waves a SIMD: five leave too few registers for the parts of Q (103 us).
template <int D, int NB>
__global__ __launch_bounds__(256, D == 128 ? 4 : 5) void mass_few_kernel(MassArgs ma) {
  const Args& a = ma.a;
  const int* it = reinterpret_cast<const int*>(a.items) + 8 * (blockIdx.x / a.Hkv);
  const int row = it[0], rows = it[1], pos = it[2], table = it[3], seg = it[4], end = it[6];
  const int h = blockIdx.x % a.Hkv, lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = lane >> 4, last = pos + rows - 1, b0 = it[5] + w;
  if (end - it[5] > 32 || b0 >= end) return;
  const int64_t at = ((int64_t)seg * a.Hkv + h) * ma.N;
  float* out = ma.out + at;
  const float* base = ma.base ? ma.base + at : out;
  const int n = (end - b0 + 3) / 4;
  if (rows == 0) {                                         // (of a segment without rows the first one may be any)
    for (int k = 0; k < n; ++k) {
      const int key = (b0 + 4 * k) * KB + lane;
      if (key < ma.N) out[key] = ma.base ? base[key] : 0.f;
    }
    return;
  }
  if (row < 0 || rows < 0 || row + rows > a.T || rows * a.G > 16) return;
  const Blocks list(pos, last, a.window, a.first);
  // blocks that no row sees give nothing: behind the last key, between the first ones and the window
  auto seen = [&](int b) { return b * KB <= last && (b < list.head || b >= list.tail); };
  const PageIds id(a.tables + table * a.ts, pos, last, a.window, a.first, lane, [&](int i) { return b0 + 4 * min(i, 7); });
  bool bad[NB];
  KFrag<4> kf[NB];
  float had[NB];
  // (without conditions, so that the waits count what is on its way: behind the last block that one again, of no row some page)
  auto fetch = [&](int x, int k) {
    k = min(k, n - 1);
    uint32_t pg[4];
    bad[x] = false;
    id.get<4>(4 * k, (uint32_t)a.n_pages, pg, bad[x]);
    load_k<D, 4>(kf[x], a.kc + h * Page<D>::BYTES, a.Hkv * Page<D>::BYTES, pg, lane);
    had[x] = base[min((b0 + 4 * k) * KB + lane, ma.N - 1)];
  };
#pragma unroll
  for (int x = 0; x < NB; ++x) fetch(x, x);
  QFrag<D> qf;
  int lim[4];
  of_rows(load_q<D>(qf, a, row, rows, pos, h, 0, lane), lim, lane);
  float l4[4];
  of_rows(load_lse(a, row, rows, h, 0, lane), l4, lane);
  const f32x4 ls = {l4[0], l4[1], l4[2], l4[3]};
  for (int k = 0; k < n; k += NB)
#pragma unroll
    for (int x = 0; x < NB; ++x) {
      const int b = b0 + 4 * (k + x), key0 = b * KB;
      float acc[4] = {};
      f32x4 s[4];
#pragma unroll
      for (int t = 0; t < 4; ++t)
        s[t] = parts_sum<D>(qf, [&](const u32x6& y, auto i, f32x4 c) { return mfma6x4<decltype(i)::value>(y, qf.s, kf[x].d[t], kf[x].s[t], c); });
      add_weights(acc, s, ls, key0 + KB - 1 > pos || (key0 <= last - a.window && key0 + KB > a.first), key0, lim, a, lane);
      float mine = quarters_sums(acc);                     // lane = key: that of tile c
      if (bad[x]) mine = __builtin_nanf("");
      if (!seen(b)) mine = 0.f;
      if (k + x < n && key0 + lane < ma.N) out[key0 + lane] = (ma.base ? had[x] : 0.f) + mine;
      fetch(x, k + x + NB);
    }
}

// Longer segments: four waves, a block of keys each, its keys widened in registers, go through the same rows, all that may see one of the
// blocks or a part of them, in stages of 64 that stay in LDS for all four (each wave's own loads of 16 rows, 256 bytes apart, would take
// 64 cycles a load of what the CU has for all its waves). A lane has one of 16 rows and a quarter of
// the keys, each key's sum by itself: no lane asks another for anything until the rows end. Parts of a block's rows are joined in their
// order by the last workgroup of them to end (attn_kernel). Exponentials and products bound it, one after the other on a SIMD: 1900 rows
// behind 1000 keys, 32/8 heads of 128, 42 us, 480 TFLOP/s (each wave with rows of its own 85 us; 500 cycles for 16 rows and 64 keys, 256 of them products).
// (11 scalar registers, of heads of 64 seven, go through lanes, outside of the products.)
// Items: first row, rows, position, table row, segment, block, first column, behind the last, first slot or -1, part | parts << 16, 0, 0.
template <int D>
__global__ __launch_bounds__(256, 3) void mass_many_kernel(MassArgs ma) {
  constexpr int CH = 64, STAGE = CH * D * 2, PIECES = STAGE / 4096;
  const Args& a = ma.a;
  // (one object: of several the compiler knows which one a load fills, and waits for it ahead of every read)
  __shared__ __attribute__((aligned(1024))) char smem[2 * STAGE + 2 * CH * 4];
  char* const rows_q = smem;
  char* const rows_l = smem + 2 * STAGE;
  const int* it = reinterpret_cast<const int*>(a.items) + 12 * (blockIdx.x / a.Hkv);
  const int row = it[0], rows = it[1], pos = it[2], table = it[3], seg = it[4], slot = it[8], part = it[9] & 0xffff, parts = it[9] >> 16;
  const int h = blockIdx.x % a.Hkv, lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = lane >> 4, last = pos + rows - 1, G = a.G, key0 = (it[5] + w) * KB;
  if (row < 0 || rows < 0 || row + rows > a.T) return;
  float acc[16] = {};
  bool bad = false, any = false;
  const int R1 = min(it[7], rows * G);
  if (it[6] < R1) {
    // x / G of x < 80
    const uint32_t inv = 65536u / G + 1;
    int tok = it[6] / G, rem = it[6] - tok * G;            // token and query head of the next stage's first column
    const int Hq = a.Hkv * G;
    const bf16* q0 = a.q + (int64_t)row * a.qs + (int64_t)h * G * D;
    const float* l0 = a.lse + (int64_t)row * Hq + h * G;
    // The 16 bytes k of row r lie at k ^ r (heads of 64: k ^ r / 2): 16 lanes read them without a bank taken twice. Behind the last row: some row.
    auto stage = [&](int buf) {
      const int t0 = min(tok, rows - 1);
      auto of = [&](int r, uint32_t& dx, uint32_t& g) {    // row and head of column r, none behind the last
        const uint32_t x = rem + r;
        dx = x * inv >> 16, g = x - dx * G;
        dx = min(dx, (uint32_t)(rows - 1 - t0));
      };
      uint32_t dx, g;
      int ln = lane;
      asm volatile("" : "+v"(ln));                         // (or its multiples of every piece stay in registers all the time)
#pragma unroll
      for (int i = 0; i < PIECES; ++i) {
        const int p = PIECES * w + i, n = D / 8, r = p * (64 / n) + ln / n, k = (ln & (n - 1)) ^ (D == 128 ? r & 15 : r >> 1 & 7);
        of(r, dx, g);
        __builtin_amdgcn_raw_ptr_buffer_load_lds(buf_rsrc(q0 + t0 * a.qs), (lds_void_t*)(rows_q + buf * STAGE + 1024 * p), 16,
                                                 2 * (dx * (uint32_t)a.qs + g * D) + 16 * k, 0, 0, 0);
      }
      if (w == 0) {
        of(ln, dx, g);
        __builtin_amdgcn_raw_ptr_buffer_load_lds(buf_rsrc(l0 + (int64_t)t0 * Hq), (lds_void_t*)(rows_l + buf * (CH * 4)), 4, 4 * (dx * Hq + g), 0, 0, 0);
      }
    };
    stage(0);
    bf16x8 k[4][D / 32];
    {
      uint32_t pg[4];
      u32x4 kw[4];
      uint32_t ks[4];
      PageIds(a.tables + table * a.ts, pos, last, a.window, a.first, lane, [&](int) { return it[5] + w; }).get<4>(0, (uint32_t)a.n_pages, pg, bad);
#pragma unroll
      for (int t = 0; t < 4; ++t) {                        // a quarter of a key, D / 4 elements, is a lane's for all steps of the products
        const uint8_t* p = a.kc + ((int64_t)pg[t] * a.Hkv + h) * Page<D>::BYTES;
        const uint8_t* kp = p + (lane & 15) * (D / 2) + c * (D / 8);
        if constexpr (D == 128) {
          kw[t] = *reinterpret_cast<const u32x4*>(kp);
        } else {
          const u32x2 y = *reinterpret_cast<const u32x2*>(kp);
          kw[t] = u32x4{y[0], y[1], 0, 0};
        }
        ks[t] = p[Page<D>::DATA + (lane & 15) * (D / 32) + c * (D / 32) / 4];
      }
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int i = 0; i < D / 32; ++i) k[t][i] = widen8(kw[t][i], scale_of(ks[t]));
    }
    int buf = 0;
    for (int R = it[6]; R < R1; R += CH, buf ^= 1) {
      const int tok0 = tok, rem0 = rem;
      rem += CH % G, tok += CH / G;
      if (rem >= G) ++tok, rem -= G;
      t3_wait_vmcnt<0>();                                  // this stage; and all have done with the one before the next takes its place
      t3_barrier();
      if (R + CH < R1) stage(buf ^ 1);
      // scores of the 16 rows from j on, times 2^(- their lse)
      const char* const qb = rows_q + buf * STAGE + (lane & 15) * (2 * D);
      const char* const lb = rows_l + buf * (CH * 4) + 4 * (lane & 15);
      auto tile = [&](int j, auto mask) {
        bf16x8 q[D / 32];
#pragma unroll
        for (int i = 0; i < D / 32; ++i)
          q[i] = *reinterpret_cast<const bf16x8*>(qb + j * (2 * D) + 16 * ((D / 32 * c + i) ^ (D == 128 ? lane & 15 : lane >> 1 & 7)));
        const float x = *reinterpret_cast<const float*>(lb + 4 * j), l = x == -INFINITY ? INFINITY : x;   // (a row that sees nothing has no weights)
#pragma unroll
        for (int u = 0; u < 4; u += 2) {
          f32x4 s[2];
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            s[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < D / 32; ++i) s[t] = mfma16(k[u + t][i], q[i], s[t]);
          }
#pragma unroll
          for (int t = 0; t < 2; ++t) asm volatile("" : "+v"(s[t]));
          mask(s, u);
#pragma unroll
          for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[4 * (u + t) + i] += fast_exp2(fmaf(s[t][i], a.scale2, -l));
        }
      };
      const int pmin = pos + tok0, pmax = pmin + (int)((rem0 + CH - 1) * inv >> 16);
      if (R + CH <= R1 && pmin >= key0 + KB - 1 && pmax <= last && (pmax - a.window < key0 || key0 + KB <= a.first)) {
        any = true;                                        // all of the rows see all of the keys
#pragma unroll
        for (int j = 0; j < CH; j += 16) tile(j, [](auto&, int) {});
        continue;
      }
#pragma unroll 1
      for (int j = 0; j < CH; j += 16) {
        const int p0 = pos + tok0 + (int)((rem0 + j) * inv >> 16), p1 = pos + tok0 + (int)((rem0 + j + 15) * inv >> 16);
        if (R + j >= R1 || p1 < key0 || (p0 - a.window >= key0 + KB - 1 && key0 >= a.first)) continue;
        any = true;
        const int t = tok0 + (int)((rem0 + j + (lane & 15)) * inv >> 16), lim = t < rows ? pos + t : -1;
        tile(j, [&](f32x4(&s)[2], int u) {
#pragma unroll
          for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (!sees(key0 + 16 * (u + t) + 4 * c + i, lim, a.window, a.first)) s[t][i] = -INFINITY;
        });
      }
    }
  }
  // over the 16 rows: halves of the sums change places until a lane has one of them
#pragma unroll
  for (int n = 8; n; n /= 2)
#pragma unroll
    for (int j = 0; j < n; ++j) {
      const bool up = lane & n;
      const float keep = up ? acc[j + n] : acc[j], give = up ? acc[j] : acc[j + n];
      acc[j] = keep + __shfl_xor(give, n, 64);
    }
  float mine = bad && any ? __builtin_nanf("") : acc[0];
  if (slot >= 0) {
    float* p = a.part + (((int64_t)slot * a.Hkv + h * parts) * 4 + w) * KB + lane;
    __hip_atomic_store(p + part * (4 * KB), mine, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    int* n = a.counters + (int64_t)slot * a.Hkv + h;
    int* const before = reinterpret_cast<int*>(smem);      // (nobody reads rows any more)
    if (threadIdx.x == 0) *before = __hip_atomic_fetch_add(n, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    if (*before != parts - 1) return;
    if (threadIdx.x == 0) __hip_atomic_store(n, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    mine = 0.f;
    for (int i0 = 0; i0 < parts; i0 += 8) {
      float x[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = __hip_atomic_load(p + min(i0 + i, parts - 1) * (4 * KB), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
#pragma unroll
      for (int i = 0; i < 8; ++i) mine += i0 + i < parts ? x[i] : 0.f;
    }
  }
  const int key = key0 + 16 * ((lane & 15) >> 2) + 4 * c + (lane & 3);
  if (key < ma.N) {
    const int64_t at = ((int64_t)seg * a.Hkv + h) * ma.N + key;
    ma.out[at] = (ma.base ? ma.base[at] : 0.f) + mine;
  }
}

}  // namespace kv4

using namespace kv4;

static Args make_args(const bf16* q, int64_t qs, const uint8_t* kc, const uint8_t* vc, int64_t n_pages, const int* tables, int64_t ts,
                      const int* items, int T, int Hkv, int G, int window, int first, float scale, bf16* out, int64_t os, float* lse,
                      float* part, float* plse, int* counters = nullptr) {
  return Args{q,   qs, kc,  vc,   n_pages, tables, ts, reinterpret_cast<const Item*>(items), T, Hkv, G, window > 0 ? window : 1 << 30,
              first, scale * 1.4426950408889634f, out, os, lse, part, plse, counters};
}

extern "C" hipError_t kafka_kv4_merge(const int* merges, int n_merges, int tile_rows, int T, int Hkv, int G, int D, bf16* out, int64_t os,
                                      float* lse, float* part, float* plse, hipStream_t st) {
  const int per = 256 / (D / 4);
  const int64_t wgs = (int64_t)Hkv * n_merges;
  if ((D != 64 && D != 128) || wgs >= 1 << 24) return hipErrorInvalidValue;
  const Args a = make_args(nullptr, 0, nullptr, nullptr, 0, nullptr, 0, nullptr, T, Hkv, G, 0, 0, 1.f, out, os, lse, part, plse);
  const dim3 grid((unsigned)wgs, (tile_rows + per - 1) / per);
  if (D == 128)
    merge_kernel<128><<<grid, 256, 0, st>>>(a, merges, tile_rows);
  else
    merge_kernel<64><<<grid, 256, 0, st>>>(a, merges, tile_rows);
  return hipGetLastError();
}

// tiles of 16 nq rows, nw waves each; wtiles (four waves): what of the cache goes to ws beside them
extern "C" hipError_t kafka_kv4_attn(const bf16* q, int64_t qs, const uint8_t* kc, const uint8_t* vc, int64_t n_pages, const int* tables,
                                     int64_t ts, const int* items, int n_items, int nq, int nw, int T, int Hkv, int G, int D, int window,
                                     int first, float scale, bf16* out, int64_t os, float* lse, float* part, float* plse, int* counters,
                                     const int* wtiles, int n_wtiles, char* ws, hipStream_t st) {
  if (n_items == 0) return hipSuccess;
  const int64_t wgs = (int64_t)Hkv * n_items, wws = (int64_t)Hkv * n_wtiles;
  if ((D != 64 && D != 128) || G < 1 || G > 16 || wgs >= 1 << 24 || wws >= 1 << 24 || (n_wtiles && nw != 4)) return hipErrorInvalidValue;
  const Args a = make_args(q, qs, kc, vc, n_pages, tables, ts, items, T, Hkv, G, window, first, scale, out, os, lse, part, plse, counters);
  const Widen wd{wtiles, ws, (uint32_t)wgs};
  auto go = [&](auto kern) { kern<<<(unsigned)(wgs + wws), 64 * nw, 0, st>>>(a, wd); };
  auto dim = [&](auto d) {
    constexpr int DD = decltype(d)::value;
    if (nq == 1 && nw == 4) n_wtiles ? go(attn_kernel<DD, 1, 4, 2, true>) : go(attn_kernel<DD, 1, 4, 2, false>);
    else if (nq == 1 && nw == 8) go(attn_kernel<DD, 1, 8, 2, false>);
    else if (nq == 2 && nw == 4) n_wtiles ? go(attn_kernel<DD, 2, 4, 2, true>) : go(attn_kernel<DD, 2, 4, 2, false>);
    else return false;
    return true;
  };
  if (!(D == 128 ? dim(std::integral_constant<int, 128>{}) : dim(std::integral_constant<int, 64>{}))) return hipErrorInvalidValue;
  return hipGetLastError();
}

// few: items of segments of at most 16 rows; many: of those of more
extern "C" hipError_t kafka_kv4_mass(const bf16* q, int64_t qs, const float* lse, const uint8_t* kc, int64_t n_pages, const int* tables,
                                     int64_t ts, const int* few, int n_few, const int* many, int n_many, int T, int Hkv, int G, int D,
                                     int window, int first, float scale, const float* base, float* out, int N, float* part, int* counters,
                                     hipStream_t st) {
  if ((D != 64 && D != 128) || G < 1 || G > 16 || (int64_t)Hkv * n_few >= 1 << 24 || (int64_t)Hkv * n_many >= 1 << 24)
    return hipErrorInvalidValue;
  auto args = [&](const int* items) {
    return MassArgs{make_args(q, qs, kc, nullptr, n_pages, tables, ts, items, T, Hkv, G, window, first, scale, nullptr, 0,
                              const_cast<float*>(lse), part, nullptr, counters),
                    base, out, N};
  };
  if (n_few) {
    const MassArgs m = args(few);
    if (D == 128)
      mass_few_kernel<128, 2><<<Hkv * n_few, 256, 0, st>>>(m);
    else
      mass_few_kernel<64, 2><<<Hkv * n_few, 256, 0, st>>>(m);
  }
  if (n_many) {
    const MassArgs m = args(many);
    if (D == 128)
      mass_many_kernel<128><<<Hkv * n_many, 256, 0, st>>>(m);
    else
      mass_many_kernel<64><<<Hkv * n_many, 256, 0, st>>>(m);
  }
  return hipGetLastError();
}

}  // namespace kafka
