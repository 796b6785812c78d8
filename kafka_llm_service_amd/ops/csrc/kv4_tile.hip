// Attention of long portions over the 4-bit cache (pages: kv4.h; segments, items and what a row sees: kv4_attn.hip; gfx950).
//
// Of many rows the products bound it, and widening four bits in front of each product would double the work beside them. So the keys
// that a portion sees are widened once, to a workspace in the order in which the matrix cores take them, and every tile of rows copies them
// from there to LDS without a register or an address in between. The workspace is 4 bytes an element pair of K and V, written once and mostly
// read from the last-level cache.
#include "attn_tile.h"
#include "kv4_widen.h"

namespace kafka {
namespace kv4 {

template <int D>
__global__ __launch_bounds__(256) void widen_kernel(const uint8_t* __restrict__ kc, const uint8_t* __restrict__ vc, int64_t n_pages,
                                                    const int* __restrict__ tables, int64_t ts, const int* __restrict__ tiles, int Hkv,
                                                    int window, int first, char* __restrict__ ws) {
  widen_tile<D>(blockIdx.x, kc, vc, n_pages, tables, ts, tiles, Hkv, window, first, ws);
}

// ---- attention ----------------------------------------------------------------------------------------------------------
struct TileItem4 {
  int row, tokens, pos;    // first row, rows (times the query heads of a group: at most 32 a wave), position of the first
  int base, head, tail;    // the segment's first tile in the workspace; its list of blocks: below head, from tail on
  int lo, hi;              // places of this item in the tile's own list
  int slot;                // < 0: rows are written, else partial results
  int pad[3];
};

struct TileArgs {
  const bf16* q;
  int64_t qs;
  const char* ws;
  const TileItem4* items;
  int T, Hkv, G, window, first;
  float scale2;
  bf16* out;
  int64_t os;
  float *lse, *part, *plse;
};

// The lane's number, where registers are few (heads of 64) counted where it is used: what is computed from one that the compiler knows stays in
// registers through the loop, and a register too many there is a load from scratch, whose wait is one for all that is on its way to LDS
// (8000 rows, 32/8 heads, 325 us for 288).
template <int D>
__device__ __forceinline__ int lane_again(int lane) {
  if constexpr (D == 64) asm volatile("v_mbcnt_lo_u32_b32 %0, -1, 0\n\tv_mbcnt_hi_u32_b32 %0, -1, %0" : "=v"(lane));
  return lane;
}

// NW waves of 32 rows each. A wave is a pipeline over tiles of keys: between the products of the next tile's keys stand the
// exponentials of this one, between those of its values the rest of them and the next one's maxima, each product behind the LDS reads of the F
// fragments after it; keys run a tile ahead of the values, and the slots that a step has read are filled again in its middle, behind one counted
// wait and one barrier. The maximum is raised only where it has grown by more than 2^24 (sums of weights up to that are exact enough in fp32).
// What bounds it, by leaving one thing out at a time: 8000 rows cold, 32/8 heads of 128, 446 us, 1175 TFLOP/s (a large product of the library
// 1400), without the copies to LDS (32 KiB a tile and workgroup, 4.6 TB/s in all) 371, which is the products' own rate, without
// the exponentials 421, without the reads from LDS 422; heads of 64, which have half the products for an exponential, 272 us, 965
// TFLOP/s, without them 227, 236 and 258. So copies first, then exponentials and reads. Masks count where most blocks are at an edge: three
// portions of 1100 rows in a window of 512, heads of 64, 28.6 us, without masks 21.6. The scalar unit runs beside: 24 million instructions for 43 million vector ones.
// Heads of 64: three workgroups of four waves a CU, of 128 one of eight, whose ring of three slots (96 KiB) leaves no room for another. Below
// about 500 rows the tiles of 32 rows (kv4_attn.hip) are as fast.
template <int D, int NW, int NSLOT>
__global__ __launch_bounds__(64 * NW, D == 64 ? 3 : 1) void tile_kernel(TileArgs a) {
  constexpr int F = D / 16, NT = D / 32, KBYTES = Image<D>::KBYTES, PB = Image<D>::PAGE_BYTES;
  constexpr int PIECES = KBYTES / 1024, DPT = 2 * PIECES / NW;             // LDS copies of 1 KiB: of K or V of a tile, of a wave for both
  constexpr float THR = 24.f;
  __shared__ __attribute__((aligned(1024))) char smem[2 * NSLOT * KBYTES];
  const TileItem4 it = a.items[blockIdx.x / a.Hkv];
  const int kvh = blockIdx.x % a.Hkv, tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r = lane & 31, h = lane >> 5, Hq = a.Hkv * a.G;
  if (it.row < 0 || it.tokens <= 0 || it.row + it.tokens > a.T || it.tokens * a.G > 32 * NW) return;
  const int R = 32 * w + r, tok = R / a.G, head = kvh * a.G + (R - tok * a.G);
  const bool valid = tok < it.tokens;
  const int limit = valid ? it.pos + tok : -1;
  // what the wave's rows see: keys up to wmin are seen by all of them if they are within the windows of all
  const int wfirst = 32 * w / a.G, wlast = min((32 * w + 31) / a.G, it.tokens - 1);
  const bool idle = wfirst >= it.tokens;
  const int wmin = idle ? 0x3fffffff : it.pos + wfirst, wmax = idle ? -1 : it.pos + wlast;
  const int tail = max(0, it.pos - a.window + 1) / TK, first = min((a.first + TK - 1) / TK, tail);
  const int ntiles = max(0, min(it.hi, first + (it.pos + it.tokens - 1) / TK + 1 - tail) - it.lo);
  auto block = [&](int i) {               // block of processing index i
    const int v = it.lo + i;
    return v < first ? v : v - first + tail;
  };
  auto image = [&](int i) {
    const int b = block(i);
    return a.ws + ((int64_t)(it.base + (b < it.head ? b : b - it.tail + it.head)) * a.Hkv + kvh) * Image<D>::BYTES;
  };
  auto issue = [&](int g) {               // group g: the keys of index g, the values of g - 1
    char* kd = smem + (g % NSLOT) * KBYTES + w * (DPT / 2) * 1024;
    char* vd = smem + (NSLOT + (g + NSLOT - 1) % NSLOT) * KBYTES + w * (DPT / 2) * 1024;
    const int at = w * (DPT / 2) * 1024, ln = lane_again<D>(lane);
    if (g < ntiles || g == 1)
      dma_pieces<DPT / 2, 0>(reinterpret_cast<const bf16*>(image(min(g, ntiles - 1)) + at), 16 * ln, kd);
    if (g > 0) dma_pieces<DPT / 2, 0>(reinterpret_cast<const bf16*>(image(g - 1) + KBYTES + at), 16 * ln, vd);
  };
  f32x16 o[NT];
  float m = -INFINITY, ls[2] = {0.f, 0.f};              // (two sums: one's additions wait for each other)
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[t][i] = 0.f;
  if (ntiles > 0) {
    issue(0);
    bf16x8 qf[F];
    const bf16* qrow = a.q + (int64_t)(it.row + (valid ? tok : 0)) * a.qs + (int64_t)head * D + 8 * h;
#pragma unroll
    for (int k = 0; k < F; ++k) {
      qf[k] = load_bf16x8(qrow + 16 * k);
      if (!valid) qf[k] = bf16x8{};
    }
#pragma unroll
    for (int g = 1; g < NSLOT; ++g)
      if (g <= ntiles) issue(g);
    int kl = (r >> 4) * PB + (h * 16 + (r & 15)) * 16, vl = NSLOT * KBYTES + r * 32 + 16 * (h ^ ((r >> 3) & 1));
    if (D == 64) asm volatile("" : "+v"(kl), "+v"(vl));  // (a register each, not one for every summand)
    const char* const Kl = smem + kl;
    const char* const Vl = smem + vl;
    bf16x8 fr[F];
    f32x16 sa[2], sb[2];
    auto kfrag = [&](const char* k, int f) { return *reinterpret_cast<const bf16x8*>(k + (f & 1) * 2 * PB + (f >> 1) * 512); };
    auto vfrag = [&](const char* v, int f) { return *reinterpret_cast<const bf16x8*>(v + (f / NT) * PB + (f % NT) * 1024); };
    auto kslot = [&](int i) { return Kl + (i % NSLOT) * KBYTES; };
    auto vslot = [&](int i) { return Vl + (i % NSLOT) * KBYTES; };
    auto mask = [&](f32x16(&s)[2], int i) {
      const int key0 = block(i) * TK;
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) {
        const int k0 = key0 + 32 * kb;
        if ((k0 + 31 > wmin) | ((k0 <= wmax - a.window) & (k0 + 32 > a.first))) {
          const int k1 = k0 + 4 * (lane_again<D>(lane) >> 5);
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const int key = k1 + (e & 3) + 8 * (e >> 2);
            if (!(key <= limit && (key > limit - a.window || key < a.first))) s[kb][e] = -INFINITY;
          }
        }
      }
    };
    auto rescale = [&](float mx) {
      const float smax = t3_xor32_max(mx) * a.scale2;
      if (__any(!(smax <= m + THR))) {
        const float mn = fmaxf(m, smax), alpha = mn == -INFINITY ? 1.f : fast_exp2(m - mn);
#pragma unroll
        for (int t = 0; t < NT; ++t) o[t] *= alpha;
        ls[0] *= alpha;
        ls[1] *= alpha;
        m = mn;
      }
    };
    // every wave has read the keys of index j + 1 and the values of j, and group j + 2 has landed: their slots are filled again
    auto meet = [&](int j) {
      __builtin_amdgcn_s_waitcnt(0xC07F);              // lgkmcnt(0)
      t3_wait_tiles<DPT>(min(NSLOT - 2, max(0, ntiles - 1 - (j + 2))));
      t3_barrier();
      if (j + 1 + NSLOT <= ntiles) issue(j + 1 + NSLOT);
    };
    auto step = [&](auto last_c, int j, f32x16(&s)[2], f32x16(&sn)[2]) {
      constexpr bool LAST = decltype(last_c)::value;
      const f32x16 zero = {};
      const char *kc = kslot(j + 1), *vc = vslot(j);
      const float mu = m == -INFINITY ? 0.f : m;
      bf16x8 pf[2], pg[2];
      auto prob = [&](float x, int i) {
        const float e = fast_exp2(fmaf(x, a.scale2, -mu));
        ls[i & 1] += e;
        return (bf16)e;
      };
      if constexpr (LAST) {
#pragma unroll
        for (int p = 0; p < F; ++p) fr[p] = vfrag(vc, p);
#pragma unroll
        for (int p = 0; p < 16; ++p) pf[p >> 3][p & 7] = prob(s[0][p], p);
      } else {
#pragma unroll
        for (int p = 0; p < 2 * F; ++p) {
          sn[p & 1] = mfma32(fr[p % F], qf[p >> 1], p < 2 ? zero : sn[p & 1]);
#pragma unroll
          for (int x = 0; x < 8 / F; ++x) {
            const int i = p * (8 / F) + x;
            pf[i >> 3][i & 7] = prob(s[0][i], i);
          }
          fr[p % F] = p < F ? kfrag(kc, p + F) : vfrag(vc, p - F);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
#pragma unroll
      for (int p = 0; p < F; ++p) {
        o[p % NT] = mfma32(fr[p], pf[p / NT], o[p % NT]);
#pragma unroll
        for (int x = 0; x < 16 / F; ++x) {
          const int i = p * (16 / F) + x;
          pg[i >> 3][i & 7] = prob(s[1][i], i);
        }
        fr[p] = vfrag(vc, p + F);
        __builtin_amdgcn_sched_barrier(0);
      }
      float ma = 0.f, mb = 0.f;
      const char* kn = kslot(j + 2);
      if constexpr (!LAST) {
        asm volatile("" : "+v"(pg[0]), "+v"(pg[1]));   // (the compiler would move the exponentials to the products that take them)
        meet(j);
        mask(sn, j + 1);
        ma = t3_max(sn[0][0], sn[1][0]);
        mb = t3_max(sn[0][1], sn[1][1]);
      }
#pragma unroll
      for (int p = 0; p < F; ++p) {
        o[p % NT] = mfma32(fr[p], pg[p / NT], o[p % NT]);
        if constexpr (!LAST) {
#pragma unroll
          for (int i = p * (16 / F); i < (p + 1) * (16 / F); i += 2)
            if (i > 0) {
              ma = t3_max(t3_max(ma, sn[0][i]), sn[1][i]);
              mb = t3_max(t3_max(mb, sn[0][i + 1]), sn[1][i + 1]);
            }
          fr[p] = kfrag(kn, p);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      if constexpr (!LAST) rescale(t3_max(ma, mb));
    };
    t3_wait_vmcnt<DPT>();                              // (group 1 is whole whatever there is: its keys are the last ones' again where they are past them)
    t3_barrier();
#pragma unroll
    for (int p = 0; p < F; ++p) fr[p] = kfrag(Kl, p);
#pragma unroll
    for (int p = 0; p < 2 * F; ++p) {
      const f32x16 zero = {};
      sa[p & 1] = mfma32(fr[p % F], qf[p >> 1], p < 2 ? zero : sa[p & 1]);
      if (p < F) fr[p] = kfrag(Kl, p + F);
    }
    meet(-1);
#pragma unroll
    for (int p = 0; p < F; ++p) fr[p] = kfrag(kslot(1), p);
    mask(sa, 0);
    float mx = t3_max(sa[0][0], sa[1][0]);
#pragma unroll
    for (int i = 1; i < 16; ++i) mx = t3_max(t3_max(mx, sa[0][i]), sa[1][i]);
    rescale(mx);
    int j = 0;
    for (; j + 2 < ntiles; j += 2) {
      step(std::false_type{}, j, sa, sb);
      step(std::false_type{}, j + 1, sb, sa);
    }
    if (j + 1 < ntiles) {
      step(std::false_type{}, j, sa, sb);
      sa[0] = sb[0];
      sa[1] = sb[1];
      ++j;
    }
    step(std::true_type{}, j, sa, sb);
  }
  const float sum = t3_xor32_sum(ls[0] + ls[1]);
  const int l2 = lane_again<D>(lane);
  const int r2 = l2 & 31, h2 = l2 >> 5, R2 = 32 * w + r2, tok2 = R2 / a.G, head2 = kvh * a.G + (R2 - tok2 * a.G);
  // ---- rows, through LDS so that whole cache lines are stored
  __syncthreads();                                     // (every wave has read the last keys and values)
  const float inv = sum == 0.f ? 0.f : 1.f / sum, lse = sum == 0.f ? -INFINITY : m + log2f(sum);
  const int64_t prow = ((int64_t)max(it.slot, 0) * a.Hkv + kvh) * (32 * NW) + R2;
  if (tok2 < it.tokens && h2 == 0) {
    if (it.slot >= 0) a.plse[prow] = lse;
    else if (a.lse) a.lse[(int64_t)(it.row + tok2) * Hq + head2] = lse;
  }
  char* slab = smem + w * 4096;                        // 32 rows of 128 bytes
  const int cc = l2 & 7, nvalid = it.tokens * a.G - 32 * w;
#pragma unroll
  for (int rd = 0; rd < NT; ++rd) {                    // 32 columns of fp32, or every second time 64 of bf16
    if (it.slot >= 0) {
#pragma unroll
      for (int i4 = 0; i4 < 4; ++i4)
        *reinterpret_cast<f32x4*>(slab + r2 * 128 + 16 * ((2 * i4 + h2) ^ (r2 & 7))) =
            f32x4{o[rd][4 * i4] * inv, o[rd][4 * i4 + 1] * inv, o[rd][4 * i4 + 2] * inv, o[rd][4 * i4 + 3] * inv};
    } else {
#pragma unroll
      for (int i4 = 0; i4 < 4; ++i4) {
        bf16x4 v;
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = (bf16)(o[rd][4 * i4 + j] * inv);
        *reinterpret_cast<bf16x4*>(slab + r2 * 128 + 16 * ((4 * (rd & 1) + i4) ^ (r2 & 7)) + 8 * h2) = v;
      }
      if (!(rd & 1)) continue;
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int row = (l2 >> 3) + 8 * k;
      const f32x4 v = *reinterpret_cast<const f32x4*>(slab + row * 128 + 16 * (cc ^ (row & 7)));
      if (row < nvalid) {
        const int R3 = 32 * w + row, tok3 = R3 / a.G, head3 = kvh * a.G + R3 - tok3 * a.G;
        if (it.slot >= 0)
          *reinterpret_cast<f32x4*>(a.part + (((int64_t)it.slot * a.Hkv + kvh) * (32 * NW) + R3) * D + 32 * rd + 4 * cc) = v;
        else
          *reinterpret_cast<f32x4*>(a.out + (int64_t)(it.row + tok3) * a.os + (int64_t)head3 * D + 32 * (rd - 1) + 8 * cc) = v;
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }
}

}  // namespace kv4

using namespace kv4;

extern "C" hipError_t kafka_kv4_merge(const int* merges, int n_merges, int tile_rows, int T, int Hkv, int G, int D, bf16* out, int64_t os,
                                      float* lse, float* part, float* plse, hipStream_t st);

// items of 256 rows (D 128) or 128 (D 64); wtiles: what of the cache the workspace has to hold, tile after tile (none: it holds it already)
extern "C" hipError_t kafka_kv4_tiles(const bf16* q, int64_t qs, const uint8_t* kc, const uint8_t* vc, int64_t n_pages, const int* tables,
                                      int64_t ts, int rows, const int* items, int n_items, const int* wtiles, int n_wtiles,
                                      const int* merges, int n_merges, int T, int Hkv, int G, int D, int window, int first, float scale, bf16* out, int64_t os,
                                      float* lse, float* part, float* plse, char* ws, hipStream_t st) {
  if (n_items == 0) return hipSuccess;
  const int64_t wgs = (int64_t)Hkv * n_items, wws = (int64_t)Hkv * n_wtiles;
  if ((D != 64 && D != 128) || rows != (D == 128 ? 256 : 128) || G < 1 || G > 16 || wgs >= 1 << 24 || wws >= 1 << 24) return hipErrorInvalidValue;
  const TileArgs a{q,  qs, ws, reinterpret_cast<const TileItem4*>(items), T, Hkv, G, window > 0 ? window : 1 << 30, first,
                   scale * 1.4426950408889634f, out, os, lse, part, plse};
  if (D == 128) {
    if (n_wtiles) widen_kernel<128><<<(unsigned)wws, 256, 0, st>>>(kc, vc, n_pages, tables, ts, wtiles, Hkv, a.window, first, ws);
    tile_kernel<128, 8, 3><<<(unsigned)wgs, 512, 0, st>>>(a);
  } else {
    if (n_wtiles) widen_kernel<64><<<(unsigned)wws, 256, 0, st>>>(kc, vc, n_pages, tables, ts, wtiles, Hkv, a.window, first, ws);
    tile_kernel<64, 4, 3><<<(unsigned)wgs, 256, 0, st>>>(a);
  }
  if (n_merges) return kafka_kv4_merge(merges, n_merges, rows, T, Hkv, G, D, out, os, lse, part, plse, st);
  return hipGetLastError();
}

}  // namespace kafka
