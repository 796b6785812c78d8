// The 4-bit cache's writer, its reader and the eviction from it (pages: kv4.h).
#include "kv4.h"

namespace kafka {
namespace kv4 {

// ---- writer -----------------------------------------------------------------------------------------------------------
// Of 32 numbers (eight in each of four neighbouring lanes) the least e with |x| <= 6 * 2^e, as a byte e + 127. With the bits of a
// bf16 as an integer, 6 * 2^e is (e + 129) << 7 | 0x40, so the carry of + 0x3f says whether the mantissa is beyond 3/2.
__device__ __forceinline__ uint32_t scale_byte(bf16x8 x) {
  const u32x4 b = __builtin_bit_cast(u32x4, x);
  uint32_t m = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) m = max(m, max(b[j] & 0x7fffu, (b[j] >> 16) & 0x7fffu));
  m = max(m, (uint32_t)__shfl_xor((int)m, 1, 64));
  m = max(m, (uint32_t)__shfl_xor((int)m, 2, 64));
  return (uint32_t)min(max((int)((m + 0x3f) >> 7) - 129, EXP_MIN), EXP_MAX) + 127u;
}

// not a number counts as zero, an infinity as the largest that the scale holds: what is read back is always a number, so that no
// masked place can spoil a product
__device__ __forceinline__ bf16x8 numbers(bf16x8 x) {
#pragma unroll
  for (int j = 0; j < 8; ++j) x[j] = x[j] == x[j] ? x[j] : (bf16)0.f;
  return x;
}

// Rotation in fp32 without fused products (each product rounded by itself, as elementary operations give it: next to a border of
// two codes the last bit decides), rounded to bf16 as the cache in bf16 holds it, then to 4 bits. A thread takes eight
// pairs of a query or key head, or eight elements of a value head; four neighbours share a scale. Bytes bound it, most of them
// the step's rows and its queries: 16-byte accesses, no LDS, two exchanges with neighbours for a scale. 4099 rows of 32/8 heads of
// 128, 91 MB: 20 us, 4.6 TB/s; one row 3 us.
template <int D>
__global__ __launch_bounds__(256) void rope_write_kernel(const bf16* __restrict__ qkv, const float* __restrict__ qp, int S, int64_t ps,
                                                         int64_t qkv_stride, const int64_t* __restrict__ positions,
                                                         const float* __restrict__ cos_sin, int64_t n_pos, bf16* __restrict__ q_out, int64_t q_stride,
                                                         uint8_t* __restrict__ kc, uint8_t* __restrict__ vc,
                                                         const int64_t* __restrict__ slots, int64_t n_slots, int64_t total, int Hq, int Hkv) {
  constexpr int HALF = D / 2, RU = HALF / 8, VU = D / 8;
  const int n_rope = (Hq + Hkv) * RU, n_row = n_rope + Hkv * VU;   // (multiples of four, as is total)
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= total) return;
  const int t = (int)(i / n_row), u = (int)(i - (int64_t)t * n_row);
  int64_t slot = slots ? slots[t] : -1;
  const int64_t pos = positions[t];
  const bool turns = pos >= 0 && pos < n_pos;                      // (a row of a position without angles: no numbers, and not into the cache)
  if (slot >= n_slots || !turns) slot = -1;
  const int64_t row = (int64_t)t * qkv_stride;
  const int64_t page = slot >> 4;
  const int o = (int)(slot & 15);
  if (u < n_rope) {
    const int head = u / RU, c = (u % RU) * 8;
    float x1[8], x2[8];
    load_in8(x1, qkv, qp, S, ps, row + head * D + c);
    load_in8(x2, qkv, qp, S, ps, row + head * D + HALF + c);
    const float* cs = cos_sin + (turns ? pos : 0) * D + c;
    bf16x8 y1, y2;
    {
#pragma clang fp contract(off)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float co = cs[j], si = cs[HALF + j];
        const float ac = x1[j] * co, bs = x2[j] * si, bc = x2[j] * co, as = x1[j] * si;
        y1[j] = (bf16)(ac - bs);
        y2[j] = (bf16)(bc + as);
      }
    }
    if (head < Hq) {
      if (!turns) {
#pragma unroll
        for (int j = 0; j < 8; ++j) y1[j] = y2[j] = (bf16)__builtin_nanf("");
      }
      bf16* dst = q_out + t * q_stride + head * D + c;
      store_bf16x8(dst, y1);
      store_bf16x8(dst + HALF, y2);
      return;
    }
    y1 = numbers(y1);
    y2 = numbers(y2);
    const uint32_t b1 = scale_byte(y1), b2 = scale_byte(y2);
    if (slot < 0) return;
    uint8_t* k = kc + (page * Hkv + head - Hq) * (int64_t)Page<D>::BYTES;
    *reinterpret_cast<uint32_t*>(k + o * (D / 2) + c / 2) = narrow8(y1, scale_of(b1));
    *reinterpret_cast<uint32_t*>(k + o * (D / 2) + (HALF + c) / 2) = narrow8(y2, scale_of(b2));
    if ((c & 31) == 0) {
      k[Page<D>::DATA + o * (D / 32) + c / 32] = (uint8_t)b1;
      k[Page<D>::DATA + o * (D / 32) + (HALF + c) / 32] = (uint8_t)b2;
    }
  } else {
    const int head = (u - n_rope) / VU, p = (u - n_rope) % VU;
    float x[8];
    load_in8(x, qkv, qp, S, ps, row + (Hq + Hkv + head) * D + p * 8);
    bf16x8 y;
#pragma unroll
    for (int j = 0; j < 8; ++j) y[j] = (bf16)x[j];
    y = numbers(y);
    const uint32_t b = scale_byte(y);
    if (slot < 0) return;
    uint8_t* v = vc + (page * Hkv + head) * (int64_t)Page<D>::BYTES;
    *reinterpret_cast<uint32_t*>(v + ((o >> 2) * VU + p) * 16 + (o & 3) * 4) = narrow8(y, scale_of(b));
    if ((p & 3) == 0) v[Page<D>::DATA + (p >> 2) * 16 + o] = (uint8_t)b;
  }
}

// ---- reader -----------------------------------------------------------------------------------------------------------
// Keys and values of slots as bf16 rows, exactly: two bits of mantissa and a power of two. Negative slots give zeros, slots behind
// the cache no numbers. A thread takes eight elements of a key and of its value; what it writes bounds it (65536 slots of 8 heads of 128:
// 73 us, 4.7 TB/s in all).
template <int D>
__global__ __launch_bounds__(256) void read_kernel(const uint8_t* __restrict__ kc, const uint8_t* __restrict__ vc,
                                                   const int64_t* __restrict__ slots, int64_t n_slots, int64_t total, int Hkv,
                                                   bf16* __restrict__ k, bf16* __restrict__ v) {
  constexpr int U = D / 8;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= total) return;
  const int p = (int)(i % U);
  const int64_t th = i / U, t = th / Hkv;
  const int h = (int)(th - t * Hkv);
  const int64_t slot = slots[t];
  bf16x8 a, b;
  if (slot < 0 || slot >= n_slots) {
    const bf16 none = slot < 0 ? (bf16)0.f : (bf16)__builtin_nanf("");
#pragma unroll
    for (int j = 0; j < 8; ++j) a[j] = b[j] = none;
  } else {
    const int o = (int)(slot & 15);
    const int64_t at = ((slot >> 4) * Hkv + h) * (int64_t)Page<D>::BYTES;
    const uint32_t kw = *reinterpret_cast<const uint32_t*>(kc + at + o * (D / 2) + p * 4);
    const uint32_t vw = *reinterpret_cast<const uint32_t*>(vc + at + ((o >> 2) * U + p) * 16 + (o & 3) * 4);
    a = widen8(kw, scale_of(kc[at + Page<D>::DATA + o * (D / 32) + (p >> 2)]));
    b = widen8(vw, scale_of(vc[at + Page<D>::DATA + (p >> 2) * 16 + o]));
  }
  store_bf16x8(k + i * 8, a);
  store_bf16x8(v + i * 8, b);
}

// ---- eviction ---------------------------------------------------------------------------------------------------------
// Order of masses as of unsigned integers: the two zeros alike, not a number below everything.
__device__ __forceinline__ uint32_t rank_of(float x) {
  const uint32_t b = __float_as_uint(x), a = b & 0x7fffffffu;   // (by its bits: comparisons take the smallest numbers for zeros)
  if (a > 0x7f800000u) return 0u;
  return a == 0u ? 0x80000000u : (b & 0x80000000u) ? ~b : b | 0x80000000u;
}

constexpr int KEEP_NT = 1024, KEEP_NW = KEEP_NT / 64;

// Inclusive sum over a wave: shifts within rows of 16, then the last lane of a row to the next one, of the first half to the second.
__device__ __forceinline__ int wave_sums(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);
  return x;
}

// Exclusive sum over the workgroup's threads, and the whole. ``ws`` holds KEEP_NW ints and is free again behind the next barrier.
__device__ __forceinline__ int before_thread(int x, int* ws, int& all) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int inc = wave_sums(x);
  if (lane == 63) ws[w] = inc;
  __syncthreads();
  const int sums = wave_sums(lane < KEEP_NW ? ws[lane] : 0);
  all = __builtin_amdgcn_readlane(sums, 63);
  return inc - x + (w ? __builtin_amdgcn_readlane(sums, w - 1) : 0);
}

// Kept keys of one (sequence, head), ascending: the first ones, the most recent ones, and of those between them the ``room`` largest, ties to
// the lowest index. Radix select: counts of 11 bits each narrow the threshold down (masses of one size share their leading byte: of 8 bits each
// many threads would wait at one counter) until its equals are as many as are wanted, then the keys are numbered in order. A thread
// holds PER neighbouring keys; of sequences that fit no such kernel (REG false) they are read again, KEEP_NT * PER at a time. Waiting bounds
// it, for barriers and for instructions that nobody has fetched yet: 2500 keys of 8 heads take 5.9 us with 4 keys a thread and 10.2 with
// 16, most of them not there; 16 sequences of 8000 keys 12 us.
template <int PER, bool REG>
__global__ __launch_bounds__(KEEP_NT) void evict_keep_kernel(const float* __restrict__ mass, int64_t ms, int64_t mh, int N,
                                                             const int* __restrict__ lens, int budget, int first, int recent,
                                                             int* __restrict__ kept, int Hkv) {
  constexpr int CHUNK = KEEP_NT * PER;
  __shared__ int hist[2048];
  __shared__ int s_digit, s_above, s_count;
  __shared__ int ws[4][KEEP_NW];
  const int h = blockIdx.x, r = blockIdx.y, tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const float* m = mass + r * ms + h * mh;
  int* out = kept + ((int64_t)r * Hkv + h) * budget;
  const int n = min(max(lens[r], 0), N);
  if (n <= budget) {
    for (int i = tid; i < budget; i += KEEP_NT) out[i] = i < n ? i : -1;
    return;
  }
  const int a = first, b = n - recent, room = budget - first - recent;   // (b - a = n - budget + room > room)
  uint32_t key[PER];
  auto load = [&](int i0) {
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      const int i = i0 + tid * PER + k;
      key[k] = i >= a && i < b ? rank_of(m[i]) : 0u;
    }
  };
  if (REG) load(0);
  // two counters a thread, from the largest digit down
  const int d0 = 2047 - 2 * tid;
  hist[d0] = hist[d0 - 1] = 0;
  __syncthreads();
  uint32_t lead = 0, known = 0;
  int need = room;                                                       // of those with the leading digits of the threshold
  for (int turn = 0; turn < 3 && need > 0; ++turn) {
    const int shift = 21 - 11 * turn, left = max(0, -shift);             // (the last digit: 10 bits)
    auto digit = [&](uint32_t x) { return (left ? x << left : x >> shift) & 2047; };
    for (int i0 = 0; i0 < (REG ? 1 : n); i0 += CHUNK) {
      if (!REG) load(i0);
#pragma unroll
      for (int k = 0; k < PER; ++k) {
        const int i = i0 + tid * PER + k;
        if (i >= a && i < b && (key[k] & known) == lead) atomicAdd(&hist[digit(key[k])], 1);
      }
    }
    __syncthreads();
    const int c0 = hist[d0], c1 = hist[d0 - 1];
    hist[d0] = hist[d0 - 1] = 0;                                         // for the next turn
    int all;
    const int before = before_thread(c0 + c1, ws[turn & 1], all);
    if (before < need && before + c0 + c1 >= need) {
      const bool first_of = before + c0 >= need;
      s_digit = first_of ? d0 : d0 - 1;
      s_above = first_of ? before : before + c0;
      s_count = first_of ? c0 : c1;
    }
    __syncthreads();
    lead |= left ? (uint32_t)s_digit >> left : (uint32_t)s_digit << shift;
    known |= left ? 2047u >> left : 2047u << shift;
    need -= s_above;
    if (s_count == need) break;
  }
  // ``lead`` is the threshold in its ``known`` bits: all above it stay, and the first ``need`` of its equals (room 0: nothing between the ends)
  int ties = 0, done = 0;                                                // in front of this chunk
  for (int i0 = 0; i0 < n; i0 += CHUNK) {
    if (!REG) load(i0);
    int mine = 0, all;
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      const int i = i0 + tid * PER + k;
      mine += room > 0 && i >= a && i < b && (key[k] & known) == lead;
    }
    int rank = ties + before_thread(mine, ws[2], all);
    ties += all;
    uint32_t keep = 0;
    int count = 0;
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      const int i = i0 + tid * PER + k;
      if (i >= n) continue;
      const bool mid = i >= a && i < b;
      bool yes = !mid;
      if (mid && room > 0) {
        const uint32_t x = key[k] & known;
        yes = x > lead || (x == lead && rank < need);
        rank += x == lead;
      }
      keep |= (uint32_t)yes << k;
      count += yes;
    }
    int at = done + before_thread(count, ws[3], all);
    done += all;
#pragma unroll
    for (int k = 0; k < PER; ++k)
      if ((keep >> k) & 1) {
        if (at < budget) out[at] = i0 + tid * PER + k;
        ++at;
      }
  }
}

// Kept keys, values and masses into new pages, a wave for a new page of a head. K goes by
// 16-byte pieces, V by the words of its keys. Keys outside of their table or cache leave their place in the new page as it was.
// Cache lines bound it: half of the keys kept, nearly every line of the old pages is read. 4096 of 8000 keys, 16 sequences, 8 heads of 128: 52 us,
// 142 MB kept and written, 213 MB with the lines' other halves (4.1 TB/s). Four pages a wave take 55, and one short sequence 6.4 us for 4.2.
template <int D>
__global__ __launch_bounds__(256) void evict_copy_kernel(uint8_t* __restrict__ kc, uint8_t* __restrict__ vc, int64_t n_pages,
                                                         const int* __restrict__ tables, int tw, int64_t ts, const int* __restrict__ kept,
                                                         int budget, const int* __restrict__ new_tables, int nw, int64_t ns, int Hkv,
                                                         const float* __restrict__ mass, int64_t ms, int64_t mh, int N,
                                                         float* __restrict__ new_mass) {
  constexpr int U = D / 8, KP = D / 32, BYTES = Page<D>::BYTES, DATA = Page<D>::DATA;   // words of a key; 16-byte pieces of it
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int h = blockIdx.y, r = blockIdx.z, pg = blockIdx.x * 4 + w, i0 = pg * PAGE;
  if (i0 >= budget) return;
  const int64_t row = ((int64_t)r * Hkv + h) * budget;
  const int np = pg < nw ? new_tables[r * ns + pg] : -1;
  const bool page = np >= 0 && np < n_pages;
  const int64_t to = ((int64_t)(page ? np : 0) * Hkv + h) * BYTES;
  // lane = key: where it is (-1: nowhere), in pages and heads
  const bool mine = lane < PAGE && i0 + lane < budget;
  const int src = mine ? kept[row + i0 + lane] : -1;
  int64_t from = -1;
  if (page && src >= 0 && (src >> 4) < tw) {
    const int p = tables[r * ts + (src >> 4)];
    if (p >= 0 && p < n_pages) from = (int64_t)p * Hkv + h;
  }
  const int so = src & 15, o = lane & 15;
  if (new_mass && mine) new_mass[row + i0 + lane] = src >= 0 && src < N ? mass[r * ms + h * mh + src] : 0.f;
  auto of = [&](int l) {
    return (int64_t)(uint32_t)__shfl((int)(uint32_t)from, l, 64) | (int64_t)__shfl((int)(from >> 32), l, 64) << 32;
  };
  const int kk = lane / KP, kp = lane % KP, c = lane / U, p = lane % U;
  u32x4 k, v;
  int there = 0;
  {                                             // K: lane = (key, piece)
    const int l = kk & 15, s = __shfl(so, l, 64);
    const int64_t f = of(l);
    if (kk < 16 && f >= 0) {
      k = *reinterpret_cast<const u32x4*>(kc + f * BYTES + s * (D / 2) + kp * 16);
      there = 16;
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {                 // V: lane = (four keys, eight elements)
    const int l = (4 * c + i) & 15, s = __shfl(so, l, 64);
    const int64_t f = of(l);
    if (c < 4 && f >= 0) {
      v[i] = *reinterpret_cast<const uint32_t*>(vc + f * BYTES + ((s >> 2) * U + p) * 16 + (s & 3) * 4);
      there |= 1 << i;
    }
  }
  if (there & 16) *reinterpret_cast<u32x4*>(kc + to + kk * (D / 2) + kp * 16) = k;
  uint8_t* vd = vc + to + (c * U + p) * 16;
  if ((there & 15) == 15) *reinterpret_cast<u32x4*>(vd) = v;
  else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if ((there >> i) & 1) *reinterpret_cast<uint32_t*>(vd + 4 * i) = v[i];
  }
  if (from >= 0) {                              // scales: lane = key
    const uint8_t *kf = kc + from * BYTES + DATA, *vf = vc + from * BYTES + DATA;
    uint8_t *kd = kc + to + DATA, *vd = vc + to + DATA;
    if constexpr (D == 128) *reinterpret_cast<uint32_t*>(kd + o * 4) = *reinterpret_cast<const uint32_t*>(kf + so * 4);
    else *reinterpret_cast<uint16_t*>(kd + o * 2) = *reinterpret_cast<const uint16_t*>(kf + so * 2);
    uint8_t vs[KP];
#pragma unroll
    for (int g = 0; g < KP; ++g) vs[g] = vf[g * 16 + so];
#pragma unroll
    for (int g = 0; g < KP; ++g) vd[g * 16 + o] = vs[g];
  }
}

}  // namespace kv4

using namespace kv4;

extern "C" hipError_t kafka_kv4_rope_write(const bf16* qkv, const float* qp, int S, int64_t ps, int64_t qkv_stride, const int64_t* positions,
                                           const float* cos_sin, int64_t n_pos, bf16* q_out, int64_t q_stride, uint8_t* kc, uint8_t* vc,
                                           const int64_t* slots, int64_t n_slots, int T, int Hq, int Hkv, int D, hipStream_t st) {
  if (T == 0) return hipSuccess;
  const int64_t total = (int64_t)T * ((Hq + Hkv) * (D / 16) + Hkv * (D / 8));
  if (n_pos < 1 || (D != 64 && D != 128) || total > 0xffffff00ll) return hipErrorInvalidValue;
  auto go = [&](auto kern) {
    kern<<<(unsigned)((total + 255) / 256), 256, 0, st>>>(qkv, qp, S, ps, qkv_stride, positions, cos_sin, n_pos, q_out, q_stride, kc, vc, slots,
                                                          n_slots, total, Hq, Hkv);
    return hipGetLastError();
  };
  return D == 64 ? go(rope_write_kernel<64>) : go(rope_write_kernel<128>);
}

extern "C" hipError_t kafka_kv4_read(const uint8_t* kc, const uint8_t* vc, const int64_t* slots, int64_t n_slots, int64_t T, int Hkv, int D,
                                     bf16* k, bf16* v, hipStream_t st) {
  if (T == 0) return hipSuccess;
  const int64_t total = T * Hkv * (D / 8);
  if ((D != 64 && D != 128) || total > 0xffffff00ll) return hipErrorInvalidValue;
  auto go = [&](auto kern) {
    kern<<<(unsigned)((total + 255) / 256), 256, 0, st>>>(kc, vc, slots, n_slots, total, Hkv, k, v);
    return hipGetLastError();
  };
  return D == 64 ? go(read_kernel<64>) : go(read_kernel<128>);
}

extern "C" hipError_t kafka_kv4_evict_keep(const float* mass, int64_t ms, int64_t mh, int N, const int* lens, int R, int Hkv, int budget,
                                           int first, int recent, int* kept, hipStream_t st) {
  if (R == 0 || Hkv == 0 || budget == 0) return hipSuccess;
  if (first < 0 || recent < 0 || (int64_t)first + recent > budget || R > 65535) return hipErrorInvalidValue;
  auto go = [&](auto kern) { kern<<<dim3(Hkv, R), KEEP_NT, 0, st>>>(mass, ms, mh, N, lens, budget, first, recent, kept, Hkv); };
  // (16 sequences of 5000 / 8300 / 12000 keys, as few a thread as hold them, 9 / 12 / 14 us, 8300 with 16 a thread 18; read again, 4 a thread at a
  // time, 12 / 16 / 19. One of 30000 keys, which no kernel holds, 4 a thread at a time 40, 16 at a time 49. With 12 and 16 a thread 18 and 51 scalar
  // registers go through lanes: in the times above)
  if (N <= KEEP_NT * 4) go(evict_keep_kernel<4, true>);
  else if (N <= KEEP_NT * 8) go(evict_keep_kernel<8, true>);
  else if (N <= KEEP_NT * 12) go(evict_keep_kernel<12, true>);
  else if (N <= KEEP_NT * 16) go(evict_keep_kernel<16, true>);
  else go(evict_keep_kernel<4, false>);
  return hipGetLastError();
}

extern "C" hipError_t kafka_kv4_evict_copy(uint8_t* kc, uint8_t* vc, int64_t n_pages, const int* tables, int tw, int64_t ts,
                                           const int* kept, int R, int Hkv, int budget, const int* new_tables, int nw, int64_t ns,
                                           const float* mass, int64_t ms, int64_t mh, int N, float* new_mass, int D, hipStream_t st) {
  if (R == 0 || budget == 0) return hipSuccess;
  if ((D != 64 && D != 128) || R > 65535 || Hkv > 65535) return hipErrorInvalidValue;
  auto go = [&](auto kern) {
    kern<<<dim3((budget + 63) / 64, Hkv, R), 256, 0, st>>>(kc, vc, n_pages, tables, tw, ts, kept, budget, new_tables, nw, ns, Hkv, mass, ms,
                                                           mh, N, new_mass);
    return hipGetLastError();
  };
  return D == 64 ? go(evict_copy_kernel<64>) : go(evict_copy_kernel<128>);
}

}  // namespace kafka
