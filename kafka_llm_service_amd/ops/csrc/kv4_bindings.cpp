// Python bindings of the 4-bit cache's kernels (kv4.hip, kv4_attn.hip). What the kernels assume of shapes, types, strides, alignment
// and devices is checked here; index values on the device (slots, page ids, kept keys) are checked by the kernels.
#include <torch/extension.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <hip/hip_runtime.h>

extern "C" {
hipError_t kafka_kv4_rope_write(const void* qkv, const float* qp, int S, int64_t ps, int64_t qkv_stride, const int64_t* positions,
                                const float* cos_sin, void* q_out, int64_t q_stride, uint8_t* kc, uint8_t* vc, const int64_t* slots,
                                int64_t n_slots, int T, int Hq, int Hkv, int D, hipStream_t st);
hipError_t kafka_kv4_read(const uint8_t* kc, const uint8_t* vc, const int64_t* slots, int64_t n_slots, int64_t T, int Hkv, int D, void* k,
                          void* v, hipStream_t st);
hipError_t kafka_kv4_evict_keep(const float* mass, int64_t ms, int64_t mh, int N, const int* lens, int R, int Hkv, int budget, int first,
                                int recent, int* kept, hipStream_t st);
hipError_t kafka_kv4_evict_copy(uint8_t* kc, uint8_t* vc, int64_t n_pages, const int* tables, int tw, int64_t ts, const int* kept, int R,
                                int Hkv, int budget, const int* new_tables, int nw, int64_t ns, const float* mass, int64_t ms, int64_t mh,
                                int N, float* new_mass, int D, hipStream_t st);
hipError_t kafka_kv4_attn(const void* q, int64_t qs, const uint8_t* kc, const uint8_t* vc, int64_t n_pages, const int* tables, int64_t ts,
                          const int* items, int n_items, int nq, const int* merges, int n_merges, int T, int Hkv, int G, int D, int window,
                          int first, float scale, void* out, int64_t os, float* lse, float* part, float* plse, hipStream_t st);
hipError_t kafka_kv4_tiles(const void* q, int64_t qs, const uint8_t* kc, const uint8_t* vc, int64_t n_pages, const int* tables, int64_t ts,
                           const int* items, int n_items, const int* wtiles, int n_wtiles, const int* merges, int n_merges, int T, int Hkv,
                           int G, int D, int window, int first, float scale, void* out, int64_t os, float* lse, float* part, float* plse,
                           char* ws, hipStream_t st);
hipError_t kafka_kv4_mass(const void* q, int64_t qs, const float* lse, const uint8_t* kc, int64_t n_pages, const int* tables, int64_t ts,
                          const int* items, int n_whole, int n_split, int T, int Hkv, int G, int D, int window, int first, float scale,
                          const float* base, float* out, int N, hipStream_t st);
}

namespace {

using at::Tensor;
using OptT = c10::optional<Tensor>;

#define KV4_HIP(e)                                                                \
  do {                                                                            \
    hipError_t _e = (e);                                                          \
    TORCH_CHECK(_e == hipSuccess, "HIP launch failed: ", hipGetErrorString(_e));  \
  } while (0)

hipStream_t stream() { return c10::hip::getCurrentHIPStream().stream(); }
bool aligned(const Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0; }

void on(const Tensor& t, const Tensor& home, at::ScalarType type, const char* name) {
  TORCH_CHECK(t.is_cuda() && t.device() == home.device(), name, ": on the cache's device expected");
  TORCH_CHECK(t.scalar_type() == type, name, ": wrong dtype");
}

// head dim of a K / V page pool
int cache(const Tensor& c, const char* name) {
  TORCH_CHECK(c.is_cuda() && c.scalar_type() == at::kByte && c.dim() == 4 && c.size(2) == 16 && c.is_contiguous() && aligned(c) &&
                  (c.size(3) == 68 || c.size(3) == 34) && c.size(1) > 0 && c.size(1) < 1 << 12 && c.size(0) < 1ll << 27,
              name, ": uint8 pages [pages, heads, 16, 34 or 68] expected");
  return c.size(3) == 68 ? 128 : 64;
}
int caches(const Tensor& k, const Tensor& v) {
  const int D = cache(k, "k_cache");
  TORCH_CHECK(cache(v, "v_cache") == D && v.sizes() == k.sizes() && v.device() == k.device(), "k_cache and v_cache differ");
  return D;
}

// rows [T, heads, D] in bf16 whose 16-byte pieces are whole
void rows3(const Tensor& t, const Tensor& home, int64_t T, int64_t heads, int D, const char* name) {
  on(t, home, at::kBFloat16, name);
  TORCH_CHECK(t.dim() == 3 && t.size(0) == T && t.size(1) == heads && t.size(2) == D, name, ": shape");
  TORCH_CHECK(t.stride(2) == 1 && t.stride(1) == D && (T < 2 || (t.stride(0) % 8 == 0 && t.stride(0) >= heads * D)) && aligned(t), name,
              ": rows of whole heads, 16-byte aligned, expected");
}
const int* table(const Tensor& t, const Tensor& home, const char* name) {
  on(t, home, at::kInt, name);
  TORCH_CHECK(t.dim() == 2 && (t.size(1) < 2 || t.stride(1) == 1) && t.size(1) < 1 << 27, name, ": int32 [rows, pages] expected");
  return t.data_ptr<int>();
}

void rope_write(Tensor qkv, Tensor positions, Tensor cos_sin, Tensor q_out, Tensor kc, Tensor vc, OptT slots, int64_t Hq, int64_t Hkv) {
  const int D = caches(kc, vc);
  const c10::DeviceGuard guard(kc.device());
  const bool slab = qkv.scalar_type() == at::kFloat;
  on(qkv, kc, slab ? at::kFloat : at::kBFloat16, "qkv");
  TORCH_CHECK(Hkv == kc.size(1) && Hq > 0 && Hq < 1 << 12, "rope_kv_write: heads");
  const int64_t W = (Hq + 2 * Hkv) * D, T = qkv.dim() < 2 ? -1 : qkv.size(qkv.dim() - 2);
  TORCH_CHECK(qkv.dim() == (slab ? 3 : 2) && qkv.size(-1) == W && T < 1 << 30 && aligned(qkv) &&
                  (slab ? qkv.is_contiguous() : qkv.stride(1) == 1 && (T < 2 || qkv.stride(0) % 8 == 0)),
              "rope_kv_write: qkv bf16 [T, (Hq + 2 Hkv) D] or contiguous fp32 slabs of it");
  on(positions, kc, at::kLong, "positions");
  on(cos_sin, kc, at::kFloat, "cos_sin");
  TORCH_CHECK(positions.is_contiguous() && positions.numel() == T && cos_sin.is_contiguous() && cos_sin.dim() == 2 && cos_sin.size(1) == D,
              "rope_kv_write: positions [T], cos_sin [positions, D]");
  rows3(q_out, kc, T, Hq, D, "q_out");
  const int64_t* sp = nullptr;
  if (slots.has_value()) {
    on(*slots, kc, at::kLong, "slot_mapping");
    TORCH_CHECK(slots->is_contiguous() && slots->numel() == T, "slot_mapping: int64 [T]");
    sp = slots->data_ptr<int64_t>();
  }
  KV4_HIP(kafka_kv4_rope_write(slab ? nullptr : qkv.data_ptr(), slab ? qkv.data_ptr<float>() : nullptr, slab ? (int)qkv.size(0) : 0,
                               slab ? T * W : 0, slab ? W : qkv.stride(0), positions.data_ptr<int64_t>(), cos_sin.data_ptr<float>(),
                               q_out.data_ptr(), q_out.stride(0), kc.data_ptr<uint8_t>(), vc.data_ptr<uint8_t>(), sp, kc.size(0) * 16,
                               (int)T, (int)Hq, (int)Hkv, D, stream()));
}

void read_slots(Tensor kc, Tensor vc, Tensor slots, Tensor k, Tensor v) {
  const int D = caches(kc, vc);
  const c10::DeviceGuard guard(kc.device());
  on(slots, kc, at::kLong, "slots");
  const int64_t T = slots.numel(), H = kc.size(1);
  TORCH_CHECK(slots.dim() == 1 && slots.is_contiguous(), "slots: int64 [T]");
  rows3(k, kc, T, H, D, "k");
  rows3(v, kc, T, H, D, "v");
  TORCH_CHECK(k.is_contiguous() && v.is_contiguous(), "k, v: contiguous");
  KV4_HIP(kafka_kv4_read(kc.data_ptr<uint8_t>(), vc.data_ptr<uint8_t>(), slots.data_ptr<int64_t>(), kc.size(0) * 16, T, (int)H, D,
                         k.data_ptr(), v.data_ptr(), stream()));
}

void masses(const Tensor& m, const Tensor& home, int64_t R, int64_t H, const char* name) {
  on(m, home, at::kFloat, name);
  TORCH_CHECK(m.dim() == 3 && m.size(0) == R && m.size(1) == H && (m.size(2) < 2 || m.stride(2) == 1) && m.size(2) < 1 << 30, name,
              ": fp32 [sequences, heads, keys] expected");
}

void evict_keep(Tensor mass, Tensor lens, int64_t budget, int64_t first, int64_t recent, Tensor kept) {
  TORCH_CHECK(mass.is_cuda(), "mass: GPU tensor expected");
  const c10::DeviceGuard guard(mass.device());
  const int64_t R = mass.size(0), H = mass.size(1);
  masses(mass, mass, R, H, "mass");
  on(lens, mass, at::kInt, "lens");
  on(kept, mass, at::kInt, "kept");
  TORCH_CHECK(lens.is_contiguous() && lens.numel() == R && kept.is_contiguous() && kept.dim() == 3 && kept.size(0) == R &&
                  kept.size(1) == H && kept.size(2) == budget && R < 65536 && H < 65536 && budget < 1 << 30, "evict_keep: lens [R], kept [R, H, budget]");
  KV4_HIP(kafka_kv4_evict_keep(mass.data_ptr<float>(), mass.stride(0), mass.stride(1), (int)mass.size(2), lens.data_ptr<int>(), (int)R,
                               (int)H, (int)budget, (int)first, (int)recent, kept.data_ptr<int>(), stream()));
}

void evict_copy(Tensor kc, Tensor vc, Tensor tables, Tensor kept, Tensor new_tables, OptT mass, OptT new_mass) {
  const int D = caches(kc, vc);
  const c10::DeviceGuard guard(kc.device());
  const int64_t R = kept.size(0), H = kc.size(1);
  on(kept, kc, at::kInt, "kept");
  TORCH_CHECK(kept.dim() == 3 && kept.size(1) == H && kept.is_contiguous() && R < 65536 && kept.size(2) < 1 << 30, "kept: int32 [R, heads, budget]");
  const int *tp = table(tables, kc, "block_tables"), *np = table(new_tables, kc, "new_tables");
  TORCH_CHECK(tables.size(0) == R && new_tables.size(0) == R, "evict: a table row for every sequence");
  const float* mp = nullptr;
  float* nm = nullptr;
  int64_t ms = 0, mh = 0, N = 0;
  if (mass.has_value()) {
    masses(*mass, kc, R, H, "mass");
    on(*new_mass, kc, at::kFloat, "new_mass");
    TORCH_CHECK(new_mass->is_contiguous() && new_mass->sizes() == kept.sizes(), "new_mass: fp32 like kept");
    mp = mass->data_ptr<float>();
    nm = new_mass->data_ptr<float>();
    ms = mass->stride(0), mh = mass->stride(1), N = mass->size(2);
  }
  KV4_HIP(kafka_kv4_evict_copy(kc.data_ptr<uint8_t>(), vc.data_ptr<uint8_t>(), kc.size(0), tp, (int)tables.size(1), tables.stride(0),
                               kept.data_ptr<int>(), (int)R, (int)H, (int)kept.size(2), np, (int)new_tables.size(1), new_tables.stride(0),
                               mp, ms, mh, (int)N, nm, D, stream()));
}

const int* ints(const Tensor& t, const Tensor& home, int64_t cols, const char* name) {
  on(t, home, at::kInt, name);
  TORCH_CHECK(t.dim() == 2 && t.size(1) == cols && t.is_contiguous() && t.size(0) < 1 << 24, name, ": plan");
  return t.data_ptr<int>();
}

// ``rows`` of a tile; ``wtiles``, ``ws``: what of the cache is widened first, and where to
void attn(Tensor q, Tensor kc, Tensor vc, Tensor tables, int64_t rows, Tensor items, Tensor merges, int64_t window, int64_t first, double scale,
          Tensor out, OptT lse, OptT part, OptT plse, int64_t slots, OptT wtiles, OptT ws) {
  const int D = caches(kc, vc);
  const c10::DeviceGuard guard(kc.device());
  const int64_t T = q.size(0), Hq = q.dim() == 3 ? q.size(1) : 0, H = kc.size(1);
  rows3(q, kc, T, Hq, D, "q");
  rows3(out, kc, T, Hq, D, "out");
  TORCH_CHECK(Hq > 0 && Hq % H == 0 && Hq / H <= 16 && T < 1 << 26, "attn: 1 to 16 query heads for each key/value head");
  const int* tp = table(tables, kc, "block_tables");
  const int *ip = ints(items, kc, wtiles.has_value() ? 12 : 8, "items"), *mp = ints(merges, kc, 4, "merges");
  float *lp = nullptr, *pp = nullptr, *pl = nullptr;
  if (lse.has_value()) {
    on(*lse, kc, at::kFloat, "lse");
    TORCH_CHECK(lse->is_contiguous() && lse->dim() == 2 && lse->size(0) == T && lse->size(1) == Hq, "lse: fp32 [T, Hq]");
    lp = lse->data_ptr<float>();
  }
  if (slots > 0) {
    TORCH_CHECK(part.has_value() && plse.has_value(), "attn: split tiles need their workspace");
    on(*part, kc, at::kFloat, "part");
    on(*plse, kc, at::kFloat, "plse");
    TORCH_CHECK(part->is_contiguous() && plse->is_contiguous() && aligned(*part) && plse->numel() >= slots * H * rows &&
                    part->numel() >= slots * H * rows * D, "attn: workspace");
    pp = part->data_ptr<float>();
    pl = plse->data_ptr<float>();
  }
  if (!wtiles.has_value()) {
    KV4_HIP(kafka_kv4_attn(q.data_ptr(), q.stride(0), kc.data_ptr<uint8_t>(), vc.data_ptr<uint8_t>(), kc.size(0), tp, tables.stride(0), ip,
                           (int)items.size(0), (int)(rows / 16), mp, (int)merges.size(0), (int)T, (int)H, (int)(Hq / H), D, (int)window,
                           (int)first, (float)scale, out.data_ptr(), out.stride(0), lp, pp, pl, stream()));
    return;
  }
  const int* wp = ints(*wtiles, kc, 4, "wtiles");
  on(*ws, kc, at::kByte, "ws");
  TORCH_CHECK(rows == 256 && ws->is_contiguous() && aligned(*ws) && ws->numel() >= wtiles->size(0) * H * 256 * D, "attn: workspace");
  KV4_HIP(kafka_kv4_tiles(q.data_ptr(), q.stride(0), kc.data_ptr<uint8_t>(), vc.data_ptr<uint8_t>(), kc.size(0), tp, tables.stride(0), ip,
                          (int)items.size(0), wp, (int)wtiles->size(0), mp, (int)merges.size(0), (int)T, (int)H, (int)(Hq / H), D,
                          (int)window, (int)first, (float)scale, out.data_ptr(), out.stride(0), lp, pp, pl,
                          reinterpret_cast<char*>(ws->data_ptr()), stream()));
}

void mass(Tensor q, Tensor lse, Tensor kc, Tensor tables, Tensor items, int64_t n_whole, int64_t window, int64_t first, double scale, OptT base,
          Tensor out, int64_t segments) {
  const int D = cache(kc, "k_cache");
  const c10::DeviceGuard guard(kc.device());
  const int64_t T = q.size(0), Hq = q.dim() == 3 ? q.size(1) : 0, H = kc.size(1);
  rows3(q, kc, T, Hq, D, "q");
  TORCH_CHECK(Hq > 0 && Hq % H == 0 && Hq / H <= 16 && T < 1 << 26, "attn_mass: 1 to 16 query heads for each key/value head");
  on(lse, kc, at::kFloat, "lse");
  TORCH_CHECK(lse.is_contiguous() && lse.dim() == 2 && lse.size(0) == T && lse.size(1) == Hq, "lse: fp32 [T, Hq]");
  const int* tp = table(tables, kc, "block_tables");
  const int* ip = ints(items, kc, 8, "items");
  masses(out, kc, segments, H, "out");
  TORCH_CHECK(out.is_contiguous() && n_whole >= 0 && n_whole <= items.size(0), "attn_mass: out contiguous");
  const float* bp = nullptr;
  if (base.has_value()) {
    masses(*base, kc, segments, H, "base");
    TORCH_CHECK(base->is_contiguous() && base->size(2) == out.size(2), "base: like out");
    bp = base->data_ptr<float>();
  }
  KV4_HIP(kafka_kv4_mass(q.data_ptr(), q.stride(0), lse.data_ptr<float>(), kc.data_ptr<uint8_t>(), kc.size(0), tp, tables.stride(0), ip,
                         (int)n_whole, (int)(items.size(0) - n_whole), (int)T, (int)H, (int)(Hq / H), D, (int)window, (int)first,
                         (float)scale, bp, out.data_ptr<float>(), (int)out.size(2), stream()));
}

}  // namespace

void kafka_bind_kv4(pybind11::module_& m) {
  m.def("kv4_rope_write", &rope_write);
  m.def("kv4_read", &read_slots);
  m.def("kv4_evict_keep", &evict_keep);
  m.def("kv4_evict_copy", &evict_copy);
  m.def("kv4_attn", &attn);
  m.def("kv4_mass", &mass);
}
