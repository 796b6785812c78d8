// Python bindings of the 4-bit cache's kernels (kv4.hip, kv4_attn.hip, kv4_tile.hip). What the kernels assume of shapes, types, strides, alignment
// and devices is checked here; index values on the device (slots, page ids, kept keys) are checked by the kernels.
#include <torch/extension.h>
#include <ATen/MemoryOverlap.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <hip/hip_runtime.h>

extern "C" {
hipError_t kafka_kv4_rope_write(const void* qkv, const float* qp, int S, int64_t ps, int64_t qkv_stride, const int64_t* positions,
                                const float* cos_sin, int64_t n_pos, void* q_out, int64_t q_stride, uint8_t* kc, uint8_t* vc, const int64_t* slots,
                                int64_t n_slots, int T, int Hq, int Hkv, int D, hipStream_t st);
hipError_t kafka_kv4_read(const uint8_t* kc, const uint8_t* vc, const int64_t* slots, int64_t n_slots, int64_t T, int Hkv, int D, void* k,
                          void* v, hipStream_t st);
hipError_t kafka_kv4_evict_keep(const float* mass, int64_t ms, int64_t mh, int N, const int* lens, int R, int Hkv, int budget, int first,
                                int recent, int* kept, hipStream_t st);
hipError_t kafka_kv4_evict_copy(uint8_t* kc, uint8_t* vc, int64_t n_pages, const int* tables, int tw, int64_t ts, const int* kept, int R,
                                int Hkv, int budget, const int* new_tables, int nw, int64_t ns, const float* mass, int64_t ms, int64_t mh,
                                int N, float* new_mass, int D, hipStream_t st);
hipError_t kafka_kv4_attn(const void* q, int64_t qs, const uint8_t* kc, const uint8_t* vc, int64_t n_pages, const int* tables, int64_t ts,
                          const int* items, int n_items, int nq, int nw, int T, int Hkv, int G, int D, int window, int first, float scale, void* out,
                          int64_t os, float* lse, float* part, float* plse, int* counters, const int* wtiles, int n_wtiles, char* ws, hipStream_t st);
hipError_t kafka_kv4_tiles(const void* q, int64_t qs, const uint8_t* kc, const uint8_t* vc, int64_t n_pages, const int* tables, int64_t ts,
                           int rows, const int* items, int n_items, const int* wtiles, int n_wtiles, const int* merges, int n_merges, int T, int Hkv,
                           int G, int D, int window, int first, float scale, void* out, int64_t os, float* lse, float* part, float* plse,
                           char* ws, hipStream_t st);
hipError_t kafka_kv4_mass(const void* q, int64_t qs, const float* lse, const uint8_t* kc, int64_t n_pages, const int* tables, int64_t ts,
                          const int* few, int n_few, const int* many, int n_many, int T, int Hkv, int G, int D, int window, int first,
                          float scale, const float* base, float* out, int N, float* part, int* counters, hipStream_t st);
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
  TORCH_CHECK_VALUE(t.is_cuda() && t.device() == home.device(), name, ": on the cache's device expected");
  TORCH_CHECK_VALUE(t.scalar_type() == type, name, ": wrong dtype");
}

// workgroups read what others may have written by then, unless both are the same memory, which each reads and writes for itself
void apart(const Tensor& out, const Tensor& in, const char* what) {
  TORCH_CHECK_VALUE(at::get_overlap_status(out, in) != at::MemOverlapStatus::Partial, what);
}

// head dim of a K / V page pool
int cache(const Tensor& c, const char* name) {
  TORCH_CHECK_VALUE(c.is_cuda() && c.scalar_type() == at::kByte && c.dim() == 4 && c.size(2) == 16 && c.is_contiguous() && aligned(c) &&
                        (c.size(3) == 68 || c.size(3) == 34) && c.size(1) > 0 && c.size(1) < 1 << 12 && c.size(0) > 0 && c.size(0) < 1ll << 27,
                    name, ": a cache of kv_cache_shapes(..., \"mx4\") with head dim 64 or 128 expected");
  return c.size(3) == 68 ? 128 : 64;
}
int caches(const Tensor& k, const Tensor& v) {
  const int D = cache(k, "k_cache");
  TORCH_CHECK_VALUE(cache(v, "v_cache") == D && v.sizes() == k.sizes() && v.device() == k.device(), "k_cache and v_cache differ");
  return D;
}

// rows [T, heads, D] in bf16 whose 16-byte pieces are whole
void rows3(const Tensor& t, const Tensor& home, int64_t T, int64_t heads, int D, const char* name) {
  on(t, home, at::kBFloat16, name);
  TORCH_CHECK_VALUE(t.dim() == 3 && t.size(0) == T && t.size(1) == heads && t.size(2) == D, name, ": shape");
  TORCH_CHECK_VALUE(t.stride(2) == 1 && (t.stride(1) == D || heads == 1) && (T < 2 || (t.stride(0) % 8 == 0 && t.stride(0) >= heads * D)) &&
                        aligned(t), name, ": rows of whole heads, 16-byte aligned, expected");
}
const int* table(const Tensor& t, const Tensor& home, const char* name) {
  on(t, home, at::kInt, name);
  TORCH_CHECK_VALUE(t.dim() == 2 && (t.size(1) < 2 || t.stride(1) == 1) && t.size(1) < 1 << 27, name, ": int32 [rows, pages] expected");
  return t.data_ptr<int>();
}

void rope_write(Tensor qkv, Tensor positions, Tensor cos_sin, Tensor q_out, Tensor kc, Tensor vc, OptT slots, int64_t Hq, int64_t Hkv) {
  const int D = caches(kc, vc);
  const c10::DeviceGuard guard(kc.device());
  const bool slab = qkv.scalar_type() == at::kFloat;
  on(qkv, kc, slab ? at::kFloat : at::kBFloat16, "qkv");
  TORCH_CHECK_VALUE(Hkv == kc.size(1) && Hq > 0 && Hq < 1 << 12, "rope_kv_write: heads");
  const int64_t W = (Hq + 2 * Hkv) * D, T = qkv.dim() < 2 ? -1 : qkv.size(qkv.dim() - 2);
  TORCH_CHECK_VALUE(qkv.dim() == (slab ? 3 : 2) && qkv.size(-1) == W && T < 1 << 30 && aligned(qkv) &&
                  (slab ? qkv.is_contiguous() : qkv.stride(1) == 1 && (T < 2 || qkv.stride(0) % 8 == 0)),
              "rope_kv_write: qkv bf16 [T, (Hq + 2 Hkv) D] or contiguous fp32 slabs of it");
  on(positions, kc, at::kLong, "positions");
  on(cos_sin, kc, at::kFloat, "cos_sin");
  TORCH_CHECK_VALUE(positions.is_contiguous() && positions.numel() == T && cos_sin.is_contiguous() && cos_sin.dim() == 2 && cos_sin.size(1) == D &&
                  (T == 0 || cos_sin.size(0) > 0),
              "rope_kv_write: positions [T], cos_sin [positions, D]");
  rows3(q_out, kc, T, Hq, D, "q_out");
  const int64_t* sp = nullptr;
  if (slots.has_value()) {
    on(*slots, kc, at::kLong, "slot_mapping");
    TORCH_CHECK_VALUE(slots->is_contiguous() && slots->numel() == T, "slot_mapping: int64 [T]");
    sp = slots->data_ptr<int64_t>();
  }
  KV4_HIP(kafka_kv4_rope_write(slab ? nullptr : qkv.data_ptr(), slab ? qkv.data_ptr<float>() : nullptr, slab ? (int)qkv.size(0) : 0,
                               slab ? T * W : 0, slab ? W : qkv.stride(0), positions.data_ptr<int64_t>(), cos_sin.data_ptr<float>(), cos_sin.size(0),
                               q_out.data_ptr(), q_out.stride(0), kc.data_ptr<uint8_t>(), vc.data_ptr<uint8_t>(), sp, kc.size(0) * 16,
                               (int)T, (int)Hq, (int)Hkv, D, stream()));
}

std::tuple<Tensor, Tensor> read_slots(Tensor kc, Tensor vc, Tensor slots) {
  const int D = caches(kc, vc);
  const c10::DeviceGuard guard(kc.device());
  on(slots, kc, at::kLong, "slots");
  const int64_t T = slots.numel(), H = kc.size(1);
  TORCH_CHECK_VALUE(slots.dim() == 1, "slots: int64 [T]");
  slots = slots.contiguous();
  const auto opt = kc.options().dtype(at::kBFloat16);
  Tensor k = at::empty({T, H, D}, opt), v = at::empty({T, H, D}, opt);
  KV4_HIP(kafka_kv4_read(kc.data_ptr<uint8_t>(), vc.data_ptr<uint8_t>(), slots.data_ptr<int64_t>(), kc.size(0) * 16, T, (int)H, D,
                         k.data_ptr(), v.data_ptr(), stream()));
  return {k, v};
}

// a step's work, made by the host for all its layers (kv4.py): tables on the device and what is known of them
struct Part {
  int64_t rows, waves, slots;     // of a tile; of its workgroup; partial results
  Tensor items, merges, keys;     // keys: tiles to widen first, none: the kernels widen as they go
};
struct Plan {
  int64_t heads, kv_heads, dim, window, first, rows, covered, keys, tables;
  int64_t segments = 0, mass_slots = 0;
  std::vector<Part> parts;
  OptT few, many;                 // items of attn_mass

  // Counters of split tiles, which every launch leaves zero: one set for each stream that the plan is used on. A captured call has a set of its
  // own, cleared in its graph, since the graph may be replayed beside anything.
  mutable std::vector<std::pair<hipStream_t, Tensor>> counters;
  int* zeros(int64_t n, Tensor& held) const {
    const auto opt = (parts.empty() ? *many : parts[0].items).options();
    hipStreamCaptureStatus status;
    KV4_HIP(hipStreamIsCapturing(stream(), &status));
    if (status != hipStreamCaptureStatusNone) {
      held = at::zeros({n}, opt);
      return held.data_ptr<int>();
    }
    for (auto& c : counters)
      if (c.first == stream() && c.second.numel() >= n) return c.second.data_ptr<int>();
    counters.emplace_back(stream(), at::zeros({n}, opt));
    return counters.back().second.data_ptr<int>();
  }

  void add(int64_t r, int64_t w, int64_t slots, Tensor items, Tensor merges, Tensor keys) {
    auto ok = [&](const Tensor& t, int64_t cols) {
      return t.is_cuda() && t.scalar_type() == at::kInt && t.dim() == 2 && t.size(1) == cols && t.is_contiguous() && t.size(0) < 1 << 24;
    };
    const bool wide = keys.numel() > 0;
    TORCH_CHECK_VALUE(ok(items, wide ? 12 : 8) && ok(merges, 4) && ok(keys, 4) && r > 0 && r <= 256 && slots >= 0 && slots < 1 << 24, "kv4: plan");
    parts.push_back({r, w, slots, items, merges, keys});
  }
  void weigh(Tensor f, Tensor m, int64_t slots, int64_t n) {
    auto ok = [&](const Tensor& t, int64_t cols) {
      return t.is_cuda() && t.scalar_type() == at::kInt && t.dim() == 2 && t.size(1) == cols && t.is_contiguous() && t.size(0) < 1 << 24;
    };
    TORCH_CHECK_VALUE(ok(f, 8) && ok(m, 12) && f.device() == m.device() && slots >= 0 && slots < 1 << 24, "kv4: plan");
    few = f;
    many = m;
    mass_slots = slots;
    segments = n;
  }
};

// q and the block tables of a call against its plan
const int* call(const Plan& p, const Tensor& q, const Tensor& kc, int D, const Tensor& tables, double scale) {
  TORCH_CHECK_VALUE(scale >= 1e-30 && scale <= 1e30, "kv4: a positive scale expected");   // (masked scores are -infinity times it)
  TORCH_CHECK_VALUE(q.dim() == 3 && q.size(1) == p.heads && D == p.dim && kc.size(1) == p.kv_heads,
                    "kv4: q bf16 [T, heads, dim] and a cache of the plan's heads expected");
  rows3(q, kc, q.size(0), p.heads, D, "q");
  TORCH_CHECK_VALUE(q.size(0) >= p.rows && q.size(0) < 1 << 26, "kv4: the plan has ", p.rows, " rows, q ", q.size(0));
  const int* tp = table(tables, kc, "block_tables");
  TORCH_CHECK_VALUE(tables.size(0) >= p.tables && tables.size(1) * 16 >= p.keys, "kv4: int32 block tables of ", p.tables, " rows for ", p.keys,
                    " keys expected");
  return tp;
}
float* row_values(const OptT& t, const Tensor& q, const Tensor& home) {
  if (!t.has_value()) return nullptr;
  on(*t, home, at::kFloat, "lse");
  TORCH_CHECK_VALUE(t->is_contiguous() && t->dim() == 2 && t->size(0) == q.size(0) && t->size(1) == q.size(1), "lse: fp32 [T, heads]");
  return t->data_ptr<float>();
}

Tensor attn(Tensor q, Tensor kc, Tensor vc, Tensor tables, const Plan& p, double scale, OptT out_, OptT lse) {
  const int D = caches(kc, vc);
  const c10::DeviceGuard guard(kc.device());
  const int* tp = call(p, q, kc, D, tables, scale);
  const int64_t T = q.size(0), Hq = p.heads, H = p.kv_heads;
  Tensor out;
  if (out_.has_value()) {
    out = *out_;
    rows3(out, kc, T, Hq, D, "out");
    apart(out, q, "attn: out and q overlap in part");
  } else {
    out = p.covered == T ? at::empty({T, Hq, D}, q.options()) : at::zeros({T, Hq, D}, q.options());
  }
  float* lp = row_values(lse, q, kc);
  // keys of long portions are widened beside the last launch of four waves before them, where there is one
  const Part *wide = nullptr, *beside = nullptr;
  for (const Part& t : p.parts) {
    TORCH_CHECK_VALUE(t.items.device() == kc.device(), "kv4: the plan was made for another device");
    if (t.keys.size(0) > 0) wide = &t;
    else if (!wide && t.waves == 4 && t.items.size(0) > 0) beside = &t;
  }
  Tensor ws;                        // (the caching allocator orders it with the stream)
  if (wide) ws = at::empty({wide->keys.size(0) * H * 256 * D}, kc.options());
  char* wp = wide ? reinterpret_cast<char*>(ws.data_ptr()) : nullptr;
  if (!wide) beside = nullptr;
  for (const Part& t : p.parts) {
    Tensor part, held;
    float *pp = nullptr, *pl = nullptr;
    if (t.slots > 0) {
      const int64_t n = t.slots * H * t.rows;
      part = at::empty({n * (D + 1)}, kc.options().dtype(at::kFloat));
      pp = part.data_ptr<float>();
      pl = pp + n * D;
    }
    const int *ip = t.items.data_ptr<int>(), *mp = t.merges.data_ptr<int>();
    const int ni = (int)t.items.size(0), nm = (int)t.merges.size(0);
    if (t.keys.size(0) == 0) {
      KV4_HIP(kafka_kv4_attn(q.data_ptr(), q.stride(0), kc.data_ptr<uint8_t>(), vc.data_ptr<uint8_t>(), kc.size(0), tp, tables.stride(0), ip, ni,
                             (int)(t.rows / 16), (int)t.waves, (int)T, (int)H, (int)(Hq / H), D, (int)p.window, (int)p.first, (float)scale,
                             out.data_ptr(), out.stride(0), lp, pp, pl, t.slots > 0 ? p.zeros(t.slots * H, held) : nullptr,
                             &t == beside ? wide->keys.data_ptr<int>() : nullptr, &t == beside ? (int)wide->keys.size(0) : 0, wp, stream()));
    } else {
      KV4_HIP(kafka_kv4_tiles(q.data_ptr(), q.stride(0), kc.data_ptr<uint8_t>(), vc.data_ptr<uint8_t>(), kc.size(0), tp, tables.stride(0),
                              (int)t.rows, ip, ni, t.keys.data_ptr<int>(), beside ? 0 : (int)t.keys.size(0), mp, nm, (int)T, (int)H, (int)(Hq / H), D,
                              (int)p.window, (int)p.first, (float)scale, out.data_ptr(), out.stride(0), lp, pp, pl,
                              wp, stream()));
    }
  }
  return out;
}

void masses(const Tensor& m, const Tensor& home, int64_t R, int64_t H, const char* name) {
  on(m, home, at::kFloat, name);
  TORCH_CHECK_VALUE(m.dim() == 3 && m.size(0) == R && m.size(1) == H && (m.size(2) < 2 || m.stride(2) == 1) && m.size(2) < 1 << 30, name,
                    ": fp32 [sequences, heads, keys] expected");
}

Tensor attn_mass(Tensor q, Tensor lse, Tensor kc, Tensor tables, const Plan& p, double scale, OptT base, OptT out_) {
  const int D = cache(kc, "k_cache");
  const c10::DeviceGuard guard(kc.device());
  const int* tp = call(p, q, kc, D, tables, scale);
  TORCH_CHECK_VALUE(p.few.has_value() && p.few->device() == kc.device(), "attn_mass: a plan of attn_plan for this device expected");
  TORCH_CHECK_VALUE(p.rows < 2 || q.stride(0) < 1 << 23, "attn_mass: q's rows less than 2^23 elements apart");
  const float* lp = row_values(lse, q, kc);
  const int64_t S = p.segments, H = p.kv_heads;
  int64_t N = p.keys;
  for (const OptT* t : {&base, &out_})
    if (t->has_value()) {
      masses(**t, kc, S, H, "base, out");
      N = (*t)->size(2);
      TORCH_CHECK_VALUE((*t)->is_contiguous() && N >= p.keys, "attn_mass: base and out contiguous, at least ", p.keys, " keys wide");
    }
  TORCH_CHECK_VALUE(!base.has_value() || !out_.has_value() || base->sizes() == out_->sizes(), "attn_mass: base and out alike");
  if (base.has_value() && out_.has_value()) apart(*out_, *base, "attn_mass: base and out overlap in part");
  Tensor out = out_.has_value() ? *out_ : at::empty({S, H, N}, lse.options());
  const int64_t done = (p.keys + 63) / 64 * 64;
  const bool same = base.has_value() && base->data_ptr() == out.data_ptr();
  if (N > done && !same) {           // (behind the plan's last block nothing is added)
    Tensor rest = out.narrow(2, done, N - done);
    if (base.has_value()) rest.copy_(base->narrow(2, done, N - done));
    else rest.zero_();
  }
  Tensor part, held;
  float* pp = nullptr;
  int* counters = nullptr;
  if (p.mass_slots > 0) {
    part = at::empty({p.mass_slots * H * 256}, lse.options());
    pp = part.data_ptr<float>();
    counters = p.zeros(p.mass_slots * H, held);
  }
  KV4_HIP(kafka_kv4_mass(q.data_ptr(), q.stride(0), lp, kc.data_ptr<uint8_t>(), kc.size(0), tp, tables.stride(0), p.few->data_ptr<int>(),
                         (int)p.few->size(0), p.many->data_ptr<int>(), (int)p.many->size(0), (int)q.size(0), (int)H, (int)(p.heads / H), D,
                         (int)p.window, (int)p.first, (float)scale, base.has_value() ? base->data_ptr<float>() : nullptr,
                         out.data_ptr<float>(), (int)N, pp, counters, stream()));
  return out;
}

Tensor evict_keep(Tensor mass, Tensor lens, int64_t budget, int64_t first, int64_t recent) {
  TORCH_CHECK_VALUE(mass.is_cuda() && mass.dim() == 3, "mass: fp32 [sequences, heads, keys] on a GPU expected");
  const c10::DeviceGuard guard(mass.device());
  const int64_t R = mass.size(0), H = mass.size(1);
  if (mass.size(2) > 1 && mass.stride(2) != 1) mass = mass.contiguous();
  masses(mass, mass, R, H, "mass");
  on(lens, mass, at::kInt, "lens");
  TORCH_CHECK_VALUE(lens.dim() == 1 && lens.numel() == R && R < 65536 && H < 65536, "evict_keep: lens int32 [sequences] expected");
  TORCH_CHECK_VALUE(budget >= 1 && budget < 1 << 26 && first >= 0 && recent >= 0 && first + recent <= budget,
                    "evict_keep: first and recent keys within a budget of at least one");
  lens = lens.contiguous();
  Tensor kept = at::empty({R, H, budget}, lens.options());
  KV4_HIP(kafka_kv4_evict_keep(mass.data_ptr<float>(), mass.stride(0), mass.stride(1), (int)mass.size(2), lens.data_ptr<int>(), (int)R,
                               (int)H, (int)budget, (int)first, (int)recent, kept.data_ptr<int>(), stream()));
  return kept;
}

OptT evict_copy(Tensor kc, Tensor vc, Tensor tables, Tensor kept, Tensor new_tables, OptT mass) {
  const int D = caches(kc, vc);
  const c10::DeviceGuard guard(kc.device());
  on(kept, kc, at::kInt, "kept");
  const int64_t R = kept.dim() == 3 ? kept.size(0) : -1, H = kc.size(1);
  TORCH_CHECK_VALUE(R >= 0 && kept.size(1) == H && R < 65536 && kept.size(2) < 1 << 26, "kept: int32 [sequences, heads, budget]");
  kept = kept.contiguous();
  const int *tp = table(tables, kc, "block_tables"), *np = table(new_tables, kc, "new_tables");
  TORCH_CHECK_VALUE(tables.size(0) == R && new_tables.size(0) == R, "evict: a table row for every sequence");
  const float* mp = nullptr;
  float* nm = nullptr;
  int64_t ms = 0, mh = 0, N = 0;
  OptT moved;
  if (mass.has_value()) {
    Tensor m = *mass;
    if (m.dim() == 3 && m.size(2) > 1 && m.stride(2) != 1) m = m.contiguous();
    masses(m, kc, R, H, "mass");
    moved = at::empty({R, H, kept.size(2)}, m.options());
    mp = m.data_ptr<float>();
    nm = moved->data_ptr<float>();
    ms = m.stride(0), mh = m.stride(1), N = m.size(2);
    mass = m;                       // (alive until the launch)
  }
  KV4_HIP(kafka_kv4_evict_copy(kc.data_ptr<uint8_t>(), vc.data_ptr<uint8_t>(), kc.size(0), tp, (int)tables.size(1), tables.stride(0),
                               kept.data_ptr<int>(), (int)R, (int)H, (int)kept.size(2), np, (int)new_tables.size(1), new_tables.stride(0),
                               mp, ms, mh, (int)N, nm, D, stream()));
  return moved;
}

}  // namespace

void kafka_bind_kv4(pybind11::module_& m) {
  namespace py = pybind11;
  py::class_<Plan>(m, "Kv4Plan")
      .def(py::init([](int64_t heads, int64_t kv_heads, int64_t dim, int64_t window, int64_t first, int64_t rows, int64_t covered, int64_t keys,
                       int64_t tables) {
        TORCH_CHECK_VALUE(kv_heads > 0 && heads % kv_heads == 0 && heads / kv_heads >= 1 && heads / kv_heads <= 16, "kv4: plan");
        return Plan{heads, kv_heads, dim, window, first, rows, covered, keys, tables};
      }))
      .def("add", &Plan::add)
      .def("weigh", &Plan::weigh);
  m.def("kv4_rope_write", &rope_write);
  m.def("kv4_read", &read_slots);
  m.def("kv4_attn", &attn);
  m.def("kv4_mass", &attn_mass);
  m.def("kv4_evict_keep", &evict_keep);
  m.def("kv4_evict_copy", &evict_copy);
}
