// Checks and marshalling of the engine's operators that a program calls for single tokens (include/omniserve_lm.h: rotary positions, the quantised cache,
// drafted tokens): a call's dozen tensors are looked over, its result and scratch allocated and the entry point called in 3 - 5 us, where the same in
// Python takes 12 - 40 (more than the kernels of such a call).  No kernel lives here; the entry points are those of the library that the Python side has
// loaded, handed over by address, one Ops per element type.  A call that does not fit is a ValueError, before anything is enqueued, the library's own refusals
// among them; a launch that fails is a RuntimeError.
#include <torch/extension.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <cstdint>
#include <initializer_list>
#include <optional>
#include <string>
#include <tuple>
#include <vector>

#include "omniserve_lm.h"

namespace py = pybind11;

namespace {

typedef torch::Tensor T;
typedef std::optional<T> OptT;
typedef std::vector<T> Pools;

constexpr int64_t PAGE = 64;
constexpr int NO_WINDOW = INT32_MAX;
constexpr int64_t MOST_HEADS = 4096, MOST_ROWS = 1 << 24;      // of a row; drafted tokens times heads

template <typename... What>
inline void need(bool ok, const What&... what) {
  if (!ok) throw py::value_error(c10::str(what...));
}

inline void done(int rc, const char* name) {
  if (rc == 0) return;
  if (rc == -22) throw py::value_error(std::string(name) + ": sizes, strides or addresses that it does not take");
  throw std::runtime_error(std::string(name) + " failed: " + (rc == -5 ? "kernel launch failed" : "error") + " (" + std::to_string(rc) + ")");
}

// from row to row (a single row's stride may be anything)
inline int64_t step(const T& t) { return t.size(0) > 1 ? t.stride(0) : 0; }
inline bool at16(const T& t) { return (uintptr_t)t.data_ptr() % 16 == 0 && step(t) * t.element_size() % 16 == 0; }
inline void* ptr(const OptT& t) { return t ? t->data_ptr() : nullptr; }

inline void index(const T& t, int64_t n, const char* name) {
  need(t.scalar_type() == torch::kInt32 && t.dim() == 1 && t.size(0) == n && t.is_contiguous(), name, ": ", n, " contiguous int32");
}

inline bool code_size(int64_t d) { return d == 64 || d == 128 || d == 256; }

struct Turn {
  const double* freq = nullptr;
  int half = 0;
  const int* pos = nullptr;
  int halves = 0;
};

struct Sizes { int64_t pages, G, dk, dv; };

class Ops {
  c10::ScalarType elem;
  decltype(&lm_rope) rope_;
  decltype(&lm_kv_store) store_;
  decltype(&lm_kv_load) load_;
  decltype(&lm_tree_attn_scratch) scratch_;
  decltype(&lm_tree_attn) tree_;

  // a matrix of at least `width` neighbouring columns, and of `n` rows (< 0: of any number)
  void rows(const T& t, int64_t width, int64_t n, const char* name) const {
    need(t.dim() == 2 && t.size(1) >= width && t.scalar_type() == elem && (t.stride(1) == 1 || t.size(1) == 1), name, ": rows of ", width, " or more ", elem);
    need(n < 0 || t.size(0) == n, name, ": ", n, " rows");
  }
  // ... that a call writes: no two of them share memory
  void results(const T& t, int64_t width, int64_t n, const char* name) const {
    rows(t, width, n, name);
    need(t.size(0) <= 1 || t.stride(0) >= width, name, ": rows that do not overlap");
  }

  static Turn turn(const OptT& freq, const OptT& pos, int64_t n, int64_t dk, const std::string& pairing) {
    need(pairing == "neighbours" || pairing == "halves", "pairing: neighbours or halves");
    need(freq.has_value() == pos.has_value(), "freq and pos come together");
    if (!freq) return {};
    need(freq->scalar_type() == torch::kFloat64 && freq->dim() == 1 && freq->is_contiguous() && freq->numel() > 0 && 2 * freq->numel() <= dk, "freq: float64 of up to half of a head");
    index(*pos, n, "pos");
    return {freq->data_ptr<double>(), (int)freq->numel(), pos->data_ptr<int>(), pairing == "halves"};
  }

  // of a quantised cache, or (codes false) of pools of elements
  Sizes pools(const Pools& c, bool codes) const {
    need(c.size() == (codes ? 4u : 2u), "a cache: pools of keys and values, and of their exponents where they are codes");
    const T &k = c[0], &v = c[1];
    need(k.dim() == 4 && v.dim() == 4 && k.size(0) == v.size(0) && k.size(1) == v.size(1) && k.size(2) == PAGE && v.size(2) == PAGE && code_size(k.size(3)) && code_size(v.size(3)),
         "pools [pages, kv heads, 64, size], sizes 64, 128 and 256");
    const auto type = codes ? torch::kUInt8 : elem;
    for (const T& t : c) need(t.scalar_type() == type && t.is_contiguous(), "contiguous pools of ", type);
    for (size_t i = 2; i < c.size(); ++i)
      need(c[i].dim() == 3 && c[i].size(0) == k.size(0) && c[i].size(1) == k.size(1) && c[i].size(2) == PAGE, "exponents [pages, kv heads, 64]");
    return {k.size(0), k.size(1), k.size(3), v.size(3)};
  }

  // where a call runs: its tensors' device, which all of them share
  static void one_device(const T& first, const Pools& c, std::initializer_list<const T*> more) {
    need(first.is_cuda(), "tensors must live on the GPU");
    const auto d = first.device();
    for (const T& t : c) need(t.device() == d, "tensors of one device");
    for (const T* t : more) need(t == nullptr || t->device() == d, "tensors of one device");
  }
  static const T* opt(const OptT& t) { return t ? &*t : nullptr; }
  static void* stream(const T& t) { return (void*)c10::hip::getCurrentHIPStream(t.get_device()).stream(); }
  static int narrow(int64_t n) {
    need(n >= INT32_MIN && n <= INT32_MAX, "a size beyond 32 bits");
    return (int)n;
  }

 public:
  Ops(bool bf16, uintptr_t rope, uintptr_t store, uintptr_t load, uintptr_t scratch, uintptr_t tree)
      : elem(bf16 ? torch::kBFloat16 : torch::kFloat32), rope_((decltype(rope_))rope), store_((decltype(store_))store), load_((decltype(load_))load),
        scratch_((decltype(scratch_))scratch), tree_((decltype(tree_))tree) {}

  T rope(const T& x, const OptT& freq, const OptT& pos, int64_t heads, int64_t dk, const std::string& pairing, double factor, const OptT& out) const {
    need(heads > 0 && heads <= MOST_HEADS && dk > 0 && dk <= INT32_MAX, "heads: 1 to ", MOST_HEADS, ", of at least one dimension");
    const int64_t w = heads * dk;
    rows(x, w, -1, "x");
    const int64_t n = x.size(0);
    const Turn t = turn(freq, pos, n, dk, pairing);
    need(t.half > 0, "freq and pos say how rope turns");
    if (out) results(*out, w, n, "out");
    one_device(x, {}, {opt(freq), opt(pos), opt(out)});
    const c10::DeviceGuard guard(x.device());
    const T o = out ? *out : torch::empty({n, w}, x.options());
    done(rope_(x.data_ptr(), step(x), o.data_ptr(), step(o), t.freq, t.half, t.pos, t.halves, factor, narrow(n), (int)heads, (int)dk, stream(x)), "lm_rope");
    return o;
  }

  void kv_store(const T& x, const Pools& cache, const T& slot, int64_t heads, const OptT& freq, const OptT& pos, const std::string& pairing, double factor, const OptT& q_out,
                const OptT& picked) const {
    const Sizes s = pools(cache, true);
    need(heads >= 0 && heads + s.G <= MOST_HEADS, "heads: none or more, ", MOST_HEADS, " at most with the kv heads");
    need((uintptr_t)cache[0].data_ptr() % 8 == 0 && (uintptr_t)cache[1].data_ptr() % 8 == 0, "cache: pools at 8 bytes");
    rows(x, (heads + s.G) * s.dk + s.G * s.dv, -1, "x");
    const int64_t n = picked ? slot.size(0) : x.size(0);
    index(slot, n, "slot");
    const Turn t = turn(freq, pos, n, s.dk, pairing);
    need(!q_out || (!picked && heads > 0 && t.half > 0), "queries are turned of all rows in order");
    if (q_out) results(*q_out, heads * s.dk, n, "q_out");
    if (picked) index(*picked, n, "rows");
    one_device(x, cache, {&slot, opt(freq), opt(pos), opt(q_out), opt(picked)});
    const c10::DeviceGuard guard(x.device());
    done(store_(x.data_ptr(), step(x), narrow(x.size(0)), (const int*)ptr(picked), t.freq, t.half, t.pos, t.halves, factor, ptr(q_out), q_out ? step(*q_out) : 0,
                slot.data_ptr<int>(), cache[0].data_ptr<uint8_t>(), cache[1].data_ptr<uint8_t>(), cache[2].data_ptr<uint8_t>(), cache[3].data_ptr<uint8_t>(), s.pages, narrow(n),
                (int)heads, narrow(s.G), (int)s.dk, (int)s.dv, stream(x)),
         "lm_kv_store");
  }

  std::tuple<T, T> kv_load(const Pools& cache, const T& slot, const std::optional<std::tuple<T, T>>& out) const {
    const Sizes s = pools(cache, true);
    need(slot.dim() == 1, "slot: a vector");
    const int64_t n = slot.size(0);
    index(slot, n, "slot");
    need(s.G <= MOST_HEADS, "kv heads: ", MOST_HEADS, " at most");
    need((uintptr_t)cache[0].data_ptr() % 16 == 0 && (uintptr_t)cache[1].data_ptr() % 16 == 0, "cache: pools at 16 bytes");
    if (out) {
      results(std::get<0>(*out), s.G * s.dk, n, "out");
      results(std::get<1>(*out), s.G * s.dv, n, "out");
      need(at16(std::get<0>(*out)) && at16(std::get<1>(*out)), "out: rows at 16 bytes");
      one_device(slot, {}, {&std::get<0>(*out), &std::get<1>(*out)});
    }
    one_device(slot, cache, {});
    const c10::DeviceGuard guard(slot.device());
    const auto options = slot.options().dtype(elem);
    const T k = out ? std::get<0>(*out) : torch::empty({n, s.G * s.dk}, options), v = out ? std::get<1>(*out) : torch::empty({n, s.G * s.dv}, options);
    done(load_(k.data_ptr(), step(k), v.data_ptr(), step(v), cache[0].data_ptr<uint8_t>(), cache[1].data_ptr<uint8_t>(), cache[2].data_ptr<uint8_t>(), cache[3].data_ptr<uint8_t>(),
               s.pages, slot.data_ptr<int>(), narrow(n), narrow(s.G), (int)s.dk, (int)s.dv, stream(slot)),
         "lm_kv_load");
    return {k, v};
  }

  T tree_attn(const T& q, const T& k, const T& v, const T& mask, const T& first, const T& pos, const Pools& cache, const T& bt, const T& length, double scale,
              const std::optional<int64_t>& window, int64_t max_draft, int64_t max_context, const OptT& out) const {
    const bool codes = cache.size() == 4;
    const Sizes s = pools(cache, codes);
    for (const T& t : cache) need((uintptr_t)t.data_ptr() % 16 == 0, "cache: pools at 16 bytes");
    need(q.dim() == 2 && s.G > 0, "q: rows, over kv heads");
    need(length.dim() == 1, "length: a vector");
    const int64_t n = q.size(0), B = length.size(0), H = q.size(1) / s.dk;
    need(H > 0 && H % s.G == 0 && q.size(1) == H * s.dk, "q: a multiple of the ", s.G, " kv heads, of ", s.dk, " each");
    rows(q, H * s.dk, n, "q");
    rows(k, s.G * s.dk, n, "k");
    rows(v, s.G * s.dv, n, "v");
    need(at16(q), "q: rows at 16 bytes");
    need(at16(k), "k: rows at 16 bytes");
    need(at16(v), "v: rows at 16 bytes");
    need(mask.scalar_type() == torch::kInt64 && mask.dim() == 2 && mask.size(0) == n && mask.is_contiguous(), "mask: contiguous int64 [tokens, words]");
    need(0 <= max_draft && max_draft <= 64 * mask.size(1), "the mask has ", 64 * mask.size(1), " bits for ", max_draft, " drafted tokens");
    index(first, B + 1, "first");
    index(pos, n, "pos");
    index(length, B, "length");
    need(bt.scalar_type() == torch::kInt32 && bt.dim() == 2 && bt.size(0) == B && (bt.stride(1) == 1 || bt.size(1) <= 1), "bt: int32 [sequences, pages]");
    need(B <= 1 || bt.stride(0) >= bt.size(1), "bt: rows that do not overlap");
    need(bt.size(1) == 0 || s.pages > 0, "a block table needs pages");
    need(max_draft * H <= MOST_ROWS, "max_draft: ", MOST_ROWS, " rows of tokens times heads at most");
    need(scale >= 0x1p-60 && scale <= 0x1p60 && (!window || *window > 0), "scale: 2^-60 to 2^60; window: positive");
    need(max_context >= 0, "max_context is a number of keys");
    if (out) {
      results(*out, H * s.dv, n, "out");
      need((uintptr_t)out->data_ptr() % (4 * out->element_size()) == 0 && step(*out) % 4 == 0, "out: rows at four elements");
    }
    one_device(q, cache, {&k, &v, &mask, &first, &pos, &bt, &length, opt(out)});
    const c10::DeviceGuard guard(q.device());
    const T o = out ? *out : torch::empty({n, H * s.dv}, q.options());
    const int draft = narrow(max_draft), context = (int)std::min<int64_t>(max_context, INT32_MAX), heads = narrow(H), kv_heads = narrow(s.G), seqs = narrow(B);
    const int64_t room = scratch_(seqs, draft, context, heads, kv_heads, (int)s.dk, (int)s.dv, codes);
    const T part = room ? torch::empty({room}, q.options().dtype(torch::kFloat32)) : T();
    done(tree_(q.data_ptr(), step(q), k.data_ptr(), step(k), v.data_ptr(), step(v), cache[0].data_ptr(), cache[1].data_ptr(), codes ? cache[2].data_ptr<uint8_t>() : nullptr,
               codes ? cache[3].data_ptr<uint8_t>() : nullptr, s.pages, bt.data_ptr<int>(), narrow(B > 1 ? bt.stride(0) : bt.size(1)), narrow(bt.size(1)), length.data_ptr<int>(),
               first.data_ptr<int>(), pos.data_ptr<int>(), mask.data_ptr<int64_t>(), narrow(mask.size(1)), o.data_ptr(), step(o), room ? part.data_ptr<float>() : nullptr,
               (float)scale, (int)std::min<int64_t>(window.value_or(NO_WINDOW), NO_WINDOW), seqs, narrow(n), draft, context, heads, kv_heads, (int)s.dk, (int)s.dv, stream(q)),
         "lm_tree_attn");
    return o;
  }
};

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("abi_version", []() { return LM_ABI_VERSION; });
  py::class_<Ops>(m, "Ops")
      .def(py::init<bool, uintptr_t, uintptr_t, uintptr_t, uintptr_t, uintptr_t>())
      .def("rope", &Ops::rope)
      .def("kv_store", &Ops::kv_store)
      .def("kv_load", &Ops::kv_load)
      .def("tree_attn", &Ops::tree_attn);
}
