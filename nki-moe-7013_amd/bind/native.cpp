// Checked calls of the cache operators for qmoe/ops.py.
//
// A decode step makes these calls around a few microseconds of kernel each, so
// what the host does for one counts as much: the checks of up to 14 tensors, the
// outputs and the workspace.  In Python that was 10 us of kv_append's 14.9 and 9
// of attn_decode_scored's 17 (each launch is 3.7 us of the rest); here it is
// about 2.  Arguments that do not fit raise ValueError before anything is
// launched, as every wrapper in ops.py does.
#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <pybind11/pybind11.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <initializer_list>
#include <optional>
#include <sstream>
#include <string>

#include "qmoe_capi.h"

namespace py = pybind11;

namespace {

constexpr at::ScalarType BF16 = at::kBFloat16, F32 = at::kFloat, I32 = at::kInt, U8 = at::kByte;
using Shape = std::initializer_list<int64_t>;

[[noreturn]] void refuse(const std::string& msg) { throw py::value_error(msg); }

std::string text(at::IntArrayRef shape) {
  std::ostringstream s;
  s << "(";
  for (size_t i = 0; i < shape.size(); ++i) s << (i ? ", " : "") << shape[i];
  s << (shape.size() == 1 ? ",)" : ")");
  return s.str();
}

const at::Tensor& tensor(py::handle h, const char* name) {
  if (!THPVariable_Check(h.ptr()))
    refuse(std::string(name) + ": expected a tensor, got " + Py_TYPE(h.ptr())->tp_name);
  return THPVariable_Unpack(h.ptr());
}

// The GPU of the operand that says the call's sizes.
int gpu_of(const at::Tensor& t, const char* name, const char* dims, int64_t n) {
  if (t.dim() != n) refuse(std::string(name) + " must be " + dims);
  if (!t.is_cuda()) refuse(std::string(name) + ": must be on a GPU (got " + t.device().str() + ")");
  return t.get_device();
}

// The kernels load and store bf16 rows 16 bytes at a time (kv_append's one element at a
// time), and everything else, lengths and scores, in single words.
constexpr uintptr_t any_alignment = 1;
constexpr uintptr_t alignment_of(at::ScalarType dtype) { return dtype == BF16 ? 16 : any_alignment; }

// Address of a contiguous tensor of this dtype, shape and alignment on GPU ix.
void* address(const at::Tensor& t, const char* name, at::ScalarType dtype, at::IntArrayRef shape, int ix,
              uintptr_t align) {
  if (!t.is_cuda()) refuse(std::string(name) + ": must be on a GPU (got " + t.device().str() + ")");
  if (t.scalar_type() != dtype)
    refuse(std::string(name) + ": dtype must be " + c10::toString(dtype) + " (got " + c10::toString(t.scalar_type()) +
           ")");
  if (!t.is_contiguous()) refuse(std::string(name) + ": must be contiguous");
  if (t.sizes() != shape)
    refuse(std::string(name) + ": shape must be " + text(shape) + " (got " + text(t.sizes()) + ")");
  if (t.get_device() != ix)
    refuse("tensors are on different devices: " + std::string(name) + " is on " + t.device().str() +
           ", expected cuda:" + std::to_string(ix));
  void* p = t.data_ptr();
  if (reinterpret_cast<uintptr_t>(p) % align)
    refuse(std::string(name) + ": must be " + std::to_string(align) + "-byte aligned");
  return p;
}

void* address(const at::Tensor& t, const char* name, at::ScalarType dtype, at::IntArrayRef shape, int ix) {
  return address(t, name, dtype, shape, ix, alignment_of(dtype));
}

template <class T>
T* arg(py::handle h, const char* name, at::ScalarType dtype, Shape shape, int ix, uintptr_t align) {
  return static_cast<T*>(address(tensor(h, name), name, dtype, at::IntArrayRef(shape), ix, align));
}

template <class T>
T* arg(py::handle h, const char* name, at::ScalarType dtype, Shape shape, int ix) {
  return arg<T>(h, name, dtype, shape, ix, alignment_of(dtype));
}

template <class T>
T* optional_arg(py::handle h, const char* name, at::ScalarType dtype, Shape shape, int ix) {
  return h.is_none() ? nullptr : arg<T>(h, name, dtype, shape, ix);
}

at::Tensor empty(at::IntArrayRef shape, at::ScalarType dtype, int ix) {
  return at::empty(shape, at::TensorOptions().dtype(dtype).device(at::kCUDA, static_cast<c10::DeviceIndex>(ix)));
}

// The output the caller gave, or a new one.
struct Output {
  py::object obj;
  void* p;
  Output(py::handle h, const char* name, at::ScalarType dtype, Shape shape, int ix, uintptr_t align) {
    if (h.is_none()) {
      at::Tensor t = empty(at::IntArrayRef(shape), dtype, ix);
      p = t.data_ptr();
      obj = py::reinterpret_steal<py::object>(THPVariable_Wrap(std::move(t)));
    } else {
      p = address(tensor(h, name), name, dtype, at::IntArrayRef(shape), ix, align);
      obj = py::reinterpret_borrow<py::object>(h);
    }
  }
};

// The caller's workspace, if it is large enough, or a new one.
struct Scratch {
  at::Tensor t;
  void* p = nullptr;
  int64_t bytes = 0;
  Scratch(py::handle h, int64_t need, int ix, uintptr_t align) {
    if (h.is_none()) {
      if (need <= 0) return;
      t = empty({need}, U8, ix);
      p = t.data_ptr();
      bytes = need;
      return;
    }
    t = tensor(h, "workspace");
    if (!t.is_cuda() || t.get_device() != ix || !t.is_contiguous())
      refuse("workspace: must be a contiguous tensor on cuda:" + std::to_string(ix));
    bytes = t.numel() * t.element_size();
    if (bytes < need)
      refuse("workspace: needs " + std::to_string(need) + " bytes (got " + std::to_string(bytes) + ")");
    p = t.data_ptr();
    if (reinterpret_cast<uintptr_t>(p) % align)
      refuse("workspace: must be " + std::to_string(align) + "-byte aligned");
  }
};

void check(int rc, const char* fn) {
  if (rc == QMOE_OK) return;
  const std::string why = qmoe_last_error();
  if (rc == QMOE_ERR_INVALID) refuse(std::string(fn) + ": invalid argument: " + why);
  py::object type = py::module_::import("qmoe._lib").attr("QmoeError");
  PyErr_SetString(type.ptr(), (std::string(fn) + ": HIP error: " + why).c_str());
  throw py::error_already_set();
}

int64_t size(int64_t n, const char* fn) {
  if (n < 0) refuse(std::string(fn) + ": bad sizes");
  return n;
}

qmoe_stream_t stream(int ix) { return c10::hip::getCurrentHIPStream(static_cast<c10::DeviceIndex>(ix)).stream(); }

// Makes GPU ix current for a call.
struct On {
  c10::OptionalDeviceGuard guard;
  explicit On(int ix) : guard(at::Device(at::kCUDA, static_cast<c10::DeviceIndex>(ix))) {}
};

void cache_sizes(const at::Tensor& k, int64_t B, int64_t D, int64_t& Hkv, int64_t& S_max) {
  if (k.dim() != 4 || k.size(0) != B || k.size(3) != D)
    refuse("k_cache must be [B=" + std::to_string(B) + ", Hkv, S_max, D=" + std::to_string(D) + "] (got " +
           text(k.sizes()) + ")");
  Hkv = k.size(1);
  S_max = k.size(2);
}

void heads(int64_t Hq, int64_t Hkv) {
  if (Hkv <= 0 || Hq % Hkv || Hq / Hkv > 16)
    refuse("need Hq a multiple of Hkv, by at most 16 (Hq=" + std::to_string(Hq) + ", Hkv=" + std::to_string(Hkv) + ")");
}

double number(py::handle h, const char* name) {
  const double x = PyFloat_AsDouble(h.ptr());
  if (x == -1.0 && PyErr_Occurred()) {
    PyErr_Clear();
    refuse(std::string(name) + " must be a number");
  }
  return x;
}

float scale_of(py::handle h, int64_t D) {
  const double s = h.is_none() ? 1.0 / std::sqrt(double(D)) : number(h, "scale");
  if (!(s > 0.0) || !std::isfinite(s)) refuse("scale must be positive and finite");
  return float(s);
}

// Any integer (an __index__ of its own included).  Arguments come as handles, not as
// typed parameters: pybind would answer another type with its own TypeError.
int64_t integer(py::handle h, const char* name) {
  const int64_t n = h.is_none() ? -1 : PyLong_AsLongLong(h.ptr());
  if (h.is_none() || (n == -1 && PyErr_Occurred())) {
    PyErr_Clear();
    refuse(std::string(name) + " must be an integer");
  }
  return n;
}

// An integer within [lo, hi].
int64_t within(py::handle h, const char* name, int64_t lo, int64_t hi) {
  const int64_t n = integer(h, name);
  if (n < lo || n > hi)
    refuse(std::string(name) + " must be in [" + std::to_string(lo) + ", " + std::to_string(hi) + "] (got " +
           std::to_string(n) + ")");
  return n;
}

// The same, or `none` where None was given.
int64_t within(py::handle h, const char* name, int64_t lo, int64_t hi, int64_t none) {
  return h.is_none() ? none : within(h, name, lo, hi);
}

// A number of rows, tokens or heads.
int64_t count(py::handle h, const char* name) { return within(h, name, 0, INT32_MAX); }

using Bf = qmoe_bf16;

struct Queries {
  int ix;
  int64_t T, Hq, D;
  const Bf* p;
  Queries(py::handle h, int64_t rows, const char* dims) {
    const at::Tensor& q = tensor(h, "q");
    ix = gpu_of(q, "q", dims, 3);
    T = q.size(0);
    Hq = q.size(1);
    D = q.size(2);
    if (rows >= 0 && T != rows)
      refuse("q must be [" + std::to_string(rows) + ", Hq, D] (got " + text(q.sizes()) + ")");
    p = static_cast<const Bf*>(address(q, "q", BF16, q.sizes(), ix));
  }
};

py::object attn_shared(py::handle q, py::handle k_prefix, py::handle v_prefix, py::handle k_cache, py::handle v_cache,
                       py::handle ctx_len, py::handle batch, py::handle queries, py::handle prefix_len,
                       py::handle scale, py::handle workspace, py::handle out, py::handle max_ctx) {
  const int64_t B = count(batch, "B"), S = count(queries, "S");
  const Queries x(q, B * S, "[B*S, Hq, D]");
  int64_t Hkv, S_max;
  cache_sizes(tensor(k_cache, "k_cache"), B, x.D, Hkv, S_max);
  heads(x.Hq, Hkv);
  const at::Tensor& kp = tensor(k_prefix, "k_prefix");
  if (kp.dim() != 3 || kp.size(0) != Hkv || kp.size(2) != x.D)
    refuse("k_prefix must be [Hkv=" + std::to_string(Hkv) + ", P_max, D=" + std::to_string(x.D) + "] (got " +
           text(kp.sizes()) + ")");
  const int64_t P_max = kp.size(1), P = within(prefix_len, "prefix_len", 0, P_max, P_max);
  const int64_t ctx = within(max_ctx, "max_ctx", 0, S_max, S_max);
  const float sc = scale_of(scale, x.D);
  const Bf* pkp = arg<Bf>(k_prefix, "k_prefix", BF16, {Hkv, P_max, x.D}, x.ix);
  const Bf* pvp = arg<Bf>(v_prefix, "v_prefix", BF16, {Hkv, P_max, x.D}, x.ix);
  const Bf* pk = arg<Bf>(k_cache, "k_cache", BF16, {B, Hkv, S_max, x.D}, x.ix);
  const Bf* pv = arg<Bf>(v_cache, "v_cache", BF16, {B, Hkv, S_max, x.D}, x.ix);
  const int32_t* pc = arg<int32_t>(ctx_len, "ctx_len", I32, {B}, x.ix);
  const On on(x.ix);
  const Output o(out, "out", BF16, {x.T, x.Hq * x.D}, x.ix, 16);
  const Scratch ws(workspace, size(qmoe_attn_shared_workspace(B, S, x.Hq, Hkv, x.D, P, ctx), "qmoe_attn_shared"),
                   x.ix, 16);
  check(qmoe_attn_shared(x.p, pkp, pvp, P, P_max, pk, pv, pc, B, S, x.Hq, Hkv, x.D, S_max, ctx, sc, ws.p, ws.bytes,
                         static_cast<Bf*>(o.p), stream(x.ix)),
        "qmoe_attn_shared");
  return o.obj;
}

py::object attn_prefill_scored(py::handle q, py::handle k_cache, py::handle v_cache, py::handle scores,
                               py::handle batch, py::handle queries, py::handle at, py::handle lengths,
                               py::handle scale, py::handle workspace, py::handle out) {
  const int64_t B = count(batch, "B"), S = count(queries, "S"), start = integer(at, "start");
  const Queries x(q, B * S, "[B*S, Hq, D]");
  int64_t Hkv, S_max;
  cache_sizes(tensor(k_cache, "k_cache"), B, x.D, Hkv, S_max);
  heads(x.Hq, Hkv);
  if (start < 0 || start > S_max - S)
    refuse("need 0 <= start and start + S <= S_max=" + std::to_string(S_max) + " (start=" + std::to_string(start) +
           ", S=" + std::to_string(S) + ")");
  const float sc = scale_of(scale, x.D);
  const Bf* pk = arg<Bf>(k_cache, "k_cache", BF16, {B, Hkv, S_max, x.D}, x.ix);
  const Bf* pv = arg<Bf>(v_cache, "v_cache", BF16, {B, Hkv, S_max, x.D}, x.ix);
  float* ps = arg<float>(scores, "scores", F32, {B, Hkv, S_max}, x.ix);
  const int32_t* pl = optional_arg<int32_t>(lengths, "lengths", I32, {B}, x.ix);
  const On on(x.ix);
  const Output o(out, "out", BF16, {x.T, x.Hq * x.D}, x.ix, 16);
  const Scratch ws(
      workspace,
      size(qmoe_attn_prefill_scored_workspace(B, S, x.Hq, Hkv, x.D, start), "qmoe_attn_prefill_scored"), x.ix, 16);
  check(qmoe_attn_prefill_scored(x.p, pk, pv, B, S, x.Hq, Hkv, x.D, S_max, start, pl, sc, ws.p, ws.bytes, ps,
                                 static_cast<Bf*>(o.p), stream(x.ix)),
        "qmoe_attn_prefill_scored");
  return o.obj;
}

py::object attn_decode_scored(py::handle q, py::handle k_cache, py::handle v_cache, py::handle ctx_len,
                              py::handle scores, py::handle scale, py::handle workspace, py::handle out,
                              py::handle max_ctx) {
  const Queries x(q, -1, "[B, Hq, D]");
  const int64_t B = x.T;
  int64_t Hkv, S_max;
  cache_sizes(tensor(k_cache, "k_cache"), B, x.D, Hkv, S_max);
  heads(x.Hq, Hkv);
  const int64_t ctx = within(max_ctx, "max_ctx", 1, S_max, S_max);
  const float sc = scale_of(scale, x.D);
  const Bf* pk = arg<Bf>(k_cache, "k_cache", BF16, {B, Hkv, S_max, x.D}, x.ix);
  const Bf* pv = arg<Bf>(v_cache, "v_cache", BF16, {B, Hkv, S_max, x.D}, x.ix);
  float* ps = arg<float>(scores, "scores", F32, {B, Hkv, S_max}, x.ix);
  const int32_t* pc = arg<int32_t>(ctx_len, "ctx_len", I32, {B}, x.ix);
  const On on(x.ix);
  const Output o(out, "out", BF16, {B, x.Hq * x.D}, x.ix, 16);
  const Scratch ws(workspace,
                   size(qmoe_attn_decode_scored_workspace(B, x.Hq, x.D, ctx), "qmoe_attn_decode_scored"), x.ix,
                   16);
  check(qmoe_attn_decode_scored(x.p, pk, pv, pc, B, x.Hq, Hkv, x.D, S_max, ctx, sc, ws.p, ws.bytes, ps,
                                static_cast<Bf*>(o.p), stream(x.ix)),
        "qmoe_attn_decode_scored");
  return o.obj;
}

py::object kv_append(py::handle qkv, py::handle q_norm_w, py::handle k_norm_w, py::handle rope_cos,
                     py::handle rope_sin, py::handle positions, py::handle slots, py::handle q_heads,
                     py::handle kv_heads, py::handle k_cache, py::handle v_cache, py::handle epsilon,
                     py::handle scores, py::handle slot_pos, py::handle q_out) {
  const int64_t Hq = count(q_heads, "Hq"), Hkv = count(kv_heads, "Hkv");
  const float eps = float(number(epsilon, "eps"));
  const at::Tensor& raw = tensor(qkv, "qkv");
  const int ix = gpu_of(raw, "qkv", "[B, (Hq + 2 Hkv) * D]", 2);
  const at::Tensor &k = tensor(k_cache, "k_cache"), &cos = tensor(rope_cos, "rope_cos");
  const int64_t B = raw.size(0), D = k.dim() == 4 ? k.size(3) : 0;
  int64_t n_kv, S_max;
  cache_sizes(k, B, D, n_kv, S_max);
  if (n_kv != Hkv)
    refuse("k_cache must have Hkv=" + std::to_string(Hkv) + " heads (got " + std::to_string(n_kv) + ")");
  if (cos.dim() != 2) refuse("rope_cos must be [max_pos, D / 2]");
  const int64_t max_pos = cos.size(0);
  const float* praw = arg<float>(qkv, "qkv", F32, {B, (Hq + 2 * Hkv) * D}, ix);
  const Bf* pqn = arg<Bf>(q_norm_w, "q_norm_w", BF16, {D}, ix, any_alignment);
  const Bf* pkn = arg<Bf>(k_norm_w, "k_norm_w", BF16, {D}, ix, any_alignment);
  const float* pcos = arg<float>(rope_cos, "rope_cos", F32, {max_pos, D / 2}, ix);
  const float* psin = arg<float>(rope_sin, "rope_sin", F32, {max_pos, D / 2}, ix);
  const int32_t* pp = arg<int32_t>(positions, "positions", I32, {B}, ix);
  const int32_t* psl = arg<int32_t>(slots, "slots", I32, {B}, ix);
  Bf* pk = arg<Bf>(k_cache, "k_cache", BF16, {B, Hkv, S_max, D}, ix, any_alignment);
  Bf* pv = arg<Bf>(v_cache, "v_cache", BF16, {B, Hkv, S_max, D}, ix, any_alignment);
  float* ps = optional_arg<float>(scores, "scores", F32, {B, Hkv, S_max}, ix);
  int32_t* psp = optional_arg<int32_t>(slot_pos, "slot_pos", I32, {B, Hkv, S_max}, ix);
  const On on(ix);
  const Output o(q_out, "q_out", BF16, {B, Hq, D}, ix, any_alignment);
  check(qmoe_kv_append(praw, pqn, pkn, pcos, psin, max_pos, pp, psl, B, Hq, Hkv, D, S_max, eps,
                       static_cast<Bf*>(o.p), pk, pv, ps, psp, stream(ix)),
        "qmoe_kv_append");
  return o.obj;
}

struct Cache {
  at::Tensor t[4];
  void* p[4];
  Cache(const py::handle (&h)[4], const char* const (&names)[4], int64_t B, int64_t Hkv, int64_t S, int64_t D,
        int ix) {
    const at::ScalarType dt[4] = {BF16, BF16, F32, I32};
    for (int i = 0; i < 4; ++i) {
      t[i] = tensor(h[i], names[i]);
      p[i] = i < 2 ? address(t[i], names[i], dt[i], {B, Hkv, S, D}, ix) : address(t[i], names[i], dt[i], {B, Hkv, S}, ix);
    }
  }
  bool overlaps(const Cache& o) const {
    for (int i = 0; i < 4; ++i)
      for (int j = 0; j < 4; ++j) {
        const char *a = static_cast<char*>(p[i]), *b = static_cast<char*>(o.p[j]);
        if (a < b + o.t[j].nbytes() && b < a + t[i].nbytes()) return true;
      }
    return false;
  }
};

void kv_evict(py::handle k_cache, py::handle v_cache, py::handle scores, py::handle slot_pos, py::handle ctx_len,
              py::handle entries, py::handle last, py::handle first, py::handle out, py::handle workspace) {
  const int64_t budget = integer(entries, "budget"), recent = integer(last, "recent"), sink = integer(first, "sink");
  const at::Tensor& k = tensor(k_cache, "k_cache");
  const int ix = gpu_of(k, "k_cache", "[B, Hkv, S_max, D]", 4);
  const int64_t B = k.size(0), Hkv = k.size(1), S_max = k.size(2), D = k.size(3);
  if (budget <= 0 || recent < 0 || sink < 0 || recent > budget - sink)
    refuse("need budget > 0 and 0 <= recent + sink <= budget (budget=" + std::to_string(budget) +
           ", recent=" + std::to_string(recent) + ", sink=" + std::to_string(sink) + ")");
  const Cache from({k_cache, v_cache, scores, slot_pos}, {"k_cache", "v_cache", "scores", "slot_pos"}, B, Hkv, S_max,
                   D, ix);
  const int32_t* pc = arg<int32_t>(ctx_len, "ctx_len", I32, {B}, ix);
  std::optional<Cache> other;
  int64_t S_out = S_max;
  if (!out.is_none()) {
    if (!PySequence_Check(out.ptr()) || PySequence_Size(out.ptr()) != 4)
      refuse("out must be (k, v, scores, slot_pos)");
    const py::object o[4] = {py::cast<py::sequence>(out)[0], py::cast<py::sequence>(out)[1],
                             py::cast<py::sequence>(out)[2], py::cast<py::sequence>(out)[3]};
    const at::Tensor& k2 = tensor(o[0], "k_out");
    if (k2.dim() != 4 || k2.size(2) < std::min(budget, S_max))
      refuse("out needs at least " + std::to_string(std::min(budget, S_max)) + " slots (got " + text(k2.sizes()) + ")");
    S_out = k2.size(2);
    other.emplace(Cache({o[0], o[1], o[2], o[3]}, {"k_out", "v_out", "scores_out", "slot_pos_out"}, B, Hkv, S_out, D, ix));
    if (from.overlaps(*other)) refuse("out overlaps the cache (leave it out to evict in place)");
  }
  const Cache& to = other ? *other : from;
  const On on(ix);
  const Scratch ws(workspace, size(qmoe_kv_evict_workspace(B, Hkv, S_max, budget), "qmoe_kv_evict"), ix,
                   alignof(int32_t));
  check(qmoe_kv_evict(static_cast<Bf*>(from.p[0]), static_cast<Bf*>(from.p[1]), static_cast<float*>(from.p[2]),
                      static_cast<int32_t*>(from.p[3]), pc, B, Hkv, D, S_max, budget, recent, sink, ws.p, ws.bytes,
                      S_out, static_cast<Bf*>(to.p[0]), static_cast<Bf*>(to.p[1]), static_cast<float*>(to.p[2]),
                      static_cast<int32_t*>(to.p[3]), stream(ix)),
        "qmoe_kv_evict");
}

// Bytes -> a workspace tensor on GPU ix (None for 0).
py::object workspace(int64_t bytes, const char* fn, int ix) {
  size(bytes, fn);
  if (bytes == 0) return py::none();
  const On on(ix);
  return py::reinterpret_steal<py::object>(THPVariable_Wrap(empty({bytes}, U8, ix)));
}

}  // namespace

PYBIND11_MODULE(_native, m) {
  m.doc() = "Checked calls of libqmoe's cache operators (see qmoe.ops).";
  m.def("attn_shared", &attn_shared);
  m.def("attn_prefill_scored", &attn_prefill_scored);
  m.def("attn_decode_scored", &attn_decode_scored);
  m.def("kv_append", &kv_append);
  m.def("kv_evict", &kv_evict);
  m.def("workspace", &workspace);
}
