// Tensor binding of the operators of include/ek.h (module `_ekops`): argument
// checks, outputs and workspaces from torch's allocator, the current stream of
// the tensors' device. Plain host code, compiled against torch's headers; the
// entry points of libek.so are handed over by address (bind), so that the
// library which `megakernels.ek` loaded is the one called.
//
// It is compiled because the checks, made attribute by attribute in Python,
// took 20 to 30 us a call, several times the kernels of a small call.
#include <ATen/ATen.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/pybind.h>

#include <algorithm>
#include <cmath>
#include <string>

#include "../../include/ek.h"

namespace py = pybind11;
using at::Tensor;

namespace {

struct Api {
  const char* (*last_error)() = nullptr;
  int (*kv_write)(const EkKvCopyArgs*, void*) = nullptr;
  int (*kv_read)(const EkKvCopyArgs*, void*) = nullptr;
  int64_t (*attention_workspace)(const EkPrefixAttnArgs*) = nullptr;
  int (*attention)(const EkPrefixAttnArgs*, void*) = nullptr;
  int (*sample)(const EkSampleArgs*, void*) = nullptr;
} api;

[[noreturn]] void refuse(const std::string& why) { throw py::value_error(why); }

void check(int rc, const char* what) {
  if (rc == EK_E_INVALID || rc == EK_E_UNSUPPORTED) refuse(std::string(what) + ": " + api.last_error());
  if (rc != 0)
    throw std::runtime_error(std::string(what) + " failed (code " + std::to_string(rc) + "): " + api.last_error());
}

std::string shape_of(const Tensor& t) {
  std::string s = "(";
  for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
  return s + ")";
}

// A CUDA tensor of one type and rank, on the device of `like`.
const Tensor& need(PyObject* o, const char* name, at::ScalarType type, int64_t dim, const Tensor* like = nullptr) {
  if (!THPVariable_Check(o)) refuse(std::string(name) + ": expected a tensor, got " + Py_TYPE(o)->tp_name);
  const Tensor& t = THPVariable_Unpack(o);
  if (t.layout() != at::kStrided) refuse(std::string(name) + ": must be a dense tensor");
  if (t.scalar_type() != type)
    refuse(std::string(name) + ": dtype " + toString(t.scalar_type()) + ", expected " + toString(type));
  if (t.dim() != dim)
    refuse(std::string(name) + ": " + std::to_string(t.dim()) + "-D, expected " + std::to_string(dim) + "-D");
  if (!t.is_cuda()) refuse(std::string(name) + ": must be a CUDA tensor");
  if (like && t.device() != like->device())
    refuse(std::string(name) + ": on " + t.device().str() + ", expected " + like->device().str());
  if (t.is_neg() || t.is_conj()) refuse(std::string(name) + ": has a pending negation or conjugation");
  if (t.requires_grad() && c10::GradMode::is_enabled())
    refuse(std::string(name) + ": requires grad, but this operator has no backward pass (use torch.no_grad)");
  if (t._fw_grad(0).defined())
    refuse(std::string(name) + ": carries a tangent, but this operator has no forward derivative (use unpack_dual)");
  return t;
}

// The last dimension contiguous, everything else on 16-byte steps.
const Tensor& rows16(const Tensor& t, const char* name) {
  if (t.numel() == 0) return t;
  if (t.size(-1) > 1 && t.stride(-1) != 1) refuse(std::string(name) + ": the last dimension must be contiguous");
  bool ok = reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
  for (int64_t i = 0; i + 1 < t.dim(); ++i)
    ok = ok && (t.size(i) == 1 || t.stride(i) * t.element_size() % 16 == 0);
  if (!ok) refuse(std::string(name) + ": rows must start on 16-byte boundaries");
  return t;
}

// Outputs whose elements share memory (an expanded dimension) are refused.
void no_overlap(const Tensor& t, const char* name) {
  if (t.numel() == 0) return;
  int64_t span = 1;
  bool used[8] = {};
  for (int64_t n = 0; n < t.dim(); ++n) {  // dimensions by rising stride
    int64_t best = -1;
    for (int64_t i = 0; i < t.dim(); ++i)
      if (!used[i] && (best < 0 || t.stride(i) < t.stride(best))) best = i;
    used[best] = true;
    if (t.size(best) == 1) continue;
    if (t.stride(best) < span) refuse(std::string(name) + ": elements overlap in memory");
    span = t.stride(best) * t.size(best);
  }
}

// Counts a write, as torch's in-place operations do: autograd checks the tensors that it saved.
void written(const Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// The bytes of a tensor: start + sum of index * step over its dimensions, neighbouring ones joined.
struct Bytes {
  int64_t start = 0, span = 0;  // addresses start .. start + span - 1; none if span is 0
  int dims = 0;
  int64_t n[9], step[9];

  explicit Bytes(const Tensor& t) {
    if (t.numel() == 0) return;
    start = (int64_t)reinterpret_cast<uintptr_t>(t.data_ptr());
    span = t.element_size();
    n[0] = span, step[0] = 1, dims = 1;
    for (int64_t i = t.dim() - 1; i >= 0; --i) {
      const int64_t size = t.size(i), at = t.stride(i) * (int64_t)t.element_size();
      if (size == 1 || at == 0) continue;
      span += (size - 1) * at;
      if (at == n[dims - 1] * step[dims - 1]) n[dims - 1] *= size;
      else n[dims] = size, step[dims] = at, ++dims;
    }
  }
};

// Whether a sum of d[i] * step[i], lo[i] <= d[i] <= hi[i], steps falling, can give `target`. Gives up with true (the
// call is refused) once `budget` is spent, which rows of ordinary layouts never do.
bool reachable(int64_t target, int dims, const int64_t* step, const int64_t* lo, const int64_t* hi, int& budget) {
  if (dims == 0) return target == 0;
  if (--budget < 0) return true;
  int64_t low = 0, high = 0;  // what the smaller steps can give
  for (int i = 1; i < dims; ++i) low += lo[i] * step[i], high += hi[i] * step[i];
  auto down = [](int64_t a, int64_t b) { return a >= 0 ? a / b : -((-a + b - 1) / b); };
  const int64_t first = std::max(lo[0], -down(high - target, step[0])), last = std::min(hi[0], down(target - low, step[0]));
  for (int64_t d = first; d <= last; ++d)
    if (reachable(target - d * step[0], dims - 1, step + 1, lo + 1, hi + 1, budget)) return true;
  return false;
}

// Whether two tensors have a byte in common. Interleaved ones (K and V of a fused projection) have none.
bool share_memory(const Bytes& a, const Bytes& b) {
  if (!a.span || !b.span || a.start + a.span <= b.start || b.start + b.span <= a.start) return false;
  int64_t step[18], lo[18], hi[18];
  int dims = 0;
  auto add = [&](int64_t s, int64_t from, int64_t to) {  // sorted by falling step, equal steps together
    int i = 0;
    while (i < dims && step[i] > s) ++i;
    if (i == dims || step[i] != s) {
      for (int j = dims++; j > i; --j) step[j] = step[j - 1], lo[j] = lo[j - 1], hi[j] = hi[j - 1];
      step[i] = s, lo[i] = hi[i] = 0;
    }
    lo[i] += from, hi[i] += to;
  };
  for (int i = 0; i < a.dims; ++i) add(a.step[i], 0, a.n[i] - 1);
  for (int i = 0; i < b.dims; ++i) add(b.step[i], 1 - b.n[i], 0);
  int budget = 10000;
  return reachable(b.start - a.start, dims, step, lo, hi, budget);
}

// Different blocks write `a` and read or write `b`, in any order.
void apart(const Bytes& a, const Bytes& b, const char* what) {
  if (share_memory(a, b)) refuse(std::string(what) + " are, in part, the same memory");
}

int64_t step(const Tensor& t, int64_t i) { return t.size(i) > 1 ? t.stride(i) : 0; }

// Descriptor of [batch, row, head, D] rows; a 3-D tensor has no batch.
EkKvTensor describe(const Tensor& data, const Tensor* scales) {
  EkKvTensor r = {};
  const int64_t d = data.dim();
  r.data = data.data_ptr();
  r.stride_batch = d == 4 ? step(data, 0) : 0;
  r.stride_row = step(data, d - 3), r.stride_head = step(data, d - 2);
  if (scales) {
    r.scales = scales->data_ptr();
    r.scale_stride_batch = step(*scales, 0), r.scale_stride_row = step(*scales, 1);
    r.scale_stride_head = step(*scales, 2);
  }
  return r;
}

// Rows [.., row, head, D] that copies of several rows can take: one row shown as many would need a stride of 0.
void distinct_rows(const Tensor& t, const char* name) {
  if (t.size(-3) > 1 && t.stride(-3) == 0) refuse(std::string(name) + ": a row repeated by expand; make it contiguous");
}

int fit32(int64_t n, const char* name) {
  if (n < 0 || n > 0x7fffffff) refuse(std::string(name) + ": size " + std::to_string(n) + " out of range");
  return (int)n;
}

void head_dim_ok(int64_t d) {
  if (d != 64 && d != 128) refuse("head_dim " + std::to_string(d) + " (supported: 64, 128)");
}

double number(py::handle o, const char* name) {
  const double x = PyFloat_AsDouble(o.ptr());
  if (PyErr_Occurred()) {
    PyErr_Clear();
    refuse(std::string(name) + ": expected a number");
  }
  return x;
}

int64_t whole_number(py::handle o, const char* name) {
  PyObject* index = PyNumber_Index(o.ptr());
  const long long x = index ? PyLong_AsLongLong(index) : -1;
  Py_XDECREF(index);
  if (PyErr_Occurred()) {
    PyErr_Clear();
    refuse(std::string(name) + ": expected a whole number of 64 bits");
  }
  return x;
}

void* stream_of(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.device().index()).stream(); }

// (codes, scales) of K and V: an 8-bit cache.
struct Cache {
  const Tensor *kc, *ks, *vc, *vs;
};

Cache take_cache(const py::tuple& t, const char* name, const Tensor* like = nullptr) {
  if (t.size() != 4) refuse(std::string(name) + ": expected KVCacheInt8");
  Cache c;
  c.kc = &rows16(need(t[0].ptr(), "k_codes", at::kChar, 4, like), "k_codes");
  c.ks = &need(t[1].ptr(), "k_scales", at::kBFloat16, 3, c.kc);
  c.vc = &rows16(need(t[2].ptr(), "v_codes", at::kChar, 4, c.kc), "v_codes");
  c.vs = &need(t[3].ptr(), "v_scales", at::kBFloat16, 3, c.kc);
  if (c.vc->sizes() != c.kc->sizes() || c.ks->sizes() != c.kc->sizes().slice(0, 3) ||
      c.vs->sizes() != c.kc->sizes().slice(0, 3))
    refuse(std::string(name) + ": codes " + shape_of(*c.kc) + " / " + shape_of(*c.vc) + " and scales " +
           shape_of(*c.ks) + " / " + shape_of(*c.vs) + " do not match");
  head_dim_ok(c.kc->size(3));
  return c;
}

void check_cache(const py::tuple& t) { take_cache(t, "cache"); }

// What the blocks of a copy write may not meet anything else of the call.
void check_memory(bool write, const Cache& c, const Tensor& k, const Tensor& v, py::handle start) {
  if (write) {
    no_overlap(*c.kc, "k_codes"), no_overlap(*c.ks, "k_scales");
    no_overlap(*c.vc, "v_codes"), no_overlap(*c.vs, "v_scales");
  } else {
    no_overlap(k, "out[0]"), no_overlap(v, "out[1]");
  }
  const Bytes values[2] = {Bytes(k), Bytes(v)}, cache[4] = {Bytes(*c.kc), Bytes(*c.ks), Bytes(*c.vc), Bytes(*c.vs)};
  for (const Bytes& x : values)
    for (const Bytes& y : cache) apart(x, y, write ? "rows and cache" : "out and cache");
  if (write) {
    for (int i = 1; i < 4; ++i)
      for (int j = 0; j < i; ++j) apart(cache[i], cache[j], "tensors of the cache");
  } else {
    apart(values[0], values[1], "out: K and V");
  }
  if (THPVariable_Check(start.ptr())) {
    const Bytes at(THPVariable_Unpack(start.ptr()));
    if (write)
      for (const Bytes& y : cache) apart(at, y, "start and cache");
    else
      for (const Bytes& x : values) apart(at, x, "start and out");
  }
}

// `fresh`: k and v are new outputs, which nothing else shares.
void kv_copy(bool write, bool fresh, const Cache& c, const Tensor& k, const Tensor& v, py::handle start) {
  if (k.sizes() != v.sizes() || k.size(0) != c.kc->size(0) || k.sizes().slice(2) != c.kc->sizes().slice(2))
    refuse("k " + shape_of(k) + " / v " + shape_of(v) + ": expected [batch, rows, kv_heads, head_dim] as in the cache " +
           shape_of(*c.kc));
  EkKvCopyArgs a = {};
  a.k_values = describe(k, nullptr), a.v_values = describe(v, nullptr);
  a.k_cache = describe(*c.kc, c.ks), a.v_cache = describe(*c.vc, c.vs);
  a.batch = fit32(k.size(0), "batch"), a.length = fit32(k.size(1), "rows");
  a.kv_heads = fit32(k.size(2), "kv_heads"), a.head_dim = (int)k.size(3);
  a.capacity = fit32(c.kc->size(1), "cache rows");
  if (THPVariable_Check(start.ptr())) {
    const Tensor& s = need(start.ptr(), "start", at::kInt, 1, c.kc);
    if (s.size(0) != a.batch || !s.is_contiguous())
      refuse("start: expected a contiguous int32 tensor of " + std::to_string(a.batch) + " positions");
    a.start = s.data_ptr<int32_t>();
  } else {
    const int64_t at = whole_number(start, "start");
    if (at < 0 || at > a.capacity - (int64_t)a.length)
      refuse("start: " + std::to_string(a.length) + " rows from " + std::to_string(at) + " on lie outside the cache of " +
             std::to_string(a.capacity) + " rows");
    a.start_all = at;
  }
  if (!fresh) check_memory(write, c, k, v, start);
  if (a.kv_heads == 0 || a.batch == 0 || a.length == 0) return;
  a.device = c.kc->device().index();
  check((write ? api.kv_write : api.kv_read)(&a, stream_of(k)), write ? "ek_kv_write" : "ek_kv_read");
  if (write) written(*c.kc), written(*c.ks), written(*c.vc), written(*c.vs);
  else written(k), written(v);
}

void kv_write(const py::tuple& cache, py::handle ko, py::handle vo, py::handle start) {
  const Cache c = take_cache(cache, "cache");
  const Tensor& k = rows16(need(ko.ptr(), "k", at::kBFloat16, 4, c.kc), "k");
  const Tensor& v = rows16(need(vo.ptr(), "v", at::kBFloat16, 4, c.kc), "v");
  kv_copy(true, false, c, k, v, start);
}

py::tuple kv_read(const py::tuple& cache, py::handle start, py::handle length_o, py::handle out) {
  const Cache c = take_cache(cache, "cache");
  const int64_t length = whole_number(length_o, "length");
  if (length < 0 || (length > c.kc->size(1) && !THPVariable_Check(start.ptr())))  // (before anything is allocated)
    refuse("length " + std::to_string(length) + ": outside the cache of " + std::to_string(c.kc->size(1)) + " rows");
  if (out.is_none()) {
    const Tensor both = at::empty({2, c.kc->size(0), length, c.kc->size(2), c.kc->size(3)}, c.ks->options());
    const Tensor k = both.select(0, 0), v = both.select(0, 1);
    kv_copy(false, true, c, k, v, start);
    return py::make_tuple(k, v);
  }
  const py::sequence pair = py::reinterpret_borrow<py::sequence>(out);
  if (!PySequence_Check(out.ptr()) || THPVariable_Check(out.ptr()) || pair.size() != 2) refuse("out: expected a (k, v) pair");
  const py::object ko = pair[0], vo = pair[1];
  const Tensor& k = rows16(need(ko.ptr(), "out[0]", at::kBFloat16, 4, c.kc), "out[0]");
  const Tensor& v = rows16(need(vo.ptr(), "out[1]", at::kBFloat16, 4, c.kc), "out[1]");
  if (k.size(1) != length) refuse("out: " + std::to_string(k.size(1)) + " rows, expected " + std::to_string(length));
  kv_copy(false, false, c, k, v, start);
  return py::make_tuple(ko, vo);
}

py::object attention(py::handle qo, const py::tuple& prefix, const py::tuple& own, py::handle lens_o,
                     py::handle scale, py::handle max_own_len, py::handle out_o,
                     bool return_lse) {
  const Tensor& q = rows16(need(qo.ptr(), "q", at::kBFloat16, 3), "q");
  const int64_t batch = q.size(0), q_heads = q.size(1), head_dim = q.size(2);
  head_dim_ok(head_dim);
  EkPrefixAttnArgs a = {};
  const Tensor *pk, *ok;
  int64_t prefix_len;
  if (prefix.size() != own.size()) refuse("prefix and own must both be KVCacheInt8 or both (k, v) pairs");
  if (prefix.size() == 4) {
    const Cache p = take_cache(prefix, "prefix", &q), o = take_cache(own, "own", &q);
    if (p.kc->size(0) != 1) refuse("prefix: batch " + std::to_string(p.kc->size(0)) + ", expected 1");
    a.prefix_k = describe(*p.kc, p.ks), a.prefix_v = describe(*p.vc, p.vs);
    a.own_k = describe(*o.kc, o.ks), a.own_v = describe(*o.vc, o.vs);
    distinct_rows(*p.kc, "prefix k_codes"), distinct_rows(*p.vc, "prefix v_codes");
    distinct_rows(*o.kc, "own k_codes"), distinct_rows(*o.vc, "own v_codes");
    pk = p.kc, ok = o.kc;
    prefix_len = pk->size(1);
  } else {
    if (prefix.size() != 2) refuse("prefix and own must be KVCacheInt8 or (k, v) pairs");
    pk = &rows16(need(prefix[0].ptr(), "prefix k", at::kBFloat16, 3, &q), "prefix k");
    const Tensor& pv = rows16(need(prefix[1].ptr(), "prefix v", at::kBFloat16, 3, &q), "prefix v");
    ok = &rows16(need(own[0].ptr(), "own k", at::kBFloat16, 4, &q), "own k");
    const Tensor& ov = rows16(need(own[1].ptr(), "own v", at::kBFloat16, 4, &q), "own v");
    if (pk->sizes() != pv.sizes() || ok->sizes() != ov.sizes()) refuse("k and v must have the same shape");
    a.prefix_k = describe(*pk, nullptr), a.prefix_v = describe(pv, nullptr);
    a.own_k = describe(*ok, nullptr), a.own_v = describe(ov, nullptr);
    distinct_rows(*pk, "prefix k"), distinct_rows(pv, "prefix v");
    distinct_rows(*ok, "own k"), distinct_rows(ov, "own v");
    prefix_len = pk->size(0);
  }
  const int64_t kv_heads = ok->size(2), rows = ok->size(1);
  if (ok->size(0) != batch || pk->sizes().slice(pk->dim() - 2) != ok->sizes().slice(2) || ok->size(3) != head_dim)
    refuse("q " + shape_of(q) + ", prefix " + shape_of(*pk) + ", own " + shape_of(*ok) + ": inconsistent");
  if (kv_heads < 1 || q_heads < 1 || q_heads % kv_heads)
    refuse("q_heads " + std::to_string(q_heads) + " must be a positive multiple of kv_heads " + std::to_string(kv_heads));
  const Tensor& lens = need(lens_o.ptr(), "own_lens", at::kInt, 1, &q);
  if (lens.size(0) != batch || !lens.is_contiguous())
    refuse("own_lens: expected a contiguous int32 tensor of " + std::to_string(batch) + " lengths");
  const int64_t bound = max_own_len.is_none() ? rows : whole_number(max_own_len, "max_own_len");
  if (bound < 0 || bound > rows)
    refuse("max_own_len " + std::to_string(bound) + " outside the " + std::to_string(rows) + " own rows");
  const double s = scale.is_none() ? 1.0 / std::sqrt((double)head_dim) : number(scale, "scale");
  if (!std::isfinite((float)s)) refuse("scale: must be finite");
  Tensor out;
  if (out_o.is_none()) {
    out = at::empty({batch, q_heads, head_dim}, q.options());
  } else {
    out = rows16(need(out_o.ptr(), "out", at::kBFloat16, 3, &q), "out");
    no_overlap(out, "out");
    if (out.sizes() != q.sizes()) refuse("out: " + shape_of(out) + ", expected " + shape_of(q));
    // (q, K and V have been read when the first result is written)
    apart(Bytes(out), Bytes(lens), "out and own_lens");
  }
  Tensor lse;
  if (return_lse) lse = at::empty({batch, q_heads}, q.options().dtype(at::kFloat));
  a.q = q.data_ptr(), a.own_lens = lens.data_ptr<int32_t>(), a.out = out.data_ptr();
  a.q_stride_batch = step(q, 0), a.q_stride_head = step(q, 1);
  a.out_stride_batch = step(out, 0), a.out_stride_head = step(out, 1);
  a.lse = return_lse ? lse.data_ptr<float>() : nullptr;
  a.batch = fit32(batch, "batch"), a.q_heads = fit32(q_heads, "q_heads"), a.kv_heads = fit32(kv_heads, "kv_heads");
  a.head_dim = (int)head_dim;
  a.prefix_len = fit32(prefix_len, "prefix rows"), a.own_capacity = fit32(rows, "own rows");
  a.max_own_len = (int)bound;
  a.scale = (float)s;
  a.device = q.device().index();
  a.workspace_bytes = api.attention_workspace(&a);
  if (a.workspace_bytes < 0) refuse(std::string("shared_prefix_attention: ") + api.last_error());
  Tensor workspace = at::empty({a.workspace_bytes}, q.options().dtype(at::kByte));
  a.workspace = workspace.data_ptr();
  check(api.attention(&a, stream_of(q)), "ek_prefix_attention");
  written(out);
  py::object result = out_o.is_none() ? py::cast(out) : py::reinterpret_borrow<py::object>(out_o);
  if (return_lse) return py::make_tuple(result, lse);
  return result;
}

// A setting given as a number, or as a tensor with one value per row.
template <typename V>
const V* per_row(py::handle o, const char* name, at::ScalarType type, const Tensor& logits) {
  if (!THPVariable_Check(o.ptr())) return nullptr;
  const Tensor& t = need(o.ptr(), name, type, 1, &logits);
  if (t.size(0) != logits.size(0) || !t.is_contiguous())
    refuse(std::string(name) + ": expected a contiguous tensor of " + std::to_string(logits.size(0)) + " values");
  return t.data_ptr<V>();
}

py::object sample(py::handle logits_o, py::handle uniforms_o, py::handle temperature, py::handle top_k,
                  py::handle top_p, py::handle min_p, py::handle out_o, int64_t max_vocab) {
  if (!THPVariable_Check(logits_o.ptr())) refuse(std::string("logits: expected a tensor, got ") + Py_TYPE(logits_o.ptr())->tp_name);
  const bool f32 = THPVariable_Unpack(logits_o.ptr()).scalar_type() == at::kFloat;
  const Tensor& logits = need(logits_o.ptr(), "logits", f32 ? at::kFloat : at::kBFloat16, 2);
  const int64_t batch = logits.size(0), vocab = logits.size(1);
  if (vocab < 1 || vocab > max_vocab)
    refuse("logits: vocabulary " + std::to_string(vocab) + " (1 .. " + std::to_string(max_vocab) + ")");
  if (vocab > 1 && logits.stride(1) != 1) refuse("logits: the last dimension must be contiguous");
  const Tensor& uniforms = need(uniforms_o.ptr(), "uniforms", at::kFloat, 1, &logits);
  if (uniforms.size(0) != batch || !uniforms.is_contiguous())
    refuse("uniforms: expected a contiguous f32 tensor of " + std::to_string(batch) + " numbers");
  EkSampleArgs a = {};
  if (!(a.temperature = per_row<float>(temperature, "temperature", at::kFloat, logits))) {
    const double t = number(temperature, "temperature");
    a.temperature_all = (float)t;
    if (!(t >= 0) || !std::isfinite(a.temperature_all)) refuse("temperature: must be finite and not negative");
    if (t > 0 && a.temperature_all == 0.f) a.temperature_all = 1e-45f;
  }
  if (!(a.top_k = per_row<int32_t>(top_k, "top_k", at::kInt, logits))) {
    const double k = number(top_k, "top_k");
    if (!(k >= 0) || k != std::floor(k)) refuse("top_k: must be a whole number >= 0");
    a.top_k_all = (int32_t)std::min(k, (double)vocab);
  }
  if (!(a.top_p = per_row<float>(top_p, "top_p", at::kFloat, logits))) {
    const double p = number(top_p, "top_p");
    if (!(p >= 0 && p <= 1)) refuse("top_p: must lie in [0, 1]");
    a.top_p_all = (float)p;
  }
  if (!(a.min_p = per_row<float>(min_p, "min_p", at::kFloat, logits))) {
    const double p = number(min_p, "min_p");
    if (!(p >= 0 && p <= 1)) refuse("min_p: must lie in [0, 1]");
    a.min_p_all = (float)p;
  }
  Tensor out;
  if (out_o.is_none()) {
    out = at::empty({batch}, logits.options().dtype(at::kLong));
  } else {
    out = need(out_o.ptr(), "out", at::kLong, 1, &logits);
    if (out.size(0) != batch || !out.is_contiguous())
      refuse("out: expected a contiguous int64 tensor of " + std::to_string(batch) + " tokens");
    const Bytes at(out);
    apart(at, Bytes(logits), "out and logits");
    for (py::handle o : {uniforms_o, temperature, top_k, top_p, min_p})
      if (THPVariable_Check(o.ptr())) apart(at, Bytes(THPVariable_Unpack(o.ptr())), "out and another input");
  }
  a.logits = logits.data_ptr(), a.uniforms = uniforms.data_ptr<float>(), a.tokens = out.data_ptr<int64_t>();
  a.row_stride = batch > 1 ? logits.stride(0) : 0;
  a.logits_f32 = f32;
  a.batch = fit32(batch, "batch"), a.vocab = (int)vocab;
  a.device = logits.device().index();
  check(api.sample(&a, stream_of(logits)), "ek_sample");
  written(out);
  return out_o.is_none() ? py::cast(out) : py::reinterpret_borrow<py::object>(out_o);
}

template <typename F>
void set(F& f, const py::dict& d, const char* name) {
  f = reinterpret_cast<F>(py::cast<uintptr_t>(d[name]));
}

void bind(const py::dict& d) {
  set(api.last_error, d, "ek_last_error");
  set(api.kv_write, d, "ek_kv_write");
  set(api.kv_read, d, "ek_kv_read");
  set(api.attention_workspace, d, "ek_prefix_attention_workspace");
  set(api.attention, d, "ek_prefix_attention");
  set(api.sample, d, "ek_sample");
}

}  // namespace

PYBIND11_MODULE(_ekops, m) {
  m.def("bind", &bind);
  m.def("check_cache", &check_cache);
  m.def("kv_write", &kv_write);
  m.def("kv_read", &kv_read);
  m.def("attention", &attention);
  m.def("sample", &sample);
}
