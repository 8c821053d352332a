// Host side of the serving operators' calls (dsrg_amd/kernels.py): argument checks, output tensors and the C-ABI call in one native
// function each.  One new token's attention, append or draw takes 4 to 6 us on the GPU; the same checks in Python and a call through
// ctypes took 11 to 13 us a call, so a loop that is not captured into a graph waited for its host.  Nothing is computed here.
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <ATen/ops/empty.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/GradMode.h>
#include <c10/hip/HIPStream.h>
#include <algorithm>
#include <climits>
#include <cstdarg>
#include <stdexcept>
#include "../../include/dsrg_hip.h"

namespace {

PyObject* g_error = nullptr;            // dsrg_amd._lib.DsrgHipError

struct Api {                            // libdsrg_hip.so's entry points, handed over by dsrg_amd._lib (which loads the library)
  decltype(&dsrg_last_error) last_error;
  decltype(&dsrg_kv_append) append;
  decltype(&dsrg_kv_read) read;
  decltype(&dsrg_attention_paged_workspace) workspace;
  decltype(&dsrg_attention_paged) attention;
  decltype(&dsrg_sample_rows) sample;
} g_api;

struct Refusal : std::runtime_error { using std::runtime_error::runtime_error; };
struct Pending : std::exception {};     // a Python error is set already

[[noreturn]] __attribute__((format(printf, 1, 2))) void refuse(const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof buf, fmt, ap);
  va_end(ap);
  throw Refusal(buf);
}

std::string shape_of(const at::Tensor& t) {
  std::string s = "(";
  for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
  return s + ")";
}

const at::Tensor& tensor(const char* what, const char* name, PyObject* o) {
  if (!THPVariable_Check(o)) refuse("%s: %s must be a tensor", what, name);
  return THPVariable_Unpack(o);
}

void on_device(const char* what, const at::Tensor& t) {
  if (!t.is_cuda()) refuse("dsrg_amd kernels need device tensors (%s got %s); there is no CPU path", what, t.device().str().c_str());
}

// These operators have no backward: what asks for a gradient is refused, since its gradient would be lost without a word
void no_grad(const char* what, const char* name, const at::Tensor& t) {
  if (c10::GradMode::is_enabled() && t.requires_grad())
    refuse("%s has no backward and %s asks for a gradient: detach it, or call under torch.no_grad()", what, name);
}

int io_dtype(const char* what, at::ScalarType t) {
  if (t == at::kFloat) return DSRG_F32;
  if (t == at::kBFloat16) return DSRG_BF16;
  refuse("%s: unsupported dtype %s (float32 / bfloat16 only)", what, c10::toString(t));
}

int as_int(const char* what, const char* name, PyObject* o) {
  const long v = PyLong_AsLong(o);
  if (v == -1 && PyErr_Occurred()) throw Pending();
  if (v > INT_MAX || v < INT_MIN) refuse("%s: %s = %ld", what, name, v);
  return (int)v;
}
double as_double(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw Pending();
  return v;
}
bool as_bool(PyObject* o) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) throw Pending();
  return v;
}
int fits(const char* what, int64_t v) {
  if (v > INT_MAX || v < INT_MIN) refuse("%s: a size or stride of %lld", what, (long long)v);
  return (int)v;
}

struct Cache { dsrg_kv_cache_t c; int H, D; at::Device dev; };

Cache cache_of(const char* what, PyObject* ko, PyObject* vo, PyObject* kso, PyObject* vso) {
  const at::Tensor &k = tensor(what, "k_pool", ko), &v = tensor(what, "v_pool", vo);
  no_grad(what, "k_pool", k);
  no_grad(what, "v_pool", v);
  on_device(what, k);
  const at::ScalarType st = k.scalar_type();
  const int dt = st == at::kBFloat16 ? DSRG_BF16 : st == at::kFloat ? DSRG_F32 : st == at::kChar ? DSRG_I8 : st == at::kFloat8_e4m3fn ? DSRG_E4M3 : -1;
  const int64_t e = dt == DSRG_F32 ? 4 : 8;
  if (dt < 0 || k.dim() != 6 || k.size(4) != 16 || k.size(5) != e) refuse("%s: k_pool %s %s is no cache (kv_pool_shapes)", what, c10::toString(st), shape_of(k).c_str());
  const int64_t P = k.size(0), H = k.size(1), S = k.size(2) * 16, D = k.size(3) * e;
  const bool vs = dt == DSRG_F32 ? v.sizes() == at::IntArrayRef({P, H, S / 16, D / 16, 4, 16, 4}) : v.sizes() == at::IntArrayRef({P, H, S / 32, D / 16, 4, 16, 2, 4});
  if (!vs || v.scalar_type() != st || !k.is_contiguous() || !v.is_contiguous() || v.device() != k.device())
    refuse("%s: pools must be contiguous, of one dtype and of the shapes of kv_pool_shapes (got %s, %s)", what, shape_of(k).c_str(), shape_of(v).c_str());
  float* scale[2] = {nullptr, nullptr};
  if (dt >= DSRG_I8) {
    PyObject* so[2] = {kso, vso};
    for (int i = 0; i < 2; ++i) {
      const bool given = so[i] != Py_None;
      if (given) {
        const at::Tensor& s = tensor(what, "scale", so[i]);
        no_grad(what, i ? "v_scale" : "k_scale", s);
        if (s.scalar_type() == at::kFloat && s.sizes() == at::IntArrayRef({P, H, S}) && s.is_contiguous() && s.device() == k.device()) { scale[i] = s.data_ptr<float>(); continue; }
      }
      refuse("%s: an 8-bit cache needs k_scale and v_scale, contiguous fp32 [pages, kv heads, page size]", what);
    }
  } else if (kso != Py_None || vso != Py_None) refuse("%s: only 8-bit caches have scales", what);
  Cache r{{k.data_ptr(), v.data_ptr(), scale[0], scale[1], fits(what, P), fits(what, S), fits(what, H), fits(what, D), dt, 0}, (int)H, (int)D, k.device()};
  return r;
}

struct Table { const int32_t* p; int ld, width; };

Table table_of(const char* what, PyObject* o, at::Device dev, int64_t B) {
  const at::Tensor& t = tensor(what, "the page table", o);
  if (t.scalar_type() != at::kInt || t.dim() != 2 || t.size(0) != B || t.size(1) < 1 || (t.stride(1) != 1 && t.size(1) > 1) || t.device() != dev)
    refuse("%s: the page table must be int32 [B, pages] with contiguous rows beside the cache", what);
  const int width = fits(what, t.size(1));
  return Table{t.data_ptr<int32_t>(), B > 1 ? fits(what, t.stride(0)) : width, width};
}

const int32_t* ints_of(const char* what, const char* name, PyObject* o, at::Device dev, int64_t B) {
  const at::Tensor& t = tensor(what, name, o);
  if (t.scalar_type() != at::kInt || t.dim() != 1 || t.size(0) != B || !t.is_contiguous() || t.device() != dev)
    refuse("%s: %s must be contiguous int32 [B] beside the cache", what, name);
  return t.data_ptr<int32_t>();
}

// [B, N, W] as it is if its rows are contiguous and 16-byte aligned, else a copy
struct Rows {
  at::Tensor t;
  int64_t bs;
  int rs;
  Rows(const char* what, const at::Tensor& x) : t(x) {
    const int64_t n = 16 / x.element_size(), W = x.size(2);
    if ((x.stride(2) != 1 && W > 1) || (uintptr_t)x.data_ptr() % 16 || (x.stride(0) % n && x.size(0) > 1) || (x.stride(1) % n && x.size(1) > 1))
      t = x.detach().clone(at::MemoryFormat::Contiguous);
    rs = fits(what, t.size(1) > 1 ? t.stride(1) : W);
    bs = t.size(0) > 1 ? t.stride(0) : t.size(1) * (int64_t)rs;
  }
};

void* stream_of(at::Device dev) { return c10::hip::getCurrentHIPStream(dev.index()).stream(); }

void done(int rc, const char* what) {
  if (rc != DSRG_OK) refuse("%s failed (%d): %s", what, rc, g_api.last_error());
}

// f's exceptions become Python's: a refusal is a DsrgHipError, torch's own (out of memory among them) keep their classes.
template <typename F> PyObject* guarded(F&& f) {
  HANDLE_TH_ERRORS
  try {
    return f();
  } catch (const Pending&) {
    return nullptr;
  } catch (const Refusal& e) {
    PyErr_SetString(g_error ? g_error : PyExc_RuntimeError, e.what());
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

void arity(const char* what, Py_ssize_t n, Py_ssize_t want) {
  if (n != want) refuse("%s: %zd arguments, %zd wanted", what, n, want);
  if (!g_api.append) refuse("%s: the kernel library is not loaded", what);
}

PyObject* init(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    if (n != 7) refuse("init: %zd arguments", n);
    void* p[6];
    for (int i = 0; i < 6; ++i) {
      p[i] = PyLong_AsVoidPtr(a[i + 1]);
      if (!p[i]) { if (PyErr_Occurred()) throw Pending(); refuse("init: NULL entry point"); }
    }
    Py_INCREF(a[0]);
    Py_XDECREF(g_error);
    g_error = a[0];
    g_api.last_error = (decltype(g_api.last_error))p[0];
    g_api.append = (decltype(g_api.append))p[1];
    g_api.read = (decltype(g_api.read))p[2];
    g_api.workspace = (decltype(g_api.workspace))p[3];
    g_api.attention = (decltype(g_api.attention))p[4];
    g_api.sample = (decltype(g_api.sample))p[5];
    Py_RETURN_NONE;
  });
}

// (k, v, k_pool, v_pool, table, start, count, k_scale, v_scale)
PyObject* kv_append(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    const char* what = "kv_append";
    arity(what, n, 9);
    const at::Tensor &k = tensor(what, "k", a[0]), &v = tensor(what, "v", a[1]);
    no_grad(what, "k", k);
    no_grad(what, "v", v);
    const Cache c = cache_of(what, a[2], a[3], a[7], a[8]);
    const int64_t W = (int64_t)c.H * c.D;
    if (k.dim() != 3 || k.size(2) != W || v.sizes() != k.sizes() || v.scalar_type() != k.scalar_type() || k.device() != c.dev || v.device() != c.dev)
      refuse("kv_append: k and v must be [B, T, %lld] of one dtype beside the cache (got %s, %s)", (long long)W, shape_of(k).c_str(), shape_of(v).c_str());
    const int dt = io_dtype(what, k.scalar_type()), B = fits(what, k.size(0)), T = fits(what, k.size(1));
    const Table t = table_of(what, a[4], c.dev, B);
    const int32_t* start = ints_of(what, "start", a[5], c.dev, B);
    const int32_t* count = a[6] == Py_None ? nullptr : ints_of(what, "count", a[6], c.dev, B);
    const c10::DeviceGuard guard(c.dev);
    const Rows kr(what, k), vr(what, v);
    done(g_api.append(&c.c, kr.t.data_ptr(), kr.bs, kr.rs, vr.t.data_ptr(), vr.bs, vr.rs, dt, t.p, t.ld, t.width, start, count, B, T, stream_of(c.dev)), "dsrg_kv_append");
    Py_RETURN_NONE;
  });
}

// (k_pool, v_pool, table, start, count, n, k_scale, v_scale, dtype)
PyObject* kv_read(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    const char* what = "kv_read";
    arity(what, n, 9);
    const Cache c = cache_of(what, a[0], a[1], a[6], a[7]);
    at::ScalarType st = c.c.dtype == DSRG_F32 ? at::kFloat : at::kBFloat16;
    if (a[8] != Py_None) {
      if (!THPDtype_Check(a[8])) refuse("kv_read: dtype must be a torch.dtype");
      st = reinterpret_cast<THPDtype*>(a[8])->scalar_type;
    }
    const int dt = io_dtype(what, st), N = as_int(what, "n", a[5]);
    const at::Tensor& tt = tensor(what, "the page table", a[2]);
    const int B = tt.dim() == 2 ? fits(what, tt.size(0)) : -1;
    const Table t = table_of(what, a[2], c.dev, B);
    const int32_t *start = ints_of(what, "start", a[3], c.dev, B), *count = ints_of(what, "count", a[4], c.dev, B);
    if (N < 0) refuse("kv_read: n = %d", N);
    const c10::DeviceGuard guard(c.dev);
    const int64_t W = (int64_t)c.H * c.D;
    const auto opt = at::TensorOptions().dtype(st).device(c.dev);
    at::Tensor k = at::empty({B, N, W}, opt), v = at::empty({B, N, W}, opt);
    done(g_api.read(&c.c, k.data_ptr(), N * W, fits(what, W), v.data_ptr(), N * W, fits(what, W), dt, t.p, t.ld, t.width, start, count, B, N, stream_of(c.dev)), "dsrg_kv_read");
    PyObject *pk = THPVariable_Wrap(std::move(k)), *pv = THPVariable_Wrap(std::move(v));
    PyObject* r = pk && pv ? PyTuple_Pack(2, pk, pv) : nullptr;
    Py_XDECREF(pk);
    Py_XDECREF(pv);
    return r;
  });
}

// (q, k_pool, v_pool, table, lens, nh, k_scale, v_scale, scale, causal, window, want_lse)
PyObject* attention_paged(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    const char* what = "attention_paged";
    arity(what, n, 12);
    const at::Tensor& q = tensor(what, "q", a[0]);
    no_grad(what, "q", q);
    const Cache c = cache_of(what, a[1], a[2], a[6], a[7]);
    const int nh = as_int(what, "nh", a[5]);
    if (q.dim() != 3 || nh < 1 || nh % c.H || q.size(2) != (int64_t)nh * c.D || q.device() != c.dev)
      refuse("attention_paged: q %s is not [B, Nq, nh * %d] with nh = %d a multiple of %d, beside the cache", shape_of(q).c_str(), c.D, nh, c.H);
    const int dt = io_dtype(what, q.scalar_type()), B = fits(what, q.size(0)), Nq = fits(what, q.size(1)), W = fits(what, q.size(2));
    const Table t = table_of(what, a[3], c.dev, B);
    const int32_t* lens = ints_of(what, "lens", a[4], c.dev, B);
    const double scale = a[8] == Py_None ? (c.D == 64 ? 0.125 : 0.08838834764831845) : as_double(a[8]);
    const bool causal = as_bool(a[9]), want_lse = as_bool(a[11]);
    const int window = as_int(what, "window", a[10]);
    const c10::DeviceGuard guard(c.dev);
    const Rows qr(what, q);
    const auto opt = at::TensorOptions().device(c.dev);
    at::Tensor o = at::empty({B, Nq, W}, opt.dtype(q.scalar_type())), lse, ws;
    if (want_lse) lse = at::empty({B, nh, Nq}, opt.dtype(at::kFloat));
    const int64_t need = g_api.workspace(&c.c, t.width, B, nh, Nq, window);
    if (need < 0) done((int)need, "dsrg_attention_paged_workspace");
    if (need) ws = at::empty({need}, opt.dtype(at::kByte));
    done(g_api.attention(&c.c, qr.t.data_ptr(), qr.bs, qr.rs, o.data_ptr(), (int64_t)Nq * W, W, want_lse ? lse.data_ptr<float>() : nullptr, t.p, t.ld, t.width, lens, B, nh, Nq,
                         (float)scale, causal, window, need ? ws.data_ptr() : nullptr, need, dt, stream_of(c.dev)), "dsrg_attention_paged");
    PyObject* po = THPVariable_Wrap(std::move(o));
    if (!want_lse || !po) return po;
    PyObject* pl = THPVariable_Wrap(std::move(lse));
    PyObject* r = pl ? PyTuple_Pack(2, po, pl) : nullptr;
    Py_DECREF(po);
    Py_XDECREF(pl);
    return r;
  });
}

// (logits, u, temperature, top_k, top_p, min_p)
PyObject* sample_rows(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    const char* what = "sample_rows";
    arity(what, n, 6);
    static const char* const names[4] = {"temperature", "top_k", "top_p", "min_p"};
    const at::Tensor &x = tensor(what, "logits", a[0]), &u = tensor(what, "u", a[1]);
    no_grad(what, "logits", x);
    no_grad(what, "u", u);
    for (int i = 0; i < 4; ++i)
      if (THPVariable_Check(a[2 + i])) no_grad(what, names[i], THPVariable_Unpack(a[2 + i]));
    on_device(what, x);
    if (x.dim() != 2 || x.size(1) < 1 || (x.stride(1) != 1 && x.size(1) > 1)) refuse("sample_rows: logits must be [B,V] with contiguous rows (got %s)", shape_of(x).c_str());
    const int dt = io_dtype(what, x.scalar_type()), B = fits(what, x.size(0)), V = fits(what, x.size(1));
    const at::Device dev = x.device();
    if (u.scalar_type() != at::kFloat || u.dim() != 1 || u.size(0) != B || !u.is_contiguous() || u.device() != dev) refuse("sample_rows: u must be contiguous fp32 [B] beside the logits");
    const void* p[4];
    double num[4];
    int k0 = 0;
    for (int i = 0; i < 4; ++i) {
      PyObject* o = a[2 + i];
      p[i] = nullptr;
      num[i] = 0;
      if (THPVariable_Check(o)) {
        const at::Tensor& t = THPVariable_Unpack(o);
        if (t.scalar_type() != (i == 1 ? at::kInt : at::kFloat) || t.dim() != 1 || t.size(0) != B || !t.is_contiguous() || t.device() != dev)
          refuse("sample_rows: %s must be a number or contiguous %s [B] beside the logits", names[i], i == 1 ? "int32" : "fp32");
        p[i] = B ? t.data_ptr() : nullptr;
      } else if (i == 1) k0 = std::max(as_int(what, names[i], o), 0);          // (below 0 is "off" here, or the largest entry, as 0 is in the C-ABI)
      else {
        num[i] = as_double(o);
        if (i != 2 && num[i] < 0) num[i] = 0;
      }
    }
    const c10::DeviceGuard guard(dev);
    const auto opt = at::TensorOptions().device(dev);
    at::Tensor token = at::empty({B}, opt.dtype(at::kLong)), logp = at::empty({B}, opt.dtype(at::kFloat));
    done(g_api.sample(x.data_ptr(), B > 1 ? x.stride(0) : V, dt, u.data_ptr<float>(), (const float*)p[0], (float)num[0], (const int32_t*)p[1], k0, (const float*)p[2], (float)num[2],
                      (const float*)p[3], (float)num[3], token.data_ptr<int64_t>(), logp.data_ptr<float>(), B, V, stream_of(dev)), "dsrg_sample_rows");
    PyObject *pt = THPVariable_Wrap(std::move(token)), *pl = THPVariable_Wrap(std::move(logp));
    PyObject* r = pt && pl ? PyTuple_Pack(2, pt, pl) : nullptr;
    Py_XDECREF(pt);
    Py_XDECREF(pl);
    return r;
  });
}

template <PyObject* (*F)(PyObject*, PyObject* const*, Py_ssize_t)> PyCFunction fast() { return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(F)); }

PyMethodDef methods[] = {{"init", fast<init>(), METH_FASTCALL, "(error class, addresses of the C-ABI's entry points)"},
                         {"kv_append", fast<kv_append>(), METH_FASTCALL, nullptr},
                         {"kv_read", fast<kv_read>(), METH_FASTCALL, nullptr},
                         {"attention_paged", fast<attention_paged>(), METH_FASTCALL, nullptr},
                         {"sample_rows", fast<sample_rows>(), METH_FASTCALL, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_dsrg_bind", "native host side of the serving operators", -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__dsrg_bind() { return PyModule_Create(&module); }
