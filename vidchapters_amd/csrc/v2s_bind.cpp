// Native argument path of the 8-bit decoding calls (lib.py): operands are looked at and the argument structs of include/vid2seq_hip.h filled here.
// A decode step is a chain of launches of a few microseconds, and a launch alone costs the host 3 us.  Reading shapes, strides, types and addresses of six
// to eight tensors from Python added as much again: a call through ctypes took 4.7 (dequant_q8), 6.1 (gemm_q8), 8.0 (kv_append_q8) us of host time, from
// here 3.4, 3.4 and 4.0.
// The library is not linked: lib.py hands over the addresses of its functions, and attach() checks that both were built from one header.
#include <torch/csrc/autograd/python_variable.h>
#include <exception>
#include <stdexcept>
#include <string>
#include "../../include/vid2seq_hip.h"

namespace {

struct Raised {};                                     // a Python error is set

[[noreturn]] void raise(PyObject* type, const std::string& what) { PyErr_SetString(type, what.c_str()); throw Raised(); }

decltype(&v2s_quant_rows_q8) f_quant;
decltype(&v2s_rmsnorm_q8) f_norm;
decltype(&v2s_dequant_q8) f_dequant;
decltype(&v2s_gemm_q8) f_gemm;
decltype(&v2s_kv_append_q8) f_append;
decltype(&v2s_kv_read_q8) f_read;
decltype(&v2s_decode_attn_q8) f_attn;
decltype(&v2s_sample_step) f_sample;
PyObject *current_device, *raw_stream;                // of torch

int64_t integer(PyObject* o) {
  const int64_t v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw Raised();
  return v;
}
int32_t small(PyObject* o, const char* name) {
  const int64_t v = integer(o);
  if (v != (int32_t)v) raise(PyExc_ValueError, std::string(name) + " does not fit 32 bits");
  return (int32_t)v;
}
int64_t given_stride(PyObject* o) {                   // 0: not given
  const int64_t v = o == Py_None ? 0 : integer(o);
  if (v > INT32_MAX) raise(PyExc_ValueError, "a row stride does not fit 32 bits");
  return v;
}
double number(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw Raised();
  return v;
}

// Elements of a tensor that lie one behind the other from its first one on, and the dimension next to them as rows (none: one row)
struct Layout { int64_t run = 1, rows = 1, stride = -1; };
Layout layout_of(const at::Tensor& t) {
  Layout l;
  int64_t d = t.dim() - 1;
  for (; d >= 0; --d) {
    if (t.size(d) == 1) continue;
    if (t.stride(d) != l.run) break;
    l.run *= t.size(d);
  }
  for (; d >= 0; --d) {
    if (t.size(d) == 1) continue;
    if (l.stride < 0) { l.rows = t.size(d); l.stride = t.stride(d); }
    else if (t.stride(d) == l.rows * l.stride) l.rows *= t.size(d);
    else break;
  }
  return l;
}

// The operands of one call: all on the current device, on whose current stream the launch goes out.
struct Call {
  const char* name;
  int64_t device = -2;                                // not looked up yet
  const char* elsewhere = nullptr;                    // an operand that is not on the GPU: said when every operand has been looked at

  const at::Tensor& tensor(PyObject* o, const char* arg) const {
    if (!THPVariable_Check(o)) raise(PyExc_TypeError, label(arg) + ": a tensor is expected");
    return THPVariable_Unpack(o);
  }
  std::string label(const char* arg) const { return std::string(name) + " " + arg; }
  // address of an operand of this type with `need` elements of storage from its first one on
  void* at_least(const at::Tensor& t, at::ScalarType type, int64_t need, const char* arg) {
    if (t.dim() > 0 && t.size(-1) > 1 && t.stride(-1) != 1) raise(PyExc_ValueError, label(arg) + ": the last dimension must be contiguous");
    if (t.scalar_type() != type)
      raise(PyExc_RuntimeError, label(arg) + ": expected dtype " + c10::toString(type) + ", got " + c10::toString(t.scalar_type()));
    const int64_t have = (int64_t)(t.storage().nbytes() / t.element_size()) - t.storage_offset();
    if (have < need)
      raise(PyExc_ValueError, label(arg) + ": " + std::to_string(need) + " elements are read or written, the tensor's storage holds " + std::to_string(have));
    if (!t.is_cuda()) {
      if (!elsewhere) elsewhere = arg;
      return nullptr;
    }
    if (device < 0) {
      PyObject* d = PyObject_CallNoArgs(current_device);
      if (!d) throw Raised();
      device = PyLong_AsLongLong(d);
      Py_DECREF(d);
    }
    if (t.get_device() != device)
      raise(PyExc_RuntimeError, label(arg) + ": tensor lives on cuda:" + std::to_string(t.get_device()) + ", the launch goes to cuda:" + std::to_string(device));
    return t.data_ptr();
  }
  void* operand(PyObject* o, at::ScalarType type, int64_t need, const char* arg) { return at_least(tensor(o, arg), type, need, arg); }
  // `need` numbers that lie one behind the other
  void* vector(const at::Tensor& t, at::ScalarType type, int64_t need, const char* arg) {
    if (!t.is_contiguous() && layout_of(t).run < need)
      raise(PyExc_ValueError, label(arg) + ": " + std::to_string(need) + " elements are expected one behind the other (contiguous) in its storage");
    return at_least(t, type, need, arg);
  }
  void* vector(PyObject* o, at::ScalarType type, int64_t need, const char* arg) { return vector(tensor(o, arg), type, need, arg); }
  void* optional(PyObject* o, at::ScalarType type, int64_t need, const char* arg) { return o == Py_None ? nullptr : vector(o, type, need, arg); }
  // Rows of `cols` elements, ld apart.  A stride of 0 stands for the tensor's own: the rows of a tensor that has so many, each of `cols` elements or more; else
  // rows laid end to end, if so many elements lie one behind the other.
  void* matrix(const at::Tensor& t, at::ScalarType type, int64_t rows, int64_t cols, int64_t& ld, const char* arg) {
    if (ld == 0) {
      ld = cols;
      const bool whole = t.is_contiguous(), wide = t.dim() > 1 && cols > 0 && t.size(-1) > cols;
      if (!whole || wide) {
        const Layout l = whole ? Layout{t.size(-1), t.numel() / t.size(-1), t.size(-1)} : layout_of(t);
        if (rows > 1 && l.run >= cols && l.rows >= rows) ld = l.stride;
        else if (!whole && l.run < rows * cols)
          raise(PyExc_ValueError, label(arg) + ": " + std::to_string(rows) + " rows of " + std::to_string(cols) + " elements at one distance are expected; give their stride");
      }
      if (ld > INT32_MAX) raise(PyExc_ValueError, "a row stride does not fit 32 bits");
    }
    return at_least(t, type, (rows - 1) * ld + cols, arg);
  }
  void* matrix(PyObject* o, at::ScalarType type, int64_t rows, int64_t cols, int64_t& ld, const char* arg) { return matrix(tensor(o, arg), type, rows, cols, ld, arg); }
  void* optional_matrix(PyObject* o, at::ScalarType type, int64_t rows, int64_t cols, int64_t& ld, const char* arg) {
    return o == Py_None ? nullptr : matrix(o, type, rows, cols, ld, arg);
  }
  void* stream() const {
    if (elsewhere) raise(PyExc_RuntimeError, label(elsewhere) + ": tensor must live on the GPU (HIP path has no CPU fallback)");
    PyObject* d = PyLong_FromLongLong(device);
    PyObject* s = d ? PyObject_CallOneArg(raw_stream, d) : nullptr;
    Py_XDECREF(d);
    if (!s) throw Raised();
    void* p = PyLong_AsVoidPtr(s);
    Py_DECREF(s);
    if (!p && PyErr_Occurred()) throw Raised();
    return p;
  }
  // sizes of codes [entries][heads][maxlen][64] and scales [entries][heads][maxlen] of keys and of values; then their addresses
  v2s_kv_q8 cache(PyObject* const* a) {
    const at::Tensor &kq = tensor(a[0], "kq"), &ks = tensor(a[1], "ks"), &vq = tensor(a[2], "vq"), &vs = tensor(a[3], "vs");
    const auto rows = ks.sizes();
    const auto codes_of = [&](const at::Tensor& t) { return t.dim() == 4 && t.sizes().slice(0, 3) == rows && t.size(3) == 64; };
    if (rows.size() != 3 || vs.sizes() != rows || !codes_of(kq) || !codes_of(vq))
      raise(PyExc_ValueError, std::string(name) + ": a cache is codes [entries, heads, maxlen, 64] and scales [entries, heads, maxlen] for keys and for values");
    const int64_t e = ks.stride(0), h = ks.stride(1);
    const auto rows_of = [&](const at::Tensor& t) { return t.stride(0) == e * 64 && t.stride(1) == h * 64 && t.stride(2) == 64 && t.stride(3) == 1; };
    if (ks.stride(2) != 1 || vs.strides() != ks.strides() || !rows_of(kq) || !rows_of(vq))
      raise(PyExc_ValueError, std::string(name) + ": codes and scales of a cache share their row strides, the rows of a head are contiguous");
    if (rows[0] > INT32_MAX || rows[1] > INT32_MAX || rows[2] > INT32_MAX) raise(PyExc_ValueError, std::string(name) + ": the cache is too large");
    v2s_kv_q8 c = {};
    c.e_rows = e; c.h_rows = h; c.entries = (int32_t)rows[0]; c.heads = (int32_t)rows[1]; c.maxlen = (int32_t)rows[2];
    return c;
  }
  void locate(v2s_kv_q8& c, PyObject* const* a) {     // the views cover what is read and written
    c.k = (int8_t*)operand(a[0], at::kChar, 0, "kq"); c.ks = (float*)operand(a[1], at::kFloat, 0, "ks");
    c.v = (int8_t*)operand(a[2], at::kChar, 0, "vq"); c.vs = (float*)operand(a[3], at::kFloat, 0, "vs");
  }
};

// the library's call, other Python threads run meanwhile (a launch waits where the device's queue is full)
template <class F, class... A> PyObject* launch(F f, A... a) {
  PyThreadState* state = PyEval_SaveThread();
  const int rc = f(a...);
  PyEval_RestoreThread(state);
  return PyLong_FromLong(rc);
}

// x q scale rows cols ldx ldq
PyObject* quant_rows_q8(PyObject* const* a) {
  Call c{"quant_rows_q8"};
  const at::Tensor& x = c.tensor(a[0], "x");
  const bool f32 = x.scalar_type() == at::kFloat;
  const int32_t rows = small(a[3], "rows"), cols = small(a[4], "cols");
  int64_t ldx = given_stride(a[5]), ldq = given_stride(a[6]);
  void* px = c.matrix(x, f32 ? at::kFloat : at::kBFloat16, rows, cols, ldx, "x");
  void *pq = c.matrix(a[1], at::kChar, rows, cols, ldq, "q"), *ps = c.vector(a[2], at::kFloat, rows, "scale");
  return launch(f_quant, px, f32 ? V2S_F32 : V2S_BF16, ldx, (int8_t*)pq, ldq, (float*)ps, rows, cols, c.stream());
}

// x w q scale rows cols eps delta h ldx ldd ldh ldq
PyObject* rmsnorm_q8(PyObject* const* a) {
  Call c{"rmsnorm_q8"};
  const int32_t rows = small(a[4], "rows"), cols = small(a[5], "cols");
  int64_t ldx = given_stride(a[9]), ldd = given_stride(a[10]), ldh = given_stride(a[11]), ldq = given_stride(a[12]);
  void *x = c.matrix(a[0], at::kBFloat16, rows, cols, ldx, "x"), *w = c.vector(a[1], at::kFloat, cols, "w");
  void *d = c.optional_matrix(a[7], at::kBFloat16, rows, cols, ldd, "delta"), *h = c.optional_matrix(a[8], at::kBFloat16, rows, cols, ldh, "h");
  void *q = c.matrix(a[2], at::kChar, rows, cols, ldq, "q"), *s = c.vector(a[3], at::kFloat, rows, "scale");
  return launch(f_norm, x, ldx, d, ldd, (float*)w, h, ldh, (int8_t*)q, ldq, (float*)s, rows, cols, (float)number(a[6]), c.stream());
}

// q scale y rows cols ldq ldy
PyObject* dequant_q8(PyObject* const* a) {
  Call c{"dequant_q8"};
  const int32_t rows = small(a[3], "rows"), cols = small(a[4], "cols");
  int64_t ldq = given_stride(a[5]), ldy = given_stride(a[6]);
  void *q = c.matrix(a[0], at::kChar, rows, cols, ldq, "q"), *s = c.vector(a[1], at::kFloat, rows, "scale");
  void* y = c.matrix(a[2], at::kBFloat16, rows, cols, ldy, "y");
  return launch(f_dequant, (int8_t*)q, ldq, (float*)s, y, ldy, rows, cols, c.stream());
}

// A B sA sB C M N K lda ldb ldc alpha bias act residual ldr
PyObject* gemm_q8(PyObject* const* a) {
  Call c{"gemm_q8"};
  v2s_gemm_q8_args g = {};
  const at::Tensor& out = c.tensor(a[4], "C");
  const bool f32 = out.scalar_type() == at::kFloat;
  g.M = small(a[5], "M"); g.N = small(a[6], "N"); g.K = small(a[7], "K");
  g.lda = given_stride(a[8]); g.ldb = given_stride(a[9]); g.ldc = given_stride(a[10]); g.ldr = given_stride(a[15]);
  g.A = (int8_t*)c.matrix(a[0], at::kChar, g.M, g.K, g.lda, "A"); g.B = (int8_t*)c.matrix(a[1], at::kChar, g.N, g.K, g.ldb, "B");
  g.sA = (float*)c.vector(a[2], at::kFloat, g.M, "sA"); g.sB = (float*)c.vector(a[3], at::kFloat, g.N, "sB");
  g.C = c.matrix(out, f32 ? at::kFloat : at::kBFloat16, g.M, g.N, g.ldc, "C");
  g.c_dtype = f32 ? V2S_F32 : V2S_BF16; g.alpha = (float)number(a[11]); g.act = small(a[13], "act");
  g.bias = (float*)c.optional(a[12], at::kFloat, g.N, "bias");
  g.residual = c.optional_matrix(a[14], at::kBFloat16, g.M, g.N, g.ldr, "residual");
  return launch(f_gemm, &g, c.stream());
}

// k v kq ks vq vs T pos0 pos pos_dev count
template <class F> PyObject* kv_move(const char* name, F f, PyObject* const* a) {
  Call c{name};
  v2s_kv_q8 cache = c.cache(a + 2);
  const at::Tensor &k = c.tensor(a[0], "k"), &v = c.tensor(a[1], "v");
  const int32_t T = small(a[6], "T"), E = cache.entries;
  const int64_t cols = (int64_t)cache.heads * 64;
  if (k.dim() != 3 || v.sizes() != k.sizes() || k.size(0) != E || k.size(1) < T || k.size(2) < cols || v.strides() != k.strides())
    raise(PyExc_ValueError, std::string(name) + ": k and v are [" + std::to_string(E) + ", >= " + std::to_string(T) + ", >= " + std::to_string(cols) +
                                "] with the same strides");
  c.locate(cache, a + 2);
  void *pk = c.at_least(k, at::kBFloat16, 0, "k"), *pv = c.at_least(v, at::kBFloat16, 0, "v");
  const auto *pos = (int32_t*)c.optional(a[8], at::kInt, E, "pos"), *ctr = (int32_t*)c.optional(a[9], at::kInt, 1, "pos_dev"),
             *count = (int32_t*)c.optional(a[10], at::kInt, E, "count");
  return launch(f, &cache, pk, pv, k.stride(0), k.stride(1), T, small(a[7], "pos0"), pos, ctr, count, c.stream());
}
PyObject* kv_append_q8(PyObject* const* a) { return kv_move("kv_append_q8", f_append, a); }
PyObject* kv_read_q8(PyObject* const* a) { return kv_move("kv_read_q8", f_read, a); }

// q kq ks vq vs o Nk group klen pos_dev bias_maxlen bias_row key_mask scale workspace
PyObject* decode_attn_q8(PyObject* const* a) {
  Call c{"decode_attn_q8"};
  v2s_decode_attn_q8_args d = {};
  d.cache = c.cache(a + 1);
  d.Nk = small(a[6], "Nk"); d.group = small(a[7], "group"); d.scale = (float)number(a[13]);
  const at::Tensor &q = c.tensor(a[0], "q"), &o = c.tensor(a[5], "o");
  const int64_t E = d.cache.entries, H = d.cache.heads, B = E * d.group;
  if (q.dim() != 2 || q.size(0) != B || q.size(1) != H * 64 || o.sizes() != q.sizes())
    raise(PyExc_ValueError, "decode_attn_q8: q and o are [" + std::to_string(B) + ", " + std::to_string(H * 64) + "]");
  if (B > INT32_MAX) raise(PyExc_ValueError, "decode_attn_q8: too many rows");
  d.B = (int32_t)B;
  c.locate(d.cache, a + 1);
  d.q = c.at_least(q, at::kBFloat16, 0, "q"); d.q_bs = q.stride(0);
  d.o = c.at_least(o, at::kBFloat16, 0, "o"); d.o_bs = o.stride(0);
  if (a[9] != Py_None) { d.pos_dev = (int32_t*)c.vector(a[9], at::kInt, 1, "pos_dev"); d.bias_maxlen = small(a[10], "bias_maxlen"); }
  if (a[11] != Py_None) {
    const at::Tensor& b = c.tensor(a[11], "bias_row");
    if (b.dim() != 2 || b.size(0) != H) raise(PyExc_ValueError, "decode_attn_q8: bias_row is [heads, keys]");
    d.bias_ld = H > 1 ? b.stride(0) : b.size(1);
    d.bias_row = (float*)c.at_least(b, at::kFloat, (H - 1) * d.bias_ld + (d.pos_dev ? 2 * (int64_t)d.bias_maxlen - 1 : d.Nk), "bias_row");
  }
  if (a[12] != Py_None) {
    const at::Tensor& m = c.tensor(a[12], "key_mask");
    if (m.dim() != 2 || m.size(0) != E) raise(PyExc_ValueError, "decode_attn_q8: key_mask is [entries, keys]");
    d.mask_ld = E > 1 ? m.stride(0) : m.size(1);
    d.key_mask = (uint8_t*)c.at_least(m, at::kByte, (E - 1) * d.mask_ld + d.Nk, "key_mask");
  }
  d.klen = (int32_t*)c.optional(a[8], at::kInt, E, "klen");
  if (a[14] != Py_None) {
    const at::Tensor& w = c.tensor(a[14], "workspace");
    d.workspace = c.vector(w, at::kFloat, w.numel(), "workspace"); d.workspace_bytes = w.numel() * 4;
  }
  return launch(f_attn, &d, c.stream());
}

// logits rows V u next_tok ld temperature top_k top_p min_p logp unfinished eos_id pad_id seq_out seq_ld pos_dev min_length
PyObject* sample_step(PyObject* const* a) {
  Call c{"sample_step"};
  const at::Tensor &z = c.tensor(a[0], "logits"), &u = c.tensor(a[3], "u");
  const bool f32 = z.scalar_type() == at::kFloat, table = a[16] != Py_None;
  const int32_t rows = small(a[1], "rows"), V = small(a[2], "V");
  int64_t ld = given_stride(a[5]);
  int64_t seq_ld = given_stride(a[15]);
  if (a[14] != Py_None && seq_ld == 0) {              // the length of its rows: the step behind the last column is not written
    const at::Tensor& t = c.tensor(a[14], "seq_out");
    if (t.dim() != 2 || t.size(0) < rows || !t.is_contiguous() || t.size(1) > INT32_MAX)
      raise(PyExc_ValueError, "sample_step seq_out: [" + std::to_string(rows) + ", columns] is expected, or seq_ld");
    seq_ld = t.size(1);
  }
  if (u.dim() != (table ? 2 : 1) || u.size(-1) < rows)
    raise(PyExc_ValueError, "sample_step: u is [rows], or [steps, rows] with pos_dev, for " + std::to_string(rows) + " rows");
  const int64_t steps = table ? u.size(0) : 0, u_ld = !table ? 0 : (steps > 1 ? u.stride(0) : u.size(1));
  if (steps > INT32_MAX) raise(PyExc_ValueError, "sample_step: too many steps");
  void *pz = c.matrix(z, f32 ? at::kFloat : at::kBFloat16, rows, V, ld, "logits"), *pu = c.at_least(u, at::kFloat, rows, "u");
  void *tok = c.vector(a[4], at::kLong, rows, "next_tok"), *lp = c.optional(a[10], at::kFloat, rows, "logp");
  void *un = c.optional(a[11], at::kInt, rows, "unfinished"), *seq = a[14] == Py_None ? nullptr : c.operand(a[14], at::kLong, rows * seq_ld, "seq_out");
  void* ctr = c.optional(a[16], at::kInt, 1, "pos_dev");
  return launch(f_sample, pz, f32 ? V2S_F32 : V2S_BF16, ld, rows, V, number(a[6]), small(a[7], "top_k"), number(a[8]), number(a[9]), (float*)pu, u_ld, (int32_t)steps,
                         (int64_t*)tok, (float*)lp, (int32_t*)un, small(a[12], "eos_id"), small(a[13], "pad_id"), (int64_t*)seq, seq_ld, (int32_t*)ctr,
                         small(a[17], "min_length"), c.stream());
}

// every entry: the number of arguments, and no C++ exception reaches the interpreter
template <PyObject* (*F)(PyObject* const*), int N> PyObject* entry(PyObject*, PyObject* const* a, Py_ssize_t n) {
  try {
    if (n != N) raise(PyExc_TypeError, "expected " + std::to_string(N) + " arguments, got " + std::to_string(n));
    if (!raw_stream) raise(PyExc_RuntimeError, "attach() has not been called");
    return F(a);
  } catch (const Raised&) {
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  } catch (...) {
    PyErr_SetString(PyExc_RuntimeError, "unknown C++ exception");
  }
  return nullptr;
}

// current_device raw_stream v2s_version v2s_sizeof, then the addresses of the library's functions in the order of the pointers above.  The structs filled here
// are laid out by the header that this file was compiled with: a library of another version, or with other sizes, is refused and nothing is attached.
PyObject* attach(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 12) { PyErr_SetString(PyExc_TypeError, "attach: twelve arguments"); return nullptr; }
  void* f[10];
  for (int i = 0; i < 10; ++i) {
    f[i] = PyLong_AsVoidPtr(a[2 + i]);
    if (!f[i]) { if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "attach: a function's address is NULL"); return nullptr; }
  }
  const int version = ((decltype(&v2s_version))f[0])();
  if (version != V2S_ABI_VERSION) {
    PyErr_Format(PyExc_RuntimeError, "ABI mismatch: the library reports V2S_ABI_VERSION %d, _bind.so was built for %d (vidchapters_amd/csrc/build.sh builds both)", version,
                 V2S_ABI_VERSION);
    return nullptr;
  }
  const struct { const char* name; size_t size; } structs[] = {
      {"v2s_gemm_q8_args", sizeof(v2s_gemm_q8_args)}, {"v2s_kv_q8", sizeof(v2s_kv_q8)}, {"v2s_decode_attn_q8_args", sizeof(v2s_decode_attn_q8_args)}};
  for (const auto& t : structs) {
    const long long size = ((decltype(&v2s_sizeof))f[1])(t.name);
    if (size != (long long)t.size) {
      PyErr_Format(PyExc_RuntimeError, "ABI mismatch: %s has %lld bytes in the library and %zu in _bind.so (vidchapters_amd/csrc/build.sh builds both)", t.name, size, t.size);
      return nullptr;
    }
  }
  Py_INCREF(a[0]); Py_INCREF(a[1]);
  current_device = a[0]; raw_stream = a[1];
  f_quant = (decltype(f_quant))f[2]; f_norm = (decltype(f_norm))f[3]; f_dequant = (decltype(f_dequant))f[4]; f_gemm = (decltype(f_gemm))f[5];
  f_append = (decltype(f_append))f[6]; f_read = (decltype(f_read))f[7]; f_attn = (decltype(f_attn))f[8]; f_sample = (decltype(f_sample))f[9];
  Py_RETURN_NONE;
}

#define V2S_ENTRY(NAME, N) {#NAME, (PyCFunction)(void*)entry<NAME, N>, METH_FASTCALL, nullptr}
PyMethodDef methods[] = {{"attach", (PyCFunction)(void*)attach, METH_FASTCALL, nullptr},
                         V2S_ENTRY(quant_rows_q8, 7), V2S_ENTRY(rmsnorm_q8, 13), V2S_ENTRY(dequant_q8, 7), V2S_ENTRY(gemm_q8, 16), V2S_ENTRY(kv_append_q8, 11),
                         V2S_ENTRY(kv_read_q8, 11), V2S_ENTRY(decode_attn_q8, 15), V2S_ENTRY(sample_step, 18), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module_def = {PyModuleDef_HEAD_INIT, "_bind", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

extern "C" __attribute__((visibility("default"))) PyObject* PyInit__bind() { return PyModule_Create(&module_def); }
