// Python bindings of the low-bit decode operators: the argument checks, output
// and workspace allocation (torch's caching allocator) and the C ABI call
// (include/b200q.h) of w4.py, block_norm.py and kv8.py.
//
// These calls are short (a one-token 5120 x 5120 linear runs 4 us on the GPU), and
// checking some forty tensor properties plus a 20-argument foreign call from
// Python cost 14 to 30 us a call; here it is 3 to 5.  Every function is a
// METH_FASTCALL method whose C++ exceptions are turned into Python ones before
// they reach the interpreter.
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <limits>

#include "../../include/b200q.h"

namespace {

using at::Tensor;

#define B2_CHECK(cond, ...) TORCH_CHECK(cond, "[b200q] ", __VA_ARGS__)

// ---------------------------------------------------------------- arguments
const Tensor& tensor(PyObject* o, const char* name) {
  if (!THPVariable_Check(o)) throw torch::TypeError(c10::str("[b200q] ", name, " must be a tensor"));
  return THPVariable_Unpack(o);
}
Tensor optional_tensor(PyObject* o, const char* name) {
  return o == Py_None ? Tensor() : tensor(o, name);
}
double number(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw python_error();
  return v;
}
int64_t integer(PyObject* o) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw python_error();
  return v;
}
bool truth(PyObject* o) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) throw python_error();
  return v != 0;
}
// The index of a string in `names`, -1 if it is none of them.
int choice(PyObject* o, std::initializer_list<const char*> names) {
  if (!PyUnicode_Check(o)) return -1;
  int i = 0;
  for (const char* n : names) {
    if (PyUnicode_CompareWithASCIIString(o, n) == 0) return i;
    ++i;
  }
  return -1;
}
void count(Py_ssize_t n, Py_ssize_t want, const char* name) {
  if (n != want) throw torch::TypeError(c10::str("[b200q] ", name, " takes ", want, " arguments, got ", n));
}
PyObject* wrap(const Tensor& t) {
  if (!t.defined()) Py_RETURN_NONE;
  return THPVariable_Wrap(t);
}
PyObject* tuple(std::initializer_list<Tensor> ts) {
  PyObject* r = PyTuple_New(static_cast<Py_ssize_t>(ts.size()));
  if (!r) throw python_error();
  Py_ssize_t i = 0;
  for (const Tensor& t : ts) PyTuple_SET_ITEM(r, i++, wrap(t));
  return r;
}

// B200Q_BF16 / F16 / F32 of a type, -1 for others.
int out_code(at::ScalarType t) {
  return t == at::kBFloat16 ? B200Q_BF16 : t == at::kHalf ? B200Q_F16 : t == at::kFloat ? B200Q_F32 : -1;
}
// B200Q_BIAS_*, -1 for others.
int bias_code(at::ScalarType t) { return out_code(t) < 0 ? -1 : out_code(t) + 1; }
int code16(const Tensor& t, const char* what) {
  const int c = out_code(t.scalar_type());
  B2_CHECK(c == B200Q_BF16 || c == B200Q_F16, what, " expects bf16/f16, got ", t.scalar_type());
  return c;
}
bool aligned(const void* p, int bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }
void on_device(const Tensor& t, const at::Device& dev, const char* name) {
  B2_CHECK(t.device() == dev, name, " is on ", t.device(), ", expected ", dev);
}
void cuda_device(const Tensor& t) { B2_CHECK(t.is_cuda(), "expected CUDA tensors, got ", t.device()); }
void* stream() { return c10::cuda::getCurrentCUDAStream().stream(); }
void status(int st) {
  B2_CHECK(st == 0, "native call failed: ", b200q_status_string(st), " (status ", st, ")");
}
Tensor empty(at::IntArrayRef shape, const Tensor& like, at::ScalarType t) {
  return at::empty(shape, like.options().dtype(t).requires_grad(false).memory_format(std::nullopt));
}
// Device pointer of a workspace of `bytes`, kept alive by `hold` until the launch.
void* workspace(size_t bytes, const Tensor& like, Tensor* hold) {
  if (!bytes) return nullptr;
  *hold = empty({static_cast<int64_t>(bytes)}, like, at::kByte);
  return hold->data_ptr();
}
// [..., D] as rows: the tensor (copied unless its rows have unit stride and one
// common row stride) and that stride.
Tensor as_rows(const Tensor& t, int64_t D, int64_t* ld) {
  if (t.is_contiguous()) {
    *ld = D;
    return t;
  }
  Tensor r = t.dim() == 2 ? t : t.reshape({-1, D});
  if ((D > 1 && r.stride(1) != 1) || (r.size(0) > 1 && r.stride(0) < D)) r = r.contiguous();
  *ld = r.size(0) > 1 ? r.stride(0) : D;
  return r;
}

// ---------------------------------------------------------------- 4-bit linear
Tensor w4a16(const Tensor& x, const Tensor& w, const Tensor& scales, const Tensor& zeros,
             const Tensor& bias_in, int act, at::ScalarType out_dtype) {
  cuda_device(x);
  const at::Device dev = x.device();
  const int xdt = code16(x, "w4a16");
  B2_CHECK(x.dim() >= 1, "w4a16: x must be [..., K]");
  const int64_t K = x.size(-1);
  B2_CHECK(w.dim() == 2 && w.scalar_type() == at::kByte && 2 * w.size(1) == K && w.stride(1) == 1,
           "w4a16: w must be uint8 [N, K/2] with K=", K, " and unit inner stride, got ",
           w.scalar_type(), " ", w.sizes());
  const int64_t N = w.size(0);
  const int64_t ldw = N > 1 ? w.stride(0) : (K / 2 + 15) / 16 * 16;
  B2_CHECK(aligned(w.data_ptr(), 16) && ldw % 16 == 0 && ldw >= K / 2,
           "w4a16: the rows of w must start on 16-byte boundaries");
  const int sdt = bias_code(scales.scalar_type());
  B2_CHECK(sdt > 0 && scales.dim() == 2 && scales.size(0) == N && scales.is_contiguous(),
           "w4a16: scales must be contiguous bf16/f16/f32 [N, K/G], got ", scales.scalar_type(), " ",
           scales.sizes());
  const int64_t groups = scales.size(1), G = groups ? K / groups : 0;
  B2_CHECK((G == 32 || G == 64 || G == 128) && G * groups == K, "w4a16: K=", K, " in ", groups,
           " groups; the group size must be 32, 64 or 128");
  on_device(w, dev, "w");
  on_device(scales, dev, "scales");
  if (zeros.defined()) {
    B2_CHECK(zeros.scalar_type() == at::kByte && zeros.sizes() == scales.sizes() && zeros.is_contiguous(),
             "w4a16: zeros must be contiguous uint8 of scales' shape");
    on_device(zeros, dev, "zeros");
  }
  const int code = out_code(out_dtype);
  B2_CHECK(code >= 0, "unsupported out dtype ", out_dtype);
  Tensor bias = bias_in;
  int bdt = B200Q_BIAS_NONE;
  const c10::cuda::CUDAGuard guard(dev);
  if (bias.defined()) {
    on_device(bias, dev, "bias");
    B2_CHECK(bias.numel() == N, "bias numel ", bias.numel(), " != N ", N);
    bias = bias.contiguous();
    if (bias_code(bias.scalar_type()) < 0) bias = bias.to(at::kFloat);
    bdt = bias_code(bias.scalar_type());
  }
  int64_t ldx;
  Tensor x2 = as_rows(x, K, &ldx);
  const int64_t M = x.numel() / K;
  const size_t bytes = b200q_w4a16_workspace_bytes(M, N, K, G, xdt, sdt);
  if (bytes && xdt == B200Q_F16 && (!aligned(x2.data_ptr(), 16) || ldx % 8)) {
    x2 = x2.clone(at::MemoryFormat::Contiguous);
    ldx = K;
  }
  at::DimVector shape(x.sizes());
  shape.back() = N;
  Tensor out = empty(shape, x, out_dtype), hold;
  void* work = workspace(bytes, x, &hold);
  status(b200q_w4a16_linear(x2.data_ptr(), xdt, ldx, static_cast<const uint8_t*>(w.data_ptr()), ldw,
                            scales.data_ptr(), sdt,
                            zeros.defined() ? static_cast<const uint8_t*>(zeros.data_ptr()) : nullptr, G,
                            bias.defined() ? bias.data_ptr() : nullptr, bdt, act, out.data_ptr(), code,
                            N, M, N, K, work, bytes, stream()));
  return out;
}

PyObject* py_w4a16(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  count(n, 7, "w4a16_linear");
  const Tensor& x = tensor(a[0], "x");
  const int act = a[5] == Py_None ? 0 : choice(a[5], {"none", "gelu_tanh", "gelu"});
  B2_CHECK(act >= 0, "unknown activation");
  if (a[6] != Py_None && !THPDtype_Check(a[6])) throw torch::TypeError(std::string("[b200q] out_dtype must be a torch.dtype"));
  const at::ScalarType od = a[6] == Py_None ? x.scalar_type() : reinterpret_cast<THPDtype*>(a[6])->scalar_type;
  return wrap(w4a16(x, tensor(a[1], "w"), tensor(a[2], "scales"), optional_tensor(a[3], "zeros"),
                    optional_tensor(a[4], "bias"), act, od));
  END_HANDLE_TH_ERRORS
}

// ---------------------------------------------------------------- block norms
struct Vector {
  const void* p = nullptr;
  int dtype = 0;
};
Vector vector(const Tensor& t, int64_t D, const at::Device& dev, const char* name) {
  if (!t.defined()) return {};
  B2_CHECK(t.dim() == 1 && t.size(0) == D && bias_code(t.scalar_type()) > 0 && (D == 1 || t.stride(0) == 1),
           name, " must be bf16/f16/f32 [", D, "] with unit stride, got ", t.scalar_type(), " ", t.sizes());
  on_device(t, dev, name);
  return {t.data_ptr(), bias_code(t.scalar_type())};
}

// [B, D] or [D] rows of gate / scale / shift.
struct Mods {
  int64_t count = -1;  // B, common to the three
  int dtype = 0;
  struct Row {
    Tensor t;  // a copy where the rows overlap
    const void* p = nullptr;
    int64_t ld = 0;
  };
  Row add(const Tensor& in, int64_t D, int64_t rows, const at::Device& dev, const char* name) {
    Row r;
    if (!in.defined()) return r;
    const int64_t b = in.dim() == 2 ? in.size(0) : 1;
    B2_CHECK((in.dim() == 1 || in.dim() == 2) && in.size(-1) == D && bias_code(in.scalar_type()) > 0 &&
                 (D == 1 || in.stride(-1) == 1),
             name, " must be bf16/f16/f32 [B, ", D, "] with unit inner stride, got ", in.scalar_type(), " ",
             in.sizes());
    on_device(in, dev, name);
    if (count < 0) {
      B2_CHECK(b > 0 && rows % b == 0, rows, " rows do not split over ", b, " rows of ", name);
      count = b;
      dtype = bias_code(in.scalar_type());
    }
    B2_CHECK(b == count && bias_code(in.scalar_type()) == dtype,
             "gate, scale and shift must agree in type and rows");
    r.t = in;
    r.ld = b > 1 ? in.stride(0) : D;
    if (r.ld < D) {  // a row expanded over the batch
      r.t = in.contiguous();
      r.ld = D;
    }
    r.p = r.t.data_ptr();
    return r;
  }
};

constexpr std::initializer_list<const char*> kKinds = {"none", "rms", "layer"};

// x, y, gate, post_weight, post_kind, residual_scale, weight, scale, shift, kind,
// eps, quant, want_out -> (h, out, codes, scales), the ones asked for.
PyObject* py_block_norm(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  count(n, 13, "block_norm");
  const Tensor& x = tensor(a[0], "x");
  Tensor y = optional_tensor(a[1], "y");
  const int post_kind = choice(a[4], kKinds), kind = choice(a[9], kKinds);
  const double res_scale = number(a[5]), eps = number(a[10]);
  const bool quant = truth(a[11]), want_out = truth(a[12]);
  B2_CHECK(kind >= 0 && post_kind >= 0, "norm kind must be 'none', 'rms' or 'layer'");
  cuda_device(x);
  const at::Device dev = x.device();
  const int code = code16(x, "block norm");
  const int64_t D = x.dim() ? x.size(-1) : 0;
  B2_CHECK(D >= 1 && D <= B200Q_NORM_MAX_D, "block norms take rows of 1 to ", B200Q_NORM_MAX_D,
           " values, got ", x.sizes());
  const int64_t rows = x.numel() / D;
  const c10::cuda::CUDAGuard guard(dev);
  int64_t ldx, ldy = 0;
  const Tensor x2 = as_rows(x, D, &ldx);
  if (y.defined()) {
    B2_CHECK(y.sizes() == x.sizes() && y.scalar_type() == x.scalar_type(), "y must match the residual: ",
             x.scalar_type(), " ", x.sizes(), ", got ", y.scalar_type(), " ", y.sizes());
    on_device(y, dev, "y");
    y = as_rows(y, D, &ldy);
  }
  const Vector pw = vector(optional_tensor(a[3], "post_weight"), D, dev, "post_weight");
  const Vector w = vector(optional_tensor(a[6], "weight"), D, dev, "weight");
  Mods mods;
  const Mods::Row gate = mods.add(optional_tensor(a[2], "gate"), D, rows, dev, "gate");
  const Mods::Row scale = mods.add(optional_tensor(a[7], "scale"), D, rows, dev, "scale");
  const Mods::Row shift = mods.add(optional_tensor(a[8], "shift"), D, rows, dev, "shift");
  const int64_t per = std::max<int64_t>(rows / std::max<int64_t>(mods.count, 1), 1);
  Tensor h, out, q, s;
  if (y.defined()) h = empty(x.sizes(), x, x.scalar_type());
  if (want_out && quant) {
    q = empty({rows, D}, x, at::kChar);
    s = empty({rows, 1}, x, at::kFloat);
  } else if (want_out) {
    out = empty(x.sizes(), x, x.scalar_type());
  }
  auto ptr = [](const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; };
  status(b200q_block_norm(x2.data_ptr(), ldx, ptr(y), ldy, code, post_kind, pw.p, pw.dtype, gate.p,
                          gate.ld, static_cast<float>(res_scale), kind, w.p, w.dtype, scale.p, scale.ld,
                          shift.p, shift.ld, mods.dtype, per, static_cast<float>(eps), ptr(h), D, ptr(out),
                          D, static_cast<int8_t*>(ptr(q)), D, static_cast<float*>(ptr(s)), rows, D, stream()));
  if (!y.defined()) return quant ? tuple({q, s}) : wrap(out);
  if (!want_out) return wrap(h);
  return quant ? tuple({h, q, s}) : tuple({h, out});
  END_HANDLE_TH_ERRORS
}

// ---------------------------------------------------------------- 8-bit cache
struct Cache {
  int64_t P, H, T, D, ld, nb;
  int8_t *k, *v;
  float *ks, *vs;
  const int32_t* table;
  at::Device dev = at::kCUDA;
};
Cache cache(PyObject* const* a, int64_t B) {
  const Tensor &kc = tensor(a[0], "k_codes"), &vc = tensor(a[1], "v_codes"), &ks = tensor(a[2], "k_scale"),
               &vs = tensor(a[3], "v_scale"), &table = tensor(a[4], "block_table");
  B2_CHECK(kc.dim() == 4 && kc.sizes() == vc.sizes() && kc.scalar_type() == at::kChar &&
               vc.scalar_type() == at::kChar && kc.is_contiguous() && vc.is_contiguous(),
           "kv8: k_codes and v_codes must be contiguous int8 [pages, heads, T, D], got ", kc.scalar_type(),
           " ", kc.sizes(), ", ", vc.scalar_type(), " ", vc.sizes());
  Cache c;
  c.P = kc.size(0);
  c.H = kc.size(1);
  c.T = kc.size(2);
  c.D = kc.size(3);
  B2_CHECK((c.T == 16 || c.T == 32 || c.T == 64 || c.T == 128) && (c.D == 64 || c.D == 128) && c.P > 0 && c.H > 0,
           "kv8: pages of ", c.T, " tokens x ", c.D, "; T must be 16, 32, 64 or 128 and D 64 or 128");
  for (const Tensor* s : {&ks, &vs})
    B2_CHECK(s->dim() == 2 && s->size(0) == c.P && s->size(1) == c.H && s->scalar_type() == at::kFloat &&
                 s->is_contiguous(),
             "kv8: scales must be contiguous fp32 [", c.P, ", ", c.H, "], got ", s->scalar_type(), " ", s->sizes());
  if (B < 0) B = table.dim() == 2 ? table.size(0) : 0;
  B2_CHECK(table.dim() == 2 && table.scalar_type() == at::kInt && table.size(0) == B && table.size(1) > 0 &&
               (table.size(1) == 1 || table.stride(1) == 1),
           "kv8: block_table must be int32 [", B, ", max_blocks], got ", table.scalar_type(), " ", table.sizes());
  cuda_device(kc);
  c.dev = kc.device();
  on_device(vc, c.dev, "v_codes");
  on_device(ks, c.dev, "k_scale");
  on_device(vs, c.dev, "v_scale");
  on_device(table, c.dev, "block_table");
  c.nb = table.size(1);
  c.ld = B > 1 ? table.stride(0) : c.nb;
  B2_CHECK(c.ld >= c.nb, "kv8: block_table rows overlap");
  c.k = kc.data_ptr<int8_t>();
  c.v = vc.data_ptr<int8_t>();
  c.ks = ks.data_ptr<float>();
  c.vs = vs.data_ptr<float>();
  c.table = table.data_ptr<int32_t>();
  return c;
}
const int32_t* per_seq(PyObject* o, int64_t B, const at::Device& dev, const char* name) {
  const Tensor& t = tensor(o, name);
  B2_CHECK(t.dim() == 1 && t.size(0) == B && t.scalar_type() == at::kInt && t.is_contiguous(), "kv8: ", name,
           " must be contiguous int32 [", B, "], got ", t.scalar_type(), " ", t.sizes());
  on_device(t, dev, name);
  return t.data_ptr<int32_t>();
}
// A [B, heads, S, D] operand with unit inner stride and 16-byte rows.
Tensor tokens(const Tensor& t, at::IntArrayRef shape, at::ScalarType dt, const at::Device& dev, const char* name) {
  B2_CHECK(t.sizes() == shape && t.scalar_type() == dt, "kv8: ", name, " must be ", dt, " ", shape, ", got ",
           t.scalar_type(), " ", t.sizes());
  on_device(t, dev, name);
  const bool ok = t.stride(3) == 1 && ((t.stride(0) | t.stride(1) | t.stride(2)) & 7) == 0 && aligned(t.data_ptr(), 16);
  return ok ? t : t.clone(at::MemoryFormat::Contiguous);
}

// k, v, the cache (5), start, counts
PyObject* py_kv8_append(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  count(n, 9, "kv8_append");
  const Tensor &k = tensor(a[0], "k"), &v = tensor(a[1], "v");
  B2_CHECK(k.dim() == 4, "kv8: k must be [B, heads, S, D], got ", k.sizes());
  const int code = code16(k, "kv8_append");
  const int64_t B = k.size(0), S = k.size(2);
  const Cache c = cache(a + 2, B);
  const c10::cuda::CUDAGuard guard(c.dev);
  const int64_t shape[4] = {B, c.H, S, c.D};
  const Tensor k2 = tokens(k, shape, k.scalar_type(), c.dev, "k"), v2 = tokens(v, shape, k.scalar_type(), c.dev, "v");
  const int32_t* start = per_seq(a[7], B, c.dev, "start");
  const int32_t* counts = a[8] == Py_None ? nullptr : per_seq(a[8], B, c.dev, "counts");
  status(b200q_kv8_append(k2.data_ptr(), v2.data_ptr(), code, B, S, k2.strides().data(), v2.strides().data(), c.k,
                          c.v, c.ks, c.vs, c.P, c.H, c.T, c.D, c.table, c.ld, c.nb, start, counts, stream()));
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

// the cache (5), first, counts, max_count, out_dtype
PyObject* py_kv8_gather(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  count(n, 9, "kv8_gather");
  const Cache c = cache(a, -1);
  const int64_t B = tensor(a[4], "block_table").size(0), S = integer(a[7]);
  if (!THPDtype_Check(a[8])) throw torch::TypeError(std::string("[b200q] out_dtype must be a torch.dtype"));
  const at::ScalarType od = reinterpret_cast<THPDtype*>(a[8])->scalar_type;
  const int code = out_code(od);
  B2_CHECK(code >= 0 && S >= 0, "kv8_gather: out dtype ", od, ", max_count ", S);
  const int32_t* first = per_seq(a[5], B, c.dev, "first");
  const int32_t* counts = per_seq(a[6], B, c.dev, "counts");
  const c10::cuda::CUDAGuard guard(c.dev);
  const Tensor& like = tensor(a[0], "k_codes");
  const Tensor k = empty({B, c.H, S, c.D}, like, od), v = empty({B, c.H, S, c.D}, like, od);
  status(b200q_kv8_gather(c.k, c.v, c.ks, c.vs, c.P, c.H, c.T, c.D, c.table, c.ld, c.nb, first, counts, k.data_ptr(),
                          v.data_ptr(), code, B, S, stream()));
  return tuple({k, v});
  END_HANDLE_TH_ERRORS
}

// q, the cache (5), lens, causal, scale, max_len
PyObject* py_kv8_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  count(n, 10, "kv8_attention");
  const Tensor& q = tensor(a[0], "q");
  B2_CHECK(q.dim() == 4, "kv8: q must be [B, heads, Tq, D], got ", q.sizes());
  const int64_t B = q.size(0), Hq = q.size(1), Tq = q.size(2), D = q.size(3);
  const int code = code16(q, "kv8_attention");
  const Cache c = cache(a + 1, B);
  B2_CHECK(Hq > 0 && Hq % c.H == 0 && D == c.D, "kv8: ", Hq, " query heads of ", D, " over ", c.H,
           " cache heads of ", c.D);
  const c10::cuda::CUDAGuard guard(c.dev);
  const Tensor q2 = tokens(q, q.sizes(), q.scalar_type(), c.dev, "q");
  const int32_t* lens = per_seq(a[6], B, c.dev, "lens");
  const bool causal = truth(a[7]);
  const double scale = a[8] == Py_None ? 1.0 / std::sqrt(static_cast<double>(D)) : number(a[8]);
  const int64_t cap = c.T * c.nb;
  const int64_t max_len = a[9] == Py_None ? cap : std::min(integer(a[9]), cap);
  B2_CHECK(max_len >= 0, "kv8: max_len ", max_len);
  const Tensor flat = empty({B, Tq, Hq, D}, q, q.scalar_type()), lse = empty({B, Hq, Tq}, q, at::kFloat);
  const Tensor out = flat.transpose(1, 2);
  const size_t bytes = b200q_kv8_attention_workspace_size(B, Hq, c.H, Tq, D, max_len);
  Tensor hold;
  void* work = workspace(bytes, q, &hold);
  status(b200q_kv8_attention(q2.data_ptr(), code, B, Hq, Tq, q2.strides().data(), c.k, c.v, c.ks, c.vs, c.P, c.H, c.T,
                             D, c.table, c.ld, c.nb, lens, max_len, causal, static_cast<float>(scale), out.data_ptr(),
                             out.strides().data(), lse.data_ptr<float>(), work, bytes, stream()));
  return tuple({out, lse});
  END_HANDLE_TH_ERRORS
}

PyMethodDef kMethods[] = {
    {"w4a16_linear", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(py_w4a16)), METH_FASTCALL, nullptr},
    {"block_norm", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(py_block_norm)), METH_FASTCALL, nullptr},
    {"kv8_append", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(py_kv8_append)), METH_FASTCALL, nullptr},
    {"kv8_gather", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(py_kv8_gather)), METH_FASTCALL, nullptr},
    {"kv8_attention", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(py_kv8_attention)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "b200q_bindings", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

extern "C" __attribute__((visibility("default"))) PyObject* PyInit_b200q_bindings(void) {
  return PyModule_Create(&kModule);
}
