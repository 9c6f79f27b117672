// Python entry of the embedding heads: the checks, output tensors and calls of scenemap_b200/products.py
// in one C++ call each (METH_FASTCALL), over the C ABI of include/smg.h.  A call from Python then costs
// the host 3.3 to 4.3 us (the norm's, with its four outputs, 6.2) instead of the 9 to 28 us of the same steps in Python,
// which is what a robot's frame loop with a handful of rows waits for.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/core/grad_mode.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <c10/core/InferenceMode.h>
#include <cuda_runtime.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>

#include <mutex>
#include <stdexcept>
#include <string>

#include "../../include/smg.h"

namespace {

PyObject* g_error = nullptr;   // scenemap_b200.smg.SmgError

struct Refusal : std::runtime_error {
  using std::runtime_error::runtime_error;
};

[[noreturn]] void refuse(const char* who, const std::string& text) { throw Refusal(std::string(who) + ": " + text); }

void check(const char* who, int rc) {
  if (rc != SMG_OK) throw Refusal(std::string(who) + " rc=" + std::to_string(rc) + ": " + smg_last_error());
}

// a tensor that a call keeps for itself, or got from one before
const at::Tensor& kept(const char* who, PyObject* o, const char* name) {
  if (!THPVariable_Check(o)) refuse(who, std::string(name) + " must be a tensor");
  return THPVariable_Unpack(o);
}

// an input; nothing is recorded for autograd, so one that asks for it is not taken in silence
const at::Tensor& tensor(const char* who, PyObject* o, const char* name) {
  const at::Tensor& t = kept(who, o, name);
  if (t.requires_grad() && at::GradMode::is_enabled())
    refuse(who, std::string(name) + " requires gradients, which this call does not record: call it under torch.no_grad() or with " + name +
                    ".detach(), and the gradients' own calls for them");
  return t;
}

// changes in place so far (inference tensors do not count theirs)
int64_t version(const at::Tensor& t) { return t.is_inference() ? 0 : (int64_t)t._version(); }

int code_of(at::ScalarType t) {
  return t == at::kFloat ? SMG_EMB_F32 : t == at::kBFloat16 ? SMG_EMB_BF16 : t == at::kHalf ? SMG_EMB_F16 : -1;
}

at::ScalarType out_type(const char* who, PyObject* o, at::ScalarType none) {
  if (o == Py_None) return none;
  if (!THPDtype_Check(o)) refuse(who, "bad out_dtype");
  const at::ScalarType t = ((THPDtype*)o)->scalar_type;
  if (code_of(t) < 0) refuse(who, "bad out_dtype");
  return t;
}

int on_device(const char* who, const at::Tensor& t) {
  if (!t.is_cuda()) refuse(who, "tensors must be on a CUDA device");
  return t.get_device();
}

void same_device(const char* who, int dev, const at::Tensor& t) {
  if (!t.is_cuda() || t.get_device() != dev) refuse(who, "all tensors must be on one CUDA device");
}

// Makes the device current where it is not.
struct Device {
  int back = -1;
  explicit Device(int dev) {
    const int now = c10::cuda::current_device();
    if (now != dev) {
      back = now;
      c10::cuda::set_device((c10::DeviceIndex)dev);
    }
  }
  ~Device() {
    if (back >= 0) c10::cuda::set_device((c10::DeviceIndex)back);
  }
};

at::Tensor make(at::IntArrayRef shape, at::ScalarType t, int dev) {
  return at::detail::empty_cuda(shape, t, at::Device(at::kCUDA, (c10::DeviceIndex)dev), std::nullopt);
}

cudaStream_t stream_of(int dev) { return c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)dev).stream(); }

// A device word of 0, made outside of what the thread may be capturing: its own allocation and stream, waited for.
int32_t* new_word() {
  cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
  cudaThreadExchangeStreamCaptureMode(&mode);
  void* p = nullptr;
  cudaStream_t s = nullptr;
  cudaError_t e = cudaMalloc(&p, 256);
  if (e == cudaSuccess) e = cudaStreamCreateWithFlags(&s, cudaStreamNonBlocking);
  if (e == cudaSuccess) e = cudaMemsetAsync(p, 0, 256, s);
  if (e == cudaSuccess) e = cudaStreamSynchronize(s);
  if (s) cudaStreamDestroy(s);
  if (e != cudaSuccess && p) cudaFree(p);
  cudaThreadExchangeStreamCaptureMode(&mode);
  if (e != cudaSuccess) throw Refusal(std::string("no error word: ") + cudaGetErrorString(e));
  return (int32_t*)p;
}

// error word of each device (the caller has made the device current), an ordinary tensor whatever the mode
at::Tensor& word(int dev) {
  static at::Tensor words[64];
  static std::mutex m;
  if (dev < 0 || dev >= 64) throw Refusal("device index outside 0 .. 63");
  std::lock_guard<std::mutex> lock(m);
  if (!words[dev].defined()) {
    const c10::InferenceMode ordinary(false);
    words[dev] = at::from_blob(new_word(), {1}, at::TensorOptions().dtype(at::kInt).device(at::kCUDA, (c10::DeviceIndex)dev));
  }
  return words[dev];
}

int32_t* word_at(int dev) { return (int32_t*)word(dev).data_ptr(); }

// ---- operands ----
struct Rows {
  at::Tensor t;
  int64_t ld;
};

int64_t up8(int64_t v) { return (v + 7) & ~(int64_t)7; }

// rows of a 16-bit matrix on 16-byte boundaries, laid out anew if they are not
Rows aligned(const at::Tensor& t) {
  const int64_t rows = t.size(0), k = t.size(1), ld = rows > 1 ? t.stride(0) : up8(k);
  if ((t.stride(1) == 1 || k == 1) && ld >= k && !(ld & 7) && !((uintptr_t)t.data_ptr() & 15)) return {t, ld};
  at::Tensor n = make({rows, up8(k)}, t.scalar_type(), t.get_device()).narrow(1, 0, k);
  n.copy_(t);
  return {n, up8(k)};
}

struct Groups {
  at::Tensor t;
  int64_t ld, stride;
};

Groups aligned3(const at::Tensor& w) {
  const int64_t g = w.size(0), n = w.size(1), k = w.size(2);
  const int64_t ld = n > 1 ? w.stride(1) : up8(k), gs = g > 1 ? w.stride(0) : n * ld;
  if ((w.stride(2) == 1 || k == 1) && ld >= k && gs >= (n - 1) * ld + k && !((ld | gs) & 7) && !((uintptr_t)w.data_ptr() & 15))
    return {w, ld, gs};
  at::Tensor c = make({g, n, up8(k)}, w.scalar_type(), w.get_device()).narrow(2, 0, k);
  c.copy_(w);
  return {c, up8(k), n * up8(k)};
}

// the values of a row next to one another
Rows plain(const at::Tensor& t) {
  if (t.size(1) > 1 && t.stride(1) != 1) {
    at::Tensor c = t.contiguous();
    return {c, c.stride(0)};
  }
  return {t, t.stride(0)};
}

int as_int(const char* who, int64_t v) {
  if (v > 0x7fffffff) refuse(who, "too many rows or values for one call");
  return (int)v;
}

const int32_t* offsets(const char* who, PyObject* o, int64_t groups, int dev) {
  if (groups < 1) refuse(who, "no groups");
  if (o == Py_None) {
    if (groups != 1) refuse(who, "several groups need offsets");
    return nullptr;
  }
  const at::Tensor& off = tensor(who, o, "off");
  if (off.scalar_type() != at::kInt || off.dim() != 1 || off.size(0) != groups + 1 || !off.is_contiguous())
    refuse(who, "off must be " + std::to_string(groups + 1) + " int32 values");
  if (!off.is_cuda() || off.get_device() != dev) refuse(who, "off must be on the device of the rows");
  return (const int32_t*)off.data_ptr();
}

void both16(const char* who, const at::Tensor& a, const at::Tensor& b) {
  if ((a.scalar_type() != at::kBFloat16 && a.scalar_type() != at::kHalf) || a.scalar_type() != b.scalar_type())
    refuse(who, "inputs must both be bf16 or both f16");
}

PyObject* wrap(const at::Tensor& t) { return THPVariable_Wrap(t); }

// ---- calls; arguments are positional, products.py gives them names and defaults ----
PyObject* grouped(PyObject* const* a) {
  const char* who = "grouped";
  const at::Tensor &x = tensor(who, a[0], "x"), &w = tensor(who, a[1], "w");
  if (x.dim() != 2 || w.dim() != 3 || x.size(1) != w.size(2)) refuse(who, "x must be rows x k and w groups x n x k");
  both16(who, x, w);
  const int dev = on_device(who, x);
  same_device(who, dev, w);
  const Device d(dev);
  const int64_t rows = x.size(0), k = x.size(1), groups = w.size(0), n = w.size(1);
  const int32_t* off = offsets(who, a[2], groups, dev);
  const at::ScalarType t = out_type(who, a[3], x.scalar_type());
  const Rows xr = aligned(x);
  const Groups wr = aligned3(w);
  at::Tensor y = make({rows, n}, t, dev);
  check("smg_group_product",
        smg_group_product(xr.t.data_ptr(), xr.ld, wr.t.data_ptr(), wr.ld, wr.stride, off, as_int(who, groups), as_int(who, rows),
                          as_int(who, n), as_int(who, k), code_of(x.scalar_type()), y.data_ptr(), n, code_of(t), word_at(dev),
                          stream_of(dev)));
  return wrap(y);
}

PyObject* grouped_dx(PyObject* const* a) {
  const char* who = "grouped_dx";
  const at::Tensor &dy = tensor(who, a[0], "dy"), &w = tensor(who, a[1], "w");
  if (dy.dim() != 2 || w.dim() != 3 || dy.size(1) != w.size(1)) refuse(who, "dy must be rows x n and w groups x n x k");
  both16(who, dy, w);
  const int dev = on_device(who, dy);
  same_device(who, dev, w);
  const Device d(dev);
  const int64_t rows = dy.size(0), n = dy.size(1), groups = w.size(0), k = w.size(2);
  const int32_t* off = offsets(who, a[2], groups, dev);
  const at::ScalarType t = out_type(who, a[3], dy.scalar_type());
  const Rows yr = aligned(dy);
  const Groups wr = aligned3(w);
  at::Tensor dx = make({rows, k}, t, dev);
  check("smg_group_product_dx",
        smg_group_product_dx(yr.t.data_ptr(), yr.ld, wr.t.data_ptr(), wr.ld, wr.stride, off, as_int(who, groups), as_int(who, rows),
                             as_int(who, n), as_int(who, k), code_of(dy.scalar_type()), dx.data_ptr(), k, code_of(t), word_at(dev),
                             stream_of(dev)));
  return wrap(dx);
}

PyObject* grouped_dw(PyObject* const* a) {
  const char* who = "grouped_dw";
  const at::Tensor &dy = tensor(who, a[0], "dy"), &x = tensor(who, a[1], "x");
  if (dy.dim() != 2 || x.dim() != 2 || dy.size(0) != x.size(0)) refuse(who, "dy and x must have the same rows");
  both16(who, dy, x);
  const int dev = on_device(who, dy);
  same_device(who, dev, x);
  const Device d(dev);
  const int64_t rows = dy.size(0), n = dy.size(1), k = x.size(1);
  const int64_t groups = a[2] == Py_None ? 1 : tensor(who, a[2], "off").numel() - 1;
  const int32_t* off = offsets(who, a[2], groups, dev);
  const at::ScalarType t = out_type(who, a[3], x.scalar_type());
  const Rows yr = aligned(dy), xr = aligned(x);
  at::Tensor dw = make({groups, n, k}, t, dev);
  check("smg_group_product_dw",
        smg_group_product_dw(yr.t.data_ptr(), yr.ld, xr.t.data_ptr(), xr.ld, off, as_int(who, groups), as_int(who, rows), as_int(who, n),
                             as_int(who, k), code_of(x.scalar_type()), dw.data_ptr(), k, n * k, code_of(t), word_at(dev), stream_of(dev)));
  return wrap(dw);
}

// bytes of a row's codes and scales
int64_t code_bytes(int64_t k, int bits) { return (k + 31) / 32 * 4 * bits; }
int64_t scale_bytes(int64_t k) { return (k + 127) / 128 * 4; }

int bits_of(const char* who, PyObject* o) {
  const long b = PyLong_AsLong(o);
  if (b == -1 && PyErr_Occurred()) PyErr_Clear();
  if (b != 4 && b != 8) refuse(who, "bits must be 4 or 8");
  return (int)b;
}

bool flag(const char* who, PyObject* o, const char* name) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) {
    PyErr_Clear();
    refuse(who, std::string(name) + " must be true or false");
  }
  return v == 1;
}

// (x, bits, values) -> (buffer of codes, then scales; values or None)
PyObject* mx_quantise(PyObject* const* a) {
  const char* who = "mx_quantise";
  const at::Tensor& x = tensor(who, a[0], "x");
  if (x.dim() != 2 || code_of(x.scalar_type()) < 0 || x.size(1) < 1) refuse(who, "x must be rows x k of f32, bf16 or f16");
  const int bits = bits_of(who, a[1]), dev = on_device(who, x);
  const bool want = flag(who, a[2], "values");
  const Device d(dev);
  const int64_t rows = x.size(0), k = x.size(1), cb = rows * code_bytes(k, bits);
  const Rows xr = plain(x);
  at::Tensor buf = make({cb + rows * scale_bytes(k)}, at::kByte, dev), v;
  if (want) v = make({rows, k}, at::kBFloat16, dev);
  uint8_t* p = (uint8_t*)buf.data_ptr();
  check("smg_mx_quantise", smg_mx_quantise(xr.t.data_ptr(), xr.ld, as_int(who, rows), as_int(who, k), code_of(x.scalar_type()), bits, p, p + cb,
                                           want ? (uint16_t*)v.data_ptr() : nullptr, stream_of(dev)));
  return Py_BuildValue("(NN)", wrap(buf), want ? wrap(v) : Py_NewRef(Py_None));
}

// Microscaled rows as products.py keeps them: codes and scales, or one buffer and None
struct Mx {
  const at::Tensor* t;
  const uint8_t *codes, *scales;
};

Mx mx_rows(const char* who, PyObject* codes, PyObject* scales, int64_t rows, int64_t k, int bits) {
  const at::Tensor& c = tensor(who, codes, "codes");
  const uint8_t* p = (const uint8_t*)c.data_ptr();
  if (scales == Py_None) return {&c, p, p + rows * code_bytes(k, bits)};
  const at::Tensor& s = tensor(who, scales, "scales");
  return {&c, p, (const uint8_t*)s.data_ptr()};
}

// (a codes, a scales, rows, b codes, b scales, groups, n, k, bits, off, out_dtype)
PyObject* mx_product(PyObject* const* a) {
  const char* who = "mx_product";
  const int64_t rows = PyLong_AsLongLong(a[2]), groups = PyLong_AsLongLong(a[5]), n = PyLong_AsLongLong(a[6]), k = PyLong_AsLongLong(a[7]);
  const int bits = bits_of(who, a[8]);
  const Mx p = mx_rows(who, a[0], a[1], rows, k, bits), q = mx_rows(who, a[3], a[4], groups * n, k, bits);
  const int dev = on_device(who, *p.t);
  same_device(who, dev, *q.t);
  const Device d(dev);
  const int32_t* off = offsets(who, a[9], groups, dev);
  const at::ScalarType t = out_type(who, a[10], at::kFloat);
  at::Tensor y = make({rows, n}, t, dev);
  check("smg_mx_product", smg_mx_product(p.codes, p.scales, q.codes, q.scales, off, as_int(who, groups), as_int(who, rows), as_int(who, n),
                                         as_int(who, k), bits, y.data_ptr(), n, code_of(t), word_at(dev), stream_of(dev)));
  return wrap(y);
}

// (codes, scales, rows, k, bits, dtype) -> rows x k
PyObject* mx_values(PyObject* const* a) {
  const char* who = "dequantise";
  const int64_t rows = PyLong_AsLongLong(a[2]), k = PyLong_AsLongLong(a[3]);
  const int bits = bits_of(who, a[4]);
  const Mx p = mx_rows(who, a[0], a[1], rows, k, bits);
  const int dev = on_device(who, *p.t);
  const Device d(dev);
  const at::ScalarType t = out_type(who, a[5], at::kBFloat16);
  at::Tensor y = make({rows, k}, t, dev);
  check("smg_mx_values", smg_mx_values(p.codes, p.scales, as_int(who, rows), as_int(who, k), bits, y.data_ptr(), k, code_of(t), stream_of(dev)));
  return wrap(y);
}

const float* gain_of(const char* who, const at::Tensor& g, const at::Tensor& x) {
  if (g.scalar_type() != at::kFloat || g.dim() != 1 || g.size(0) != x.size(1) || !g.is_contiguous())
    refuse(who, "gain must be dim float32 values");
  return (const float*)g.data_ptr();
}

bool like(const at::Tensor& a, const at::Tensor& b) { return a.scalar_type() == b.scalar_type() && a.sizes() == b.sizes(); }

// changes in place of both inputs of a norm, in one number
int64_t versions(const at::Tensor& x, const at::Tensor* r) { return version(x) << 32 | (r ? version(*r) : 0); }

// (x, residual, gain, eps, bits, values) -> (h; buffer of codes, scales, 1 / rms; values; x; residual as read; their versions)
PyObject* norm_add(PyObject* const* a) {
  const char* who = "norm_add";
  const at::Tensor &x = tensor(who, a[0], "x"), &gain = tensor(who, a[2], "gain");
  if (x.dim() != 2 || code_of(x.scalar_type()) < 0 || x.size(1) < 1) refuse(who, "x must be rows x dim of f32, bf16 or f16");
  const int bits = bits_of(who, a[4]);
  const float* g = gain_of(who, gain, x);
  const int dev = on_device(who, x);
  same_device(who, dev, gain);
  const double eps = PyFloat_AsDouble(a[3]);
  if (eps == -1.0 && PyErr_Occurred()) { PyErr_Clear(); refuse(who, "eps must be a number"); }
  const bool want = flag(who, a[5], "values"), res = a[1] != Py_None;
  Rows r = {at::Tensor(), 0};
  if (res) {
    const at::Tensor& t = tensor(who, a[1], "residual");
    if (!like(t, x)) refuse(who, "the residual must be like x");
    same_device(who, dev, t);
  }
  const Device d(dev);
  if (res) r = plain(THPVariable_Unpack(a[1]));
  const Rows xr = plain(x);
  const int64_t rows = x.size(0), dim = x.size(1), cb = rows * code_bytes(dim, bits), sb = rows * scale_bytes(dim);
  at::Tensor h = make({rows, dim}, x.scalar_type(), dev), buf = make({cb + sb + 4 * rows}, at::kByte, dev), v;
  if (want) v = make({rows, dim}, at::kBFloat16, dev);
  uint8_t* p = (uint8_t*)buf.data_ptr();
  check("smg_norm_add",
        smg_norm_add(xr.t.data_ptr(), xr.ld, res ? r.t.data_ptr() : nullptr, r.ld, g, as_int(who, rows), as_int(who, dim),
                     code_of(x.scalar_type()), (float)eps, h.data_ptr(), dim, (float*)(p + cb + sb), bits, p, p + cb,
                     want ? (uint16_t*)v.data_ptr() : nullptr, stream_of(dev)));
  return Py_BuildValue("(NNNNNL)", wrap(h), wrap(buf), want ? wrap(v) : Py_NewRef(Py_None), wrap(xr.t), res ? wrap(r.t) : Py_NewRef(Py_None),
                       (long long)versions(xr.t, res ? &r.t : nullptr));
}

// (dy, x, residual, rstd buffer, byte offset in it, gain, dh, versions or -1) -> (dx, dgain)
PyObject* norm_add_backward(PyObject* const* a) {
  const char* who = "norm_add_backward";
  const at::Tensor &dy = tensor(who, a[0], "dy"), &x = kept(who, a[1], "x"), &buf = kept(who, a[3], "rstd"), &gain = tensor(who, a[5], "gain");
  if (!like(dy, x)) refuse(who, "dy must be like x");
  const long long was = PyLong_AsLongLong(a[7]);
  if (was >= 0 && was != versions(x, a[2] == Py_None ? nullptr : &kept(who, a[2], "residual")))
    refuse(who, "x or the residual was changed in place since the norm; its gradient reads them again");
  const bool res = a[2] != Py_None, past = a[6] != Py_None;
  if (past && !like(tensor(who, a[6], "dh"), x)) refuse(who, "dh must be like x");
  const float* g = gain_of(who, gain, x);
  const int dev = on_device(who, dy);
  same_device(who, dev, x);
  same_device(who, dev, gain);
  if (past) same_device(who, dev, THPVariable_Unpack(a[6]));
  const Device d(dev);
  const Rows yr = plain(dy), xr = plain(x);
  Rows r = {at::Tensor(), 0}, h = {at::Tensor(), 0};
  if (res) r = plain(kept(who, a[2], "residual"));
  if (past) h = plain(THPVariable_Unpack(a[6]));
  const int64_t rows = x.size(0), dim = x.size(1);
  at::Tensor dx = make({rows, dim}, x.scalar_type(), dev), dgain = make({dim}, at::kFloat, dev);
  at::Tensor work = make({smg_norm_add_bwd_work(as_int(who, dim))}, at::kByte, dev);
  const float* rstd = (const float*)((const uint8_t*)buf.data_ptr() + PyLong_AsLongLong(a[4]));
  check("smg_norm_add_bwd",
        smg_norm_add_bwd(yr.t.data_ptr(), yr.ld, xr.t.data_ptr(), xr.ld, res ? r.t.data_ptr() : nullptr, r.ld, rstd, g,
                         past ? h.t.data_ptr() : nullptr, h.ld, as_int(who, rows), as_int(who, dim), code_of(x.scalar_type()), dx.data_ptr(),
                         dim, (float*)dgain.data_ptr(), work.data_ptr(), stream_of(dev)));
  return Py_BuildValue("(NN)", wrap(dx), wrap(dgain));
}

PyObject* error_word(PyObject* const* a) {
  const int dev = (int)PyLong_AsLong(a[0]);
  const Device d(dev);
  return wrap(word(dev));
}

// Refusals become SmgError; what torch throws (out of memory, say) becomes RuntimeError: no C++ exception
// leaves a call.
template <PyObject* (*F)(PyObject* const*), int N>
PyObject* entry(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != N) {
    PyErr_Format(PyExc_TypeError, "%d arguments expected, %zd given", N, n);
    return nullptr;
  }
  try {
    return F(args);
  } catch (const Refusal& e) {
    PyErr_SetString(g_error, e.what());
  } catch (const c10::OutOfMemoryError& e) {
    PyErr_SetString(PyExc_MemoryError, e.what_without_backtrace());
  } catch (const c10::Error& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what_without_backtrace());
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  } catch (...) {
    PyErr_SetString(PyExc_RuntimeError, "unknown error");
  }
  return nullptr;
}

PyObject* set_error(PyObject*, PyObject* type) {
  Py_INCREF(type);
  Py_XSETREF(g_error, type);
  Py_RETURN_NONE;
}

#define ENTRY(name, n) \
  { #name, (PyCFunction)(void (*)(void))entry<name, n>, METH_FASTCALL, nullptr }

PyMethodDef methods[] = {ENTRY(grouped, 4),    ENTRY(grouped_dx, 4), ENTRY(grouped_dw, 4), ENTRY(mx_quantise, 3), ENTRY(mx_product, 11),
                         ENTRY(mx_values, 6),  ENTRY(norm_add, 6),   ENTRY(norm_add_backward, 8), ENTRY(error_word, 1),
                         {"set_error", set_error, METH_O, nullptr}, {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_heads", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}   // namespace

PyMODINIT_FUNC PyInit__heads(void) {
  g_error = Py_NewRef(PyExc_RuntimeError);
  return PyModule_Create(&module);
}
