// Python binding of the block-scaled FP8 operators (runtime/fp8_block.py): the
// checks of the arguments, the outputs' allocation and the call of the C entry
// point in one extension call. These operators take a few microseconds on the
// device, and the same steps in Python, argument by argument, take longer than
// that (13-18 us a call against 5-7).
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/recavsr_b200.h"

namespace {

constexpr int64_t kBlock = 128;

int64_t up(int64_t a, int64_t b) { return (a + b - 1) / b; }

const at::Tensor& tensor(PyObject* o, const char* what, const char* name) {
  TORCH_CHECK_VALUE(THPVariable_Check(o), what, ": ", name, " must be a tensor.");
  return THPVariable_Unpack(o);
}

int dtype_code(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return 0;
    case at::kBFloat16: return 1;
    case at::kHalf: return 2;
    default: return -1;
  }
}

bool aligned16(const at::Tensor& t) { return reinterpret_cast<uintptr_t>(t.const_data_ptr()) % 16 == 0; }

// Rows whose columns are contiguous; a single row has its length as stride.
bool is_rows(const at::Tensor& t) { return t.is_contiguous() || (t.stride(1) == 1 && t.stride(0) >= t.size(1)); }
int64_t row_stride(const at::Tensor& t) { return t.is_contiguous() ? t.size(1) : t.stride(0); }

// x as rows the kernels can read: unit column stride, 16-byte rows.
at::Tensor rows(const at::Tensor& x, const char* what) {
  TORCH_CHECK_VALUE(x.is_cuda(), what, ": the B200 kernels need CUDA tensors (got ", x.device(), ")");
  TORCH_CHECK_VALUE(dtype_code(x.scalar_type()) >= 0, what, " takes float32 / bfloat16 / float16 rows (got ",
                    x.scalar_type(), ").");
  TORCH_CHECK_VALUE(x.dim() == 2, what, " expects a 2-D matrix (got ", x.dim(), "-D).");
  TORCH_CHECK_VALUE(x.size(1) > 0 && x.size(1) % 16 == 0, what, ": columns must be a positive multiple of 16 (got ",
                    x.size(1), ").");
  TORCH_CHECK_VALUE(x.size(0) <= INT32_MAX && x.size(1) <= INT32_MAX, what, ": ", x.size(0), " x ", x.size(1),
                    " is too large.");
  if (is_rows(x) && row_stride(x) * x.element_size() % 16 == 0 && aligned16(x)) return x;
  return x.clone(at::MemoryFormat::Contiguous);
}

at::Tensor vector(const at::Tensor& t, int64_t n, const at::Tensor& like, const char* what) {
  TORCH_CHECK_VALUE(t.dim() == 1 && t.size(0) == n && t.device() == like.device(), what, " must have ", n,
                    " elements on ", like.device(), " (got ", t.sizes(), " on ", t.device(), ").");
  at::Tensor v = t.scalar_type() == at::kFloat && t.is_contiguous() ? t : t.to(at::kFloat).contiguous();
  return aligned16(v) ? v : v.clone();
}

int64_t scale_numel(int64_t rows, int64_t cols) { return up(rows, kBlock) * kBlock * up(cols, 4 * kBlock) * 4; }

at::Tensor empty(at::IntArrayRef size, at::ScalarType type, const at::Tensor& like) {
  return at::detail::empty_cuda(size, type, like.device(), c10::nullopt);    // at::empty without its dispatch
}

// Codes [rows, K] and their scales; codes as rows the kernels can read.
at::Tensor operand(const at::Tensor& codes, const at::Tensor& scales, const char* what) {
  TORCH_CHECK_VALUE(codes.is_cuda() && scales.device() == codes.device(), what,
                    ": codes and scales must be on one CUDA device (got ", codes.device(), ", ", scales.device(), ").");
  // Other 8-bit types would be read as what they are not (a float8_e5m2 code as E4M3).
  TORCH_CHECK_VALUE(codes.dim() == 2 && (codes.scalar_type() == at::kByte || codes.scalar_type() == at::kFloat8_e4m3fn) &&
                        (scales.scalar_type() == at::kByte || scales.scalar_type() == at::kFloat8_e8m0fnu),
                    what, ": operands are uint8 or float8_e4m3fn codes [rows, K] with uint8 or float8_e8m0fnu scales (got ",
                    codes.dim(), "-D ", codes.scalar_type(), ", ", scales.scalar_type(), ").");
  const int64_t n = codes.size(0), k = codes.size(1);
  TORCH_CHECK_VALUE(k > 0 && k % 16 == 0, what, ": K must be a positive multiple of 16 (got ", k, ").");
  TORCH_CHECK_VALUE(n <= INT32_MAX && k <= INT32_MAX, what, ": ", n, " x ", k, " is too large.");
  TORCH_CHECK_VALUE(scales.numel() == scale_numel(n, k) && scales.is_contiguous() && aligned16(scales), what, ": a ", n,
                    " x ", k, " operand has ", scale_numel(n, k), " contiguous, 16-byte aligned scale bytes.");
  if (is_rows(codes) && row_stride(codes) % 16 == 0 && aligned16(codes)) return codes;
  return codes.clone(at::MemoryFormat::Contiguous);
}

// Whether rows of two matrices share memory: [t.size(0), bytes] pieces every row
// stride. Rows of one stride side by side (column ranges of one buffer) do not.
bool share(const at::Tensor& a, const at::Tensor& b) {
  if (!a.numel() || !b.numel()) return false;
  const bool matrix = a.dim() == 2 && b.dim() == 2;
  auto span = [](const at::Tensor& t) {
    const int64_t last = t.dim() == 2 ? (t.size(0) - 1) * row_stride(t) + t.size(1) : t.numel();
    return last * (int64_t)t.element_size();
  };
  const int64_t at = reinterpret_cast<int64_t>(a.const_data_ptr()), bt = reinterpret_cast<int64_t>(b.const_data_ptr());
  if (at + span(a) <= bt || bt + span(b) <= at) return false;
  const int64_t step = matrix ? row_stride(a) * (int64_t)a.element_size() : 0;
  if (!matrix || step != row_stride(b) * (int64_t)b.element_size()) return true;
  const int64_t from = ((bt - at) % step + step) % step;     // b's rows start here in a's
  return from < a.size(1) * (int64_t)a.element_size() || from + b.size(1) * (int64_t)b.element_size() > step;
}

void check(int status) {
  if (!status) return;
  char text[1024];
  rc_get_last_error(text, sizeof(text));
  TORCH_CHECK_VALUE(status != 1 && status != 4, text);
  TORCH_CHECK(false, text, " (status ", status, ")");
}

uint8_t* bytes(const at::Tensor& t) { return static_cast<uint8_t*>(t.data_ptr()); }

rc_stream_t stream_of(const at::Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.get_device()).stream(); }

PyObject* pair(const at::Tensor& a, const at::Tensor& b) {
  PyObject* x = THPVariable_Wrap(a);
  PyObject* y = THPVariable_Wrap(b);
  PyObject* t = PyTuple_Pack(2, x, y);
  Py_XDECREF(x);
  Py_XDECREF(y);
  return t;
}

// A gradient would be asked for: the caller takes the call through a custom op,
// whose result raises in backward.
bool wants_grad(const at::Tensor& t) { return t.defined() && t.requires_grad() && c10::GradMode::is_enabled(); }

#define EXPECT_ARGS(count) TORCH_CHECK(nargs == (count), "expected ", (count), " arguments (got ", nargs, ")")

// quantize(x, what, weight) -> (codes, scales)
PyObject* quantize(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  EXPECT_ARGS(2);
  const bool weight = args[1] == Py_True;
  const char* what = weight ? "fp8_block.quantize_weight" : "fp8_block.quantize";
  const at::Tensor x = rows(tensor(args[0], what, "x"), what);
  const int m = (int)x.size(0), k = (int)x.size(1);
  c10::cuda::CUDAGuard guard(x.device());
  const at::Tensor codes = empty({m, k}, at::kByte, x), scales = empty({scale_numel(m, k)}, at::kByte, x);
  auto call = weight ? rc_fp8_block_quantize_weight : rc_fp8_block_quantize;
  check(call(x.const_data_ptr(), dtype_code(x.scalar_type()), m, k, row_stride(x), bytes(codes), bytes(scales),
             stream_of(x)));
  return pair(codes, scales);
  END_HANDLE_TH_ERRORS
}

// rms_norm_quantize(x, weight, eps, residual | None) -> (codes, scales, hidden | None) or NotImplemented (wants_grad)
PyObject* rms_norm_quantize(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  EXPECT_ARGS(4);
  const char* what = "fp8_block.rms_norm_quantize";
  const at::Tensor x = rows(tensor(args[0], what, "x"), what);
  const int m = (int)x.size(0), n = (int)x.size(1);
  const at::Tensor weight = vector(tensor(args[1], what, "weight"), n, x, "fp8_block.rms_norm_quantize: weight");
  const double eps = PyFloat_AsDouble(args[2]);
  if (eps == -1.0 && PyErr_Occurred()) return nullptr;
  c10::cuda::CUDAGuard guard(x.device());
  at::Tensor residual, hidden;
  if (args[3] != Py_None) {
    const at::Tensor& r = tensor(args[3], what, "residual");
    TORCH_CHECK_VALUE(r.sizes() == x.sizes() && r.scalar_type() == x.scalar_type() && r.device() == x.device(), what,
                      ": residual must match x's shape, dtype and device.");
    if (wants_grad(x) || wants_grad(r)) return Py_NewRef(Py_NotImplemented);
    residual = rows(r, what);
    hidden = empty({m, n}, x.scalar_type(), x);
  }
  const at::Tensor codes = empty({m, n}, at::kByte, x), scales = empty({scale_numel(m, n)}, at::kByte, x);
  const bool with = residual.defined();
  check(rc_fp8_block_rms_norm(x.const_data_ptr(), row_stride(x), with ? residual.const_data_ptr() : nullptr,
                              with ? row_stride(residual) : 0, dtype_code(x.scalar_type()), m, n,
                              static_cast<const float*>(weight.const_data_ptr()), (float)eps,
                              with ? hidden.data_ptr() : nullptr, bytes(codes), bytes(scales), stream_of(x)));
  PyObject* c = THPVariable_Wrap(codes);
  PyObject* s = THPVariable_Wrap(scales);
  PyObject* h = with ? THPVariable_Wrap(hidden) : Py_NewRef(Py_None);
  PyObject* t = PyTuple_Pack(3, c, s, h);
  Py_XDECREF(c);
  Py_XDECREF(s);
  Py_XDECREF(h);
  return t;
  END_HANDLE_TH_ERRORS
}

// mm(values, weights, scales, weight_scales, bias, residual, dtype, out), the last four or None; -> out or NotImplemented
// (wants_grad)
PyObject* mm(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  EXPECT_ARGS(8);
  const char* what = "fp8_block.mm";
  const at::Tensor &scales = tensor(args[2], what, "scales"), &weight_scales = tensor(args[3], what, "weight_scales");
  const at::Tensor a = operand(tensor(args[0], what, "values"), scales, what);
  const at::Tensor b = operand(tensor(args[1], what, "weights"), weight_scales, what);
  const int m = (int)a.size(0), n = (int)b.size(0), k = (int)a.size(1);
  TORCH_CHECK_VALUE(b.size(1) == k && b.device() == a.device() && n > 0, what, ": operands of ", m, " x ", k, " on ",
                    a.device(), " and ", n, " x ", b.size(1), " on ", b.device(), ".");
  at::ScalarType dtype = at::kBFloat16;
  if (args[6] != Py_None) {
    TORCH_CHECK_VALUE(THPDtype_Check(args[6]), what, ": dtype must be a torch.dtype.");
    dtype = reinterpret_cast<THPDtype*>(args[6])->scalar_type;
  } else if (args[7] != Py_None) {
    dtype = tensor(args[7], what, "out").scalar_type();
  } else if (args[5] != Py_None) {
    dtype = tensor(args[5], what, "residual").scalar_type();
  }
  TORCH_CHECK_VALUE(dtype == at::kBFloat16 || dtype == at::kHalf, what, " produces bfloat16 or float16 (got ", dtype, ").");
  c10::cuda::CUDAGuard guard(a.device());
  at::Tensor bias, residual, out;
  if (args[4] != Py_None) bias = vector(tensor(args[4], what, "bias"), n, a, "fp8_block.mm: bias");
  bool grad = wants_grad(bias);
  if (args[5] != Py_None) {
    residual = tensor(args[5], what, "residual");
    TORCH_CHECK_VALUE(residual.dim() == 2 && residual.size(0) == m && residual.size(1) == n &&
                          residual.scalar_type() == dtype && residual.device() == a.device(),
                      what, ": residual must be ", m, " x ", n, " ", dtype, " on ", a.device(), ".");
    grad |= wants_grad(residual);
    if (!is_rows(residual)) residual = residual.clone(at::MemoryFormat::Contiguous);
  }
  if (args[7] != Py_None) {
    out = tensor(args[7], what, "out");
    TORCH_CHECK_VALUE(out.dim() == 2 && out.size(0) == m && out.size(1) == n && out.scalar_type() == dtype &&
                          out.device() == a.device() && is_rows(out),
                      what, ": out must be ", m, " x ", n, " ", dtype, " rows on ", a.device(), ".");
    grad |= wants_grad(out);
    // Tiles are written while others still read: out may be the residual, element for element, and no other input.
    const bool same = residual.defined() && out.const_data_ptr() == residual.const_data_ptr() &&
                      (row_stride(out) == row_stride(residual) || m == 1);
    TORCH_CHECK_VALUE((!residual.defined() || same || !share(out, residual)) && !share(out, a) && !share(out, b) &&
                          !share(out, scales) && !share(out, weight_scales) && (!bias.defined() || !share(out, bias)),
                      what, ": out shares memory with an input (it may be the residual itself).");
  }
  if (grad) return Py_NewRef(Py_NotImplemented);
  if (!out.defined()) out = empty({m, n}, dtype, a);
  check(rc_fp8_block_gemm(bytes(a), row_stride(a), bytes(scales), bytes(b), row_stride(b), bytes(weight_scales),
                          bias.defined() ? static_cast<const float*>(bias.const_data_ptr()) : nullptr, m, n, k,
                          dtype_code(dtype), residual.defined() ? residual.const_data_ptr() : nullptr,
                          residual.defined() ? row_stride(residual) : 0, out.data_ptr(), row_stride(out), stream_of(a)));
  return THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

// swiglu_mm(values, weights, scales, weight_scales, bias | None, features | None) -> (codes, scales)
PyObject* swiglu_mm(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  EXPECT_ARGS(6);
  const char* what = "fp8_block.swiglu_mm";
  const at::Tensor &scales = tensor(args[2], what, "scales"), &weight_scales = tensor(args[3], what, "weight_scales");
  const at::Tensor a = operand(tensor(args[0], what, "values"), scales, what);
  const at::Tensor b = operand(tensor(args[1], what, "weights"), weight_scales, what);
  const int64_t m = a.size(0), n = b.size(0), k = a.size(1);
  TORCH_CHECK_VALUE(b.size(1) == k && b.device() == a.device(), what, ": operands of ", m, " x ", k, " on ", a.device(),
                    " and ", n, " x ", b.size(1), " on ", b.device(), ".");
  int64_t h = n / 2;
  if (args[5] != Py_None) {
    h = PyLong_AsLongLong(args[5]);
    if (h == -1 && PyErr_Occurred()) return nullptr;
  }
  TORCH_CHECK_VALUE(h > 0 && h % 16 == 0 && up(h, kBlock) * 2 * kBlock == n, what, ": ", h, " features need ",
                    up(h, kBlock) * 2 * kBlock, " interleaved weight rows (got ", n, ").");
  c10::cuda::CUDAGuard guard(a.device());
  at::Tensor bias;
  if (args[4] != Py_None) bias = vector(tensor(args[4], what, "bias"), n, a, "fp8_block.swiglu_mm: bias");
  const at::Tensor codes = empty({m, h}, at::kByte, a), out_scales = empty({scale_numel(m, h)}, at::kByte, a);
  check(rc_fp8_block_swiglu_gemm(bytes(a), row_stride(a), bytes(scales), bytes(b), row_stride(b), bytes(weight_scales),
                                 bias.defined() ? static_cast<const float*>(bias.const_data_ptr()) : nullptr, (int)m,
                                 (int)h, (int)k, bytes(codes), bytes(out_scales), stream_of(a)));
  return pair(codes, out_scales);
  END_HANDLE_TH_ERRORS
}

#define METHOD(name) {#name, (PyCFunction)(void (*)(void))name, METH_FASTCALL, nullptr}
PyMethodDef kMethods[] = {METHOD(quantize), METHOD(rms_norm_quantize), METHOD(mm), METHOD(swiglu_mm),
                          {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_fp8_block", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__fp8_block(void) { return PyModule_Create(&kModule); }
