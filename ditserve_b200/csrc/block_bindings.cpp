// torch bindings of the block operators: rms_norm_quant, linear_fp8, rope_axes, cross_attention.
//
// Each entry checks its arguments, allocates what it returns and launches, in one call: at a few rows the
// host's time is what a user waits for.  A call whose arguments are not laid out as its kernel takes them,
// or are wrong, launches nothing and returns None; ops/ then either brings them into that layout and calls
// again, or says what is wrong.  What keeps a launch inside its buffers is checked here alone.
//
// The entries are plain C functions over the argument vector: converting eight tensor arguments through
// the binding library took 1.5 us, a quarter of a small call.
#include <torch/extension.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAException.h>
#include <c10/cuda/CUDAGuard.h>

#include <cfloat>
#include <cmath>
#include <mutex>
#include <numeric>

#include "kernels.h"

namespace {

namespace py = pybind11;

// An optional tensor argument: a borrowed tensor, or nothing for None
struct OptTensor {
  const at::Tensor* t = nullptr;
  bool has_value() const { return t != nullptr; }
  const at::Tensor& operator*() const { return *t; }
  const at::Tensor* operator->() const { return t; }
};

struct BadArgument : std::runtime_error {
  using std::runtime_error::runtime_error;
};

const at::Tensor& tensor_arg(PyObject* o) {
  if (!THPVariable_Check(o)) throw BadArgument(std::string("expected a tensor, got ") + Py_TYPE(o)->tp_name);
  return THPVariable_Unpack(o);
}
OptTensor opt_arg(PyObject* o) { return o == Py_None ? OptTensor{} : OptTensor{&tensor_arg(o)}; }
int64_t int_arg(PyObject* o) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw py::error_already_set();
  return v;
}
double float_arg(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw py::error_already_set();
  return v;
}
bool bool_arg(PyObject* o) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) throw py::error_already_set();
  return v != 0;
}

PyObject* nothing() { Py_RETURN_NONE; }
PyObject* wrap(at::Tensor t) {
  PyObject* o = THPVariable_Wrap(std::move(t));
  if (o == nullptr) throw py::error_already_set();
  return o;
}
// a new tuple of its arguments' references (nullptr: None)
PyObject* tuple_of(std::initializer_list<PyObject*> items) {
  PyObject* t = PyTuple_New(static_cast<Py_ssize_t>(items.size()));
  Py_ssize_t i = 0;
  for (PyObject* o : items) {
    if (o == nullptr) {
      o = Py_None;
      Py_INCREF(o);
    }
    if (t != nullptr) PyTuple_SET_ITEM(t, i++, o);
    else Py_DECREF(o);
  }
  if (t == nullptr) throw py::error_already_set();
  return t;
}

// An entry: a function over `kCount` arguments whose C++ exceptions become Python's
template <PyObject* (*kBody)(PyObject* const*), int kCount>
PyObject* entry(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != kCount) {
    PyErr_Format(PyExc_TypeError, "expected %d arguments, got %zd", kCount, n);
    return nullptr;
  }
  try {
    return kBody(args);
  } catch (py::error_already_set& e) {
    e.restore();
  } catch (const BadArgument& e) {
    PyErr_SetString(PyExc_TypeError, e.what());
  } catch (...) {  // torch's own classes: torch.OutOfMemoryError among them
    torch::translate_exception_to_python(std::current_exception());
  }
  return nullptr;
}

// The device status words that ops/_ext.py made, by device index.
std::mutex status_mu;
std::vector<at::Tensor> status_words;

void bind_status(const at::Tensor& word) {
  TORCH_CHECK(word.is_cuda() && word.scalar_type() == at::kInt && word.numel() >= 2 && word.is_contiguous(),
              "a status word is int32 with 2 elements on a CUDA device");
  std::lock_guard<std::mutex> lock(status_mu);
  const size_t i = static_cast<size_t>(word.device().index());
  if (status_words.size() <= i) status_words.resize(i + 1);
  status_words[i] = word;
}

// A device's status word, cleared.  It lives as long as the process, so it comes from neither the stream that asks
// for it nor the allocator: made while that stream is captured, a tensor would be part of the graph, whose every
// replay would clear it again and with it what other launches reported.
at::Tensor new_status(int64_t index) {
  const c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(index));
  cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
  C10_CUDA_CHECK(cudaThreadExchangeStreamCaptureMode(&mode));
  void* word = nullptr;
  cudaStream_t s = nullptr;
  cudaError_t e = cudaMalloc(&word, 2 * sizeof(int));
  if (e == cudaSuccess) e = cudaStreamCreateWithFlags(&s, cudaStreamNonBlocking);
  if (e == cudaSuccess) e = cudaMemsetAsync(word, 0, 2 * sizeof(int), s);
  if (e == cudaSuccess) e = cudaStreamSynchronize(s);
  if (s != nullptr) cudaStreamDestroy(s);
  C10_CUDA_CHECK(cudaThreadExchangeStreamCaptureMode(&mode));
  C10_CUDA_CHECK(e);
  return at::from_blob(word, {2}, at::TensorOptions().dtype(at::kInt).device(at::kCUDA, static_cast<c10::DeviceIndex>(index)));
}

int* status_of(const at::Device& dev) {
  std::lock_guard<std::mutex> lock(status_mu);
  const size_t i = static_cast<size_t>(dev.index());
  return i < status_words.size() && status_words[i].defined() ? status_words[i].data_ptr<int>() : nullptr;
}

int elem_type(const at::Tensor& t) {
  switch (t.scalar_type()) {
    case at::kBFloat16: return ds::kBF16;
    case at::kHalf: return ds::kFP16;
    case at::kFloat: return ds::kFP32;
    default: return -1;
  }
}

at::Tensor empty(at::IntArrayRef sizes, at::ScalarType type, const at::Device& dev) {
  return at::detail::empty_cuda(sizes, type, dev, c10::nullopt);
}

// A tensor as rows of its last axis: any row stride in two dimensions, packed in more.
struct Rows {
  int64_t rows = 0, cols = 0, stride = 0;
};

bool as_rows(const at::Tensor& t, const at::Device& dev, Rows& r) {
  const int64_t d = t.dim();
  if (d < 1 || t.device() != dev) return false;
  r.cols = t.size(d - 1);
  if (r.cols <= 0 || r.cols >= (int64_t{1} << 30) || (r.cols > 1 && t.stride(d - 1) != 1)) return false;
  if (d == 2) {
    r.rows = t.size(0);
    r.stride = t.stride(0);
    return true;
  }
  r.rows = t.numel() / r.cols;
  r.stride = r.cols;
  return t.is_contiguous();
}

// as_rows for a tensor that is written: its rows do not overlap each other
bool as_output(const at::Tensor& t, const at::Device& dev, Rows& r) {
  return as_rows(t, dev, r) && (r.rows <= 1 || r.stride >= r.cols);
}

bool is_vector(const at::Tensor& t, const at::Device& dev, int64_t n, at::ScalarType type) {
  return t.dim() == 1 && t.size(0) == n && t.scalar_type() == type && t.device() == dev && (n <= 1 || t.stride(0) == 1);
}

// whether `out` (rows o) shares no byte with `in` (rows i): spans that do not meet, or other columns of one buffer.
// By addresses, since a storage may be another's memory (DLPack).
bool apart(const at::Tensor& out, const Rows& o, const at::Tensor& in, const Rows& i) {
  if (o.rows == 0 || i.rows == 0) return true;
  const int64_t eo = out.element_size(), ei = in.element_size();
  const int64_t lo = reinterpret_cast<int64_t>(out.data_ptr()), at = reinterpret_cast<int64_t>(in.data_ptr());
  const int64_t hi = lo + ((o.rows - 1) * o.stride + o.cols) * eo, end = at + ((i.rows - 1) * i.stride + i.cols) * ei;
  if (hi <= at || end <= lo) return true;
  // all rows of either start in one place of this pitch; a single row in one of any
  if ((o.rows > 1 && o.stride <= 0) || (i.rows > 1 && i.stride <= 0)) return false;
  const int64_t pitch = std::gcd(o.rows > 1 ? o.stride * eo : 0, i.rows > 1 ? i.stride * ei : 0);
  if (pitch == 0) return false;
  const int64_t d = ((lo - at) % pitch + pitch) % pitch;
  return d >= i.cols * ei && d + o.cols * eo <= pitch;
}

// ... the same for a vector of `n` elements that lie together
bool apart_from_vector(const at::Tensor& out, const Rows& o, const at::Tensor& in, int64_t n) {
  return n == 0 || apart(out, o, in, Rows{1, n, n});
}

// ... or is `in` itself, element by element
bool apart_or_same(const at::Tensor& out, const Rows& o, const at::Tensor& in, const Rows& i) {
  return apart(out, o, in, i) || (out.data_ptr() == in.data_ptr() && out.element_size() == in.element_size() &&
                                  o.rows == i.rows && o.cols == i.cols && (o.rows <= 1 || o.stride == i.stride));
}

// whether the bytes that two tensors span meet
bool spans_meet(const at::Tensor& x, const at::Tensor& y) {
  auto span = [](const at::Tensor& t) {
    int64_t n = 1;
    for (int64_t i = 0; i < t.dim(); ++i) n += (t.size(i) - 1) * t.stride(i);
    const int64_t lo = reinterpret_cast<int64_t>(t.data_ptr());
    return std::make_pair(lo, lo + n * static_cast<int64_t>(t.element_size()));
  };
  const auto a = span(x), b = span(y);
  return a.first < b.second && b.first < a.second;
}

// e4m3 of x's shape with rows that start on 16 bytes
at::Tensor empty_fp8_like(const at::Tensor& x, const Rows& r) {
  if (r.cols % 16 == 0) return empty(x.sizes(), at::kFloat8_e4m3fn, x.device());
  const int64_t pitch = (r.cols + 15) / 16 * 16;
  at::Tensor buf = empty({r.rows, pitch}, at::kFloat8_e4m3fn, x.device());
  std::vector<int64_t> strides(x.dim(), 1);
  int64_t s = pitch;
  for (int64_t i = x.dim() - 2; i >= 0; --i) {
    strides[i] = s;
    s *= x.size(i);
  }
  return at::as_strided(buf, x.sizes(), strides);
}

// (x, weight, residual, eps, out, scale_out, residual_out) -> (q, scale, h)
PyObject* rms_norm_quant(PyObject* const* args) {
  const at::Tensor& x = tensor_arg(args[0]);
  const OptTensor weight = opt_arg(args[1]), residual = opt_arg(args[2]);
  const double eps = float_arg(args[3]);
  const OptTensor out = opt_arg(args[4]), scale_out = opt_arg(args[5]), residual_out = opt_arg(args[6]);
  const at::Device dev = x.device();
  ds::NormQuantArgs a;
  a.type = elem_type(x);
  Rows rx, rr, rh, rq;
  if (!x.is_cuda() || a.type < 0 || !as_rows(x, dev, rx)) return nothing();
  if (weight.has_value()) {
    if (!is_vector(*weight, dev, rx.cols, x.scalar_type())) return nothing();
    a.weight = weight->data_ptr();
  }
  if (residual_out.has_value() && !residual.has_value()) return nothing();
  const c10::cuda::CUDAGuard guard(dev);
  at::Tensor h;
  if (residual.has_value()) {
    if (residual->sizes() != x.sizes() || residual->scalar_type() != x.scalar_type() || !as_rows(*residual, dev, rr))
      return nothing();
    if (residual_out.has_value()) {
      h = *residual_out;
      if (h.sizes() != x.sizes() || h.scalar_type() != x.scalar_type() || !as_output(h, dev, rh)) return nothing();
      if (!apart_or_same(h, rh, x, rx) || !apart_or_same(h, rh, *residual, rr)) return nothing();
    }
  }
  if (out.has_value() && (out->sizes() != x.sizes() || out->scalar_type() != at::kFloat8_e4m3fn || !as_output(*out, dev, rq)))
    return nothing();
  if (scale_out.has_value() && (scale_out->sizes() != x.sizes().slice(0, x.dim() - 1) || !scale_out->is_contiguous() ||
                                scale_out->scalar_type() != at::kFloat || scale_out->device() != dev))
    return nothing();
  // the row's codes, scale and sum leave while other rows, and the weight, are still read
  const Rows rs{1, rx.rows, rx.rows};
  if (weight.has_value() && rx.rows > 0 &&
      ((out.has_value() && !apart_from_vector(*out, rq, *weight, rx.cols)) ||
       (scale_out.has_value() && !apart_from_vector(*scale_out, rs, *weight, rx.cols)) ||
       (residual_out.has_value() && !apart_from_vector(*residual_out, rh, *weight, rx.cols))))
    return nothing();
  auto clear_of = [&](const at::Tensor& t, const Rows& r) {
    return (!out.has_value() || apart(*out, rq, t, r)) && (!scale_out.has_value() || apart(*scale_out, rs, t, r));
  };
  if (rx.rows > 0 && (!clear_of(x, rx) || (residual.has_value() && !clear_of(*residual, rr)) ||
                      (residual_out.has_value() && !clear_of(*residual_out, rh)) ||
                      (out.has_value() && scale_out.has_value() && !apart(*scale_out, rs, *out, rq))))
    return nothing();
  if (residual.has_value()) {
    if (!residual_out.has_value()) {
      h = empty(x.sizes(), x.scalar_type(), dev);
      rh.stride = rx.cols;
    }
    a.residual = residual->data_ptr();
    a.r_stride = rr.stride;
    a.h = h.data_ptr();
    a.h_stride = rh.stride;
  }
  at::Tensor q = out.has_value() ? *out : empty_fp8_like(x, rx);
  if (!out.has_value()) rq.stride = (rx.cols + 15) / 16 * 16;
  at::Tensor scale = scale_out.has_value() ? *scale_out : empty(x.sizes().slice(0, x.dim() - 1), at::kFloat, dev);
  a.x = x.data_ptr();
  a.x_stride = rx.stride;
  a.q = reinterpret_cast<uint8_t*>(q.data_ptr());
  a.q_stride = rq.stride;
  a.scale = reinterpret_cast<float*>(scale.data_ptr());
  a.rows = rx.rows;
  a.dim = static_cast<int>(rx.cols);
  a.eps = static_cast<float>(eps);
  ds::launch_norm_quant(a, at::cuda::getCurrentCUDAStream());
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  return tuple_of({wrap(std::move(q)), wrap(std::move(scale)), residual.has_value() ? wrap(std::move(h)) : nullptr});
}

// e4m3 rows that the product's 16-byte loads and tile loads can take
bool fp8_rows(const at::Tensor& t, const at::Device& dev, Rows& r) {
  if (t.scalar_type() != at::kFloat8_e4m3fn || !as_rows(t, dev, r)) return false;
  if (reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 != 0) return false;
  if (r.rows <= 1) r.stride = (r.cols + 15) / 16 * 16;
  return r.stride % 16 == 0 && r.stride >= r.cols;
}

// (x, x_scale, w, w_scale, bias, gelu, residual, gate, rows_per_batch, row_batch, out, out_dtype) -> y
PyObject* linear_fp8(PyObject* const* args) {
  const at::Tensor &x = tensor_arg(args[0]), &sx = tensor_arg(args[1]), &w = tensor_arg(args[2]), &sw = tensor_arg(args[3]);
  const OptTensor bias = opt_arg(args[4]);
  const bool gelu = bool_arg(args[5]);
  const OptTensor residual = opt_arg(args[6]), gate = opt_arg(args[7]);
  const int64_t rows_per_batch = args[8] == Py_None ? 0 : int_arg(args[8]);  // 0: not given
  const OptTensor row_batch = opt_arg(args[9]), out = opt_arg(args[10]);
  if (!THPDtype_Check(args[11])) throw BadArgument("out_dtype must be a dtype");
  at::ScalarType out_type = reinterpret_cast<THPDtype*>(args[11])->scalar_type;
  if (!x.is_cuda()) return nothing();
  const at::Device dev = x.device();
  Rows rx, rw, ry, rr;
  ds::LinearFp8Args a;
  a.status = status_of(dev);
  if (a.status == nullptr || !fp8_rows(x, dev, rx) || w.dim() != 2 || !fp8_rows(w, dev, rw) || rw.cols != rx.cols)
    return nothing();
  const int64_t M = rx.rows, K = rx.cols, N = rw.rows;
  // a tile's products over more values would outlast the kernels' wait for them (2^28: 0.8 s of 2)
  if (M > (1 << 30) || N > (1 << 30) || K > (1 << 28)) return nothing();
  if (sx.sizes() != x.sizes().slice(0, x.dim() - 1) || sx.scalar_type() != at::kFloat || sx.device() != dev ||
      !sx.is_contiguous() || !is_vector(sw, dev, N, at::kFloat))
    return nothing();
  if (gelu && residual.has_value()) return nothing();
  at::DimVector shape(x.sizes());
  shape.back() = N;
  if (out.has_value()) {
    out_type = out->scalar_type();
    if (out->sizes() != at::IntArrayRef(shape) || (N > 0 && !as_output(*out, dev, ry))) return nothing();
    if (N > 0 && (!apart(*out, ry, x, rx) || !apart(*out, ry, w, rw))) return nothing();
  } else {
    ry.stride = N;
  }
  if (out_type != at::kBFloat16 && out_type != at::kHalf && out_type != at::kFloat) return nothing();
  if (bias.has_value()) {
    if (!is_vector(*bias, dev, N, out_type)) return nothing();
    a.bias = bias->data_ptr();
  }
  if (residual.has_value()) {
    if (residual->sizes() != at::IntArrayRef(shape) || residual->scalar_type() != out_type ||
        (N > 0 && !as_rows(*residual, dev, rr)))
      return nothing();
    if (out.has_value() && N > 0 && !apart_or_same(*out, ry, *residual, rr)) return nothing();
    a.residual = residual->data_ptr();
    a.ldr = rr.stride;
  }
  if (gate.has_value()) {
    const at::Tensor& g = *gate;
    if (!residual.has_value() || g.scalar_type() != at::kFloat || g.device() != dev || g.dim() < 1 || g.dim() > 2 ||
        g.size(-1) != N || (N > 1 && g.stride(-1) != 1))
      return nothing();
    const int64_t batches = g.dim() == 2 ? g.size(0) : 1;
    const int64_t per = args[8] != Py_None ? rows_per_batch : std::max<int64_t>(M, 1);
    if (batches < 1 || per < 1) return nothing();
    a.gate = g.data_ptr<float>();
    a.gate_stride = g.dim() == 2 ? g.stride(0) : 0;
    a.batches = static_cast<int>(std::min<int64_t>(batches, 1 << 30));
    a.rows_per_batch = static_cast<int>(std::min<int64_t>(per, 1 << 30));
    if (row_batch.has_value()) {
      if (!is_vector(*row_batch, dev, M, at::kInt)) return nothing();
      a.row_batch = row_batch->data_ptr<int>();
    } else if ((M + per - 1) / per > batches) {
      return nothing();
    }
  }
  // blocks read these while others store
  if (out.has_value() && N > 0) {
    if (!apart_from_vector(*out, ry, sx, M) || !apart_from_vector(*out, ry, sw, N) ||
        (bias.has_value() && !apart_from_vector(*out, ry, *bias, N)))
      return nothing();
    if (gate.has_value() && (!apart(*out, ry, *gate, Rows{a.gate_stride == 0 ? 1 : a.batches, N, a.gate_stride}) ||
                             (row_batch.has_value() && !apart_from_vector(*out, ry, *row_batch, M))))
      return nothing();
  }
  const c10::cuda::CUDAGuard guard(dev);
  at::Tensor y = out.has_value() ? *out : empty(shape, out_type, dev);
  a.out_type = elem_type(y);
  a.x = reinterpret_cast<const uint8_t*>(x.data_ptr());
  a.ldx = rx.stride;
  a.w = reinterpret_cast<const uint8_t*>(w.data_ptr());
  a.ldw = rw.stride;
  a.sx = reinterpret_cast<const float*>(sx.data_ptr());
  a.sw = reinterpret_cast<const float*>(sw.data_ptr());
  a.y = y.data_ptr();
  a.ldy = ry.stride;
  a.M = static_cast<int>(M);
  a.N = static_cast<int>(N);
  a.K = static_cast<int>(K);
  a.gelu = gelu ? 1 : 0;
  ds::launch_linear_fp8(a, at::cuda::getCurrentCUDAStream());
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  return wrap(std::move(y));
}

// What a rotation's axes and thetas fix: the axis and frequency of every pair.
struct RopePlan {
  int axes = 0, pairs = 0;
  double turns[ds::kRopeMaxPairs];
  uint8_t axis[ds::kRopeMaxPairs];
};

// None where the axes are not one to kRopeMaxAxes, each with positive even dims and a positive theta
py::object rope_plan(const std::vector<int64_t>& dims, const std::vector<double>& theta) {
  if (dims.empty() || dims.size() > ds::kRopeMaxAxes || dims.size() != theta.size()) return py::none();
  int64_t pairs = 0;
  for (size_t i = 0; i < dims.size(); ++i) {
    if (dims[i] <= 0 || dims[i] % 2 != 0 || dims[i] > 2 * ds::kRopeMaxPairs || !(theta[i] > 0.0) || !std::isfinite(theta[i]))
      return py::none();
    pairs += dims[i] / 2;
  }
  if (pairs > ds::kRopeMaxPairs) return py::none();
  RopePlan p;
  p.axes = static_cast<int>(dims.size());
  for (int i = 0; i < p.axes; ++i)
    for (int64_t j = 0; j < dims[i] / 2; ++j, ++p.pairs) {
      p.axis[p.pairs] = static_cast<uint8_t>(i);
      p.turns[p.pairs] = std::pow(theta[i], -2.0 * static_cast<double>(j) / static_cast<double>(dims[i])) / (2.0 * M_PI);
    }
  return py::cast(p);
}

// (x, k, positions, plan, head_dim, half, inverse, out, k_out) -> x' or (x', k')
PyObject* rope_axes(PyObject* const* args) {
  const at::Tensor& x = tensor_arg(args[0]);
  const OptTensor k = opt_arg(args[1]);
  const at::Tensor& pos = tensor_arg(args[2]);
  const RopePlan& plan = py::handle(args[3]).cast<const RopePlan&>();
  const int64_t head_dim = int_arg(args[4]);
  const bool half = bool_arg(args[5]), inverse = bool_arg(args[6]);
  const OptTensor out = opt_arg(args[7]), k_out = opt_arg(args[8]);
  if (!x.is_cuda()) return nothing();
  const at::Device dev = x.device();
  ds::RopeAxesArgs a;
  a.type = elem_type(x);
  if (a.type < 0 || head_dim < 2 * plan.pairs || head_dim > (1 << 20) || (k_out.has_value() && !k.has_value()))
    return nothing();
  const int64_t pos_axes = pos.dim() == 1 ? 1 : (pos.dim() == 2 ? pos.size(1) : 0);
  if (pos.device() != dev || pos_axes != plan.axes) return nothing();
  switch (pos.scalar_type()) {
    case at::kLong: a.pos_type = 0; break;
    case at::kInt: a.pos_type = 1; break;
    case at::kFloat: a.pos_type = 2; break;
    case at::kDouble: a.pos_type = 3; break;
    default: return nothing();
  }
  Rows in[2], to[2];
  const at::Tensor* t[2] = {&x, k.t};
  const OptTensor o[2] = {out, k_out};
  for (int i = 0; i < 2 && t[i] != nullptr; ++i) {
    if (t[i]->dim() < 2 || t[i]->scalar_type() != x.scalar_type() || !as_rows(*t[i], dev, in[i]) ||
        in[i].cols % head_dim != 0 || in[i].rows != in[0].rows)
      return nothing();
    if (o[i].has_value()) {
      const at::Tensor& y = *o[i];
      if (y.sizes() != t[i]->sizes() || y.scalar_type() != x.scalar_type() || !as_output(y, dev, to[i]) ||
          !apart_or_same(y, to[i], *t[i], in[i]))
        return nothing();
    } else {
      to[i].stride = in[i].cols;
    }
  }
  // with k: neither output on the other's input, nor the outputs on each other
  if (k.has_value() && ((out.has_value() && !apart(*out, to[0], *k, in[1])) ||
                        (k_out.has_value() && !apart(*k_out, to[1], x, in[0])) ||
                        (out.has_value() && k_out.has_value() && !apart(*out, to[0], *k_out, to[1]))))
    return nothing();
  const int64_t rows = in[0].rows;
  // positions are read while rows leave
  if (rows > 0 && pos.numel() > 0) {
    const bool packed = pos.dim() == 1 || pos_axes == 1 || pos.stride(1) == 1;
    const Rows rp{pos.stride(0) == 0 ? 1 : pos.size(0), pos_axes, pos.stride(0)};
    for (int i = 0; i < 2; ++i)
      if (o[i].has_value() && (packed ? !apart(*o[i], to[i], pos, rp) : spans_meet(*o[i], pos))) return nothing();
  }
  if (rows > 0 && (pos.size(0) == 0 || rows % pos.size(0) != 0)) return nothing();
  const c10::cuda::CUDAGuard guard(dev);
  at::Tensor y[2];
  for (int i = 0; i < 2 && t[i] != nullptr; ++i) {
    y[i] = o[i].has_value() ? *o[i] : empty(t[i]->sizes(), x.scalar_type(), dev);
    a.t[i].x = t[i]->data_ptr();
    a.t[i].x_stride = in[i].stride;
    a.t[i].y = y[i].data_ptr();
    a.t[i].y_stride = to[i].stride;
    a.t[i].heads = static_cast<int>(in[i].cols / head_dim);
  }
  a.rows = rows;
  a.head_dim = static_cast<int>(head_dim);
  a.pairs = plan.pairs;
  a.half = half ? 1 : 0;
  a.inverse = inverse ? 1 : 0;
  a.pos = pos.data_ptr();
  a.pos_rows = pos.size(0);
  a.pos_stride = pos.stride(0);
  a.axis_stride = pos.dim() == 2 ? pos.stride(1) : 0;
  std::copy(plan.turns, plan.turns + plan.pairs, a.turns);
  std::copy(plan.axis, plan.axis + plan.pairs, a.axis);
  ds::launch_rope_axes(a, at::cuda::getCurrentCUDAStream());
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  if (t[1] == nullptr) return wrap(std::move(y[0]));
  return tuple_of({wrap(std::move(y[0])), wrap(std::move(y[1]))});
}

// (q, k, v, heads, heads_kv, kv_lens, key_mask, scale, out, return_lse) -> out or (out, lse)
PyObject* cross_attention(PyObject* const* args) {
  const at::Tensor &q = tensor_arg(args[0]), &k = tensor_arg(args[1]), &v = tensor_arg(args[2]);
  const int64_t heads = int_arg(args[3]), heads_kv = int_arg(args[4]);
  const OptTensor kv_lens = opt_arg(args[5]), key_mask = opt_arg(args[6]), out = opt_arg(args[8]);
  const bool return_lse = bool_arg(args[9]);
  if (!q.is_cuda() || q.dim() != 3 || k.dim() != 3 || heads < 1 || heads_kv < 1 || heads % heads_kv != 0) return nothing();
  const at::Device dev = q.device();
  ds::CrossAttnArgs a;
  a.type = elem_type(q);
  a.status = status_of(dev);
  const int64_t B = q.size(0), Sq = q.size(1), width = q.size(2), Sk = k.size(1), d = width / heads;
  if (a.status == nullptr || (a.type != ds::kBF16 && a.type != ds::kFP16) || width % heads != 0 || (d != 64 && d != 128))
    return nothing();
  if (B < 1 || B > 65535 || heads_kv > 65535 || Sq < 1 || Sk < 1 || Sk >= (int64_t{1} << 30) ||
      Sq * (heads / heads_kv) >= (int64_t{1} << 30) || width >= (int64_t{1} << 30))
    return nothing();
  auto fits = [&](const at::Tensor& t, int64_t rows, int64_t cols, bool output) {
    if (t.device() != dev || t.scalar_type() != q.scalar_type() || t.dim() != 3 || t.size(0) != B || t.size(1) != rows ||
        t.size(2) != cols || t.stride(2) != 1 || t.stride(1) % 8 != 0 || t.stride(0) % 8 != 0 ||
        reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 != 0)
      return false;
    if (rows > 1 && t.stride(1) < (output ? cols : 8)) return false;
    if (!output || B == 1) return true;
    // an output's entries lie behind one another, or between one another's rows
    const int64_t entry = (rows - 1) * t.stride(1) + cols, row = (B - 1) * t.stride(0) + cols;
    return t.stride(0) >= entry || (t.stride(0) >= cols && (rows == 1 || t.stride(1) >= row));
  };
  if (!fits(q, Sq, width, false) || !fits(k, Sk, heads_kv * d, false) || !fits(v, Sk, heads_kv * d, false)) return nothing();
  if (out.has_value()) {
    if (!fits(*out, Sq, width, true)) return nothing();
    for (const at::Tensor* t : {&q, &k, &v})
      if (spans_meet(*out, *t)) return nothing();
  }
  if (kv_lens.has_value()) {
    if (!is_vector(*kv_lens, dev, B, at::kInt)) return nothing();
    a.kv_lens = kv_lens->data_ptr<int>();
  }
  if (key_mask.has_value()) {
    const at::Tensor& m = *key_mask;
    if (m.device() != dev || m.scalar_type() != at::kBool || m.dim() != 2 || m.size(0) != B || m.size(1) != Sk)
      return nothing();
    a.key_mask = reinterpret_cast<const uint8_t*>(m.data_ptr());
    a.mask_row = m.stride(0);
    a.mask_col = m.stride(1);
  }
  // lengths and mask are read while outputs leave
  if (out.has_value() && ((kv_lens.has_value() && spans_meet(*out, *kv_lens)) ||
                          (key_mask.has_value() && spans_meet(*out, *key_mask))))
    return nothing();
  const double s = args[7] == Py_None ? 1.0 / std::sqrt(static_cast<double>(d)) : float_arg(args[7]);
  // the kernels multiply scores, -inf among them, by scale * log2(e) in fp32: neither zero nor infinite there
  if (!(s >= FLT_TRUE_MIN) || !(s * M_LOG2E <= FLT_MAX)) return nothing();
  const c10::cuda::CUDAGuard guard(dev);
  at::Tensor o = out.has_value() ? *out : empty(q.sizes(), q.scalar_type(), dev), lse;
  if (return_lse) {
    lse = empty({B, heads, Sq}, at::kFloat, dev);
    a.lse = lse.data_ptr<float>();
  }
  a.q = q.data_ptr();
  a.k = k.data_ptr();
  a.v = v.data_ptr();
  a.o = o.data_ptr();
  a.q_batch = q.stride(0), a.q_row = q.stride(1);
  a.k_batch = k.stride(0), a.k_row = k.stride(1);
  a.v_batch = v.stride(0), a.v_row = v.stride(1);
  a.o_batch = o.stride(0), a.o_row = o.stride(1);
  a.batch = static_cast<int>(B);
  a.seq_q = static_cast<int>(Sq);
  a.seq_k = static_cast<int>(Sk);
  a.heads = static_cast<int>(heads);
  a.heads_kv = static_cast<int>(heads_kv);
  a.head_dim = static_cast<int>(d);
  a.scale = static_cast<float>(s);
  ds::launch_cross_attention(a, at::cuda::getCurrentCUDAStream());
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  if (!return_lse) return wrap(std::move(o));
  return tuple_of({wrap(std::move(o)), wrap(std::move(lse))});
}

template <PyObject* (*kBody)(PyObject* const*), int kCount>
void add_entry(pybind11::module_& m, const char* name, const char* doc) {
  static PyMethodDef def = {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&entry<kBody, kCount>)),
                            METH_FASTCALL, doc};
  m.add_object(name, py::reinterpret_steal<py::object>(PyCFunction_New(&def, nullptr)));
}

}  // namespace

void bind_block_ops(pybind11::module_& m) {
  m.def("new_status", &new_status, "a cleared status word of a device, outside of streams and graphs");
  m.def("bind_status", &bind_status, "names a device's status word to the block operators");
  py::class_<RopePlan>(m, "RopePlan");
  m.def("rope_plan", &rope_plan, "the frequencies of a set of axes, or None");
  add_entry<&rms_norm_quant, 7>(m, "rms_norm_quant", "residual addition + RMS norm + e4m3 rows with scales");
  add_entry<&linear_fp8, 12>(m, "linear_fp8", "linear layer on e4m3 operands with row scales");
  add_entry<&rope_axes, 9>(m, "rope_axes", "rotary positions with several axes");
  add_entry<&cross_attention, 10>(m, "cross_attention", "attention to padded, masked encoder states");
}
