// Python module of the block-FP8 operators: checks of arguments, outputs, and the call of the C ABI (include/mono_linear.h) on the
// current stream. Arguments come positionally from unimonomoe_b200/linear.py, which has the documentation. In C++ because a call
// is to cost the host a few microseconds.
#include <ATen/ATen.h>
#include <c10/core/InferenceMode.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <array>
#include <utility>

#include "../../../include/mono_linear.h"

namespace {

using at::Tensor;

// ---- arguments
const Tensor& tensor(PyObject* o, const char* name) {
  if (!THPVariable_Check(o)) throw c10::TypeError({__func__, __FILE__, static_cast<uint32_t>(__LINE__)}, c10::str(name, " must be a tensor, got ", Py_TYPE(o)->tp_name));
  return THPVariable_Unpack(o);
}
int64_t integer(PyObject* o, const char* name) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) {
    PyErr_Clear();
    throw c10::TypeError({__func__, __FILE__, static_cast<uint32_t>(__LINE__)}, c10::str(name, " must be a 64-bit whole number, got ", Py_TYPE(o)->tp_name));
  }
  return v;
}
bool truth(PyObject* o) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) throw python_error();
  return v != 0;
}
void on_gpu(const Tensor& t, const char* name) {
  TORCH_CHECK_VALUE(t.is_cuda(), name, " is on ", t.device(), "; these operators need a CUDA device, there is no CPU path");
  TORCH_CHECK_VALUE(t.layout() == at::kStrided && !t.is_neg(), name, " is sparse, or a view whose memory holds the negative");
}
void typed(const Tensor& t, const char* name, at::ScalarType type, c10::Device device) {
  on_gpu(t, name);
  TORCH_CHECK_VALUE(t.scalar_type() == type, name, " has dtype ", t.scalar_type(), ", expected ", type);
  TORCH_CHECK_VALUE(t.device() == device, name, " is on ", t.device(), ", expected ", device);
}
bool aligned(const Tensor& t) { return (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0; }
// Contiguous and on a 16-byte boundary: as it is, or as a copy.
Tensor packed(const Tensor& t) {
  Tensor c = t.is_contiguous() ? t : t.contiguous();
  return aligned(c) ? c : c.clone();
}
// e4m3, as such or as bytes.
void bytes8(const Tensor& t, const char* name, c10::Device device) {
  on_gpu(t, name);
  TORCH_CHECK_VALUE(t.scalar_type() == at::kFloat8_e4m3fn || t.scalar_type() == at::kByte, name, " has dtype ", t.scalar_type(),
                    ", expected float8_e4m3fn (or uint8, its bytes)");
  TORCH_CHECK_VALUE(t.device() == device, name, " is on ", t.device(), ", expected ", device);
}
int64_t groups(int64_t k) { return (k + 127) / 128; }
void inner(int64_t k, const char* name) {
  TORCH_CHECK_VALUE(k >= 16 && k % 16 == 0 && k <= (1 << 24), name, " has rows of ", k, "; a multiple of 16 up to 2^24 is needed");
}

Tensor empty(at::IntArrayRef shape, at::ScalarType type, c10::Device device) {
  return at::empty(shape, at::TensorOptions().dtype(type).device(device));
}
// Several tensors in one allocation: an allocation costs the host more than all the rest of one.
class Block {
 public:
  using Part = std::pair<c10::SmallVector<int64_t, 6>, at::ScalarType>;
  Block(c10::Device device, std::initializer_list<Part> parts) {
    int64_t bytes = 0;
    for (const Part& p : parts) bytes += padded(p);
    base_ = empty({bytes}, at::kByte, device);
    int64_t at = 0;
    for (const Part& p : parts) {
      Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(base_.storage()), base_.key_set(), c10::scalarTypeToTypeMeta(p.second));
      t.unsafeGetTensorImpl()->set_storage_offset(at / static_cast<int64_t>(c10::elementSize(p.second)));
      t.unsafeGetTensorImpl()->set_sizes_contiguous(p.first);
      tensors_.push_back(std::move(t));
      at += padded(p);
    }
  }
  const Tensor& operator[](size_t i) const { return tensors_[i]; }

 private:
  static int64_t padded(const Part& p) {
    int64_t n = static_cast<int64_t>(c10::elementSize(p.second));
    for (const int64_t s : p.first) n *= s;
    return (n + 15) / 16 * 16;
  }
  Tensor base_;
  c10::SmallVector<Tensor, 4> tensors_;
};
template <typename T>
T* ptr(const Tensor& t) { return t.defined() ? static_cast<T*>(t.data_ptr()) : nullptr; }

// ---- the status word of a device. Zeroed once, before any launch that may report into it, on a stream that is not being captured, and
// waited for: as part of a graph it would wipe what was reported before at each replay. Never freed: a captured graph may hold its
// address. Not an inference tensor, which check_status could not write outside of that mode.
Tensor& status_word(c10::DeviceIndex device) {
  static auto* words = new std::array<Tensor, 64>();
  Tensor& t = words->at(device);
  if (t.defined()) return t;
  const c10::InferenceMode normal(false);
  const c10::cuda::CUDAStreamCaptureModeGuard relaxed(cudaStreamCaptureModeRelaxed);
  c10::cuda::CUDAStreamGuard side(c10::cuda::getStreamFromPool(true, device));
  while (c10::cuda::currentStreamCaptureStatusMayInitCtx() != c10::cuda::CaptureStatus::None) side.reset_stream(c10::cuda::getStreamFromPool(true, device));
  const Tensor w = at::zeros({2}, at::TensorOptions().dtype(at::kInt).device(at::kCUDA, device));
  side.current_stream().synchronize();
  return t = w;
}
uint32_t* status(c10::Device device) { return static_cast<uint32_t*>(status_word(device.index()).data_ptr()); }
mono_lin_stream_t stream_of(c10::Device device) {
  return reinterpret_cast<mono_lin_stream_t>(c10::cuda::getCurrentCUDAStream(device.index()).stream());
}
void launched(const char* name, int rc) {
  const char* why = rc == MONO_LIN_NULL        ? " (a required pointer is null)"
                    : rc == MONO_LIN_BAD_SIZE  ? " (a size is out of its range)"
                    : rc == MONO_LIN_ALIGNMENT ? " (a pointer or a stride is not aligned)"
                    : rc == MONO_LIN_DRIVER    ? " (the driver refuses a tensor map)"
                                               : "";
  TORCH_CHECK(rc == 0, name, " failed: rc=", rc, why);
}
PyObject* tuple(std::initializer_list<Tensor> tensors) {
  PyObject* r = PyTuple_New(static_cast<Py_ssize_t>(tensors.size()));
  if (!r) throw python_error();
  Py_ssize_t i = 0;
  for (const Tensor& t : tensors) PyTuple_SET_ITEM(r, i++, THPVariable_Wrap(t));
  return r;
}
void expect(Py_ssize_t have, Py_ssize_t want) {
  if (have != want) throw c10::TypeError({__func__, __FILE__, static_cast<uint32_t>(__LINE__)}, c10::str("expected ", want, " arguments, got ", have));
}
// The shape of `t` with its last size replaced.
c10::SmallVector<int64_t, 6> with_last(const Tensor& t, int64_t last) {
  c10::SmallVector<int64_t, 6> s(t.sizes().begin(), t.sizes().end());
  s.back() = last;
  return s;
}

// bf16 [..., K] as rows a stride apart: as it is where the rows lie evenly on 16-byte boundaries, else as a copy.
struct Rows {
  Tensor t;
  int64_t rows = 1, cols = 0, stride = 0;
  Rows(const Tensor& in, const char* name) : t(in) {
    on_gpu(in, name);
    TORCH_CHECK_VALUE(in.scalar_type() == at::kBFloat16, name, " has dtype ", in.scalar_type(), ", expected bfloat16");
    TORCH_CHECK_VALUE(in.dim() >= 1, name, " has no dimension");
    cols = in.size(-1);
    for (int64_t i = 0; i + 1 < in.dim(); ++i) rows *= in.size(i);
    stride = cols;
    bool even = cols <= 1 || in.stride(-1) == 1;
    if (in.dim() >= 2 && rows > 1) {
      // the leading dimensions have to be one
      int64_t expected = -1;
      for (int64_t i = in.dim() - 2; i >= 0 && even; --i) {
        if (in.size(i) == 1) continue;
        if (expected < 0) { stride = in.stride(i); expected = stride; }
        even = in.stride(i) == expected;
        expected *= in.size(i);
      }
    }
    if (rows > 0 && (!even || stride < 0 || stride % 8 || !aligned(in))) {
      t = packed(in);
      stride = cols;
    }
  }
};

struct Weight {
  const Tensor &w, &s;
  int64_t experts = 1, n, k;
  Weight(const Tensor& weight, const Tensor& weight_scale, bool many, bool gate, c10::Device dev) : w(weight), s(weight_scale) {
    bytes8(w, "weight", dev);
    TORCH_CHECK_VALUE(w.dim() == (many ? 3 : 2) && w.is_contiguous() && aligned(w), "weight must be contiguous ", many ? "[experts, N, K]" : "[N, K]",
                      " on a 16-byte boundary, got ", w.sizes());
    if (many) experts = w.size(0);
    n = w.size(-2);
    k = w.size(-1);
    TORCH_CHECK_VALUE(n >= 1 && n <= (1 << 24), "weight has ", n, " rows");
    inner(k, "weight");
    TORCH_CHECK_VALUE(experts >= 1 && experts <= MONO_LIN_MAX_EXPERTS, experts, " experts; 1 to ", MONO_LIN_MAX_EXPERTS, " are taken");
    TORCH_CHECK_VALUE(!gate || n % 256 == 0, "weight has ", n, " rows; with silu_mul each half needs a multiple of 128");
    typed(s, "weight_scale", at::kFloat, dev);
    const bool fits = s.dim() == w.dim() && s.size(-1) == groups(k) && s.size(-2) == groups(n) && (!many || s.size(0) == experts);
    TORCH_CHECK_VALUE(fits, "weight_scale has shape ", s.sizes(), ", expected one number for each block of 128 x 128 of the weight ", w.sizes());
  }
  Tensor scale() const { return s.is_contiguous() ? s : s.contiguous(); }
};

// Codes and scales of rows that are given in 8 bits.
struct Codes {
  Tensor q, s;
  int64_t rows = 1;
  Codes(const Tensor& x, const Tensor& xs, int64_t k) {
    const c10::Device dev = x.device();
    bytes8(x, "x", dev);
    typed(xs, "x_scale", at::kFloat, dev);
    TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) == k, "x has shape ", x.sizes(), ", the weight's rows have ", k);
    for (int64_t i = 0; i + 1 < x.dim(); ++i) rows *= x.size(i);
    bool fits = xs.dim() == x.dim() && xs.size(-1) == groups(k);
    for (int64_t i = 0; fits && i + 1 < x.dim(); ++i) fits = xs.size(i) == x.size(i);
    TORCH_CHECK_VALUE(fits, "x_scale has shape ", xs.sizes(), ", expected one number for 128 columns of x ", x.sizes());
    q = packed(x);
    s = xs.is_contiguous() ? xs : xs.contiguous();
  }
};

// ---- operators
PyObject* quantize(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  expect(n, 2);
  const bool silu = truth(a[1]);
  const Rows x(tensor(a[0], "x"), "x");
  TORCH_CHECK_VALUE(!silu || x.cols % 2 == 0, "x has rows of ", x.cols, "; with silu_mul they have two halves");
  const int64_t k = silu ? x.cols / 2 : x.cols;
  inner(k, silu ? "each half of x" : "x");
  const c10::Device dev = x.t.device();
  const c10::cuda::CUDAGuard guard(dev);
  const Block block(dev, {{with_last(x.t, k), at::kFloat8_e4m3fn}, {with_last(x.t, groups(k)), at::kFloat}});
  const Tensor &q = block[0], &s = block[1];
  launched("mono_lin_quantize", mono_lin_quantize(x.t.data_ptr(), x.stride, x.rows, static_cast<int>(k), silu, ptr<uint8_t>(q), ptr<float>(s), stream_of(dev)));
  return tuple({q, s});
  END_HANDLE_TH_ERRORS
}

PyObject* linear(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  expect(n, 7);
  const Tensor& x = tensor(a[0], "x");
  on_gpu(x, "x");
  const c10::Device dev = x.device();
  const bool silu = truth(a[5]), fp32 = truth(a[6]);
  const Weight w(tensor(a[1], "weight"), tensor(a[2], "weight_scale"), false, silu, dev);
  TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) == w.k, "x has shape ", x.sizes(), ", the weight's rows have ", w.k);
  TORCH_CHECK_VALUE(!(silu && (fp32 || a[4] != Py_None)), "silu_mul returns codes and scales; it takes no residual and no out_dtype");
  const c10::cuda::CUDAGuard guard(dev);
  Tensor residual;
  if (a[4] != Py_None) {
    const Tensor& r = tensor(a[4], "residual");
    typed(r, "residual", at::kBFloat16, dev);
    TORCH_CHECK_VALUE(r.sizes().equals(with_last(x, w.n)), "residual has shape ", r.sizes(), ", expected ", c10::IntArrayRef(with_last(x, w.n)));
    residual = packed(r);
  }
  Tensor out, out_s;
  if (silu) {
    const Block block(dev, {{with_last(x, w.n / 2), at::kFloat8_e4m3fn}, {with_last(x, w.n / 256), at::kFloat}});
    out = block[0];
    out_s = block[1];
  } else {
    out = empty(with_last(x, w.n), fp32 ? at::kFloat : at::kBFloat16, dev);
  }
  void* to = silu ? nullptr : out.data_ptr();
  uint8_t* codes_to = silu ? ptr<uint8_t>(out) : nullptr;
  const int wn = static_cast<int>(w.n), wk = static_cast<int>(w.k);
  const Tensor scale = w.scale();
  if (a[3] == Py_None) {
    const Rows in(x, "x");
    TORCH_CHECK_VALUE(in.rows <= INT32_MAX, "x has ", in.rows, " rows");
    if (in.rows <= MONO_LIN_FEW_ROWS && mono_lin_takes_rows(static_cast<int>(in.rows), wn, wk, silu)) {
      launched("mono_lin_product_rows", mono_lin_product_rows(in.t.data_ptr(), in.stride, static_cast<int>(in.rows), ptr<uint8_t>(w.w), ptr<float>(scale), wn, wk, to, fp32,
                                                              ptr<void>(residual), codes_to, ptr<float>(out_s), status(dev), stream_of(dev)));
    } else {
      const int64_t of_codes = in.rows * w.k;
      const Tensor q = empty({of_codes + in.rows * groups(w.k) * 4}, at::kByte, dev);      // codes, then scales
      uint8_t* codes = ptr<uint8_t>(q);
      float* scales = reinterpret_cast<float*>(codes + of_codes);
      launched("mono_lin_quantize", mono_lin_quantize(in.t.data_ptr(), in.stride, in.rows, wk, 0, codes, scales, stream_of(dev)));
      launched("mono_lin_product", mono_lin_product(codes, scales, in.rows, ptr<uint8_t>(w.w), ptr<float>(scale), wn, wk, to, fp32, ptr<void>(residual), codes_to,
                                                    ptr<float>(out_s), 1, status(dev), stream_of(dev)));
    }
  } else {
    const Codes in(x, tensor(a[3], "x_scale"), w.k);
    TORCH_CHECK_VALUE(in.rows <= INT32_MAX, "x has ", in.rows, " rows");
    launched("mono_lin_product", mono_lin_product(ptr<uint8_t>(in.q), ptr<float>(in.s), in.rows, ptr<uint8_t>(w.w), ptr<float>(scale), wn, wk, to, fp32, ptr<void>(residual),
                                                  codes_to, ptr<float>(out_s), 0, status(dev), stream_of(dev)));
  }
  if (silu) return tuple({out, out_s});
  return THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

const Tensor& ids_of(PyObject* o) {
  const Tensor& in = tensor(o, "ids");
  on_gpu(in, "ids");
  TORCH_CHECK_VALUE(in.scalar_type() == at::kInt || in.scalar_type() == at::kLong, "ids has dtype ", in.scalar_type(), ", expected int32 or int64");
  TORCH_CHECK_VALUE(in.dim() == 2 && in.size(1) >= 1 && in.size(1) <= MONO_LIN_MAX_TOP, "ids has shape ", in.sizes(), ", expected [tokens, 1 to ", MONO_LIN_MAX_TOP, "]");
  TORCH_CHECK_VALUE(in.numel() <= INT32_MAX, "ids has ", in.numel(), " slots; 2^31 - 1 are counted");
  return in;
}

PyObject* plan(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  expect(n, 2);
  const Tensor& in = ids_of(a[0]);
  const c10::Device dev = in.device();
  const int64_t experts = integer(a[1], "num_experts"), tokens = in.size(0), top = in.size(1);
  TORCH_CHECK_VALUE(experts >= 1 && experts <= MONO_LIN_MAX_EXPERTS, experts, " experts; 1 to ", MONO_LIN_MAX_EXPERTS, " are taken");
  const c10::cuda::CUDAGuard guard(dev);
  const Tensor ids = in.is_contiguous() ? in : in.contiguous();
  const Block block(dev, {{{experts + 1}, at::kInt}, {{tokens * top}, at::kInt}, {{tokens, top}, at::kInt}});
  const Tensor &offsets = block[0], &rows = block[1], &positions = block[2];
  launched("mono_lin_plan", mono_lin_plan(ids.data_ptr(), ids.scalar_type() == at::kLong, tokens, static_cast<int>(top), static_cast<int>(experts),
                                          ptr<int32_t>(offsets), ptr<int32_t>(rows), ptr<int32_t>(positions), status(dev), stream_of(dev)));
  return tuple({offsets, rows, positions});
  END_HANDLE_TH_ERRORS
}

Tensor vector(const Tensor& t, const char* name, c10::Device dev) {
  typed(t, name, at::kInt, dev);
  TORCH_CHECK_VALUE(t.dim() == 1, name, " has shape ", t.sizes(), ", expected one dimension");
  return t.is_contiguous() ? t : t.contiguous();
}

PyObject* experts(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  expect(n, 8);
  const Tensor& x = tensor(a[0], "x");
  on_gpu(x, "x");
  const c10::Device dev = x.device();
  const bool gather = truth(a[6]), silu = truth(a[7]);
  const Weight w(tensor(a[1], "weight"), tensor(a[2], "weight_scale"), true, silu, dev);
  TORCH_CHECK_VALUE(x.dim() == 2 && x.size(1) == w.k, "x has shape ", x.sizes(), ", expected [rows, ", w.k, "]");
  const c10::cuda::CUDAGuard guard(dev);
  const Tensor offsets = vector(tensor(a[3], "plan.offsets"), "plan.offsets", dev), tokens = vector(tensor(a[4], "plan.tokens"), "plan.tokens", dev);
  TORCH_CHECK_VALUE(offsets.numel() == w.experts + 1, "plan is one of ", offsets.numel() - 1, " experts, the weight of ", w.experts);
  const int64_t rows = tokens.numel();
  TORCH_CHECK_VALUE(gather || x.size(0) == rows, "x has ", x.size(0), " rows, the plan ", rows, "; with gather the tokens' rows are taken");
  TORCH_CHECK_VALUE(!gather || x.size(0) > 0 || rows == 0, "x has no rows for a plan of ", rows);
  TORCH_CHECK_VALUE(rows <= INT32_MAX && x.size(0) <= INT32_MAX, "x has ", x.size(0), " rows");
  Tensor out, out_s;
  if (silu) {
    const Block block(dev, {{{rows, w.n / 2}, at::kFloat8_e4m3fn}, {{rows, w.n / 256}, at::kFloat}});
    out = block[0];
    out_s = block[1];
  } else {
    out = empty({rows, w.n}, at::kBFloat16, dev);
  }
  const Tensor scale = w.scale();
  Tensor q, s;
  if (a[5] == Py_None) {
    const Rows in(x, "x");
    const Block block(dev, {{{x.size(0), w.k}, at::kByte}, {{x.size(0), groups(w.k)}, at::kFloat}});
    q = block[0];
    s = block[1];
    launched("mono_lin_quantize", mono_lin_quantize(in.t.data_ptr(), in.stride, in.rows, static_cast<int>(w.k), 0, ptr<uint8_t>(q), ptr<float>(s), stream_of(dev)));
  } else {
    const Codes in(x, tensor(a[5], "x_scale"), w.k);
    q = in.q;
    s = in.s;
  }
  if (rows > 0)
    launched("mono_lin_experts",
             mono_lin_experts(ptr<uint8_t>(q), ptr<float>(s), x.size(0), gather ? ptr<int32_t>(tokens) : nullptr, ptr<int32_t>(offsets), rows,
                              static_cast<int>(w.experts), ptr<uint8_t>(w.w), ptr<float>(scale), static_cast<int>(w.n), static_cast<int>(w.k),
                              silu ? nullptr : out.data_ptr(), silu ? ptr<uint8_t>(out) : nullptr, ptr<float>(out_s), status(dev), stream_of(dev)));
  if (silu) return tuple({out, out_s});
  return THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

void residual_fits(const Tensor& r, int64_t tokens, int64_t cols, c10::Device dev) {
  typed(r, "residual", at::kBFloat16, dev);
  TORCH_CHECK_VALUE(r.dim() == 2 && r.size(0) == tokens && r.size(1) == cols, "residual has shape ", r.sizes(), ", expected [", tokens, ", ", cols, "]");
}

PyObject* combine(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  expect(n, 4);
  const Tensor& partial_in = tensor(a[0], "partial");
  on_gpu(partial_in, "partial");
  const c10::Device dev = partial_in.device();
  typed(partial_in, "partial", at::kBFloat16, dev);
  TORCH_CHECK_VALUE(partial_in.dim() == 2, "partial has shape ", partial_in.sizes(), ", expected [rows, columns]");
  const int64_t cols = partial_in.size(1);
  TORCH_CHECK_VALUE(cols >= 8 && cols % 8 == 0 && cols <= (1 << 24), "partial has rows of ", cols, "; a multiple of 8 up to 2^24 is needed");
  const Tensor &pos_in = tensor(a[1], "positions"), &w_in = tensor(a[2], "weights");
  typed(pos_in, "positions", at::kInt, dev);
  typed(w_in, "weights", at::kFloat, dev);
  TORCH_CHECK_VALUE(pos_in.dim() == 2 && pos_in.size(1) >= 1 && pos_in.size(1) <= MONO_LIN_MAX_TOP, "positions has shape ", pos_in.sizes(), ", expected [tokens, 1 to ",
                    MONO_LIN_MAX_TOP, "]");
  TORCH_CHECK_VALUE(w_in.sizes() == pos_in.sizes(), "weights has shape ", w_in.sizes(), ", positions ", pos_in.sizes());
  const int64_t tokens = pos_in.size(0);
  const c10::cuda::CUDAGuard guard(dev);
  const Tensor partial = packed(partial_in), pos = pos_in.is_contiguous() ? pos_in : pos_in.contiguous(), w = w_in.is_contiguous() ? w_in : w_in.contiguous();
  Tensor residual;
  if (a[3] != Py_None) {
    const Tensor& r = tensor(a[3], "residual");
    residual_fits(r, tokens, cols, dev);
    residual = packed(r);
  }
  const Tensor out = empty({tokens, cols}, at::kBFloat16, dev);
  launched("mono_lin_combine", mono_lin_combine(partial.data_ptr(), partial.size(0), ptr<int32_t>(pos), ptr<float>(w), tokens, static_cast<int>(pos.size(1)),
                                                static_cast<int>(cols), ptr<void>(residual), out.data_ptr(), status(dev), stream_of(dev)));
  return THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

// What the operators of a layer refuse of its arguments (x, ids, weights, w13, w13_scale, w2, w2_scale, residual), before the first of them runs.
PyObject* check_layer(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  expect(n, 8);
  const Tensor& x = tensor(a[0], "x");
  on_gpu(x, "x");
  const c10::Device dev = x.device();
  typed(x, "x", at::kBFloat16, dev);
  const Tensor &ids = ids_of(a[1]), &weights = tensor(a[2], "weights");
  TORCH_CHECK_VALUE(ids.device() == dev, "ids is on ", ids.device(), ", expected ", dev);
  typed(weights, "weights", at::kFloat, dev);
  const Weight w13(tensor(a[3], "w13"), tensor(a[4], "w13_scale"), true, true, dev), w2(tensor(a[5], "w2"), tensor(a[6], "w2_scale"), true, false, dev);
  const bool fits = x.dim() == 2 && ids.size(0) == x.size(0) && weights.sizes() == ids.sizes() && w13.k == x.size(1) && w2.n == x.size(1) &&
                    w2.k == w13.n / 2 && w2.experts == w13.experts;
  TORCH_CHECK_VALUE(fits, "x ", x.sizes(), ", ids ", ids.sizes(), ", weights ", weights.sizes(), ", w13 ", w13.w.sizes(), " and w2 ", w2.w.sizes(),
                    " are not of one layer; expected [tokens, H], [tokens, top] twice, [experts, 2 I, H] and [experts, H, I]");
  if (a[7] != Py_None) residual_fits(tensor(a[7], "residual"), x.size(0), x.size(1), dev);
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

// The status word of a device, int32 [2].
PyObject* status_tensor(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  expect(n, 1);
  return THPVariable_Wrap(status_word(static_cast<c10::DeviceIndex>(integer(a[0], "device"))));
  END_HANDLE_TH_ERRORS
}

#define FAST(f) {#f, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(f)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {FAST(quantize), FAST(linear), FAST(plan), FAST(experts), FAST(combine), FAST(check_layer), FAST(status_tensor), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_mono_linear", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__mono_linear() { return PyModule_Create(&module); }
