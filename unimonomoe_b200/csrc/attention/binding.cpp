// Python module of the attention operators: checks of arguments, outputs and workspaces, and the call of the C ABI
// (include/mono_attention.h) on the current stream. Arguments come positionally from unimonomoe_b200/attention.py, which has the
// documentation. In C++ because a call is to cost the host a few microseconds: in Python the checks and allocations alone took
// fifteen to twenty, several times what the small launches take on the GPU.
#include <ATen/ATen.h>
#include <c10/core/InferenceMode.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <array>
#include <cmath>
#include <map>
#include <utility>
#include <vector>

#include "../../../include/mono_attention.h"

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
double number(PyObject* o, const char* name) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) {
    PyErr_Clear();
    throw c10::TypeError({__func__, __FILE__, static_cast<uint32_t>(__LINE__)}, c10::str(name, " must be a number, got ", Py_TYPE(o)->tp_name));
  }
  return v;
}
bool truth(PyObject* o) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) throw python_error();
  return v != 0;
}
int size32(int64_t v, const char* name) {
  TORCH_CHECK_VALUE(v >= 0 && v <= INT32_MAX, name, " is ", v);
  return static_cast<int>(v);
}

void on_gpu(const Tensor& t, const char* name) {
  TORCH_CHECK_VALUE(t.is_cuda(), name, " is on ", t.device(), "; these operators need a CUDA device, there is no CPU path");
}
void typed(const Tensor& t, const char* name, at::ScalarType type, c10::Device device) {
  on_gpu(t, name);
  TORCH_CHECK_VALUE(t.scalar_type() == type, name, " has dtype ", t.scalar_type(), ", expected ", type);
  TORCH_CHECK_VALUE(t.device() == device, name, " is on ", t.device(), ", expected ", device);
}
Tensor vector(const Tensor& t, const char* name, int64_t n, c10::Device device, at::ScalarType type = at::kInt) {
  typed(t, name, type, device);
  TORCH_CHECK_VALUE(t.dim() == 1 && t.size(0) == n, name, " has shape ", t.sizes(), ", expected [", n, "]");
  return t.is_contiguous() ? t : t.contiguous();
}
bool aligned(const Tensor& t) { return (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0; }

// bf16 [tokens, heads, head_dim] with 16-byte rows; any other layout is copied into one.
Tensor rows(const Tensor& t, const char* name, c10::Device device) {
  typed(t, name, at::kBFloat16, device);
  TORCH_CHECK_VALUE(t.dim() == 3, name, " has shape ", t.sizes(), ", expected [tokens, heads, head_dim]");
  if (t.stride(2) == 1 && ((t.stride(0) | t.stride(1)) & 7) == 0 && aligned(t)) return t;
  Tensor c = t.contiguous();
  return aligned(c) ? c : c.clone();
}
void head_dim(int64_t d) { TORCH_CHECK_VALUE(d == 64 || d == 128 || d == 256, "head size ", d, "; the kernels have 64, 128 and 256"); }
void page_size(int64_t p) {
  TORCH_CHECK_VALUE(p >= 16 && p <= 1024 && !(p & (p - 1)), "page size ", p, "; a power of two from 16 to 1024 is needed");
}

// The cache's tensor, checked as KV4Cache does when it is made: here is where its pointer and sizes are used.
struct Cache {
  const Tensor& data;
  int64_t pages, heads, dim;
  int page;
  explicit Cache(const Tensor& d) : data(d) {
    TORCH_CHECK_VALUE(d.dim() == 4 && d.scalar_type() == at::kByte && d.is_contiguous() && d.size(0) > 0 && d.size(1) > 0 && d.size(3) % 17 == 0 && aligned(d),
                      "cache must be contiguous uint8 [num_pages, kv_heads, page_size / 16, 17 * head_dim] on a 16-byte boundary, got ", d.sizes(), " ",
                      d.scalar_type());
    pages = d.size(0);
    heads = d.size(1);
    dim = d.size(3) / 17;
    head_dim(dim);
    page_size(std::min<int64_t>(d.size(2), 1 << 20) * 16);
    page = static_cast<int>(d.size(2)) * 16;
  }
  uint8_t* ptr() const { return static_cast<uint8_t*>(data.data_ptr()); }
  void check(int64_t kv_heads, int64_t d, c10::Device device) const {
    TORCH_CHECK_VALUE(heads == kv_heads && dim == d && data.device() == device, "cache holds ", heads, " KV heads of ", dim, " on ",
                      data.device(), ", the call has ", kv_heads, " of ", d, " on ", device);
  }
};

Tensor empty(at::IntArrayRef shape, at::ScalarType type, c10::Device device) {
  return at::empty(shape, at::TensorOptions().dtype(type).device(device));
}

// Several one-dimensional tensors in one allocation: an allocation costs the host more than all the rest of one.
class Block {
 public:
  Block(c10::Device device, std::initializer_list<std::pair<int64_t, at::ScalarType>> parts) {
    int64_t bytes = 0;
    for (const auto& [n, type] : parts) bytes += padded(n, type);
    base_ = empty({bytes}, at::kByte, device);
    int64_t at = 0;
    for (const auto& [n, type] : parts) {
      Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(base_.storage()), base_.key_set(), c10::scalarTypeToTypeMeta(type));
      t.unsafeGetTensorImpl()->set_storage_offset(at / static_cast<int64_t>(c10::elementSize(type)));
      t.unsafeGetTensorImpl()->set_sizes_contiguous({n});
      tensors_.push_back(std::move(t));
      at += padded(n, type);
    }
  }
  const Tensor& operator[](size_t i) const { return tensors_[i]; }

 private:
  static int64_t padded(int64_t n, at::ScalarType type) { return (n * static_cast<int64_t>(c10::elementSize(type)) + 15) / 16 * 16; }
  Tensor base_;
  std::vector<Tensor> tensors_;
};

// ---- what is kept: a status word for each device, a workspace for each stream of a device. Never freed: a captured graph may
// hold their addresses, and at exit the allocator is gone before them.
//
// The word is zeroed once, before any launch that may report into it, whatever stream that goes to; and not as a part of a graph, each replay of which
// would wipe what was reported before. So it is made on a stream that is not being captured, and waited for. Nor as an inference tensor, which
// check_status could not write outside of that mode.
Tensor& status_word(c10::DeviceIndex device) {
  static auto* words = new std::array<Tensor, 64>();
  Tensor& t = words->at(device);
  if (t.defined()) return t;
  const c10::InferenceMode normal(false);
  const c10::cuda::CUDAStreamCaptureModeGuard relaxed(cudaStreamCaptureModeRelaxed);   // allocating and waiting beside a capture
  c10::cuda::CUDAStreamGuard side(c10::cuda::getStreamFromPool(true, device));
  while (c10::cuda::currentStreamCaptureStatusMayInitCtx() != c10::cuda::CaptureStatus::None) side.reset_stream(c10::cuda::getStreamFromPool(true, device));
  const Tensor w = at::zeros({2}, at::TensorOptions().dtype(at::kInt).device(at::kCUDA, device));
  side.current_stream().synchronize();
  return t = w;
}
uint32_t* status(c10::DeviceIndex device) { return static_cast<uint32_t*>(status_word(device).data_ptr()); }

// Counters zero. A capture that finds none gets a workspace of its own, so that the capture's memory pool owns it.
Tensor workspace(c10::DeviceIndex device, cudaStream_t stream) {
  static auto* kept = new std::map<std::pair<int, cudaStream_t>, Tensor>();
  const auto it = kept->find({device, stream});
  if (it != kept->end()) return it->second;
  Tensor w = at::empty({static_cast<int64_t>(mono_attn_workspace_bytes())}, at::TensorOptions().dtype(at::kByte).device(at::kCUDA, device));
  w.narrow(0, 0, MONO_ATTN_COUNTERS * 4).zero_();
  if (c10::cuda::currentStreamCaptureStatusMayInitCtx() == c10::cuda::CaptureStatus::None) kept->emplace(std::make_pair(static_cast<int>(device), stream), w);
  return w;
}

void launched(const char* name, int rc) {
  const char* why = rc == MONO_ATTN_NULL          ? " (a required pointer is null)"
                    : rc == MONO_ATTN_BAD_SIZE     ? " (a size is out of its range)"
                    : rc == MONO_ATTN_BAD_HEAD_DIM ? " (head size is not 64, 128 or 256)"
                    : rc == MONO_ATTN_WORKSPACE    ? " (workspace too small)"
                                                   : "";
  TORCH_CHECK(rc == 0, name, " failed: rc=", rc, why);
}

template <typename T>
T* ptr(const Tensor& t) { return static_cast<T*>(t.data_ptr()); }
mono_attn_stream_t stream_of(c10::Device device) {
  return reinterpret_cast<mono_attn_stream_t>(c10::cuda::getCurrentCUDAStream(device.index()).stream());
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

// ---- operators
PyObject* plan(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  expect(n, 7);
  const Tensor &cached_in = tensor(a[0], "cached_lens"), &table = tensor(a[2], "block_table");
  on_gpu(cached_in, "cached_lens");
  const c10::Device dev = cached_in.device();
  const int64_t batch = cached_in.numel();
  TORCH_CHECK_VALUE(batch >= 1 && batch <= MONO_ATTN_MAX_REQUESTS, batch, " requests; 1 to ", MONO_ATTN_MAX_REQUESTS, " are planned at a time");
  const Tensor cached = vector(cached_in, "cached_lens", batch, dev), fresh = vector(tensor(a[1], "new_lens"), "new_lens", batch, dev);
  typed(table, "block_table", at::kInt, dev);
  TORCH_CHECK_VALUE(table.dim() == 2 && table.size(0) == batch && table.size(1) >= 1 && table.is_contiguous(), "block_table must be contiguous int32 [",
                    batch, ", pages], got ", table.sizes());
  const Tensor &free_in = tensor(a[3], "free_pages"), free = vector(free_in, "free_pages", free_in.numel(), dev);
  const Tensor taken = vector(tensor(a[4], "taken"), "taken", 1, dev);
  const int64_t page = integer(a[5], "page_size");
  page_size(page);
  const int tokens = size32(integer(a[6], "num_tokens"), "num_tokens");
  const c10::cuda::CUDAGuard guard(dev);
  const Block block(dev, {{batch + 1, at::kInt}, {batch, at::kInt}, {tokens, at::kInt}, {tokens, at::kLong}, {tokens, at::kInt}, {1, at::kInt}});
  const Tensor &start = block[0], &lens = block[1], &positions = block[2], &slots = block[3], &requests = block[4], &taken_out = block[5];
  launched("mono_attn_plan",
           mono_attn_plan(ptr<int32_t>(cached), ptr<int32_t>(fresh), static_cast<int>(batch), ptr<int32_t>(table), size32(table.size(1), "pages of block_table"),
                          ptr<int32_t>(free), size32(free.numel(), "free_pages"), ptr<int32_t>(taken), static_cast<int>(page), tokens,
                          ptr<int32_t>(start), ptr<int32_t>(lens), ptr<int32_t>(positions), ptr<int64_t>(slots), ptr<int32_t>(requests),
                          ptr<int32_t>(taken_out), status(dev.index()), stream_of(dev)));
  return tuple({start, lens, positions, slots, requests, taken_out});
  END_HANDLE_TH_ERRORS
}

PyObject* qk_norm_rope(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  expect(n, 12);
  const Tensor& q_in = tensor(a[0], "q");
  on_gpu(q_in, "q");
  const c10::Device dev = q_in.device();
  const Tensor q = rows(q_in, "q", dev), k = rows(tensor(a[1], "k"), "k", dev);
  const int64_t T = q.size(0), H = q.size(1), D = q.size(2), K = k.size(1);
  head_dim(D);
  TORCH_CHECK_VALUE(k.size(0) == T && k.size(2) == D && H > 0 && K > 0, "q is ", q.sizes(), ", k is ", k.sizes(), ": tokens and head size must agree");
  const Tensor &wq = tensor(a[2], "q_weight"), &wk = tensor(a[3], "k_weight");
  const at::ScalarType wt = wq.scalar_type();
  TORCH_CHECK_VALUE((wt == at::kBFloat16 || wt == at::kFloat) && wk.scalar_type() == wt, "norm weights must both be bfloat16 or float32, got ", wt,
                    " and ", wk.scalar_type());
  for (const auto& [name, w] : {std::pair<const char*, const Tensor&>{"q_weight", wq}, {"k_weight", wk}}) {
    typed(w, name, wt, dev);
    TORCH_CHECK_VALUE(w.dim() == 1 && w.size(0) == D && w.is_contiguous() && aligned(w), name, " must be contiguous [", D, "] on a 16-byte boundary, got ",
                      w.sizes());
  }
  const Tensor& table = tensor(a[4], "cos_sin");
  typed(table, "cos_sin", at::kFloat, dev);
  TORCH_CHECK_VALUE(table.dim() == 2 && table.is_contiguous() && aligned(table), "cos_sin must be contiguous fp32 [positions, rotary_dim], got ", table.sizes());
  const int64_t R = table.size(1);
  TORCH_CHECK_VALUE(R % 16 == 0 && R <= D, "rotary dim ", R, "; a multiple of 16 up to the head size ", D, " is needed");
  TORCH_CHECK_VALUE(R == 0 || table.size(0) > 0, "cos_sin has no rows");
  const Tensor positions = vector(tensor(a[5], "positions"), "positions", T, dev);
  const double eps = number(a[6], "eps");
  const bool interleaved = truth(a[7]), unit = truth(a[8]), store = a[10] != Py_None;
  Tensor v, slots;
  const Tensor* data = nullptr;
  if (store) {
    TORCH_CHECK_VALUE(a[9] != Py_None && a[11] != Py_None, "storing into a cache needs v and slots");
    data = &tensor(a[10], "cache");
    v = rows(tensor(a[9], "v"), "v", dev);
    TORCH_CHECK_VALUE(v.sizes() == k.sizes(), "v is ", v.sizes(), ", k is ", k.sizes());
    Cache(*data).check(K, D, dev);
    slots = vector(tensor(a[11], "slots"), "slots", T, dev, at::kLong);
  } else {
    TORCH_CHECK_VALUE(a[9] == Py_None && a[11] == Py_None, "v and slots are stored in a cache, and none is given");
  }
  const c10::cuda::CUDAGuard guard(dev);
  const Tensor q_out = empty({T, H, D}, at::kBFloat16, dev), k_out = store ? Tensor() : empty({T, K, D}, at::kBFloat16, dev);
  if (T > 0)
    launched("mono_attn_qk_norm_rope",
             mono_attn_qk_norm_rope(q.data_ptr(), q.stride(0), q.stride(1), k.data_ptr(), k.stride(0), k.stride(1), wq.data_ptr(), wk.data_ptr(),
                                    wt == at::kFloat, unit, static_cast<float>(eps), ptr<float>(table), size32(table.size(0), "positions of cos_sin"),
                                    static_cast<int>(R), interleaved, ptr<int32_t>(positions), size32(T, "tokens"), size32(H, "heads"), size32(K, "KV heads"),
                                    static_cast<int>(D), q_out.data_ptr(), store ? nullptr : k_out.data_ptr(), store ? v.data_ptr() : nullptr,
                                    store ? v.stride(0) : 0, store ? v.stride(1) : 0, store ? ptr<uint8_t>(*data) : nullptr, store ? data->size(0) : 0,
                                    store ? Cache(*data).page : 16, store ? ptr<int64_t>(slots) : nullptr, status(dev.index()), stream_of(dev)));
  if (store) return THPVariable_Wrap(q_out);
  return tuple({q_out, k_out});
  END_HANDLE_TH_ERRORS
}

PyObject* kv4_append(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  expect(n, 4);
  const Tensor& k_in = tensor(a[0], "k");
  on_gpu(k_in, "k");
  const c10::Device dev = k_in.device();
  const Tensor k = rows(k_in, "k", dev), v = rows(tensor(a[1], "v"), "v", dev);
  const int64_t T = k.size(0), K = k.size(1), D = k.size(2);
  TORCH_CHECK_VALUE(v.sizes() == k.sizes(), "v is ", v.sizes(), ", k is ", k.sizes());
  const Cache cache(tensor(a[2], "cache"));
  cache.check(K, D, dev);
  const Tensor slots = vector(tensor(a[3], "slots"), "slots", T, dev, at::kLong);
  if (T > 0) {
    const c10::cuda::CUDAGuard guard(dev);
    launched("mono_attn_kv4_append",
             mono_attn_kv4_append(k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(), v.stride(0), v.stride(1), size32(T, "tokens"), static_cast<int>(K),
                                  static_cast<int>(D), cache.ptr(), cache.pages, cache.page, ptr<int64_t>(slots), status(dev.index()), stream_of(dev)));
  }
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

PyObject* kv4_read(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  expect(n, 2);
  const Cache cache(tensor(a[0], "cache"));
  on_gpu(cache.data, "cache");
  const c10::Device dev = cache.data.device();
  const Tensor& slots_in = tensor(a[1], "slots");
  const int64_t T = slots_in.numel();
  const Tensor slots = vector(slots_in, "slots", T, dev, at::kLong);
  const c10::cuda::CUDAGuard guard(dev);
  const Tensor k = empty({T, cache.heads, cache.dim}, at::kBFloat16, dev), v = empty({T, cache.heads, cache.dim}, at::kBFloat16, dev);
  if (T > 0)
    launched("mono_attn_kv4_read", mono_attn_kv4_read(cache.ptr(), cache.pages, cache.page, ptr<int64_t>(slots), size32(T, "tokens"), static_cast<int>(cache.heads),
                                                      static_cast<int>(cache.dim), k.data_ptr(), v.data_ptr(), status(dev.index()), stream_of(dev)));
  return tuple({k, v});
  END_HANDLE_TH_ERRORS
}

PyObject* kv4_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  expect(n, 10);
  const Tensor& q_in = tensor(a[0], "q");
  on_gpu(q_in, "q");
  const c10::Device dev = q_in.device();
  const Tensor q = rows(q_in, "q", dev);
  const int64_t T = q.size(0), H = q.size(1), D = q.size(2);
  const Cache cache(tensor(a[1], "cache"));
  cache.check(cache.heads, D, dev);
  TORCH_CHECK_VALUE(H > 0 && H % cache.heads == 0, H, " query heads over ", cache.heads, " KV heads");
  const Tensor &table = tensor(a[2], "block_table"), &lens_in = tensor(a[3], "seq_lens");
  const int64_t B = lens_in.numel();
  typed(table, "block_table", at::kInt, dev);
  TORCH_CHECK_VALUE(table.dim() == 2 && table.size(0) == B && table.size(1) >= 1 && table.is_contiguous(), "block_table must be contiguous int32 [", B,
                    ", pages], got ", table.sizes());
  TORCH_CHECK_VALUE(B <= MONO_ATTN_MAX_REQUESTS, B, " requests; up to ", MONO_ATTN_MAX_REQUESTS, " are taken at a time");
  const Tensor lens = vector(lens_in, "seq_lens", B, dev), start = vector(tensor(a[4], "query_start"), "query_start", B + 1, dev);
  const int64_t longest = integer(a[5], "max_query_len"), window = integer(a[7], "window");
  TORCH_CHECK_VALUE(window >= 0 && longest >= 0, "window is ", window, ", max_query_len is ", longest);
  const double scale = a[6] == Py_None ? 1.0 / std::sqrt(static_cast<double>(D)) : number(a[6], "scale");
  TORCH_CHECK_VALUE(std::isfinite(static_cast<float>(scale)), "scale is ", scale, "; a finite number of 32 bits is needed");
  const bool want_lse = truth(a[9]);
  const c10::cuda::CUDAGuard guard(dev);
  Tensor out;
  if (a[8] == Py_None) {
    out = empty({T, H, D}, at::kBFloat16, dev);
  } else {
    out = tensor(a[8], "out");
    typed(out, "out", at::kBFloat16, dev);
    TORCH_CHECK_VALUE(out.sizes() == q.sizes() && out.is_contiguous() && aligned(out), "out must be contiguous bfloat16 [", T, ", ", H, ", ", D,
                      "] on a 16-byte boundary, got ", out.sizes());
  }
  const Tensor lse = want_lse ? empty({T, H}, at::kFloat, dev) : Tensor();
  if (T > 0 && B > 0) {
    const mono_attn_stream_t stream = stream_of(dev);
    const Tensor ws = workspace(dev.index(), reinterpret_cast<cudaStream_t>(stream));
    launched("mono_attn_kv4_attention",
             mono_attn_kv4_attention(q.data_ptr(), q.stride(0), q.stride(1), cache.ptr(), cache.pages, cache.page, ptr<int32_t>(table),
                                     size32(table.size(1), "pages of block_table"), ptr<int32_t>(lens), ptr<int32_t>(start), static_cast<int>(B),
                                     size32(T, "tokens"), static_cast<int>(std::min<int64_t>(longest, INT32_MAX)), size32(H, "heads"),
                                     static_cast<int>(cache.heads), static_cast<int>(D), static_cast<float>(scale),
                                     static_cast<int>(std::min<int64_t>(window, INT32_MAX)), out.data_ptr(), want_lse ? ptr<float>(lse) : nullptr, ws.data_ptr(),
                                     static_cast<size_t>(ws.numel()), status(dev.index()), stream));
  }
  PyObject* o = a[8] == Py_None ? THPVariable_Wrap(out) : Py_NewRef(a[8]);
  if (!want_lse) return o;
  PyObject* r = PyTuple_New(2);
  if (!r) throw python_error();
  PyTuple_SET_ITEM(r, 0, o);
  PyTuple_SET_ITEM(r, 1, THPVariable_Wrap(lse));
  return r;
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
PyMethodDef methods[] = {FAST(plan), FAST(qk_norm_rope), FAST(kv4_append), FAST(kv4_read), FAST(kv4_attention), FAST(status_tensor), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_mono_attention", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__mono_attention() { return PyModule_Create(&module); }
