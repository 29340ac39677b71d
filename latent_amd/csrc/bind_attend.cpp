// The attention calls of include/latent_ffn.h on torch tensors: argument checks,
// the copies that strides or alignment ask for, outputs, scratch, the stream.
//
// A step's calls are a few microseconds of GPU each, less than the interpreter
// takes to look at their ten tensors (append of one token: 11 us a call from
// Python and ctypes, of which the launch is 3; 5 from here).  The library itself
// keeps its C ABI and knows no torch: its entry points come as addresses.
#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <c10/core/AutogradState.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/GradMode.h>
#include <c10/core/impl/VirtualGuardImpl.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>

#include "../../include/latent_ffn.h"

namespace {

using at::Tensor;

decltype(&latent_kv_append) append_entry;
decltype(&latent_attn_decode_workspace_size) decode_size_entry;
decltype(&latent_attn_decode) decode_entry;
decltype(&latent_attn_prompt_workspace_size) prompt_size_entry;
decltype(&latent_attn_prompt) prompt_entry;
PyObject* error_type;  // LatentError(status, call)

struct LatentFailure {
  int status;
  const char* call;
};
void check(int status, const char* call) {
  if (status != LATENT_OK) throw LatentFailure{status, call};
}

const Tensor& tensor(PyObject* o, const char* name) {
  TORCH_CHECK_TYPE(THPVariable_Check(o), name, " must be a tensor");
  return THPVariable_Unpack(o);
}

void check_grad(const Tensor& t) {
  TORCH_CHECK(!t.requires_grad() || !c10::GradMode::is_enabled(),
              "attention here has no backward pass: call it under torch.no_grad()");
  TORCH_CHECK(!c10::AutogradState::get_tls_state().get_fw_grad_mode() || !t._fw_grad(0).defined(),
              "attention here has no forward-mode derivative: its operands may not carry tangents");
}

// What a call wrote in place, for autograd's check of what it saved.  Inference tensors have no counter.
void written(const Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}
void written(PyObject* o) {
  if (o != Py_None) written(THPVariable_Unpack(o));
}

// The device of a call's first tensor.
c10::Device first(const Tensor& t, const char* name) {
  TORCH_CHECK_VALUE(t.is_cuda(), name, " must be a CUDA tensor");
  TORCH_CHECK_TYPE(t.scalar_type() == at::kHalf || t.scalar_type() == at::kBFloat16, name, " must be f16 or bf16");
  return t.device();
}
int32_t dtype_of(const Tensor& t) { return t.scalar_type() == at::kHalf ? LATENT_F16 : LATENT_BF16; }

bool fits(int64_t token, int64_t head, int64_t element, int64_t dim, const void* p) {
  return (element == 1 || dim < 2) && !((token | head) & 7) && !(reinterpret_cast<uintptr_t>(p) & 15);
}

// [tokens, heads, D] as the kernels read it: a copy where strides or base do not fit.
struct Heads {
  Tensor t;
  void* p;
  int64_t token, head;      // strides
  int64_t tokens, heads, D;
};
// Tokens further apart than this (elements) are copied together: the kernels step over a tile of them in 32 bits.
constexpr int64_t kFar = 1 << 22;
Heads heads(const Tensor& t, const char* name, c10::ScalarType dt, c10::Device dev) {
  TORCH_CHECK_VALUE(t.dim() == 3, name, " must be [tokens, heads, D]");
  TORCH_CHECK_TYPE(t.scalar_type() == dt, name, " must be ", dt, ", as the queries and the cache are");
  TORCH_CHECK_VALUE(t.device() == dev, name, " must be on ", dev);
  check_grad(t);
  Heads h{t, t.data_ptr(), t.stride(0), t.stride(1), t.size(0), t.size(1), t.size(2)};
  if (!fits(h.token, h.head, t.stride(2), h.D, h.p) || h.token >= kFar) {
    h.t = t.clone(at::MemoryFormat::Contiguous);
    h.p = h.t.data_ptr();
    h.token = h.t.stride(0);
    h.head = h.t.stride(1);
  }
  return h;
}

// The output: the one given, or a new one like q.
Heads output(PyObject* o, const Heads& q, const char* name) {
  Heads h = q;
  if (o == Py_None) {
    h.t = at::empty({q.tokens, q.heads, q.D}, q.t.options().requires_grad(false));
    h.head = q.D;
    h.token = q.heads * q.D;
  } else {
    h.t = tensor(o, name);
    TORCH_CHECK_VALUE(h.t.sizes() == q.t.sizes() && h.t.scalar_type() == q.t.scalar_type() && h.t.device() == q.t.device(), name,
                      " must be ", q.t.scalar_type(), " ", q.t.sizes(), " on ", q.t.device());
    check_grad(h.t);
    h.token = h.t.stride(0);
    h.head = h.t.stride(1);
    TORCH_CHECK_VALUE(fits(h.token, h.head, h.t.stride(2), h.D, h.t.data_ptr()), name,
                      " must have adjacent D, strides that are multiples of 8 and a 16-byte aligned base");
  }
  h.p = h.t.data_ptr();
  return h;
}
PyObject* result(PyObject* given, const Heads& out) {
  if (given == Py_None) return THPVariable_Wrap(out.t);
  Py_INCREF(given);
  return given;
}

Tensor ints(const Tensor& t, const char* name, int64_t n, c10::Device dev) {
  TORCH_CHECK_VALUE(t.scalar_type() == at::kInt && t.dim() == 1 && t.size(0) == n && t.device() == dev, name, " must be int32 [", n,
                    "] on ", dev);
  return t.is_contiguous() ? t : t.contiguous();
}

float* lse_of(PyObject* o, const Heads& q) {
  if (o == Py_None) return nullptr;
  const Tensor& t = tensor(o, "lse");
  TORCH_CHECK_VALUE(t.scalar_type() == at::kFloat && t.dim() == 2 && t.size(0) == q.tokens && t.size(1) == q.heads &&
                        t.device() == q.t.device() && t.is_contiguous(),
                    "lse must be contiguous f32 [", q.tokens, ", ", q.heads, "] on ", q.t.device());
  check_grad(t);
  return static_cast<float*>(t.data_ptr());
}

float scale_of(PyObject* o, int64_t D) {
  double s = o == Py_None ? 1.0 / std::sqrt(static_cast<double>(D)) : PyFloat_AsDouble(o);
  if (s == -1.0 && PyErr_Occurred()) throw python_error();
  TORCH_CHECK_VALUE(s > 0.0 && s < INFINITY, "scale must be positive and finite");
  return static_cast<float>(s);
}

bool truth(PyObject* o) {
  const int r = PyObject_IsTrue(o);
  if (r < 0) throw python_error();
  return r;
}

latent_kv_cache cache_of(const Tensor& k, const Tensor& v, const Tensor& pages, c10::ScalarType dt, c10::Device dev) {
  TORCH_CHECK_VALUE(k.dim() == 4 && v.sizes() == k.sizes(), "k_cache and v_cache must be [pages, page rows, kv heads, D], of one shape");
  TORCH_CHECK_TYPE(k.scalar_type() == dt && v.scalar_type() == dt, "k_cache and v_cache must be ", dt, ", as the call's other operands are");
  check_grad(k);
  check_grad(v);
  TORCH_CHECK_VALUE(k.device() == dev && v.device() == dev && pages.device() == dev, "the cache and its page table must be on ", dev);
  TORCH_CHECK_VALUE(pages.scalar_type() == at::kInt && pages.dim() == 2, "pages must be int32 [sequences, max_pages]");
  TORCH_CHECK_VALUE(((k.stride(3) == 1 && v.stride(3) == 1) || k.size(3) < 2) && (pages.stride(1) == 1 || pages.size(1) < 2),
                    "the last dimensions of k_cache, v_cache and pages must be adjacent");
  // A size of one makes its stride meaningless to torch, and so to the library.
  auto stride = [](const Tensor& t, int i) { return t.size(i) > 1 ? t.stride(i) : 0; };
  latent_kv_cache c{};
  c.k = k.data_ptr();
  c.v = v.data_ptr();
  c.pages = static_cast<const int32_t*>(pages.data_ptr());
  c.n_pages = k.size(0);
  c.page_size = k.size(1);
  c.n_seq = pages.size(0);
  c.max_pages = pages.size(1);
  c.pages_stride = c.n_seq > 1 ? pages.stride(0) : c.max_pages;
  c.k_page_stride = stride(k, 0), c.k_row_stride = stride(k, 1), c.k_head_stride = stride(k, 2);
  c.v_page_stride = stride(v, 0), c.v_row_stride = stride(v, 1), c.v_head_stride = stride(v, 2);
  return c;
}

// The scratch that is given, or what the call wants of its own.
struct Scratch {
  Tensor own;
  void* p = nullptr;
  size_t bytes = 0;
};
template <typename Args, typename Size>
Scratch scratch(PyObject* given, const Args& a, Size size, const char* call, const Tensor& q) {
  Scratch s;
  if (given != Py_None) {
    const Tensor& t = tensor(given, "workspace");
    TORCH_CHECK_VALUE(t.device() == q.device() && t.is_contiguous(), "workspace must be contiguous and on ", q.device());
    s.bytes = t.nbytes();
    s.p = s.bytes ? t.data_ptr() : nullptr;
    return s;
  }
  check(size(&a, &s.bytes), call);
  if (s.bytes) {
    s.own = at::empty({static_cast<int64_t>(s.bytes)}, q.options().dtype(at::kByte).requires_grad(false));
    s.p = s.own.data_ptr();
  }
  return s;
}

// Runs f with the tensors' device current and its current stream's handle.  Everything that f allocates it allocates there.
template <typename F>
PyObject* on_device(c10::Device dev, F f) {
  const c10::impl::VirtualGuardImpl impl(dev.type());
  c10::OptionalDeviceGuard guard;
  if (impl.getDevice() != dev) guard.reset_device(dev);
  return f(reinterpret_cast<latent_stream_t>(c10::hip::getCurrentHIPStream(dev.index()).stream()));
}
template <typename Entry, typename Args>
void launch(Entry entry, const Args& a, latent_stream_t stream, const char* call) {
  PyThreadState* state = PyEval_SaveThread();
  const int status = entry(&a, stream);
  PyEval_RestoreThread(state);
  check(status, call);
}

// f's errors as Python's.
template <typename F>
PyObject* guarded(Py_ssize_t n, Py_ssize_t want, F f) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == want, "expected ", want, " arguments");
  TORCH_CHECK(error_type, "the library's entry points are not set");
  try {
    return f();
  } catch (const LatentFailure& e) {
    if (PyObject* x = PyObject_CallFunction(error_type, "is", e.status, e.call)) {
      PyErr_SetObject(error_type, x);
      Py_DECREF(x);
    }
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

// kv_append(k, v, k_cache, v_cache, pages, positions, seqs, q, rope, interleaved, q_out)
PyObject* kv_append(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded(n, 11, [&]() -> PyObject* {
    const Tensor& k0 = tensor(args[0], "k");
    const c10::Device dev = first(k0, "k");
    return on_device(dev, [&](latent_stream_t stream) -> PyObject* {
      const auto dt = k0.scalar_type();
      latent_kv_append_args a{};
      a.cache = cache_of(tensor(args[2], "k_cache"), tensor(args[3], "v_cache"), tensor(args[4], "pages"), dt, dev);
      const Heads k = heads(k0, "k", dt, dev), v = heads(tensor(args[1], "v"), "v", dt, dev);
      const Tensor& cache = THPVariable_Unpack(args[2]);
      TORCH_CHECK_VALUE(cache.size(2) == k.heads && cache.size(3) == k.D && v.t.sizes() == k.t.sizes(), "k ", k.t.sizes(), ", v ",
                        v.t.sizes(), " and the cache ", cache.sizes(), " do not fit");
      Tensor seqs;
      if (args[6] != Py_None) {
        seqs = ints(tensor(args[6], "seqs"), "seqs", k.tokens, dev);
        a.seqs = static_cast<const int32_t*>(seqs.data_ptr());
      } else {
        TORCH_CHECK_VALUE(k.tokens <= a.cache.n_seq, "more tokens than sequences: give seqs");
      }
      const Tensor positions = ints(tensor(args[5], "positions"), "positions", k.tokens, dev);
      a.positions = static_cast<const int32_t*>(positions.data_ptr());
      Tensor rope;
      if (args[8] != Py_None) {
        rope = tensor(args[8], "rope");
        TORCH_CHECK_VALUE(rope.scalar_type() == at::kFloat && rope.dim() == 3 && rope.size(1) == 2 && rope.device() == dev,
                          "rope must be f32 [positions, 2, rot / 2] on ", dev);
        check_grad(rope);
        if (!rope.is_contiguous() || (reinterpret_cast<uintptr_t>(rope.data_ptr()) & 15)) rope = rope.clone(at::MemoryFormat::Contiguous);
        // A table without rows has no base, and no base would mean no rotation: any address serves, none of it is read.
        a.rope = static_cast<const float*>(rope.numel() ? rope.data_ptr() : k.p);
        a.rope_rows = rope.size(0);
        a.rot_dim = 2 * rope.size(2);
        TORCH_CHECK_VALUE(0 < a.rot_dim && a.rot_dim <= k.D, "rope turns ", a.rot_dim, " dimensions of ", k.D);
      }
      Heads q{}, out{};
      if (args[7] != Py_None) {
        q = heads(tensor(args[7], "q"), "q", dt, dev);
        TORCH_CHECK_VALUE(q.tokens == k.tokens && q.D == k.D, "q ", q.t.sizes(), " does not fit k ", k.t.sizes());
        out = output(args[10], q, "q_out");
      } else {
        TORCH_CHECK_VALUE(args[10] == Py_None, "q_out without q");
      }
      if (k.tokens) {
        a.q = q.p, a.q_out = out.p, a.k = k.p, a.v = v.p;
        a.q_token_stride = q.token, a.q_head_stride = q.head;
        a.q_out_token_stride = out.token, a.q_out_head_stride = out.head;
        a.k_token_stride = k.token, a.k_head_stride = k.head;
        a.v_token_stride = v.token, a.v_head_stride = v.head;
        a.n_tokens = k.tokens, a.n_head = q.heads, a.n_kv_head = k.heads, a.head_dim = k.D;
        a.dtype = dtype_of(k.t);
        a.rope_kind = truth(args[9]) ? LATENT_ROPE_INTERLEAVED : LATENT_ROPE_HALF;
        launch(append_entry, a, stream, "latent_kv_append");
        written(args[2]), written(args[3]), written(args[10]);
      }
      if (args[7] == Py_None) Py_RETURN_NONE;
      return result(args[10], out);
    });
  });
}

// attend_decode(q, k_cache, v_cache, pages, lengths, scale, out, lse, workspace)
PyObject* attend_decode(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded(n, 9, [&]() -> PyObject* {
    const Tensor& q0 = tensor(args[0], "q");
    const c10::Device dev = first(q0, "q");
    return on_device(dev, [&](latent_stream_t stream) -> PyObject* {
      const auto dt = q0.scalar_type();
      const Tensor& kc = tensor(args[1], "k_cache");
      latent_attn_decode_args a{};
      a.cache = cache_of(kc, tensor(args[2], "v_cache"), tensor(args[3], "pages"), dt, dev);
      const Heads q = heads(q0, "q", dt, dev);
      const int64_t kv = kc.size(2);
      TORCH_CHECK_VALUE(q.tokens == a.cache.n_seq && q.D == kc.size(3) && kv && q.heads % kv == 0, "q ", q.t.sizes(),
                        " does not fit the cache ", kc.sizes(), " of ", a.cache.n_seq, " sequences");
      const Tensor lengths = ints(tensor(args[4], "lengths"), "lengths", q.tokens, dev);
      const Heads out = output(args[6], q, "out");
      a.lse = lse_of(args[7], q);
      a.scale = scale_of(args[5], q.D);
      if (q.tokens && q.heads) {
        a.q = q.p, a.out = out.p;
        a.lengths = static_cast<const int32_t*>(lengths.data_ptr());
        a.q_token_stride = q.token, a.q_head_stride = q.head;
        a.out_token_stride = out.token, a.out_head_stride = out.head;
        a.n_head = q.heads, a.n_kv_head = kv, a.head_dim = q.D;
        a.dtype = dtype_of(q.t);
        const Scratch s = scratch(args[8], a, decode_size_entry, "latent_attn_decode", q.t);
        a.workspace = s.p, a.workspace_bytes = s.bytes;
        launch(decode_entry, a, stream, "latent_attn_decode");
        written(args[6]), written(args[7]);
      }
      return result(args[6], out);
    });
  });
}

// What attend_prompt and attend_prompt_paged share: queries, outputs, the call.  a holds keys, sequences and n_kv_head.
PyObject* prompt(latent_attn_prompt_args& a, const Heads& q, PyObject* starts_arg, bool causal, PyObject* const* rest /* scale, out, lse, workspace */,
                 c10::Device dev, latent_stream_t stream) {
  TORCH_CHECK_VALUE(a.n_kv_head && q.heads % a.n_kv_head == 0, q.heads, " heads are no multiple of ", a.n_kv_head, " key and value heads");
  const Tensor starts = ints(tensor(starts_arg, "starts"), "starts", a.cache.n_seq + 1, dev);
  const Heads out = output(rest[1], q, "out");
  a.lse = lse_of(rest[2], q);
  a.scale = scale_of(rest[0], q.D);
  if (q.tokens && q.heads && a.cache.n_seq) {
    a.q = q.p, a.out = out.p;
    a.starts = static_cast<const int32_t*>(starts.data_ptr());
    a.q_token_stride = q.token, a.q_head_stride = q.head;
    a.out_token_stride = out.token, a.out_head_stride = out.head;
    a.n_tokens = q.tokens, a.n_head = q.heads, a.head_dim = q.D;
    a.dtype = dtype_of(q.t);
    a.causal = causal;
    const Scratch s = scratch(rest[3], a, prompt_size_entry, "latent_attn_prompt", q.t);
    a.workspace = s.p, a.workspace_bytes = s.bytes;
    launch(prompt_entry, a, stream, "latent_attn_prompt");
    written(rest[1]), written(rest[2]);
  }
  return result(rest[1], out);
}

// attend_prompt(q, k, v, starts, k_starts, causal, scale, out, lse, workspace)
PyObject* attend_prompt(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded(n, 10, [&]() -> PyObject* {
    const Tensor& q0 = tensor(args[0], "q");
    const c10::Device dev = first(q0, "q");
    return on_device(dev, [&](latent_stream_t stream) -> PyObject* {
      const auto dt = q0.scalar_type();
      const Heads q = heads(q0, "q", dt, dev), k = heads(tensor(args[1], "k"), "k", dt, dev), v = heads(tensor(args[2], "v"), "v", dt, dev);
      TORCH_CHECK_VALUE(v.t.sizes() == k.t.sizes() && k.D == q.D, "q ", q.t.sizes(), ", k ", k.t.sizes(), " and v ", v.t.sizes(), " do not fit");
      const Tensor& starts = tensor(args[3], "starts");
      TORCH_CHECK_VALUE(starts.dim() == 1 && starts.size(0) > 0, "starts must be int32 [sequences + 1]");
      latent_attn_prompt_args a{};
      a.cache.n_seq = starts.size(0) - 1;
      a.cache.page_size = 1;
      TORCH_CHECK_VALUE(args[4] != Py_None || k.tokens == q.tokens, "k has other rows than q: give k_starts");
      const Tensor k_starts = ints(args[4] == Py_None ? starts : tensor(args[4], "k_starts"), "k_starts", a.cache.n_seq + 1, dev);
      a.k_starts = static_cast<const int32_t*>(k_starts.data_ptr());
      a.k = k.tokens ? k.p : q.p;  // a tensor without rows has no base
      a.v = k.tokens ? v.p : q.p;
      a.k_token_stride = k.token, a.k_head_stride = k.head;
      a.v_token_stride = v.token, a.v_head_stride = v.head;
      a.n_keys = k.tokens, a.n_kv_head = k.heads;
      return prompt(a, q, args[3], truth(args[5]), args + 6, dev, stream);
    });
  });
}

// attend_prompt_paged(q, k_cache, v_cache, pages, lengths, starts, causal, scale, out, lse, workspace)
PyObject* attend_prompt_paged(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded(n, 11, [&]() -> PyObject* {
    const Tensor& q0 = tensor(args[0], "q");
    const c10::Device dev = first(q0, "q");
    return on_device(dev, [&](latent_stream_t stream) -> PyObject* {
      const auto dt = q0.scalar_type();
      const Tensor& kc = tensor(args[1], "k_cache");
      latent_attn_prompt_args a{};
      a.cache = cache_of(kc, tensor(args[2], "v_cache"), tensor(args[3], "pages"), dt, dev);
      const Heads q = heads(q0, "q", dt, dev);
      TORCH_CHECK_VALUE(q.D == kc.size(3), "q ", q.t.sizes(), " does not fit the cache ", kc.sizes());
      const Tensor lengths = ints(tensor(args[4], "lengths"), "lengths", a.cache.n_seq, dev);
      a.lengths = static_cast<const int32_t*>(lengths.data_ptr());
      a.n_kv_head = kc.size(2);
      return prompt(a, q, args[5], truth(args[6]), args + 7, dev, stream);
    });
  });
}

// entries(append, decode size, decode, prompt size, prompt, LatentError): addresses of the library's functions
PyObject* entries(PyObject*, PyObject* args) {
  unsigned long long e[5];
  PyObject* error;
  if (!PyArg_ParseTuple(args, "KKKKKO", &e[0], &e[1], &e[2], &e[3], &e[4], &error)) return nullptr;
  append_entry = reinterpret_cast<decltype(append_entry)>(e[0]);
  decode_size_entry = reinterpret_cast<decltype(decode_size_entry)>(e[1]);
  decode_entry = reinterpret_cast<decltype(decode_entry)>(e[2]);
  prompt_size_entry = reinterpret_cast<decltype(prompt_size_entry)>(e[3]);
  prompt_entry = reinterpret_cast<decltype(prompt_entry)>(e[4]);
  Py_INCREF(error);
  Py_XSETREF(error_type, error);
  Py_RETURN_NONE;
}

template <typename F>
PyCFunction fast(F f) {
  return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f));
}
PyMethodDef methods[] = {
    {"entries", entries, METH_VARARGS, nullptr},
    {"kv_append", fast(kv_append), METH_FASTCALL, nullptr},
    {"attend_decode", fast(attend_decode), METH_FASTCALL, nullptr},
    {"attend_prompt", fast(attend_prompt), METH_FASTCALL, nullptr},
    {"attend_prompt_paged", fast(attend_prompt_paged), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_attend", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__attend() { return PyModule_Create(&module); }
