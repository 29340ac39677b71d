// The attention calls and residual_norm of include/latent_ffn.h on torch tensors: argument checks,
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
#include <cstring>

#include "../../include/latent_ffn.h"

namespace {

using at::Tensor;

decltype(&latent_kv_append) append_entry;
decltype(&latent_attn_decode_workspace_size) decode_size_entry;
decltype(&latent_attn_decode) decode_entry;
decltype(&latent_attn_prompt_workspace_size) prompt_size_entry;
decltype(&latent_attn_prompt) prompt_entry;
decltype(&latent_kv_append_q8) append8_entry;
decltype(&latent_kv_read) read_entry;
decltype(&latent_attn_decode_q8_workspace_size) decode8_size_entry;
decltype(&latent_attn_decode_q8) decode8_entry;
decltype(&latent_attn_prompt_q8) prompt8_entry;
decltype(&latent_attn_decode_shared_workspace_size) shared_size_entry;
decltype(&latent_attn_decode_shared) shared_entry;
decltype(&latent_residual_norm) norm_entry;
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

// A cache, and its scales where it holds codes.
struct CacheArg {
  latent_kv_cache c{};
  latent_kv_scales s{};
  bool codes = false;
  const latent_kv_scales* scales() const { return codes ? &s : nullptr; }
};
bool is_code(c10::ScalarType t) { return t == at::kChar || t == at::kFloat8_e4m3fn; }

// dt: the type of the call's other operands.
CacheArg cache_of(const Tensor& k, const Tensor& v, const Tensor& pages, c10::ScalarType dt, c10::Device dev, PyObject* k_scale, PyObject* v_scale) {
  CacheArg r;
  TORCH_CHECK_VALUE(k.dim() == 4 && v.sizes() == k.sizes(), "k_cache and v_cache must be [pages, page rows, kv heads, D], of one shape");
  r.codes = is_code(k.scalar_type());
  TORCH_CHECK_TYPE(r.codes ? v.scalar_type() == k.scalar_type() : k.scalar_type() == dt && v.scalar_type() == dt,
                   "k_cache and v_cache must be ", dt, ", as the call's other operands are, or both int8 or both float8_e4m3fn");
  check_grad(k);
  check_grad(v);
  TORCH_CHECK_VALUE(k.device() == dev && v.device() == dev && pages.device() == dev, "the cache and its page table must be on ", dev);
  TORCH_CHECK_VALUE(pages.scalar_type() == at::kInt && pages.dim() == 2, "pages must be int32 [sequences, max_pages]");
  TORCH_CHECK_VALUE(((k.stride(3) == 1 && v.stride(3) == 1) || k.size(3) < 2) && (pages.stride(1) == 1 || pages.size(1) < 2),
                    "the last dimensions of k_cache, v_cache and pages must be adjacent");
  // A size of one makes its stride meaningless to torch, and so to the library.
  auto stride = [](const Tensor& t, int i) { return t.size(i) > 1 ? t.stride(i) : 0; };
  latent_kv_cache& c = r.c;
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
  if (!r.codes) {
    TORCH_CHECK_VALUE(k_scale == Py_None && v_scale == Py_None, "k_scale and v_scale belong to a cache of int8 or float8_e4m3fn");
    return r;
  }
  auto scale = [&](PyObject* o, const char* name, float** p, int64_t* page, int64_t* head) {
    const Tensor& t = tensor(o, name);
    TORCH_CHECK_VALUE(t.scalar_type() == at::kFloat && t.dim() == 3 && t.size(0) == c.n_pages && t.size(1) == k.size(2) && t.size(2) == c.page_size &&
                          t.device() == dev && (t.stride(2) == 1 || t.size(2) < 2),
                      name, " must be f32 [", c.n_pages, ", ", k.size(2), ", ", c.page_size, "] on ", dev, ", its last dimension adjacent");
    check_grad(t);
    *p = static_cast<float*>(t.data_ptr());
    *page = stride(t, 0);
    *head = stride(t, 1);
  };
  scale(k_scale, "k_scale", &r.s.k, &r.s.k_page_stride, &r.s.k_head_stride);
  scale(v_scale, "v_scale", &r.s.v, &r.s.v_page_stride, &r.s.v_head_stride);
  r.s.code = k.scalar_type() == at::kChar ? LATENT_CODE_INT8 : LATENT_CODE_E4M3;
  return r;
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
template <typename Entry, typename... Args>
void launch(Entry entry, latent_stream_t stream, const char* call, const Args*... a) {
  PyThreadState* state = PyEval_SaveThread();
  const int status = entry(a..., stream);
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

// kv_append(k, v, k_cache, v_cache, pages, positions, seqs, q, rope, interleaved, q_out, k_scale, v_scale)
PyObject* kv_append(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded(n, 13, [&]() -> PyObject* {
    const Tensor& k0 = tensor(args[0], "k");
    const c10::Device dev = first(k0, "k");
    return on_device(dev, [&](latent_stream_t stream) -> PyObject* {
      const auto dt = k0.scalar_type();
      latent_kv_append_args a{};
      const CacheArg ca = cache_of(tensor(args[2], "k_cache"), tensor(args[3], "v_cache"), tensor(args[4], "pages"), dt, dev, args[11], args[12]);
      a.cache = ca.c;
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
        if (ca.codes)
          launch(append8_entry, stream, "latent_kv_append_q8", &a, ca.scales());
        else
          launch(append_entry, stream, "latent_kv_append", &a);
        written(args[2]), written(args[3]), written(args[10]), written(args[11]), written(args[12]);
      }
      if (args[7] == Py_None) Py_RETURN_NONE;
      return result(args[10], out);
    });
  });
}

// kv_read(k_cache, v_cache, pages, positions, seqs, k_scale, v_scale, dtype: 0 the cache's own, or the library's)
PyObject* kv_read(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded(n, 8, [&]() -> PyObject* {
    const Tensor& kc = tensor(args[0], "k_cache");
    TORCH_CHECK_VALUE(kc.is_cuda(), "k_cache must be a CUDA tensor");
    const long want = PyLong_AsLong(args[7]);
    if (want == -1 && PyErr_Occurred()) throw python_error();
    const auto dt = want == LATENT_F16 ? at::kHalf : want == LATENT_BF16 ? at::kBFloat16 : kc.scalar_type();
    TORCH_CHECK_TYPE(dt == at::kHalf || dt == at::kBFloat16, "an 8-bit cache is read as f16 or bf16: give dtype; other caches hold one of them");
    const c10::Device dev = kc.device();
    return on_device(dev, [&](latent_stream_t stream) -> PyObject* {
      latent_kv_read_args a{};
      const CacheArg ca = cache_of(kc, tensor(args[1], "v_cache"), tensor(args[2], "pages"), dt, dev, args[5], args[6]);
      a.cache = ca.c;
      const Tensor& at0 = tensor(args[3], "positions");
      TORCH_CHECK_VALUE(at0.dim() == 1, "positions must be int32 [T]");
      const int64_t T = at0.size(0);
      const Tensor positions = ints(at0, "positions", T, dev);
      Tensor seqs;
      if (args[4] != Py_None) {
        seqs = ints(tensor(args[4], "seqs"), "seqs", T, dev);
        a.seqs = static_cast<const int32_t*>(seqs.data_ptr());
      } else {
        TORCH_CHECK_VALUE(T <= a.cache.n_seq, "more tokens than sequences: give seqs");
      }
      const auto options = kc.options().dtype(dt).requires_grad(false);
      const Tensor k = at::empty({T, kc.size(2), kc.size(3)}, options), v = at::empty({T, kc.size(2), kc.size(3)}, options);
      if (k.numel()) {
        a.k = k.data_ptr(), a.v = v.data_ptr();
        a.k_token_stride = a.v_token_stride = kc.size(2) * kc.size(3);
        a.k_head_stride = a.v_head_stride = kc.size(3);
        a.positions = static_cast<const int32_t*>(positions.data_ptr());
        a.n_tokens = T, a.n_kv_head = kc.size(2), a.head_dim = kc.size(3);
        a.dtype = dtype_of(k);
        launch(read_entry, stream, "latent_kv_read", &a, ca.scales());
      }
      PyObject* pair = PyTuple_New(2);
      if (!pair) throw python_error();
      PyTuple_SET_ITEM(pair, 0, THPVariable_Wrap(k));
      PyTuple_SET_ITEM(pair, 1, THPVariable_Wrap(v));
      return pair;
    });
  });
}

// What attend_decode and attend_decode_shared (prefix given) share.  rest: lengths, scale, out, lse, workspace, k_scale, v_scale
PyObject* decode(PyObject* q_arg, PyObject* k_arg, PyObject* v_arg, PyObject* prefix_arg, PyObject* pages_arg, PyObject* const* rest) {
  const Tensor& q0 = tensor(q_arg, "q");
  const c10::Device dev = first(q0, "q");
  return on_device(dev, [&](latent_stream_t stream) -> PyObject* {
    const auto dt = q0.scalar_type();
    const Tensor& kc = tensor(k_arg, "k_cache");
    latent_attn_shared_args shared{};
    latent_attn_decode_args& a = shared.decode;
    const CacheArg ca = cache_of(kc, tensor(v_arg, "v_cache"), tensor(pages_arg, "pages"), dt, dev, rest[5], rest[6]);
    a.cache = ca.c;
    const Heads q = heads(q0, "q", dt, dev);
    const int64_t kv = kc.size(2);
    TORCH_CHECK_VALUE(q.tokens == a.cache.n_seq && q.D == kc.size(3) && kv && q.heads % kv == 0, "q ", q.t.sizes(),
                      " does not fit the cache ", kc.sizes(), " of ", a.cache.n_seq, " sequences");
    const Tensor lengths = ints(tensor(rest[0], "lengths"), "lengths", q.tokens, dev);
    Tensor prefix;
    if (prefix_arg) {
      const Tensor& t = tensor(prefix_arg, "prefix");
      TORCH_CHECK_VALUE(t.dim() == 1 && t.size(0) <= a.cache.max_pages, "prefix must be int32 [pages], at most the ", a.cache.max_pages, " of a sequence");
      prefix = ints(t, "prefix", t.size(0), dev);
      shared.prefix = static_cast<const int32_t*>(prefix.data_ptr());
      shared.n_prefix = prefix.size(0);
      shared.scales = ca.scales();
    }
    const Heads out = output(rest[2], q, "out");
    a.lse = lse_of(rest[3], q);
    a.scale = scale_of(rest[1], q.D);
    if (q.tokens && q.heads) {
      a.q = q.p, a.out = out.p;
      a.lengths = static_cast<const int32_t*>(lengths.data_ptr());
      a.q_token_stride = q.token, a.q_head_stride = q.head;
      a.out_token_stride = out.token, a.out_head_stride = out.head;
      a.n_head = q.heads, a.n_kv_head = kv, a.head_dim = q.D;
      a.dtype = dtype_of(q.t);
      const Scratch s = prefix_arg ? scratch(rest[4], shared, shared_size_entry, "latent_attn_decode_shared", q.t)
                        : ca.codes ? scratch(rest[4], a, decode8_size_entry, "latent_attn_decode_q8", q.t)
                                   : scratch(rest[4], a, decode_size_entry, "latent_attn_decode", q.t);
      a.workspace = s.p, a.workspace_bytes = s.bytes;
      if (prefix_arg)
        launch(shared_entry, stream, "latent_attn_decode_shared", &shared);
      else if (ca.codes)
        launch(decode8_entry, stream, "latent_attn_decode_q8", &a, ca.scales());
      else
        launch(decode_entry, stream, "latent_attn_decode", &a);
      written(rest[2]), written(rest[3]);
    }
    return result(rest[2], out);
  });
}
// attend_decode(q, k_cache, v_cache, pages, lengths, scale, out, lse, workspace, k_scale, v_scale)
PyObject* attend_decode(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded(n, 11, [&]() -> PyObject* { return decode(args[0], args[1], args[2], nullptr, args[3], args + 4); });
}
// attend_decode_shared(q, k_cache, v_cache, prefix, pages, lengths, scale, out, lse, workspace, k_scale, v_scale)
PyObject* attend_decode_shared(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded(n, 12, [&]() -> PyObject* { return decode(args[0], args[1], args[2], args[3], args[4], args + 5); });
}

// What attend_prompt and attend_prompt_paged share: queries, outputs, the call.  a holds keys, sequences and n_kv_head.
PyObject* prompt(latent_attn_prompt_args& a, const Heads& q, PyObject* starts_arg, bool causal, PyObject* const* rest /* scale, out, lse, workspace */,
                 c10::Device dev, latent_stream_t stream, const latent_kv_scales* scales) {
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
    if (scales)
      launch(prompt8_entry, stream, "latent_attn_prompt_q8", &a, scales);
    else
      launch(prompt_entry, stream, "latent_attn_prompt", &a);
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
      return prompt(a, q, args[3], truth(args[5]), args + 6, dev, stream, nullptr);
    });
  });
}

// attend_prompt_paged(q, k_cache, v_cache, pages, lengths, starts, causal, scale, out, lse, workspace, k_scale, v_scale)
PyObject* attend_prompt_paged(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded(n, 13, [&]() -> PyObject* {
    const Tensor& q0 = tensor(args[0], "q");
    const c10::Device dev = first(q0, "q");
    return on_device(dev, [&](latent_stream_t stream) -> PyObject* {
      const auto dt = q0.scalar_type();
      const Tensor& kc = tensor(args[1], "k_cache");
      latent_attn_prompt_args a{};
      const CacheArg ca = cache_of(kc, tensor(args[2], "v_cache"), tensor(args[3], "pages"), dt, dev, args[11], args[12]);
      a.cache = ca.c;
      const Heads q = heads(q0, "q", dt, dev);
      TORCH_CHECK_VALUE(q.D == kc.size(3), "q ", q.t.sizes(), " does not fit the cache ", kc.sizes());
      const Tensor lengths = ints(tensor(args[4], "lengths"), "lengths", a.cache.n_seq, dev);
      a.lengths = static_cast<const int32_t*>(lengths.data_ptr());
      a.n_kv_head = kc.size(2);
      return prompt(a, q, args[5], truth(args[6]), args + 7, dev, stream, ca.scales());
    });
  });
}

// ---- residual_norm ----------------------------------------------------------------
int32_t any_dtype(const Tensor& t, const char* name) {
  const auto dt = t.scalar_type();
  TORCH_CHECK_TYPE(dt == at::kFloat || dt == at::kHalf || dt == at::kBFloat16, name, " must be f32, f16 or bf16");
  return dt == at::kFloat ? LATENT_F32 : dt == at::kHalf ? LATENT_F16 : LATENT_BF16;
}
void check_norm_grad(const Tensor& t) {
  TORCH_CHECK(!t.requires_grad() || !c10::GradMode::is_enabled(), "residual_norm has no backward pass: call it under torch.no_grad()");
  TORCH_CHECK(!c10::AutogradState::get_tls_state().get_fw_grad_mode() || !t._fw_grad(0).defined(),
              "residual_norm has no forward-mode derivative: its operands may not carry tangents");
}
// Rows of d adjacent elements: a copy where they are not.
Tensor rows(const Tensor& t, const char* name, int64_t T, int64_t d, c10::Device dev) {
  TORCH_CHECK_VALUE(t.dim() == 2 && t.size(0) == T && t.size(1) == d && t.device() == dev, name, " must be [", T, ", ", d, "] on ", dev);
  check_norm_grad(t);
  return (t.stride(1) == 1 || d < 2) && t.stride(0) >= 0 ? t : t.contiguous();
}
int64_t row_stride(const Tensor& t) { return t.size(0) > 1 ? t.stride(0) : 0; }

// residual_norm(x, y, post, gate, scale, pre, dtype of n (the library's), x_out, n_out); post and pre: None or (kind, eps, weight, bias)
PyObject* residual_norm(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded(n, 9, [&]() -> PyObject* {
    const Tensor& x0 = tensor(args[0], "x");
    TORCH_CHECK_VALUE(x0.is_cuda() && x0.dim() == 2, "x must be a CUDA tensor [T, d]");
    const c10::Device dev = x0.device();
    return on_device(dev, [&](latent_stream_t stream) -> PyObject* {
      latent_residual_norm_args a{};
      const int64_t T = x0.size(0), d = x0.size(1);
      const Tensor x = rows(x0, "x", T, d, dev);
      a.n_tokens = T, a.n_embd = d;
      a.x_dtype = any_dtype(x, "x");
      a.x = x.data_ptr(), a.x_stride = row_stride(x);
      Tensor y, gate, held[4];
      auto norm = [&](PyObject* o, latent_norm* to, Tensor* hold, const char* name) {
        if (o == Py_None) return;
        TORCH_CHECK_TYPE(PyTuple_Check(o) && PyTuple_GET_SIZE(o) == 4, name, " must be a Norm");
        to->kind = static_cast<int32_t>(PyLong_AsLong(PyTuple_GET_ITEM(o, 0)));
        to->eps = static_cast<float>(PyFloat_AsDouble(PyTuple_GET_ITEM(o, 1)));
        if (PyErr_Occurred()) throw python_error();
        const void** at[2] = {&to->weight, &to->bias};
        for (int i = 0; i < 2; ++i) {
          PyObject* w = PyTuple_GET_ITEM(o, 2 + i);
          if (w == Py_None) continue;
          const Tensor& t = tensor(w, i ? "bias" : "weight");
          TORCH_CHECK_VALUE(t.dim() == 1 && t.size(0) == d && t.device() == dev, name, "'s weight and bias must be [", d, "] on ", dev);
          check_norm_grad(t);
          const int32_t dt = any_dtype(t, name);
          TORCH_CHECK_TYPE(!(i && to->weight) || to->dtype == dt, name, "'s weight and bias must be of one type");
          to->dtype = dt;
          hold[i] = t.is_contiguous() ? t : t.contiguous();
          *at[i] = d ? hold[i].data_ptr() : nullptr;
        }
      };
      if (args[1] != Py_None) {
        y = rows(tensor(args[1], "y"), "y", T, d, dev);
        a.y_dtype = any_dtype(y, "y");
        a.y = y.data_ptr(), a.y_stride = row_stride(y);
        norm(args[2], &a.post, held, "post");
        if (args[3] != Py_None) {
          const Tensor& g = tensor(args[3], "gate");
          TORCH_CHECK_VALUE(g.dim() == 1 ? g.size(0) == d : g.dim() == 2 && g.size(0) == T && (g.size(1) == d || g.size(1) == 1), "gate must be [", d, "], [",
                            T, ", 1] or [", T, ", ", d, "]");
          check_norm_grad(g);
          gate = rows(g.dim() == 1 ? g.unsqueeze(0).expand({T, d}) : g.dim() == 2 && g.size(1) == 1 && d != 1 ? g.expand({g.size(0), d}) : g, "gate", T, d, dev);
          a.gate_dtype = any_dtype(gate, "gate");
          a.gate = gate.data_ptr(), a.gate_stride = row_stride(gate);
        }
      } else {
        TORCH_CHECK_VALUE(args[2] == Py_None && args[3] == Py_None, "post and gate belong to y");
      }
      a.scale = static_cast<float>(PyFloat_AsDouble(args[4]));
      if (PyErr_Occurred()) throw python_error();
      norm(args[5], &a.pre, held + 2, "pre");
      // Outputs: the ones given, or new ones; without y the stream is x itself, without pre there is no n.
      auto output_rows = [&](PyObject* o, c10::ScalarType dt, const char* name) {
        if (o == Py_None) return at::empty({T, d}, x.options().dtype(dt).requires_grad(false));
        const Tensor& t = tensor(o, name);
        TORCH_CHECK_VALUE(t.dim() == 2 && t.size(0) == T && t.size(1) == d && t.scalar_type() == dt && t.device() == dev && (t.stride(1) == 1 || d < 2) &&
                              (T < 2 || t.stride(0) >= d),
                          name, " must be ", dt, " [", T, ", ", d, "] on ", dev, " with adjacent columns");
        check_norm_grad(t);
        return t;
      };
      const bool has_x = args[1] != Py_None || args[7] != Py_None, has_n = args[5] != Py_None;
      TORCH_CHECK_VALUE(has_n || args[8] == Py_None, "n_out without pre");
      Tensor x_out, n_out;
      if (has_x) {
        x_out = output_rows(args[7], x0.scalar_type(), "x_out");
        a.x_out = x_out.data_ptr(), a.x_out_stride = row_stride(x_out);
      }
      if (has_n) {
        const long want = PyLong_AsLong(args[6]);
        if (want == -1 && PyErr_Occurred()) throw python_error();
        n_out = output_rows(args[8], want == LATENT_F32 ? at::kFloat : want == LATENT_F16 ? at::kHalf : at::kBFloat16, "n_out");
        a.n_dtype = static_cast<int32_t>(want);
        a.n_out = n_out.data_ptr(), a.n_out_stride = row_stride(n_out);
      }
      if (x.numel() && (has_x || has_n)) {
        launch(norm_entry, stream, "latent_residual_norm", &a);
        written(args[7]), written(args[8]);
      }
      PyObject* pair = PyTuple_New(2);
      if (!pair) throw python_error();
      auto put = [&](int i, PyObject* o) {
        PyTuple_SET_ITEM(pair, i, o);
      };
      auto given = [](PyObject* o) {
        Py_INCREF(o);
        return o;
      };
      put(0, args[7] != Py_None ? given(args[7]) : has_x ? THPVariable_Wrap(x_out) : given(args[0]));
      put(1, args[8] != Py_None ? given(args[8]) : has_n ? THPVariable_Wrap(n_out) : given(Py_None));
      return pair;
    });
  });
}

// entries({name: address of the library's function}, LatentError)
PyObject* entries(PyObject*, PyObject* args) {
  PyObject *table, *error;
  if (!PyArg_ParseTuple(args, "O!O", &PyDict_Type, &table, &error)) return nullptr;
  const struct {
    const char* name;
    void* to;
  } all[] = {{"latent_kv_append", &append_entry}, {"latent_kv_append_q8", &append8_entry}, {"latent_kv_read", &read_entry},
             {"latent_attn_decode_workspace_size", &decode_size_entry}, {"latent_attn_decode", &decode_entry},
             {"latent_attn_decode_q8_workspace_size", &decode8_size_entry}, {"latent_attn_decode_q8", &decode8_entry},
             {"latent_attn_decode_shared_workspace_size", &shared_size_entry}, {"latent_attn_decode_shared", &shared_entry},
             {"latent_attn_prompt_workspace_size", &prompt_size_entry}, {"latent_attn_prompt", &prompt_entry},
             {"latent_attn_prompt_q8", &prompt8_entry}, {"latent_residual_norm", &norm_entry}};
  for (const auto& e : all) {
    PyObject* o = PyDict_GetItemString(table, e.name);
    if (!o) {
      PyErr_Format(PyExc_KeyError, "%s", e.name);
      return nullptr;
    }
    void* address = PyLong_AsVoidPtr(o);
    if (!address && PyErr_Occurred()) return nullptr;
    std::memcpy(e.to, &address, sizeof address);
  }
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
    {"kv_read", fast(kv_read), METH_FASTCALL, nullptr},
    {"attend_decode", fast(attend_decode), METH_FASTCALL, nullptr},
    {"attend_decode_shared", fast(attend_decode_shared), METH_FASTCALL, nullptr},
    {"residual_norm", fast(residual_norm), METH_FASTCALL, nullptr},
    {"attend_prompt", fast(attend_prompt), METH_FASTCALL, nullptr},
    {"attend_prompt_paged", fast(attend_prompt_paged), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_attend", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__attend() { return PyModule_Create(&module); }
