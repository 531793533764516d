// Calls of token_log_probs, packed_attention and AdamW from Python, as a CPython extension against PyTorch's C++ interface.
//
// Through Python and a foreign function call a forward pass took 25 us of the host, and a backward pass, whose node the autograd
// engine runs on a thread of its own that must first get the interpreter lock, 80 us besides the engine's own 45: more than the kernels
// of all but large inputs. Here the nodes are C++ ones.
//
// A call answers None for whatever is not plain (other types, layouts that must be refused, subclasses of Tensor): the caller then
// goes through the Python form (ops/tokens.py, ops/attention.py), which checks, refuses and explains. Nothing is remembered
// from one call for the next but the entry points of the native library and the status words that Python hands over.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/TensorSubclassLikeUtils.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include <cmath>
#include <cstdint>

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// ---- entry points of the native library ---------------------------------------------------------
struct Entry {
  const char* (*error)() = nullptr;
  int (*token)(const void*, int, long long, int, long long, const void*, int, long long, float, int, float*, float*, float*, float*, long long*, void*) = nullptr;
  int (*token_grad)(const void*, int, long long, int, long long, void*, long long, const void*, int, long long, float, int, const float*, const float*,
                    const long long*, const float*, const float*, const float*, void*) = nullptr;
  int (*attention)(const void*, const void*, const void*, const long long*, const int*, int, int, int, int, int, int, int, float, void*, void*, float*, int*, int*,
                   void*) = nullptr;
  long long (*attention_plan_ints)(int, int) = nullptr;
  int (*attention_backward)(const void*, const void*, const void*, const void*, const long long*, const int*, int, int, int, int, int, int, int, float,
                            const void*, const void*, const float*, float*, void*, void*, void*, int*, int*, void*) = nullptr;
  int (*adamw)(const void*, int, int, int, double, const float*, double, double, double, double, double, double, unsigned, int*, void*) = nullptr;
} entry;

constexpr int MOST_DEVICES = 64;
struct Status {
  volatile int* host = nullptr;   // written by kernels whose waits ran out
  int* device = nullptr;
} statuses[MOST_DEVICES];

void check(int code, const char* what) { TORCH_CHECK(code == 0, what, " failed (code ", code, "): ", entry.error ? entry.error() : ""); }

int type_code(at::ScalarType t) { return t == at::kFloat ? 0 : t == at::kBFloat16 ? 1 : t == at::kHalf ? 2 : -1; }

const Tensor* plain(PyObject* object) {
  if (!THPVariable_CheckExact(object)) return nullptr;
  const Tensor& t = THPVariable_Unpack(object);
  if (!t.defined() || t.layout() != at::kStrided || !t.unsafeGetTensorImpl()->has_storage() || at::isTensorSubclassLike(t) || t.is_neg() || t.is_conj()) return nullptr;
  return &t;
}

// Does the tensor carry a tangent of forward-mode differentiation? Results here would lose it.
bool has_tangent(const Tensor& t) { return t.defined() && t._fw_grad(/*level=*/0).defined(); }
void refuse_tangents(const variable_list& grads, const char* what) {
  for (const Tensor& g : grads) TORCH_CHECK_NOT_IMPLEMENTED(!has_tangent(g), what, ": forward-mode differentiation is not supported");
}

void* current_stream(const Tensor& t) { return (void*)c10::cuda::getCurrentCUDAStream(t.get_device()).stream(); }

// What a backward pass returns cannot be differentiated again: asking for it raises.
variable_list once(variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  for (Tensor& g : grads)
    if (g.defined()) g = g.detach().set_requires_grad(true);
  return (*std::make_shared<torch::autograd::DelayedError>("trying to differentiate twice a function that was marked with @once_differentiable", (int64_t)grads.size()))(std::move(grads));
}

// ---- log probabilities --------------------------------------------------------------------------
// Rows of a tensor whose last dimension is the row: their distance, where all other dimensions are steps of one; else -1.
int64_t row_stride(const Tensor& t) {
  const auto n = t.sizes(), s = t.strides();
  const int64_t vocab = n.back();
  if (vocab != 1 && s.back() != 1) return -1;
  int64_t stride = -1, expected = -1;
  for (int64_t i = (int64_t)n.size() - 2; i >= 0; --i) {
    if (n[i] == 1) continue;
    if (stride < 0) stride = s[i];
    else if (s[i] != expected) return -1;
    expected = s[i] * n[i];
  }
  if (stride < 0) return vocab;   // one row
  return stride >= vocab ? stride : -1;
}
// The numbers that a tensor stands for, in memory: some only say that what they refer to is to be negated, or that all of it is zero.
Tensor in_memory(const Tensor& t) { return t._is_zerotensor() ? at::zeros(t.sizes(), t.options()) : t.resolve_neg(); }
// `t`, or a contiguous copy where its rows do not lie as the kernels take them.
Tensor as_rows(const Tensor& t, int64_t& stride) {
  stride = row_stride(t);
  if (stride >= 0) return t;
  stride = t.sizes().back();
  return t.contiguous();
}

struct Tokens {
  Tensor log_probs, entropy, values, tokens, stats;
};

Tokens token_forward(const Tensor& logits, const Tensor& targets, int64_t top, bool entropy, int64_t ignore_index, double temperature) {
  const c10::cuda::CUDAGuard guard(logits.device());
  int64_t stride;
  const Tensor z = as_rows(logits, stride), t = targets.contiguous();
  const int64_t n = targets.numel(), vocab = logits.sizes().back();
  const auto f32 = z.options().dtype(at::kFloat);
  Tokens o;
  o.log_probs = at::empty(targets.sizes(), f32);
  o.stats = at::empty({n, 2}, f32);
  if (entropy) o.entropy = at::empty(targets.sizes(), f32);
  if (top > 0) {
    std::vector<int64_t> shape = targets.sizes().vec();
    shape.push_back(top);
    o.values = at::empty(shape, f32);
    o.tokens = at::empty(shape, z.options().dtype(at::kLong));
  }
  if (n > 0)
    check(entry.token(z.const_data_ptr(), type_code(z.scalar_type()), n, (int)vocab, stride, t.const_data_ptr(), t.scalar_type() == at::kLong, ignore_index,
                      (float)(1.0 / temperature), (int)top, (float*)o.log_probs.data_ptr(), (float*)o.stats.data_ptr(),
                      entropy ? (float*)o.entropy.data_ptr() : nullptr, top > 0 ? (float*)o.values.data_ptr() : nullptr,
                      top > 0 ? (long long*)o.tokens.data_ptr() : nullptr, current_stream(z)),
          "psgd_token_logprob");
  return o;
}

struct TokenLogProbs : torch::autograd::Function<TokenLogProbs> {
  // outputs: log probabilities, then the entropy and the listed tokens with their log probabilities, where asked for
  static variable_list forward(AutogradContext* ctx, const Tensor& logits, const Tensor& targets, int64_t top, bool entropy, int64_t ignore_index, double temperature) {
    const Tokens o = token_forward(logits, targets, top, entropy, ignore_index, temperature);
    ctx->save_for_backward({logits, targets, o.stats, o.entropy, o.tokens});
    ctx->saved_data["ignore_index"] = ignore_index;
    ctx->saved_data["temperature"] = temperature;
    ctx->set_materialize_grads(false);
    variable_list out = {o.log_probs};
    if (entropy) out.push_back(o.entropy);
    if (top > 0) {
      out.push_back(o.values);
      out.push_back(o.tokens);
      ctx->mark_non_differentiable({o.tokens});
    }
    return out;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    refuse_tangents(grads, "token_log_probs");
    const auto saved = ctx->get_saved_variables();
    const Tensor &logits = saved[0], &targets = saved[1], &stats = saved[2], &entropy = saved[3], &tokens = saved[4];
    Tensor grad;
    {
      const at::NoGradGuard no_grad;
      size_t next = 1;
      Tensor g = grads[0], g_entropy, g_top;
      if (entropy.defined()) g_entropy = grads[next++];
      if (tokens.defined()) g_top = grads[next];
      if (!g.defined() && !g_entropy.defined() && !g_top.defined()) return variable_list(6);
      const c10::cuda::CUDAGuard guard(logits.device());
      int64_t stride;
      const Tensor z = as_rows(logits, stride), t = targets.contiguous();
      const int64_t n = targets.numel(), vocab = logits.sizes().back(), size = z.element_size();
      // each row as far from a 16-byte boundary as that of the logits, see _grad_like in ops/tokens.py
      const int64_t lead = (int64_t)((uintptr_t)z.const_data_ptr() % 16) / size, between = n > 1 ? (stride - vocab) % (16 / size) : 0, pitch = vocab + between;
      if (lead == 0 && between == 0) {
        grad = at::empty(logits.sizes(), z.options());
      } else {
        std::vector<int64_t> strides(logits.dim(), 1);
        int64_t step = pitch;
        for (int64_t i = logits.dim() - 2; i >= 0; --i) {
          strides[i] = step;
          step *= logits.size(i);
        }
        grad = at::empty({lead + n * pitch}, z.options()).as_strided(logits.sizes(), strides, lead);
      }
      if (n > 0) {
        auto f32 = [](const Tensor& x) { return x.defined() ? in_memory(x).to(at::kFloat).contiguous() : x; };
        auto at_of = [](const Tensor& x) { return x.defined() ? (const float*)x.const_data_ptr() : nullptr; };
        g = f32(g), g_entropy = f32(g_entropy), g_top = f32(g_top);
        check(entry.token_grad(z.const_data_ptr(), type_code(z.scalar_type()), n, (int)vocab, stride, grad.data_ptr(), pitch, t.const_data_ptr(),
                               t.scalar_type() == at::kLong, ctx->saved_data["ignore_index"].toInt(), (float)(1.0 / ctx->saved_data["temperature"].toDouble()),
                               g_top.defined() ? (int)tokens.sizes().back() : 0, (const float*)stats.const_data_ptr(),
                               g_entropy.defined() ? at_of(entropy) : nullptr, g_top.defined() ? (const long long*)tokens.const_data_ptr() : nullptr, at_of(g),
                               at_of(g_entropy), at_of(g_top), current_stream(z)),
              "psgd_token_logprob_grad");
      }
    }
    variable_list out(6);
    out[0] = grad;
    return once(std::move(out));
  }
};

PyObject* wrap(const Tensor& t) {
  if (!t.defined()) Py_RETURN_NONE;
  return THPVariable_Wrap(t);
}

// No C++ exception leaves the module: each becomes the Python exception that PyTorch's own calls raise for it.
template <class F>
PyObject* guarded(F body) {
  HANDLE_TH_ERRORS
  return body();
  END_HANDLE_TH_ERRORS
}

// token_log_probs(logits, targets, top, entropy, ignore_index, temperature): the four results, or None.
PyObject* token_log_probs(PyObject*, PyObject* args) {
  return guarded([&]() -> PyObject* {
    PyObject *logits_object, *targets_object;
    long long top, ignore_index;
    int entropy;
    double temperature;
    if (!PyArg_ParseTuple(args, "OOLpLd", &logits_object, &targets_object, &top, &entropy, &ignore_index, &temperature)) {
      PyErr_Clear();
      Py_RETURN_NONE;
    }
    const Tensor *logits = plain(logits_object), *targets = plain(targets_object);
    if (entry.token == nullptr || logits == nullptr || targets == nullptr) Py_RETURN_NONE;
    const int64_t vocab = logits->dim() > 0 ? logits->sizes().back() : 0;
    const auto index = targets->scalar_type();
    if (!logits->is_cuda() || logits->device() != targets->device() || type_code(logits->scalar_type()) < 0 || (index != at::kLong && index != at::kInt) || vocab < 1 ||
        vocab >= (1ll << 31) - (1 << 16) || logits->sizes().slice(0, logits->dim() - 1) != targets->sizes() || top < 0 || top > 32 || top > vocab ||
        !(temperature >= 0x1p-100 && temperature <= 0x1p100) || has_tangent(*logits) || torch::jit::tracer::isTracing())
      Py_RETURN_NONE;
    Tensor out[4];
    if (at::GradMode::is_enabled() && logits->requires_grad()) {
      const variable_list r = TokenLogProbs::apply(*logits, *targets, (int64_t)top, entropy != 0, (int64_t)ignore_index, temperature);
      size_t next = 1;
      out[0] = r[0];
      if (entropy) out[1] = r[next++];
      if (top > 0) {
        out[2] = r[next];
        out[3] = r[next + 1];
      }
    } else {
      const Tokens o = token_forward(*logits, *targets, top, entropy != 0, ignore_index, temperature);
      out[0] = o.log_probs, out[1] = o.entropy, out[2] = o.values, out[3] = o.tokens;
    }
    PyObject* result = PyTuple_New(4);
    for (int i = 0; i < 4 && result != nullptr; ++i) PyTuple_SET_ITEM(result, i, wrap(out[i]));
    return result;
  });
}

// ---- attention ----------------------------------------------------------------------------------
// As the kernels address it, see _usable in ops/attention.py.
Tensor usable(const Tensor& t) {
  const int64_t tokens = t.size(0), heads = t.size(1), size = t.size(2);
  const bool fits = (uintptr_t)t.const_data_ptr() % 16 == 0 && t.stride(2) == 1 && (tokens == 1 || (t.stride(0) % 8 == 0 && t.stride(0) >= size)) &&
                    (heads == 1 || (t.stride(1) % 8 == 0 && t.stride(1) >= size));
  return fits ? t : t.clone(at::MemoryFormat::Contiguous);
}
void strides_of(const Tensor& t, long long* out) {
  out[0] = t.size(0) > 1 ? t.stride(0) : t.size(1) * t.size(2);
  out[1] = t.size(1) > 1 ? t.stride(1) : t.size(2);
}
int* status_of(const Tensor& t) {
  const Status& s = statuses[t.get_device()];
  TORCH_CHECK(s.host == nullptr || *s.host == 0, "packed_attention: a wait of an earlier call ran out on ", t.device(), " (status ", *s.host, "); its results are not valid");
  return s.device;
}

// Scratch for the order of the tiles, where there are many sequences.
Tensor plan_of(int64_t sequences, int64_t tokens, const Tensor& like) {
  const long long ints = entry.attention_plan_ints((int)sequences, (int)tokens);
  return ints ? at::empty({ints}, like.options().dtype(at::kInt)) : Tensor();
}

struct Attended {
  Tensor out, lse, rest;
};
Attended attention_forward(const Tensor& q0, const Tensor& k0, const Tensor& v0, const Tensor& offsets0, bool causal, double scale, bool gradient) {
  const c10::cuda::CUDAGuard guard(q0.device());
  const int64_t tokens = q0.size(0), heads = q0.size(1), size = q0.size(2), sequences = offsets0.size(0) - 1;
  Attended o;
  o.out = at::empty({tokens, heads, size}, q0.options());
  if (tokens == 0 || sequences == 0) {
    o.out.zero_();
    return o;
  }
  o.lse = at::empty({heads, tokens}, q0.options().dtype(at::kFloat));
  if (gradient) o.rest = at::empty({tokens, heads, size}, q0.options());
  const Tensor q = usable(q0), k = usable(k0), v = usable(v0), offsets = offsets0.contiguous(), plan = plan_of(sequences, tokens, q);
  long long strides[6];
  strides_of(q, strides);
  strides_of(k, strides + 2);
  strides_of(v, strides + 4);
  check(entry.attention(q.const_data_ptr(), k.const_data_ptr(), v.const_data_ptr(), strides, (const int*)offsets.const_data_ptr(), (int)sequences, (int)tokens, (int)heads,
                        (int)k.size(1), (int)size, type_code(q.scalar_type()), causal, (float)scale, o.out.data_ptr(), gradient ? o.rest.data_ptr() : nullptr,
                        (float*)o.lse.data_ptr(), plan.defined() ? (int*)plan.data_ptr() : nullptr, status_of(q), current_stream(q)),
        "psgd_attention");
  return o;
}

struct PackedAttention : torch::autograd::Function<PackedAttention> {
  static Tensor forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& offsets, bool causal, double scale) {
    const Attended o = attention_forward(q, k, v, offsets, causal, scale, true);
    ctx->save_for_backward({q, k, v, offsets, o.out, o.lse, o.rest});
    ctx->saved_data["causal"] = causal;
    ctx->saved_data["scale"] = scale;
    return o.out;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    refuse_tangents(grads, "packed_attention");
    const auto saved = ctx->get_saved_variables();
    variable_list result(6);
    {
      const at::NoGradGuard no_grad;
      const Tensor &out = saved[4], &lse = saved[5], &rest = saved[6];
      const c10::cuda::CUDAGuard guard(out.device());
      const int64_t tokens = out.size(0), heads = out.size(1), size = out.size(2), groups = saved[1].size(1);
      Tensor dq = at::empty({tokens, heads, size}, out.options()), dk = at::empty({tokens, groups, size}, out.options()), dv = at::empty({tokens, groups, size}, out.options());
      if (!lse.defined()) {
        dq.zero_(), dk.zero_(), dv.zero_();
      } else {
        const Tensor q = usable(saved[0]), k = usable(saved[1]), v = usable(saved[2]), offsets = saved[3].contiguous();
        const Tensor plan = plan_of(offsets.size(0) - 1, tokens, q), g = usable(in_memory(grads[0])), delta = at::empty({out.scalar_type() == at::kHalf ? 2 * heads + groups : heads, tokens}, lse.options());
        long long strides[8];
        strides_of(q, strides);
        strides_of(k, strides + 2);
        strides_of(v, strides + 4);
        strides_of(g, strides + 6);
        check(entry.attention_backward(q.const_data_ptr(), k.const_data_ptr(), v.const_data_ptr(), g.const_data_ptr(), strides, (const int*)offsets.const_data_ptr(),
                                       (int)(offsets.size(0) - 1), (int)tokens, (int)heads, (int)groups, (int)size, type_code(out.scalar_type()),
                                       ctx->saved_data["causal"].toBool(), (float)ctx->saved_data["scale"].toDouble(), out.const_data_ptr(), rest.const_data_ptr(),
                                       (const float*)lse.const_data_ptr(), (float*)delta.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(),
                                       plan.defined() ? (int*)plan.data_ptr() : nullptr, status_of(q),
                                       current_stream(q)),
              "psgd_attention_backward");
      }
      result[0] = dq, result[1] = dk, result[2] = dv;
    }
    return once(std::move(result));
  }
};

// packed_attention(q, k, v, offsets, causal, scale): the output, or None. A scale of zero stands for the usual one.
PyObject* packed_attention(PyObject*, PyObject* args) {
  return guarded([&]() -> PyObject* {
    PyObject* objects[4];
    int causal;
    double scale;
    if (!PyArg_ParseTuple(args, "OOOOpd", objects, objects + 1, objects + 2, objects + 3, &causal, &scale)) {
      PyErr_Clear();
      Py_RETURN_NONE;
    }
    const Tensor* t[4];
    for (int i = 0; i < 4; ++i) {
      t[i] = plain(objects[i]);
      if (t[i] == nullptr || !t[i]->is_cuda() || t[i]->device() != t[0]->device()) Py_RETURN_NONE;
    }
    const Tensor &q = *t[0], &k = *t[1], &v = *t[2], &offsets = *t[3];
    const auto type = q.scalar_type();
    if (entry.attention == nullptr || q.dim() != 3 || k.dim() != 3 || k.sizes() != v.sizes() || q.size(0) != k.size(0) || q.size(2) != k.size(2) || k.size(1) < 1 ||
        q.size(1) < 1 || q.size(1) % k.size(1) != 0 || q.size(2) < 8 || q.size(2) > 128 || q.size(2) % 8 != 0 || (type != at::kBFloat16 && type != at::kHalf) ||
        k.scalar_type() != type || v.scalar_type() != type || offsets.scalar_type() != at::kInt || offsets.dim() != 1 || offsets.size(0) < 1 ||
        offsets.size(0) > (1ll << 31) - (1 << 16) || q.size(0) >= (1ll << 31) - (1 << 16) || !(scale == 0 || (scale >= 0x1p-100 && scale <= 0x1p100)) || q.get_device() >= MOST_DEVICES ||
        has_tangent(q) || has_tangent(k) || has_tangent(v) || torch::jit::tracer::isTracing())
      Py_RETURN_NONE;
    const Status& status = statuses[q.get_device()];
    if (status.host == nullptr || *status.host != 0) Py_RETURN_NONE;
    if (scale == 0) scale = 1.0 / std::sqrt((double)q.size(2));
    if (at::GradMode::is_enabled() && (q.requires_grad() || k.requires_grad() || v.requires_grad()))
      return wrap(PackedAttention::apply(q, k, v, offsets, causal != 0, scale));
    return wrap(attention_forward(q, k, v, offsets, causal != 0, scale, false).out);
  });
}

// ---- AdamW --------------------------------------------------------------------------------------
// adamw_step(items, count, device, type, bits, lr, address of lr, betas and their logarithms, eps, decay, seed, ticket): the native step on the
// device's current stream. Returns its code.
PyObject* adamw_step(PyObject*, PyObject* args) {
  return guarded([&]() -> PyObject* {
    const char* items;
    Py_ssize_t bytes;
    int count, device, type, bits;
    double lr, beta1, beta2, log1, log2, eps, decay;
    unsigned long long lr_at, ticket;
    unsigned int seed;
    if (!PyArg_ParseTuple(args, "y#iiiidKddddddIK", &items, &bytes, &count, &device, &type, &bits, &lr, &lr_at, &beta1, &beta2, &log1, &log2, &eps, &decay, &seed, &ticket))
      return nullptr;
    const c10::cuda::CUDAGuard guard((c10::DeviceIndex)device);
    void* stream = (void*)c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)device).stream();
    return PyLong_FromLong(entry.adamw(items, count, type, bits, lr, (const float*)lr_at, beta1, beta2, log1, log2, eps, decay, seed, (int*)ticket, stream));
  });
}

// ---- what Python hands over ---------------------------------------------------------------------
// bind(error, token, token_grad, attention, attention_backward, adamw, attention_plan_ints): addresses of the native library's entry points.
PyObject* bind(PyObject*, PyObject* args) {
  unsigned long long a[7];
  if (!PyArg_ParseTuple(args, "KKKKKKK", a, a + 1, a + 2, a + 3, a + 4, a + 5, a + 6)) return nullptr;
  entry.error = (decltype(entry.error))a[0];
  entry.token = (decltype(entry.token))a[1];
  entry.token_grad = (decltype(entry.token_grad))a[2];
  entry.attention = (decltype(entry.attention))a[3];
  entry.attention_backward = (decltype(entry.attention_backward))a[4];
  entry.adamw = (decltype(entry.adamw))a[5];
  entry.attention_plan_ints = (decltype(entry.attention_plan_ints))a[6];
  Py_RETURN_NONE;
}
// status(device, host address, device address): the status word of a device.
PyObject* status(PyObject*, PyObject* args) {
  int device;
  unsigned long long host, dev;
  if (!PyArg_ParseTuple(args, "iKK", &device, &host, &dev)) return nullptr;
  if (device >= 0 && device < MOST_DEVICES) {
    statuses[device].device = (int*)dev;
    statuses[device].host = (volatile int*)host;
  }
  Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"bind", bind, METH_VARARGS, nullptr},
    {"status", status, METH_VARARGS, nullptr},
    {"token_log_probs", token_log_probs, METH_VARARGS, nullptr},
    {"packed_attention", packed_attention, METH_VARARGS, nullptr},
    {"adamw_step", adamw_step, METH_VARARGS, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_operators", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__operators() {
  PyObject* m = PyModule_Create(&module);
  // what this was compiled for, which the loader compares (csrc/build.py, scan_target)
  if (m != nullptr && (PyModule_AddStringConstant(m, "target", PSGD_SCAN_TARGET) != 0 || PyModule_AddIntConstant(m, "entry_points", 7) != 0)) {
    Py_DECREF(m);
    return nullptr;
  }
  return m;
}
