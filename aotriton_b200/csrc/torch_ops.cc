// The autograd entry points' native route: attention on ordinary torch tensors, forward and backward, without Python in
// between; in the same way sink attention, the relative position bias and dropout of hidden states.  Outputs, gradients and scratch
// come from torch's caching allocator, launches go to torch's current stream through the C++ operator API (include/aotriton/flash.h), the backward is a torch::autograd::Function: version checks and CUDA-graph
// capture see what they see of the Python Function, saved-tensor hooks the inputs, the output and the log-sum-exp.
//
// What bounds a small call is the host.  Measured, us a pass, the Python way against this: training step of 2 x 4 heads x 128 tokens of 64 (20
// of kernels) 160 / 77; cross attention, 4 x 8 heads x 1024 x 77 of 80 (47 of kernels), 332 / 78; one token of 4 sequences against 6007
// keys, 32:8 heads of 128 (14), 33.5 / 20.6.
//
// attend() returns None for whatever is not ordinary, and the caller then goes the Python way: tensors that are not plain CUDA tensors of
// one type on the current device with unit innermost stride, and every mode in which an operator call means more than its kernels
// (dispatch and function modes, functorch transforms, forward-mode gradients, tracing).  The backward asks the same of its
// gradient, of what was saved and of the modes it runs under, and otherwise leaves itself to the operator or to the Python Function's.
#include <torch/csrc/Dtype.h>
#include <torch/csrc/DynamicTypes.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <ATen/ATen.h>
#include <ATen/PythonTorchFunctionTLS.h>
#include <ATen/core/dispatch/Dispatcher.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>

#include <aotriton/flash.h>
#include <aotriton/util.h>
#include <aotriton_b200.h>

#include <atomic>
#include <map>
#include <string>

namespace aotriton = AOTRITON_NS;
namespace flash = AOTRITON_NS::v3::flash;
using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

namespace {

// Kernel family of the most recent backward: the library keeps it per thread, and autograd runs backwards on a thread of
// its own.
std::atomic<int> g_last_bwd_family{0};

// The Function's backward as Python has it (autograd.py), for what Attend::backward leaves to it.  Set once, at import.
PyObject* g_python_backward = nullptr;

// A call's numbers.  `packed`: token-packed sequences (cu_q, cu_k); `op`: the call stands for the registered operators, whose
// backward may use the fused form and is itself an operator.
struct Call {
  double sm_scale, dropout_p;
  int64_t causal_type, left, right, max_q, max_k;
  uint64_t seed, offset;      // of the dropout; offset is the whole of it
  bool packed, op;
};

aotriton::DType dtype_of(at::ScalarType t) {
  return t == at::kFloat ? aotriton::kFloat32 : (t == at::kHalf ? aotriton::kFloat16 : aotriton::kBFloat16);
}
template <int Rank>
aotriton::TensorView<Rank> view_of(const Tensor& t, aotriton::DType dt) {
  std::array<uint64_t, Rank> n, s;
  for (int i = 0; i < Rank; ++i) { n[i] = (uint64_t)t.size(i); s[i] = (uint64_t)t.stride(i); }
  return aotriton::TensorView<Rank>(reinterpret_cast<intptr_t>(t.data_ptr()), n, s, dt);
}
aotriton::TensorView<4> view_or_null(const Tensor& t, aotriton::DType dt) {
  return t.defined() ? view_of<4>(t, dt) : aotriton::TensorView<4>(0, {}, {}, dt);
}
Tensor fresh(at::IntArrayRef sizes, at::ScalarType dt) {
  return at::detail::empty_cuda(sizes, dt, c10::Device(c10::kCUDA, c10::cuda::current_device()), std::nullopt);
}
// torch.empty_like: the tensor's strides where they are dense
Tensor gradient_of(const Tensor& t) { return t.is_contiguous() ? fresh(t.sizes(), t.scalar_type()) : at::empty_like(t); }

void check(hipError_t e, const char* what) {
  if (e == hipSuccess) return;
  const char* name = e == hipErrorInvalidValue ? "hipErrorInvalidValue" : e == hipErrorNoBinaryForGpu ? "hipErrorNoBinaryForGpu"
                     : e == hipErrorNotSupported ? "hipErrorNotSupported" : e == hipErrorLaunchFailure ? "hipErrorLaunchFailure"
                                                                                                       : nullptr;
  throw std::runtime_error(std::string(what) + " failed: " + (name ? std::string("hipError_t.") + name : std::to_string((int)e)));
}

template <typename P>
void fill_common(P& p, const Call& c, const Tensor& cu_q, const Tensor& cu_k, const Tensor& seed) {
  p.Sm_scale = (float)c.sm_scale;
  p.dropout_p = (float)c.dropout_p;
  p.philox_seed_ptr = aotriton::TensorView<0>(seed.defined() ? reinterpret_cast<intptr_t>(seed.data_ptr()) : 0, aotriton::kUInt64);
  p.philox_offset1 = aotriton::TensorView<0>(0, aotriton::kUInt64);
  p.philox_offset2 = c.offset;
  p.causal_type = (int8_t)c.causal_type;
  p.window_left = (int32_t)c.left;
  p.window_right = (int32_t)c.right;
  p.varlen_type = c.packed ? AB200_VARLEN_COMPACT : AB200_VARLEN_NONE;
  if (c.packed) {
    p.cu_seqlens_q = view_of<1>(cu_q, aotriton::kInt32);
    p.cu_seqlens_k = view_of<1>(cu_k, aotriton::kInt32);
    p.Max_seqlen_q = (int32_t)c.max_q;
    p.Max_seqlen_k = (int32_t)c.max_k;
  }
}

aotriton::Stream current_stream() { return aotriton::Stream(c10::cuda::getCurrentCUDAStream().stream()); }

// `lse` is left undefined where nobody will read it.
void forward(const Call& c, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& b, const Tensor& cu_q, const Tensor& cu_k,
             bool want_lse, Tensor& out, Tensor& lse, Tensor& seed) {
  at::AutoDispatchBelowADInplaceOrView guard;
  const aotriton::DType dt = dtype_of(q.scalar_type());
  if (c.packed) {      // (1, H, tokens, D) views of (tokens, H, D) storage
    out = fresh({1, q.size(2), q.size(1), v.size(3)}, q.scalar_type()).transpose(1, 2);
    if (want_lse) lse = fresh({q.size(1), q.size(2)}, at::kFloat);
  } else {
    out = fresh({q.size(0), q.size(1), q.size(2), v.size(3)}, q.scalar_type());
    if (want_lse) lse = fresh({q.size(0) * q.size(1), q.size(2)}, at::kFloat);
  }
  // one fill on the stream; the offset goes by value
  if (c.dropout_p > 0) seed = at::full({1}, (int64_t)c.seed, out.options().dtype(at::kLong));
  flash::attn_fwd_params p;
  p.Q = view_of<4>(q, dt); p.K = view_of<4>(k, dt); p.V = view_of<4>(v, dt); p.B = view_or_null(b, dt); p.Out = view_of<4>(out, dt);
  p.L = want_lse ? view_of<2>(lse, aotriton::kFloat32) : aotriton::TensorView<2>(0, {}, {}, aotriton::kFloat32);
  p.encoded_softmax = aotriton::TensorView<4>(0, {}, {}, dt);
  fill_common(p, c, cu_q, cu_k, seed);
  check(flash::attn_fwd(p, flash::attn_fwd_params::kVersion, current_stream(), nullptr), c.packed ? "attn_fwd (varlen)" : "attn_fwd");
}

// The fp32 dQ accumulator of the fused form, made when the backward asks for it.
struct DqAcc {
  const Tensor* dq;
  Tensor acc;
  static aotriton::TensorView<4> acquire(aotriton::LazyTensor<4>* self) {
    auto* a = static_cast<DqAcc*>(self->cookie);
    a->acc = at::zeros(a->dq->sizes(), a->dq->options().dtype(at::kFloat));
    return view_of<4>(a->acc, aotriton::kFloat32);
  }
};

bool plain_modes() {
  const auto& tls = c10::impl::tls_local_dispatch_key_set();
  return !c10::impl::TorchDispatchModeTLS::any_modes_set() && !at::impl::torch_function_mode_enabled() && !torch::jit::tracer::isTracing() &&
         !tls.included_.has(c10::DispatchKey::Python) && !tls.included_.has(c10::DispatchKey::FuncTorchDynamicLayerFrontMode) &&
         !tls.included_.has(c10::DispatchKey::Functionalize);
}

// Nothing but a strided CUDA tensor on device `dev`, with elements, without a forward-mode gradient.
bool plain(const Tensor& t, int dev) {
  static const uint64_t allowed =
      (c10::DispatchKeySet(c10::DispatchKey::CUDA) | c10::DispatchKeySet(c10::DispatchKey::AutogradCUDA) |
       c10::DispatchKeySet(c10::DispatchKey::ADInplaceOrView) | c10::DispatchKeySet(c10::DispatchKey::AutocastCUDA)).raw_repr();
  return t.defined() && (t.key_set().raw_repr() & ~allowed) == 0 && t.is_cuda() && t.get_device() == dev && t.layout() == at::kStrided &&
         t.numel() != 0 && !t._fw_grad(0).defined();
}
// ... of this type and rank, with a unit innermost stride
bool plain_operand(const Tensor& t, int dev, at::ScalarType type, int64_t dim) {
  return plain(t, dev) && t.scalar_type() == type && t.dim() == dim && t.stride(-1) == 1;
}

struct Attend : torch::autograd::Function<Attend> {
  using Maybe = std::optional<Tensor>;      // (an undefined Tensor is no argument to apply())
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, const Maybe& bias,
                               const Maybe& seqs_q, const Maybe& seqs_k, const Call& c, bool return_lse) {
    const Tensor b = bias.value_or(Tensor()), cu_q = seqs_q.value_or(Tensor()), cu_k = seqs_k.value_or(Tensor());
    Tensor out, lse, seed;
    ::forward(c, q, k, v, b, cu_q, cu_k, true, out, lse, seed);
    ctx->save_for_backward({q, k, v, b, out, lse, cu_q, cu_k});
    if (seed.defined()) ctx->saved_data["seed"] = seed;      // (a number of the call, nothing for a saved-tensor hook to change)
    ctx->saved_data["numbers"] = std::vector<int64_t>{c.causal_type, c.left, c.right, c.max_q, c.max_k, (int64_t)c.seed,
                                                      (int64_t)c.offset, c.packed, c.op};
    ctx->saved_data["scales"] = std::vector<double>{c.sm_scale, c.dropout_p};
    ctx->set_materialize_grads(false);
    return return_lse ? variable_list{out, lse} : variable_list{out};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &q = saved[0], &k = saved[1], &v = saved[2], &b = saved[3], &out = saved[4], &lse = saved[5], &cu_q = saved[6], &cu_k = saved[7];
    const auto found = ctx->saved_data.find("seed");
    const Tensor seed = found == ctx->saved_data.end() ? Tensor() : found->second.toTensor();
    const auto n = ctx->saved_data["numbers"].toIntVector();
    const auto s = ctx->saved_data["scales"].toDoubleVector();
    const Call c{s[0], s[1], n[0], n[1], n[2], n[3], n[4], (uint64_t)n[5], (uint64_t)n[6], n[7] != 0, n[8] != 0};
    variable_list r(8);
    Tensor dout = grads[0].defined() ? grads[0] : at::zeros_like(out);
    // create_graph: the operator, which knows that it has no derivative
    if (c.op && at::GradMode::is_enabled()) {
      operator_backward(c, q, k, v, b, out, dout, lse, seed, r);
      return r;
    }
    // A gradient that is not an ordinary tensor (a batch of them under vmap), a mode that only this pass runs under, or a saved-tensor
    // hook that handed back something else than it was given: what the call stands for deals with it.
    if (!as_saved(q, k, v, b, out, dout, lse, cu_q, cu_k)) {
      if (c.op) operator_backward(c, q, k, v, b, out, dout, lse, seed, r);
      else python_backward(c, q, k, v, b, out, dout, lse, cu_q, cu_k, seed, r);
      return r;
    }
    if (dout.stride(-1) != 1) dout = dout.contiguous();
    const aotriton::DType dt = dtype_of(q.scalar_type());
    r[0] = gradient_of(q);
    r[1] = gradient_of(k);
    r[2] = gradient_of(v);
    if (b.defined()) r[3] = gradient_of(b);
    const Tensor delta = fresh(lse.sizes(), at::kFloat);
    DqAcc acc{&r[0], {}};
    flash::attn_options options;
    flash::attn_bwd_params p;
    p.Q = view_of<4>(q, dt); p.K = view_of<4>(k, dt); p.V = view_of<4>(v, dt); p.B = view_or_null(b, dt);
    p.Out = view_of<4>(out, dt); p.DO = view_of<4>(dout, dt);
    p.DQ = view_of<4>(r[0], dt); p.DK = view_of<4>(r[1], dt); p.DV = view_of<4>(r[2], dt); p.DB = view_or_null(r[3], dt);
    p.L = view_of<2>(lse, aotriton::kFloat32);
    p.D.eager = view_of<2>(delta, aotriton::kFloat32);
    if (c.op) {
      options.deterministic = at::globalContext().deterministicAlgorithms();
      p.DQ_ACC.cookie = &acc;
      p.DQ_ACC.acquire = &DqAcc::acquire;
    }
    fill_common(p, c, cu_q, cu_k, seed);
    check(flash::attn_bwd(p, flash::attn_bwd_params::kVersion, current_stream(), &options), c.packed ? "attn_bwd (varlen)" : "attn_bwd");
    g_last_bwd_family.store(ab200_last_bwd_family(), std::memory_order_relaxed);
    return r;
  }

  static bool as_saved(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& b, const Tensor& out, const Tensor& dout,
                       const Tensor& lse, const Tensor& cu_q, const Tensor& cu_k) {
    if (!plain_modes()) return false;
    const int dev = c10::cuda::current_device();
    const auto type = q.scalar_type();
    for (const Tensor* t : {&q, &k, &v, &out})
      if (!plain_operand(*t, dev, type, 4)) return false;
    for (const Tensor* t : {&cu_q, &cu_k})
      if (t->defined() && !plain_operand(*t, dev, at::kInt, 1)) return false;
    return (!b.defined() || plain_operand(b, dev, type, 4)) && plain_operand(lse, dev, at::kFloat, 2) && lse.is_contiguous() &&
           lse.numel() == q.size(0) * q.size(1) * q.size(2) && plain(dout, dev) && dout.scalar_type() == type && dout.sizes() == out.sizes();
  }

  static void python_backward(const Call& c, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& b, const Tensor& out,
                              const Tensor& dout, const Tensor& lse, const Tensor& cu_q, const Tensor& cu_k, const Tensor& seed,
                              variable_list& r) {
    pybind11::gil_scoped_acquire gil;
    auto wrap = [](const Tensor& t) {
      return t.defined() ? pybind11::reinterpret_steal<pybind11::object>(THPVariable_Wrap(t)) : pybind11::object(pybind11::none());
    };
    const pybind11::object t[] = {wrap(q), wrap(k), wrap(v), wrap(b), wrap(out), wrap(dout), wrap(lse), wrap(cu_q), wrap(cu_k), wrap(seed)};
    const auto result = pybind11::reinterpret_steal<pybind11::object>(PyObject_CallFunction(
        g_python_backward, "OOOOOOOOOOKddLLLLL", t[0].ptr(), t[1].ptr(), t[2].ptr(), t[3].ptr(), t[4].ptr(), t[5].ptr(), t[6].ptr(), t[7].ptr(),
        t[8].ptr(), t[9].ptr(), (unsigned long long)c.offset, c.sm_scale, c.dropout_p, (long long)c.causal_type, (long long)c.left,
        (long long)c.right, (long long)c.max_q, (long long)c.max_k));
    if (!result) {
      python_error e;
      e.persist();
      throw e;
    }
    for (int i = 0; i < (b.defined() ? 4 : 3); ++i) r[i] = THPVariable_Unpack(PyTuple_GET_ITEM(result.ptr(), i));
  }

  static void operator_backward(const Call& c, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& b, const Tensor& out,
                                const Tensor& dout, const Tensor& lse, const Tensor& seed, variable_list& r) {
    const auto one = lse.options().dtype(at::kLong);
    const Tensor sd = (seed.defined() ? seed : at::zeros({1}, one)).view(at::kUInt64);
    const Tensor off = at::full({1}, (int64_t)(c.dropout_p > 0 ? c.offset : 0), one).view(at::kUInt64);
    torch::jit::Stack stack;
    for (const Tensor& t : {q, k, v}) stack.emplace_back(t);
    stack.emplace_back(b.defined() ? c10::IValue(b) : c10::IValue());
    for (const Tensor& t : {out, dout, lse, sd, off}) stack.emplace_back(t);
    stack.emplace_back(c.sm_scale);
    stack.emplace_back(c.dropout_p);
    for (int64_t i : {c.causal_type, c.left, c.right}) stack.emplace_back(i);
    stack.emplace_back(at::globalContext().deterministicAlgorithms());
    c10::Dispatcher::singleton().findSchemaOrThrow("aotriton_b200::attn_bwd", "").callBoxed(&stack);
    for (int i = 0; i < (b.defined() ? 4 : 3); ++i) r[i] = stack[i].toTensor();
  }
};

// ---- what stands around attention -------------------------------------------------------------------------
// The Python Functions that stand for these operators' backwards where the gradient or the modes are not ordinary ones, or where the
// backward is to be differentiated in turn.  By name, set at import, kept for the life of the process.
std::map<std::string, PyObject*>& python_functions() {
  static std::map<std::string, PyObject*> table;
  return table;
}
pybind11::object wrapped(const Tensor& t) {
  return t.defined() ? pybind11::reinterpret_steal<pybind11::object>(THPVariable_Wrap(t)) : pybind11::object(pybind11::none());
}
// (the GIL is held)
pybind11::object call_python(const char* name, const pybind11::tuple& args) {
  auto r = pybind11::reinterpret_steal<pybind11::object>(PyObject_CallObject(python_functions()[name], args.ptr()));
  if (!r) {
    python_error e;
    e.persist();
    throw e;
  }
  return r;
}
PyObject* dtype_object(at::ScalarType t) { return reinterpret_cast<PyObject*>(torch::getTHPDtype(t)); }

int32_t code_of(at::ScalarType t) { return t == at::kFloat ? AB200_DTYPE_FP32 : (t == at::kHalf ? AB200_DTYPE_FP16 : AB200_DTYPE_BF16); }
bool floating(at::ScalarType t) { return t == at::kFloat || t == at::kHalf || t == at::kBFloat16; }
void* stream_handle() { return c10::cuda::getCurrentCUDAStream().stream(); }
ab200_view4 c_view(const Tensor& t) {
  ab200_view4 v;
  v.ptr = t.data_ptr();
  for (int i = 0; i < 4; ++i) { v.size[i] = t.size(i); v.stride[i] = t.stride(i); }
  return v;
}
// A gradient that this file's backwards take as it is.
bool ordinary_gradient(const Tensor& g, at::ScalarType type) {
  return !at::GradMode::is_enabled() && plain_modes() && plain(g, c10::cuda::current_device()) && g.scalar_type() == type;
}

// ---- attention with a sliding window and first keys that stay visible ----
struct SinkCall {
  int64_t max_q, max_k, window, sinks, varlen;      // varlen: AB200_VARLEN_*
  double sm_scale;
};
ab200_attn_problem sink_problem(const SinkCall& c, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& cu_q, const Tensor& cu_k) {
  ab200_attn_problem p{};
  p.dtype = code_of(q.scalar_type());
  p.batch = (int32_t)q.size(0);
  p.num_head_q = (int32_t)q.size(1);
  p.num_head_k = (int32_t)k.size(1);
  p.max_seqlen_q = (int32_t)q.size(2);
  p.max_seqlen_k = (int32_t)k.size(2);
  p.head_dim_qk = (int32_t)q.size(3);
  p.head_dim_vo = (int32_t)v.size(3);
  p.sm_scale = (float)c.sm_scale;
  if (c.varlen) {
    p.batch = (int32_t)cu_q.numel() - 1;
    p.max_seqlen_q = (int32_t)c.max_q;
    p.max_seqlen_k = (int32_t)c.max_k;
    p.varlen_type = (int32_t)c.varlen;
    p.cu_seqlens_q = cu_q.data_ptr<int32_t>();
    p.cu_seqlens_k = cu_k.data_ptr<int32_t>();
  }
  return p;
}
// `lse` is left undefined where nobody will read it.
void sink_forward(const SinkCall& c, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& cu_q, const Tensor& cu_k, bool want_lse, Tensor& out,
                  Tensor& lse) {
  at::AutoDispatchBelowADInplaceOrView guard;
  if (c.varlen == AB200_VARLEN_COMPACT) out = fresh({1, q.size(2), q.size(1), v.size(3)}, q.scalar_type()).transpose(1, 2);
  else out = fresh({q.size(0), q.size(1), q.size(2), v.size(3)}, q.scalar_type());
  if (want_lse) lse = fresh({q.size(0) * q.size(1), q.size(2)}, at::kFloat);
  ab200_attn_fwd_args a{};
  a.prob = sink_problem(c, q, k, v, cu_q, cu_k);
  a.q = c_view(q); a.k = c_view(k); a.v = c_view(v); a.out = c_view(out);
  a.lse = want_lse ? lse.data_ptr<float>() : nullptr;
  check((hipError_t)ab200_sink_attn_fwd(&a, (int32_t)c.window, (int32_t)c.sinks, stream_handle()), "sink_attn_fwd");
}
struct SinkAttend : torch::autograd::Function<SinkAttend> {
  using Maybe = std::optional<Tensor>;
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, const Maybe& seqs_q, const Maybe& seqs_k,
                               const SinkCall& c, bool return_lse) {
    const Tensor cu_q = seqs_q.value_or(Tensor()), cu_k = seqs_k.value_or(Tensor());
    Tensor out, lse;
    sink_forward(c, q, k, v, cu_q, cu_k, true, out, lse);
    ctx->save_for_backward({q, k, v, out, lse, cu_q, cu_k});
    ctx->saved_data["numbers"] = std::vector<int64_t>{c.max_q, c.max_k, c.window, c.sinks, c.varlen};
    ctx->saved_data["scale"] = c.sm_scale;
    ctx->mark_non_differentiable({lse});
    ctx->set_materialize_grads(false);
    return return_lse ? variable_list{out, lse} : variable_list{out};
  }
  // (a saved-tensor hook may hand back anything: what does not match is refused in Python)
  static bool sizes_match(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& out, const Tensor& cu_q, const Tensor& cu_k) {
    for (int i = 0; i < 3; ++i)
      if (k.size(i) != v.size(i) || q.size(i) != out.size(i)) return false;
    return k.size(0) == q.size(0) && k.size(3) == q.size(3) && v.size(3) == out.size(3) && cu_q.defined() == cu_k.defined() &&
           (!cu_q.defined() || cu_q.numel() == cu_k.numel());
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &q = saved[0], &k = saved[1], &v = saved[2], &out = saved[3], &lse = saved[4], &cu_q = saved[5], &cu_k = saved[6];
    const auto n = ctx->saved_data["numbers"].toIntVector();
    const SinkCall c{n[0], n[1], n[2], n[3], n[4], ctx->saved_data["scale"].toDouble()};
    variable_list r(7);
    if (!grads[0].defined()) return r;
    Tensor dout = grads[0];
    // (create_graph: the operator, which knows that it has no derivative; the rest as in Attend::backward)
    if (at::GradMode::is_enabled() || !Attend::as_saved(q, k, v, Tensor(), out, dout, lse, cu_q, cu_k) || !sizes_match(q, k, v, out, cu_q, cu_k)) {
      pybind11::gil_scoped_acquire gil;
      const auto o = call_python("sink_attention", pybind11::make_tuple(wrapped(q), wrapped(k), wrapped(v), wrapped(out), wrapped(dout), wrapped(lse),
                                                                        wrapped(cu_q), wrapped(cu_k), c.max_q, c.max_k, c.window, c.sinks, c.sm_scale, c.varlen));
      for (int i = 0; i < 3; ++i) r[i] = THPVariable_Unpack(PyTuple_GET_ITEM(o.ptr(), i));
      return r;
    }
    if (dout.stride(-1) != 1) dout = dout.size(-1) == 1 ? dout.squeeze(-1).unsqueeze(-1) : dout.contiguous();      // (contiguous() leaves one column's stride)
    r[0] = gradient_of(q);
    r[1] = gradient_of(k);
    r[2] = gradient_of(v);
    const Tensor delta = fresh(lse.sizes(), at::kFloat);
    ab200_attn_bwd_args a{};
    a.prob = sink_problem(c, q, k, v, cu_q, cu_k);
    a.q = c_view(q); a.k = c_view(k); a.v = c_view(v); a.out = c_view(out); a.dout = c_view(dout);
    a.dq = c_view(r[0]); a.dk = c_view(r[1]); a.dv = c_view(r[2]);
    a.lse = lse.data_ptr<float>();
    a.delta = delta.data_ptr<float>();
    const int64_t need = ab200_sink_attn_bwd_workspace(&a, (int32_t)c.window, (int32_t)c.sinks, stream_handle());
    if (need < 0) check((hipError_t)-need, "sink_attn_bwd");
    const Tensor workspace = need > 0 ? fresh({need}, at::kFloat) : Tensor();
    check((hipError_t)ab200_sink_attn_bwd(&a, (int32_t)c.window, (int32_t)c.sinks, need > 0 ? workspace.data_ptr<float>() : nullptr, (uint64_t)need,
                                          stream_handle()),
          "sink_attn_bwd");
    g_last_bwd_family.store(ab200_last_bwd_family(), std::memory_order_relaxed);
    return r;
  }
};

// ---- dropout with the residual's addition ----
// t as rows of unit stride: (rows, cols, stride between rows); false where its strides give none.
bool rows_of(const Tensor& t, int64_t* rows, int64_t* cols, int64_t* stride) {
  if (t.is_contiguous()) {
    *cols = t.dim() ? t.size(-1) : 1;
    *rows = t.numel() / *cols;
    *stride = *cols;
    return true;
  }
  if (t.stride(-1) != 1 && t.size(-1) != 1) return false;
  *cols = t.size(-1);
  *rows = 1;
  *stride = *cols;
  for (int64_t i = t.dim() - 2; i >= 0; --i) {      // (from the innermost: one stride for all rows)
    if (t.size(i) == 1) continue;
    if (*rows == 1) *stride = t.stride(i);
    else if (t.stride(i) != *stride * *rows) return false;
    *rows *= t.size(i);
  }
  return true;
}
Tensor drop(const Tensor& x, const Tensor& residual, double p, uint64_t seed, uint64_t offset) {
  at::AutoDispatchBelowADInplaceOrView guard;
  Tensor out = fresh(x.sizes(), x.scalar_type()), from = x, add = residual;
  ab200_dropout_args a{};
  a.dtype = code_of(x.scalar_type());
  a.dropout_p = (float)p;
  if (!rows_of(from, &a.rows, &a.cols, &a.x_stride)) {
    from = from.contiguous();
    rows_of(from, &a.rows, &a.cols, &a.x_stride);
  }
  int64_t rows, cols;
  if (add.defined() && !rows_of(add, &rows, &cols, &a.residual_stride)) {
    add = add.contiguous();
    rows_of(add, &rows, &cols, &a.residual_stride);
  }
  a.x = from.data_ptr();
  a.residual = add.defined() ? add.data_ptr() : nullptr;
  a.out = out.data_ptr();
  a.out_stride = a.cols;
  a.philox_seed_value = seed;
  a.philox_offset2 = offset;
  check((hipError_t)ab200_dropout(&a, stream_handle()), "dropout");
  return out;
}

struct Drop : torch::autograd::Function<Drop> {
  using Maybe = std::optional<Tensor>;
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Maybe& residual, double p, uint64_t seed, uint64_t offset) {
    ctx->saved_data["p"] = p;
    ctx->saved_data["numbers"] = std::vector<int64_t>{(int64_t)seed, (int64_t)offset, residual.has_value(), (int64_t)x.scalar_type()};
    ctx->set_materialize_grads(false);
    return drop(x, residual.value_or(Tensor()), p, seed, offset);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list r(5);
    const Tensor& g = grads[0];
    if (!g.defined()) return r;
    const double p = ctx->saved_data["p"].toDouble();
    const auto n = ctx->saved_data["numbers"].toIntVector();
    if (n[2] && ctx->needs_input_grad(1)) r[1] = g;
    if (!ctx->needs_input_grad(0)) return r;
    if (ordinary_gradient(g, (at::ScalarType)n[3])) {
      r[0] = drop(g, Tensor(), p, (uint64_t)n[0], (uint64_t)n[1]);
    } else {
      pybind11::gil_scoped_acquire gil;
      const auto o = call_python("dropout", pybind11::make_tuple(wrapped(g), p, (uint64_t)n[0], (uint64_t)n[1]));
      r[0] = THPVariable_Unpack(o.ptr());
    }
    return r;
  }
};

// ---- learned relative position bias ----
struct BiasCall {
  int64_t sq, sk, batch, offset;
  bool both;
  at::ScalarType type;
  std::string borders;      // int32 each
};
ab200_relative_bias_args bias_args(const Tensor& table, const Tensor& bias, const std::string& borders, bool both, int64_t offset) {
  ab200_relative_bias_args a{};
  a.dtype = code_of(bias.scalar_type());
  a.table_dtype = code_of(table.scalar_type());
  a.num_buckets = (int32_t)table.size(0);
  a.num_heads = (int32_t)table.size(1);
  a.bidirectional = both;
  a.query_offset = (int32_t)offset;
  a.borders = reinterpret_cast<const int32_t*>(borders.data());
  a.table = table.data_ptr();
  a.table_stride[0] = table.stride(0);
  a.table_stride[1] = table.stride(1);
  a.bias = c_view(bias);
  return a;
}
// Rows of a multiple of 32 bytes, which the kernels that write and read them take 16 or 32 bytes at a time.
Tensor make_bias(const Tensor& table, const BiasCall& c) {
  at::AutoDispatchBelowADInplaceOrView guard;
  const int64_t per = c.type == at::kFloat ? 8 : 16, heads = table.size(1), pitch = (c.sk + per - 1) / per * per;
  const Tensor store = fresh({heads, c.sq, pitch}, c.type);
  const Tensor one = store.as_strided({1, heads, c.sq, c.sk}, {0, c.sq * pitch, pitch, 1});
  const auto a = bias_args(table, one, c.borders, c.both, c.offset);
  check((hipError_t)ab200_relative_bias_fwd(&a, stream_handle()), "relative_bias_fwd");
  return store.as_strided({c.batch, heads, c.sq, c.sk}, {0, c.sq * pitch, pitch, 1});
}
struct RelativeBias : torch::autograd::Function<RelativeBias> {
  static Tensor forward(AutogradContext* ctx, const Tensor& table, const BiasCall& c) {
    ctx->saved_data["numbers"] = std::vector<int64_t>{table.size(0), table.size(1), (int64_t)table.scalar_type(), (int64_t)c.type, c.both, c.offset};
    ctx->saved_data["borders"] = c.borders;
    ctx->set_materialize_grads(false);
    return make_bias(table, c);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list r(2);
    const Tensor& g = grads[0];
    if (!g.defined()) return r;
    const auto n = ctx->saved_data["numbers"].toIntVector();
    const std::string& borders = ctx->saved_data["borders"].toStringRef();
    const auto table_type = (at::ScalarType)n[2];
    if (!ordinary_gradient(g, (at::ScalarType)n[3])) {
      pybind11::gil_scoped_acquire gil;
      const auto dt = pybind11::reinterpret_borrow<pybind11::object>(dtype_object(table_type));
      const auto o = call_python("relative_bias", pybind11::make_tuple(wrapped(g), n[0], n[1], dt, pybind11::bytes(borders), n[4] != 0, n[5]));
      r[0] = THPVariable_Unpack(o.ptr());
      return r;
    }
    r[0] = fresh({n[0], n[1]}, table_type);
    auto a = bias_args(r[0], g, borders, n[4] != 0, n[5]);
    const int64_t need = ab200_relative_bias_workspace(&a, stream_handle());
    if (need < 0) check((hipError_t)-need, "relative_bias_bwd");
    const Tensor workspace = fresh({need}, at::kFloat);
    a.workspace = static_cast<float*>(workspace.data_ptr());
    a.workspace_floats = (uint64_t)need;
    check((hipError_t)ab200_relative_bias_bwd(&a, stream_handle()), "relative_bias_bwd");
    return r;
  }
};

// ---- from Python ------------------------------------------------------------------------------------------

// A torch.Tensor or Parameter (no subclass) that is plain().  The tensor itself goes to *out.
bool plain_tensor(PyObject* o, int dev, Tensor* out) {
  if (!THPVariable_CheckExact(o)) return false;
  const Tensor& t = THPVariable_Unpack(o);
  if (!plain(t, dev) || t.stride(-1) != 1) return false;
  *out = t;
  return true;
}
bool attention_operand(PyObject* o, int dev, Tensor* out) {
  if (!plain_tensor(o, dev, out)) return false;
  const auto t = out->scalar_type();
  return out->dim() == 4 && (t == at::kFloat || t == at::kHalf || t == at::kBFloat16);
}
bool small_int(PyObject* o, int64_t* out) {      // fits the C API's int32
  if (!PyLong_CheckExact(o)) return false;
  *out = PyLong_AsLongLong(o);
  if (*out == -1 && PyErr_Occurred()) { PyErr_Clear(); return false; }
  return *out >= INT32_MIN && *out <= INT32_MAX;
}
bool u64(PyObject* o, uint64_t* out) {
  if (!PyLong_CheckExact(o)) return false;
  *out = PyLong_AsUnsignedLongLong(o);
  if (*out == (uint64_t)-1 && PyErr_Occurred()) { PyErr_Clear(); return false; }
  return true;
}
bool number(PyObject* o, double* out) {
  if (!PyFloat_CheckExact(o) && !PyLong_CheckExact(o)) return false;
  *out = PyFloat_AsDouble(o);
  if (*out == -1.0 && PyErr_Occurred()) { PyErr_Clear(); return false; }
  return true;
}

// attend(q, k, v, bias, cu_seqlens_q, cu_seqlens_k, max_seqlen_q, max_seqlen_k, sm_scale, dropout_p, causal_type, window_left,
// window_right, return_lse, philox_seed, philox_offset, op): out, or (out, lse), or None: not an ordinary call.
PyObject* attend(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 17) {
    PyErr_SetString(PyExc_TypeError, "attend takes 17 arguments");
    return nullptr;
  }
  Call c{};
  Tensor q, k, v, b, cu_q, cu_k;
  // (a process without a CUDA context yet has no tensor to look at either)
  if (!THPVariable_CheckExact(a[0]) || !THPVariable_Unpack(a[0]).is_cuda() || !plain_modes()) Py_RETURN_NONE;
  const int dev = c10::cuda::current_device();
  if (!attention_operand(a[0], dev, &q) || !attention_operand(a[1], dev, &k) || !attention_operand(a[2], dev, &v)) Py_RETURN_NONE;
  if (a[3] != Py_None && !attention_operand(a[3], dev, &b)) Py_RETURN_NONE;
  if (k.scalar_type() != q.scalar_type() || v.scalar_type() != q.scalar_type() || (b.defined() && b.scalar_type() != q.scalar_type()))
    Py_RETURN_NONE;
  c.packed = a[4] != Py_None;
  if (c.packed) {
    for (int i = 0; i < 2; ++i) {
      Tensor& cu = i ? cu_k : cu_q;
      if (!plain_tensor(a[4 + i], dev, &cu) || cu.dim() != 1 || cu.numel() < 2 || cu.scalar_type() != at::kInt) Py_RETURN_NONE;
    }
    if (b.defined() || q.size(0) != 1 || !small_int(a[6], &c.max_q) || !small_int(a[7], &c.max_k)) Py_RETURN_NONE;
  }
  if (!number(a[8], &c.sm_scale) || !number(a[9], &c.dropout_p) || !small_int(a[10], &c.causal_type) || !small_int(a[11], &c.left) ||
      !small_int(a[12], &c.right))
    Py_RETURN_NONE;
  const bool return_lse = a[13] == Py_True;
  if (!return_lse && a[13] != Py_False) Py_RETURN_NONE;
  if (c.dropout_p > 0 && (!u64(a[14], &c.seed) || !u64(a[15], &c.offset))) Py_RETURN_NONE;
  c.op = a[16] == Py_True;
  Tensor out, lse;
  {
    pybind11::gil_scoped_release release;
    const bool grad = at::GradMode::is_enabled() &&
                      (q.requires_grad() || k.requires_grad() || v.requires_grad() || (b.defined() && b.requires_grad()));
    if (grad) {
      auto maybe = [](const Tensor& t) { return t.defined() ? Attend::Maybe(t) : Attend::Maybe(); };
      variable_list r = Attend::apply(q, k, v, maybe(b), maybe(cu_q), maybe(cu_k), c, return_lse);
      out = std::move(r[0]);
      if (return_lse) lse = std::move(r[1]);
    } else {
      Tensor seed;
      forward(c, q, k, v, b, cu_q, cu_k, return_lse, out, lse, seed);
    }
  }
  if (!return_lse) return THPVariable_Wrap(std::move(out));
  return PyTuple_Pack(2, pybind11::reinterpret_steal<pybind11::object>(THPVariable_Wrap(std::move(out))).ptr(),
                      pybind11::reinterpret_steal<pybind11::object>(THPVariable_Wrap(std::move(lse))).ptr());
  END_HANDLE_TH_ERRORS
}

// sink_attend(q, k, v, cu_seqlens_q, cu_seqlens_k, max_seqlen_q, max_seqlen_k, window, sinks, sm_scale, return_lse, varlen): out, or (out, lse),
// or None: not an ordinary call, or one whose arguments the caller is to look at.
PyObject* sink_attend(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 12) {
    PyErr_SetString(PyExc_TypeError, "sink_attend takes 12 arguments");
    return nullptr;
  }
  if (!THPVariable_CheckExact(a[0]) || !THPVariable_Unpack(a[0]).is_cuda() || !plain_modes()) Py_RETURN_NONE;
  const int dev = c10::cuda::current_device();
  SinkCall c{};
  Tensor q, k, v, cu_q, cu_k;
  if (!attention_operand(a[0], dev, &q) || !attention_operand(a[1], dev, &k) || !attention_operand(a[2], dev, &v)) Py_RETURN_NONE;
  if (k.scalar_type() != q.scalar_type() || v.scalar_type() != q.scalar_type()) Py_RETURN_NONE;
  if (!small_int(a[11], &c.varlen) || !small_int(a[7], &c.window) || !small_int(a[8], &c.sinks) || !number(a[9], &c.sm_scale)) Py_RETURN_NONE;
  const bool return_lse = a[10] == Py_True;
  if (!return_lse && a[10] != Py_False) Py_RETURN_NONE;
  if (c.window < 1 || c.sinks < 0 || k.size(0) != q.size(0) || v.size(0) != k.size(0) || v.size(1) != k.size(1) || v.size(2) != k.size(2) ||
      k.size(3) != q.size(3) || q.size(1) % k.size(1) != 0 || q.size(3) > 512 || v.size(3) > 512)
    Py_RETURN_NONE;
  if (c.varlen) {
    for (int i = 0; i < 2; ++i) {
      Tensor& cu = i ? cu_k : cu_q;
      if (!plain_tensor(a[3 + i], dev, &cu) || cu.dim() != 1 || cu.numel() < 2 || cu.scalar_type() != at::kInt) Py_RETURN_NONE;
    }
    if (cu_q.numel() != cu_k.numel() || !small_int(a[5], &c.max_q) || !small_int(a[6], &c.max_k)) Py_RETURN_NONE;
    if (c.max_q < 1 || c.max_q > q.size(2) || c.max_k < 1 || c.max_k > k.size(2)) Py_RETURN_NONE;
    if (c.varlen == AB200_VARLEN_COMPACT ? q.size(0) != 1 : cu_q.numel() != q.size(0) + 1) Py_RETURN_NONE;
    if (c.varlen == AB200_VARLEN_PADDED) c.max_q = q.size(2);
  }
  Tensor out, lse;
  {
    pybind11::gil_scoped_release release;
    if (at::GradMode::is_enabled() && (q.requires_grad() || k.requires_grad() || v.requires_grad())) {
      auto maybe = [](const Tensor& t) { return t.defined() ? SinkAttend::Maybe(t) : SinkAttend::Maybe(); };
      variable_list r = SinkAttend::apply(q, k, v, maybe(cu_q), maybe(cu_k), c, return_lse);
      out = std::move(r[0]);
      if (return_lse) lse = std::move(r[1]);
    } else {
      sink_forward(c, q, k, v, cu_q, cu_k, return_lse, out, lse);
    }
  }
  if (!return_lse) return THPVariable_Wrap(std::move(out));
  return PyTuple_Pack(2, pybind11::reinterpret_steal<pybind11::object>(THPVariable_Wrap(std::move(out))).ptr(),
                      pybind11::reinterpret_steal<pybind11::object>(THPVariable_Wrap(std::move(lse))).ptr());
  END_HANDLE_TH_ERRORS
}

// A floating-point tensor this file's operators take, of any shape and strides; or not.
bool floating_tensor(PyObject* o, int dev, Tensor* out) {
  if (!THPVariable_CheckExact(o)) return false;
  const Tensor& t = THPVariable_Unpack(o);
  if (!plain(t, dev) || !floating(t.scalar_type())) return false;
  *out = t;
  return true;
}
bool ordinary_first(PyObject* o) { return THPVariable_CheckExact(o) && THPVariable_Unpack(o).is_cuda() && plain_modes(); }

// dropout(x, residual, dropout_p, philox_seed, philox_offset): the output, or None: not an ordinary call.
PyObject* dropout(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 5) {
    PyErr_SetString(PyExc_TypeError, "dropout takes 5 arguments");
    return nullptr;
  }
  if (!ordinary_first(a[0])) Py_RETURN_NONE;
  const int dev = c10::cuda::current_device();
  Tensor x, residual;
  double p;
  uint64_t seed, offset;
  if (!floating_tensor(a[0], dev, &x) || (a[1] != Py_None && !floating_tensor(a[1], dev, &residual))) Py_RETURN_NONE;
  if (!number(a[2], &p) || !u64(a[3], &seed) || !u64(a[4], &offset)) Py_RETURN_NONE;
  Tensor out;
  {
    pybind11::gil_scoped_release release;
    if (at::GradMode::is_enabled() && (x.requires_grad() || (residual.defined() && residual.requires_grad())))
      out = Drop::apply(x, residual.defined() ? Drop::Maybe(residual) : Drop::Maybe(), p, seed, offset);
    else
      out = drop(x, residual, p, seed, offset);
  }
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// relative_bias(table, seqlen_q, seqlen_k, batch, borders, bidirectional, query_offset, dtype): the bias, or None: not an ordinary call.
PyObject* relative_bias(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 8) {
    PyErr_SetString(PyExc_TypeError, "relative_bias takes 8 arguments");
    return nullptr;
  }
  if (!ordinary_first(a[0])) Py_RETURN_NONE;
  const int dev = c10::cuda::current_device();
  Tensor table;
  BiasCall c{};
  if (!floating_tensor(a[0], dev, &table) || table.dim() != 2) Py_RETURN_NONE;
  if (!small_int(a[1], &c.sq) || !small_int(a[2], &c.sk) || !small_int(a[3], &c.batch) || !small_int(a[6], &c.offset)) Py_RETURN_NONE;
  if (c.sq <= 0 || c.sk <= 0 || c.batch <= 0 || !PyBytes_CheckExact(a[4]) || !THPDtype_Check(a[7])) Py_RETURN_NONE;
  c.borders.assign(PyBytes_AS_STRING(a[4]), PyBytes_GET_SIZE(a[4]));
  c.both = a[5] == Py_True;
  c.type = reinterpret_cast<THPDtype*>(a[7])->scalar_type;
  if (!floating(c.type)) Py_RETURN_NONE;
  Tensor out;
  {
    pybind11::gil_scoped_release release;
    out = at::GradMode::is_enabled() && table.requires_grad() ? RelativeBias::apply(table, c) : make_bias(table, c);
  }
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// set_python_function(name, fn): what python_functions() holds.
PyObject* set_python_function(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 2 || !PyUnicode_Check(a[0])) {
    PyErr_SetString(PyExc_TypeError, "set_python_function takes a name and a function");
    return nullptr;
  }
  Py_INCREF(a[1]);
  PyObject*& slot = python_functions()[PyUnicode_AsUTF8(a[0])];
  Py_XDECREF(slot);
  slot = a[1];
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

PyObject* last_bwd_family(PyObject*, PyObject*) { return PyLong_FromLong(g_last_bwd_family.load(std::memory_order_relaxed)); }
// ... of a backward that ran on this thread by the Python way
PyObject* note_bwd_family(PyObject*, PyObject*) {
  g_last_bwd_family.store(ab200_last_bwd_family(), std::memory_order_relaxed);
  Py_RETURN_NONE;
}

// The Function's backward: (q, k, v, bias, out, dout, logsumexp, cu_seqlens_q, cu_seqlens_k, seed, offset, sm_scale, dropout_p, causal_type,
// window_left, window_right, max_seqlen_q, max_seqlen_k) -> (dq, dk, dv, dbias).  Kept for the life of the process.
PyObject* set_python_backward(PyObject*, PyObject* fn) {
  Py_INCREF(fn);
  std::swap(g_python_backward, fn);
  Py_XDECREF(fn);
  Py_RETURN_NONE;
}

PyMethodDef kMethods[] = {{"attend", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&attend)), METH_FASTCALL, nullptr},
                          {"sink_attend", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&sink_attend)), METH_FASTCALL, nullptr},
                          {"dropout", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&dropout)), METH_FASTCALL, nullptr},
                          {"relative_bias", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&relative_bias)), METH_FASTCALL, nullptr},
                          {"set_python_function", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&set_python_function)), METH_FASTCALL, nullptr},
                          {"set_python_backward", &set_python_backward, METH_O, nullptr},
                          {"last_bwd_family", &last_bwd_family, METH_NOARGS, nullptr},
                          {"note_bwd_family", &note_bwd_family, METH_NOARGS, nullptr},
                          {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_torch_ops", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__torch_ops() { return PyModule_Create(&kModule); }
