// dfs_torch_attn.cpp -- autograd glue of the local attention and its learned
// relative position bias (include/dfsink.h: dfs_window_attn_*, dfs_relbias_*).
// Nothing here computes: shapes are checked, outputs and workspaces come from
// the caching allocator, and the C ABI runs on the current stream.
//
// Device errors (a bounded wait that gave up) are written by the kernels
// straight into one word of mapped host memory per device, so a call pays
// nothing for them: the next attention call (or its check_status) reads the
// word, which the other operators' calls leave alone.
#include <ATen/cuda/CUDAContext.h>
#include <torch/csrc/autograd/functions/basic_ops.h>

#include <initializer_list>
#include <limits>
#include <mutex>

#include "dfs_torch.h"

namespace dfs_torch {
namespace {

using at::Tensor;
using c10::optional;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

constexpr int kMaxDevices = 64;
std::mutex g_mu;
int32_t* g_word[kMaxDevices] = {};  // never freed: kernels may still write at exit

int32_t* status_word(const at::Device& dev) {
  const int i = dev.index();
  require(i >= 0 && i < kMaxDevices, "device index out of range");
  std::lock_guard<std::mutex> lock(g_mu);
  if (g_word[i] == nullptr) {
    void* p = nullptr;
    require(cudaHostAlloc(&p, sizeof(int32_t), cudaHostAllocMapped | cudaHostAllocPortable) == cudaSuccess,
            "cudaHostAlloc failed");
    *static_cast<int32_t*>(p) = 0;
    g_word[i] = static_cast<int32_t*>(p);
  }
  return g_word[i];
}

// A call's status word, after raising for an error that an earlier call left there.
int32_t* checked_status(const at::Device& dev) {
  int32_t* w = status_word(dev);
  const int v = __atomic_load_n(w, __ATOMIC_RELAXED);
  if (v != 0) {
    __atomic_store_n(w, 0, __ATOMIC_RELAXED);
    fail(std::string("a previous window attention call reported a device error: ") + dfs_status_string(v) +
         " (status " + std::to_string(v) + ")");
  }
  return w;
}

int32_t narrow32(int64_t v, const char* what) {
  if (v > std::numeric_limits<int32_t>::max() || v < std::numeric_limits<int32_t>::min())
    fail(std::string(what) + " does not fit 32 bits");
  return static_cast<int32_t>(v);
}

bool float_type(const Tensor& t) {
  const auto s = t.scalar_type();
  return s == at::kBFloat16 || s == at::kHalf || s == at::kFloat;
}

// No kernel computes a tangent: a call on dual tensors (forward-mode derivatives) that went on would drop theirs,
// which reads as a derivative of 0.
void refuse_tangents(std::initializer_list<optional<Tensor>> operands) {
  for (const auto& t : operands)
    require(!t.has_value() || !t->defined() || !t->_fw_grad(/*level=*/0).defined(),
            "deepfold B200 attention and position bias have no forward-mode derivatives");
}

// What a backward returns.  Where it is itself recorded (create_graph) its gradients carry an error in place of the
// second derivative that the kernels lack: without a history they would count as constants.
variable_list once_differentiable(variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  variable_list in;
  for (const Tensor& g : grads)
    if (g.defined()) in.push_back(g.detach().requires_grad_());
  const auto n = static_cast<int64_t>(in.size());
  variable_list out = torch::autograd::DelayedError(
      "deepfold B200 attention and position bias are differentiable once only", n).apply(std::move(in));
  auto next = out.begin();
  for (Tensor& g : grads)
    if (g.defined()) g = *next++;
  return grads;
}

// The tensor itself where the kernels can walk it (unit stride along d, no row
// that is several rows' memory), else a dense copy.
Tensor walkable(const Tensor& t) {
  bool ok = t.size(-1) <= 1 || t.stride(-1) == 1;
  for (int64_t i = 0; i + 1 < t.dim(); ++i) ok = ok && (t.size(i) <= 1 || t.stride(i) > 0);
  return ok ? t : t.contiguous();
}
// An output laid out as `t` is.
Tensor like(const Tensor& t) { return t.numel() ? at::empty_like(t) : at::empty(t.sizes(), t.options()); }

// (B, heads, n, d); a (B, heads, d) tensor has one row per head
dfs_strided strided(const Tensor& t) {
  return {t.data_ptr(), t.stride(0), t.stride(1), t.dim() == 4 ? t.stride(2) : 0};
}

dfs_relbias bias_of(const Tensor& w, const Tensor& lut, int64_t max_distance) {
  dfs_relbias b{};
  if (!w.defined()) return b;
  b.weight = w.data_ptr();
  b.lut = lut.data_ptr<int32_t>();
  b.num_buckets = narrow32(w.size(1), "num_buckets");
  b.max_distance = narrow32(max_distance, "max_distance");
  b.dtype = dtype_code(w.scalar_type());
  return b;
}

void check_bias(const Tensor& w, const optional<Tensor>& lut, int64_t H, int64_t max_distance, const at::Device& dev) {
  require(lut.has_value() && lut->defined(), "pos_weight needs buckets");
  require(w.device() == dev && lut->device() == dev, "pos_weight and buckets must be on the operands' device");
  require(float_type(w), "pos_weight must be bfloat16, float16 or float32");
  require(w.dim() == 2 && w.size(0) == H && w.size(1) > 0, "pos_weight must be (H, num_buckets)");
  require(lut->scalar_type() == at::kInt && lut->is_contiguous() && lut->numel() == 2 * max_distance + 1,
          "buckets: int32 (2 max_distance + 1)");
}

struct Problem {
  dfs_attn_problem p{};
  Tensor q, k, v, mask, w, lut;
  int64_t max_distance = 0;
};

Problem make_problem(const Tensor& Q, const Tensor& K, const Tensor& V, const optional<Tensor>& mask,
                     const optional<Tensor>& weight, const optional<Tensor>& lut, int64_t max_distance, int64_t window,
                     int64_t sinks, bool causal, int64_t q_start, double scale) {
  require(Q.is_cuda() && K.is_cuda() && V.is_cuda(), "deepfold B200 attention runs on CUDA tensors only (no CPU path)");
  require(K.device() == Q.device() && V.device() == Q.device(), "Q, K, V must be on one device");
  require(K.dim() == 4 && V.sizes() == K.sizes() && K.size(0) == Q.size(0) && K.size(3) == Q.size(-1),
          "Q must be (B, H, n_q, d); K and V (B, H_kv, n_k, d)");
  require(float_type(Q) && K.scalar_type() == Q.scalar_type() && V.scalar_type() == Q.scalar_type(),
          "Q, K, V must share one type: bfloat16, float16 or float32");
  const int64_t B = Q.size(0), H = Q.size(1), Hkv = K.size(1), d = Q.size(-1);
  require(H == 0 || (Hkv > 0 && H % Hkv == 0), "the query heads must be a multiple of the key heads");
  require(d >= 1 && d <= 64, "head dims 1 to 64 are supported");
  Problem r;
  r.q = walkable(Q);
  r.k = walkable(K);
  r.v = walkable(V);
  if (mask.has_value() && mask->defined()) {
    require(mask->device() == Q.device(), "mask must be on the operands' device");
    require(mask->dim() == 2 && mask->size(0) == B && mask->size(1) == K.size(2), "mask must be (B, n_k)");
    const auto t = mask->scalar_type();
    r.mask = (t == at::kBool || t == at::kByte) ? mask->contiguous() : mask->ne(0).contiguous();
  }
  if (weight.has_value() && weight->defined()) {
    check_bias(*weight, lut, H, max_distance, Q.device());
    r.w = weight->contiguous();
    r.lut = *lut;
    r.max_distance = max_distance;
  }
  dfs_attn_problem& p = r.p;
  p.B = narrow32(B, "B");
  p.H = narrow32(H, "H");
  p.H_kv = narrow32(Hkv, "H_kv");
  p.n_q = Q.dim() == 4 ? narrow32(Q.size(2), "n_q") : 1;
  p.n_k = narrow32(K.size(2), "n_k");
  p.d = static_cast<int32_t>(d);
  p.dtype = dtype_code(Q.scalar_type());
  p.causal = causal;
  p.window = narrow32(window, "window");
  p.sinks = narrow32(sinks, "sinks");
  p.q_start = narrow32(q_start, "q_start");
  p.scale = static_cast<float>(scale);
  return r;
}

dfs_attn_args args_of(const Problem& r, const Tensor& o, const Tensor& lse, const Tensor& o_lo) {
  dfs_attn_args a{};
  a.q = strided(r.q);
  a.k = strided(r.k);
  a.v = strided(r.v);
  a.o = strided(o);
  a.lse = lse.defined() ? lse.data_ptr<float>() : nullptr;
  a.mask = r.mask.defined() ? static_cast<const uint8_t*>(r.mask.data_ptr()) : nullptr;
  a.bias = bias_of(r.w, r.lut, r.max_distance);
  a.o_lo = o_lo.defined() ? o_lo.data_ptr() : nullptr;
  return a;
}

cudaStream_t stream_of(const Tensor& t) { return at::cuda::getCurrentCUDAStream(t.device().index()).stream(); }

// keep: what the backward needs, lse and (16-bit types) what the rounding of o took
Tensor run_forward(const Problem& r, bool keep, Tensor* lse, Tensor* o_lo) {
  const DeviceSwitch guard(r.q.device());
  Tensor o = like(r.q);
  if (keep) *lse = at::empty({r.q.size(0), r.q.size(1), r.q.size(2)}, r.q.options().dtype(at::kFloat));
  if (keep && r.p.dtype != DFS_F32) *o_lo = like(r.q);
  dfs_attn_args a = args_of(r, o, keep ? *lse : Tensor(), keep ? *o_lo : Tensor());
  a.status = checked_status(r.q.device());
  check_rc(dfs_window_attn_fwd(&r.p, &a, stream_of(r.q)), "dfs_window_attn_fwd");
  return o;
}

struct WindowAttnFn : public torch::autograd::Function<WindowAttnFn> {
  static Tensor forward(AutogradContext* ctx, Tensor Q, Tensor K, Tensor V, optional<Tensor> weight,
                        optional<Tensor> mask, optional<Tensor> lut, int64_t max_distance, int64_t window,
                        int64_t sinks, bool causal, int64_t q_start, double scale) {
    const Problem r = make_problem(Q, K, V, mask, weight, lut, max_distance, window, sinks, causal, q_start, scale);
    Tensor lse, o_lo;
    Tensor o = run_forward(r, true, &lse, &o_lo);
    ctx->save_for_backward({r.q, r.k, r.v, r.mask, r.w, r.lut, o, lse, o_lo});
    ctx->saved_data["max_distance"] = max_distance;
    ctx->saved_data["window"] = window;
    ctx->saved_data["sinks"] = sinks;
    ctx->saved_data["causal"] = causal;
    ctx->saved_data["q_start"] = q_start;
    ctx->saved_data["scale"] = scale;
    return o;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto s = ctx->get_saved_variables();
    variable_list out(12);
    if (!grads[0].defined()) return out;
    auto opt = [](const Tensor& t) { return t.defined() ? optional<Tensor>(t) : c10::nullopt; };
    const Problem r = make_problem(s[0], s[1], s[2], opt(s[3]), opt(s[4]), opt(s[5]),
                                   ctx->saved_data["max_distance"].toInt(), ctx->saved_data["window"].toInt(),
                                   ctx->saved_data["sinks"].toInt(), ctx->saved_data["causal"].toBool(),
                                   ctx->saved_data["q_start"].toInt(), ctx->saved_data["scale"].toDouble());
    const Tensor &o = s[6], &lse = s[7], &o_lo = s[8];
    const DeviceSwitch guard(r.q.device());
    const Tensor dO = walkable(grads[0].to(r.q.scalar_type()));
    Tensor dq = like(r.q), dk = like(r.k), dv = like(r.v), dw;
    const bool want_w = r.w.defined() && ctx->needs_input_grad(3);  // the edge after Q, K, V where there is one
    if (want_w) dw = at::empty_like(r.w);
    dfs_attn_args a = args_of(r, o, lse, o_lo);
    a.d_o = strided(dO);
    a.d_q = strided(dq);
    a.d_k = strided(dk);
    a.d_v = strided(dv);
    a.d_weight = want_w ? dw.data_ptr() : nullptr;
    a.status = status_word(r.q.device());  // errors are raised by the next forward: autograd's threads stay clean
    const size_t bytes = dfs_window_attn_bwd_work(&r.p, want_w ? &a.bias : nullptr);
    const Tensor work = at::empty({static_cast<int64_t>(bytes)}, r.q.options().dtype(at::kByte));
    check_rc(dfs_window_attn_bwd(&r.p, &a, bytes ? work.data_ptr() : nullptr, bytes, stream_of(r.q)),
             "dfs_window_attn_bwd");
    out[0] = dq;
    out[1] = dk;
    out[2] = dv;
    if (want_w) out[3] = dw;
    return once_differentiable(out);
  }
};

Tensor window_attn(Tensor Q, Tensor K, Tensor V, optional<Tensor> mask, optional<Tensor> weight, optional<Tensor> lut,
                   int64_t max_distance, int64_t window, int64_t sinks, bool causal, int64_t q_start, double scale) {
  refuse_tangents({Q, K, V, weight});
  const bool has_w = weight.has_value() && weight->defined();
  const bool grad = at::GradMode::is_enabled() && (Q.requires_grad() || K.requires_grad() || V.requires_grad() ||
                                                   (has_w && weight->requires_grad()));
  require(Q.dim() == 4, "Q must be (B, H, n_q, d)");
  if (grad)
    return WindowAttnFn::apply(Q, K, V, has_w ? weight : c10::nullopt, mask, lut, max_distance, window, sinks,
                               causal, q_start, scale);
  return run_forward(make_problem(Q, K, V, mask, weight, lut, max_distance, window, sinks, causal, q_start, scale),
                     false, nullptr, nullptr);
}

Tensor window_attn_decode(Tensor q, Tensor K, Tensor V, Tensor lengths, optional<Tensor> weight, optional<Tensor> lut,
                          int64_t max_distance, int64_t window, int64_t sinks, double scale) {
  refuse_tangents({q, K, V, weight});
  require(q.dim() == 3, "q must be (B, H, d)");
  const Problem r = make_problem(q, K, V, c10::nullopt, weight, lut, max_distance, window, sinks, true, 0,
                                 scale);
  require(lengths.is_cuda() && lengths.device() == q.device() && lengths.dim() == 1 && lengths.size(0) == q.size(0) &&
              (lengths.scalar_type() == at::kInt || lengths.scalar_type() == at::kLong),
          "lengths must be (B,) int32 or int64 on the operands' device");
  const Tensor len = lengths.contiguous();
  const DeviceSwitch guard(q.device());
  Tensor o = at::empty(q.sizes(), q.options());
  dfs_attn_args a = args_of(r, o, Tensor(), Tensor());
  a.status = checked_status(q.device());
  check_rc(len.scalar_type() == at::kInt
               ? dfs_window_attn_decode(&r.p, &a, len.data_ptr<int32_t>(), stream_of(q))
               : dfs_window_attn_decode_i64(&r.p, &a, len.data_ptr<int64_t>(), stream_of(q)),
           "dfs_window_attn_decode");
  return o;
}

// ---------------------------------------------------------------- the dense bias
Tensor relbias_forward(const Tensor& w, const Tensor& lut, int64_t max_distance, int64_t n_q, int64_t n_k,
                       int64_t q_start) {
  require(w.is_cuda(), "deepfold B200 position bias runs on CUDA tensors only (no CPU path)");
  check_bias(w, lut, w.dim() == 2 ? w.size(0) : 0, max_distance, w.device());
  const DeviceSwitch guard(w.device());
  const Tensor wc = w.contiguous();
  Tensor out = at::empty({w.size(0), n_q, n_k}, w.options());
  const dfs_relbias b = bias_of(wc, lut, max_distance);
  check_rc(dfs_relbias_fwd(narrow32(w.size(0), "H"), narrow32(n_q, "n_q"), narrow32(n_k, "n_k"),
                           narrow32(q_start, "q_start"), &b, out.data_ptr(), stream_of(w)),
           "dfs_relbias_fwd");
  return out;
}

struct RelBiasFn : public torch::autograd::Function<RelBiasFn> {
  static Tensor forward(AutogradContext* ctx, Tensor w, Tensor lut, int64_t max_distance, int64_t n_q, int64_t n_k,
                        int64_t q_start) {
    Tensor out = relbias_forward(w, lut, max_distance, n_q, n_k, q_start);
    ctx->save_for_backward({lut});
    ctx->saved_data["max_distance"] = max_distance;
    ctx->saved_data["q_start"] = q_start;
    ctx->saved_data["buckets"] = w.size(1);
    ctx->saved_data["dtype"] = static_cast<int64_t>(w.scalar_type());
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list out(6);
    if (!grads[0].defined()) return out;
    const Tensor lut = ctx->get_saved_variables()[0];
    const DeviceSwitch guard(lut.device());
    const Tensor g = grads[0].to(static_cast<at::ScalarType>(ctx->saved_data["dtype"].toInt())).contiguous();
    const int64_t max_distance = ctx->saved_data["max_distance"].toInt();
    Tensor dw = at::empty({g.size(0), ctx->saved_data["buckets"].toInt()}, g.options());
    dfs_relbias b = bias_of(dw, lut, max_distance);
    const int H = narrow32(g.size(0), "H"), nq = narrow32(g.size(1), "n_q"), nk = narrow32(g.size(2), "n_k");
    const size_t bytes = dfs_relbias_bwd_work(H, nq, nk, &b);
    const Tensor work = at::empty({static_cast<int64_t>(bytes)}, g.options().dtype(at::kByte));
    b.weight = nullptr;
    check_rc(dfs_relbias_bwd(H, nq, nk, narrow32(ctx->saved_data["q_start"].toInt(), "q_start"), &b, g.data_ptr(),
                             dw.data_ptr(), bytes ? work.data_ptr() : nullptr, bytes, stream_of(g)),
             "dfs_relbias_bwd");
    out[0] = dw;
    return once_differentiable(out);
  }
};

Tensor relative_position_bias(Tensor w, Tensor lut, int64_t max_distance, int64_t n_q, int64_t n_k, int64_t q_start) {
  refuse_tangents({w});
  if (at::GradMode::is_enabled() && w.requires_grad())
    return RelBiasFn::apply(w, lut, max_distance, n_q, n_k, q_start);
  return relbias_forward(w, lut, max_distance, n_q, n_k, q_start);
}

// For Python: raises for an error that an attention call on the current device left (wait: any made so far).
void check_status(bool wait) {
  require(!wait || cudaDeviceSynchronize() == cudaSuccess, "cudaDeviceSynchronize failed");
  checked_status(at::Device(at::kCUDA, c10::cuda::current_device()));
}

}  // namespace

void bind_window_attn(pybind11::module_& m) {
  m.def("window_attn", &window_attn, "sliding-window softmax attention with sinks and a bucketed position bias",
        py::arg("Q"), py::arg("K"), py::arg("V"), py::arg("mask"), py::arg("weight"), py::arg("lut"),
        py::arg("max_distance"), py::arg("window"), py::arg("sinks"), py::arg("causal"), py::arg("q_start"),
        py::arg("scale"));
  m.def("window_attn_decode", &window_attn_decode, "the same for one query per sequence over a cache", py::arg("q"),
        py::arg("K"), py::arg("V"), py::arg("lengths"), py::arg("weight"), py::arg("lut"), py::arg("max_distance"),
        py::arg("window"), py::arg("sinks"), py::arg("scale"));
  m.def("window_attn_check_status", &check_status, "raise for a device error of an earlier window attention call",
        py::arg("wait") = true);
  m.def("window_attn_plant_status", [](int code) {
    *status_word(at::Device(at::kCUDA, c10::cuda::current_device())) = code;
  }, "TEST-ONLY: the status that a kernel of the current device would leave", py::arg("code"));
  m.def("relative_position_bias", &relative_position_bias, "(H, n_q, n_k) bias by distance buckets", py::arg("weight"),
        py::arg("lut"), py::arg("max_distance"), py::arg("n_q"), py::arg("n_k"), py::arg("q_start"));
}

}  // namespace dfs_torch
