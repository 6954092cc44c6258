// torch binding for the language-model training operators: LayerNorm of any
// width (layernorm.hip), log probabilities of given tokens
// (token_logprobs.hip) and AdamW over many tensors (multi_adamw.hip).
// Arguments are checked here before any launch; work goes to the current
// stream of the tensors' device, whichever device is current.
#include <torch/extension.h>
#include <ATen/hip/EmptyTensor.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/VirtualGuardImpl.h>
#include <c10/hip/HIPException.h>
#include <c10/hip/HIPStream.h>

#include <cstring>
#include <limits>
#include <vector>

#include "kernels/lm.h"

namespace {

using torch::Tensor;
using OptTensor = c10::optional<Tensor>;

hipStream_t stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

bool given(const OptTensor& t) { return t.has_value() && t->defined(); }

int elem_type(const Tensor& t, const char* nm) {
  switch (t.scalar_type()) {
    case torch::kFloat32: return mfl::ELEM_F32;
    case torch::kBFloat16: return mfl::ELEM_BF16;
    case torch::kFloat16: return mfl::ELEM_F16;
    default: TORCH_CHECK(false, nm, " must be float32, bfloat16 or float16, got ", t.scalar_type());
  }
}

// A tensor of any dimensions as rows of its last one: columns one element
// apart, rows a fixed stride apart (a copy where the strides allow no such view).
struct Rows {
  Tensor keep;
  void* p = nullptr;
  int64_t rows = 1, cols = 0, stride = 0;

  Rows(const Tensor& t, const char* nm) : keep(t) {
    TORCH_CHECK(t.is_cuda(), nm, " must be a device tensor");
    TORCH_CHECK_VALUE(t.dim() > 0, nm, " must have at least one dimension");
    const int64_t d = t.dim();
    cols = t.size(d - 1);
    for (int64_t i = 0; i + 1 < d; ++i) rows *= t.size(i);
    TORCH_CHECK(rows < std::numeric_limits<int>::max() && cols < std::numeric_limits<int>::max() - 65536, nm,
                " has too many rows or columns");
    if (t.is_contiguous()) {
      stride = cols;
    } else if (d == 2 && (t.stride(1) == 1 || cols == 1)) {
      stride = t.stride(0);
    } else {
      if (cols > 1 && t.stride(d - 1) != 1) keep = t.contiguous();
      if (d != 2) keep = keep.reshape({rows, cols});
      stride = keep.dim() == 2 ? keep.stride(0) : cols;
    }
    p = keep.data_ptr();
  }
};

void same_device(const Tensor& t, const Tensor& x, const char* nm) {
  TORCH_CHECK(t.device() == x.device(), nm, " is on ", t.device(), ", expected ", x.device());
}

void vector_of(const Tensor& t, const Tensor& x, torch::ScalarType dt, int64_t n, const char* nm) {
  same_device(t, x, nm);
  TORCH_CHECK(t.scalar_type() == dt, nm, " has dtype ", t.scalar_type(), ", expected ", dt);
  TORCH_CHECK(t.is_contiguous() && t.numel() == n, nm, " must be contiguous with ", n, " elements");
}

int param_type(const Tensor& p, const Tensor& x, int64_t H, const char* nm) {
  const int t = elem_type(p, nm);
  TORCH_CHECK(t == mfl::ELEM_F32 || p.scalar_type() == x.scalar_type(), nm, " must be float32 or of the input's type");
  vector_of(p, x, p.scalar_type(), H, nm);
  return t;
}

// A result or workspace of its own, from the allocator of the current stream
// (or of a capture).  Straight to the device's form: through the dispatcher a
// call of five results on one row is 1.2 us longer (6.6 against 5.3 us).
Tensor fresh(c10::IntArrayRef sizes, const Tensor& x, torch::ScalarType dt) {
  return Tensor(at::detail::empty_cuda(sizes, dt, x.device(), c10::nullopt));
}

c10::IntArrayRef lead_of(const Tensor& t) { return t.sizes().slice(0, t.dim() - 1); }

void norm_weights(const Tensor& x, int64_t H, const OptTensor& gamma, const OptTensor& beta) {
  TORCH_CHECK_VALUE(H > 0, "x has rows of no elements");
  TORCH_CHECK_VALUE(!given(beta) || given(gamma), "beta without gamma");
  for (const auto* p : {&gamma, &beta})
    TORCH_CHECK_VALUE(!given(*p) || ((*p)->dim() == 1 && (*p)->size(0) == H), p == &gamma ? "gamma" : "beta",
                      " has shape ", (*p)->sizes(), ", expected (", H, ")");
}

std::tuple<Tensor, Tensor, Tensor> layer_norm_fwd(const Tensor& x, const OptTensor& gamma, const OptTensor& beta,
                                                  double eps) {
  const Rows r(x, "x");
  norm_weights(x, r.cols, gamma, beta);
  c10::DeviceGuard guard(x.device());
  mfl::LayerNormFwd a{};
  a.type = elem_type(x, "x");
  a.param_type = mfl::ELEM_F32;
  if (given(gamma)) {
    a.param_type = param_type(*gamma, x, r.cols, "gamma");
    a.gamma = gamma->data_ptr();
  }
  if (given(beta)) {
    TORCH_CHECK(param_type(*beta, x, r.cols, "beta") == a.param_type, "gamma and beta must have the same type");
    a.beta = beta->data_ptr();
  }
  Tensor y = fresh(x.sizes(), x, x.scalar_type()), mean = fresh(lead_of(x), x, torch::kFloat32),
         rstd = fresh(lead_of(x), x, torch::kFloat32);
  if (r.rows == 0) return {y, mean, rstd};
  a.x = r.p;
  a.y = y.data_ptr();
  a.mean = mean.data_ptr<float>();
  a.rstd = rstd.data_ptr<float>();
  a.ldx = r.stride;
  a.M = (int)r.rows;
  a.H = (int)r.cols;
  a.eps = (float)eps;
  mfl::launch_layer_norm_fwd(a, stream_of(x));
  C10_HIP_KERNEL_LAUNCH_CHECK();
  return {y, mean, rstd};
}

std::tuple<Tensor, OptTensor, OptTensor> layer_norm_bwd(const Tensor& dy, const Tensor& x, const Tensor& mean,
                                                        const Tensor& rstd, const OptTensor& gamma) {
  TORCH_CHECK_VALUE(dy.sizes() == x.sizes(), "dy has shape ", dy.sizes(), ", expected ", x.sizes());
  const Rows r(x, "x"), d(dy, "dy");
  norm_weights(x, r.cols, gamma, c10::nullopt);
  c10::DeviceGuard guard(x.device());
  mfl::LayerNormBwd a{};
  a.type = elem_type(x, "x");
  same_device(dy, x, "dy");
  TORCH_CHECK(dy.scalar_type() == x.scalar_type(), "dy must have x's type and shape");
  vector_of(mean, x, torch::kFloat32, r.rows, "mean");
  vector_of(rstd, x, torch::kFloat32, r.rows, "rstd");
  a.param_type = given(gamma) ? param_type(*gamma, x, r.cols, "gamma") : mfl::ELEM_F32;
  Tensor dx = fresh(x.sizes(), x, x.scalar_type());
  OptTensor dgamma, dbeta;
  if (given(gamma)) {
    dgamma = fresh({r.cols}, x, gamma->scalar_type());
    dbeta = fresh({r.cols}, x, gamma->scalar_type());
  }
  if (r.rows == 0) {
    if (given(gamma)) {
      dgamma->zero_();
      dbeta->zero_();
    }
    return {dx, dgamma, dbeta};
  }
  Tensor part;  // the workgroups' partial sums, from the allocator of the current stream (or of a capture)
  a.dy = d.p;
  a.x = r.p;
  a.mean = mean.data_ptr<float>();
  a.rstd = rstd.data_ptr<float>();
  a.dx = dx.data_ptr();
  a.ldx = r.stride;
  a.lddy = d.stride;
  a.M = (int)r.rows;
  a.H = (int)r.cols;
  if (given(gamma)) {
    if (const int64_t G = mfl::layer_norm_bwd_parts(a.M, a.H, a.type)) {
      part = fresh({G * 2 * r.cols}, x, torch::kFloat32);
      a.part = part.data_ptr<float>();
    }
    a.gamma = gamma->data_ptr();
    a.dgamma = dgamma->data_ptr();
    a.dbeta = dbeta->data_ptr();
  }
  mfl::launch_layer_norm_bwd(a, stream_of(x));
  C10_HIP_KERNEL_LAUNCH_CHECK();
  return {dx, dgamma, dbeta};
}

// The targets of rows of logits: one whole number each.
struct Targets {
  Tensor keep;
  const int64_t* t64 = nullptr;
  const int32_t* t32 = nullptr;

  Targets(const Tensor& t, const Tensor& x) : keep(t) {
    TORCH_CHECK_VALUE(t.sizes() == lead_of(x), "targets have shape ", t.sizes(), ", expected ", lead_of(x));
    TORCH_CHECK_TYPE(t.scalar_type() == torch::kInt64 || t.scalar_type() == torch::kInt32,
                     "targets must be int64 or int32, got ", t.scalar_type());
    same_device(t, x, "targets");
    if (!t.is_contiguous()) keep = t.contiguous();
    if (t.scalar_type() == torch::kInt64) t64 = keep.data_ptr<int64_t>();
    else t32 = keep.data_ptr<int32_t>();
  }
};

int64_t vocab_of(const Rows& r, const c10::optional<int64_t>& vocab) {
  const int64_t V = vocab.value_or(r.cols);
  TORCH_CHECK_VALUE(V > 0 && V <= r.cols, "vocab must be between 1 and the logits' ", r.cols, " columns, got ", V);
  return V;
}

std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor> token_logprobs_fwd(const Tensor& x, const Tensor& target,
                                                                      int64_t K, c10::optional<int64_t> vocab) {
  const Rows r(x, "logits");
  const int64_t V = vocab_of(r, vocab);
  TORCH_CHECK_VALUE(K >= 0 && K <= mfl::kTopMax && K <= V, "top_k must be between 0 and ", mfl::kTopMax,
                    " and at most vocab, got ", K);
  const Targets t(target, x);
  c10::DeviceGuard guard(x.device());
  mfl::TokenLogprobs a{};
  a.type = elem_type(x, "logits");
  const auto f32 = torch::kFloat32;
  auto shape = lead_of(x).vec();
  Tensor logp = fresh(shape, x, f32), entropy = fresh(shape, x, f32);
  shape.push_back(3);
  Tensor stats = fresh(shape, x, f32);
  shape.back() = K;
  Tensor top = fresh(shape, x, f32), ids = fresh(shape, x, torch::kInt64);
  if (r.rows == 0) return {logp, entropy, top, ids, stats};
  Tensor work;  // parts of split rows, from the allocator of the current stream (or of a capture)
  if (const size_t bytes = mfl::token_logprobs_workspace((int)r.rows, (int)V, (int)K, a.type)) {
    work = fresh({(int64_t)bytes}, x, torch::kUInt8);
    a.work = work.data_ptr();
  }
  a.x = r.p;
  a.target64 = t.t64;
  a.target32 = t.t32;
  a.logp = logp.data_ptr<float>();
  a.entropy = entropy.data_ptr<float>();
  a.stats = stats.data_ptr<float>();
  a.top_logp = top.data_ptr<float>();
  a.top_ids = ids.data_ptr<int64_t>();
  a.ldx = r.stride;
  a.N = (int)r.rows;
  a.V = (int)V;
  a.K = (int)K;
  mfl::launch_token_logprobs(a, stream_of(x));
  C10_HIP_KERNEL_LAUNCH_CHECK();
  return {logp, entropy, top, ids, stats};
}

Tensor token_logprobs_bwd(const Tensor& x, const Tensor& target, const Tensor& stats, const OptTensor& d_logp,
                          const OptTensor& d_entropy, const OptTensor& d_top, const OptTensor& top_ids,
                          c10::optional<int64_t> vocab) {
  const Rows r(x, "logits");
  const int64_t V = vocab_of(r, vocab), N = r.rows;
  const Targets t(target, x);
  const auto lead = lead_of(x);
  auto rows_by = [&](const Tensor& v) { return v.dim() == x.dim() && lead_of(v) == lead; };
  TORCH_CHECK_VALUE(rows_by(stats) && stats.size(-1) == 3, "stats have shape ", stats.sizes(),
                    ", expected the rows' shape and 3");
  for (const auto* d : {&d_logp, &d_entropy})
    TORCH_CHECK_VALUE(!given(*d) || (*d)->sizes() == lead, d == &d_logp ? "d_logp" : "d_entropy", " has shape ",
                      (*d)->sizes(), ", expected ", lead);
  TORCH_CHECK_VALUE(!given(d_top) || (given(top_ids) && rows_by(*d_top) && d_top->sizes() == top_ids->sizes()),
                    "d_top needs top_ids, both with the rows' shape and one column for each alternative");
  c10::DeviceGuard guard(x.device());
  mfl::TokenLogprobsBwd a{};
  a.type = elem_type(x, "logits");
  std::vector<Tensor> keep;  // contiguous copies (the gradient of a sum is an expanded number)
  auto whole = [&](const Tensor& v, torch::ScalarType dt, int64_t n, const char* nm) {
    keep.push_back(v.contiguous());
    vector_of(keep.back(), x, dt, n, nm);
    return keep.back().data_ptr();
  };
  a.stats = static_cast<const float*>(whole(stats, torch::kFloat32, 3 * N, "stats"));
  if (given(d_logp)) a.d_logp = static_cast<const float*>(whole(*d_logp, torch::kFloat32, N, "d_logp"));
  if (given(d_entropy)) a.d_entropy = static_cast<const float*>(whole(*d_entropy, torch::kFloat32, N, "d_entropy"));
  if (given(d_top) && d_top->size(-1)) {
    TORCH_CHECK_VALUE(d_top->size(-1) <= mfl::kTopMax, "d_top has more than ", mfl::kTopMax, " columns");
    a.K = (int)d_top->size(-1);
    a.d_top = static_cast<const float*>(whole(*d_top, torch::kFloat32, N * a.K, "d_top"));
    a.top_ids = static_cast<const int64_t*>(whole(*top_ids, torch::kInt64, N * a.K, "top_ids"));
  }
  Tensor dx = fresh(x.sizes(), x, x.scalar_type());
  if (N == 0) return dx;
  a.x = r.p;
  a.target64 = t.t64;
  a.target32 = t.t32;
  a.dx = dx.data_ptr();
  a.ldx = r.stride;
  a.N = (int)N;
  a.V = (int)V;
  a.C = (int)r.cols;
  mfl::launch_token_logprobs_bwd(a, stream_of(x));
  C10_HIP_KERNEL_LAUNCH_CHECK();
  return dx;
}

// The device side of ops.optim.MultiTensorAdamW: holds the parameters, their
// table and chunk list, and the states' buffers.
class AdamPlan {
 public:
  AdamPlan(std::vector<Tensor> params, std::vector<OptTensor> mirrors, std::vector<bool> decay, Tensor m, Tensor v,
           OptTensor m_scale, OptTensor v_scale, Tensor step, OptTensor lr_scale, std::vector<int64_t> offsets)
      : params_(std::move(params)), mirrors_(std::move(mirrors)), m_(m), v_(v), step_(step) {
    TORCH_CHECK(!params_.empty(), "no parameters");
    TORCH_CHECK(mirrors_.size() == params_.size() && decay.size() == params_.size() && offsets.size() == params_.size(),
                "mirrors, decay and offsets must have one entry for each parameter");
    const Tensor& first = params_[0];
    TORCH_CHECK(first.is_cuda(), "parameters must be device tensors");
    c10::DeviceGuard guard(first.device());
    int64_t total = 0;
    std::vector<mfl::AdamTensor> table(params_.size());
    std::vector<mfl::AdamChunk> list;
    for (size_t i = 0; i < params_.size(); ++i) {
      const Tensor& p = params_[i];
      same_device(p, first, "a parameter");
      TORCH_CHECK(p.scalar_type() == torch::kFloat32 || p.scalar_type() == torch::kBFloat16,
                  "parameters must be float32 or bfloat16, got ", p.scalar_type());
      TORCH_CHECK(p.is_contiguous(), "parameters must be contiguous");
      TORCH_CHECK(p.numel() < (1LL << 41), "a parameter has too many elements");
      TORCH_CHECK(offsets[i] >= total && offsets[i] % mfl::kAdamBlock == 0, "state offsets must grow in whole blocks");
      mfl::AdamTensor& t = table[i];
      t.p = p.data_ptr();
      t.mirror = nullptr;
      if (given(mirrors_[i])) {
        vector_of(*mirrors_[i], first, torch::kBFloat16, p.numel(), "a mirror");
        t.mirror = reinterpret_cast<uint16_t*>(mirrors_[i]->data_ptr());
      }
      t.offset = offsets[i];
      t.numel = p.numel();
      t.decays = decay[i];
      t.param_type = p.scalar_type() == torch::kFloat32 ? mfl::ELEM_F32 : mfl::ELEM_BF16;
      total = offsets[i] + (p.numel() + mfl::kAdamBlock - 1) / mfl::kAdamBlock * mfl::kAdamBlock;
      if (i % mfl::kAdamGrads == 0) firsts_.push_back((int64_t)list.size());
      for (int64_t c = 0; c * mfl::kAdamChunk < p.numel(); ++c) list.push_back({(int)i, (int)c});
    }
    firsts_.push_back((int64_t)list.size());
    TORCH_CHECK(list.size() < (size_t)1 << 24, "the parameters have too many elements for one optimizer");
    total_ = total;
    bits_ = given(m_scale) ? 8 : 32;
    if (bits_ == 8) {
      TORCH_CHECK(given(v_scale), "8-bit states need both scales");
      m_scale_ = *m_scale;
      v_scale_ = *v_scale;
    }
    if (given(lr_scale)) lr_scale_ = *lr_scale;
    check_states();
    for (const Tensor& p : params_) held_.emplace_back(p);
    for (const OptTensor& q : mirrors_) held_.push_back(given(q) ? Held(*q) : Held());
    // one copy: the table, the chunks, and zeros for the scalars and the arrivals
    const size_t tb = table.size() * sizeof(table[0]), cb = list.size() * sizeof(mfl::AdamChunk);
    Tensor host = torch::zeros({(int64_t)(tb + cb + sizeof(mfl::AdamScalars) + sizeof(int))}, torch::kUInt8);
    uint8_t* h = host.data_ptr<uint8_t>();
    memcpy(h, table.data(), tb);
    if (cb) memcpy(h + tb, list.data(), cb);
    chunks_at_ = tb;
    scalars_at_ = tb + cb;
    tables_ = host.to(first.device());
    hold_on_stream();  // their own
  }

  void step(const std::vector<OptTensor>& grads, double lr, double beta1, double beta2, double eps, double wd,
            int64_t seed) {
    const Tensor& first = params_[0];
    TORCH_CHECK(grads.size() == params_.size(), "got ", grads.size(), " gradients for ", params_.size(), " parameters");
    for (size_t i = 0; i < grads.size(); ++i) {
      TORCH_CHECK(held_[i].same(params_[i]), "parameter ", i, " has another storage, size or type than at construction");
      TORCH_CHECK(!given(mirrors_[i]) || held_[grads.size() + i].same(*mirrors_[i]), "mirror ", i,
                  " has another storage, size or type than at construction");
      if (!given(grads[i])) continue;
      const Tensor& g = *grads[i];
      same_device(g, first, "a gradient");
      elem_type(g, "a gradient");
      TORCH_CHECK(g.is_contiguous() && g.numel() == held_[i].numel, "gradient ", i,
                  " must be contiguous with its parameter's ", held_[i].numel, " elements");
    }
    check_states();
    c10::DeviceGuard guard(first.device());
    const hipStream_t s = stream_of(first);
    hold_on_stream();
    mfl::AdamStep a{};
    uint8_t* tables = tables_.data_ptr<uint8_t>();
    a.tensors = reinterpret_cast<const mfl::AdamTensor*>(tables);
    a.chunks = reinterpret_cast<const mfl::AdamChunk*>(tables + chunks_at_);
    a.scalars = reinterpret_cast<mfl::AdamScalars*>(tables + scalars_at_);
    a.arrived = reinterpret_cast<int*>(a.scalars + 1);
    a.step = step_.data_ptr<int>();
    a.lr_scale = lr_scale_.defined() ? lr_scale_.data_ptr<float>() : nullptr;
    a.m = m_.data_ptr();
    a.v = v_.data_ptr();
    if (bits_ == 8) {
      a.m_scale = m_scale_.data_ptr<float>();
      a.v_scale = v_scale_.data_ptr<float>();
    }
    a.beta1 = beta1;
    a.beta2 = beta2;
    a.eps = (float)eps;
    a.lr = (float)lr;
    a.wd = (float)wd;
    a.seed = (uint32_t)seed;
    a.state_bits = bits_;
    const bool whole = firsts_.size() == 2 && firsts_[1] > 0 && firsts_[1] <= mfl::kAdamWhole;
    if (!whole) mfl::launch_adam_begin(a, s);
    C10_HIP_KERNEL_LAUNCH_CHECK();
    for (size_t i = 0; i < grads.size(); ++i)  // autograd learns of the change, as of any in place
      if (given(grads[i]))
        for (const OptTensor& t : {OptTensor(params_[i]), mirrors_[i]})
          if (given(t) && !t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
    mfl::AdamGrads g;
    for (size_t part = 0; part + 1 < firsts_.size(); ++part) {
      const size_t lo = part * mfl::kAdamGrads, hi = std::min(grads.size(), lo + mfl::kAdamGrads);
      const int64_t n = firsts_[part + 1] - firsts_[part];
      if (n == 0) continue;
      for (size_t i = lo; i < hi; ++i) {
        g.g[i - lo] = given(grads[i]) ? grads[i]->data_ptr() : nullptr;
        g.type[i - lo] = given(grads[i]) ? (uint8_t)elem_type(*grads[i], "a gradient") : 0;
      }
      mfl::launch_adam_chunks(a, g, (int)lo, firsts_[part], n, whole, s);
      C10_HIP_KERNEL_LAUNCH_CHECK();
    }
  }

 private:
  // A tensor as the device table has it; a kernel goes by the table, so a step
  // refuses one that is another by then (moved, cut, of another type).
  struct Held {
    void* p = nullptr;
    int64_t numel = 0;
    torch::ScalarType type = torch::kFloat32;
    Held() = default;
    explicit Held(const Tensor& t) : p(t.data_ptr()), numel(t.numel()), type(t.scalar_type()) {}
    bool same(const Tensor& t) const {
      return t.data_ptr() == p && t.numel() == numel && t.scalar_type() == type && t.is_contiguous();
    }
  };

  void check_states() const {
    const Tensor& first = params_[0];
    const auto st = bits_ == 8 ? torch::kFloat8_e4m3fn : torch::kFloat32;
    vector_of(m_, first, st, total_, "state m");
    vector_of(v_, first, st, total_, "state v");
    if (bits_ == 8) {
      vector_of(m_scale_, first, torch::kFloat32, total_ / mfl::kAdamBlock, "m_scale");
      vector_of(v_scale_, first, torch::kFloat32, total_ / mfl::kAdamBlock, "v_scale");
    }
    vector_of(step_, first, torch::kInt32, 1, "step");
    if (lr_scale_.defined()) vector_of(lr_scale_, first, torch::kFloat32, 1, "lr_scale");
  }

  // The allocator reuses what is freed in the order of the stream that
  // allocated it; a step on another stream may still run when the optimizer is
  // dropped.  Nobody else can tell it of the tables.
  void hold_on_stream() {
    const c10::Stream now = c10::impl::VirtualGuardImpl(step_.device().type()).getStream(step_.device());
    for (const c10::Stream& known : streams_)
      if (known == now) return;
    for (const Tensor& t : {tables_, m_, v_, m_scale_, v_scale_, step_})
      if (t.defined() && !streams_.empty()) t.record_stream(now);
    streams_.push_back(now);
  }

  std::vector<Tensor> params_;
  std::vector<OptTensor> mirrors_;
  Tensor m_, v_, m_scale_, v_scale_, step_, lr_scale_, tables_;
  std::vector<Held> held_;       // the parameters, then their mirrors
  int64_t total_ = 0;            // elements of a state's buffer
  std::vector<c10::Stream> streams_;  // that steps ran on, the first the construction's
  size_t chunks_at_ = 0, scalars_at_ = 0;
  std::vector<int64_t> firsts_;  // first chunk of each launch's tensors, and the end
  int bits_ = 32;
};

}  // namespace

void register_lm(pybind11::module& m) {
  m.def("layer_norm_fwd", &layer_norm_fwd);
  m.def("layer_norm_bwd", &layer_norm_bwd);
  m.def("token_logprobs_fwd", &token_logprobs_fwd);
  m.def("token_logprobs_bwd", &token_logprobs_bwd);
  pybind11::class_<AdamPlan>(m, "AdamPlan")
      .def(pybind11::init<std::vector<Tensor>, std::vector<OptTensor>, std::vector<bool>, Tensor, Tensor, OptTensor,
                          OptTensor, Tensor, OptTensor, std::vector<int64_t>>())
      .def("step", &AdamPlan::step);
}
