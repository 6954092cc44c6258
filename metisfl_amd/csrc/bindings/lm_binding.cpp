// torch binding for the language-model training operators: LayerNorm of any
// width (layernorm.hip), log probabilities of given tokens
// (token_logprobs.hip) and AdamW over many tensors (multi_adamw.hip).
// Arguments are checked here before any launch; work goes to the current
// stream of the tensors' device, whichever device is current.
#include <torch/extension.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPException.h>
#include <c10/hip/HIPStream.h>

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

// [rows][cols] with the columns one element apart -> the row stride
int64_t rows_stride(const Tensor& t, const char* nm) {
  TORCH_CHECK(t.is_cuda(), nm, " must be a device tensor");
  TORCH_CHECK(t.dim() == 2, nm, " must have two dimensions");
  TORCH_CHECK(t.size(1) <= 1 || t.stride(1) == 1, nm, " must have its columns one element apart");
  TORCH_CHECK(t.size(0) < std::numeric_limits<int>::max() && t.size(1) < std::numeric_limits<int>::max() - 65536, nm,
              " has too many rows or columns");
  return t.size(0) > 1 ? t.stride(0) : t.size(1);
}

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

std::tuple<Tensor, Tensor, Tensor> layer_norm_fwd(const Tensor& x, const OptTensor& gamma, const OptTensor& beta,
                                                  double eps) {
  const int64_t ldx = rows_stride(x, "x"), M = x.size(0), H = x.size(1);
  c10::DeviceGuard guard(x.device());
  mfl::LayerNormFwd a{};
  a.type = elem_type(x, "x");
  TORCH_CHECK(H > 0, "x has rows of no elements");
  a.param_type = mfl::ELEM_F32;
  if (given(gamma)) a.param_type = param_type(*gamma, x, H, "gamma");
  if (given(beta)) {
    TORCH_CHECK(given(gamma), "beta without gamma");
    TORCH_CHECK(param_type(*beta, x, H, "beta") == a.param_type, "gamma and beta must have the same type");
  }
  Tensor y = torch::empty({M, H}, x.options());
  Tensor mean = torch::empty({M}, x.options().dtype(torch::kFloat32));
  Tensor rstd = torch::empty({M}, x.options().dtype(torch::kFloat32));
  if (M == 0) return {y, mean, rstd};
  a.x = x.data_ptr();
  a.gamma = given(gamma) ? gamma->data_ptr() : nullptr;
  a.beta = given(beta) ? beta->data_ptr() : nullptr;
  a.y = y.data_ptr();
  a.mean = mean.data_ptr<float>();
  a.rstd = rstd.data_ptr<float>();
  a.ldx = ldx;
  a.M = (int)M;
  a.H = (int)H;
  a.eps = (float)eps;
  mfl::launch_layer_norm_fwd(a, stream_of(x));
  C10_HIP_KERNEL_LAUNCH_CHECK();
  return {y, mean, rstd};
}

std::tuple<Tensor, OptTensor, OptTensor> layer_norm_bwd(const Tensor& dy, const Tensor& x, const Tensor& mean,
                                                        const Tensor& rstd, const OptTensor& gamma) {
  const int64_t ldx = rows_stride(x, "x"), lddy = rows_stride(dy, "dy"), M = x.size(0), H = x.size(1);
  c10::DeviceGuard guard(x.device());
  mfl::LayerNormBwd a{};
  a.type = elem_type(x, "x");
  TORCH_CHECK(H > 0, "x has rows of no elements");
  same_device(dy, x, "dy");
  TORCH_CHECK(dy.scalar_type() == x.scalar_type() && dy.sizes() == x.sizes(), "dy must have x's type and shape");
  vector_of(mean, x, torch::kFloat32, M, "mean");
  vector_of(rstd, x, torch::kFloat32, M, "rstd");
  a.param_type = given(gamma) ? param_type(*gamma, x, H, "gamma") : mfl::ELEM_F32;
  Tensor dx = torch::empty({M, H}, x.options());
  OptTensor dgamma, dbeta;
  if (given(gamma)) {
    dgamma = M ? torch::empty({H}, gamma->options()) : torch::zeros({H}, gamma->options());
    dbeta = M ? torch::empty({H}, gamma->options()) : torch::zeros({H}, gamma->options());
  }
  if (M == 0) return {dx, dgamma, dbeta};
  Tensor part;  // the workgroups' partial sums, from the allocator of the current stream (or of a capture)
  a.dy = dy.data_ptr();
  a.x = x.data_ptr();
  a.mean = mean.data_ptr<float>();
  a.rstd = rstd.data_ptr<float>();
  a.dx = dx.data_ptr();
  a.ldx = ldx;
  a.lddy = lddy;
  a.M = (int)M;
  a.H = (int)H;
  if (given(gamma)) {
    const int64_t G = mfl::layer_norm_bwd_blocks((int)M, (int)H, a.type);
    part = torch::empty({G * 2 * H}, x.options().dtype(torch::kFloat32));
    a.part = part.data_ptr<float>();
    a.gamma = gamma->data_ptr();
    a.dgamma = dgamma->data_ptr();
    a.dbeta = dbeta->data_ptr();
  }
  mfl::launch_layer_norm_bwd(a, stream_of(x));
  C10_HIP_KERNEL_LAUNCH_CHECK();
  return {dx, dgamma, dbeta};
}

// targets of any whole type the kernels read
void set_target(const Tensor& target, const Tensor& x, int64_t N, const int64_t*& t64, const int32_t*& t32) {
  same_device(target, x, "targets");
  TORCH_CHECK(target.is_contiguous() && target.numel() == N, "targets must be contiguous, one for each row");
  if (target.scalar_type() == torch::kInt64) t64 = target.data_ptr<int64_t>();
  else if (target.scalar_type() == torch::kInt32) t32 = target.data_ptr<int32_t>();
  else TORCH_CHECK(false, "targets must be int64 or int32, got ", target.scalar_type());
}

std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor> token_logprobs_fwd(const Tensor& x, const Tensor& target,
                                                                      int64_t V, int64_t K) {
  const int64_t ldx = rows_stride(x, "logits"), N = x.size(0);
  c10::DeviceGuard guard(x.device());
  mfl::TokenLogprobs a{};
  a.type = elem_type(x, "logits");
  TORCH_CHECK(V > 0 && V <= x.size(1), "vocab must be between 1 and the logits' ", x.size(1), " columns, got ", V);
  TORCH_CHECK(K >= 0 && K <= mfl::kTopMax && K <= V, "top_k must be between 0 and ", mfl::kTopMax,
              " and at most vocab, got ", K);
  set_target(target, x, N, a.target64, a.target32);
  const auto f32 = x.options().dtype(torch::kFloat32);
  Tensor logp = torch::empty({N}, f32), entropy = torch::empty({N}, f32), stats = torch::empty({N, 3}, f32);
  Tensor top = torch::empty({N, K}, f32), ids = torch::empty({N, K}, x.options().dtype(torch::kInt64));
  if (N == 0) return {logp, entropy, stats, top, ids};
  Tensor work;
  const size_t bytes = mfl::token_logprobs_workspace((int)N, (int)V, (int)K, a.type);
  if (bytes) {
    work = torch::empty({(int64_t)bytes}, x.options().dtype(torch::kUInt8));
    a.work = work.data_ptr();
  }
  a.x = x.data_ptr();
  a.logp = logp.data_ptr<float>();
  a.entropy = entropy.data_ptr<float>();
  a.stats = stats.data_ptr<float>();
  a.top_logp = top.data_ptr<float>();
  a.top_ids = ids.data_ptr<int64_t>();
  a.ldx = ldx;
  a.N = (int)N;
  a.V = (int)V;
  a.K = (int)K;
  mfl::launch_token_logprobs(a, stream_of(x));
  C10_HIP_KERNEL_LAUNCH_CHECK();
  return {logp, entropy, stats, top, ids};
}

Tensor token_logprobs_bwd(const Tensor& x, const Tensor& target, const Tensor& stats, const OptTensor& d_logp,
                          const OptTensor& d_entropy, const OptTensor& d_top, const OptTensor& top_ids,
                          int64_t V) {
  const int64_t ldx = rows_stride(x, "logits"), N = x.size(0), C = x.size(1);
  c10::DeviceGuard guard(x.device());
  mfl::TokenLogprobsBwd a{};
  a.type = elem_type(x, "logits");
  TORCH_CHECK(V > 0 && V <= C, "vocab must be between 1 and the logits' ", C, " columns, got ", V);
  set_target(target, x, N, a.target64, a.target32);
  vector_of(stats, x, torch::kFloat32, 3 * N, "stats");
  if (given(d_logp)) vector_of(*d_logp, x, torch::kFloat32, N, "d_logp");
  if (given(d_entropy)) vector_of(*d_entropy, x, torch::kFloat32, N, "d_entropy");
  if (given(d_top)) {
    TORCH_CHECK(given(top_ids) && d_top->dim() == 2, "d_top needs top_ids and two dimensions");
    a.K = (int)d_top->size(1);
    TORCH_CHECK(d_top->size(1) <= mfl::kTopMax, "d_top has more than ", mfl::kTopMax, " columns");
    vector_of(*d_top, x, torch::kFloat32, N * a.K, "d_top");
    vector_of(*top_ids, x, torch::kInt64, N * a.K, "top_ids");
  }
  Tensor dx = torch::empty({N, C}, x.options());
  if (N == 0) return dx;
  a.x = x.data_ptr();
  a.stats = stats.data_ptr<float>();
  a.d_logp = given(d_logp) ? d_logp->data_ptr<float>() : nullptr;
  a.d_entropy = given(d_entropy) ? d_entropy->data_ptr<float>() : nullptr;
  if (given(d_top) && a.K) {
    a.d_top = d_top->data_ptr<float>();
    a.top_ids = top_ids->data_ptr<int64_t>();
  }
  a.dx = dx.data_ptr();
  a.ldx = ldx;
  a.N = (int)N;
  a.V = (int)V;
  a.C = (int)C;
  mfl::launch_token_logprobs_bwd(a, stream_of(x));
  C10_HIP_KERNEL_LAUNCH_CHECK();
  return dx;
}

// The device side of ops.optim.MultiTensorAdamW: holds the parameters, their
// table and chunk list, and the states' buffers.
class AdamPlan {
 public:
  AdamPlan(std::vector<Tensor> params, std::vector<OptTensor> mirrors, std::vector<double> decay, Tensor m, Tensor v,
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
      t.wd = (float)decay[i];
      t.param_type = p.scalar_type() == torch::kFloat32 ? mfl::ELEM_F32 : mfl::ELEM_BF16;
      total = offsets[i] + (p.numel() + mfl::kAdamBlock - 1) / mfl::kAdamBlock * mfl::kAdamBlock;
      if (i % mfl::kAdamGrads == 0) firsts_.push_back((int64_t)list.size());
      for (int64_t c = 0; c * mfl::kAdamChunk < p.numel(); ++c) list.push_back({(int)i, (int)c});
    }
    firsts_.push_back((int64_t)list.size());
    TORCH_CHECK(list.size() < (size_t)1 << 24, "the parameters have too many elements for one optimizer");
    bits_ = given(m_scale) ? 8 : 32;
    const auto st = bits_ == 8 ? torch::kFloat8_e4m3fn : torch::kFloat32;
    for (const Tensor* t : {&m_, &v_}) {
      same_device(*t, first, "a state");
      TORCH_CHECK(t->scalar_type() == st && t->is_contiguous() && t->numel() == total, "state buffer");
    }
    if (bits_ == 8) {
      TORCH_CHECK(given(v_scale), "8-bit states need both scales");
      vector_of(*m_scale, first, torch::kFloat32, total / mfl::kAdamBlock, "m_scale");
      vector_of(*v_scale, first, torch::kFloat32, total / mfl::kAdamBlock, "v_scale");
      m_scale_ = *m_scale;
      v_scale_ = *v_scale;
    }
    vector_of(step_, first, torch::kInt32, 1, "step");
    if (given(lr_scale)) {
      vector_of(*lr_scale, first, torch::kFloat32, 1, "lr_scale");
      lr_scale_ = *lr_scale;
    }
    auto upload = [&](const void* from, size_t bytes) {
      Tensor host = torch::empty({(int64_t)std::max<size_t>(bytes, 1)}, torch::kUInt8);
      if (bytes) memcpy(host.data_ptr(), from, bytes);
      return host.to(first.device());
    };
    table_ = upload(table.data(), table.size() * sizeof(table[0]));
    chunks_ = upload(list.data(), list.size() * sizeof(mfl::AdamChunk));
    scalars_ = torch::empty({(int64_t)sizeof(mfl::AdamScalars)}, first.options().dtype(torch::kUInt8));
  }

  void step(const std::vector<OptTensor>& grads, double lr, double beta1, double beta2, double eps, int64_t seed) {
    const Tensor& first = params_[0];
    TORCH_CHECK(grads.size() == params_.size(), "got ", grads.size(), " gradients for ", params_.size(), " parameters");
    for (size_t i = 0; i < grads.size(); ++i) {
      if (!given(grads[i])) continue;
      const Tensor& g = *grads[i];
      same_device(g, first, "a gradient");
      elem_type(g, "a gradient");
      TORCH_CHECK(g.is_contiguous() && g.numel() == params_[i].numel(), "gradient ", i,
                  " must be contiguous with its parameter's ", params_[i].numel(), " elements");
    }
    c10::DeviceGuard guard(first.device());
    const hipStream_t s = stream_of(first);
    mfl::AdamStep a{};
    a.tensors = reinterpret_cast<const mfl::AdamTensor*>(table_.data_ptr());
    a.chunks = reinterpret_cast<const mfl::AdamChunk*>(chunks_.data_ptr());
    a.scalars = reinterpret_cast<mfl::AdamScalars*>(scalars_.data_ptr());
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
    a.seed = (uint32_t)seed;
    a.state_bits = bits_;
    mfl::launch_adam_begin(a, s);
    C10_HIP_KERNEL_LAUNCH_CHECK();
    mfl::AdamGrads g;
    for (size_t part = 0; part + 1 < firsts_.size(); ++part) {
      const size_t lo = part * mfl::kAdamGrads, hi = std::min(grads.size(), lo + mfl::kAdamGrads);
      const int64_t n = firsts_[part + 1] - firsts_[part];
      if (n == 0) continue;
      for (size_t i = lo; i < hi; ++i) {
        g.g[i - lo] = given(grads[i]) ? grads[i]->data_ptr() : nullptr;
        g.type[i - lo] = given(grads[i]) ? (uint8_t)elem_type(*grads[i], "a gradient") : 0;
      }
      mfl::launch_adam_chunks(a, g, (int)lo, firsts_[part], n, s);
      C10_HIP_KERNEL_LAUNCH_CHECK();
    }
  }

 private:
  std::vector<Tensor> params_;
  std::vector<OptTensor> mirrors_;
  Tensor m_, v_, m_scale_, v_scale_, step_, lr_scale_, table_, chunks_, scalars_;
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
      .def(pybind11::init<std::vector<Tensor>, std::vector<OptTensor>, std::vector<double>, Tensor, Tensor, OptTensor,
                          OptTensor, Tensor, OptTensor, std::vector<int64_t>>())
      .def("step", &AdamPlan::step);
}
