// PyTorch side of the vocabulary objectives: argument checks, outputs, the current stream.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAException.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/types.h>

#include "objectives.h"

using torch::Tensor;
using OptTensor = c10::optional<Tensor>;

namespace {

using OptDouble = c10::optional<double>;

// Arguments that are wrong by themselves: the Python side turns this error into a ValueError. (What the kernels
// cannot take, a device, strides or a type, stays a RuntimeError.) TORCH_CHECK throws within PyTorch's library.
#define ME_CHECK_VALUE(cond, ...) TORCH_CHECK(cond, "value: ", __VA_ARGS__)

// Numbers go into messages as text: a stream's number formatting would tie this file to the C++ runtime that
// its compiler came with, and PyTorch loads its own.
std::string text(int64_t v) { return std::to_string(v); }
std::string text(double v) {
  char s[32];
  snprintf(s, sizeof s, "%g", v);
  return s;
}
std::string shape(const Tensor& t) {
  std::string s = "[";
  for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
  return s + "]";
}

float check_cap(const OptDouble& cap) {
  const double c = cap.value_or(0.0);
  ME_CHECK_VALUE(c >= 0.0 && c < INFINITY, "softcap: a positive number or None, got ", text(c));
  return (float)c;
}
double check_temperature(double t) {
  ME_CHECK_VALUE(t > 0.0 && t < INFINITY, "temperature: a positive number, got ", text(t));
  return t;
}

me::Logits check_logits(const Tensor& x, const OptDouble& cap, const char* what) {
  TORCH_CHECK(x.is_cuda(), what, ": a CUDA tensor is needed");
  ME_CHECK_VALUE(x.dim() == 2 && x.is_floating_point(), what, ": logits [rows, V] of a floating type are needed, got ",
                    x.scalar_type(), " of shape ", shape(x));
  ME_CHECK_VALUE(x.size(1) > 0 && x.size(1) <= me::kMaxColumns, what, ": a vocabulary of 1 to ", text(me::kMaxColumns),
                    " entries is needed, got ", text(x.size(1)));
  TORCH_CHECK(x.size(0) < (1 << 28), what, ": 2^28 - 1 rows at most, got ", text(x.size(0)));
  TORCH_CHECK(x.size(1) == 1 || x.stride(1) == 1, what, ": a row's logits have to be contiguous");
  me::LogitType type = me::LogitType::kF32;
  if (x.scalar_type() == torch::kBFloat16) type = me::LogitType::kBF16;
  else if (x.scalar_type() == torch::kHalf) type = me::LogitType::kF16;
  else TORCH_CHECK(x.scalar_type() == torch::kFloat32, what, ": bfloat16, float16 or float32 is needed, got ",
                   x.scalar_type());
  return {x.data_ptr(), x.stride(0), x.size(0), x.size(1), type, check_cap(cap)};
}

// One value a row of x, as `type`.
Tensor check_rows(const Tensor& t, const Tensor& x, torch::ScalarType type, const char* what) {
  ME_CHECK_VALUE(t.dim() == 1 && t.size(0) == x.size(0), what, ": one value a row of logits is needed (", text(x.size(0)),
                    "), got shape ", shape(t));
  TORCH_CHECK(t.device() == x.device(), what, ": on another device than the logits");
  return t.scalar_type() == type && t.is_contiguous() ? t : t.to(type).contiguous();
}
// A gradient's coefficient for each row of x, as it comes (autograd's are often one number expanded). `hold` keeps it.
me::RowValues check_coefficients(const Tensor& g, const Tensor& x, Tensor& hold) {
  ME_CHECK_VALUE(g.dim() == 1 && g.size(0) == x.size(0), "coefficients: one value a row of logits is needed (",
                 text(x.size(0)), "), got shape ", shape(g));
  TORCH_CHECK(g.device() == x.device(), "coefficients: on another device than the logits");
  hold = g.scalar_type() == torch::kFloat32 ? g : g.to(torch::kFloat32);
  return {hold.data_ptr<float>(), hold.size(0) > 1 ? hold.stride(0) : 0};
}
Tensor check_whole(const Tensor& t, const Tensor& x, const char* what) {
  ME_CHECK_VALUE(t.scalar_type() == torch::kLong || t.scalar_type() == torch::kInt, what,
                    ": int64 or int32 is needed, got ", t.scalar_type());
  return check_rows(t, x, torch::kLong, what);
}

Tensor gradient_like(const Tensor& x, const OptTensor& out, const char* what) {
  if (!out.has_value()) {
    const auto opts = x.options().requires_grad(false);
    // rows a little apart (a padded vocabulary): the gradient's too, so that both are aligned alike
    if (x.size(0) > 1 && x.stride(0) > x.size(1) && x.stride(0) <= x.size(1) + 64)
      return torch::empty_strided(x.sizes(), {x.stride(0), 1}, opts);
    return torch::empty(x.sizes(), opts);
  }
  const Tensor& o = *out;
  ME_CHECK_VALUE(o.sizes() == x.sizes() && o.scalar_type() == x.scalar_type() && o.device() == x.device(), what,
                    ": out has another shape, type or device than the logits");
  TORCH_CHECK((o.size(1) == 1 || o.stride(1) == 1) && (o.size(0) <= 1 || o.stride(0) >= o.size(1)), what,
              ": out's rows have to be contiguous and apart from one another");
  // The kernels write through the pointer: a graph that has saved these values (an earlier objective's, of the same
  // logits) learns of it by the version.
  o.unsafeGetTensorImpl()->bump_version();
  return o;
}

me::Gradient gradient_of(const Tensor& o) { return {o.data_ptr(), o.stride(0)}; }

struct Teacher {
  Tensor ids, top, lse, weight;
  me::TeacherArgs args;
};

Teacher check_teacher(const Tensor& x, const Tensor& ids, const Tensor& top, const OptTensor& lse,
                      const OptTensor& weight, double temp) {
  ME_CHECK_VALUE(ids.dim() == 2 && ids.sizes() == top.sizes() && ids.size(0) == x.size(0),
                    "teacher_ids and teacher_logits: [rows, k] with the logits' rows is needed, got ", shape(ids), " and ", shape(top));
  ME_CHECK_VALUE(ids.size(1) >= 1 && ids.size(1) <= me::kMaxTop, "teacher_ids: 1 to ", text((int64_t)me::kMaxTop),
                    " entries a row, got ", text(ids.size(1)));
  ME_CHECK_VALUE(ids.scalar_type() == torch::kLong || ids.scalar_type() == torch::kInt,
                    "teacher_ids: int64 or int32 is needed, got ", ids.scalar_type());
  TORCH_CHECK(ids.device() == x.device() && top.device() == x.device(),
              "distill_loss: the teacher's tensors are on another device than the logits");
  check_temperature(temp);
  Teacher t;
  t.ids = ids.to(torch::kLong).contiguous();
  t.top = top.to(torch::kFloat32).contiguous();
  if (lse.has_value()) t.lse = check_rows(*lse, x, torch::kFloat32, "teacher_lse");
  if (weight.has_value()) t.weight = check_rows(*weight, x, torch::kFloat32, "weights");
  t.args = {t.ids.data_ptr<int64_t>(),
            t.top.data_ptr<float>(),
            lse.has_value() ? t.lse.data_ptr<float>() : nullptr,
            weight.has_value() ? t.weight.data_ptr<float>() : nullptr,
            (int)t.ids.size(1),
            (float)temp};
  return t;
}

float2* as2(const Tensor& t) { return reinterpret_cast<float2*>(t.data_ptr<float>()); }
float4* as4(const Tensor& t) { return reinterpret_cast<float4*>(t.data_ptr<float>()); }

}  // namespace

// (logp [N], stats [N, 2])
std::vector<Tensor> token_logprobs_fwd(Tensor x, Tensor target, OptDouble cap) {
  const auto in = check_logits(x, cap, "token_logprobs");
  const at::cuda::CUDAGuard guard(x.device());
  auto t = check_whole(target, x, "targets");
  auto opts = x.options().dtype(torch::kFloat32).requires_grad(false);
  auto logp = torch::empty({in.N}, opts), stats = torch::empty({in.N, 2}, opts);
  if (in.N == 0) return {logp, stats};
  me::launch_logprob_fwd(in, t.data_ptr<int64_t>(), logp.data_ptr<float>(), as2(stats),
                         at::cuda::getCurrentCUDAStream());
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  return {logp, stats};
}

Tensor token_logprobs_bwd(Tensor x, Tensor target, OptDouble cap, Tensor stats, Tensor g, OptTensor out) {
  const auto in = check_logits(x, cap, "token_logprobs");
  const at::cuda::CUDAGuard guard(x.device());
  auto t = check_whole(target, x, "targets");
  Tensor hold;
  const auto gr = check_coefficients(g, x, hold);
  auto o = gradient_like(x, out, "token_logprobs");
  if (in.N == 0) return o;
  me::launch_logprob_bwd(in, t.data_ptr<int64_t>(), as2(stats), gr, gradient_of(o),
                         at::cuda::getCurrentCUDAStream());
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  return o;
}

// (logp [N], gradient of sum(coef * logp) in the logits [N, V]); coef: 1 unless given
std::vector<Tensor> token_logprobs_grad(Tensor x, Tensor target, OptTensor coef, OptDouble cap, OptTensor out) {
  auto t = check_whole(target, x, "targets");
  Tensor g = coef.has_value() ? *coef : torch::ones({1}, x.options().dtype(torch::kFloat32).requires_grad(false)).expand(x.size(0));
  auto f = token_logprobs_fwd(x, t, cap);
  return {f[0], token_logprobs_bwd(x, t, cap, f[1], g, out)};
}

namespace {
// The kernels' view of the teacher's rows: k entries of 4 and one of 8 floats a row.
struct TeacherRows {
  Tensor buffer;
  float* entries;
  float* rows;
};
TeacherRows teacher_rows(const Tensor& x, int64_t k) {
  TeacherRows t;
  t.buffer = torch::empty({x.size(0), k + 2, me::kEntryBytes / 4}, x.options().dtype(torch::kFloat32));
  t.entries = t.buffer.data_ptr<float>();
  t.rows = t.entries + x.size(0) * k * (me::kEntryBytes / 4);
  return t;
}
}  // namespace

// (loss [N], stats [N, 4], the teacher's rows, which distill_bwd takes)
std::vector<Tensor> distill_fwd(Tensor x, Tensor ids, Tensor top, OptTensor lse, OptTensor weight, OptDouble cap,
                                double temp) {
  const auto in = check_logits(x, cap, "distill_loss");
  const at::cuda::CUDAGuard guard(x.device());
  const auto te = check_teacher(x, ids, top, lse, weight, temp);
  auto opts = x.options().dtype(torch::kFloat32).requires_grad(false);
  auto loss = torch::empty({in.N}, opts), stats = torch::empty({in.N, 4}, opts);
  const auto rows = teacher_rows(x, te.args.k);
  if (in.N == 0) return {loss, stats, rows.buffer};
  const auto stream = at::cuda::getCurrentCUDAStream();
  me::launch_teacher(in, te.args, rows.entries, rows.rows, stream);
  me::launch_distill_fwd(in, te.args, rows.entries, rows.rows, loss.data_ptr<float>(), as4(stats), stream);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  return {loss, stats, rows.buffer};
}

Tensor distill_bwd(Tensor x, Tensor rows, OptTensor weight, OptDouble cap, double temp, Tensor stats, Tensor g,
                   OptTensor out) {
  const auto in = check_logits(x, cap, "distill_loss");
  const at::cuda::CUDAGuard guard(x.device());
  Tensor hold;
  const auto gr = check_coefficients(g, x, hold);
  Tensor w;
  if (weight.has_value()) w = check_rows(*weight, x, torch::kFloat32, "weights");
  auto o = gradient_like(x, out, "distill_loss");
  if (in.N == 0) return o;
  me::TeacherArgs te = {};
  te.k = (int)rows.size(1) - 2;
  te.weight = weight.has_value() ? w.data_ptr<float>() : nullptr;
  te.temp = (float)temp;
  const float* entries = rows.data_ptr<float>();
  me::launch_distill_bwd(in, te, entries, entries + in.N * te.k * (me::kEntryBytes / 4), as4(stats),
                         gr, gradient_of(o), at::cuda::getCurrentCUDAStream());
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  return o;
}

// (loss [N], dL/dx [N, V])
std::vector<Tensor> distill_grad(Tensor x, Tensor ids, Tensor top, OptTensor lse, OptTensor weight, OptDouble cap,
                                 double temp, OptTensor out) {
  const auto in = check_logits(x, cap, "distill_loss");
  const at::cuda::CUDAGuard guard(x.device());
  const auto te = check_teacher(x, ids, top, lse, weight, temp);
  auto o = gradient_like(x, out, "distill_loss");
  auto loss = torch::empty({in.N}, x.options().dtype(torch::kFloat32));
  if (in.N == 0) return {loss, o};
  const auto rows = teacher_rows(x, te.args.k);
  const auto stream = at::cuda::getCurrentCUDAStream();
  me::launch_teacher(in, te.args, rows.entries, rows.rows, stream);
  me::launch_distill_grad(in, te.args, rows.entries, rows.rows, loss.data_ptr<float>(), gradient_of(o), stream);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  return {loss, o};
}

// (values [N, k] fp32, ids [N, k] int64, lse [N] fp32)
std::vector<Tensor> top_logits(Tensor x, int64_t k, OptDouble cap, double temp) {
  const auto in = check_logits(x, cap, "top_logits");
  const at::cuda::CUDAGuard guard(x.device());
  const int64_t most = std::min<int64_t>(in.V, me::kMaxTop);
  ME_CHECK_VALUE(k >= 1 && k <= most, "k: 1 to ", text(most), ", got ", text(k));
  check_temperature(temp);
  auto opts = x.options().dtype(torch::kFloat32).requires_grad(false);
  auto values = torch::empty({in.N, k}, opts), lse = torch::empty({in.N}, opts);
  auto ids = torch::empty({in.N, k}, x.options().dtype(torch::kLong));
  if (in.N == 0) return {values, ids, lse};
  me::launch_top_logits(in, (int)k, (float)temp, values.data_ptr<float>(), ids.data_ptr<int64_t>(),
                        lse.data_ptr<float>(), at::cuda::getCurrentCUDAStream());
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  return {values, ids, lse};
}

// (loss [P], rewards [P, 2], scale * d sum(loss) / d logp [T]); scale: 1 / P unless given
std::vector<Tensor> preference_pairs(Tensor logp, OptTensor ref, Tensor cu, int64_t kind, double beta, double smooth,
                                     OptDouble scale, OptTensor target) {
  ME_CHECK_VALUE(logp.dim() == 1 && logp.is_floating_point(), "log-probabilities [tokens] are needed, got ",
                    logp.scalar_type(), " of shape ", shape(logp));
  ME_CHECK_VALUE(cu.dim() == 1 && cu.size(0) % 2 == 1,
                    "cu_seqlens: offsets [2 pairs + 1] of packed sequences (chosen, rejected, chosen, ...) are needed, got shape ",
                    shape(cu));
  ME_CHECK_VALUE(cu.scalar_type() == torch::kInt || cu.scalar_type() == torch::kLong,
                    "cu_seqlens: int64 or int32 is needed, got ", cu.scalar_type());
  TORCH_CHECK(logp.is_cuda() && cu.device() == logp.device(),
              "preference_loss: the log-probabilities and cu_seqlens have to be on one GPU device");
  const at::cuda::CUDAGuard guard(logp.device());
  const int64_t n = logp.size(0), pairs = cu.size(0) / 2;
  TORCH_CHECK(pairs <= INT32_MAX, "preference_loss: 2^31 - 1 pairs at most");
  auto lp = logp.scalar_type() == torch::kFloat32 && logp.is_contiguous() ? logp : logp.to(torch::kFloat32).contiguous();
  Tensor rf, tg;
  if (ref.has_value()) rf = check_rows(*ref, logp, torch::kFloat32, "ref_logps");
  if (target.has_value()) tg = check_rows(*target, logp, torch::kLong, "targets");
  auto off = cu.contiguous();
  auto opts = lp.options().requires_grad(false);
  auto loss = torch::empty({pairs}, opts), rewards = torch::empty({pairs, 2}, opts);
  if (pairs == 0) return {loss, rewards, torch::zeros({n}, opts)};
  auto grad = torch::empty({n}, opts);
  me::launch_preference({lp.data_ptr<float>(), ref.has_value() ? rf.data_ptr<float>() : nullptr,
                         target.has_value() ? tg.data_ptr<int64_t>() : nullptr, off.data_ptr(),
                         off.scalar_type() == torch::kLong, n, pairs, (int)kind, (float)beta, (float)smooth,
                         (float)scale.value_or(1.0 / (double)pairs)},
                        loss.data_ptr<float>(), as2(rewards), grad.data_ptr<float>(),
                        at::cuda::getCurrentCUDAStream());
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  return {loss, rewards, grad};
}

// (loss [P], rewards [P, 2], logp [T], d (scale * sum(loss)) / d logits [T, V])
std::vector<Tensor> preference_logits(Tensor x, Tensor target, OptTensor ref, Tensor cu, int64_t kind, double beta,
                                      double smooth, OptDouble scale, OptDouble cap, OptTensor out) {
  auto t = check_whole(target, x, "targets");
  auto f = token_logprobs_fwd(x, t, cap);
  auto p = preference_pairs(f[0], ref, cu, kind, beta, smooth, scale, t);
  return {p[0], p[1], f[0], token_logprobs_bwd(x, t, cap, f[1], p[2], out)};
}

// ------------------------------------------------------------------------------- autograd
// (in C++: a Python autograd function costs some 60 us a training step, several times a small call's kernels)
namespace {
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// The gradients are not differentiable themselves (create_graph would make a graph without them).
void check_once() {
  TORCH_CHECK(!at::GradMode::is_enabled(), "the gradient of this objective cannot be differentiated (create_graph)");
}

OptTensor optional(const Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); }

struct TokenLogprobs : torch::autograd::Function<TokenLogprobs> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& target, OptDouble cap) {
    auto f = token_logprobs_fwd(x, target, cap);
    ctx->saved_data["cap"] = cap.value_or(0.0);
    ctx->save_for_backward({x, target, f[1]});
    return f[0];
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    check_once();
    const auto s = ctx->get_saved_variables();
    return {token_logprobs_bwd(s[0], s[1], ctx->saved_data["cap"].toDouble(), s[2], g[0], OptTensor()), Tensor(),
            Tensor()};
  }
};

struct Distill : torch::autograd::Function<Distill> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& ids, const Tensor& top,
                        const OptTensor& lse, const OptTensor& weight, OptDouble cap, double temp) {
    auto f = distill_fwd(x, ids, top, lse, weight, cap, temp);
    ctx->saved_data["cap"] = cap.value_or(0.0);
    ctx->saved_data["temp"] = temp;
    ctx->save_for_backward({x, weight.has_value() ? *weight : Tensor(), f[1], f[2]});
    return f[0];
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    check_once();
    const auto s = ctx->get_saved_variables();
    auto dx = distill_bwd(s[0], s[3], optional(s[1]), ctx->saved_data["cap"].toDouble(),
                          ctx->saved_data["temp"].toDouble(), s[2], g[0], OptTensor());
    return {dx, Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};
struct Preference : torch::autograd::Function<Preference> {
  static variable_list forward(AutogradContext* ctx, const Tensor& logp, const OptTensor& ref, const Tensor& cu,
                               int64_t kind, double beta, double smooth) {
    auto p = preference_pairs(logp, ref, cu, kind, beta, smooth, 1.0, OptTensor());
    ctx->saved_data["type"] = logp.scalar_type();
    ctx->save_for_backward({p[2], cu});
    ctx->mark_non_differentiable({p[1]});
    return {p[0], p[1]};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    check_once();
    const auto s = ctx->get_saved_variables();
    const at::cuda::CUDAGuard guard(s[0].device());
    auto gp = g[0].to(torch::kFloat32).contiguous(), out = torch::empty_like(s[0]), off = s[1].contiguous();
    if (out.numel() > 0)
      me::launch_preference_scale(s[0].data_ptr<float>(), gp.data_ptr<float>(), off.data_ptr(),
                                  off.scalar_type() == torch::kLong, s[0].size(0), off.size(0) / 2,
                                  out.data_ptr<float>(), at::cuda::getCurrentCUDAStream());
    C10_CUDA_KERNEL_LAUNCH_CHECK();
    return {out.to(ctx->saved_data["type"].toScalarType()), Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};
}  // namespace

std::vector<Tensor> preference_loss(Tensor logp, OptTensor ref, Tensor cu, int64_t kind, double beta, double smooth) {
  return Preference::apply(logp, ref, cu, kind, beta, smooth);
}

Tensor token_logprobs(Tensor x, Tensor target, OptDouble cap) { return TokenLogprobs::apply(x, target, cap); }

Tensor distill_loss(Tensor x, Tensor ids, Tensor top, OptTensor lse, OptTensor weight, OptDouble cap, double temp) {
  return Distill::apply(x, ids, top, lse, weight, cap, temp);
}
