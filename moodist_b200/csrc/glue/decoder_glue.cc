// Tensor-level entry points of the decoder operators (layer normalisation, rotary positions, distillation loss, gated
// projection): checks of arguments, autograd and the launches on the current stream of the tensors' device. The *_check
// functions are the same checks for CPU tensors, whose arithmetic is in Python.
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/extension.h>

#include <atomic>
#include <cmath>
#include <string>

#include "bindings.h"
#include "kernels/kernels_api.h"

namespace moodist {
namespace {

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptTensor = c10::optional<at::Tensor>;

std::atomic<int64_t> g_launches{0};

void run(int rc, int launches, const char* what) {
  TORCH_CHECK(rc == MB_OK, "moodist ", what, ": ",
              rc == MB_ERR_ALIGN ? "pointers and row pitches must be 16-byte aligned"
              : rc == MB_ERR_ARG ? "unsupported shape"
                                 : "launch failed",
              " (code ", rc, ")");
  g_launches += launches;
}

void* cur_stream() { return c10::cuda::getCurrentCUDAStream().stream(); }

int dtype_code(at::ScalarType t) {
  switch (t) {
    case at::kBFloat16: return MB_BF16;
    case at::kHalf: return MB_F16;
    case at::kFloat: return MB_F32;
    default: return -1;
  }
}

bool wants_grad(const at::Tensor& t) { return t.defined() && t.requires_grad() && at::GradMode::is_enabled(); }

at::Tensor value(const OptTensor& t) { return t.has_value() ? *t : at::Tensor(); }

// What every backward pass asks for. The kernels' backward passes give no graph of their own. And one that is being captured
// must not hand its gradients to a node of the default stream, which cannot join a capture: a leaf keeps its node as long as
// any graph that used it lives, an eager one included, and an engine that finds the wait impossible ends the process.
void backward_check(const char* what, const at::Device& device) {
  TORCH_CHECK(!at::GradMode::is_enabled(), "moodist ", what, ": differentiable once (no create_graph)");
  const auto stream = c10::cuda::getCurrentCUDAStream(device.index()), plain = c10::cuda::getDefaultCUDAStream(device.index());
  const auto node = stream == plain ? nullptr : torch::autograd::get_current_node();
  if (!node) return;
  bool plain_receiver = false;
  for (const auto& edge : node->next_edges())
    if (edge.function) plain_receiver |= edge.function->stream() == std::optional<c10::Stream>(plain.unwrap());
  if (!plain_receiver) return;
  c10::cuda::CUDAGuard guard(device);
  TORCH_CHECK(c10::cuda::currentStreamCaptureStatusMayInitCtx() == c10::cuda::CaptureStatus::None, "moodist ", what,
              ": the gradient of a captured backward pass would go to the default stream. An earlier graph of the same tensors, made "
              "there, is still alive: release its outputs before the capture, or make it on another stream");
}

const void* ptr(const at::Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }

// [rows, D] with contiguous rows, without a copy where the layout allows it
at::Tensor as_rows(const at::Tensor& x) {
  const int64_t D = x.size(-1);
  at::Tensor r = x.dim() == 2 ? x : x.reshape({x.numel() / D, D});
  return r.stride(1) == 1 || D == 1 ? r : r.contiguous();
}

// ---- layer normalisation ------------------------------------------------------------------------------------------------

void layer_norm_check(const at::Tensor& x, const OptTensor& weight, const OptTensor& bias, double eps) {
  TORCH_CHECK(dtype_code(x.scalar_type()) >= 0, "moodist layer_norm: x must be bf16, fp16 or fp32, not ", x.scalar_type());
  TORCH_CHECK(x.dim() >= 1 && x.size(-1) >= 1, "moodist layer_norm: x needs a last dimension of at least 1");
  TORCH_CHECK(x.size(-1) <= (1 << 30), "moodist layer_norm: last dimension too long");
  TORCH_CHECK(eps >= 0, "moodist layer_norm: eps must not be negative");
  for (const OptTensor* o : {&weight, &bias}) {
    if (!o->has_value()) continue;
    const at::Tensor& t = **o;
    TORCH_CHECK(t.dim() == 1 && t.size(0) == x.size(-1), "moodist layer_norm: weight and bias must be [", x.size(-1), "], got ",
                t.sizes());
    TORCH_CHECK(t.scalar_type() == x.scalar_type() || t.scalar_type() == at::kFloat,
                "moodist layer_norm: weight and bias must be of x's type or fp32, got ", t.scalar_type());
    TORCH_CHECK(t.device() == x.device(), "moodist layer_norm: weight and bias must be on x's device");
  }
  TORCH_CHECK(!weight.has_value() || !bias.has_value() || weight->scalar_type() == bias->scalar_type(),
              "moodist layer_norm: weight and bias must be of one type");
}

int weight_code(const at::Tensor& x, const at::Tensor& w, const at::Tensor& b) {
  return dtype_code(w.defined() ? w.scalar_type() : b.defined() ? b.scalar_type() : x.scalar_type());
}

at::Tensor layer_norm_run(const at::Tensor& x2, const at::Tensor& w, const at::Tensor& b, at::IntArrayRef shape, double eps,
                          at::Tensor* stats) {
  const int64_t rows = x2.size(0), D = x2.size(1);
  at::Tensor y = at::empty(shape, x2.options());
  float* mean = nullptr;
  if (stats) {
    *stats = at::empty({2, rows}, x2.options().dtype(at::kFloat));  // means, then 1 / deviations
    mean = stats->data_ptr<float>();
  }
  run(mb_layernorm_fwd(x2.const_data_ptr(), ptr(w), ptr(b), y.data_ptr(), mean, mean ? mean + rows : nullptr, rows, D, x2.stride(0), D,
                       dtype_code(x2.scalar_type()), weight_code(x2, w, b), (float)eps, cur_stream()),
      1, "layer_norm");
  return y;
}

struct LayerNorm : torch::autograd::Function<LayerNorm> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const OptTensor& weight_in, const OptTensor& bias_in,
                            double eps) {
    const at::Tensor weight = value(weight_in), bias = value(bias_in);
    at::Tensor x2 = as_rows(x), stats;
    at::Tensor w = weight.defined() ? weight.contiguous() : weight, b = bias.defined() ? bias.contiguous() : bias;
    at::Tensor y = layer_norm_run(x2, w, b, x.sizes(), eps, &stats);
    ctx->save_for_backward({x2, w, stats});
    ctx->saved_data["wants"] = (int64_t)(x.requires_grad() | (weight.defined() && weight.requires_grad()) << 1 |
                                         (bias.defined() && bias.requires_grad()) << 2 | (weight_code(x, w, b) == MB_F32) << 3);
    return y;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const at::Tensor &x2 = saved[0], &w = saved[1], &stats = saved[2];
    backward_check("layer_norm", x2.device());
    if (!grads[0].defined()) return {at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor()};
    c10::cuda::CUDAGuard guard(x2.device());
    const int64_t rows = x2.size(0), D = x2.size(1), wants = ctx->saved_data["wants"].toInt();
    const int w_code = wants & 8 ? MB_F32 : dtype_code(x2.scalar_type());
    const auto w_options = x2.options().dtype(w_code == MB_F32 ? at::kFloat : x2.scalar_type());
    at::Tensor dy = as_rows(grads[0]), dx, dw, db, partial;
    if (wants & 1) dx = at::empty(grads[0].sizes(), x2.options());
    if (wants & 2) dw = rows ? at::empty({D}, w_options) : at::zeros({D}, w_options);
    if (wants & 4) db = rows ? at::empty({D}, w_options) : at::zeros({D}, w_options);
    if (rows && wants & 6) partial = at::empty({mb_layernorm_bwd_parts(rows, D), 2, D}, x2.options().dtype(at::kFloat));
    const float* mean = stats.data_ptr<float>();
    run(mb_layernorm_bwd(x2.const_data_ptr(), ptr(w), dy.const_data_ptr(), mean, mean + rows, dx.defined() ? dx.data_ptr() : nullptr,
                         dw.defined() ? dw.data_ptr() : nullptr, db.defined() ? db.data_ptr() : nullptr,
                         partial.defined() ? partial.data_ptr<float>() : nullptr, rows, D, x2.stride(0), dy.stride(0), D,
                         dtype_code(x2.scalar_type()), w_code, cur_stream()),
        rows ? 1 + (wants & 6 ? 1 : 0) : 0, "layer_norm backward");
    return {dx, dw, db, at::Tensor()};
  }
};

at::Tensor layer_norm(const at::Tensor& x, const OptTensor& weight, const OptTensor& bias, double eps) {
  TORCH_CHECK(x.is_cuda(), "moodist layer_norm: a CUDA tensor is required");
  layer_norm_check(x, weight, bias, eps);
  c10::cuda::CUDAGuard guard(x.device());
  at::Tensor w = value(weight), b = value(bias);
  if (wants_grad(x) || wants_grad(w) || wants_grad(b)) return LayerNorm::apply(x, weight, bias, eps);
  return layer_norm_run(as_rows(x), w.defined() ? w.contiguous() : w, b.defined() ? b.contiguous() : b, x.sizes(), eps, nullptr);
}

// ---- rotary positions -----------------------------------------------------------------------------------------------------

void rotary_check(const at::Tensor& q, const OptTensor& k, const at::Tensor& cos, const at::Tensor& sin,
                  const OptTensor& positions) {
  TORCH_CHECK(dtype_code(q.scalar_type()) >= 0, "moodist rotary: q must be bf16, fp16 or fp32, not ", q.scalar_type());
  TORCH_CHECK(q.dim() == 3 || q.dim() == 4, "moodist rotary: q must be [batch, tokens, heads, dim] or [tokens, heads, dim], got ",
              q.sizes());
  TORCH_CHECK(q.size(-1) <= (1 << 20) && q.size(-2) <= (1 << 20) && (!k.has_value() || k->dim() < 2 || k->size(-2) <= (1 << 20)),
              "moodist rotary: at most 2^20 heads of 2^20 dimensions");
  if (k.has_value()) {
    TORCH_CHECK(k->dim() == q.dim() && k->size(-1) == q.size(-1) && k->sizes().slice(0, q.dim() - 2) == q.sizes().slice(0, q.dim() - 2),
                "moodist rotary: k must have q's batch, tokens and head dimension, got ", k->sizes(), " for ", q.sizes());
    TORCH_CHECK(k->scalar_type() == q.scalar_type() && k->device() == q.device(), "moodist rotary: k must be of q's type and device");
  }
  TORCH_CHECK(cos.dim() == 2 && sin.sizes() == cos.sizes() && cos.size(0) >= 1 && cos.size(1) >= 1,
              "moodist rotary: cos and sin must be [positions, rotated dimensions / 2], got ", cos.sizes(), " and ", sin.sizes());
  TORCH_CHECK(cos.scalar_type() == at::kFloat && sin.scalar_type() == at::kFloat && cos.is_contiguous() && sin.is_contiguous() &&
                  cos.device() == q.device() && sin.device() == q.device(),
              "moodist rotary: contiguous fp32 tables on q's device required");
  TORCH_CHECK(!cos.requires_grad() && !sin.requires_grad(), "moodist rotary: the tables have no gradient");
  TORCH_CHECK(2 * cos.size(1) <= q.size(-1), "moodist rotary: the tables turn ", 2 * cos.size(1), " dimensions, a head has ",
              q.size(-1));
  const int64_t seq = q.size(-3);
  if (positions.has_value()) {
    const at::Tensor& p = *positions;
    TORCH_CHECK(p.scalar_type() == at::kLong || p.scalar_type() == at::kInt, "moodist rotary: positions must be int64 or int32, not ",
                p.scalar_type());
    TORCH_CHECK(p.device() == q.device(), "moodist rotary: positions must be on q's device");
    const bool per_token = p.dim() == 1 && p.size(0) == seq;
    const bool per_row = q.dim() == 4 && p.dim() == 2 && p.size(0) == q.size(0) && p.size(1) == seq;
    TORCH_CHECK(per_token || per_row, "moodist rotary: positions must be [tokens] or [batch, tokens], got ", p.sizes(), " for ",
                q.sizes());
  } else {
    TORCH_CHECK(seq <= cos.size(0), "moodist rotary: ", seq, " tokens, the tables have ", cos.size(0), " positions");
  }
}

void fill_heads(mb_rotary_heads_t& h, int& heads, const at::Tensor& in, const at::Tensor& out) {
  if (!in.defined()) return;
  const bool b = in.dim() == 4;
  heads = (int)in.size(-2);
  h.in = in.const_data_ptr();
  h.out = out.data_ptr();
  h.in_batch = b ? in.stride(0) : 0;
  h.in_seq = in.stride(-3);
  h.in_head = in.stride(-2);
  h.out_batch = b ? out.stride(0) : 0;
  h.out_seq = out.stride(-3);
  h.out_head = out.stride(-2);
}

at::Tensor dense_last(const at::Tensor& t) { return !t.defined() || t.stride(-1) == 1 || t.size(-1) == 1 ? t : t.contiguous(); }

// one launch for both; either of q and k may be undefined. qo / ko: where the result goes
void rotary_run(const at::Tensor& q, const at::Tensor& k, const at::Tensor& qo, const at::Tensor& ko, const at::Tensor& cos,
                const at::Tensor& sin, const at::Tensor& positions, bool interleaved, bool inverse, bool in_place) {
  const at::Tensor& any = q.defined() ? q : k;
  mb_rotary_t p = {};
  fill_heads(p.q, p.q_heads, q, qo);
  fill_heads(p.k, p.k_heads, k, ko);
  p.batch = any.dim() == 4 ? any.size(0) : 1;
  p.seq = any.size(-3);
  p.dim = (int)any.size(-1);
  p.rot = (int)(2 * cos.size(1));
  p.dtype = dtype_code(any.scalar_type());
  p.interleaved = interleaved;
  p.inverse = inverse;
  p.in_place = in_place;
  p.cos_tab = cos.const_data_ptr<float>();
  p.sin_tab = sin.const_data_ptr<float>();
  p.length = cos.size(0);
  if (positions.defined()) {
    p.positions = positions.const_data_ptr();
    p.pos_batch = positions.dim() == 2 ? positions.stride(0) : 0;
    p.pos_seq = positions.stride(-1);
    p.pos_i64 = positions.scalar_type() == at::kLong;
  }
  run(mb_rotary(&p, cur_stream()), 1, "rotary");
}

struct Rotary : torch::autograd::Function<Rotary> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& q, const OptTensor& k_in, const at::Tensor& cos,
                               const at::Tensor& sin, const OptTensor& positions_in, bool interleaved) {
    const at::Tensor k = value(k_in), positions = value(positions_in);
    at::Tensor qo = at::empty(q.sizes(), q.options()), ko = k.defined() ? at::empty(k.sizes(), k.options()) : at::Tensor();
    rotary_run(dense_last(q), dense_last(k), qo, ko, cos, sin, positions, interleaved, false, false);
    ctx->save_for_backward({cos, sin, positions});
    ctx->saved_data["interleaved"] = interleaved;
    ctx->set_materialize_grads(false);
    return k.defined() ? variable_list{qo, ko} : variable_list{qo};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    backward_check("rotary", saved[0].device());
    at::Tensor gq = dense_last(grads[0]), gk = grads.size() > 1 ? dense_last(grads[1]) : at::Tensor();
    at::Tensor dq, dk;
    if (gq.defined()) dq = at::empty(gq.sizes(), gq.options());
    if (gk.defined()) dk = at::empty(gk.sizes(), gk.options());
    if (gq.defined() || gk.defined()) {
      c10::cuda::CUDAGuard guard(saved[0].device());
      rotary_run(gq, gk, dq, dk, saved[0], saved[1], saved[2], ctx->saved_data["interleaved"].toBool(), true, false);
    }
    return {dq, dk, at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor()};
  }
};

std::tuple<at::Tensor, OptTensor> rotary(const at::Tensor& q, const OptTensor& k, const at::Tensor& cos, const at::Tensor& sin,
                                         const OptTensor& positions, bool interleaved) {
  TORCH_CHECK(q.is_cuda(), "moodist rotary: CUDA tensors are required");
  rotary_check(q, k, cos, sin, positions);
  c10::cuda::CUDAGuard guard(q.device());
  at::Tensor kt = value(k), pt = value(positions);
  if (wants_grad(q) || wants_grad(kt)) {
    auto out = Rotary::apply(q, k, cos, sin, positions, interleaved);
    return {out[0], out.size() > 1 ? OptTensor(out[1]) : OptTensor()};
  }
  at::Tensor qo = at::empty(q.sizes(), q.options()), ko = kt.defined() ? at::empty(kt.sizes(), kt.options()) : at::Tensor();
  rotary_run(dense_last(q), dense_last(kt), qo, ko, cos, sin, pt, interleaved, false, false);
  return {qo, kt.defined() ? OptTensor(ko) : OptTensor()};
}

void rotary_in_place_check(const at::Tensor& q, const OptTensor& k) {
  TORCH_CHECK(!k.has_value() || q.numel() == 0 || k->numel() == 0 || q.const_data_ptr() != k->const_data_ptr(),
              "moodist rotary_: q and k are the same memory");
  for (const at::Tensor& t : {q, value(k)}) {
    if (!t.defined()) continue;
    TORCH_CHECK(!wants_grad(t), "moodist rotary_: no gradient passes through the in-place form, use rotary");
    TORCH_CHECK(t.numel() == 0 || t.stride(-1) == 1, "moodist rotary_: contiguous head dimensions required");
    for (int64_t i = 0; i < t.dim(); ++i)
      TORCH_CHECK(t.size(i) <= 1 || t.stride(i) != 0, "moodist rotary_: an expanded tensor cannot be written in place");
  }
}

void rotary_(at::Tensor q, const OptTensor& k, const at::Tensor& cos, const at::Tensor& sin, const OptTensor& positions,
             bool interleaved) {
  TORCH_CHECK(q.is_cuda(), "moodist rotary_: CUDA tensors are required");
  rotary_check(q, k, cos, sin, positions);
  rotary_in_place_check(q, k);
  c10::cuda::CUDAGuard guard(q.device());
  at::Tensor kt = value(k);
  q.unsafeGetTensorImpl()->bump_version();
  if (kt.defined()) kt.unsafeGetTensorImpl()->bump_version();
  rotary_run(q, kt, q, kt, cos, sin, value(positions), interleaved, false, true);
}

// ---- distillation loss ------------------------------------------------------------------------------------------------------

void distill_check(const at::Tensor& logits, const at::Tensor& ids, const at::Tensor& top, const OptTensor& targets, double tau,
                   double hard) {
  TORCH_CHECK(dtype_code(logits.scalar_type()) >= 0, "moodist distill_loss: logits must be bf16, fp16 or fp32, not ",
              logits.scalar_type());
  TORCH_CHECK(logits.dim() >= 1 && logits.size(-1) >= 1 && logits.size(-1) <= (1 << 30),
              "moodist distill_loss: logits need a vocabulary of 1 to 2^30 words, got ", logits.sizes());
  TORCH_CHECK(ids.sizes() == top.sizes() && ids.dim() == logits.dim() && ids.size(-1) >= 1 && ids.size(-1) <= (1 << 30) &&
                  ids.sizes().slice(0, ids.dim() - 1) == logits.sizes().slice(0, logits.dim() - 1),
              "moodist distill_loss: teacher ids and logits must be [..., entries] over the rows of logits, got ", ids.sizes(), " and ",
              top.sizes(), " for ", logits.sizes());
  TORCH_CHECK(ids.scalar_type() == at::kLong || ids.scalar_type() == at::kInt, "moodist distill_loss: ids must be int64 or int32, not ",
              ids.scalar_type());
  TORCH_CHECK(dtype_code(top.scalar_type()) >= 0, "moodist distill_loss: teacher logits must be bf16, fp16 or fp32, not ",
              top.scalar_type());
  TORCH_CHECK(!top.requires_grad(), "moodist distill_loss: the teacher has no gradient (detach its logits)");
  TORCH_CHECK(ids.device() == logits.device() && top.device() == logits.device(), "moodist distill_loss: tensors on one device required");
  TORCH_CHECK((float)tau > 0 && std::isfinite((float)tau) && std::isfinite(1 / (float)tau),
              "moodist distill_loss: temperature must be positive, and it and its inverse finite in fp32");
  TORCH_CHECK(hard >= 0 && hard <= 1, "moodist distill_loss: hard_weight must be in [0, 1]");
  TORCH_CHECK(hard == 0 || targets.has_value(), "moodist distill_loss: hard_weight needs targets");
  if (targets.has_value()) {
    TORCH_CHECK(targets->scalar_type() == at::kLong && targets->sizes() == logits.sizes().slice(0, logits.dim() - 1) &&
                    targets->device() == logits.device(),
                "moodist distill_loss: targets must be int64, one for each row of logits");
  }
}

mb_distill_t distill_args(const at::Tensor& z, const at::Tensor& ids, const at::Tensor& top, const at::Tensor& targets, double tau,
                          double hard, int64_t ignore_index, bool mean, double scale, const at::Tensor& work) {
  const int64_t rows = z.size(0), K = ids.size(1);
  mb_distill_t d = {};
  d.logits = z.const_data_ptr();
  d.rows = rows;
  d.stride = z.stride(0);
  d.V = (int)z.size(1);
  d.K = (int)K;
  d.dtype = dtype_code(z.scalar_type());
  d.top_dtype = dtype_code(top.scalar_type());
  d.ids_i64 = ids.scalar_type() == at::kLong;
  d.ids = ids.const_data_ptr();
  d.top = top.const_data_ptr();
  d.targets = targets.defined() ? targets.const_data_ptr<int64_t>() : nullptr;
  d.ignore_index = ignore_index;
  d.tau = (float)tau;
  d.hard = (float)hard;
  d.scale = (float)scale;
  d.mean = mean;
  // one workspace: MB_DISTILL_COUNTS counts, [rows] entropy, [rows, 3] stats, [rows] row losses, [rows] live, [rows, K] p
  float* w = work.data_ptr<float>();
  d.counts = reinterpret_cast<int*>(w);
  d.entropy = w + MB_DISTILL_COUNTS;
  d.stats = d.entropy + rows;
  d.row_loss = d.stats + 3 * rows;
  d.live = reinterpret_cast<int*>(d.row_loss + rows);
  d.p = d.row_loss + 2 * rows;
  return d;
}

struct Distill : torch::autograd::Function<Distill> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& logits, const at::Tensor& ids_in, const at::Tensor& top_in,
                            const OptTensor& targets_opt, double tau, double hard, int64_t ignore_index, bool mean, double scale) {
    const at::Tensor targets_in = value(targets_opt);
    const int64_t rows = logits.numel() / logits.size(-1), K = ids_in.size(-1);
    if (!rows) {
      if (ctx) ctx->saved_data["grad"] = at::empty(logits.sizes(), logits.options());
      return at::zeros({}, logits.options().dtype(at::kFloat));
    }
    at::Tensor z = as_rows(logits);
    at::Tensor ids = ids_in.reshape({rows, K}).contiguous(), top = top_in.reshape({rows, K}).contiguous();
    at::Tensor targets = targets_in.defined() ? targets_in.reshape({rows}).contiguous() : targets_in;
    at::Tensor work = at::empty({MB_DISTILL_COUNTS + rows * (6 + K)}, z.options().dtype(at::kFloat));
    at::Tensor loss = at::empty({}, z.options().dtype(at::kFloat)), dz;
    mb_distill_t d = distill_args(z, ids, top, targets, tau, hard, ignore_index, mean, scale, work);
    d.loss = loss.data_ptr<float>();
    // fp16 gradients wait for the incoming scale, which keeps them from underflowing
    const bool now = ctx && logits.scalar_type() != at::kHalf;
    if (now) dz = at::empty(logits.sizes(), logits.options());
    run(mb_distill_fwd(&d, now ? dz.data_ptr() : nullptr, d.V, cur_stream()), 2, "distill_loss");
    if (now) {
      ctx->saved_data["grad"] = dz;
    } else if (ctx) {
      ctx->save_for_backward({z, ids, top, targets, work});
      ctx->saved_data["shape"] = logits.sizes();
      ctx->saved_data["tau"] = tau;
      ctx->saved_data["hard"] = hard;
      ctx->saved_data["ignore"] = ignore_index;
      ctx->saved_data["mean"] = mean;
      ctx->saved_data["scale"] = scale;
    }
    return loss;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list out(9);
    if (!grads[0].defined()) return out;
    backward_check("distill_loss", grads[0].device());
    auto& a = ctx->saved_data;
    at::Tensor g = grads[0].contiguous();
    if (a.count("grad")) {
      // the forward pass made the gradient; it is given away, and only scaled if the loss was
      TORCH_CHECK(a["grad"].isTensor(), "moodist distill_loss: the gradient of this call has been taken already (a second backward pass "
                  "through it needs a second forward pass)");
      at::Tensor dz = a["grad"].toTensor();
      a["grad"] = c10::IValue();
      c10::cuda::CUDAGuard guard(dz.device());
      run(mb_scale_by(dz.data_ptr(), dz.numel(), dtype_code(dz.scalar_type()), g.data_ptr<float>(), cur_stream()), 1,
          "distill_loss backward");
      out[0] = dz;
      return out;
    }
    const auto s = ctx->get_saved_variables();
    c10::cuda::CUDAGuard guard(s[0].device());
    mb_distill_t d = distill_args(s[0], s[1], s[2], s[3], a["tau"].toDouble(), a["hard"].toDouble(), a["ignore"].toInt(),
                                  a["mean"].toBool(), a["scale"].toDouble(), s[4]);
    at::Tensor dz = at::empty(a["shape"].toIntVector(), s[0].options());
    run(mb_distill_bwd(&d, g.data_ptr<float>(), dz.data_ptr(), d.V, cur_stream()), 1, "distill_loss backward");
    out[0] = dz;
    return out;
  }
};

at::Tensor distill_loss(const at::Tensor& logits, const at::Tensor& ids, const at::Tensor& top, const OptTensor& targets, double tau,
                        double hard, int64_t ignore_index, bool mean, double scale) {
  TORCH_CHECK(logits.is_cuda(), "moodist distill_loss: CUDA tensors are required");
  distill_check(logits, ids, top, targets, tau, hard);
  c10::cuda::CUDAGuard guard(logits.device());
  if (wants_grad(logits)) return Distill::apply(logits, ids, top, targets, tau, hard, ignore_index, mean, scale);
  return Distill::forward(nullptr, logits, ids, top, targets, tau, hard, ignore_index, mean, scale);
}

// ---- gated projection -------------------------------------------------------------------------------------------------------

int act_code(const std::string& name) {
  const int act = name == "silu" ? 0 : name == "gelu" ? 1 : name == "gelu_tanh" ? 2 : -1;
  TORCH_CHECK(act >= 0, "moodist gated_linear: activation must be 'silu', 'gelu' or 'gelu_tanh', not '", name, "'");
  return act;
}

void gated_check(const at::Tensor& x, const at::Tensor& w, const std::string& activation) {
  act_code(activation);
  TORCH_CHECK(x.scalar_type() == at::kBFloat16 && w.scalar_type() == at::kBFloat16, "moodist gated_linear: bf16 tensors required, got ",
              x.scalar_type(), " and ", w.scalar_type());
  TORCH_CHECK(x.dim() >= 1 && w.dim() == 2 && w.size(1) == x.size(-1) && w.size(0) >= 2 && w.size(0) % 2 == 0,
              "moodist gated_linear: the weight must be [2 * features, ", x.dim() ? x.size(-1) : 0, "], gate rows first, got ", w.sizes());
  TORCH_CHECK(w.size(0) % 16 == 0 && w.size(1) % 8 == 0 && w.size(1) > 0,
              "moodist gated_linear: features and inputs must be multiples of 8, got a weight of ", w.sizes());
  TORCH_CHECK(w.numel() < (1ll << 40) && w.size(0) <= (1 << 30) && w.size(1) <= (1 << 30) && x.numel() / x.size(-1) <= (1 << 30),
              "moodist gated_linear: at most 2^30 rows, inputs and rows of weight, got ", x.sizes(), " and ", w.sizes());
  TORCH_CHECK(x.device() == w.device(), "moodist gated_linear: tensors on one device required");
}

// rows that the tensor-memory copies can take: contiguous, 16-byte aligned start and pitch
at::Tensor as_tiles(const at::Tensor& t) {
  at::Tensor r = as_rows(t);
  const bool fits = r.stride(1) == 1 && (r.size(0) <= 1 || r.stride(0) % 8 == 0) &&
                    (reinterpret_cast<uintptr_t>(r.const_data_ptr()) & 15) == 0 && (r.size(0) <= 1 || r.stride(0) >= r.size(1));
  return fits ? r : r.contiguous().data_ptr() == r.const_data_ptr() ? r.clone(at::MemoryFormat::Contiguous) : r.contiguous();
}
int64_t pitch(const at::Tensor& t) { return t.size(0) <= 1 ? t.size(1) : t.stride(0); }

// gu, scales: where the projections are kept for the backward pass, or null
at::Tensor gated_run(const at::Tensor& x2, const at::Tensor& w2, at::IntArrayRef shape, int act, at::Tensor* gu, at::Tensor* scales) {
  const int64_t T = x2.size(0), K = x2.size(1), F = w2.size(0) / 2;
  at::Tensor h = at::empty(shape, x2.options());
  if (gu) {
    *gu = at::empty({T, 2 * F}, x2.options().dtype(at::kHalf));
    *scales = at::empty({T, 2 * (int64_t)mb_gated_scale_pitch((int)F)}, x2.options().dtype(at::kByte));
  }
  const int dev = x2.get_device();
  check_kernel_status(dev);
  run(mb_gated_fwd_bf16(x2.const_data_ptr(), w2.const_data_ptr(), h.data_ptr(), gu ? gu->data_ptr() : nullptr,
                        gu ? scales->data_ptr() : nullptr, T, (int)F, (int)K, pitch(x2), pitch(w2), F, act, kernel_status(dev), 0, cur_stream()),
      1, "gated_linear");
  return h;
}

std::vector<int64_t> gated_shape(const at::Tensor& x, const at::Tensor& w) {
  std::vector<int64_t> shape = x.sizes().vec();
  shape.back() = w.size(0) / 2;
  return shape;
}

struct Gated : torch::autograd::Function<Gated> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& w, int64_t act) {
    at::Tensor x2 = as_tiles(x), w2 = as_tiles(w), gu, scales;
    at::Tensor h = gated_run(x2, w2, gated_shape(x, w), (int)act, &gu, &scales);
    ctx->save_for_backward({x2, w2, gu, scales});
    ctx->saved_data["act"] = act;
    ctx->saved_data["wants"] = (int64_t)(x.requires_grad() | w.requires_grad() << 1);
    return h;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    if (!grads[0].defined()) return {at::Tensor(), at::Tensor(), at::Tensor()};
    backward_check("gated_linear", grads[0].device());
    const auto saved = ctx->get_saved_variables();
    const at::Tensor &x2 = saved[0], &w2 = saved[1], &gu = saved[2], &scales = saved[3];
    c10::cuda::CUDAGuard guard(x2.device());
    const int64_t T = x2.size(0), K = x2.size(1), F = w2.size(0) / 2;
    const int64_t wants = ctx->saved_data["wants"].toInt();
    std::vector<int64_t> shape = grads[0].sizes().vec();
    shape.back() = K;
    at::Tensor dh = as_tiles(grads[0]), dgu = at::empty({T, 2 * F}, x2.options()), dx, dw;
    if (wants & 1) dx = at::empty(shape, x2.options());
    if (wants & 2) dw = T ? at::empty({2 * F, K}, x2.options()) : at::zeros({2 * F, K}, x2.options());
    if (T) {
      const int dev = x2.get_device();
      uint32_t* status = kernel_status(dev);
      check_kernel_status(dev);
      run(mb_gated_bwd_bf16(gu.const_data_ptr(), scales.const_data_ptr(), dh.const_data_ptr(), dgu.data_ptr(), T, (int)F, pitch(dh),
                            (int)ctx->saved_data["act"].toInt(), cur_stream()),
          1, "gated_linear backward");
      // dx[T, K] = dgu[T, 2F] w[2F, K], dw[2F, K] = dgu^T x: the transposed operands are read as they lie
      if (dx.defined())
        run(mb_gated_dx_bf16(dgu.const_data_ptr(), w2.const_data_ptr(), dx.data_ptr(), T, (int)F, (int)K, 2 * F, pitch(w2), K, status, 0,
                             cur_stream()),
            1, "gated_linear backward");
      if (dw.defined())
        run(mb_gemm_bf16(dgu.const_data_ptr(), x2.const_data_ptr(), dw.data_ptr(), (int)(2 * F), (int)K, (int)T, 2 * F, pitch(x2), K, 1, 1,
                         0, 0, status, 0, cur_stream()),
            1, "gated_linear backward");
    }
    return {dx, dw, at::Tensor()};
  }
};

at::Tensor gated_linear(const at::Tensor& x, const at::Tensor& w, const std::string& activation) {
  TORCH_CHECK(x.is_cuda(), "moodist gated_linear: CUDA tensors are required");
  gated_check(x, w, activation);
  c10::cuda::CUDAGuard guard(x.device());
  const int act = act_code(activation);
  if (wants_grad(x) || wants_grad(w)) return Gated::apply(x, w, (int64_t)act);
  return gated_run(as_tiles(x), as_tiles(w), gated_shape(x, w), act, nullptr, nullptr);
}

}  // namespace

void bind_decoder_ops(pybind11::module_& m) {
  namespace py = pybind11;
  m.def("decoder_op_launches", [] { return g_launches.load(); });
  m.def("layer_norm", &layer_norm);
  m.def("layer_norm_check", &layer_norm_check);
  m.def("rotary", &rotary);
  m.def("rotary_", &rotary_);
  m.def("rotary_check", &rotary_check);
  m.def("rotary_in_place_check", &rotary_in_place_check);
  m.def("distill_loss", &distill_loss);
  m.def("distill_check", &distill_check);
  m.def("gated_linear", &gated_linear);
  m.def("gated_check", &gated_check);
}

}  // namespace moodist
