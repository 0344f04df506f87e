// The model kernels as differentiable functions on torch tensors: they allocate
// results and workspaces from torch's allocator, fill in the argument structures
// and call the C entries on the current stream of the tensors' device. Checking
// what a caller passes is workloads/kernels.py's part.
//
// In C++ because of what a call costs the host: forward and backward of a small
// call take 60 us, of which torch's engine takes 45; the same in Python took 120.

#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/extension.h>

#include <array>
#include <cstring>
#include <memory>
#include <optional>
#include <tuple>
#include <vector>

#include "model_api.h"

namespace {

using at::Tensor;
using sofa_model::AttentionArgs;
using sofa_model::LogprobArgs;
using sofa_model::NormArgs;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

using Optional = std::optional<Tensor>;

void* stream_of(const Tensor& t) {
  return c10::hip::getCurrentHIPStream(t.get_device()).stream();
}

void check(int status, const char* what) {
  if (status < 0) TORCH_CHECK(false, what, " failed: bad argument");
  TORCH_CHECK(status == 0, what, " failed: HIP error ", status);
}

template <typename T = void>
T* ptr(const Tensor& t) {
  return t.defined() ? static_cast<T*>(t.data_ptr()) : nullptr;
}

Tensor unpack(const Optional& t) { return t ? *t : Tensor(); }

int type_of(at::ScalarType t) {
  return t == at::kFloat      ? sofa_model::kFloat32
         : t == at::kBFloat16 ? sofa_model::kBFloat16
                              : sofa_model::kFloat16;
}

// The values in memory are a tensor's own unless it is a lazily negated view.
Tensor dense(const Tensor& t) {
  return t.defined() ? t.resolve_neg().contiguous() : t;
}

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

at::ScalarType known_type(const Tensor& t) {
  const at::ScalarType type = t.scalar_type();
  TORCH_CHECK(type == at::kFloat || type == at::kBFloat16 || type == at::kHalf,
              "the model kernels have no ", type);
  return type;
}

// What a backward pass is given was saved by the forward pass, but hooks on saved
// tensors may return it laid out anew, which every one of them allows for, or as
// something else, which is refused.
void expect(const char* what, const Tensor& t, bool fits, at::ScalarType type,
            const Tensor& like) {
  TORCH_CHECK(t.defined() && fits && t.scalar_type() == type &&
                  t.device() == like.device(),
              what, " came back from a hook as another tensor than it was");
}

// Whether autograd will ask for a backward pass
bool recorded(std::initializer_list<Tensor> tensors) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor& t : tensors)
    if (t.defined() && t.requires_grad()) return true;
  return false;
}

// The gradients as they are, or, where a second derivative may be asked for, such
// that asking for it is an error.
variable_list first_derivatives(variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  variable_list there;
  for (const Tensor& g : grads)
    if (g.defined()) there.push_back(g.detach().requires_grad_());
  auto error = std::make_shared<torch::autograd::DelayedError>(
      "the model kernels have first derivatives only", there.size());
  there = (*error)(std::move(there));
  size_t at = 0;
  for (Tensor& g : grads)
    if (g.defined()) g = there[at++];
  return grads;
}

// ---------------------------------------------------------------- attention

// t, or a copy, with dense rows that start at multiples of 16 bytes and are not
// further apart than the kernels' offsets within a tile reach
Tensor rows16(const Tensor& t) {
  const auto s = t.strides();
  if (s[3] == 1 && s[2] <= sofa_model::kMaxTokenStride &&
      (s[0] | s[1] | s[2]) % 8 == 0 &&
      reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0)
    return t;
  return t.clone(at::MemoryFormat::Contiguous);
}

// (batch, heads, tokens, dim) laid out as (batch, tokens, heads, dim): what the
// projection behind it reads as one matrix without a copy
Tensor token_major(const Tensor& like) {
  const auto s = like.sizes();
  return at::empty_strided(s, {s[2] * s[1] * s[3], s[3], s[1] * s[3], 1},
                           like.options());
}

// t, or a copy, laid out so
Tensor as_token_major(const Tensor& t) {
  const auto s = t.sizes();
  if (t.strides() == at::IntArrayRef{s[2] * s[1] * s[3], s[3], s[1] * s[3], 1} &&
      reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0)
    return t;
  return token_major(t).copy_(t);
}

void put_strides(int64_t (&to)[3], const Tensor& t) {
  for (int i = 0; i < 3; ++i) to[i] = t.stride(i);
}

AttentionArgs attention_args(const Tensor& q, const Tensor& k, const Tensor& v,
                             const Tensor& o, const Tensor& o_low,
                             const Tensor& lse, const Tensor& lengths,
                             double scale, bool causal) {
  AttentionArgs a{};
  a.q = ptr<sofa_model::bf16>(q);
  a.k = ptr<sofa_model::bf16>(k);
  a.v = ptr<sofa_model::bf16>(v);
  a.o = ptr<sofa_model::bf16>(o);
  a.o_low = ptr<sofa_model::bf16>(o_low);
  a.lse = ptr<float>(lse);
  a.lengths = ptr<int>(lengths);
  a.stream = stream_of(q);
  put_strides(a.q_stride, q);
  put_strides(a.k_stride, k);
  put_strides(a.v_stride, v);
  put_strides(a.o_stride, o);
  a.scale = (float) scale;
  a.batch = (int) q.size(0);
  a.heads = (int) q.size(1);
  a.kv_heads = (int) k.size(1);
  a.tokens = (int) q.size(2);
  a.dim = (int) q.size(3);
  a.causal = causal;
  a.key_parts = 1;
  a.device = q.get_device();
  return a;
}

// Workgroups that share the rows behind one block of 128 keys. Two fit a compute
// unit, so 512 fill the card; under a causal mask the blocks differ in work and
// twice as many even it out (8192 tokens, 8 key heads of 128: 1.15 ms with two
// parts, 1.71 with one). Parts cost a pass over their sums, and one of less than
// four steps gains nothing.
int key_parts(int64_t batch, int64_t heads, int64_t kv_heads, int64_t tokens,
              int64_t dim, bool causal) {
  const int64_t groups = batch * kv_heads * ceil_div(tokens, 128);
  const int64_t steps = ceil_div(tokens, dim <= 64 ? 64 : 32) *
                        (heads / kv_heads) / (causal ? 2 : 1);
  const int64_t parts =
      std::min({(int64_t) sofa_model::kMaxKeyParts,
                ceil_div(causal ? 1024 : 512, groups), steps / 4});
  return (int) std::max<int64_t>(1, parts);
}

struct Attention : torch::autograd::Function<Attention> {
  static Tensor forward(AutogradContext* ctx, const Tensor& q_in,
                        const Tensor& k_in, const Tensor& v_in,
                        const Optional& lengths_in, double scale, bool causal) {
    const Tensor lengths = dense(unpack(lengths_in));
    const Tensor q = rows16(q_in), k = rows16(k_in), v = rows16(v_in);
    const Tensor o = token_major(q), o_low = token_major(q);
    const Tensor lse = at::empty({q.size(0), q.size(1), q.size(2)},
                                 q.options().dtype(at::kFloat));
    const AttentionArgs a =
        attention_args(q, k, v, o, o_low, lse, lengths, scale, causal);
    check(sofa_attention_forward(&a), "attention");
    ctx->save_for_backward({q, k, v, o, o_low, lse, lengths});
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["causal"] = causal;
    return o;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    const Tensor& like = grads[0];
    const auto sizes = like.sizes(), kv_sizes = saved[1].sizes();
    expect("attention: q", saved[0], saved[0].sizes() == sizes, at::kBFloat16, like);
    expect("attention: k", saved[1],
           kv_sizes.size() == 4 && kv_sizes[0] == sizes[0] && kv_sizes[1] > 0 &&
               sizes[1] % kv_sizes[1] == 0 && kv_sizes.slice(2) == sizes.slice(2),
           at::kBFloat16, like);
    expect("attention: v", saved[2], saved[2].sizes() == kv_sizes, at::kBFloat16, like);
    for (int i : {3, 4})
      expect("attention: o", saved[i], saved[i].sizes() == sizes, at::kBFloat16, like);
    expect("attention: lse", saved[5], saved[5].sizes() == sizes.slice(0, 3), at::kFloat,
           like);
    if (saved[6].defined())
      expect("attention: lengths", saved[6], saved[6].sizes() == sizes.slice(0, 1),
             at::kInt, like);
    const Tensor q = rows16(saved[0]), k = rows16(saved[1]), v = rows16(saved[2]),
                 o = as_token_major(saved[3]), o_low = as_token_major(saved[4]),
                 lse = dense(saved[5]), lengths = dense(saved[6]);
    const Tensor dout = rows16(grads[0]);
    const Tensor dq = token_major(q), dk = token_major(k), dv = token_major(v);
    const Tensor delta = at::empty_like(lse);
    AttentionArgs a = attention_args(q, k, v, o, o_low, lse, lengths,
                                     ctx->saved_data["scale"].toDouble(),
                                     ctx->saved_data["causal"].toBool());
    a.dout = ptr<sofa_model::bf16>(dout);
    a.delta = ptr<float>(delta);
    a.dq = ptr<sofa_model::bf16>(dq);
    a.dk = ptr<sofa_model::bf16>(dk);
    a.dv = ptr<sofa_model::bf16>(dv);
    put_strides(a.dout_stride, dout);
    put_strides(a.dq_stride, dq);
    put_strides(a.dk_stride, dk);
    put_strides(a.dv_stride, dv);
    a.key_parts = key_parts(a.batch, a.heads, a.kv_heads, a.tokens, a.dim,
                            a.causal);
    Tensor partial;
    if (a.key_parts > 1) {
      partial = at::empty({a.key_parts, 2, k.numel()},
                          q.options().dtype(at::kFloat));
      a.partial = ptr<float>(partial);
    }
    check(sofa_attention_backward(&a), "attention");
    return first_derivatives({dq, dk, dv, {}, {}, {}});
  }
};

Tensor attention(const Tensor& q_in, const Tensor& k_in, const Tensor& v_in,
                 const Optional& lengths_in, double scale, bool causal) {
  if (recorded({q_in, k_in, v_in}))
    return Attention::apply(q_in, k_in, v_in, lengths_in, scale, causal);
  // the arguments hold addresses only: copies live until the launch
  const Tensor lengths = dense(unpack(lengths_in));
  const Tensor q = rows16(q_in), k = rows16(k_in), v = rows16(v_in);
  const Tensor o = token_major(q);
  const AttentionArgs a =
      attention_args(q, k, v, o, {}, {}, lengths, scale, causal);
  check(sofa_attention_forward(&a), "attention");
  return o;
}

// ---------------------------------------------------------------- log probabilities

// Element i of a tensor's first axes is at i / inner * outer_stride +
// i % inner * inner_stride.
struct Split {
  int64_t inner, outer_stride, inner_stride;
};

std::optional<Split> two_level(const Tensor& t, int64_t axes) {
  Split s{1, 0, 0};
  int levels = 0;
  int64_t outer_size = 1;
  for (int64_t i = axes - 1; i >= 0; --i) {
    const int64_t n = t.size(i), stride = t.stride(i);
    if (n == 1) continue;
    if (levels == 0) {
      s.inner = n;
      s.inner_stride = stride;
      levels = 1;
    } else if (levels == 1 && stride == s.inner * s.inner_stride) {
      s.inner *= n;
    } else if (levels == 1) {
      outer_size = n;
      s.outer_stride = stride;
      levels = 2;
    } else if (stride == outer_size * s.outer_stride) {
      outer_size *= n;
    } else {
      return std::nullopt;
    }
  }
  return s;
}

// t, or a copy, and its strides over rows that are split at `inner`
std::tuple<Tensor, int64_t, int64_t> same_split(int64_t inner, int64_t rows,
                                                const Tensor& t, int64_t axes) {
  if (const auto s = t.is_neg() ? std::nullopt : two_level(t, axes)) {
    if (s->inner == inner) return {t, s->outer_stride, s->inner_stride};
    if (s->inner >= rows)  // one level: it can be split anywhere
      return {t, inner * s->inner_stride, s->inner_stride};
  }
  return {dense(t), inner, 1};
}

// A row goes to one workgroup where there are rows for every compute unit, which
// then read all that memory gives; below that it is cut into parts, multiples of
// what a workgroup reads at a time.
std::pair<int, int> vocab_parts(int64_t rows, int64_t vocab) {
  constexpr int64_t kStep = 2048;
  const int64_t most = std::max<int64_t>(
      1, std::min({(int64_t) sofa_model::kMaxVocabParts, ceil_div(256, rows),
                   ceil_div(vocab, kStep)}));
  const int64_t size = ceil_div(vocab, most * kStep) * kStep;
  return {(int) ceil_div(vocab, size), (int) size};
}

// dense rows in two levels
Tensor logit_rows(const Tensor& logits) {
  if (!logits.is_neg() && logits.stride(-1) == 1 &&
      two_level(logits, logits.dim() - 1))
    return logits;
  return dense(logits);
}

LogprobArgs logprob_args(const Tensor& logits, Tensor& tokens, int64_t top,
                         int64_t ignore_index) {
  LogprobArgs a{};
  const int64_t axes = tokens.dim();
  const Split split = *two_level(logits, axes);
  a.rows = tokens.numel();
  a.inner = split.inner;
  a.outer_stride = split.outer_stride;
  a.inner_stride = split.inner_stride;
  std::tie(tokens, a.token_outer_stride, a.token_inner_stride) =
      same_split(a.inner, a.rows, tokens, axes);
  a.logits = ptr(logits);
  a.tokens = ptr<int64_t>(tokens);
  a.ignore_index = ignore_index;
  a.vocab = (int) logits.size(-1);
  a.top = (int) top;
  std::tie(a.parts, a.part_size) = vocab_parts(a.rows, a.vocab);
  a.type = type_of(logits.scalar_type());
  a.device = logits.get_device();
  a.stream = stream_of(logits);
  return a;
}

struct LogprobResults {
  Tensor logprob, entropy, norm, ids, values;
};

LogprobResults logprob_forward(const Tensor& logits, Tensor& tokens, int64_t top,
                               int64_t ignore_index) {
  LogprobArgs a = logprob_args(logits, tokens, top, ignore_index);
  const auto floats = logits.options().dtype(at::kFloat);
  const auto longs = tokens.options();
  LogprobResults r{at::empty(tokens.sizes(), floats),
                   at::empty(tokens.sizes(), floats),
                   at::empty({a.rows, 2}, floats), {}, {}};
  Tensor part_sums, part_top;
  if (top) {
    std::vector<int64_t> shape = tokens.sizes().vec();
    shape.push_back(top);
    r.ids = at::empty(shape, longs);
    r.values = at::empty(shape, floats);
  }
  if (a.parts > 1) {
    part_sums = at::empty({a.rows, a.parts, 3}, floats);
    if (top) part_top = at::empty({a.rows, a.parts, top}, longs);
  }
  a.logprob = ptr<float>(r.logprob);
  a.entropy = ptr<float>(r.entropy);
  a.norm = ptr<float>(r.norm);
  a.top_ids = ptr<int64_t>(r.ids);
  a.top_logprobs = ptr<float>(r.values);
  a.part_sums = ptr<float>(part_sums);
  a.part_top = ptr<uint64_t>(part_top);
  check(sofa_logprob_forward(&a), "token_logprobs");
  return r;
}

struct TokenLogprobs : torch::autograd::Function<TokenLogprobs> {
  static variable_list forward(AutogradContext* ctx, const Tensor& logits_in,
                               const Tensor& tokens_in, int64_t top,
                               int64_t ignore_index) {
    const Tensor logits = logit_rows(logits_in);
    Tensor tokens = tokens_in;
    const LogprobResults r = logprob_forward(logits, tokens, top, ignore_index);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({logits, tokens, r.entropy, r.norm});
    ctx->saved_data["ignore_index"] = ignore_index;
    if (!top) return {r.logprob, r.entropy};
    ctx->mark_non_differentiable({r.ids, r.values});
    return {r.logprob, r.entropy, r.ids, r.values};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    if (!grads[0].defined() && !grads[1].defined()) return variable_list(4);
    const variable_list saved = ctx->get_saved_variables();
    Tensor tokens = saved[1];
    const Tensor& like = grads[0].defined() ? grads[0] : grads[1];
    const auto sizes = like.sizes();
    expect("token_logprobs: logits", saved[0],
           saved[0].dim() == like.dim() + 1 && saved[0].size(-1) > 0 &&
               saved[0].sizes().slice(0, like.dim()) == sizes,
           known_type(saved[0]), like);
    expect("token_logprobs: tokens", tokens, tokens.sizes() == sizes, at::kLong, like);
    expect("token_logprobs: entropy", saved[2], saved[2].sizes() == sizes, at::kFloat,
           like);
    expect("token_logprobs: norm", saved[3],
           saved[3].sizes() == at::IntArrayRef{tokens.numel(), 2}, at::kFloat, like);
    const Tensor logits = logit_rows(saved[0]), entropy = dense(saved[2]),
                 norm = dense(saved[3]);
    LogprobArgs a = logprob_args(logits, tokens, 0,
                                 ctx->saved_data["ignore_index"].toInt());
    const int64_t axes = tokens.dim();
    Tensor g = grads[0], h = grads[1];
    if (g.defined())
      std::tie(g, a.grad_outer_stride, a.grad_inner_stride) =
          same_split(a.inner, a.rows, g, axes);
    if (h.defined())
      std::tie(h, a.grad2_outer_stride, a.grad2_inner_stride) =
          same_split(a.inner, a.rows, h, axes);
    const Tensor dlogits =
        at::empty_like(logits, at::MemoryFormat::Contiguous);
    a.logprob = a.entropy = ptr<float>(entropy);
    a.norm = ptr<float>(norm);
    a.dlogprob = ptr<float>(g);
    a.dentropy = ptr<float>(h);
    a.dlogits = ptr(dlogits);
    check(sofa_logprob_backward(&a), "token_logprobs");
    return first_derivatives({dlogits, {}, {}, {}});
  }
};

std::tuple<Tensor, Tensor, Optional, Optional> token_logprobs(
    const Tensor& logits, const Tensor& tokens, int64_t top,
    int64_t ignore_index) {
  if (recorded({logits})) {
    const variable_list r =
        TokenLogprobs::apply(logits, tokens, top, ignore_index);
    if (!top) return {r[0], r[1], std::nullopt, std::nullopt};
    return {r[0], r[1], r[2], r[3]};
  }
  Tensor ids = tokens;
  const LogprobResults r =
      logprob_forward(logit_rows(logits), ids, top, ignore_index);
  if (!top) return {r.logprob, r.entropy, std::nullopt, std::nullopt};
  return {r.logprob, r.entropy, r.ids, r.values};
}

// ---------------------------------------------------------------- residual norm

// Workgroups of the backward pass that share the rows of one gate. About 512 fill
// the card twice; more would only add partial sums.
int norm_blocks(int64_t rows, int64_t groups, int64_t dim) {
  rows /= groups;
  return (int) std::max<int64_t>(
      1, std::min(512 / groups, dim <= 1024 ? ceil_div(rows, 4) : rows));
}

NormArgs norm_args(const Tensor& x, const Tensor& branch, const Tensor& weight,
                   const Tensor& post, const Tensor& gate, double scale,
                   double eps, at::ScalarType branch_type,
                   at::ScalarType y_type) {
  NormArgs a{};
  a.x = ptr(x);
  a.branch = ptr(branch);
  a.weight = ptr(weight);
  a.post = ptr(post);
  a.gate = ptr(gate);
  a.stream = stream_of(x);
  a.dim = (int) x.size(-1);
  a.rows = x.numel() / a.dim;
  a.group_rows = gate.defined() ? a.rows / (gate.numel() / a.dim) : a.rows;
  a.eps = (float) eps;
  a.scale = (float) scale;
  a.x_type = type_of(x.scalar_type());
  a.branch_type = type_of(branch_type);
  a.y_type = type_of(y_type);
  a.weight_type = type_of(weight.scalar_type());
  if (post.defined()) a.post_type = type_of(post.scalar_type());
  if (gate.defined()) a.gate_type = type_of(gate.scalar_type());
  a.device = x.get_device();
  return a;
}

// (r, y); r is not there without a branch, whose type then only chooses a kernel
std::pair<Tensor, Tensor> norm_forward(const Tensor& x, const Tensor& branch,
                                       const Tensor& weight, const Tensor& post,
                                       const Tensor& gate, double scale,
                                       double eps, at::ScalarType y_type) {
  const Tensor y = at::empty_like(x, x.options().dtype(y_type));
  const Tensor r = branch.defined() ? at::empty_like(x) : Tensor();
  NormArgs a =
      norm_args(x, branch, weight, post, gate, scale, eps,
                branch.defined() ? branch.scalar_type() : y_type, y_type);
  a.r = ptr(r);
  a.y = ptr(y);
  check(sofa_norm_forward(&a), "residual_norm");
  return {r, y};
}

struct ResidualNorm : torch::autograd::Function<ResidualNorm> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x,
                               const Optional& branch_in,
                               const Tensor& weight, const Optional& post_in,
                               const Optional& gate_in, double scale, double eps,
                               at::ScalarType y_type) {
    const Tensor branch = unpack(branch_in), post = unpack(post_in),
                 gate = unpack(gate_in);
    const auto [r, y] =
        norm_forward(x, branch, weight, post, gate, scale, eps, y_type);
    ctx->set_materialize_grads(false);
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["y_type"] = (int64_t) y_type;
    ctx->saved_data["branch_type"] =
        (int64_t) (branch.defined() ? branch.scalar_type() : y_type);
    // which gradients to compute, in the order of the arguments
    int64_t needed = 0, bit = 1;
    for (const Tensor* t : {&x, &branch, &weight, &post, &gate}) {
      if (t->defined() && t->requires_grad()) needed |= bit;
      bit <<= 1;
    }
    ctx->saved_data["needed"] = needed;
    if (!r.defined()) {
      ctx->save_for_backward({x, {}, weight, post, gate});
      return {y};
    }
    // a 32-bit sum is kept, one rounded to 16 bits is computed again
    const bool keep = x.scalar_type() == at::kFloat;
    const bool uses_branch = !keep || post.defined() || gate.defined();
    ctx->save_for_backward(
        {keep ? r : x, uses_branch ? branch : Tensor(), weight, post, gate});
    return {y, r};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const Tensor dy = dense(grads[0]);
    const Tensor dr = grads.size() > 1 ? dense(grads[1]) : Tensor();
    if (!dr.defined() && !dy.defined()) return variable_list(8);
    const variable_list saved = ctx->get_saved_variables();
    const Tensor& like = dy.defined() ? dy : dr;
    const auto branch_type =
        (at::ScalarType) ctx->saved_data["branch_type"].toInt();
    const auto y_type = (at::ScalarType) ctx->saved_data["y_type"].toInt();
    const auto sizes = like.sizes(), dim = sizes.slice(sizes.size() - 1);
    expect("residual_norm: x", saved[0], saved[0].sizes() == sizes,
           dr.defined() ? dr.scalar_type() : known_type(saved[0]), like);
    if (saved[1].defined())
      expect("residual_norm: branch", saved[1], saved[1].sizes() == sizes, branch_type,
             like);
    expect("residual_norm: weight", saved[2], saved[2].sizes() == dim,
           known_type(saved[2]), like);
    if (saved[3].defined())
      expect("residual_norm: post_weight", saved[3], saved[3].sizes() == dim,
             known_type(saved[3]), like);
    if (saved[4].defined())
      expect("residual_norm: gate", saved[4],
             saved[4].dim() > 0 && saved[4].size(-1) == dim[0] &&
                 (saved[4].dim() == 1 || (saved[4].dim() == like.dim() &&
                                          saved[4].size(0) == sizes[0] &&
                                          saved[4].numel() == sizes[0] * dim[0])),
             known_type(saved[4]), like);
    const Tensor x = dense(saved[0]), branch = dense(saved[1]),
                 weight = dense(saved[2]), post = dense(saved[3]),
                 gate = dense(saved[4]);
    NormArgs a = norm_args(x, branch, weight, post, gate,
                           ctx->saved_data["scale"].toDouble(),
                           ctx->saved_data["eps"].toDouble(), branch_type, y_type);
    const int64_t needed = ctx->saved_data["needed"].toInt();
    const Tensor dx = at::empty_like(x);
    Tensor dbranch, dweight, dpost, dgate, partial;
    if (needed & 2) dbranch = at::empty_like(x, x.options().dtype(branch_type));
    if (needed & 4) dweight = at::empty_like(weight);
    if (needed & 8) dpost = at::empty_like(post);
    if (needed & 16) dgate = at::empty_like(gate);
    const int64_t groups = a.rows / a.group_rows;
    a.group_blocks = norm_blocks(a.rows, groups, a.dim);
    const int sums = dweight.defined() + dpost.defined() + dgate.defined();
    if (sums)
      partial = at::empty({sums, groups * a.group_blocks, a.dim},
                          x.options().dtype(at::kFloat));
    a.dr = ptr(dr);
    a.dy = ptr(dy);
    a.dx = ptr(dx);
    a.dbranch = ptr(dbranch);
    a.partial = ptr<float>(partial);
    a.dweight = ptr(dweight);
    a.dpost = ptr(dpost);
    a.dgate = ptr(dgate);
    check(sofa_norm_backward(&a), "residual_norm");
    return first_derivatives(
        {needed & 1 ? dx : Tensor(), dbranch, dweight, dpost, dgate, {}, {}, {}});
  }
};

std::tuple<Tensor, Tensor> residual_norm(const Tensor& x_in,
                                         const Optional& branch_in,
                                         const Tensor& weight_in,
                                         const Optional& post_in,
                                         const Optional& gate_in, double scale,
                                         double eps, at::ScalarType y_type) {
  const Tensor x = dense(x_in), branch = dense(unpack(branch_in)),
               weight = dense(weight_in), post = dense(unpack(post_in)),
               gate = dense(unpack(gate_in));
  if (recorded({x, branch, weight, post, gate})) {
    const auto given = [](const Tensor& t) {
      return t.defined() ? Optional(t) : std::nullopt;
    };
    const variable_list out =
        ResidualNorm::apply(x, given(branch), weight, given(post), given(gate),
                            scale, eps, y_type);
    return {out.size() > 1 ? out[1] : x_in, out[0]};
  }
  const auto [r, y] =
      norm_forward(x, branch, weight, post, gate, scale, eps, y_type);
  return {r.defined() ? r : x_in, y};
}

}  // namespace

PYBIND11_MODULE(sofa_model, m) {
  m.def("attention", &attention);
  m.def("token_logprobs", &token_logprobs);
  m.def("residual_norm", [](const Tensor& x, const Optional& branch,
                            const Tensor& weight, const Optional& post,
                            const Optional& gate, double scale, double eps,
                            const py::object& y_type) {
    return residual_norm(x, branch, weight, post, gate, scale, eps,
                         torch::python::detail::py_object_to_dtype(y_type));
  });
  // the choices of sizes, to be tested
  m.def("key_parts", &key_parts);
  m.def("vocab_parts", &vocab_parts);
  m.def("norm_blocks", &norm_blocks);
  m.def("two_level", [](const Tensor& t, int64_t axes)
                         -> std::optional<std::array<int64_t, 3>> {
    const auto s = two_level(t, axes);
    if (!s) return std::nullopt;
    return std::array<int64_t, 3>{s->inner, s->outer_stride, s->inner_stride};
  });
}
