// The model kernels as operators of torch's dispatcher: they allocate results and
// workspaces from torch's allocator, fill in the argument structures and call the
// C entries on the current stream of the tensors' device. Being known to the
// dispatcher is what lets tracers record them, and fake tensors pass through.
//
// Each has a kernel (CUDA: what it computes; Meta: the shapes alone, the same
// function up to the launch) and, where it is differentiable, an Autograd kernel,
// which calls operators of its own for what a backward pass needs. Kernels check
// what they could read or write out of bounds; telling a caller what is wrong is
// workloads/kernels.py's part.
//
// In C++ because of what a call costs the host: forward and backward of a small
// call take 60 us, of which torch's engine takes 45; the same in Python took 120.

#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/extension.h>
#include <torch/library.h>

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
using Below = at::AutoDispatchBelowADInplaceOrView;

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
Optional given(const Tensor& t) { return t.defined() ? Optional(t) : std::nullopt; }

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

at::ScalarType known(at::ScalarType type) {
  TORCH_CHECK(type == at::kFloat || type == at::kBFloat16 || type == at::kHalf,
              "the model kernels have no ", type);
  return type;
}

at::ScalarType known_type(const Tensor& t) { return known(t.scalar_type()); }

// `fits`: the sizes do. Backward passes check as well: hooks on saved tensors may
// return them laid out anew, which every kernel allows for, or as something else.
void expect(const char* what, const Tensor& t, bool fits, at::ScalarType type,
            const Tensor& like) {
  TORCH_CHECK(t.defined() && fits && t.scalar_type() == type &&
                  t.device() == like.device(),
              what, " does not belong to the other tensors");
}

// The operator whose kernel is F
template <auto* F>
const auto& op(const char* name) {
  static const auto handle =
      c10::Dispatcher::singleton()
          .findSchemaOrThrow(name, "")
          .typed<std::remove_pointer_t<decltype(F)>>();
  return handle;
}

// Whether autograd will ask for a backward pass. Derivatives that are carried
// forward are refused here: a result without one would read as not depending on
// the input.
bool recorded(std::initializer_list<Tensor> tensors) {
  for (const Tensor& t : tensors)
    TORCH_CHECK(!t.defined() || !t._fw_grad(0).defined(),
                "the model kernels have no forward-mode derivatives");
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

// t, or a copy, with dense rows that start at multiples of 16 bytes of its memory
// and are not further apart than the kernels' offsets within a tile reach
Tensor rows16(const Tensor& t) {
  const auto s = t.strides();
  if (s[3] == 1 && s[2] <= sofa_model::kMaxTokenStride &&
      (s[0] | s[1] | s[2] | t.storage_offset()) % 8 == 0)
    return t;
  return t.clone(at::MemoryFormat::Contiguous);
}

bool at16(const Tensor& t) {
  return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
}

// The same, and that memory too
Tensor aligned(const Tensor& t) {
  const Tensor rows = rows16(t);
  return at16(rows) ? rows : rows.clone(at::MemoryFormat::Contiguous);
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
      at16(t))
    return t;
  return token_major(t).copy_(t);
}

void put_strides(int64_t (&to)[3], const Tensor& t) {
  for (int i = 0; i < 3; ++i) to[i] = t.stride(i);
}

void check_attention(const Tensor& q, const Tensor& k, const Tensor& v,
                     const Tensor& lengths) {
  const auto s = q.sizes(), kv = k.sizes();
  expect("attention: q", q,
         s.size() == 4 && q.numel() > 0 && s[0] <= sofa_model::kMaxBlocks &&
             s[1] <= sofa_model::kMaxBlocks && s[2] <= sofa_model::kMaxTokens &&
             s[3] % 8 == 0 && s[3] <= sofa_model::kMaxHeadDim,
         at::kBFloat16, q);
  expect("attention: k", k,
         kv.size() == 4 && kv[0] == s[0] && kv[1] > 0 && s[1] % kv[1] == 0 &&
             kv.slice(2) == s.slice(2),
         at::kBFloat16, q);
  expect("attention: v", v, v.sizes() == kv, at::kBFloat16, q);
  if (lengths.defined())
    expect("attention: lengths", lengths, lengths.sizes() == s.slice(0, 1), at::kInt, q);
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
// twice as many even it out (8 key heads of 128: 8192 tokens 1040 us with two parts
// and 25 to join them, 1810 with one; 2 x 2048 tokens 172 and 23 with four, 462 with
// one). One of less than four steps gains nothing.
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

Tensor attention(const Tensor& q_in, const Tensor& k_in, const Tensor& v_in,
                 const Optional& lengths_in, double scale, bool causal) {
  check_attention(q_in, k_in, v_in, unpack(lengths_in));
  const Tensor o = token_major(q_in);
  if (o.is_meta()) return o;
  // the arguments hold addresses only: copies live until the launch
  const Tensor lengths = dense(unpack(lengths_in));
  const Tensor q = aligned(q_in), k = aligned(k_in), v = aligned(v_in);
  const AttentionArgs a =
      attention_args(q, k, v, o, {}, {}, lengths, scale, causal);
  check(sofa_attention_forward(&a), "attention");
  return o;
}

// with the rest of o and lse, for a backward pass
std::tuple<Tensor, Tensor, Tensor> attention_forward(
    const Tensor& q_in, const Tensor& k_in, const Tensor& v_in,
    const Optional& lengths_in, double scale, bool causal) {
  check_attention(q_in, k_in, v_in, unpack(lengths_in));
  const Tensor o = token_major(q_in), o_low = token_major(q_in);
  const Tensor lse = at::empty({q_in.size(0), q_in.size(1), q_in.size(2)},
                               q_in.options().dtype(at::kFloat));
  if (o.is_meta()) return {o, o_low, lse};
  const Tensor lengths = dense(unpack(lengths_in));
  const Tensor q = aligned(q_in), k = aligned(k_in), v = aligned(v_in);
  const AttentionArgs a =
      attention_args(q, k, v, o, o_low, lse, lengths, scale, causal);
  check(sofa_attention_forward(&a), "attention");
  return {o, o_low, lse};
}

std::tuple<Tensor, Tensor, Tensor> attention_backward(
    const Tensor& dout_in, const Tensor& q_in, const Tensor& k_in,
    const Tensor& v_in, const Tensor& o_in, const Tensor& o_low_in,
    const Tensor& lse_in, const Optional& lengths_in, double scale, bool causal) {
  check_attention(q_in, k_in, v_in, unpack(lengths_in));
  const auto sizes = q_in.sizes();
  for (const Tensor* t : {&dout_in, &o_in, &o_low_in})
    expect("attention: o", *t, t->sizes() == sizes, at::kBFloat16, q_in);
  expect("attention: lse", lse_in, lse_in.sizes() == sizes.slice(0, 3), at::kFloat, q_in);
  const Tensor dq = token_major(q_in), dk = token_major(k_in), dv = token_major(v_in);
  if (dq.is_meta()) return {dq, dk, dv};
  const Tensor q = aligned(q_in), k = aligned(k_in), v = aligned(v_in),
               dout = aligned(dout_in), o = as_token_major(o_in),
               o_low = as_token_major(o_low_in), lse = dense(lse_in),
               lengths = dense(unpack(lengths_in));
  const Tensor delta = at::empty_like(lse);
  AttentionArgs a = attention_args(q, k, v, o, o_low, lse, lengths, scale, causal);
  a.dout = ptr<sofa_model::bf16>(dout);
  a.delta = ptr<float>(delta);
  a.dq = ptr<sofa_model::bf16>(dq);
  a.dk = ptr<sofa_model::bf16>(dk);
  a.dv = ptr<sofa_model::bf16>(dv);
  put_strides(a.dout_stride, dout);
  put_strides(a.dq_stride, dq);
  put_strides(a.dk_stride, dk);
  put_strides(a.dv_stride, dv);
  a.key_parts = key_parts(a.batch, a.heads, a.kv_heads, a.tokens, a.dim, a.causal);
  Tensor partial;
  if (a.key_parts > 1) {
    partial = at::empty({a.key_parts, 2, k.numel()}, q.options().dtype(at::kFloat));
    a.partial = ptr<float>(partial);
  }
  check(sofa_attention_backward(&a), "attention");
  return {dq, dk, dv};
}

struct Attention : torch::autograd::Function<Attention> {
  static Tensor forward(AutogradContext* ctx, const Tensor& q_in,
                        const Tensor& k_in, const Tensor& v_in,
                        const Optional& lengths, double scale, bool causal) {
    const Below below;
    check_attention(q_in, k_in, v_in, unpack(lengths));  // before strides are read
    const Tensor q = rows16(q_in), k = rows16(k_in), v = rows16(v_in);
    const auto [o, o_low, lse] =
        op<&attention_forward>("sofa_model::attention_forward")
            .call(q, k, v, lengths, scale, causal);
    ctx->save_for_backward({q, k, v, o, o_low, lse, unpack(lengths)});
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["causal"] = causal;
    return o;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    variable_list d(6);
    {
      const Below below;
      std::tie(d[0], d[1], d[2]) =
          op<&attention_backward>("sofa_model::attention_backward")
              .call(grads[0], saved[0], saved[1], saved[2], saved[3], saved[4],
                    saved[5], given(saved[6]),
                    ctx->saved_data["scale"].toDouble(),
                    ctx->saved_data["causal"].toBool());
    }
    return first_derivatives(d);
  }
};

Tensor attention_autograd(const Tensor& q, const Tensor& k, const Tensor& v,
                          const Optional& lengths, double scale, bool causal) {
  if (recorded({q, k, v}))
    return Attention::apply(q, k, v, lengths, scale, causal);
  const Below below;
  return op<&attention>("sofa_model::attention").call(q, k, v, lengths, scale, causal);
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

void check_logits(const Tensor& logits, const Tensor& tokens, int64_t top) {
  const int64_t axes = tokens.dim();
  expect("token_logprobs: logits", logits,
         logits.dim() == axes + 1 && logits.numel() > 0 &&
             logits.sizes().slice(0, axes) == tokens.sizes() &&
             logits.size(-1) <= sofa_model::kMaxVocab && top >= 0 &&
             top <= std::min<int64_t>(sofa_model::kMaxTop, logits.size(-1)),
         known_type(logits), logits);
  expect("token_logprobs: tokens", tokens, true, at::kLong, logits);
}

// (log p, entropy, the sums for a backward pass, alternatives if there are any)
std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor> token_logprobs_forward(
    const Tensor& logits_in, const Tensor& tokens_in, int64_t top,
    int64_t ignore_index) {
  check_logits(logits_in, tokens_in, top);
  const auto floats = logits_in.options().dtype(at::kFloat);
  const auto longs = tokens_in.options();
  const auto sizes = tokens_in.sizes();
  const Tensor logprob = at::empty(sizes, floats), entropy = at::empty(sizes, floats),
               norm = at::empty({tokens_in.numel(), 2}, floats);
  Tensor ids, values;
  if (top) {
    std::vector<int64_t> shape = sizes.vec();
    shape.push_back(top);
    ids = at::empty(shape, longs);
    values = at::empty(shape, floats);
  }
  if (logprob.is_meta()) return {logprob, entropy, norm, ids, values};
  const Tensor logits = logit_rows(logits_in);
  Tensor tokens = tokens_in;
  LogprobArgs a = logprob_args(logits, tokens, top, ignore_index);
  Tensor part_sums, part_top;
  if (a.parts > 1) {
    part_sums = at::empty({a.rows, a.parts, 3}, floats);
    if (top) part_top = at::empty({a.rows, a.parts, top}, longs);
  }
  a.logprob = ptr<float>(logprob);
  a.entropy = ptr<float>(entropy);
  a.norm = ptr<float>(norm);
  a.top_ids = ptr<int64_t>(ids);
  a.top_logprobs = ptr<float>(values);
  a.part_sums = ptr<float>(part_sums);
  a.part_top = ptr<uint64_t>(part_top);
  check(sofa_logprob_forward(&a), "token_logprobs");
  return {logprob, entropy, norm, ids, values};
}

std::tuple<Tensor, Tensor> token_logprobs(const Tensor& logits, const Tensor& tokens,
                                          int64_t ignore_index) {
  const auto r = token_logprobs_forward(logits, tokens, 0, ignore_index);
  return {std::get<0>(r), std::get<1>(r)};
}

std::tuple<Tensor, Tensor, Tensor, Tensor> token_logprobs_top(const Tensor& logits,
                                                              const Tensor& tokens,
                                                              int64_t top,
                                                              int64_t ignore_index) {
  TORCH_CHECK(top > 0, "token_logprobs: no alternatives to look for");
  const auto r = token_logprobs_forward(logits, tokens, top, ignore_index);
  return {std::get<0>(r), std::get<1>(r), std::get<3>(r), std::get<4>(r)};
}

Tensor token_logprobs_backward(const Optional& dlogprob, const Optional& dentropy,
                               const Tensor& logits_in, const Tensor& tokens_in,
                               const Tensor& entropy_in, const Tensor& norm_in,
                               int64_t ignore_index) {
  check_logits(logits_in, tokens_in, 0);
  const auto sizes = tokens_in.sizes();
  Tensor g = unpack(dlogprob), h = unpack(dentropy);
  for (const Tensor* t : {&g, &h})
    if (t->defined())
      expect("token_logprobs: a gradient", *t, t->sizes() == sizes, at::kFloat, logits_in);
  expect("token_logprobs: entropy", entropy_in, entropy_in.sizes() == sizes, at::kFloat,
         logits_in);
  expect("token_logprobs: norm", norm_in,
         norm_in.sizes() == at::IntArrayRef{tokens_in.numel(), 2}, at::kFloat, logits_in);
  const Tensor dlogits = at::empty_like(logits_in, at::MemoryFormat::Contiguous);
  if (dlogits.is_meta()) return dlogits;
  const Tensor logits = logit_rows(logits_in), entropy = dense(entropy_in),
               norm = dense(norm_in);
  Tensor tokens = tokens_in;
  LogprobArgs a = logprob_args(logits, tokens, 0, ignore_index);
  const int64_t axes = tokens_in.dim();
  if (g.defined())
    std::tie(g, a.grad_outer_stride, a.grad_inner_stride) =
        same_split(a.inner, a.rows, g, axes);
  if (h.defined())
    std::tie(h, a.grad2_outer_stride, a.grad2_inner_stride) =
        same_split(a.inner, a.rows, h, axes);
  a.logprob = a.entropy = ptr<float>(entropy);
  a.norm = ptr<float>(norm);
  a.dlogprob = ptr<float>(g);
  a.dentropy = ptr<float>(h);
  a.dlogits = ptr(dlogits);
  check(sofa_logprob_backward(&a), "token_logprobs");
  return dlogits;
}

struct TokenLogprobs : torch::autograd::Function<TokenLogprobs> {
  static variable_list forward(AutogradContext* ctx, const Tensor& logits_in,
                               const Tensor& tokens, int64_t top,
                               int64_t ignore_index) {
    const Below below;
    const Tensor logits = logit_rows(logits_in);
    const auto [logprob, entropy, norm, ids, values] =
        op<&token_logprobs_forward>("sofa_model::token_logprobs_forward")
            .call(logits, tokens, top, ignore_index);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({logits, tokens, entropy, norm});
    ctx->saved_data["ignore_index"] = ignore_index;
    if (!top) return {logprob, entropy};
    ctx->mark_non_differentiable({ids, values});
    return {logprob, entropy, ids, values};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list d(4);
    if (!grads[0].defined() && !grads[1].defined()) return d;
    const variable_list saved = ctx->get_saved_variables();
    {
      const Below below;
      d[0] = op<&token_logprobs_backward>("sofa_model::token_logprobs_backward")
                 .call(given(grads[0]), given(grads[1]), saved[0], saved[1], saved[2],
                       saved[3], ctx->saved_data["ignore_index"].toInt());
    }
    return first_derivatives(d);
  }
};

std::tuple<Tensor, Tensor> token_logprobs_autograd(const Tensor& logits,
                                                   const Tensor& tokens,
                                                   int64_t ignore_index) {
  if (recorded({logits})) {
    const variable_list r = TokenLogprobs::apply(logits, tokens, 0, ignore_index);
    return {r[0], r[1]};
  }
  const Below below;
  return op<&token_logprobs>("sofa_model::token_logprobs").call(logits, tokens, ignore_index);
}

std::tuple<Tensor, Tensor, Tensor, Tensor> token_logprobs_top_autograd(
    const Tensor& logits, const Tensor& tokens, int64_t top, int64_t ignore_index) {
  if (recorded({logits})) {
    TORCH_CHECK(top > 0, "token_logprobs: no alternatives to look for");
    const variable_list r = TokenLogprobs::apply(logits, tokens, top, ignore_index);
    return {r[0], r[1], r[2], r[3]};
  }
  const Below below;
  return op<&token_logprobs_top>("sofa_model::token_logprobs_top")
      .call(logits, tokens, top, ignore_index);
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

void check_norm(const Tensor& x, const Tensor& branch, at::ScalarType branch_type,
                const Tensor& weight, const Tensor& post, const Tensor& gate) {
  const int64_t dim = x.dim() ? x.size(-1) : 0;
  expect("residual_norm: x", x, x.numel() > 0 && dim <= sofa_model::kMaxNormDim,
         known_type(x), x);
  if (branch.defined())
    expect("residual_norm: branch", branch, branch.sizes() == x.sizes(), branch_type, x);
  expect("residual_norm: weight", weight, weight.sizes() == dim, known_type(weight), x);
  if (post.defined())
    expect("residual_norm: post_weight", post, post.sizes() == dim, known_type(post), x);
  if (gate.defined())
    expect("residual_norm: gate", gate,
           gate.sizes() == dim ||
               (gate.dim() == x.dim() && gate.size(-1) == dim &&
                gate.size(0) == x.size(0) && gate.numel() == x.size(0) * dim),
           known_type(gate), x);
}

// (r, y); r is not there without a branch, whose type then only chooses a kernel
std::pair<Tensor, Tensor> norm_forward(const Tensor& x_in, const Tensor& branch_in,
                                       const Tensor& weight_in, const Tensor& post_in,
                                       const Tensor& gate_in, double scale,
                                       double eps, at::ScalarType y_type) {
  const auto branch_type = branch_in.defined() ? known_type(branch_in) : known(y_type);
  check_norm(x_in, branch_in, branch_type, weight_in, post_in, gate_in);
  const Tensor x = dense(x_in);
  const Tensor y = at::empty_like(x, x.options().dtype(known(y_type)));
  const Tensor r = branch_in.defined() ? at::empty_like(x) : Tensor();
  if (y.is_meta()) return {r, y};
  const Tensor branch = dense(branch_in), weight = dense(weight_in),
               post = dense(post_in), gate = dense(gate_in);
  NormArgs a = norm_args(x, branch, weight, post, gate, scale, eps, branch_type, y_type);
  a.r = ptr(r);
  a.y = ptr(y);
  check(sofa_norm_forward(&a), "residual_norm");
  return {r, y};
}

std::tuple<Tensor, Tensor> residual_norm(const Tensor& x, const Tensor& branch,
                                         const Tensor& weight, const Optional& post,
                                         const Optional& gate, double scale,
                                         double eps, at::ScalarType y_type) {
  return norm_forward(x, branch, weight, unpack(post), unpack(gate), scale, eps, y_type);
}

// without a branch
Tensor rms_norm(const Tensor& x, const Tensor& weight, double eps, at::ScalarType y_type) {
  return norm_forward(x, {}, weight, {}, {}, 1., eps, y_type).second;
}

// `x`: r where that is held in 32 bits. `needed`: bits, in the order of the
// results; those not needed are not there.
std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor> residual_norm_backward(
    const Optional& dr_in, const Optional& dy_in, const Tensor& x_in,
    const Optional& branch_in, const Tensor& weight_in, const Optional& post_in,
    const Optional& gate_in, double scale, double eps, at::ScalarType branch_type,
    at::ScalarType y_type, int64_t needed) {
  check_norm(x_in, unpack(branch_in), known(branch_type), weight_in, unpack(post_in),
             unpack(gate_in));
  const Tensor x = dense(x_in), weight = dense(weight_in), post = dense(unpack(post_in)),
               gate = dense(unpack(gate_in)), branch = dense(unpack(branch_in)),
               dr = dense(unpack(dr_in)), dy = dense(unpack(dy_in));
  TORCH_CHECK(dr.defined() || dy.defined(), "residual_norm: a gradient is needed");
  TORCH_CHECK((post.defined() || !(needed & 8)) && (gate.defined() || !(needed & 16)),
              "residual_norm: no gradient of what is not there");
  if (dr.defined())
    expect("residual_norm: dr", dr, dr.sizes() == x.sizes(), x.scalar_type(), x);
  if (dy.defined()) expect("residual_norm: dy", dy, dy.sizes() == x.sizes(), known(y_type), x);
  const Tensor dx = at::empty_like(x);
  Tensor dbranch, dweight, dpost, dgate, partial;
  if (needed & 2) dbranch = at::empty_like(x, x.options().dtype(branch_type));
  if (needed & 4) dweight = at::empty_like(weight);
  if (needed & 8) dpost = at::empty_like(post);
  if (needed & 16) dgate = at::empty_like(gate);
  const Tensor first = needed & 1 ? dx : Tensor();
  if (dx.is_meta()) return {first, dbranch, dweight, dpost, dgate};
  NormArgs a = norm_args(x, branch, weight, post, gate, scale, eps, branch_type, y_type);
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
  return {first, dbranch, dweight, dpost, dgate};
}

struct ResidualNorm : torch::autograd::Function<ResidualNorm> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x,
                               const Optional& branch_in,
                               const Tensor& weight, const Optional& post_in,
                               const Optional& gate_in, double scale, double eps,
                               at::ScalarType y_type) {
    const Below below;
    const Tensor branch = unpack(branch_in), post = unpack(post_in),
                 gate = unpack(gate_in);
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
    if (!branch.defined()) {
      ctx->save_for_backward({x, {}, weight, post, gate});
      return {op<&rms_norm>("sofa_model::rms_norm").call(x, weight, eps, y_type)};
    }
    const auto [r, y] = op<&residual_norm>("sofa_model::residual_norm")
                            .call(x, branch, weight, post_in, gate_in, scale, eps, y_type);
    // a 32-bit sum is kept, one rounded to 16 bits is computed again
    const bool keep = x.scalar_type() == at::kFloat;
    const bool uses_branch = !keep || post.defined() || gate.defined();
    ctx->save_for_backward(
        {keep ? r : x, uses_branch ? branch : Tensor(), weight, post, gate});
    return {y, r};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list d(8);
    const Tensor dr = grads.size() > 1 ? grads[1] : Tensor();
    if (!dr.defined() && !grads[0].defined()) return d;
    const variable_list saved = ctx->get_saved_variables();
    {
      const Below below;
      std::tie(d[0], d[1], d[2], d[3], d[4]) =
          op<&residual_norm_backward>("sofa_model::residual_norm_backward")
              .call(given(dr), given(grads[0]), saved[0], given(saved[1]), saved[2],
                    given(saved[3]), given(saved[4]),
                    ctx->saved_data["scale"].toDouble(),
                    ctx->saved_data["eps"].toDouble(),
                    (at::ScalarType) ctx->saved_data["branch_type"].toInt(),
                    (at::ScalarType) ctx->saved_data["y_type"].toInt(),
                    ctx->saved_data["needed"].toInt());
    }
    return first_derivatives(d);
  }
};

std::tuple<Tensor, Tensor> residual_norm_autograd(
    const Tensor& x, const Tensor& branch, const Tensor& weight, const Optional& post,
    const Optional& gate, double scale, double eps, at::ScalarType y_type) {
  if (recorded({x, branch, weight, unpack(post), unpack(gate)})) {
    const variable_list out = ResidualNorm::apply(
        dense(x), Optional(dense(branch)), dense(weight), given(dense(unpack(post))),
        given(dense(unpack(gate))), scale, eps, y_type);
    return {out[1], out[0]};
  }
  const Below below;
  return op<&residual_norm>("sofa_model::residual_norm")
      .call(x, branch, weight, post, gate, scale, eps, y_type);
}

Tensor rms_norm_autograd(const Tensor& x, const Tensor& weight, double eps,
                         at::ScalarType y_type) {
  if (recorded({x, weight}))
    return ResidualNorm::apply(dense(x), Optional(), dense(weight), Optional(), Optional(),
                               1., eps, y_type)[0];
  const Below below;
  return op<&rms_norm>("sofa_model::rms_norm").call(x, weight, eps, y_type);
}

void implement(torch::Library& m) {
  m.impl("attention", &attention);
  m.impl("attention_forward", &attention_forward);
  m.impl("attention_backward", &attention_backward);
  m.impl("token_logprobs", &token_logprobs);
  m.impl("token_logprobs_top", &token_logprobs_top);
  m.impl("token_logprobs_forward", &token_logprobs_forward);
  m.impl("token_logprobs_backward", &token_logprobs_backward);
  m.impl("residual_norm", &residual_norm);
  m.impl("rms_norm", &rms_norm);
  m.impl("residual_norm_backward", &residual_norm_backward);
}

TORCH_LIBRARY(sofa_model, m) {
  m.def("attention(Tensor q, Tensor k, Tensor v, Tensor? lengths, float scale, bool causal) "
        "-> Tensor");
  m.def("attention_forward(Tensor q, Tensor k, Tensor v, Tensor? lengths, float scale, "
        "bool causal) -> (Tensor o, Tensor o_low, Tensor lse)");
  m.def("attention_backward(Tensor dout, Tensor q, Tensor k, Tensor v, Tensor o, "
        "Tensor o_low, Tensor lse, Tensor? lengths, float scale, bool causal) "
        "-> (Tensor dq, Tensor dk, Tensor dv)");
  m.def("token_logprobs(Tensor logits, Tensor tokens, int ignore_index) "
        "-> (Tensor logprob, Tensor entropy)");
  m.def("token_logprobs_top(Tensor logits, Tensor tokens, int top, int ignore_index) "
        "-> (Tensor logprob, Tensor entropy, Tensor ids, Tensor values)");
  m.def("token_logprobs_forward(Tensor logits, Tensor tokens, int top, int ignore_index) "
        "-> (Tensor logprob, Tensor entropy, Tensor norm, Tensor ids, Tensor values)");
  m.def("token_logprobs_backward(Tensor? dlogprob, Tensor? dentropy, Tensor logits, "
        "Tensor tokens, Tensor entropy, Tensor norm, int ignore_index) -> Tensor");
  m.def("residual_norm(Tensor x, Tensor branch, Tensor weight, Tensor? post_weight, "
        "Tensor? gate, float scale, float eps, ScalarType out_dtype) -> (Tensor r, Tensor y)");
  m.def("rms_norm(Tensor x, Tensor weight, float eps, ScalarType out_dtype) -> Tensor");
  m.def("residual_norm_backward(Tensor? dr, Tensor? dy, Tensor x, Tensor? branch, "
        "Tensor weight, Tensor? post_weight, Tensor? gate, float scale, float eps, "
        "ScalarType branch_dtype, ScalarType out_dtype, int needed) -> (Tensor dx, "
        "Tensor dbranch, Tensor dweight, Tensor dpost, Tensor dgate)");
}

TORCH_LIBRARY_IMPL(sofa_model, CUDA, m) { implement(m); }
TORCH_LIBRARY_IMPL(sofa_model, Meta, m) { implement(m); }

TORCH_LIBRARY_IMPL(sofa_model, Autograd, m) {
  m.impl("attention", &attention_autograd);
  m.impl("token_logprobs", &token_logprobs_autograd);
  m.impl("token_logprobs_top", &token_logprobs_top_autograd);
  m.impl("residual_norm", &residual_norm_autograd);
  m.impl("rms_norm", &rms_norm_autograd);
}

}  // namespace

PYBIND11_MODULE(sofa_model, m) {
  m.def("attention", [](const Tensor& q, const Tensor& k, const Tensor& v,
                        const Optional& lengths, double scale, bool causal) {
    return op<&attention>("sofa_model::attention").call(q, k, v, lengths, scale, causal);
  });
  m.def("token_logprobs", [](const Tensor& logits, const Tensor& tokens,
                             int64_t ignore_index) {
    return op<&token_logprobs>("sofa_model::token_logprobs")
        .call(logits, tokens, ignore_index);
  });
  m.def("token_logprobs_top", [](const Tensor& logits, const Tensor& tokens, int64_t top,
                                 int64_t ignore_index) {
    return op<&token_logprobs_top>("sofa_model::token_logprobs_top")
        .call(logits, tokens, top, ignore_index);
  });
  m.def("residual_norm", [](const Tensor& x, const Tensor& branch, const Tensor& weight,
                            const Optional& post, const Optional& gate, double scale,
                            double eps, const py::object& y_type) {
    return op<&residual_norm>("sofa_model::residual_norm")
        .call(x, branch, weight, post, gate, scale, eps,
              torch::python::detail::py_object_to_dtype(y_type));
  });
  m.def("rms_norm", [](const Tensor& x, const Tensor& weight, double eps,
                       const py::object& y_type) {
    return op<&rms_norm>("sofa_model::rms_norm")
        .call(x, weight, eps, torch::python::detail::py_object_to_dtype(y_type));
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
